"""Batches in which requests have no new tokens, first, last and all of them: the
others' outputs are those of the batch without them, bit for bit, from rows of Q and
masks that are exactly as many as the batch has."""
import random

import pytest

from tests.test_gpu_attention import counters_clear, gen, i32
from tests.test_gpu_attention_q8 import dev, make_cache as cache8  # noqa: F401
from tests.test_gpu_drafts import cu_of, make_cache as cache16, signed, tree_masks
from tests.test_gpu_parity import note

pytestmark = pytest.mark.gpu


def attend(dev, cache, table, q, kv, new, masks, max_q, max_kv, ws, out=None):  # noqa: F811
    from inferflux_amd import attention as at, attention_q8 as q8, drafts
    args = table, i32(cu_of(new), dev), i32(kv, dev)
    if len(cache) == 3:
        return q8.paged_attention(q, cache, *args, max_q, max_kv, masks=masks, workspace=ws, out=out)
    if masks is None:
        return at.paged_attention(q, *cache, *args, max_q, max_kv, workspace=ws, out=out)
    return drafts.tree_attention(q, *cache, *args, masks, max_q, max_kv, workspace=ws, out=out)


# Many rows, a block each among row tiles; up to 16 and 32 rows; blocks of rows; more
# requests than lanes.  Long enough that idle requests do not change how many chunks
# there are room for.
BATCHES = {
    "mixed": ([9000, 3000, 40, 700, 129], [1, 60, 33, 2, 50]),
    "few": ([9000, 3000, 40, 700], [3, 1, 2, 3]),
    "rows": ([9000, 3000, 40, 700], [5, 1, 4, 6]),
    "blocks": ([9000, 3000, 40, 700, 129], [13, 7, 2, 1, 5]),
    "crowd": ([9000] + [i * 37 % 900 for i in range(69)], [64] + [(1, 2, 40)[i % 3] for i in range(69)]),
}


@pytest.mark.parametrize("where", ["first", "last", "both", "between"])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("what", BATCHES)
@pytest.mark.parametrize("bits", [8, 16])
def test_idle_requests(dev, bits, what, tree, where):  # noqa: F811
    import torch
    from inferflux_amd import attention as at
    note(f"idle {bits} bits {what} tree={tree} {where}")
    Hq, Hkv, D, P = 40, 8, 128, 16
    ctx, new = BATCHES[what]
    if bits == 16 and tree and what == "blocks":  # as few units as have blocks of rows there
        Hq, Hkv = 10, 2
    if where == "between":
        at_, idle = [x for b in range(len(ctx)) for x in (b, None)], len(ctx)
    else:
        at_ = [None] * (where != "last") + list(range(len(ctx))) + [None] * (where != "first")
        idle = at_.count(None)
    rng = random.Random(len(ctx) + idle)
    kv = [0 if b is None else ctx[b] + new[b] for b in at_]
    idle_kv = [rng.choice([0, 50, 1000]) if b is None else k for b, k in zip(at_, kv)]
    n_all = [0 if b is None else new[b] for b in at_]
    if bits == 8:
        cache, table, _ = cache8(dev, [k - n for k, n in zip(idle_kv, n_all)], n_all, Hkv, D, P, 3)
    else:
        *cache, table, _ = cache16(dev, torch.float16, [k - n for k, n in zip(idle_kv, n_all)], n_all, Hkv, D, P, 3)
    T = sum(new)
    q = torch.randn(T, Hq, D, generator=gen(dev, 5), device=dev).half()
    masks = torch.tensor([signed(m) for m in tree_masks(rng, new)], device=dev) if tree else None
    ws = at.workspace(dev)
    got = attend(dev, cache, table, q, idle_kv, n_all, masks, max(new), max(kv), ws)
    some = [i for i, b in enumerate(at_) if b is not None]
    want = attend(dev, cache, table[some].contiguous(), q, [kv[i] for i in some], new, masks, max(new), max(kv), ws)
    assert torch.isfinite(want).all() and torch.equal(got, want)
    assert counters_clear(ws)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("max_q", [1, 6, 13, 64])
@pytest.mark.parametrize("B", [2, 5, 70])
def test_a_plan_that_failed(dev, bits, max_q, B):  # noqa: F811
    """cu_q all 0 and lengths left at the context, as plan_batch leaves them: nothing
    is written, and the workspace serves the next call."""
    import torch
    from inferflux_amd import attention as at
    note(f"failed plan {bits} bits max_q={max_q} B={B}")
    Hq, Hkv, D, P, T = 40, 8, 128, 16, 64
    ctx = [(3000, 1, 500, 0, 64)[b % 5] for b in range(B)]
    if bits == 8:
        cache, table, _ = cache8(dev, ctx, [0] * B, Hkv, D, P, 4)
    else:
        *cache, table, _ = cache16(dev, torch.float16, ctx, [0] * B, Hkv, D, P, 4)
    q = torch.randn(T, Hq, D, generator=gen(dev, 6), device=dev).half()
    masks = torch.full((T,), -1, device=dev)
    ws = at.workspace(dev)
    for m in (masks, None):
        out = torch.full_like(q, 7.0)
        attend(dev, cache, table, q, ctx, [0] * B, m, max_q, 3000, ws, out=out)
        assert torch.all(out == 7.0) and counters_clear(ws)
