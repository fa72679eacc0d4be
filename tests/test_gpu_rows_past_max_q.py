"""A request with more rows than max_q: its first max_q rows and all rows of the
batch's other requests are computed, whichever kernel max_q leads to."""
import random

import pytest

from tests import drafts_ref
from tests.attn_ref import U, check
from tests.test_gpu_attention import counters_clear, gen, i32
from tests.test_gpu_attention_q8 import dev, make_cache as cache8  # noqa: F401
from tests.test_gpu_drafts import cu_of, make_cache as cache16, signed, tree_masks
from tests.test_gpu_idle_requests import attend
from tests.test_gpu_parity import note
from tests import q8_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,tree", [(8, False), (8, True), (16, False), (16, True)])
@pytest.mark.parametrize("Hq,Hkv", [(16, 2), (40, 8), (8, 1)])
@pytest.mark.parametrize("max_q", [1, 2, 3, 4, 6])
@pytest.mark.parametrize("ctx", [40, 1500])
def test_rows_past_max_q(dev, bits, tree, Hq, Hkv, max_q, ctx):  # noqa: F811
    import torch
    from inferflux_amd import attention as at
    note(f"past max_q={max_q} {bits} bits tree={tree} {Hq}/{Hkv} {ctx}")
    D, P = 128, 16
    new = [40, 1, 0, max_q, 63, 1, max_q, max_q]
    ctx = [ctx, 3, 70, 0, 5, 90, 33, ctx]
    rng = random.Random(max_q + Hq)
    kv = [c + n for c, n in zip(ctx, new)]
    if bits == 8:
        cache, table, slots = cache8(dev, ctx, new, Hkv, D, P, 7)
        rows = [q8_ref.get(cache, s) for s in slots]
    else:
        *cache, table, rows = cache16(dev, torch.float16, ctx, new, Hkv, D, P, 7)
    T = sum(new)
    q = torch.randn(T, Hq, D, generator=gen(dev, 8), device=dev).half()
    bits_of = tree_masks(rng, new)
    masks = torch.tensor([signed(m) for m in bits_of], device=dev) if tree else None
    out, ws = torch.full_like(q, 7.0), at.workspace(dev)
    attend(dev, cache, table, q, kv, new, masks, max_q, max(kv), ws, out=out)
    t = 0
    for b, n in enumerate(new):
        if n:
            some = min(n, max_q)
            if tree:
                seen = drafts_ref.seen_by_tree(bits_of[t:t + n], ctx[b], n, kv[b])[:some]
            else:
                seen = torch.arange(kv[b]) <= ctx[b] + torch.arange(some)[:, None]
            k, v = rows[b][:2]
            want, bound = drafts_ref.attend_seen(q[t:t + some], k, v, seen, D ** -0.5, weigh=U[torch.float16])
            if bits == 8:  # fp16 of probability times V's scale, as in the attention's own tests
                bound = bound + kv[b] * 2.0 ** -30 * 127 * float(rows[b][2].amax())
            check(out[t:t + some], want, bound, f"request {b} of {n} rows")
        t += n
    assert counters_clear(ws)
