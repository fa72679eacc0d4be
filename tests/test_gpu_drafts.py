"""Drafted tokens on the GPU against their plain forms (tests/drafts_ref.py):
trees' positions and masks, the attention of their nodes, verification, and
what the cache keeps, alone and as a serving step runs them."""
import math
import random

import pytest

from tests import drafts_ref as ref
from tests.attn_ref import check, gather_cache, put_cache
from tests.test_gpu_attention import dt_of, gen, i32
from tests.test_gpu_parity import note

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from inferflux_amd import _lib
    _lib.load()  # raises if the HIP library is missing: no fallback exists
    return torch.device("cuda:0")


def cu_of(new):
    return [sum(new[:i]) for i in range(len(new) + 1)]


def signed(m):
    return m - (1 << 64) if m >> 63 else m


# ---------------------------------------------------------------------- plans
@pytest.mark.parametrize("B,hi,extra,wild", [(1, 1, 0, False), (1, 64, 3, False), (5, 9, 0, True), (40, 64, 1, True),
                                             (3, 100, 2, False), (300, 7, 0, False), (2, 64, 0, True)])
def test_plan_tree(dev, B, hi, extra, wild):
    from inferflux_amd import drafts
    note(f"plan_tree B={B} hi={hi}")
    rng = random.Random(B * 7 + hi)
    new = [hi] + [rng.choice([0, 1, hi, rng.randint(1, hi)]) for _ in range(B - 1)]
    ctx = [rng.randint(0, 5000) for _ in new]
    trees = [ref.tree(rng, n, rng.choice([1, 3, 64])) if n else [] for n in new]
    if wild:  # numbers that are no earlier row: no parent
        for t in trees:
            for j in range(len(t)):
                if rng.random() < 0.3:
                    t[j] = rng.choice([-1, -9, j, j + 1, 1 << 30, -(1 << 31)])
    positions, masks = [], []
    for c, t in zip(ctx, trees):
        for i, way in enumerate(ref.ways(t)):
            positions.append(c + len(way) - 1 if i < 64 else 0)
            masks.append(signed(sum(1 << j for j in way)) if i < 64 else 0)
    gap = [0] * extra
    p = drafts.plan_tree(i32(sum(trees, []) + [5] * extra, dev), i32(cu_of(new), dev),
                         i32([c + n for c, n in zip(ctx, new)], dev))
    assert p.positions.tolist() == positions + gap
    assert p.masks.tolist() == masks + gap


@pytest.mark.parametrize("B,P,hi,full", [(1, 16, 5, False), (7, 16, 64, False), (33, 64, 40, False), (300, 16, 20, False),
                                         (4096, 16, 3, False), (5, 16, 40, True)])
def test_plan_kept(dev, B, P, hi, full):
    """A plan, taken back but for what is kept: the next plan gets the same pages."""
    import torch
    from inferflux_amd import attention as at, drafts
    note(f"plan_kept B={B} P={P}")
    rng = random.Random(B + P)
    ctx = [rng.randint(0, 3 * P) for _ in range(B)]
    new = ref.rand_lengths(rng, B, hi)
    held = [-(-c // P) for c in ctx]
    total = [-(-(c + n) // P) for c, n in zip(ctx, new)]
    pages = list(range(sum(total) + 3))
    rng.shuffle(pages)
    W, at0, table = max(total) + 1, 0, []
    for h in held:
        table.append(pages[at0:at0 + h] + [-1] * (W - h))
        at0 += h
    free = pages[at0:]
    t, f = i32(table, dev), i32(free, dev)
    p = at.plan_batch(i32(ctx, dev), i32(new, dev), t, f, i32([len(free)], dev), P, sum(new))
    assert int(p.status) == 0
    accepted = [rng.choice([-1, 0, n - 1, rng.randint(0, n), n + 5]) if n else rng.choice([-1, 3]) for n in new]
    keep = [c + (min(a + 1, n) if n else 0) for c, a, n in zip(ctx, accepted, new)]
    give = [-(-(c + n) // P) - -(-k // P) for c, n, k in zip(ctx, new, keep)]
    left = int(p.free_left)
    stack = f.tolist()[:left]
    now = t.tolist()
    for b in reversed(range(B)):
        last = -(-(ctx[b] + new[b]) // P)
        stack += [now[b][last - 1 - i] for i in range(give[b])]
    if full:  # room for all but one
        f = f[:left + sum(give) - 1].contiguous()
        before = f.clone()
    r = drafts.plan_kept(p.cu_q, p.kv_len, i32(accepted, dev), t, f, p.free_left, P)
    assert r.ctx_len.tolist() == keep and t.tolist() == now
    if full:
        assert int(r.status) == drafts.NO_SPACE and int(r.free_left) == left and torch.equal(f, before)
        return
    assert int(r.status) == 0 and int(r.free_left) == len(stack) and f.tolist()[:len(stack)] == stack
    if keep == ctx:
        assert f.tolist() == free


# ------------------------------------------------------------------ attention
def make_cache(dev, dtype, ctx, new, Hkv, D, P, seed, extra=3):
    """Cache, table and per request K, V [ctx + n, Hkv, D]; unwritten slots NaN."""
    import torch
    from inferflux_amd import attention as at
    g = gen(dev, seed)
    total = [-(-max(c + n, 0) // P) for c, n in zip(ctx, new)]
    order = torch.randperm(sum(total) + extra, generator=g, device=dev).int()
    k, v = at.kv_cache(sum(total) + extra, Hkv, D, P, dtype=dtype, device=dev)
    k.fill_(math.nan), v.fill_(math.nan)
    W = max(total) + 1
    table = torch.full((len(ctx), W), -5, dtype=torch.int32, device=dev)
    used, rows = 0, []
    for b, (c, n) in enumerate(zip(ctx, new)):
        table[b, :total[b]] = order[used:used + total[b]]
        used += total[b]
        x = torch.randn(2, max(c + n, 0), Hkv, D, generator=g, device=dev).to(dtype)
        rows.append((x[0], x[1]))
        if c + n > 0:
            put_cache(k, v, table[b], x[0], x[1])
    return k, v, table, rows


def run_tree(dev, dtype, ctx, new, masks, Hq, Hkv, D, P, seed=1, spoil=None, out_dtype=None, scale=None,
             max_kv=None, workspace=None):
    """tree_attention of requests with masks (integers, row by row) against 64 bits."""
    import torch
    from inferflux_amd import attention as at, drafts
    dtype = dt_of(dtype)
    k, v, table, rows = make_cache(dev, dtype, ctx, new, Hkv, D, P, seed)
    if spoil:
        spoil(k, v, table, rows)
    T = sum(new)
    q = torch.randn(T + 2, Hq, D, generator=gen(dev, seed + 1), device=dev).to(dtype)
    kv = [max(c + n, 0) for c, n in zip(ctx, new)]
    out = torch.full((T + 2, Hq, D), 7.0, dtype=out_dtype or dtype, device=dev)
    ws = at.workspace(dev) if workspace is None else workspace
    scale = scale or 1.5 * D ** -0.5
    m = torch.tensor([signed(x) for x in masks] + [-1, -1], device=dev)
    drafts.tree_attention(q, k, v, table, i32(cu_of(new), dev), i32(kv, dev), m, max(max(new), 1),
                          max_kv or max(max(kv), 1), scale=scale, out=out, workspace=ws)
    t = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        if n:
            seen = ref.seen_by_tree(masks[t:t + n], c, n, kv[b])
            kk, vv = gather_cache(k, v, table[b], kv[b]) if spoil else rows[b]
            want, bound = ref.attend_seen(q[t:t + n], kk, vv, seen, scale)
            check(out[t:t + n], want, bound, f"request {b}")
        t += n
    assert torch.all(out[T:] == 7.0), "rows behind the last request"
    assert not ws[:32768].any(), "counters left"
    return out


def tree_masks(rng, new, reach=4):
    return [sum(1 << j for j in way) for n in new for way in ref.ways(ref.tree(rng, n, reach) if n else [])]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,D,P", [(16, 2, 128, 64), (40, 8, 128, 16), (6, 6, 64, 32), (9, 3, 96, 16), (8, 2, 256, 128),
                                        (7, 1, 128, 256)])
@pytest.mark.parametrize("shape", ["one", "few", "wide", "mixed", "crowd"])
def test_tree_attention(dev, dtype, Hq, Hkv, D, P, shape):
    note(f"tree {dtype} {Hq}/{Hkv} D={D} P={P} {shape}")
    rng = random.Random(Hq * 131 + D + P + len(shape))
    ctx, new = {"one": ([1700], [3]), "few": ([0, 5, 300, 64], [4, 1, 3, 4]), "wide": ([700, 63], [64, 33]),
                "mixed": ([900, 0, 17, 130, 64], [1, 20, 0, 61, 7]),
                "crowd": ([rng.randint(0, 400) for _ in range(34)], [rng.choice([1, 2, 40]) for _ in range(33)] + [40])}[shape]
    run_tree(dev, dtype, ctx, new, tree_masks(rng, new), Hq, Hkv, D, P, seed=D + P)


@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 128), (16, 2, 64)])
@pytest.mark.parametrize("ctx", [[0, 0], [-3, 40], [-70, -64], [1000, 1]])
def test_tree_masks_of_any_kind(dev, Hq, Hkv, D, ctx):
    """Rows that see nothing, not themselves, later rows, bits past the last
    row; requests with fewer tokens than rows."""
    note(f"tree any {Hq}/{Hkv} D={D} {ctx}")
    rng = random.Random(D + ctx[0])
    for n in (3, 12, 64):
        masks = [rng.choice([0, 0, 1 << rng.randrange(64), rng.getrandbits(64)]) for _ in range(2 * n)]
        run_tree(dev, "f16", ctx, [n, n], masks, Hq, Hkv, D, 16, seed=n)


@pytest.mark.parametrize("n,Hq,Hkv", [(1, 4, 4), (6, 4, 2), (40, 16, 2)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_tree_unseen_values_have_no_influence(dev, n, Hq, Hkv, bad):
    """Nodes whose K and V are not finite: only rows that see them are hit."""
    import torch
    note(f"tree spoilt n={n} {bad}")
    rng = random.Random(n)
    ctx, new, P = [130, 61], [n, n], 16
    masks = tree_masks(rng, new, 6)
    if n == 1:
        masks = [0, 1]

    def spoil(k, v, table, rows):
        for b in range(2):
            for j in {0, n // 2, n - 1} - ({0} if n > 1 else set()):
                t = ctx[b] + j
                page, at = int(table[b, t // P]), t % P
                v[page, :, at // 8, 3:9, at % 8] = bad
                if bad == math.nan:
                    k[page, :, :, at] = bad
    out = run_tree(dev, "bf16", ctx, new, masks, Hq, Hkv, 128, P, spoil=spoil)
    assert torch.isfinite(out[:n]).any()


def test_tree_split_sums_and_chain_as_paged(dev):
    """Long contexts cut into chunks, twice the same bits; a chain's masks and
    paged_attention have the same definition.  (Their bits may differ: a stage of
    keys that all later rows see whole is one seen in part for a tree, and the
    two add a row's weights in different orders.)"""
    import torch
    from inferflux_amd import attention as at, drafts
    for n, Hq, Hkv in ((4, 16, 2), (60, 16, 2)):
        note(f"tree split n={n}")
        ctx, new = [9000, 300], [n, n]
        rng = random.Random(n)
        ws = at.workspace(dev)
        masks = tree_masks(rng, new)
        a = run_tree(dev, "f16", ctx, new, masks, Hq, Hkv, 128, 64, workspace=ws)
        b = run_tree(dev, "f16", ctx, new, masks, Hq, Hkv, 128, 64, workspace=ws)
        assert torch.equal(a, b)
        k, v, table, rows = make_cache(dev, torch.float16, ctx, new, Hkv, 128, 64, 3)
        q = torch.randn(2 * n, Hq, 128, generator=gen(dev, 4), device=dev).half()
        cu, kv = i32(cu_of(new), dev), i32([c + n for c in ctx], dev)
        t = drafts.plan_tree(i32(2 * list(range(-1, n - 1)), dev), cu, kv)
        x = drafts.tree_attention(q, k, v, table, cu, kv, t.masks, n, 9100, workspace=ws)
        y = at.paged_attention(q, k, v, table, cu, kv, n, 9100, workspace=ws)
        for i in range(2):
            seen = ref.seen_by_tree([(2 << j) - 1 for j in range(n)], ctx[i], n, ctx[i] + n)
            want, bound = ref.attend_seen(q[i * n:i * n + n], *rows[i], seen, 128 ** -0.5)
            check(x[i * n:i * n + n], want, bound, "masks")
            check(y[i * n:i * n + n], want, bound, "paged")


# --------------------------------------------------------------- verification
def run_verify(dev, new, parents, tokens, p, au, su, q=None, max_q=64, dtype="f32", pad=0, behind=0):
    """p, q: float32 tensors [T, V] on the device."""
    import torch
    from inferflux_amd import attention as at, drafts
    T, V = p.shape
    dt = dt_of(dtype)

    def strided(x):
        buf = torch.full((T, V + pad), math.nan, dtype=dt, device=dev)
        buf[:, :V] = x.to(dt)
        return buf[:, :V]
    ps, qs = strided(p), None if q is None else strided(q)
    cu = cu_of(new)
    ws = at.workspace(dev)
    out = drafts.Verified(*(torch.full((n + behind,), 77, dtype=torch.int32, device=dev)
                            for n in (len(new), T, T)))
    f32 = lambda x: torch.tensor(x, dtype=torch.float32, device=dev)  # noqa: E731
    au, su = f32(au), f32(su)
    drafts.verify(i32(tokens, dev), i32(cu, dev), ps, au, su, max_q,
                  parents=None if parents is None else i32(parents, dev), draft_probs=qs, out=out, workspace=ws)
    want = ref.verify(parents, tokens, cu, ps.float().cpu().tolist(), au.tolist(), su.tolist(),
                      None if q is None else qs.float().cpu().tolist(), max_q)
    n = cu[-1]
    got = (out.accepted.tolist()[:len(new)], out.path.tolist()[:n], out.emitted.tolist()[:n])
    assert got[0] == want[0], "accepted"
    assert got[1] == want[1], "path"
    assert got[2] == want[2], "emitted"
    assert out.path.tolist()[n:] == [77] * (T + behind - n) and out.accepted.tolist()[len(new):] == [77] * behind
    assert not ws[:32768].any(), "counters left"
    return got


def draws(rng, n):
    """Numbers as a generator gives them: 24 bits, 0 among them."""
    return [rng.choice([0.0, rng.randrange(1 << 24) / (1 << 24), rng.randrange(1 << 24) / (1 << 24)]) for _ in range(n)]


def top_tokens(rng, p, new, trees):
    """The parent's most likely tokens, a child each; some the same, some none."""
    tokens, at = [], 0
    best = p.topk(min(8, p.shape[1]), 1).indices.tolist()
    for n, t in zip(new, trees):
        for j in range(n):
            x = rng.choice(best[at + t[j]]) if 0 <= t[j] < j else 0
            tokens.append(rng.choice([x] * 12 + [-1, p.shape[1], rng.randrange(p.shape[1])]))
        at += n
    return tokens


@pytest.mark.parametrize("V,B,hi", [(1, 3, 4), (3, 20, 9), (5, 6, 64), (1000, 40, 20), (1025, 3, 64), (4099, 9, 30),
                                    (33000, 2, 12), (151936, 1, 6)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_verify_trees(dev, V, B, hi, dtype):
    import torch
    note(f"verify trees V={V} B={B} {dtype}")
    rng = random.Random(V + B)
    new = [hi] + ref.rand_lengths(rng, B - 1, hi)
    trees = [ref.tree(rng, n) if n else [] for n in new]
    for t in trees:
        for j in range(len(t)):
            if rng.random() < 0.05:
                t[j] = rng.choice([-1, j, 1 << 30])
    T = sum(new)
    p = torch.softmax(torch.randn(T, V, generator=gen(dev, V), device=dev) * 4, 1)
    tokens = top_tokens(rng, p, new, trees)
    run_verify(dev, new, sum(trees, []), tokens, p, draws(rng, T), draws(rng, B), dtype=dtype, pad=V % 4, behind=2)


@pytest.mark.parametrize("V,B,hi", [(1, 2, 3), (2, 20, 9), (7, 9, 64), (1000, 40, 9), (5003, 5, 64), (151936, 1, 5)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_verify_chains(dev, V, B, hi, dtype):
    import torch
    note(f"verify chains V={V} B={B} {dtype}")
    rng = random.Random(V + B)
    new = [hi] + ref.rand_lengths(rng, B - 1, hi)
    T = sum(new)
    g = gen(dev, V)
    x = torch.randn(T, V, generator=g, device=dev) * 4
    p = torch.softmax(x, 1)
    q = torch.softmax(x + 0.5 * torch.randn(T, V, generator=g, device=dev), 1)
    tokens = [0] + torch.multinomial(q, 1, generator=g)[:-1, 0].tolist()
    tokens = [rng.choice([t] * 20 + [-1, V]) for t in tokens]
    got = run_verify(dev, new, None, tokens, p, draws(rng, T), draws(rng, B), q=q, dtype=dtype, pad=3)
    if V == 1000:
        assert len(set(got[0])) > 2  # some go far, some stop at once
    run_verify(dev, new, None, tokens, p, draws(rng, T), draws(rng, B), dtype=dtype)  # a chain of choices


def test_verify_corners(dev):
    """Rows of zeros, NaN and negative values, one-hot rows, all mass on the
    drafts, numbers at the ends, a max_q below the rows."""
    import torch
    note("verify corners")
    V, nan = 2100, math.nan
    rows = torch.zeros(9, V)
    rows[0, 5] = 1.0                      # goes to 5 whatever is drawn
    rows[1, 7], rows[1, 2000] = 0.5, 0.5  # all mass on its children
    rows[2] = -1.0
    rows[2, 3] = nan                      # nothing counts: -1
    rows[3] = nan
    rows[3, 2099] = 1e-30                 # the last token, hardly any mass
    rows[4, 1023], rows[4, 1024] = 0.25, 0.75
    rows[5:] = 1.0 / V
    p = rows.to(dev)
    one = 1.0 - 2.0 ** -24
    for parents, tokens in (([-1, 0, 1, 1, 0, 4, 4, 6, 6], [0, 5, 7, 2000, 8, 1023, 1024, 9, 9]),
                            ([-1, 0, 1, 2, 3, 4, 5, 6, 7], [0, 5, 7, 3, 2099, 1024, 0, 1, 2])):
        for u in (0.0, 0.3, 0.5, 0.9, one):
            for s in (0.0, 0.25, one, 1.0, 2.0, -1.0):
                run_verify(dev, [9], parents, tokens, p, [u] * 9, [s])
        run_verify(dev, [9], parents, tokens, p, [one, 0.2, 0.0] * 3, [0.1], max_q=4)
    for i in range(6):  # one row alone, and against itself: no weight left
        run_verify(dev, [1], None, [0], p[i:i + 1], [0.5], [0.7])
        run_verify(dev, [2], None, [0, 8], p[[i, 4]], [0.5, 0.5], [0.7], q=p[[i, 4]])
    run_verify(dev, [0, 2, 0], None, [0, 5], p[:2], [0.5] * 2, [0.7] * 3)


@pytest.mark.parametrize("V", [4095, 4096, 4097, 8193, 20000])
@pytest.mark.parametrize("B", [1, 30, 700])
def test_verify_at_the_ends_of_chunks(dev, V, B):
    """A few equal weights around multiples of 4096, where rows are cut: numbers
    exactly at their sums and next to them, children among them."""
    import torch
    note(f"verify chunks V={V} B={B}")
    rng = random.Random(V + B)
    at = sorted({x for c in range(0, V + 1, 4096) for x in (c - 1, c, c + 1) if 0 <= x < V} | {V - 1})[:16]
    p = torch.zeros(2 * B, V, device=dev)
    p[:, at] = 0.0625
    trees = [[-1, 0]] * B
    tokens = [rng.choice(at) for _ in range(2 * B)]
    total = len(at) * 0.0625
    numbers = [x / 16 / total for x in range(len(at))]
    au = [rng.choice([0.0, 0.0625, 0.9]) for _ in range(2 * B)]
    su = [max(rng.choice(numbers) + rng.choice([0.0, 2.0 ** -20, -2.0 ** -20]), 0.0) for _ in range(B)]
    run_verify(dev, [2] * B, sum(trees, []), tokens, p, au, su)


def test_verify_accepts_as_often_as_the_target_says(dev):
    """The token behind the root, accepted or drawn, has the target's
    probabilities: 4000 requests, each count within six of its deviations."""
    import torch
    from inferflux_amd import attention as at, drafts
    note("verify distribution")
    V, B = 6, 4000
    g = gen(dev, 9)
    p = torch.tensor([0.4, 0.25, 0.15, 0.1, 0.07, 0.03], device=dev)
    d = torch.tensor([0.1, 0.1, 0.5, 0.1, 0.1, 0.1], device=dev)
    cu = torch.arange(0, 2 * B + 1, 2, dtype=torch.int32, device=dev)
    drawn = torch.multinomial(d.expand(B, V), 1, generator=g)[:, 0].int()
    tokens = torch.stack([torch.zeros_like(drawn), drawn], 1).flatten().contiguous()
    for chain in (True, False):
        u, s = torch.rand(2 * B, generator=g, device=dev), torch.rand(B, generator=g, device=dev)
        r = drafts.verify(tokens, cu, p.repeat(2 * B, 1), u, s, 2, workspace=at.workspace(dev),
                          draft_probs=d.repeat(2 * B, 1) if chain else None)
        first = r.emitted.view(B, 2)[:, 0]
        for x in range(V):
            want, dev_ = B * float(p[x]), math.sqrt(B * float(p[x]) * (1 - float(p[x])))
            assert abs(int((first == x).sum()) - want) <= 6 * dev_


# ----------------------------------------------------------------- what is kept
@pytest.mark.parametrize("P,Hkv,D,dtype", [(16, 2, 128, "f16"), (64, 8, 128, "bf16"), (32, 3, 64, "f16"), (16, 1, 256, "f16"),
                                           (16, 5, 24, "bf16")])
def test_keep_path(dev, P, Hkv, D, dtype):
    import torch
    from inferflux_amd import drafts
    note(f"keep P={P} Hkv={Hkv} D={D}")
    rng = random.Random(P + D)
    new = [64, 0, 1, 30, 12, 64, 17, 9]
    ctx = [rng.choice([0, P - 1, 3 * P, rng.randint(0, 200)]) for _ in new]
    k, v, table, rows = make_cache(dev, dt_of(dtype), ctx, new, Hkv, D, P, 5)
    paths, accepted = [], []
    for n in new:
        a = rng.choice([0, n // 2, n - 1, min(3, n - 1)]) if n else -1
        path = [0] + sorted(rng.sample(range(1, n), a)) if n else []
        paths += path + [-1] * (n - len(path))
        accepted.append(a)
    accepted[6] = -1
    want_k, want_v = k.clone(), v.clone()
    at = 0
    for b, n in enumerate(new):
        for src, dst in ref.keep(ctx[b], n, paths[at:at + n], accepted[b]):
            (sp, si), (dp, di) = ((int(table[b, x // P]), x % P) for x in (src, dst))
            want_k[dp, :, :, di] = k[sp, :, :, si]
            want_v[dp, :, di // 8, :, di % 8] = v[sp, :, si // 8, :, si % 8]
        at += n
    drafts.keep_path((k, v), table, i32(cu_of(new), dev), i32([c + n for c, n in zip(ctx, new)], dev),
                     i32(paths, dev), i32(accepted, dev), 64)
    assert torch.equal(k.view(torch.int16), want_k.view(torch.int16))
    assert torch.equal(v.view(torch.int16), want_v.view(torch.int16))


def test_keep_bad_pages_and_lengths(dev):
    """Page numbers outside the cache and tokens outside the table move nothing."""
    import torch
    from inferflux_amd import drafts
    note("keep bad pages")
    k, v, table, _ = make_cache(dev, torch.float16, [10, 10, 10], [20, 20, 20], 2, 64, 16, 5)
    table[0, :] = 1 << 30
    table[1, 1:] = -1
    before = k.clone(), v.clone()
    path = [0] + list(range(12, 20)) + [-1] * 11
    drafts.keep_path((k, v), table, i32([0, 20, 40, 60], dev), i32([30, 30, 1 << 30], dev), i32(path * 3, dev),
                     i32([8, 8, 8], dev), 20)
    assert torch.equal(k.view(torch.int16), before[0].view(torch.int16))
    assert torch.equal(v.view(torch.int16), before[1].view(torch.int16))


# ------------------------------------------------------------------ as it is used
@pytest.mark.parametrize("graph", [False, True])
def test_step_of_drafts(dev, graph):
    """Steps of trees through one layer: plan, rotate and append, attention,
    verification, what is kept, the next step's lengths.  The cache must hold
    what the accepted tokens, one behind the other, would have put there."""
    import torch
    from inferflux_amd import attention as at, drafts
    note(f"step graph={graph}")
    B, Hq, Hkv, D, P, V, N = 3, 8, 2, 64, 16, 50, 12
    rng = random.Random(3)
    g = gen(dev, 3)
    k_cache, v_cache = at.kv_cache(40, Hkv, D, P, device=dev)
    table = torch.full((B, 12), -1, dtype=torch.int32, device=dev)
    free, count = torch.randperm(40, generator=g, device=dev).int(), i32([40], dev)
    ctx = i32([0] * B, dev)
    freq = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D)
    # a token's rows depend on the token alone, so that the cache can be foretold
    wk, wv, wq = (torch.randn(V, h, D, generator=g, device=dev).half() for h in (Hkv, Hkv, Hq))
    probs = torch.softmax(torch.randn(V, V, generator=g, device=dev) * 3, 1)
    ws = at.workspace(dev)
    tokens, parents = i32([0] * (B * N), dev), i32([-1] * (B * N), dev)
    new = i32([N] * B, dev)
    au, su = torch.zeros(B * N, device=dev), torch.zeros(B, device=dev)
    bufs = {}

    def step():
        p = at.plan_batch(ctx, new, table, free, count, P, B * N, out=bufs.get("p"))
        t = drafts.plan_tree(parents, p.cu_q, p.kv_len, out=bufs.get("t"))
        x = tokens.long()
        q = at.rope_append(wq[x], wk[x], wv[x], t.positions, p.slots, k_cache, v_cache, freq)
        o = drafts.tree_attention(q, k_cache, v_cache, table, p.cu_q, p.kv_len, t.masks, N, 12 * P, workspace=ws)
        r = drafts.verify(tokens, p.cu_q, probs[x], au, su, N, parents=parents, out=bufs.get("r"), workspace=ws)
        drafts.keep_path((k_cache, v_cache), table, p.cu_q, p.kv_len, r.path, r.accepted, N)
        kept = drafts.plan_kept(p.cu_q, p.kv_len, r.accepted, table, free, p.free_left, P, out=bufs.get("k"))
        bufs.update(p=p, t=t, r=r, k=kept)
        ctx.copy_(kept.ctx_len)
        count.copy_(kept.free_left)
        return o

    if graph:
        saved = [x.clone() for x in (k_cache, v_cache, table, free, count, ctx)]
        step()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured, stream=s):
            out = step()
        for x, y in zip((k_cache, v_cache, table, free, count, ctx), saved):
            x.copy_(y)
    said = [[rng.randrange(V)] for _ in range(B)]  # what each request's cache will hold, and its next root
    accepted = 0
    for _ in range(6):
        trees = [ref.tree(rng, N, 3) for _ in range(B)]
        flat, toks = sum(trees, []), []
        best = probs.topk(5, 1).indices.tolist()
        for b in range(B):
            mine = [said[b][-1]]
            for j in range(1, N):
                mine.append(rng.choice(best[mine[trees[b][j]]]))
            toks += mine
        tokens.copy_(i32(toks, dev)), parents.copy_(i32(flat, dev))
        au.copy_(torch.rand(B * N, generator=g, device=dev)), su.copy_(torch.rand(B, generator=g, device=dev))
        had = ctx.tolist()
        if graph:
            captured.replay()
            o = out
        else:
            o = step()
        p, r = bufs["p"], bufs["r"]
        assert int(p.status) == 0 and int(bufs["k"].status) == 0
        want = ref.verify(flat, toks, [0, N, 2 * N, 3 * N], probs[tokens.long()].cpu().tolist(), au.tolist(), su.tolist())
        assert [x.tolist() for x in r] == list(want)
        for b in range(B):
            n = int(r.accepted[b]) + 1
            accepted += n - 1
            held = said[b][:]
            said[b] += r.emitted[b * N:b * N + n].tolist()
            assert int(ctx[b]) == had[b] + n == len(said[b]) - 1
            # the attention of the root: all tokens before it and itself
            x = torch.tensor(held, device=dev)
            pos = torch.arange(len(held), device=dev)
            angle = pos.double()[:, None, None] * freq
            rot = lambda y: torch.cat([y[..., :D // 2].double() * angle.cos() - y[..., D // 2:].double() * angle.sin(),
                                       y[..., D // 2:].double() * angle.cos() + y[..., :D // 2].double() * angle.sin()], -1)  # noqa: E731
            kk, qq = rot(wk[x]).half(), rot(wq[x]).half()[-1:]
            ref_o, bound = ref.attend_seen(qq, kk, wv[x], torch.ones(1, len(held), dtype=torch.bool), D ** -0.5)
            # the rotated rows, formed in 32 bits there, may round to a neighbour here
            check(o[b * N:b * N + 1], ref_o, bound + 4 * 2.0 ** -11, "root")
    assert accepted > 3
    pages = sorted(free.tolist()[:int(count)] + [x for b in range(B) for x in table[b, :-(-int(ctx[b]) // P)].tolist()])
    assert pages == list(range(40))


def test_verify_offsets_past_32_bits(dev):
    """Rows of probabilities further than 2^32 bytes from the first."""
    import torch
    from inferflux_amd import attention as at, drafts
    note("verify large")
    V, n, B = 151936, 64, 129
    T = n * B
    p = torch.zeros(T, V, device=dev)
    assert p.nbytes > 1 << 32
    rng = random.Random(1)
    p[-n:] = torch.softmax(4 * torch.randn(n, V, generator=gen(dev, 1), device=dev), 1)
    parents, tokens = ref.tree(rng, n), [5]
    best = p[-n:].topk(4, 1).indices.tolist()
    for j in range(1, n):
        tokens.append(best[parents[j]][rng.randrange(4)])
    au, su = torch.full((T,), 0.2, device=dev), torch.full((B,), 0.6, device=dev)
    r = drafts.verify(i32([1] * (T - n) + tokens, dev), i32([n * b for b in range(B + 1)], dev), p, au, su, n,
                      parents=i32(parents * B, dev), workspace=at.workspace(dev))
    want = ref.verify(parents, tokens, [0, n], p[-n:].cpu().tolist(), [float(au[0])] * n, [float(su[0])])
    assert r.accepted.tolist() == [0] * (B - 1) + want[0]
    assert r.path[-n:].tolist() == want[1] and r.emitted[-n:].tolist() == want[2]
    assert r.emitted[:-n].eq(-1).all() and r.path[:-n].view(-1, n)[:, 0].eq(0).all()
