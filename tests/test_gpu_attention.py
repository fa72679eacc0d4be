"""The attention operators on the GPU against their plain 64-bit forms
(tests/attn_ref.py): batch plans, rotation with the cache write, attention over
the paged cache and over packed prompts, alone and as a serving step runs
them."""
import math
import random

import pytest

from tests.attn_ref import TINY, U, attend, check, gather_cache, put_cache
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


def i32(v, dev):
    import torch
    return torch.tensor(v, dtype=torch.int32, device=dev)


def gen(dev, seed):
    import torch
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def dt_of(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


# ---------------------------------------------------------------------- plans
def plan_by_hand(ctx, new, table, free, count, P, T):
    """The definition, request by request."""
    W = len(table[0])
    table = [list(r) for r in table]
    n_new = sum(max(n, 0) for n in new)
    bad = 8 if any(c < 0 or n < 0 or c + n > 2 ** 31 - 1 for c, n in zip(ctx, new)) else 0
    ok = [(c, n) if c >= 0 and n >= 0 and c + n <= 2 ** 31 - 1 else (0, 0) for c, n in zip(ctx, new)]
    need = sum(-(-(c + n) // P) - -(-c // P) for c, n in ok)
    n_new = sum(n for _, n in ok)
    status = bad | (need > min(max(count, 0), len(free))) | 2 * any(-(-(c + n) // P) > W for c, n in ok)
    status |= 4 * (n_new > T)
    if status:
        return [0] * (len(ctx) + 1), list(ctx), [0] * T, [-1] * T, count, status, table
    at, cu, pos, slots = min(count, len(free)), [0], [], []
    for b, (c, n) in enumerate(zip(ctx, new)):
        for p in range(c, c + n):
            if p % P == 0:
                at -= 1
                table[b][p // P] = free[at]
            pos.append(p)
            slots.append(table[b][p // P] * P + p % P)
        cu.append(cu[-1] + n)
    gap = T - len(pos)
    return cu, [c + n for c, n in zip(ctx, new)], pos + [0] * gap, slots + [-1] * gap, at, 0, table


def run_plan(dev, ctx, new, table, free, count, P, T):
    from inferflux_amd import attention as at
    t = i32(table, dev)
    p = at.plan_batch(i32(ctx, dev), i32(new, dev), t, i32(free, dev), i32([count], dev), P, T)
    want = plan_by_hand(ctx, new, table, free, count, P, T)
    got = [x.tolist() for x in p] + [t.tolist()]
    got[4], got[5] = got[4][0], got[5][0]
    for name, g, w in zip(("cu_q", "kv_len", "positions", "slots", "free_left", "status", "table"), got, want):
        assert g == w, name
    return p


@pytest.mark.parametrize("B,P,hi,qhi,extra", [
    (1, 16, 0, 1, 0), (1, 64, 200, 1, 3), (7, 16, 40, 3, 0), (32, 64, 3000, 1, 0), (33, 128, 500, 300, 9),
    (256, 32, 300, 20, 1), (257, 256, 900, 2, 0), (1500, 16, 100, 5, 70)])
def test_plan(dev, B, P, hi, qhi, extra):
    note(f"plan B={B} P={P} hi={hi} qhi={qhi}")
    rng = random.Random(B * 31 + P)
    ctx = [rng.randint(0, hi) for _ in range(B)]
    new = [rng.choice([0, 1, qhi, rng.randint(0, qhi)]) for _ in range(B)]
    W = -(-(hi + qhi) // P) + 1
    held = [-(-c // P) for c in ctx]
    pages = list(range(sum(held) + sum(-(-(c + n) // P) - h for c, n, h in zip(ctx, new, held)) + 2))
    rng.shuffle(pages)
    table, k = [], 0
    for h in held:
        table.append(pages[k:k + h] + [-7] * (W - h))
        k += h
    free = pages[k:] + [-9] * 3  # the stack's array is longer than what is in it
    run_plan(dev, ctx, new, table, free, len(free) - 3, P, sum(new) + extra)


@pytest.mark.parametrize("ctx,new,count,W,T,want", [
    ([10, 20], [7, 13], 1, 4, 20, 1),        # two pages needed, one free
    ([10, 20], [7, 45], 9, 4, 60, 2),        # five pages in a row of four
    ([10, 20], [7, 13], 9, 4, 19, 4),        # a token more than there is room for
    ([10, -1], [7, 13], 9, 4, 40, 8),
    ([10, 20], [7, -13], 9, 4, 40, 8),
    ([2 ** 31 - 1, 20], [1, 1], 9, 4, 40, 8),
    ([2 ** 31 - 1, 20], [0, 1], 9, 4, 40, 2),
    ([2 ** 31 - 5, 20], [2, 2 ** 31 - 50], 0, 4, 40, 7),
    ([10, 20], [7, 13], -3, 4, 20, 1),
    ([0, 0], [0, 0], 0, 4, 0, 0)])
def test_plan_status(dev, ctx, new, count, W, T, want):
    """A plan that cannot be made takes nothing and says why."""
    note(f"plan status {want}")
    table = [[5, 6, -1, -1][:W], [8, 9, -1, -1][:W]]
    p = run_plan(dev, ctx, new, table, [1, 2, 3, 4, 7, 10, 11, 12, 13], count, 16, T)
    assert p.status.item() == want


def test_plan_page_number_past_31_bits_has_no_slot(dev):
    """A table entry that no cache can have gives slot -1, not another slot."""
    from inferflux_amd import attention as at
    note("plan bad page numbers")
    t = i32([[2 ** 31 - 1, -4, 3]], dev)
    p = at.plan_batch(i32([40], dev), i32([1], dev), t, i32([2 ** 30], dev), i32([1], dev), 16, 2)
    assert p.slots.tolist() == [3 * 16 + 8, -1]
    p = at.plan_batch(i32([16], dev), i32([9], dev), t, i32([2 ** 30], dev), i32([1], dev), 16, 9)
    assert p.status.item() == 0 and p.slots.tolist() == [-1] * 9


# --------------------------------------------------------------------- append
def rotate(x, pos, freq, inter):
    """x [T, H, D] (float64) rotated, and the sum of magnitudes of each value."""
    import torch
    r = 2 * freq.numel()
    ang = pos.double()[:, None] * freq
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    y, m = x.clone(), x.abs().clone()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if inter else (x[..., :r // 2], x[..., r // 2:r])
    ya, yb, mm = a * c - b * s, b * c + a * s, a.abs() + b.abs()
    if inter:
        y[..., 0:r:2], y[..., 1:r:2], m[..., 0:r:2], m[..., 1:r:2] = ya, yb, mm, mm
    else:
        y[..., :r // 2], y[..., r // 2:r], m[..., :r // 2], m[..., r // 2:r] = ya, yb, mm, mm
    return y, m


@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("T,Hq,Hkv,D,P,rot,inter", [
    (1, 16, 2, 128, 64, 128, False), (8, 5, 1, 96, 16, 96, False), (37, 4, 4, 64, 16, 32, True),
    (50, 3, 3, 256, 32, 256, True), (64, 2, 1, 40, 128, 16, False), (33, 2, 1, 24, 16, 0, False),
    (2311, 4, 2, 128, 16, 128, False), (2050, 2, 1, 72, 256, 48, True)])
def test_append(dev, src, dt, T, Hq, Hkv, D, P, rot, inter):
    """Rotation and cache write: tolerances are one rounding to the cache's
    type and, before it, 4 fp32 roundings of |a| + |b| (products, sum, sine and
    cosine to 2 ulp); nothing but the slots is written."""
    import torch
    from inferflux_amd import attention as at
    note(f"append {src}->{dt} T={T} Hq={Hq} Hkv={Hkv} D={D} P={P} rot={rot} inter={inter}")
    g, rng = gen(dev, T + D), random.Random(T * D)
    # runs of consecutive slots of every length and start, some tokens left out
    pages = -(-2 * T // P) + 3
    slots, at_slot = [], rng.randint(0, 5)
    while len(slots) < T:
        n = rng.choice([1, 2, 7, 8, 9, 30])
        for s in range(at_slot, at_slot + n):
            slots.append(s if s < pages * P else -1)
        at_slot += n + rng.choice([0, 0, 1, 5])
    slots = slots[:T]
    for i in range(0, T, 11):
        if T > 8:
            slots[i] = rng.choice([-1, pages * P, 2 ** 31 - 1, -2 ** 31])
    order = torch.randperm(pages, generator=g, device=dev)
    s = torch.tensor(slots, device=dev)
    live = (s >= 0) & (s < pages * P)
    s = torch.where(live, order[(s.clamp(0, pages * P - 1)) // P] * P + s % P, s)
    pos = torch.randint(0, 200000, (T,), generator=g, device=dev)
    freq = 1e4 ** (-torch.arange(rot // 2, dtype=torch.float64, device=dev) * 2 / max(rot, 1))
    rows = torch.randn(T, (Hq + 2 * Hkv) * D + 3, generator=g, device=dev).to(dt_of(src))
    q, k, v = (x.unflatten(1, (-1, D)) for x in
               (rows[:, :Hq * D], rows[:, Hq * D:(Hq + Hkv) * D], rows[:, (Hq + Hkv) * D:(Hq + 2 * Hkv) * D]))
    kc, vc = at.kv_cache(pages, Hkv, D, P, dt_of(dt), dev)
    kc.fill_(7.0), vc.fill_(-7.0)
    want_k, want_v = kc.double(), vc.double()
    buf = torch.full((T, Hq * D + 8), 3.0, dtype=dt_of(dt), device=dev)
    out = buf[:, :Hq * D].unflatten(1, (Hq, D))
    got = at.rope_append(q, k, v, pos.int(), s.int(), kc, vc, freq if rot else None, inter, q_out=out)
    assert got is out and bool((buf[:, Hq * D:] == 3).all()) and bool((out[~live] == 3).all())
    tol = lambda y, m: U[dt_of(dt)] * y.abs() + 2 * 4 * 2.0 ** -24 * m + TINY[dt_of(dt)]  # noqa: E731
    yq, mq = rotate(q.double(), pos, freq, inter)
    assert bool(((out.double() - yq).abs() <= tol(yq, mq))[live].all())
    yk, mk = rotate(k.double(), pos, freq, inter)
    sl = s[live].long()
    page, place = sl // P, sl % P
    gk = kc[page, :, :, place].double().flatten(2)
    assert bool(((gk - yk[live]).abs() <= tol(yk, mk)[live]).all())
    want_k[page, :, :, place] = gk.unflatten(2, (-1, 8))
    want_v[page, :, place // 8, :, place % 8] = v[live].to(dt_of(dt)).double()
    assert torch.equal(vc.double(), want_v) and torch.equal(kc.double(), want_k)


def test_append_far_positions(dev):
    """Positions near 2^31 keep their angle: 64-bit turns leave 2^-20 of a
    radian there (2^31 radians at 2^-52), and the rest is fp32's."""
    import torch
    from inferflux_amd import attention as at
    note("append far positions")
    D, T = 64, 9
    pos = torch.arange(2 ** 31 - 1 - T, 2 ** 31 - 1, device=dev)
    freq = 1e6 ** (-torch.arange(D // 2, dtype=torch.float64, device=dev) * 2 / D)
    x = torch.randn(T, 1, D, generator=gen(dev, 5), device=dev)
    kc, vc = at.kv_cache(2, 1, D, 16, torch.float16, dev)
    out = at.rope_append(x, x, x, pos.int(), torch.arange(T, dtype=torch.int32, device=dev), kc, vc, freq)
    y, m = rotate(x.double(), pos, freq, False)
    assert bool(((out.double() - y).abs() <= 2.0 ** -11 * y.abs() + (2.0 ** -19 + 2.0 ** -21) * m).all())


# ---------------------------------------------------------------- paged: setup
class Batch:
    """B requests in a paged cache with shuffled pages: kv tokens in all, the
    last n of them new.  Unwritten slots, pages no request has and table
    entries behind a request's pages hold NaN or nonsense."""

    def __init__(self, dev, kv, new, Hq, Hkv, D, P, dt, seed=0, extra_rows=0, out_dtype=None, scale_q=1.5):
        import torch
        g, rng = gen(dev, seed + 17), random.Random(seed)
        self.dev, self.kv, self.new, self.P, self.dt = dev, kv, new, P, dt_of(dt)
        need = [-(-n // P) for n in kv]
        W = max(need + [1]) + 2
        pages = list(range(sum(need) + 3))
        rng.shuffle(pages)
        rows, at = [], 0
        for n in need:
            rows.append(pages[at:at + n] + [rng.choice([-1, 2 ** 31 - 1, 0]) for _ in range(W - n)])
            at += n
        self.table = i32(rows, dev)
        shape = (len(pages), Hkv)
        nan = float("nan")
        self.kc = torch.full(shape + (D // 8, P, 8), nan, dtype=self.dt, device=dev)
        self.vc = torch.full(shape + (P // 8, D, 8), nan, dtype=self.dt, device=dev)
        for b, n in enumerate(kv):
            if n:
                put_cache(self.kc, self.vc, self.table[b], torch.randn(n, Hkv, D, generator=g, device=dev),
                          torch.randn(n, Hkv, D, generator=g, device=dev))
        self.T = sum(new)
        self.cu = i32([sum(new[:b]) for b in range(len(new) + 1)], dev)
        self.kvt = i32(kv, dev)
        R = self.T + extra_rows
        wide = torch.randn(R, Hq * D + 24, generator=g, device=dev) * scale_q
        self.q = wide.to(self.dt)[:, 8:8 + Hq * D].unflatten(1, (Hq, D))  # rows of a wider buffer
        self.out = torch.full((R, Hq, D), 9.0, dtype=dt_of(out_dtype or dt), device=dev)

    def run(self, ws, window=0, scale=None, max_q=None, max_kv=None, out=None, stream=None):
        from inferflux_amd import attention as at
        return at.paged_attention(self.q, self.kc, self.vc, self.table, self.cu, self.kvt,
                                  max_q or max(self.new + [1]), max_kv or max(self.kv + [1]), scale=scale,
                                  window=window, out=self.out if out is None else out, workspace=ws,
                                  stream=stream)

    def verify(self, out=None, window=0, scale=None):
        out = self.out if out is None else out
        at = 0
        for b, (n, L) in enumerate(zip(self.new, self.kv)):
            if n:
                k, v = gather_cache(self.kc, self.vc, self.table[b], L)
                ref, bound = attend(self.q[at:at + n], k, v, L - n, scale or self.q.shape[2] ** -0.5, True, window)
                check(out[at:at + n], ref, bound, f"request {b}: {n} new of {L}")
            at += n
        assert bool((out[at:] == 9).all()), "rows behind the last request were written"


@pytest.fixture(scope="module")
def ws(dev):
    from inferflux_amd import attention as at
    return at.workspace(dev)


def counters_clear(ws):
    return not bool(ws[:32768].any())


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,D,P,kv,new", [
    (16, 2, 128, 64, [1, 2, 63, 64, 65, 200], [1] * 6),
    (40, 8, 128, 16, [31, 32, 33, 500, 1], [1] * 5),
    (4, 4, 64, 16, [17, 129, 1000], [1] * 3),
    (6, 2, 96, 32, [5, 31, 77, 300], [1] * 4),
    (8, 1, 256, 128, [1, 130, 513], [1] * 3),
    (32, 1, 128, 256, [300, 255], [1] * 2),              # the most rows of this kernel
    (16, 2, 128, 32, [10, 0, 3, 100], [1, 0, 1, 0]),     # requests without new tokens
    (8, 2, 128, 16, [4, 90, 31, 33, 7], [4, 3, 1, 8, 7]),  # several tokens (drafts)
    (5, 5, 64, 16, [3, 40, 2], [5, 32, 1]),              # rows before the first key: empty
])
def test_paged_few_rows(dev, ws, dt, Hq, Hkv, D, P, kv, new):
    from inferflux_amd import ops
    note(f"paged rows {dt} Hq={Hq} Hkv={Hkv} D={D} P={P} kv={kv} new={new}")
    x = Batch(dev, kv, new, Hq, Hkv, D, P, dt, seed=D + P, extra_rows=2)
    with ops.launch_log() as lg:
        x.run(ws)
    assert lg.kernels[0].startswith("k_attn_rows<")
    x.verify()
    assert counters_clear(ws)


@pytest.mark.parametrize("dt,Hq,Hkv,D,P,kv,new", [
    ("f16", 16, 2, 128, 64, [5000], [1]), ("bf16", 16, 2, 128, 64, [5000, 40, 3000], [1, 1, 1]),
    ("bf16", 10, 2, 96, 16, [4001, 1, 2], [2, 2, 2]), ("f16", 4, 1, 256, 32, [2500, 700], [1, 1]),
    ("f16", 3, 3, 64, 16, [1, 9000], [1, 1])])
def test_paged_split_keys(dev, ws, dt, Hq, Hkv, D, P, kv, new):
    """Long requests are split over workgroups: the same bits on every call, and
    a request far longer than the plan was told is computed whole."""
    import torch
    note(f"paged split {dt} Hq={Hq} Hkv={Hkv} D={D} P={P} kv={kv} new={new}")
    from inferflux_amd import attention as at
    assert at.paged_workspace_bytes(len(kv), sum(new), Hq, Hkv, D, max(new), max(kv)) > 0
    x = Batch(dev, kv, new, Hq, Hkv, D, P, dt, seed=D + P)
    x.run(ws)
    first = x.out.clone()
    x.verify()
    for _ in range(3):
        x.out.fill_(9.0)
        x.run(ws)
        assert torch.equal(first, x.out)
    x.run(ws, max_kv=300)
    x.verify()
    x.run(ws, max_kv=20)
    x.verify()
    assert counters_clear(ws)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,D,P,kv,new", [
    (16, 2, 128, 64, [100, 1, 64], [100, 1, 37]),
    (40, 8, 128, 16, [300, 77, 5], [65, 77, 1]),
    (4, 4, 64, 32, [33, 500], [33, 130]),
    (6, 2, 96, 16, [200, 45, 129], [64, 45, 127]),
    (2, 1, 256, 64, [190, 64], [100, 20]),
    (16, 2, 128, 128, [0, 700, 30, 9], [0, 3, 30, 0]),
    (8, 2, 128, 16, [3, 20, 100], [9, 64, 2]),           # rows before the first key
    (2, 2, 64, 16, [2000, 1500], [300, 1]),
])
def test_paged_chunks(dev, ws, dt, Hq, Hkv, D, P, kv, new):
    from inferflux_amd import ops
    note(f"paged tile {dt} Hq={Hq} Hkv={Hkv} D={D} P={P} kv={kv} new={new}")
    x = Batch(dev, kv, new, Hq, Hkv, D, P, dt, seed=D + P, extra_rows=3)
    with ops.launch_log() as lg:
        x.run(ws)
    assert lg.kernels[0].startswith("k_attn_tile<")
    x.verify()
    assert counters_clear(ws)


@pytest.mark.parametrize("dt,Hq,Hkv,D,P,kv,new", [
    ("bf16", 40, 8, 128, 64, [3000, 900, 1], [64, 64, 1]), ("f16", 8, 2, 64, 16, [5000], [70]),
    ("bf16", 2, 1, 256, 32, [2100, 2000], [90, 1])])
def test_paged_chunks_split(dev, ws, dt, Hq, Hkv, D, P, kv, new):
    import torch
    note(f"paged tile split {dt} Hq={Hq} Hkv={Hkv} D={D} P={P} kv={kv} new={new}")
    from inferflux_amd import attention as at
    assert at.paged_workspace_bytes(len(kv), sum(new), Hq, Hkv, D, max(new), max(kv)) > 0
    x = Batch(dev, kv, new, Hq, Hkv, D, P, dt, seed=D + P)
    x.run(ws)
    first = x.out.clone()
    x.verify()
    for _ in range(2):
        x.run(ws)
        assert torch.equal(first, x.out)
    x.run(ws, max_kv=600)
    x.verify()
    assert counters_clear(ws)


@pytest.mark.parametrize("dt,Hq,Hkv,D,P,B,qhi,long", [
    ("f16", 8, 2, 64, 16, 65, 1, 5000),    # one request more than the lanes of a wave
    ("bf16", 4, 4, 96, 32, 200, 2, 3000),  # some without new tokens
    ("f16", 5, 1, 128, 16, 300, 1, 700),
    ("f16", 24, 24, 64, 16, 70, 1, 4000),  # more requests than work items are wanted
    ("f16", 2, 1, 64, 16, 4096, 1, 2000),  # the largest batch
    ("f16", 2, 1, 64, 16, 4096, 17, 1500),
    ("bf16", 4, 2, 64, 16, 70, 40, 4000),  # row tiles
    ("f16", 2, 2, 128, 64, 130, 90, 2500),
    ("f16", 24, 24, 128, 16, 40, 60, 2600),  # more row tiles than work items are wanted
])
def test_paged_large_batches(dev, ws, dt, Hq, Hkv, D, P, B, qhi, long):
    """Work is found in batches of more requests than a wave has lanes, of very
    different lengths."""
    import torch
    note(f"paged large batch {dt} Hq={Hq} Hkv={Hkv} D={D} P={P} B={B} qhi={qhi}")
    r = random.Random(B)
    new = [r.choice([0, 1, r.randint(1, qhi)]) for _ in range(B)]
    kv = [n + r.randint(0, 150) for n in new]
    for b in (B // 3, B - 1):
        new[b], kv[b] = qhi, long + b
    x = Batch(dev, kv, new, Hq, Hkv, D, P, dt, seed=B, extra_rows=1)
    x.run(ws)
    x.verify()
    first = x.out.clone()
    x.run(ws)
    assert torch.equal(first, x.out)
    assert counters_clear(ws)


@pytest.mark.parametrize("window", [1, 5, 64, 100, 2 ** 31 - 1])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 2, 1], [80, 33, 1]])
def test_paged_window(dev, ws, window, new):
    note(f"paged window={window} new={new}")
    x = Batch(dev, [700, 81, 64], new, 8, 2, 128, 16, "f16", seed=window % 97)
    x.run(ws, window=window)
    x.verify(window=window)
    assert counters_clear(ws)


@pytest.mark.parametrize("window", [2, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1])
@pytest.mark.parametrize("new,kv", [([9, 4], [3, 70]), ([90, 60], [41, 300])])
def test_paged_window_rows_before_the_first_key(dev, ws, window, new, kv):
    """Positions below 0 less the widest windows."""
    note(f"paged window {window} new={new} kv={kv}")
    x = Batch(dev, kv, new, 6, 2, 128, 16, "f16", seed=3)
    x.run(ws, window=window)
    x.verify(window=window)


@pytest.mark.parametrize("out_dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,kv", [([1, 1], [70, 3000]), ([60, 5], [60, 2000])])
def test_paged_output_types(dev, ws, out_dtype, new, kv):
    note(f"paged out {out_dtype} new={new}")
    x = Batch(dev, kv, new, 8, 2, 128, 64, "bf16", out_dtype=out_dtype, extra_rows=1)
    x.run(ws, scale=0.05)
    x.verify(scale=0.05)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("new,window", [([1, 1], 0), ([4, 3], 0), ([70, 90], 0), ([70, 90], 20), ([3, 2], 9)])
def test_paged_non_finite(dev, ws, dt, new, window):
    """Infinities and NaN reach the rows that see them, and no other: in keys
    and values behind a row's position, before its window, and everywhere in
    sight.  (The fixture's unwritten slots and free pages are NaN throughout.)"""
    import torch
    note(f"paged non-finite {dt} new={new} window={window}")
    x = Batch(dev, [300, 131], new, 8, 2, 128, 16, dt, seed=3)
    P, inf = x.P, float("inf")

    def poke(cache, b, j, dims, val, v):
        page, at = int(x.table[b, j // P]), j % P
        if v:
            cache[page, 1, at // 8, dims, at % 8] = val
        else:
            cache[page, 1, dims // 8, at, dims % 8] = val

    poke(x.vc, 0, 299, 5, float("nan"), True)     # the last token's value
    poke(x.vc, 0, 298, 70, inf, True)
    poke(x.vc, 0, 297, 127, -inf, True)
    poke(x.vc, 1, 129, 0, inf, True)
    poke(x.kc, 1, 130, 64, float("nan"), False)   # the last token's key
    poke(x.vc, 1, 100, 31, float("nan"), True)    # in sight of all, or of some in a window
    x.run(ws, window=window)
    x.verify(window=window)
    # a row all of whose scores are -inf is not a number
    x.q[:, 4:, 0] = 1.0
    for j in range(131):
        poke(x.kc, 1, j, 0, -inf, False)
    x.run(ws, window=window)
    a = x.new[0]
    assert bool(torch.isnan(x.out[a:, 4:]).all()) and not bool(torch.isnan(x.out[:a, :4]).any())


def test_paged_extreme_scores(dev, ws):
    """Scores of thousands (a single key takes all) and all-equal ones."""
    note("paged extreme scores")
    for q in (60.0, 0.0):
        for new in ([1], [50]):
            x = Batch(dev, [900], new, 8, 2, 128, 64, "f16", scale_q=q, seed=7)
            x.run(ws, scale=1.0)
            x.verify(scale=1.0)


def test_paged_many_light_keys(dev, ws):
    """One heavy key and 30000 that weigh 2^-20 of it each: together a 35th of
    the result, below fp16's smallest step if the probabilities were taken
    relative to the maximum alone."""
    import torch
    note("paged light keys")
    for new in ([1], [40]):
        x = Batch(dev, [30000], new, 8, 2, 128, 64, "f16", seed=11)
        x.kc.zero_()
        x.vc.fill_(1.0)
        x.q.zero_()
        x.q[..., 0] = 20.0 * math.log(2)
        page = int(x.table[0, 0])
        x.kc[page, :, 0, 0, 0] = 1.0
        x.vc[page, :, 0, :, 0] = 0.0
        x.run(ws, scale=1.0)
        x.verify(scale=1.0)


def test_paged_mixed_stays_within_bounds(dev, ws):
    """Lengths, row offsets and page numbers that are nonsense are clamped by
    the kernels: the call ends, and requests that are sound are right."""
    import torch
    note("paged nonsense")
    for new in ([1, 1, 1], [50, 1, 20]):
        x = Batch(dev, [100, 90, 80], new, 8, 2, 128, 16, "f16", seed=4)
        x.table[1] = 2 ** 30
        x.kvt[2] = 2 ** 31 - 1
        x.run(ws)
        k, v = gather_cache(x.kc, x.vc, x.table[0], 100)
        ref, bound = attend(x.q[:new[0]], k, v, 100 - new[0], 128 ** -0.5)
        check(x.out[:new[0]], ref, bound)
        x.kvt[2] = -5
        x.cu[2:] = 2 ** 31 - 1
        x.run(ws)
        x.kvt.fill_(0)
        x.out.fill_(9.0)
        x.cu[:] = i32([0, new[0], new[0] + new[1], sum(new)], dev)
        x.run(ws)
        assert bool((x.out == 0).all())
    assert counters_clear(ws)


def test_paged_offsets_past_32_bits(dev, ws):
    """A cache of more than 2^32 bytes, the request's pages at its end."""
    import torch
    from inferflux_amd import attention as at
    note("paged 5 GB cache")
    P, Hkv, D, pages = 64, 8, 128, 40000  # 5.2 GB each of K and V
    kc = torch.empty(pages, Hkv, D // 8, P, 8, dtype=torch.float16, device=dev)
    vc = torch.empty(pages, Hkv, P // 8, D, 8, dtype=torch.float16, device=dev)
    g = gen(dev, 1)
    n = 150
    table = i32([[pages - 1, pages - 3, pages - 2]], dev)
    freq = 1e4 ** (-torch.arange(64, dtype=torch.float64, device=dev) / 64)
    j = torch.arange(n, device=dev)
    slots = (table[0, (j // P)].long() * P + j % P).int()
    rows = [torch.randn(n, h, D, generator=g, device=dev) for h in (16, Hkv, Hkv)]
    q = at.rope_append(*rows, j.int(), slots, kc, vc, freq)
    k, v = gather_cache(kc, vc, table[0], n)
    assert torch.equal(v, rows[2].half().double())
    for m in (1, n):
        out = at.paged_attention(q[n - m:], kc, vc, table, i32([0, m], dev), i32([n], dev), m, n, workspace=ws)
        check(out, *attend(q[n - m:], k, v, n - m, D ** -0.5))


# --------------------------------------------------------------------- prompts
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 50)])
@pytest.mark.parametrize("Hq,Hkv,D,lens", [
    (16, 2, 128, [1, 2, 64, 65, 200]), (4, 4, 64, [129, 0, 63, 1]), (10, 2, 96, [300, 31]),
    (3, 1, 256, [70, 140]), (5, 5, 128, [257])])
def test_prompt(dev, dt, causal, window, Hq, Hkv, D, lens):
    import torch
    from inferflux_amd import attention as at
    note(f"prompt {dt} causal={causal} window={window} Hq={Hq} Hkv={Hkv} D={D} lens={lens}")
    g, T = gen(dev, D + Hq), sum(lens)
    # Q, K and V side by side, starting two bytes past an aligned address
    w = (Hq + 2 * Hkv) * D
    rows = torch.randn(T * w + 1, generator=g, device=dev).to(dt_of(dt))[1:].view(T, w)
    q, k, v = (x.unflatten(1, (-1, D)) for x in rows.split([Hq * D, Hkv * D, Hkv * D], dim=1))
    buf = torch.full((T + 2, Hq, D), 9.0, dtype=dt_of(dt), device=dev)
    cu = i32([sum(lens[:b]) for b in range(len(lens) + 1)], dev)
    got = at.prompt_attention(q, k, v, cu, max(lens), causal=causal, window=window, out=buf[:T])
    again = at.prompt_attention(q, k, v, cu, max(lens), causal=causal, window=window)
    assert torch.equal(got, again) and bool((buf[T:] == 9).all())
    a = 0
    for n in lens:
        if n:
            ref, bound = attend(q[a:a + n], k[a:a + n], v[a:a + n], 0, D ** -0.5, causal, window)
            check(got[a:a + n], ref, bound, f"prompt of {n}")
        a += n


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Hq,Hkv,D,B,hi", [(4, 2, 64, 64, 300), (8, 1, 128, 65, 90), (3, 3, 64, 300, 40),
                                           (10, 2, 96, 130, 60), (2, 1, 64, 4096, 3)])
def test_prompt_large_batches(dev, causal, Hq, Hkv, D, B, hi):
    """Row tiles are found in batches of as many requests as a wave has lanes,
    and of more, some of them empty."""
    import torch
    from inferflux_amd import attention as at
    note(f"prompt large batch causal={causal} Hq={Hq} Hkv={Hkv} D={D} B={B}")
    r = random.Random(B)
    lens = [r.choice([0, 1, r.randint(1, hi)]) for _ in range(B)]
    lens[B // 2] = 700
    g, T = gen(dev, B), sum(lens)
    q, k, v = (torch.randn(T, h, D, generator=g, device=dev).half() for h in (Hq, Hkv, Hkv))
    buf = torch.full((T + 1, Hq, D), 9.0, dtype=torch.float16, device=dev)
    cu = i32([sum(lens[:b]) for b in range(B + 1)], dev)
    got = at.prompt_attention(q, k, v, cu, max(lens), causal=causal, out=buf[:T])
    assert bool((buf[T:] == 9).all())
    a = 0
    for n in lens:
        if n:
            ref, bound = attend(q[a:a + n], k[a:a + n], v[a:a + n], 0, D ** -0.5, causal, 0)
            check(got[a:a + n], ref, bound, f"prompt of {n}")
        a += n


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_prompt_non_finite(dev, dt, D):
    """A later token's infinities and NaN do not reach earlier rows."""
    import torch
    from inferflux_amd import attention as at
    note(f"prompt non-finite {dt} D={D}")
    g, n = gen(dev, D), 150
    q, k, v = (torch.randn(n, h, D, generator=g, device=dev).to(dt_of(dt)) for h in (4, 2, 2))
    v[100, 0, 3], v[120, 1, D - 1], v[121, 1, D - 1] = float("nan"), float("inf"), -float("inf")
    k[140, 0, 7] = float("nan")
    k[130, 1, 1] = float("inf")
    cu = i32([0, n], dev)
    got = at.prompt_attention(q, k, v, cu, n)
    check(got, *attend(q, k, v, 0, D ** -0.5))
    assert bool(torch.isfinite(got[:100]).all())


def test_prompt_out_types_and_stray_rows(dev):
    """fp32 output; rows that belong to no prompt are left as they were."""
    import torch
    from inferflux_amd import attention as at
    note("prompt fp32 out")
    g = gen(dev, 2)
    q, k, v = (torch.randn(90, h, 128, generator=g, device=dev).half() for h in (4, 2, 2))
    out = torch.full((90, 4, 128), 9.0, device=dev)
    at.prompt_attention(q, k, v, i32([10, 40, 80], dev), 40, out=out)
    for a, b in ((10, 40), (40, 80)):
        check(out[a:b], *attend(q[a:b], k[a:b], v[a:b], 0, 128 ** -0.5))
    assert bool((out[:10] == 9).all()) and bool((out[80:] == 9).all())


# ------------------------------------------------------------ a serving program
def test_step_after_step(dev, ws):
    """Prompts read in chunks, then decoded token by token, next to each other
    in one paged cache: after every step each request's rows equal the
    attention over all of its tokens so far, taken from the rows themselves."""
    import torch
    from inferflux_amd import attention as at
    note("serving steps")
    Hq, Hkv, D, P, B = 8, 2, 128, 16, 5
    g = gen(dev, 9)
    steps = [[40, 3, 0, 17, 1], [25, 1, 60, 1, 1], [1, 1, 1, 1, 0], [1, 0, 1, 30, 1], [1, 1, 1, 1, 1]]
    pages = 40
    kc, vc = at.kv_cache(pages, Hkv, D, P, torch.bfloat16, dev)
    kc.fill_(float("nan")), vc.fill_(float("nan"))
    table = torch.full((B, 10), -1, dtype=torch.int32, device=dev)
    free, count = torch.randperm(pages, generator=g, device=dev).int(), i32([pages], dev)
    freq = 1e6 ** (-torch.arange(D // 2, dtype=torch.float64, device=dev) * 2 / D)
    ctx = torch.zeros(B, dtype=torch.int32, device=dev)
    have = [[] for _ in range(B)]
    room = 130
    for new in steps:
        p = at.plan_batch(ctx, i32(new, dev), table, free, count, P, room)
        rows = torch.randn(room, (Hq + 2 * Hkv) * D, generator=g, device=dev)
        q, k, v = (x.unflatten(1, (-1, D)) for x in rows.split([Hq * D, Hkv * D, Hkv * D], dim=1))
        qr = torch.zeros(room, Hq, D, dtype=torch.bfloat16, device=dev)
        at.rope_append(q, k, v, p.positions, p.slots, kc, vc, freq, q_out=qr)
        out = torch.full((room, Hq, D), 9.0, device=dev)
        at.paged_attention(qr, kc, vc, table, p.cu_q, p.kv_len, max(new), 160, out=out, workspace=ws)
        assert p.status.item() == 0 and p.cu_q.tolist() == [sum(new[:b]) for b in range(B + 1)]
        a = 0
        for b, n in enumerate(new):
            pos = torch.arange(len(have[b]), len(have[b]) + n, device=dev)
            kr = rotate(k[a:a + n].double(), pos, freq, False)[0].bfloat16()
            have[b] += list(zip(kr, v[a:a + n].bfloat16()))
            if n:
                kk, vv = (torch.stack([x[i] for x in have[b]]) for i in (0, 1))
                # the cache's keys may differ from these by one rounding where
                # fp32 and fp64 fall to different sides; take the cache's own
                ck, cv = gather_cache(kc, vc, table[b], len(have[b]))
                assert torch.equal(cv, vv.double())
                assert bool(((ck - kk.double()).abs() <= 2.0 ** -7 * kk.double().abs() + 1e-30).all())
                check(out[a:a + n], *attend(qr[a:a + n], ck, cv, len(have[b]) - n, D ** -0.5))
            a += n
        assert bool((out[a:] == 9).all())
        ctx, count = p.kv_len, p.free_left
    assert count.item() == pages - sum(-(-len(h) // P) for h in have)


def test_between_the_projections(dev, ws):
    """A decoder layer's attention from the residual and back to it: RMSNorm +
    Q8_1, Q/K/V by the grouped Q4_K GEMV, plan, rotation and cache write, paged
    attention, Q8_1, O accumulated.  The attention is checked on what the GEMV
    wrote, the O projection on what the attention wrote."""
    import torch
    from inferflux_amd import attention as at
    from inferflux_amd import ops, synth
    note("attention between the projections")
    Hq, Hkv, D, hidden, P = 4, 2, 128, 512, 16
    new = [1, 1, 6, 1]
    T = sum(new)
    g = gen(dev, 4)
    W = [torch.from_numpy(synth.blocks(ops.Q4_K, n, hidden, seed=i)).to(dev)
         for i, n in enumerate((Hq * D, Hkv * D, Hkv * D))]
    Wo = torch.from_numpy(synth.blocks(ops.Q4_K, hidden, Hq * D, seed=8)).to(dev)
    x = torch.randn(T, hidden, generator=g, device=dev)
    norm = torch.ones(hidden, dtype=torch.float16, device=dev)
    kc, vc = at.kv_cache(12, Hkv, D, P, torch.float16, dev)
    ctx = [20, 0, 33, 15]
    table = i32([[1, 2, -1], [-1, -1, -1], [5, 6, 7], [8, -1, -1]], dev)
    for b, c in enumerate(ctx):
        if c:
            put_cache(kc, vc, table[b], torch.randn(c, Hkv, D, generator=g, device=dev),
                      torch.randn(c, Hkv, D, generator=g, device=dev))
    a8 = ops.rmsnorm_quantize_q8_1(x, norm)
    q, k, v = (y.view(T, -1, D) * 0.1 for y in
               ops.qgemv_grouped(ops.Q4_K, W, a8, T, [Hq * D, Hkv * D, Hkv * D], hidden))
    p = at.plan_batch(i32(ctx, dev), i32(new, dev), table, i32([9, 10, 11, 0], dev), i32([4], dev), P, T)
    freq = 1e6 ** (-torch.arange(D // 2, dtype=torch.float64, device=dev) * 2 / D)
    qr = at.rope_append(q, k, v, p.positions, p.slots, kc, vc, freq)
    o = at.paged_attention(qr, kc, vc, table, p.cu_q, p.kv_len, 6, 48, workspace=ws)
    y = x.clone()
    ops.qgemv(ops.Q4_K, Wo, ops.quantize_q8_1(o.view(T, Hq * D)), T, hidden, Hq * D, out=y, mode=ops.ACCUM)
    # pages of 16: 20 + 1, 33 + 6 and 15 + 1 tokens fit the pages held, 0 + 1 takes one
    assert p.status.item() == 0 and p.free_left.item() == 3
    a = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        kk, vv = gather_cache(kc, vc, table[b], c + n)
        assert torch.equal(vv[c:], v[a:a + n].half().double())
        check(o[a:a + n], *attend(qr[a:a + n], kk, vv, c, D ** -0.5))
        a += n
    wd = ops.dequantize(ops.Q4_K, Wo, hidden, Hq * D).double()
    want = x.double() + o.view(T, -1).double() @ wd.T
    # Q8_1 of the attention's rows: half a step of 1/127 of a block's largest
    # value, over 512 of them
    tol = (o.view(T, -1, 32).abs().amax(-1, keepdim=True).double() / 254).expand(-1, -1, 32).reshape(T, -1) @ wd.abs().T
    assert bool(((y.double() - want).abs() <= 1.1 * tol + 1e-3 * want.norm(dim=1, keepdim=True)).all())


def test_captured_steps_share_a_workspace(dev):
    """Two captured steps (different shapes, one workspace, one stream) replayed
    in turn with new inputs, eager calls between them: each replay equals the
    eager result."""
    import torch
    from inferflux_amd import attention as at
    note("graphs")
    ws = at.workspace(dev)
    xs = [Batch(dev, [3000, 50, 700], [1, 1, 1], 16, 2, 128, 64, "f16", seed=1),
          Batch(dev, [1500, 64], [60, 2], 8, 2, 128, 16, "f16", seed=2)]
    graphs = []
    for x in xs:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            x.run(ws)
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            x.run(ws)
        graphs.append(gr)
    for i in range(3):
        for x, gr in zip(xs, graphs):
            x.q.copy_(torch.randn(x.q.shape, generator=gen(dev, 50 + i), device=dev))
            x.out.fill_(9.0)
            gr.replay()
            torch.cuda.synchronize()
            got = x.out.clone()
            x.verify()
            x.run(ws)
            assert torch.equal(got, x.out)
    # a plan and an append replayed for another step's lengths
    ctx, new = i32([5, 70], dev), i32([3, 2], dev)
    table, free, count = i32([[0, 1, 2], [3, 4, 5]], dev), i32([6, 7, 8], dev), i32([3], dev)
    kc, vc = at.kv_cache(9, 1, 64, 64, torch.float16, dev)
    q, k, v = (torch.randn(8, h, 64, generator=gen(dev, 3), device=dev) for h in (2, 1, 1))
    freq = torch.ones(32, dtype=torch.float64, device=dev)
    out = at.plan_batch(ctx, new, table, free, count, 64, 8)
    qo = torch.zeros(8, 2, 64, dtype=torch.float16, device=dev)
    gr = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(gr):
        at.plan_batch(ctx, new, table, free, count, 64, 8, out=out)
        at.rope_append(q, k, v, out.positions, out.slots, kc, vc, freq, q_out=qo)
    for c, n in (([5, 70], [3, 2]), ([0, 128], [1, 6]), ([9, 9], [0, 0])):
        ctx.copy_(i32(c, dev)), new.copy_(i32(n, dev))
        qo.zero_(), kc.zero_(), vc.zero_()
        table.copy_(i32([[0, 1, 2], [3, 4, 5]], dev))
        gr.replay()
        torch.cuda.synchronize()
        assert out.cu_q.tolist() == [0, n[0], sum(n)]
        m = sum(n)
        assert bool((qo[m:] == 0).all()) and (m == 0 or bool((qo[:m] != 0).any()))
        sl = out.slots[:m].long()
        assert torch.equal(vc[sl // 64, :, sl % 64 // 8, :, sl % 8], v[:m].half())
        assert int((vc != 0).sum()) == int((v[:m].half() != 0).sum())


def test_other_stream(dev, ws):
    import torch
    from inferflux_amd import attention as at
    note("other stream")
    x = Batch(dev, [2000, 90], [1, 1], 16, 2, 128, 64, "bf16", seed=1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    x.run(ws, stream=s)
    o = at.prompt_attention(x.q, x.q[:, :2], x.q[:, 2:4], i32([0, 2], dev), 2, stream=s)
    s.synchronize()
    x.verify()
    check(o, *attend(x.q, x.q[:, :2], x.q[:, 2:4], 0, 128 ** -0.5))


def test_wrapper_refusals(dev, ws):
    import torch
    from inferflux_amd import attention as at
    from inferflux_amd import ops
    note("refusals")
    x = Batch(dev, [20, 30], [1, 1], 8, 2, 128, 16, "f16")
    with pytest.raises(TypeError):
        at.paged_attention(x.q.bfloat16(), x.kc, x.vc, x.table, x.cu, x.kvt, 1, 30, workspace=ws)
    with pytest.raises(TypeError):
        at.paged_attention(x.q, x.kc, x.vc, x.table.long(), x.cu, x.kvt, 1, 30, workspace=ws)
    with pytest.raises(ValueError):
        at.paged_attention(x.q, x.kc, x.vc, x.table, x.cu[:2], x.kvt, 1, 30, workspace=ws)
    with pytest.raises(ValueError):
        at.paged_attention(x.q, x.kc, x.vc, x.table[:, ::2], x.cu, x.kvt, 1, 30, workspace=ws)
    with pytest.raises(ValueError):
        at.paged_attention(x.q, x.kc.cpu(), x.vc.cpu(), x.table, x.cu, x.kvt, 1, 30, workspace=ws)
    with pytest.raises(ops.NotHandled):
        at.paged_attention(x.q, x.kc, x.vc, x.table, x.cu, x.kvt, 1, 3000)  # no workspace
    with pytest.raises(ops.NotHandled):
        at.paged_attention(x.q, x.kc, x.vc, x.table, x.cu, x.kvt, 1, 30, scale=-1.0, workspace=ws)
    with pytest.raises(ValueError):
        at.rope_append(x.q, x.q[:, :3], x.q[:, :2], x.cu[:2], x.cu[:2], x.kc, x.vc)
    with pytest.raises(TypeError):
        at.rope_append(x.q, x.q[:, :2].float(), x.q[:, :2], x.cu[:2], x.cu[:2], x.kc, x.vc)
    with pytest.raises(TypeError):
        at.prompt_attention(x.q.float(), x.q[:, :2].float(), x.q[:, :2].float(), x.cu, 2)
    with pytest.raises(ops.NotHandled):
        at.prompt_attention(x.q, x.q[:, :2], x.q[:, :2], x.cu, 2, causal=False, window=3)
    with pytest.raises(ops.NotHandled):  # an output in an input's place
        at.plan_batch(x.kvt, x.cu, x.table, x.cu, x.cu, 16, 2, out=at.BatchPlan(*([x.cu] * 6)))
    with pytest.raises(ValueError):
        at.plan_batch(x.kvt, x.cu, x.table, x.cu, x.cu, 16, 9, out=at.BatchPlan(*([x.cu] * 6)))
    assert at.paged_attention(x.q[:0], x.kc, x.vc, x.table, x.cu, x.kvt, 1, 30).shape[0] == 0
