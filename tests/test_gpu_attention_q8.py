"""The 8-bit cache on the GPU against its definition in 64 bits (tests/q8_ref.py):
codes and scales as they are written, tokens read back, and the attention over
them, of single tokens, chunks and trees of drafts."""
import math
import random

import pytest

from tests import drafts_ref, q8_ref
from tests.attn_ref import TINY, U, check
from tests.test_gpu_attention import dt_of, gen, i32
from tests.test_gpu_drafts import cu_of, signed, tree_masks
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


def wild_cache(dev, pages, Hkv, D, P):
    """A cache of slots that nobody has written: codes of -128, scales NaN."""
    from inferflux_amd import attention_q8 as q8
    c = q8.kv_cache(pages, Hkv, D, P, device=dev)
    c.k.fill_(-128), c.v.fill_(-128), c.scales.fill_(math.nan)
    return c


# --------------------------------------------------------------- write and read
def run_append(dev, T, Hq, Hkv, D, P, src, qdt, rot, inter, slots=None, pos=None, side=0, spoil=None, pages=None):
    import torch
    from inferflux_amd import attention_q8 as q8
    g = gen(dev, T + D)
    pages = pages or -(-T // P) + 2
    n = ((Hq + 2 * Hkv) * D) + side
    rows = torch.randn(T, n, generator=g, device=dev).to(dt_of(src))
    q, k, v = (x.unflatten(1, (-1, D)) for x in rows[:, :n - side].split([Hq * D, Hkv * D, Hkv * D], 1))
    v.mul_(torch.exp(torch.randn(T, Hkv, 1, generator=g, device=dev)).to(v.dtype))
    if spoil:
        spoil(k, v)
    if slots is None:
        slots = torch.randperm(pages * P, generator=g, device=dev)[:T].int()
    if pos is None:
        pos = torch.randint(0, 100000, (T,), generator=g, device=dev).int()
    freq = None if not rot else 1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
    c = wild_cache(dev, pages, Hkv, D, P)
    want = q8.Q8Cache(*(x.clone() for x in c))
    q_out = torch.full((T, Hq, D), 7.0, dtype=dt_of(qdt), device=dev)
    q8.rope_append(q, k, v, pos, slots, c, freq, interleaved=inter, q_out=q_out)
    ok = (slots >= 0) & (slots < pages * P)
    at = slots[ok]
    kr = q8_ref.rotate(k, pos, freq, inter)
    kc, ks = q8_ref.quantise(kr[ok])
    vc, vs = q8_ref.quantise(v[ok].double())
    q8_ref.put(want, at, kc, ks, vc, vs)
    assert torch.equal(c.scales.nan_to_num(-1), want.scales.nan_to_num(-1)), "scales"
    assert torch.equal(c.v, want.v), "V's codes"
    # the definition's angles carry 1e-5 / 2^52 turns: a code at a border may go either way
    off = (c.k.int() - want.k.int()).abs()
    assert int(off.max()) <= 1 and int((off > 0).sum()) <= 1 + off.numel() // 10 ** 8, "K's codes"
    # Q in 32 bits: an angle to 2^-23 of half a turn, two products and their sum, one rounding
    qr = q8_ref.rotate(q, pos, freq, inter)
    bound = (q.double().abs().amax(-1, keepdim=True) * 8 * 2.0 ** -23).expand_as(qr)
    tol = bound + U[dt_of(qdt)] * (qr.abs() + bound) + TINY[dt_of(qdt)]
    diff = (q_out.double() - qr).abs() - tol
    assert float(diff[ok].max() if ok.any() else -1.0) <= 0, "q"
    assert torch.all(q_out[~ok] == 7.0), "q of tokens without a slot"
    # read back, slots outside the cache among them
    ask = torch.cat([slots, i32([-1, pages * P, 1 << 30, -(1 << 31)], dev)])
    inside = (ask >= 0) & (ask < pages * P)
    for dt in ("f32", "f16", "bf16"):
        kk, vv = q8.read_rows(c, ask, dtype=dt_of(dt))
        a, b, _ = q8_ref.get(c, ask[inside])
        # a product of 7 and 8 bits is exact in 32
        for got, ref in ((kk, a), (vv, b)):
            assert torch.equal(got[inside].nan_to_num(-3.0), ref.to(torch.float32).to(dt_of(dt)).nan_to_num(-3.0)), "read"
            assert not got[~inside].any(), "read outside"
    return c, kr, v


@pytest.mark.parametrize("src,qdt", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("Hq,Hkv,D,P,rot,inter", [
    (16, 2, 128, 64, 128, False), (40, 8, 128, 16, 128, True), (6, 6, 64, 32, 32, False), (9, 3, 96, 16, 96, False),
    (8, 2, 256, 128, 256, False), (3, 1, 32, 256, 16, True), (2, 1, 160, 16, 80, False), (4, 4, 224, 16, 0, False),
    (1, 1, 64, 16, 64, False)])
@pytest.mark.parametrize("T", [1, 37])
def test_append_and_read(dev, src, qdt, Hq, Hkv, D, P, rot, inter, T):
    note(f"append q8 {src} {Hq}/{Hkv} D={D} P={P} rot={rot} {inter} T={T}")
    run_append(dev, T, Hq, Hkv, D, P, src, qdt, rot, inter, side=(0, 5)[T > 1])


@pytest.mark.parametrize("T,Hkv,P,first", [(2048, 8, 16, 0), (2500, 2, 64, 7), (5000, 1, 16, 13), (2100, 3, 256, 1),
                                           (4096, 2, 32, 0)])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_append_runs_of_tokens(dev, T, Hkv, P, first, D):
    """Prompts: slots one behind the other from anywhere in a page, holes, runs of
    requests next to each other."""
    import torch
    note(f"append q8 runs T={T} Hkv={Hkv} P={P} D={D}")
    rng = random.Random(T + D)
    pages = -(-(T + first + 40) // P) + 1
    slots = list(range(first, first + T))
    for i in range(0, T, rng.randint(50, 90)):
        slots[i] = -1
    cut = T // 3  # the last third to the front of the cache's end, backwards by requests
    slots = slots[cut:] + slots[:cut]
    run_append(dev, T, 2, Hkv, D, P, "f16", "f16", 64, False, slots=i32(slots, dev), pages=pages,
               pos=torch.arange(T, device=dev).int())


def test_append_corners(dev):
    """Rows of zeros, of one value, of ties, of the smallest and largest values,
    of infinities and NaN; tokens without a slot."""
    import torch
    from inferflux_amd import attention_q8 as q8
    note("append q8 corners")

    def spoil(k, v):
        for x in (k, v):
            x[0] = 0.0
            x[1, 0] = 0.0
            x[1, 0, 3] = -2.5
            x[2, 1, 5] = math.inf
            x[3, 0, 64] = math.nan
            x[4, 1, 127] = -math.inf
            x[5] = torch.finfo(x.dtype).max
            x[6] = torch.finfo(x.dtype).smallest_normal
            # scale exactly 1: ties at .5 go to the even code
            x[7] = torch.arange(128, device=x.device) - 63.5
            x[7, :, 0] = 127.0
            # a largest value just above and just below 127 * 1.0078125
            x[8] = 1.0
            x[8, :, 9] = 127.0 * 1.0078125
            x[9, :, 9] = 127.0 * 1.0
    for src in ("f32", "bf16", "f16"):
        c, kr, v = run_append(dev, 12, 3, 2, 128, 16, src, "f16", 0, False, spoil=spoil,
                              slots=i32([0, 1, 2, 3, 4, 5, 6, 7, 8, 9, -1, 1 << 20], dev))
        k, _ = q8.read_rows(c, i32([2, 3, 4, 0], dev))
        assert k[0, 1].isnan().all() and not k[0, 0].isnan().any() and k[1, 0].isnan().all()
        assert k[2, 1].isnan().all() and not k[3].any()
    run_append(dev, 3, 3, 2, 128, 16, "f32", "f16", 128, False, slots=i32([-1, -1, -5], dev))


# ------------------------------------------------------------------ attention
def make_cache(dev, ctx, new, Hkv, D, P, seed, spread=0.5, extra=3):
    """Cache, table and the slots of each request's tokens."""
    import torch
    g = gen(dev, seed)
    kv = [max(c + n, 0) for c, n in zip(ctx, new)]
    total = [-(-x // P) for x in kv]
    order = torch.randperm(sum(total) + extra, generator=g, device=dev).int()
    cache = wild_cache(dev, sum(total) + extra, Hkv, D, P)
    W = max(total) + 1
    table = torch.full((len(ctx), W), -5, dtype=torch.int32, device=dev)
    used, slots = 0, []
    for b, x in enumerate(kv):
        table[b, :total[b]] = order[used:used + total[b]]
        used += total[b]
        j = torch.arange(x, device=dev)
        s = table[b].long()[j // P] * P + j % P
        k, v = torch.randn(2, x, Hkv, D, generator=g, device=dev, dtype=torch.float64)
        v = v * torch.exp(spread * torch.randn(x, Hkv, 1, generator=g, device=dev))
        if x:
            q8_ref.put(cache, s, *q8_ref.quantise(k), *q8_ref.quantise(v))
        slots.append(s)
    return cache, table, slots


def run_paged(dev, qdt, ctx, new, Hq, Hkv, D, P, masks=None, window=0, seed=1, spread=0.5, spoil=None, out_dtype=None,
              scale=None, max_kv=None, workspace=None, q_scale=1.0, side=0):
    """paged_attention of the 8-bit cache against 64 bits."""
    import torch
    from inferflux_amd import attention as at, attention_q8 as q8
    dtype = dt_of(qdt)
    cache, table, slots = make_cache(dev, ctx, new, Hkv, D, P, seed, spread)
    if spoil:
        spoil(cache, slots)
    T = sum(new)
    q = (torch.randn(T + 2, Hq * D + side, generator=gen(dev, seed + 1), device=dev) * q_scale).to(dtype)
    q = q[:, :Hq * D].unflatten(1, (Hq, D))
    kv = [max(c + n, 0) for c, n in zip(ctx, new)]
    out = torch.full((T + 2, Hq, D), 7.0, dtype=out_dtype or dtype, device=dev)
    ws = at.workspace(dev) if workspace is None else workspace
    scale = scale or 1.5 * D ** -0.5
    m = None if masks is None else torch.tensor([signed(x) for x in masks] + [-1, -1], device=dev)
    q8.paged_attention(q, cache, table, i32(cu_of(new), dev), i32(kv, dev), max(max(new), 1), max_kv or max(max(kv), 1),
                       scale=scale, window=window, masks=m, out=out, workspace=ws)
    t = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        if n:
            if masks is not None:
                seen = drafts_ref.seen_by_tree(masks[t:t + n], c, n, kv[b])
            else:
                j, pos = torch.arange(kv[b]), c + torch.arange(n)[:, None]
                seen = (j <= pos) & ((j > pos - window) if window else True)
            k, v, vs = q8_ref.get(cache, slots[b])
            want, bound = drafts_ref.attend_seen(q[t:t + n], k, v, seen, scale, weigh=U[torch.float16])
            # fp16 of probability times scale: half of 2^-24, scaled by 2^6 against a size of up to twice the largest
            # scale, times a code
            if kv[b]:
                bound = bound + kv[b] * 2.0 ** -30 * 127 * float(vs.nan_to_num(0).amax())
            check(out[t:t + n], want, bound, f"request {b}")
        t += n
    assert torch.all(out[T:] == 7.0), "rows behind the last request"
    assert not ws[:32768].any(), "counters left"
    return out


SHAPES = [(16, 2, 128, 64), (40, 8, 128, 16), (6, 6, 64, 32), (9, 3, 96, 16), (8, 2, 256, 128), (7, 1, 128, 256),
          (32, 1, 64, 16)]


@pytest.mark.parametrize("qdt", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,D,P", SHAPES)
@pytest.mark.parametrize("lens", ["one", "many", "long"])
def test_decode(dev, qdt, Hq, Hkv, D, P, lens):
    note(f"q8 decode {qdt} {Hq}/{Hkv} D={D} P={P} {lens}")
    ctx, new = {"one": ([0], [1]), "many": ([0, 1, 15, 31, 32, 127, 300, 64, 5], [1, 1, 1, 1, 0, 1, 1, 1, 1]),
                "long": ([5000, 130, 2047], [1, 1, 1])}[lens]
    run_paged(dev, qdt, ctx, new, Hq, Hkv, D, P, seed=D + P)


@pytest.mark.parametrize("qdt", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,D,P", SHAPES)
@pytest.mark.parametrize("lens", ["prompt", "chunk", "mixed", "crowd"])
def test_chunks(dev, qdt, Hq, Hkv, D, P, lens):
    note(f"q8 chunks {qdt} {Hq}/{Hkv} D={D} P={P} {lens}")
    ctx, new = {"prompt": ([0, 0], [150, 33]), "chunk": ([1500], [70]), "mixed": ([900, 0, 17, 130, 64], [1, 65, 0, 40, 7]),
                "crowd": ([i * 37 % 400 for i in range(34)], [(1, 2, 70)[i % 3] for i in range(34)])}[lens]
    run_paged(dev, qdt, ctx, new, Hq, Hkv, D, P, seed=D + P, side=8)


@pytest.mark.parametrize("n,Hq,Hkv,D", [(1, 16, 2, 128), (3, 4, 2, 64), (100, 8, 2, 128), (40, 3, 3, 256), (2, 6, 2, 96)])
@pytest.mark.parametrize("window", [1, 30, 64, 500, 1 << 30])
def test_windows(dev, n, Hq, Hkv, D, window):
    note(f"q8 window={window} n={n} D={D}")
    run_paged(dev, "f16", [700, 3, 0], [n, n, n], Hq, Hkv, D, 16, window=window)


@pytest.mark.parametrize("qdt", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,D,P", SHAPES)
@pytest.mark.parametrize("shape", ["few", "wide", "crowd"])
def test_trees(dev, qdt, Hq, Hkv, D, P, shape):
    note(f"q8 tree {qdt} {Hq}/{Hkv} D={D} P={P} {shape}")
    rng = random.Random(Hq * 131 + D + P + len(shape))
    ctx, new = {"few": ([0, 5, 300, 64], [4, 1, 3, 4]), "wide": ([700, 63, 0], [64, 33, 9]),
                "crowd": ([rng.randint(0, 400) for _ in range(34)], [rng.choice([1, 2, 40]) for _ in range(33)] + [40])}[shape]
    run_paged(dev, qdt, ctx, new, Hq, Hkv, D, P, masks=tree_masks(rng, new), seed=D + P)


@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 128), (16, 2, 64)])
@pytest.mark.parametrize("ctx", [[0, 0], [-3, 40], [-70, -64], [1000, 1]])
@pytest.mark.parametrize("tree", [False, True])
def test_rows_that_see_nothing(dev, Hq, Hkv, D, ctx, tree):
    note(f"q8 any {Hq}/{Hkv} D={D} {ctx} {tree}")
    rng = random.Random(D + ctx[0])
    for n in (3, 12, 64):
        masks = [rng.choice([0, 0, 1 << rng.randrange(64), rng.getrandbits(64)]) for _ in range(2 * n)]
        run_paged(dev, "f16", ctx, [n, n], Hq, Hkv, D, 16, masks=masks if tree else None, seed=n)


@pytest.mark.parametrize("n,Hq,Hkv", [(1, 4, 4), (6, 4, 2), (40, 16, 2)])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("what", ["k", "v", "both", "huge"])
def test_unseen_rows_have_no_influence(dev, n, Hq, Hkv, tree, what):
    """Tokens whose K or V reads as NaN, or is far larger than the others': only
    rows that see them are hit."""
    import torch
    note(f"q8 spoilt n={n} tree={tree} {what}")
    rng = random.Random(n)
    ctx, new = [130, 61], [n, n]
    masks = tree_masks(rng, new, 6)
    if n == 1:
        masks = [0, 1]

    def spoil(cache, slots):
        P = cache.k.shape[3]
        for b in range(2):
            for j in {n // 2, n - 1} - ({0} if n > 1 else set()):
                s = int(slots[b][ctx[b] + j])
                if what in ("k", "both"):
                    cache.scales[s // P, :, s % P, 0] = math.nan
                if what in ("v", "both"):
                    cache.scales[s // P, :, s % P, 1] = math.nan
                if what == "huge":
                    cache.scales[s // P, :, s % P, 1] = 1e30
    run_paged(dev, "bf16", ctx, new, Hq, Hkv, 128, 16, masks=masks if tree else None, spoil=spoil,
              out_dtype=torch.float32)


@pytest.mark.parametrize("n,G", [(1, 4), (50, 4)])
def test_sizes_of_scales(dev, n, G):
    """V's rows of very different size, tiny and huge ones, scales of 0; scores
    far apart; queries of bfloat16 that fp16 does not hold."""
    import torch
    note(f"q8 sizes n={n}")
    run_paged(dev, "f16", [600, 40], [n, n], 2 * G, 2, 128, 16, spread=3.0, out_dtype=torch.float32)
    run_paged(dev, "f16", [600, 40], [n, n], 2 * G, 2, 128, 16, scale=3.0, out_dtype=torch.float32)
    for factor in (1e-22, 1e22):
        def spoil(cache, slots):
            cache.scales.mul_(torch.tensor([1.0, factor], device=dev))
        run_paged(dev, "bf16", [600, 40], [n, n], 2 * G, 2, 128, 16, spoil=spoil, out_dtype=torch.float32)

        def inverse(cache, slots):
            cache.scales.mul_(torch.tensor([1 / factor, 1.0], device=dev))
        run_paged(dev, "bf16", [600, 40], [n, n], 2 * G, 2, 128, 16, spoil=inverse, q_scale=factor, out_dtype=torch.float32)

    def zeros(cache, slots):
        cache.scales[:, :, ::3] = 0.0
    run_paged(dev, "f16", [600, 40], [n, n], 2 * G, 2, 128, 16, spoil=zeros)
    run_paged(dev, "bf16", [60, 40], [n, n], 2 * G, 2, 128, 16, q_scale=0.0)


@pytest.mark.parametrize("B,n,Hq,Hkv,D", [(1, 1, 16, 2, 128), (3, 1, 40, 8, 128), (70, 1, 8, 2, 64), (2, 4, 16, 2, 256),
                                          (1, 60, 16, 2, 128), (70, 33, 4, 1, 64), (300, 1, 2, 1, 128)])
def test_split_keys_repeat(dev, B, n, Hq, Hkv, D):
    """Keys cut into chunks, lengths far apart; the same bits on every call."""
    import torch
    from inferflux_amd import attention as at
    note(f"q8 split B={B} n={n} D={D}")
    rng = random.Random(B + D)
    ctx = [rng.choice([0, 30, rng.randint(0, 3000 if B < 50 else 300), 12000 if B < 5 else 1500]) for _ in range(B)]
    ctx[0] = 9000 if B < 50 else 2500
    ws = at.workspace(dev)
    a = run_paged(dev, "f16", ctx, [n] * B, Hq, Hkv, D, 16, workspace=ws)
    b = run_paged(dev, "f16", ctx, [n] * B, Hq, Hkv, D, 16, workspace=ws)
    assert torch.equal(a, b)


def test_every_kernel_is_reached(dev):
    """The shapes above go through all kernels and head sizes."""
    import torch
    from inferflux_amd import _lib, attention as at, attention_q8 as q8, drafts
    note("q8 kernels")
    lib = _lib.load()
    lib.ifx_launch_log_begin(0)
    for Hq, Hkv, D, P in SHAPES[:5]:
        for B, n in ((1, 1), (1, 64), (1, 700), (34, 40)):
            cache = q8.kv_cache(4, Hkv, D, P, device=dev)
            table = torch.zeros(B, 700 // P + 1, dtype=torch.int32, device=dev)
            q = torch.zeros(B * n, Hq, D, dtype=torch.float16, device=dev)
            cu, kv = i32([i * n for i in range(B + 1)], dev), i32([n] * B, dev)
            q8.paged_attention(q, cache, table, cu, kv, n, 60, workspace=at.workspace(dev))
    torch.cuda.synchronize()
    log = lib.ifx_launch_log_end().decode()
    for D in (64, 96, 128, 256):
        for k in ("rows16_q8", "rows_q8", "tile_q8"):
            assert f"k_attn_{k}<{D}>" in log, (k, D)
        assert f"k_attn_tile_q8<{D},1>" in log, D  # of several requests


def test_bounds_below_the_lengths(dev):
    """max_kv below a request's keys: computed whole, as the 16-bit cache's."""
    note("q8 bounds")
    run_paged(dev, "f16", [3000, 50], [1, 1], 16, 2, 128, 64, max_kv=100)
    run_paged(dev, "f16", [3000, 50], [40, 40], 16, 2, 128, 64, max_kv=100)


def test_bad_pages_stay_inside(dev):
    """Page numbers outside the cache and lengths past the table are clamped."""
    import torch
    from inferflux_amd import attention as at, attention_q8 as q8
    note("q8 bad pages")
    for n in (1, 40):
        cache, table, _ = make_cache(dev, [100, 100], [n, n], 2, 128, 16, 3)
        table[0] = 1 << 30
        q = torch.randn(2 * n, 8, 128, device=dev).half()
        o = q8.paged_attention(q, cache, table, i32([0, n, 2 * n], dev), i32([1 << 30, 100 + n], dev), n, 200,
                               workspace=at.workspace(dev))
        assert torch.isfinite(o[n:]).all()


def test_offsets_past_32_bits(dev):
    """A cache of more than 2^32 bytes of codes: pages at its end."""
    import torch
    from inferflux_amd import attention as at, attention_q8 as q8, drafts
    note("q8 large cache")
    Hkv, D, P = 8, 128, 64
    pages = (1 << 32) // (Hkv * D * P) + 40
    c = q8.kv_cache(pages, Hkv, D, P, device=dev)
    for n in (1, 40):
        ctx = 300
        table = torch.arange(pages - 8, pages, device=dev, dtype=torch.int32)[None].contiguous()
        g = gen(dev, n)
        k, v = torch.randn(2, ctx + n, Hkv, D, generator=g, device=dev)
        j = torch.arange(ctx + n, device=dev)
        slots = (table[0].long()[j // P] * P + j % P).int()
        q8.rope_append(torch.zeros(ctx + n, 16, D, device=dev), k, v, slots, slots, c)
        kk, vv = q8.read_rows(c, slots, dtype=torch.float32)
        for a, b in ((k, kk), (v, vv)):
            code, s = q8_ref.quantise(a.double())
            assert torch.equal((code * s).float(), b)
        q = torch.randn(n, 16, D, generator=g, device=dev).half()
        o = q8.paged_attention(q, c, table, i32([0, n], dev), i32([ctx + n], dev), n, ctx + n, workspace=at.workspace(dev))
        seen = torch.arange(ctx + n) <= ctx + torch.arange(n)[:, None]
        want, bound = drafts_ref.attend_seen(q, kk.double(), vv.double(), seen, D ** -0.5)
        check(o, want, bound + 400 * 2.0 ** -30 * 127 * 0.05, "large")
        if n > 1:  # the last node to the first place
            before = q8.read_rows(c, slots[-1:], dtype=torch.float32)
            drafts.keep_path(c, table, i32([0, n], dev), i32([ctx + n], dev), i32([0, n - 1] + [-1] * (n - 2), dev),
                             i32([1], dev), n)
            after = q8.read_rows(c, slots[ctx + 1:ctx + 2], dtype=torch.float32)
            assert torch.equal(before[0], after[0]) and torch.equal(before[1], after[1])


def test_keep_path(dev):
    import torch
    from inferflux_amd import attention_q8 as q8, drafts
    note("q8 keep")
    for P, Hkv, D in ((16, 2, 128), (64, 3, 32), (32, 1, 256)):
        rng = random.Random(P)
        new, ctx = [64, 0, 1, 30, 12], [5, 9, P - 1, 0, 77]
        cache, table, slots = make_cache(dev, ctx, new, Hkv, D, P, 5)
        want = q8.Q8Cache(*(x.clone() for x in cache))
        paths, accepted = [], []
        for b, n in enumerate(new):
            a = rng.choice([n // 2, n - 1, min(3, n - 1)]) if n else -1
            path = [0] + sorted(rng.sample(range(1, n), a)) if n else []
            for src, dst in drafts_ref.keep(ctx[b], n, path, a):
                (sp, si), (dp, di) = (divmod(int(slots[b][x]), P) for x in (src, dst))
                want.k[dp, :, :, di] = cache.k[sp, :, :, si]
                want.v[dp, :, di // 16, :, di % 16] = cache.v[sp, :, si // 16, :, si % 16]
                want.scales[dp, :, di] = cache.scales[sp, :, si]
            paths += path + [-1] * (n - len(path))
            accepted.append(a)
        drafts.keep_path(cache, table, i32(cu_of(new), dev), i32([c + n for c, n in zip(ctx, new)], dev), i32(paths, dev),
                         i32(accepted, dev), 64)
        assert torch.equal(cache.k, want.k) and torch.equal(cache.v, want.v)
        assert torch.equal(cache.scales.view(torch.int16), want.scales.view(torch.int16))
