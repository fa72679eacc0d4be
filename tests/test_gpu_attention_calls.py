"""The attention operators in calls that a serving program makes beside the
plain ones: on other streams without a wait, next to memory that holds
nonsense, with windows inside long chunks."""
import pytest

from tests.attn_ref import attend, check
from tests.test_gpu_attention import Batch, counters_clear, dev, dt_of, gen, i32, ws  # noqa: F401
from tests.test_gpu_parity import note

pytestmark = pytest.mark.gpu


def test_outputs_on_a_stream_that_waits_for_nothing(dev, ws):
    """Inputs are of stream s, and the current stream still has work to do on
    blocks of the outputs' sizes that were freed there: it writes to none of
    the outputs made on s."""
    import torch
    from inferflux_amd import attention as at
    note("outputs on another stream")
    x = Batch(dev, [300, 90], [40, 1], 8, 2, 128, 16, "f16", seed=2)
    ctx, new = i32([260, 89], dev), i32([40, 1], dev)
    free, count = i32([3, 1, 2, 0], dev), i32([4], dev)
    table = torch.zeros_like(x.table)
    kc, vc = at.kv_cache(64, 2, 128, 16, torch.float16, dev)
    slots = torch.arange(x.T, dtype=torch.int32, device=dev)
    calls = {
        "plan": lambda s: at.plan_batch(ctx, new, table, free, count, 16, x.T, stream=s),
        "append": lambda s: at.rope_append(x.q, x.q[:, :2], x.q[:, 2:4], slots, slots, kc, vc, stream=s),
        "paged": lambda s: at.paged_attention(x.q, x.kc, x.vc, x.table, x.cu, x.kvt, 40, 300, workspace=ws,
                                              stream=s),
        "prompt": lambda s: at.prompt_attention(x.q, x.q[:, :2], x.q[:, 2:4], x.cu, 40, stream=s),
    }
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for what, call in calls.items():
        want = call(None)  # and the sizes of the blocks that a call asks for
        torch.cuda.synchronize()
        want = [w.clone() for w in want] if what == "plan" else [want.clone()]
        n = sum(w.numel() * w.element_size() for w in want)
        blocks = [torch.empty(n, dtype=torch.uint8, device=dev) for _ in range(4)]
        torch.cuda.synchronize()
        torch.cuda._sleep(20_000_000)
        for b in blocks:
            b.fill_(77)
        del blocks, b  # free for the current stream, with the fills pending
        got = call(s)
        s.synchronize()
        torch.cuda.synchronize()  # the fills are done
        for g, w in zip(got if what == "plan" else [got], want):
            assert torch.equal(g, w), what


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 40)])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 64), (3, 1, 96), (4, 2, 128), (2, 1, 256)])
@pytest.mark.parametrize("lens", [(70, 33, 1), (127, 64, 200), (16, 129, 33)])
def test_prompt_rows_around_a_prompt_are_not_read(dev, dt, causal, window, Hq, Hkv, D, lens):
    """K and V rows behind a prompt's last, its neighbour's or no prompt's, hold
    NaN and infinities: the outer prompts have the same bits as beside zeros.
    (A value read there would meet a probability of 0, and the wave would take
    its rows again in another order of sums.)"""
    import torch
    from inferflux_amd import attention as at
    note(f"prompt neighbours {dt} causal={causal} window={window} D={D} lens={lens}")
    g = gen(dev, D + lens[0])
    stray, T = 5, sum(lens) + 10
    a, b, c, d = (stray + sum(lens[:i]) for i in range(4))
    q, k, v = (torch.randn(T, h, D, generator=g, device=dev).to(dt_of(dt)) for h in (Hq, Hkv, Hkv))
    cu = i32([a, b, c, d], dev)
    outs = []
    for fill in ((0.0, 0.0), (float("nan"), float("inf"))):
        for t in (k, v):
            t[:a], t[b:c], t[d:] = fill[0], fill[1], fill[0]
            t[b:c:2] = fill[0]
        out = torch.full((T, Hq, D), 9.0, dtype=dt_of(dt), device=dev)
        at.prompt_attention(q, k, v, cu, max(lens), causal=causal, window=window, out=out)
        assert bool((out[:a] == 9).all()) and bool((out[d:] == 9).all())
        outs.append(out)
    for lo, hi in ((a, b), (c, d)):
        assert torch.equal(outs[0][lo:hi], outs[1][lo:hi])
        check(outs[1][lo:hi], *attend(q[lo:hi], k[lo:hi], v[lo:hi], 0, D ** -0.5, causal, window))
    assert bool(torch.isnan(outs[1][b:c]).any())


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("window", [300, 1501, 2944])
@pytest.mark.parametrize("Hq,Hkv,D,P,kv,new", [
    (4, 2, 64, 16, [4300, 700, 40], [200, 130, 1]), (6, 2, 96, 32, [4100], [131]),
    (8, 2, 128, 64, [4500, 4001, 90], [100, 33, 90]), (2, 1, 256, 16, [4200, 650], [150, 7])])
def test_paged_chunks_in_windows(dev, ws, dt, window, Hq, Hkv, D, P, kv, new):
    """Row tiles that see stages in part where their windows begin, whole ones
    behind them and their causal end: cut into chunks, whose number differs
    between the tiles of a request, and not; then with nonsense in the pages
    before the window."""
    import torch
    from inferflux_amd import attention as at
    note(f"paged tile window={window} {dt} Hq={Hq} Hkv={Hkv} D={D} P={P} kv={kv} new={new}")
    assert at.paged_workspace_bytes(len(kv), sum(new), Hq, Hkv, D, max(new), max(kv)) > 0
    x = Batch(dev, kv, new, Hq, Hkv, D, P, dt, seed=D + window, extra_rows=2)
    x.run(ws, window=window)
    first = x.out.clone()
    x.verify(window=window)
    for _ in range(2):
        x.out.fill_(9.0)
        x.run(ws, window=window)
        assert torch.equal(first, x.out)
    x.run(ws, window=window, max_kv=600)  # needs no workspace: not split
    x.verify(window=window)
    for b, (n, L) in enumerate(zip(new, kv)):
        gone = x.table[b, :max(0, (L - n - window + 1) // P)].long()  # pages that no row sees
        x.kc[gone], x.vc[gone] = float("nan"), float("inf")
    x.run(ws, window=window)
    x.verify(window=window)
    assert counters_clear(ws)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("kv,new", [([5000], [70]), ([2300, 3000, 1], [64, 129, 1])])
def test_paged_chunks_split_heads_of_96(dev, ws, dt, kv, new):
    """Split sums of an odd number of dim tiles."""
    import torch
    from inferflux_amd import attention as at
    note(f"paged tile split {dt} D=96 kv={kv} new={new}")
    assert at.paged_workspace_bytes(len(kv), sum(new), 6, 2, 96, max(new), max(kv)) > 0
    x = Batch(dev, kv, new, 6, 2, 96, 16, dt, seed=5)
    x.run(ws)
    first = x.out.clone()
    x.verify()
    x.run(ws)
    assert torch.equal(first, x.out)
    assert counters_clear(ws)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("window", [129, 400, 1000])
@pytest.mark.parametrize("Hq,Hkv,D,lens", [
    (4, 2, 64, [1201, 500]), (3, 1, 96, [1100]), (4, 2, 128, [30, 1333]), (2, 1, 256, [1050, 401])])
def test_prompt_in_windows(dev, dt, window, Hq, Hkv, D, lens):
    """Prompts longer than their window."""
    import torch
    from inferflux_amd import attention as at
    note(f"prompt window={window} {dt} Hq={Hq} Hkv={Hkv} D={D} lens={lens}")
    g, T = gen(dev, D + window), sum(lens)
    q, k, v = (torch.randn(T, h, D, generator=g, device=dev).to(dt_of(dt)) for h in (Hq, Hkv, Hkv))
    cu = i32([sum(lens[:b]) for b in range(len(lens) + 1)], dev)
    got = at.prompt_attention(q, k, v, cu, max(lens), window=window)
    assert torch.equal(got, at.prompt_attention(q, k, v, cu, max(lens), window=window))
    a = 0
    for n in lens:
        check(got[a:a + n], *attend(q[a:a + n], k[a:a + n], v[a:a + n], 0, D ** -0.5, True, window),
              f"prompt of {n}")
        a += n


def test_counts_that_pass_32_bits(dev, ws):
    from inferflux_amd import attention as at
    note("counts past 32 bits")
    x = Batch(dev, [20, 30], [1, 1], 8, 2, 128, 16, "f16")
    for bad in (dict(window=2 ** 32 + 1), dict(max_q=2 ** 32 + 1), dict(max_kv=-1)):
        with pytest.raises(ValueError):
            x.run(ws, **bad)
    with pytest.raises(ValueError):
        at.prompt_attention(x.q, x.q[:, :2], x.q[:, 2:4], x.cu, 2, window=2 ** 32 + 1)
    for bad in (dict(page_size=2 ** 32 + 16, max_tokens=2), dict(page_size=16, max_tokens=-1),
                dict(page_size=16, max_tokens=2 ** 32)):
        with pytest.raises(ValueError):
            at.plan_batch(x.kvt, x.kvt, x.table, x.cu, x.cu, **bad)


def test_captured_calls_on_a_side_stream(dev, ws):
    """Calls on a stream that a capture forks to, their outputs allocated in the
    capture: replays with new inputs equal the eager results."""
    import torch
    from inferflux_amd import attention as at
    note("capture with a side stream")
    x = Batch(dev, [300, 90], [40, 1], 8, 2, 128, 16, "f16", seed=6)
    side, ws2 = torch.cuda.Stream(), at.workspace(dev)

    def both(stream, w):
        o = at.paged_attention(x.q, x.kc, x.vc, x.table, x.cu, x.kvt, 40, 300, workspace=w, stream=stream)
        return o, at.prompt_attention(x.q, x.q[:, :2], x.q[:, 2:4], x.cu, 40, stream=stream)

    both(None, ws2)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        o, p = both(side, ws2)
        here.wait_stream(side)
        outs = o + 0, p + 0
    for i in range(3):
        x.q.copy_(torch.randn(x.q.shape, generator=gen(dev, i), device=dev))
        gr.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        for a, b in zip(got, both(None, ws)):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_two_calls_at_once(dev):
    """Split calls on two streams, each with its workspace, at the same time."""
    import torch
    from inferflux_amd import attention as at
    note("two streams")
    xs = [Batch(dev, [6000, 50, 3000], [1, 1, 1], 16, 2, 128, 64, "f16", seed=1),
          Batch(dev, [4000, 64], [70, 2], 8, 2, 128, 16, "f16", seed=2)]
    wss = [at.workspace(dev) for _ in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(20):
        for x, w, s in zip(xs, wss, streams):
            x.run(w, stream=s)
    torch.cuda.synchronize()
    for x, w in zip(xs, wss):
        x.verify()
        assert counters_clear(w)
