"""Drafts and the 8-bit cache in calls that a serving program makes beside the
plain ones: on other streams, two at once, captured and replayed, with one
workspace for all, and what is refused."""
import random

import pytest

from tests import drafts_ref as ref
from tests.attn_ref import check
from tests.test_gpu_attention import counters_clear, gen, i32
from tests.test_gpu_attention_q8 import dev, make_cache as cache8, run_append, run_paged  # noqa: F401
from tests.test_gpu_drafts import cu_of, make_cache as cache16, signed, tree_masks
from tests.test_gpu_parity import note

pytestmark = pytest.mark.gpu


class Step:
    """Inputs of every operator for one batch of trees, 16-bit and 8-bit caches."""

    def __init__(self, dev, ctx, new, Hq, Hkv, D, P, V=3001, seed=1, behind=3):
        import torch
        rng, g = random.Random(seed), gen(dev, seed)
        self.dev, self.P, self.max_q, self.max_kv = dev, P, max(max(new), 1), max(c + n for c, n in zip(ctx, new))
        self.c8, self.table, self.slots8 = cache8(dev, ctx, new, Hkv, D, P, seed)
        *self.c16, self.table16, _ = cache16(dev, torch.float16, ctx, new, Hkv, D, P, seed)
        n, self.T = sum(new), sum(new) + behind
        trees = [ref.tree(rng, x) for x in new if x]
        pad = [0] * behind
        self.cu, self.kv = i32(cu_of(new), dev), i32([c + x for c, x in zip(ctx, new)], dev)
        self.parents = i32(sum(trees, []) + pad, dev)
        self.masks = torch.tensor([signed(m) for m in tree_masks(rng, new)] + pad, device=dev)
        self.rows = torch.randn(self.T, Hq + 2 * Hkv, D, generator=g, device=dev)
        self.heads = Hq, Hkv
        self.q = self.rows[:, :Hq].half()
        # kept: the root and the last node
        self.path = i32(sum(([0, x - 1] + [-1] * (x - 2) if x > 1 else [0] * x for x in new), []) + pad, dev)
        self.one, self.zero = i32([1] * len(new), dev), i32([0] * len(new), dev)
        self.freq = 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D)
        self.pos = torch.randint(0, 5000, (self.T,), generator=g, device=dev).int()
        # appended to places of their own behind the requests' pages
        self.own = cache8(dev, [0], [self.T], Hkv, D, P, seed)
        self.own_slots = torch.cat([self.own[2][0][:n], torch.full((behind,), -1, device=dev)]).int()
        self.tokens = torch.randint(0, V, (self.T,), generator=g, device=dev).int()
        self.probs = torch.softmax(3 * torch.randn(self.T, V, generator=g, device=dev), 1)
        self.au, self.su = torch.rand(self.T, generator=g, device=dev), torch.rand(len(new), generator=g, device=dev)
        self.scratch8 = type(self.c8)(*(x.clone() for x in self.c8))
        self.free = torch.zeros(4096, dtype=torch.int32, device=dev)
        self.count = i32([0], dev)

    def new_inputs(self, seed):
        import torch
        g = gen(self.dev, seed)
        self.rows.copy_(torch.randn(self.rows.shape, generator=g, device=self.dev))
        self.q.copy_(self.rows[:, :self.heads[0]])
        self.au.copy_(torch.rand(self.au.shape, generator=g, device=self.dev))
        self.su.copy_(torch.rand(self.su.shape, generator=g, device=self.dev))

    def calls(self, ws):
        """name: call(stream) that returns its outputs, all of them newly made."""
        import torch
        from inferflux_amd import attention_q8 as q8, drafts
        Hq, Hkv = self.heads
        n = self.T - 3

        def append(s):
            q, k, v = self.rows.split([Hq, Hkv, Hkv], 1)
            o = q8.rope_append(q, k, v, self.pos, self.own_slots, self.own[0], self.freq, stream=s)
            return [o[:n]] + list(q8.read_rows(self.own[0], self.own_slots, stream=s))

        def paged(s, masks=None):
            return [q8.paged_attention(self.q, self.c8, self.table, self.cu, self.kv, self.max_q, self.max_kv,
                                       masks=masks, workspace=ws, stream=s)[:n]]

        def tree(s):
            return [drafts.tree_attention(self.q, *self.c16, self.table16, self.cu, self.kv, self.masks, self.max_q,
                                          self.max_kv, workspace=ws, stream=s)[:n]]

        def verify(s):
            r = drafts.verify(self.tokens, self.cu, self.probs, self.au, self.su, self.max_q, parents=self.parents,
                              workspace=ws, stream=s)
            return [r.accepted, r.path[:n], r.emitted[:n]]

        def keep(s):
            with torch.cuda.stream(s or torch.cuda.current_stream()):
                for x, y in zip(self.scratch8, self.c8):
                    x.copy_(y)
                drafts.keep_path(self.scratch8, self.table, self.cu, self.kv, self.path, self.one, self.max_q, stream=s)
                return [x.clone() for x in self.scratch8]

        def kept(s):
            return list(drafts.plan_kept(self.cu, self.kv, self.zero, self.table, self.free, self.count, self.P, stream=s))

        def plan(s):
            return list(drafts.plan_tree(self.parents, self.cu, self.kv, stream=s))

        return {"plan": plan, "append": append, "paged": paged, "masked": lambda s: paged(s, self.masks), "tree": tree,
                "verify": verify, "keep": keep, "kept": kept}


def same(a, b, what):
    import torch
    for x, y in zip(a, b):
        assert torch.equal(x.nan_to_num(-7) if x.is_floating_point() else x,
                           y.nan_to_num(-7) if y.is_floating_point() else y), what


LENGTHS = ([3000, 0, 40, 700], [20, 1, 0, 61])


def test_outputs_on_a_stream_that_waits_for_nothing(dev):  # noqa: F811
    """Outputs made on stream s while the current stream still writes to blocks
    of their sizes that were freed there."""
    import torch
    from inferflux_amd import attention as at
    note("drafts: outputs on another stream")
    x, ws, s = Step(dev, *LENGTHS, 8, 2, 128, 16), at.workspace(dev), torch.cuda.Stream()
    torch.cuda.synchronize()
    for what, call in x.calls(ws).items():
        want = [y.clone() for y in call(None)]
        torch.cuda.synchronize()
        n = sum(y.numel() * y.element_size() for y in want)
        blocks = [torch.empty(n, dtype=torch.uint8, device=dev) for _ in range(4)]
        torch.cuda.synchronize()
        torch.cuda._sleep(20_000_000)
        for b in blocks:
            b.fill_(77)
        del blocks, b
        got = call(s)
        s.synchronize()
        torch.cuda.synchronize()
        same(got, want, what)
    assert counters_clear(ws)


@pytest.mark.parametrize("shape,lens", [((8, 2, 128, 16), LENGTHS), ((16, 2, 64, 64), ([2500], [60])),
                                        ((5, 1, 256, 32), ([600] * 40, [1, 2] * 20))])
def test_captured_and_replayed(dev, shape, lens):  # noqa: F811
    """All operators in one graph with one workspace, which a second graph and
    eager calls between the replays use too."""
    import torch
    from inferflux_amd import attention as at
    note(f"drafts: graph {shape}")
    x, ws, ws2 = Step(dev, *lens, *shape), at.workspace(dev), at.workspace(dev)
    calls = x.calls(ws)
    for call in calls.values():
        call(None)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=side):
            outs = {what: [y + 0 for y in call(None)] for what, call in calls.items()}
        graphs.append((g, outs))
    eager = x.calls(ws2)
    for i in range(4):
        x.new_inputs(i)
        g, outs = graphs[i % 2]
        g.replay()
        if i == 2:
            graphs[1][0].replay()
        torch.cuda.synchronize()
        got = {what: [y.clone() for y in o] for what, o in outs.items()}
        for what, call in eager.items():
            same(got[what], call(None), (what, i))
        for call in calls.values():  # the graphs' workspace
            call(None)
        torch.cuda.synchronize()
    assert counters_clear(ws) and counters_clear(ws2)


def test_two_calls_at_once(dev):  # noqa: F811
    """Split sums and verifications on two streams, each with its workspace."""
    import torch
    from inferflux_amd import attention as at
    note("drafts: two streams")
    xs = [Step(dev, *LENGTHS, 16, 2, 128, 64, seed=3), Step(dev, [5000, 64], [3, 40], 8, 2, 128, 16, V=40000, seed=4)]
    wss, streams = [at.workspace(dev) for _ in xs], [torch.cuda.Stream() for _ in xs]
    names = "paged", "masked", "tree", "verify"
    sets = [x.calls(w) for x, w in zip(xs, wss)]
    want = [{n: [y.clone() for y in c[n](None)] for n in names} for c in sets]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for c, s in zip(sets, streams):
            with torch.cuda.stream(s):
                got.append({n: c[n](s) for n in names})
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for n in names:
                same(a[n], b[n], n)
    assert all(counters_clear(w) for w in wss)


@pytest.mark.parametrize("T,Hq,Hkv,D,P,rot,inter,src", [
    (2800, 3, 3, 256, 16, 256, True, "bf16"), (150, 48, 16, 128, 64, 128, False, "f32"), (130, 32, 32, 96, 16, 96, False, "f16"),
    (350, 20, 5, 64, 32, 32, True, "f16"), (111, 40, 13, 160, 16, 80, False, "bf16"), (4100, 1, 1, 32, 256, 0, False, "f32"),
    (1031, 17, 17, 224, 128, 64, False, "f16")])
def test_append_heads_shared_out(dev, T, Hq, Hkv, D, P, rot, inter, src):  # noqa: F811
    """Heads over several workgroups, the last with fewer; tokens not by eights."""
    note(f"append q8 heads T={T} {Hq}/{Hkv} D={D}")
    run_append(dev, T, Hq, Hkv, D, P, src, "f16", rot, inter)


def test_refusals_on_device(dev):  # noqa: F811
    """Arguments of another type, shape or device are refused before any launch."""
    import torch
    from inferflux_amd import attention as at, attention_q8 as q8, drafts
    x, ws = Step(dev, [30], [5], 4, 2, 64, 16), at.workspace(dev)
    q = x.q
    k, v = x.rows[:, 4:6], x.rows[:, 6:8]
    c = x.c8

    def paged(**kw):
        a = dict(q=q, cache=c, block_table=x.table, cu_q=x.cu, kv_len=x.kv, max_q=5, max_kv=35, workspace=ws)
        return q8.paged_attention(**{**a, **kw})

    def tree(**kw):
        a = dict(q=q, k_cache=x.c16[0], v_cache=x.c16[1], block_table=x.table16, cu_q=x.cu, kv_len=x.kv, masks=x.masks,
                 max_q=5, max_kv=35, workspace=ws)
        return drafts.tree_attention(**{**a, **kw})

    def append(**kw):
        a = dict(q=x.rows[:, :4], k=k, v=v, positions=x.pos, slots=x.own_slots, cache=x.own[0], inv_freq=x.freq)
        return q8.rope_append(**{**a, **kw})

    def verify(**kw):
        a = dict(tokens=x.tokens, cu_q=x.cu, target_probs=x.probs, accept_u=x.au, sample_u=x.su, max_q=5,
                 parents=x.parents, workspace=ws)
        return drafts.verify(**{**a, **kw})

    def keep(**kw):
        a = dict(cache=c, block_table=x.table, cu_q=x.cu, kv_len=x.kv, path=x.parents, accepted=x.zero, max_q=5)
        return drafts.keep_path(**{**a, **kw})

    for call in (paged, tree, append, verify, keep):
        call()
    torch.cuda.synchronize()
    host = q8.Q8Cache(c.k, c.v.cpu(), c.scales)
    bad = [(paged, dict(q=q.float())), (paged, dict(cache=host)), (paged, dict(cache=q8.Q8Cache(c.k, c.v, c.scales.half()))),
           (paged, dict(cache=q8.Q8Cache(c.k[:, :1], c.v, c.scales))), (paged, dict(window=8, masks=x.masks)),
           (paged, dict(masks=x.masks.int())), (paged, dict(masks=x.masks[:3])), (paged, dict(max_q=65, masks=x.masks)),
           (paged, dict(block_table=x.table.long())), (paged, dict(kv_len=x.kv.cpu())), (paged, dict(scale=0.0)),
           (paged, dict(out=torch.empty(3, 4, 64, device=dev))), (paged, dict(cu_q=x.cu[:1])), (paged, dict(max_kv=0)),
           (tree, dict(max_q=65)), (tree, dict(masks=x.masks.cpu())), (tree, dict(q=q.bfloat16())),
           (tree, dict(v_cache=x.c16[1].cpu())), (tree, dict(masks=x.masks[::2])), (tree, dict(block_table=x.table16[0])),
           (append, dict(k=k.half())), (append, dict(v=v.cpu())), (append, dict(slots=x.own_slots[:4])),
           (append, dict(inv_freq=x.freq.float())), (append, dict(q_dtype=torch.float32)), (append, dict(k=k[:, :1])),
           (append, dict(q_out=torch.empty(x.T, 4, 64, device=dev))), (append, dict(positions=x.pos.long())),
           (verify, dict(workspace=None)), (verify, dict(workspace=ws[:1024])), (verify, dict(max_q=65)),
           (verify, dict(target_probs=x.probs.double())), (verify, dict(target_probs=x.probs[:, ::2])),
           (verify, dict(draft_probs=x.probs)), (verify, dict(parents=None, draft_probs=x.probs.half())),
           (verify, dict(accept_u=x.au.half())), (verify, dict(sample_u=x.su.cpu())), (verify, dict(tokens=x.tokens[:4])),
           (keep, dict(cache=host)), (keep, dict(path=x.parents.long())), (keep, dict(max_q=0)),
           (keep, dict(accepted=x.zero[:0])), (keep, dict(block_table=x.table[0]))]
    for call, change in bad:
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call(**change)
    torch.cuda.synchronize()


@pytest.mark.parametrize("qdt,Hq,Hkv,D,P", [("f16", 16, 2, 128, 64), ("bf16", 40, 8, 128, 16), ("f16", 6, 6, 64, 32),
                                            ("f16", 9, 3, 96, 16), ("bf16", 8, 2, 256, 128)])
@pytest.mark.parametrize("window", [0, 100, 2000])
def test_few_rows_beside_many(dev, qdt, Hq, Hkv, D, P, window):  # noqa: F811
    """Requests of up to 32 rows of a key/value head in a batch with larger ones:
    split and whole, at their bound, in windows; the same bits again."""
    import torch
    from inferflux_amd import attention as at
    note(f"q8 few beside many {Hq}/{Hkv} D={D} window={window}")
    G = Hq // Hkv
    ctx = [9000, 3000, 40, 0, 700, 129, 0, 2500, 5]
    new = [1, 60, 33, 2, 32 // G, 200, 0, 32 // G + 1, 1]
    ws = at.workspace(dev)
    a, b = (run_paged(dev, qdt, ctx, new, Hq, Hkv, D, P, window=window, workspace=ws) for _ in range(2))
    assert torch.equal(a, b)


@pytest.mark.parametrize("B", [3, 70])
def test_few_rows_beside_trees(dev, B):  # noqa: F811
    note(f"q8 trees, few beside many B={B}")
    rng = random.Random(B)
    new = [64] + [rng.choice([0, 1, 1, 2, 6, 7, 40]) for _ in range(B - 1)]
    ctx = [rng.choice([0, 50, rng.randint(0, 700)]) for _ in new]
    ctx[-1], new[-1] = 4000, 1
    run_paged(dev, "f16", ctx, new, 40, 8, 128, 16, masks=tree_masks(rng, new))


def test_few_rows_past_their_bound(dev):  # noqa: F811
    """A request of few rows and more keys than its chunks' weights have room for
    goes the way of the others."""
    import torch
    from inferflux_amd import attention as at, attention_q8 as q8
    note("q8 few rows, many keys")
    D, P, kv = 64, 256, 300000
    c = q8.kv_cache(kv // P + 1, 1, D, P, device=dev)
    g = gen(dev, 1)
    slots = torch.arange(kv, device=dev).int()
    k = torch.randn(kv, 1, D, generator=g, device=dev)
    q8.rope_append(torch.zeros(kv, 1, D, device=dev), k, k, slots, slots, c)
    table = torch.arange(kv // P + 1, device=dev).int().expand(2, -1).contiguous()
    for few in (130000, 150000, 300000):
        q = torch.randn(41, 1, D, generator=g, device=dev).half()
        o = q8.paged_attention(q, c, table, i32([0, 1, 41], dev), i32([few, 300], dev), 40, kv, scale=0.3,
                               workspace=at.workspace(dev))
        kk, vv = q8.read_rows(c, slots[:few], dtype=torch.float32)
        want, bound = ref.attend_seen(q[:1], kk.double(), vv.double(), torch.ones(1, few, dtype=torch.bool), 0.3,
                                      weigh=2.0 ** -11)
        check(o[:1], want, bound + few * 2.0 ** -30 * 127 * 0.05, "few")
