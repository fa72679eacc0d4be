"""Drafted tokens and an 8-bit cache in a serving step, as cases that can be timed.

A serving program that drafts tokens, or keeps its cache in 8 bits, does these
things with this library besides what perf/operators.py holds:

  append  rotates the new tokens' Q and K, writes K and V into the 8-bit cache
          (attention_q8.rope_append), and reads the written rows back as the
          values that the cache then stands for (attention_q8.read_rows)
  paged   attention of the new tokens over the 8-bit cache
          (attention_q8.paged_attention)
  tree    positions and masks of drafted trees (drafts.plan_tree) and the
          attention of their nodes over the cache (drafts.tree_attention, or
          attention_q8.paged_attention with the masks)
  verify  which drafts the target's probabilities accept, and the next token
          (drafts.verify)
  keep    moves the accepted drafts' K and V behind the tokens that were there
          (drafts.keep_path)

Case values:
  op               one of the five
  B                requests
  lo, hi, lens     the requests' cached tokens: spread between lo and hi evenly
                   over their logarithm, in an order that `lens` gives
  qlo, qhi, ones   new tokens a request (nodes of its tree, the last accepted
                   token its root), likewise; the first `ones` requests have one
  page             tokens in a page
  hq, hkv, d       query heads, key/value heads, head size
  dtype            "f16" or "bf16": the rows of Q, and a 16-bit cache
  src              append: what the projections wrote, "f32", "f16" or "bf16"
  inter            append: rotated pairs are (2i, 2i + 1), else (i, i + r/2)
  rot              append: rotated values of a head (r)
  window           paged: keys a query sees, its own among them; 0: all before it
  q8               tree: whether the cache has 8 bits
  vocab            verify: tokens a row of probabilities holds
  chain            verify: drafts one behind the other, drawn from probabilities
                   that are given; else trees without
  prob             verify: type of the probabilities

Heads and vocabulary are the configurations of inferflux_amd/workloads.py (3B:
16 / 2 heads of 128, 14B: 40 / 8), and others of the same kind.  The 8-bit cache
holds K as [page][kv head][d / 16][token][16] and V as
[page][kv head][token / 16][d][16], and for each token and head the scales of
its K and V side by side; the 16-bit one K as [page][kv head][d / 8][token][8]
and V as [page][kv head][token / 8][d][8].
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
B3 = dict(hq=16, hkv=2, d=128)
B14 = dict(hq=40, hkv=8, d=128)
VOCAB = 151936
THETA = 1e6
OPS = ("append", "paged", "tree", "verify", "keep")


def listed():
    return [
        # the decode step of a small batch in the 3B model, fp32 projections
        dict(name="append q8 3B B=8", op="append", B=8, lo=50, hi=4000, lens=3, qlo=1, qhi=1, ones=0,
             page=64, dtype="f16", src="f32", rot=128, inter=False, **B3),
        # prompts of a 14B model packed into one step, fp16 projections
        dict(name="append q8 14B prompts", op="append", B=21, lo=1, hi=1000, lens=4, qlo=20, qhi=1500,
             ones=3, page=16, dtype="f16", src="f16", rot=128, inter=False, **B14),
        # one chat: the latency of a single token in the 3B model
        dict(name="paged q8 3B B=1 kv 3000", op="paged", B=1, lo=2999, hi=2999, lens=5, qlo=1, qhi=1,
             ones=0, page=64, dtype="f16", window=0, **B3),
        # a full decode batch of the 14B model, lengths far apart
        dict(name="paged q8 14B B=32", op="paged", B=32, lo=500, hi=24000, lens=6, qlo=1, qhi=1, ones=0,
             page=16, dtype="f16", window=0, **B14),
        # a prefill chunk behind a long context
        dict(name="paged q8 14B chunk 512", op="paged", B=1, lo=7430, hi=7430, lens=7, qlo=512, qhi=512,
             ones=0, page=64, dtype="bf16", window=0, **B14),
        # one chat with a wide tree of drafts
        dict(name="tree 3B B=1 61 nodes", op="tree", B=1, lo=2950, hi=2950, lens=8, qlo=61, qhi=61, ones=0,
             page=64, dtype="f16", q8=False, **B3),
        # a batch of small trees in the 14B model
        dict(name="tree 14B B=16 6 nodes", op="tree", B=16, lo=200, hi=9000, lens=9, qlo=6, qhi=6, ones=0,
             page=16, dtype="bf16", q8=False, **B14),
        # trees of different sizes next to requests without drafts, 8-bit cache
        dict(name="tree q8 14B B=24", op="tree", B=24, lo=100, hi=8000, lens=10, qlo=5, qhi=40, ones=6,
             page=32, dtype="f16", q8=True, **B14),
        # a small model's chain of seven drafts for one chat
        dict(name="verify chain B=1", op="verify", B=1, lens=11, qlo=8, qhi=8, ones=0, vocab=VOCAB,
             chain=True, prob="f32"),
        # trees of a whole batch
        dict(name="verify trees B=48", op="verify", B=48, lens=12, qlo=9, qhi=33, ones=5, vocab=VOCAB,
             chain=False, prob="f32"),
        # what the chat's tree leaves behind, one layer
        dict(name="keep 3B B=1", op="keep", B=1, lo=2950, hi=2950, lens=13, qlo=61, qhi=61, ones=0, page=64,
             dtype="f16", **B3),
        # the same for a full batch of the 14B model
        dict(name="keep 14B B=32", op="keep", B=32, lo=100, hi=3000, lens=14, qlo=9, qhi=33, ones=0, page=16,
             dtype="f16", **B14),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    if rng.random() < 0.4:
        return dict(rng.choice([B3, B14]))
    hkv = rng.choice([1, 2, 3, 4, 8, 12, 16])
    return dict(hkv=hkv, hq=hkv * rng.choice([1, 1, 2, 3, 4, 5, 7, 8]), d=rng.choice([64, 96, 128, 256]))


def draw(rng):
    """One more case: any operator, sizes over the listed ones' range."""
    top = {op: max(work(c)["flops"] + work(c)["bytes"] for c in listed() if c["op"] == op) for op in OPS}
    while True:
        op = rng.choice(OPS)
        c = dict(op=op, B=_log(rng, 1, 64), lens=rng.randrange(1 << 20))
        c["ones"] = rng.randint(0, c["B"] // 2)
        if op in ("append", "paged"):
            qhi = 1 if rng.random() < 0.4 else _log(rng, 2, 1500)
        else:
            qhi = _log(rng, 2, 64)
        c.update(qlo=max(1, int(qhi * rng.uniform(0.02, 1.0))), qhi=qhi)
        if op == "verify":
            c.update(vocab=_log(rng, 1000, VOCAB), chain=rng.random() < 0.5,
                     prob=rng.choice(["f32", "f32", "f16", "bf16"]))
        else:
            hi = _log(rng, 2, 20000 if op == "paged" else 8000 if op != "keep" else 3000)
            c.update(lo=max(1, int(hi * rng.uniform(0.02, 1.0))), hi=hi, page=rng.choice([16, 32, 64, 128]),
                     dtype=rng.choice(["f16", "bf16"]), **_heads(rng))
        if op == "append":
            c.update(src=rng.choice(["f32", "f16", "bf16"]), inter=rng.random() < 0.3,
                     rot=c["d"] if rng.random() < 0.7 else c["d"] // 2)
        if op == "paged":
            c["window"] = 0 if rng.random() < 0.8 else _log(rng, 2, 4096)
        if op == "tree":
            c["q8"] = rng.random() < 0.5
        w = work(c)
        if w["flops"] + w["bytes"] <= top[op] and _held(c) <= 2.0e9:
            return c


# ------------------------------------------------------------------- lengths
def _spread(n, lo, hi, order):
    """n lengths between lo and hi, evenly over their logarithm."""
    v = [int(round(lo * (hi / lo) ** ((i + 0.5) / n))) for i in range(n)]
    random.Random(order).shuffle(v)
    return v


def _lengths(c):
    """(cached tokens, new tokens) of every request."""
    n = _spread(c["B"], c["lo"], c["hi"], c["lens"]) if "lo" in c else [0] * c["B"]
    q = _spread(c["B"], c["qlo"], c["qhi"], c["lens"] + 1)
    return n, [1 if i < c["ones"] else x for i, x in enumerate(q)]


def _held(c):
    """Values that the plain form or the inputs hold at once."""
    ctx, new = _lengths(c)
    if c["op"] == "verify":
        return sum(new) * c["vocab"] * 2
    cache = sum(a + b + c["page"] for a, b in zip(ctx, new)) * c["hkv"] * c["d"] * 2
    if c["op"] in ("append", "keep"):
        return cache
    return max(cache, c["B"] * c["hq"] * max(new) * max(a + b for a, b in zip(ctx, new)))


def _parents(c):
    """Every request's tree, drawn from the case alone: its nodes' parents, the
    root first.  Most nodes hang on one of the last few."""
    r = random.Random(c["lens"] + 2)
    return [[-1] + [r.randint(max(0, j - 4), j - 1) for j in range(1, n)] for n in _lengths(c)[1]]


def _depth(parents):
    depth = []
    for p in parents:
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return depth


def _paths(c):
    """The nodes that each request keeps, the root first: some of those behind
    the places that they move to."""
    r = random.Random(c["lens"] + 3)
    got = []
    for n in _lengths(c)[1]:
        a = min((n - 1) // 2, r.randint(0, 6))
        got.append([0] + sorted(r.sample(range(a + 1, n), a)))
    return got


def _pairs(c):
    """Query-key pairs that the masks leave."""
    ctx, new = _lengths(c)
    if c["op"] == "tree":
        return sum(n * a + sum(_depth(p)) + n for a, n, p in zip(ctx, new, _parents(c)))
    if not c["window"]:
        return sum(n * a + n * (n + 1) // 2 for a, n in zip(ctx, new))
    return sum(sum(min(a + i + 1, c["window"]) for i in range(n)) for a, n in zip(ctx, new))


def work(c):
    ctx, new = _lengths(c)
    T = sum(new)
    if c["op"] == "verify":  # the row that the next token is drawn from, and the drafter's
        size = 4 if c["prob"] == "f32" else 2
        return {"bytes": c["B"] * c["vocab"] * size * (2 if c["chain"] else 1) + 20 * T, "flops": 0}
    row = c["hkv"] * c["d"]
    if c["op"] == "append":  # rows in; Q, codes and scales out; the rows read back
        size = 4 if c["src"] == "f32" else 2
        return {"bytes": T * ((c["hq"] * c["d"] + 2 * row) * size + c["hq"] * c["d"] * 2
                              + 2 * (2 * row + 4 * c["hkv"]) + 4 * row) + 8 * T, "flops": 0}
    if c["op"] == "keep":
        moved = sum(len(p) - 1 for p in _paths(c))
        return {"bytes": 2 * moved * row * 4 + 4 * T, "flops": 0}
    kv = sum(a + b for a, b in zip(ctx, new))
    if c.get("window"):  # keys behind every new token's window are not read
        kv = sum(min(a + b, b + c["window"] - 1) for a, b in zip(ctx, new))
    q8 = c.get("q8", True)
    return {"bytes": kv * (2 * row + 4 * c["hkv"] if q8 else 4 * row) + 4 * T * c["hq"] * c["d"],
            "flops": 4 * c["d"] * c["hq"] * _pairs(c)}


# -------------------------------------------------------------------- inputs
class _State:
    """What the program keeps from step to step, and this step's inputs."""


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _normal(shape, dtype, g):
    return torch.randn(shape, dtype=TYPES[dtype], device="cuda", generator=g)


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 2654435761 + 97) % (1 << 31))
    s = _State()
    s.c = c
    ctx, new = _lengths(c)
    B, T = c["B"], sum(new)
    s.T, s.max_q, s.max_kv = T, max(new), max(a + b for a, b in zip(ctx, new))
    s.cu = _i32([sum(new[:i]) for i in range(B + 1)])
    s.kv = _i32([a + b for a, b in zip(ctx, new)])
    if c["op"] in ("tree", "verify"):
        s.parents = _i32(sum(_parents(c), []))
    # the buffer that the program keeps for split sums, zeroed once
    s.ws = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    if c["op"] == "verify":
        return _drafts(s, g)

    P = c["page"]
    s.W = -(-s.max_kv // P) + 2  # the table has room for more
    total = [-(-(a + b) // P) for a, b in zip(ctx, new)]
    s.pages = sum(total) + 7
    order = torch.randperm(s.pages, device="cuda", generator=g).int()
    start = _i32([sum(total[:i]) for i in range(B)])[:, None]
    w = torch.arange(s.W, device="cuda")[None]
    s.table = torch.where(w < _i32(total)[:, None], order[(start + w).clamp(max=s.pages - 1)], 0).int()
    shape = (s.pages, c["hkv"])
    if c.get("q8", c["op"] != "keep"):
        k = _normal(shape + (c["d"] // 16, P, 16), "f16", g)
        s.k_cache = (k * 40).round().clamp(-127, 127).to(torch.int8)
        v = _normal(shape + (P // 16, c["d"], 16), "f16", g)
        s.v_cache = (v * 40).round().clamp(-127, 127).to(torch.int8)
        # tokens' keys and values differ in size
        spread = _normal(shape + (P, 2), "f32", g) * torch.tensor([0.2, 0.5], device="cuda")
        s.scales = (spread.exp() * 0.025).bfloat16()
    else:
        s.k_cache = _normal(shape + (c["d"] // 8, P, 8), c["dtype"], g)
        s.v_cache = _normal(shape + (P // 8, c["d"], 8), c["dtype"], g)
    if c["op"] == "keep":
        paths = _paths(c)
        s.accepted = _i32([len(p) - 1 for p in paths])
        s.path = _i32(sum((p + [-1] * (n - len(p)) for p, n in zip(paths, new)), []))
        return s
    if c["op"] == "append":
        pos = torch.cat([torch.arange(a, a + b, device="cuda") for a, b in zip(ctx, new)])
        req = torch.repeat_interleave(torch.arange(B, device="cuda"), _i32(new))
        s.pos = pos.int()
        s.slots = (s.table[req, pos // P] * P + pos % P).int()
        i = torch.arange(c["rot"] // 2, dtype=torch.float64, device="cuda")
        s.freq = THETA ** (-2.0 * i / c["rot"])
        # Q, K and V as one projection launch writes them, side by side
        n = (c["hq"], c["hkv"], c["hkv"])
        rows = _normal((T, sum(n) * c["d"]), c["src"], g)
        s.q, s.k, s.v = (x.view(T, -1, c["d"]) for x in rows.split([x * c["d"] for x in n], dim=1))
        s.q_out = torch.empty(T, c["hq"], c["d"], dtype=TYPES[c["dtype"]], device="cuda")
        return s
    # queries that single some keys out: scores spread over several units
    s.q = _normal((T, c["hq"], c["d"]), c["dtype"], g) * 1.5
    s.out = torch.empty_like(s.q)
    s.scale = c["d"] ** -0.5
    return s


def _drafts(s, g):
    """Probabilities of a target that prefers few tokens, and drafts that are
    often among them."""
    c, T, V = s.c, s.T, s.c["vocab"]
    s.p = torch.softmax(_normal((T, V), "f32", g) * 5.0, 1).to(TYPES[c["prob"]])
    s.accept_u = torch.rand(T, device="cuda", generator=g)
    s.sample_u = torch.rand(c["B"], device="cuda", generator=g)
    t = torch.arange(T, device="cuda")
    req = torch.searchsorted(s.cu[1:].long(), t, right=True)
    if c["chain"]:
        # the drafter's probabilities are the target's, disturbed
        s.q = torch.softmax(s.p.float().log().clamp(min=-40.0) + _normal((T, V), "f32", g), 1).to(TYPES[c["prob"]])
        drawn = torch.multinomial(s.q.float(), 1, generator=g)[:, 0]
        s.tokens = torch.where(t == s.cu[req], t * 7 % V, drawn.roll(1)).int()
    else:
        # the parent's most likely tokens, a child each
        s.q = None
        parent = torch.where(s.parents >= 0, s.cu[req] + s.parents, t).long()
        same = (parent[:, None] == parent[None]) & (t[None] < t[:, None]) & (s.parents >= 0)[None]
        rank = same.sum(1)
        s.tokens = s.p.float().topk(8, 1).indices[parent, rank.clamp(max=7)].int()
    return s


# ----------------------------------------------------------------------- run
def run(s):
    if own:
        return _own(s)
    return {"append": _append, "paged": _paged, "tree": _tree, "verify": _verify, "keep": _keep}[s.c["op"]](s)


def _own(s):
    from inferflux_amd import attention_q8, drafts
    c = s.c
    if c["op"] == "verify":
        r = drafts.verify(s.tokens, s.cu, s.p, s.accept_u, s.sample_u, s.max_q,
                          parents=None if c["chain"] else s.parents, draft_probs=s.q, workspace=s.ws)
        return [r.accepted, r.path, r.emitted]
    if c["op"] == "keep":
        drafts.keep_path((s.k_cache, s.v_cache), s.table, s.cu, s.kv, s.path, s.accepted, s.max_q)
        return [s.k_cache, s.v_cache]
    q8 = c.get("q8", True)
    cache = attention_q8.Q8Cache(s.k_cache, s.v_cache, s.scales) if q8 else (s.k_cache, s.v_cache)
    if c["op"] == "append":
        attention_q8.rope_append(s.q, s.k, s.v, s.pos, s.slots, cache, s.freq, interleaved=c["inter"],
                                 q_out=s.q_out)
        k, v = attention_q8.read_rows(cache, s.slots, dtype=TYPES[c["dtype"]])
        return [s.q_out, k, v]
    if c["op"] == "paged":
        return attention_q8.paged_attention(s.q, cache, s.table, s.cu, s.kv, s.max_q, s.max_kv, scale=s.scale,
                                            window=c["window"], out=s.out, workspace=s.ws)
    t = drafts.plan_tree(s.parents, s.cu, s.kv)
    if q8:
        attention_q8.paged_attention(s.q, cache, s.table, s.cu, s.kv, s.max_q, s.max_kv, scale=s.scale,
                                     masks=t.masks, out=s.out, workspace=s.ws)
    else:
        drafts.tree_attention(s.q, *cache, s.table, s.cu, s.kv, t.masks, s.max_q, s.max_kv, scale=s.scale,
                              out=s.out, workspace=s.ws)
    return [t.positions, t.masks, s.out]


def _codes(x):
    """Codes and scales of rows of float64: the scale is the smallest bfloat16
    that is no less than the largest value / 127."""
    want = x.abs().amax(-1, keepdim=True) / 127
    f = want.float()
    f = torch.where(f.double() < want, torch.nextafter(f, torch.full_like(f, math.inf)), f)
    scale = ((f.view(torch.int32) + 0xFFFF) & ~0xFFFF).view(torch.float32)
    return torch.where(scale > 0, x / scale.double(), 0.0).round(), scale


def _append(s):
    c, dt = s.c, TYPES[s.c["dtype"]]
    h, d, P = c["rot"] // 2, c["d"], c["page"]
    # 64 bits: positions times frequencies reach far, and codes change at borders
    angle = s.pos.double()[:, None, None] * s.freq
    cos, sin = angle.cos(), angle.sin()

    def rotate(x):
        x = x.double()
        if c["inter"]:
            a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
        else:
            a, b = x[..., :h], x[..., h:2 * h]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
        return torch.cat([y, x[..., 2 * h:]], dim=-1)

    s.q_out.copy_(rotate(s.q))
    page, at = s.slots.long() // P, s.slots.long() % P
    (k, ks), (v, vs) = _codes(rotate(s.k)), _codes(s.v.double())
    s.k_cache[page, :, :, at] = k.to(torch.int8).view(s.T, c["hkv"], d // 16, 16)
    s.v_cache[page, :, at // 16, :, at % 16] = v.to(torch.int8)
    s.scales[page, :, at] = torch.cat([ks, vs], -1).bfloat16()
    scale = s.scales[page, :, at].float()
    k = s.k_cache[page, :, :, at].view(s.T, c["hkv"], d).float() * scale[..., :1]
    v = s.v_cache[page, :, at // 16, :, at % 16].float() * scale[..., 1:]
    return [s.q_out, k.to(dt), v.to(dt)]


def _rows(s):
    """Row numbers of the padded form [B, max_q], and (request, row) of every
    token."""
    i = torch.arange(s.max_q, device="cuda")
    at = (s.cu[:-1, None] + i).clamp(max=s.T - 1).long()
    t = torch.arange(s.T, device="cuda")
    r = torch.searchsorted(s.cu[1:].long(), t, right=True)
    return at, r, t - s.cu[r]


def _ancestors(s, at):
    """[B, n, n]: whether node j is on the way from the root to node i."""
    n = s.max_q
    i = torch.arange(n, device="cuda")
    up = (s.parents[at][:, :, None] == i) & (i < (s.cu[1:] - s.cu[:-1])[:, None])[:, :, None]
    seen = (up | torch.eye(n, dtype=torch.bool, device="cuda")).float()
    for _ in range(max(1, (n - 1).bit_length())):  # twice as far each time
        seen = (torch.bmm(seen, seen) > 0).float()
    return seen > 0


def _cache_rows(s):
    """K and V [B, hkv, L, d] in 32 bits of the padded requests."""
    c, P = s.c, s.c["page"]
    W = -(-s.max_kv // P)
    page = s.table[:, :W].long()
    shape = (c["B"], c["hkv"], W * P, c["d"])
    k = s.k_cache[page].float().permute(0, 2, 1, 4, 3, 5).reshape(shape)
    v = s.v_cache[page].float().permute(0, 2, 1, 3, 5, 4).reshape(shape)
    if c.get("q8", True):
        scale = s.scales[page].float().permute(0, 2, 1, 3, 4).reshape(shape[:3] + (2,))
        k, v = k * scale[..., :1], v * scale[..., 1:]
    return k, v


def _softmax_v(s, seen):
    """Attention of the padded queries in 32 bits; seen [B, max_q, L]."""
    c = s.c
    k, v = _cache_rows(s)
    B, L, G = c["B"], k.shape[2], c["hq"] // c["hkv"]
    at, r, row = _rows(s)
    q = s.q[at].float().view(B, s.max_q, c["hkv"], G, c["d"]).permute(0, 2, 3, 1, 4)
    q = q.reshape(B * c["hkv"], G * s.max_q, c["d"])
    x = torch.bmm(q, k.reshape(B * c["hkv"], L, c["d"]).transpose(1, 2).contiguous()) * s.scale
    x = x.view(B, c["hkv"], G, s.max_q, L)
    x.masked_fill_(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    x.sub_(top).exp_()
    o = torch.bmm(x.view(B * c["hkv"], G * s.max_q, L), v.reshape(B * c["hkv"], L, c["d"]))
    total = x.sum(-1).view(B * c["hkv"], G * s.max_q, 1)
    o = torch.where(total > 0, o / total, 0.0).view(B, c["hq"], s.max_q, c["d"])
    s.out.copy_(o[r, :, row])
    return s.out


def _keys(s):
    """Key numbers of the padded requests and the position of their first row."""
    L = -(-s.max_kv // s.c["page"]) * s.c["page"]
    return torch.arange(L, device="cuda"), s.kv - (s.cu[1:] - s.cu[:-1])


def _paged(s):
    j, first = _keys(s)
    p = (first[:, None] + torch.arange(s.max_q, device="cuda"))[:, :, None]
    seen = (j < s.kv[:, None, None]) & (j <= p)
    if s.c["window"]:
        seen = seen & (j > p - s.c["window"])
    return _softmax_v(s, seen)


def _tree(s):
    at, r, row = _rows(s)
    up = _ancestors(s, at)
    j, first = _keys(s)
    node = (j - first[:, None])[:, None]  # of the request's tree; below 0: a cached token
    inside = torch.gather(up, 2, node.clamp(0, s.max_q - 1).expand(-1, s.max_q, -1))
    out = _softmax_v(s, (node < 0) | inside & (j < s.kv[:, None, None]))
    positions = (first[:, None] + up.sum(2) - 1)[r, row].int()
    masks = (up.long() << torch.arange(s.max_q, device="cuda")).sum(2)[r, row]
    return [positions, masks, out]


def _verify(s):
    c, V, B, n = s.c, s.c["vocab"], s.c["B"], s.max_q
    at, r, row = _rows(s)
    i = torch.arange(n, device="cuda")
    live = i < (s.cu[1:] - s.cu[:-1])[:, None]
    parent = (i - 1).expand(B, n) if c["chain"] else s.parents[at].long()
    above = at.gather(1, parent.clamp(min=0))  # the parent's row
    tokens = s.tokens[at].long()
    drafted = live & (parent >= 0)
    child = drafted[:, None] & (parent[:, None] == i[:, None])  # [B, node, its children]
    u = s.accept_u[above].double()
    p = s.p[above, tokens].double()  # 64 bits: sums next to a border
    if c["chain"]:
        taken = drafted & (u * s.q[above, tokens].double() < p)
    else:
        before = (parent[:, None] == parent[:, :, None]) & (i < i[:, None]) & drafted[:, None]
        new = drafted & ~(before & (tokens[:, None] == tokens[:, :, None])).any(2)
        p = torch.where(new, p, 0.0)
        less = (before * p[:, None]).sum(2)
        taken = new & (u < less + p) & ~(u < less)
    # a node is reached where all on its way but the root are taken
    step = torch.where(child.transpose(1, 2), 1.0, 0.0) + torch.eye(n, device="cuda")
    way = step
    for _ in range(max(1, (n - 1).bit_length())):
        way = (torch.bmm(way, way) > 0).float()
    reached = live & ((way > 0) & ~(taken | (i == 0))[:, None]).logical_not().all(2)
    accepted = reached.sum(1).int() - 1
    last = torch.where(reached, i, 0).amax(1)
    # what the next token is drawn from
    at_last = at.gather(1, last[:, None])[:, 0]
    w = s.p[at_last].double()
    if c["chain"]:
        w = torch.where((last + 1 == live.sum(1))[:, None], w, (w - s.q[at_last].double()).clamp(min=0))
    else:
        mine = child.gather(1, last[:, None, None].expand(B, 1, n))[:, 0]
        gone = torch.zeros(B, V + 1, dtype=torch.bool, device="cuda")
        gone.scatter_(1, torch.where(mine, tokens, V), True)
        w = w.masked_fill(gone[:, :V], 0.0)
    w = torch.where((w.sum(1) > 0)[:, None], w, s.p[at_last].double())
    total = w.cumsum(1)
    drawn = (total <= (s.sample_u.double() * total[:, -1])[:, None]).sum(1)
    # the nodes and tokens in their order
    rank = torch.where(reached, reached.cumsum(1) - 1, n)
    path = torch.full((B, n + 1), -1, device="cuda").scatter_(1, rank, i.expand(B, n))[:, :n]
    after = torch.cat([path[:, 1:], torch.full((B, 1), -1, device="cuda")], 1)
    emitted = torch.where(after >= 0, tokens.gather(1, after.clamp(min=0)), -1)
    emitted = torch.where(i == accepted[:, None], drawn[:, None], emitted)
    return [accepted, path[r, row].int(), emitted[r, row].int()]


def _keep(s):
    P = s.c["page"]
    _, r, row = _rows(s)
    first = (s.kv - (s.cu[1:] - s.cu[:-1]))[r]
    moves = (row <= s.accepted[r]) & (s.path >= 0)
    a, b = (first + torch.where(moves, s.path, row)).long(), (first + row).long()
    a, b = s.table[r, a // P].long() * P + a % P, s.table[r, b // P].long() * P + b % P
    s.k_cache[b // P, :, :, b % P] = s.k_cache[a // P, :, :, a % P]
    s.v_cache[b // P, :, b % P // 8, :, b % P % 8] = s.v_cache[a // P, :, a % P // 8, :, a % P % 8]
    return [s.k_cache, s.v_cache]


# ------------------------------------------------------------ the definition
def exact(c, seed):
    """The outputs in 64 bits, request by request."""
    s = prepare(c, seed)
    if c["op"] in ("paged", "tree"):
        return _exact_attention(s)
    return _exact_append(s) if c["op"] == "append" else _exact_verify(s) if c["op"] == "verify" else None


def _exact_append(s):
    c = s.c
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"),
                       s.pos.double()[:, None] * s.freq)[:, None]
    got = []
    for x in (s.q, s.k):
        x = x.double().clone()
        if c["inter"]:
            z = torch.view_as_complex(x[..., :c["rot"]].unflatten(-1, (-1, 2)).contiguous()) * turn
            x[..., :c["rot"]] = torch.view_as_real(z).flatten(-2)
        else:
            half = c["rot"] // 2
            z = torch.complex(x[..., :half], x[..., half:c["rot"]]) * turn
            x[..., :c["rot"]] = torch.cat([z.real, z.imag], dim=-1)
        got.append(x)
    for x in (got.pop(), s.v.double()):
        need = x.abs().amax(-1, keepdim=True) / 127
        # eight significant bits, away from zero
        unit = torch.exp2(torch.floor(torch.log2(need)) - 7)
        scale = torch.ceil(need / unit) * unit
        got.append(torch.round(x / scale) * scale)
    return got


def _exact_attention(s):
    c, P = s.c, s.c["page"]
    ctx, new = _lengths(c)
    q8, trees = c.get("q8", True), _parents(c) if c["op"] == "tree" else None
    out = torch.zeros(s.T, c["hq"], c["d"], dtype=torch.float64, device="cuda")
    G, t0 = c["hq"] // c["hkv"], 0
    positions, masks = [], []
    for b in range(c["B"]):
        L, n = ctx[b] + new[b], new[b]
        where = torch.arange(L, device="cuda")
        page, at = s.table[b].long()[where // P], where % P
        hide = None
        if trees:
            hide = torch.ones(n, n, dtype=torch.bool)
            for i, up in enumerate(trees[b]):
                if up >= 0:
                    hide[i] = hide[up]
                hide[i, i] = False
            positions += [ctx[b] + x for x in _depth(trees[b])]
            for row in hide.tolist():
                m = sum(1 << j for j, x in enumerate(row) if not x)
                masks.append(m - (1 << 64) if m >> 63 else m)
        for h in range(c["hkv"]):
            e = 16 if q8 else 8
            k = s.k_cache[page, h, :, at].double().reshape(L, c["d"])
            v = s.v_cache[page, h, at // e, :, at % e].double()
            if q8:
                k = k * s.scales[page, h, at, 0].double()[:, None]
                v = v * s.scales[page, h, at, 1].double()[:, None]
            gone = torch.zeros(n, L, dtype=torch.bool, device="cuda")
            if trees:
                gone[:, ctx[b]:] = hide.cuda()
            else:
                mine = torch.arange(ctx[b], L, device="cuda")[:, None]
                gone |= where > mine
                if c["window"]:
                    gone |= where <= mine - c["window"]
            for j in range(h * G, (h + 1) * G):
                x = s.q[t0:t0 + n, j].double() @ k.T * s.scale
                x[gone] = -math.inf
                x = (x - x.max(1, keepdim=True).values).exp()
                out[t0:t0 + n, j] = (x @ v) / x.sum(1, keepdim=True)
        t0 += n
    return [None, None, out] if trees else out


def _exact_verify(s):
    c, V = s.c, s.c["vocab"]
    new, trees = _lengths(c)[1], _parents(c)
    tokens, accept = s.tokens.tolist(), s.accept_u.tolist()
    accepted, paths, emitted, t0 = [], [], [], 0
    for b, n in enumerate(new):
        path = [0]
        while True:
            i = path[-1]
            p = s.p[t0 + i].double()
            w, after = p, None
            if c["chain"]:
                if i + 1 < n:
                    x, q = tokens[t0 + i + 1], s.q[t0 + i].double()
                    after = i + 1 if accept[t0 + i] * float(q[x]) < float(p[x]) else None
                    w = torch.relu(p - q)
            else:
                children = [j for j in range(n) if trees[b][j] == i]
                part, met = 0.0, set()
                for j in children:
                    x = tokens[t0 + j]
                    part += 0.0 if x in met else float(p[x])
                    if after is None and x not in met and accept[t0 + i] < part:
                        after = j
                    met.add(x)
                w = p.clone()
                w[list(met)] = 0.0
            if after is None:
                break
            path.append(after)
        if not float(w.sum()) > 0:
            w = p
        below = torch.cumsum(w, 0)
        x = int(torch.searchsorted(below, below[-1:] * float(s.sample_u[b]), right=True))
        accepted.append(len(path) - 1)
        emitted += [tokens[t0 + j] for j in path[1:]] + [x] + [-1] * (n - len(path))
        paths += path + [-1] * (n - len(path))
        t0 += n
    return [_i32(accepted), _i32(paths), _i32(emitted)]
