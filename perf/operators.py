"""The attention of a serving step, as cases that can be timed.

Between the Q/K/V projections of a decoder layer and its O projection a
serving program does four things with this library:

  plan    from the requests' lengths: pages for the new tokens, the block
          table, slots, positions and row offsets (attention.plan_batch)
  append  rotates the new tokens' Q and K and writes K and V into the paged
          cache (attention.rope_append)
  paged   attention of the new tokens (one a request, or a chunk) over the
          paged cache (attention.paged_attention)
  prompt  attention over whole prompts packed one after the other, without a
          cache: scoring and embedding requests (attention.prompt_attention)

Case values:
  op               one of the four
  B                requests
  lo, hi, lens     the requests' lengths: spread between lo and hi evenly over
                   their logarithm, in an order that `lens` gives (cached
                   tokens for plan, append and paged; prompt lengths)
  qlo, qhi, ones   new tokens a request, likewise; the first `ones` requests
                   have a single one (requests that decode)
  page             tokens in a page
  hq, hkv, d       query heads, key/value heads, head size
  dtype            "f16" or "bf16": the cache and the rows of Q
  src              append: what the projections wrote, "f32", "f16" or "bf16"
  inter            append: rotated pairs are (2i, 2i + 1), else (i, i + r/2)
  rot              append: rotated values of a head (r)
  window           keys a query sees, its own among them; 0: all before it
  causal           prompt: whether a query sees only what is before it

Heads are the configurations of inferflux_amd/workloads.py (3B: 16 / 2 heads
of 128, 14B and 32B: 40 / 8), and others of the same kind.  The cache holds K
as [page][kv head][d / 8][token][8] and V as [page][kv head][token / 8][d][8].
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
B3 = dict(hq=16, hkv=2, d=128)
B14 = dict(hq=40, hkv=8, d=128)
THETA = 1e6


def listed():
    return [
        # every step of a decode batch begins with this: 32 requests, a token each
        dict(name="plan decode B=32", op="plan", B=32, lo=100, hi=6000, lens=1, qlo=1, qhi=1,
             ones=0, page=64),
        # a scheduler that packs many prompts' chunks into one step, small pages
        dict(name="plan chunks B=300", op="plan", B=300, lo=1, hi=3000, lens=2, qlo=1, qhi=1500,
             ones=100, page=16),
        # the decode step of a small batch in the 3B model, fp32 projections
        dict(name="append 3B B=8", op="append", B=8, lo=50, hi=4000, lens=3, qlo=1, qhi=1, ones=0,
             page=64, dtype="f16", src="f32", rot=128, inter=False, **B3),
        # prompts of a 14B model packed into one step, fp16 projections
        dict(name="append 14B prompts", op="append", B=21, lo=1, hi=1000, lens=4, qlo=20, qhi=1500,
             ones=3, page=16, dtype="f16", src="f16", rot=128, inter=False, **B14),
        # one chat: the latency of a single token in the 3B model
        dict(name="paged 3B B=1 kv 3000", op="paged", B=1, lo=2999, hi=2999, lens=5, qlo=1, qhi=1,
             ones=0, page=64, dtype="f16", window=0, **B3),
        # a full decode batch of the 14B model, lengths far apart
        dict(name="paged 14B B=32", op="paged", B=32, lo=500, hi=24000, lens=6, qlo=1, qhi=1, ones=0,
             page=16, dtype="f16", window=0, **B14),
        # a prefill chunk behind a long context
        dict(name="paged 14B chunk 512", op="paged", B=1, lo=7430, hi=7430, lens=7, qlo=512, qhi=512,
             ones=0, page=64, dtype="bf16", window=0, **B14),
        # a mixed step: requests that decode next to prompts' chunks
        dict(name="paged 3B mixed B=24", op="paged", B=24, lo=30, hi=9000, lens=8, qlo=16, qhi=600,
             ones=16, page=32, dtype="f16", window=0, **B3),
        # one short prompt
        dict(name="prompt 3B 500", op="prompt", B=1, lo=500, hi=500, lens=9, dtype="f16", causal=True,
             window=0, **B3),
        # embedding requests: short texts, both directions, small heads
        dict(name="prompt embed B=64", op="prompt", B=64, lo=3, hi=500, lens=10, dtype="f16",
             causal=False, window=0, hq=12, hkv=12, d=64),
        # prompts of very different lengths packed together
        dict(name="prompt 14B packed", op="prompt", B=9, lo=70, hi=4100, lens=11, dtype="bf16",
             causal=True, window=0, **B14),
        # one long prompt
        dict(name="prompt 14B 8111", op="prompt", B=1, lo=8111, hi=8111, lens=12, dtype="bf16",
             causal=True, window=0, **B14),
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
    top = {op: max(work(c)["flops"] + work(c)["bytes"] for c in listed() if c["op"] == op)
           for op in ("plan", "append", "paged", "prompt")}
    while True:
        op = rng.choice(["plan", "append", "paged", "paged", "prompt"])
        B = _log(rng, 1, {"plan": 400, "append": 64, "paged": 48, "prompt": 80}[op])
        hi = _log(rng, 2, 20000 if op == "paged" else 8000)
        lo = max(1, int(hi * rng.uniform(0.02, 1.0)))
        c = dict(op=op, B=B, lo=lo, hi=hi, lens=rng.randrange(1 << 20))
        if op != "prompt":
            qhi = 1 if rng.random() < 0.4 else _log(rng, 2, 1500)
            c.update(qlo=max(1, int(qhi * rng.uniform(0.02, 1.0))), qhi=qhi,
                     ones=rng.randint(0, B // 2), page=rng.choice([16, 32, 64, 128]))
        if op != "plan":
            c.update(dtype=rng.choice(["f16", "bf16"]), **_heads(rng))
        if op == "append":
            c.update(src=rng.choice(["f32", "f16", "bf16"]), inter=rng.random() < 0.3,
                     rot=c["d"] if rng.random() < 0.7 else c["d"] // 2)
        if op in ("paged", "prompt"):
            c["window"] = 0 if rng.random() < 0.8 else _log(rng, 2, 4096)
        if op == "prompt":
            c["causal"] = rng.random() < 0.75
            c["window"] = c["window"] if c["causal"] else 0
        w = work(c)
        if w["flops"] + w["bytes"] <= top[op] and _padded(c) <= 3.0e9:
            return c


# ------------------------------------------------------------------- lengths
def _spread(n, lo, hi, order):
    """n lengths between lo and hi, evenly over their logarithm."""
    v = [int(round(lo * (hi / lo) ** ((i + 0.5) / n))) for i in range(n)]
    random.Random(order).shuffle(v)
    return v


def _lengths(c):
    """(cached tokens, new tokens) of every request; a prompt has none cached."""
    n = _spread(c["B"], c["lo"], c["hi"], c["lens"])
    if c["op"] == "prompt":
        return [0] * c["B"], n
    q = _spread(c["B"], c["qlo"], c["qhi"], c["lens"] + 1)
    return n, [1 if i < c["ones"] else x for i, x in enumerate(q)]


def _padded(c):
    """Scores that the padded plain form holds at once."""
    if c["op"] not in ("paged", "prompt"):
        return 0
    ctx, new = _lengths(c)
    return c["B"] * c["hq"] * max(new) * max(a + b for a, b in zip(ctx, new))


def _pairs(c):
    """Query-key pairs that the masks leave."""
    ctx, new = _lengths(c)
    total = 0
    for a, n in zip(ctx, new):
        if c["op"] == "prompt" and not c["causal"]:
            total += n * n
        elif not c["window"]:
            total += n * a + n * (n + 1) // 2
        else:
            total += sum(min(a + i + 1, c["window"]) for i in range(n))
    return total


def work(c):
    ctx, new = _lengths(c)
    T, kv = sum(new), sum(a + b for a, b in zip(ctx, new))
    if c["op"] == "plan":
        table = sum(-(-(a + b) // c["page"]) for a, b in zip(ctx, new))
        return {"bytes": 4 * (2 * c["B"] + table) + 8 * T + 4 * (2 * c["B"] + 1), "flops": 0}
    if c["op"] == "append":
        values = T * (c["hq"] + 2 * c["hkv"]) * c["d"]
        return {"bytes": values * (2 + (4 if c["src"] == "f32" else 2)) + 8 * T, "flops": 0}
    if c["window"]:  # keys behind every new token's window are not read
        kv = sum(min(a + b, b + c["window"] - 1) for a, b in zip(ctx, new))
    return {"bytes": 4 * kv * c["hkv"] * c["d"] + 4 * T * c["hq"] * c["d"],
            "flops": 4 * c["d"] * c["hq"] * _pairs(c)}


# -------------------------------------------------------------------- inputs
class _State:
    """What the program keeps from step to step, and this step's inputs."""


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


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

    if c["op"] != "prompt":
        P = c["page"]
        s.W = -(-s.max_kv // P) + 2  # the table has room for more
        held = [-(-a // P) for a in ctx]
        total = [-(-(a + b) // P) for a, b in zip(ctx, new)]
        s.pages = sum(total) + 7
        order = torch.randperm(s.pages, device="cuda", generator=g).int()
    if c["op"] == "plan":
        s.ctx, s.new = _i32(ctx), _i32(new)
        start = _i32([sum(held[:i]) for i in range(B)])[:, None]
        w = torch.arange(s.W, device="cuda")[None]
        has = w < _i32(held)[:, None]
        s.table = torch.where(has, order[(start + w).clamp(max=s.pages - 1)], -1).int()
        n = s.pages - sum(held)
        s.free = torch.full((s.pages,), -1, dtype=torch.int32, device="cuda")
        s.free[:n] = order[sum(held):]
        s.free_count = _i32([n])
        # a step has room for more tokens than it carries, as a captured one does
        s.room = T + 5
        return s

    if c["op"] != "prompt":  # the step's plan: filled tables
        start = _i32([sum(total[:i]) for i in range(B)])[:, None]
        w = torch.arange(s.W, device="cuda")[None]
        s.table = torch.where(w < _i32(total)[:, None], order[(start + w).clamp(max=s.pages - 1)], 0).int()
        shape = (s.pages, c["hkv"])
        s.k_cache = _normal(shape + (c["d"] // 8, P, 8), c["dtype"], g)
        s.v_cache = _normal(shape + (P // 8, c["d"], 8), c["dtype"], g)
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
    if c["op"] == "prompt":
        s.k = _normal((T, c["hkv"], c["d"]), c["dtype"], g)
        s.v = _normal((T, c["hkv"], c["d"]), c["dtype"], g)
    else:  # the buffer that the program keeps for split sums, zeroed once
        s.ws = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    return s


def _normal(shape, dtype, g):
    return torch.randn(shape, dtype=TYPES[dtype], device="cuda", generator=g)


# ----------------------------------------------------------------------- run
def run(s):
    if own:
        return _own(s)
    return {"plan": _plan, "append": _append, "paged": _paged, "prompt": _prompt}[s.c["op"]](s)


def _own(s):
    from inferflux_amd import attention
    c = s.c
    if c["op"] == "plan":
        p = attention.plan_batch(s.ctx, s.new, s.table, s.free, s.free_count, c["page"], s.room)
        return [p.cu_q, p.kv_len, p.positions, p.slots, p.free_left, p.status, s.table]
    if c["op"] == "append":
        attention.rope_append(s.q, s.k, s.v, s.pos, s.slots, s.k_cache, s.v_cache, s.freq,
                              interleaved=c["inter"], q_out=s.q_out)
        return [s.q_out, s.k_cache, s.v_cache]
    if c["op"] == "paged":
        return attention.paged_attention(s.q, s.k_cache, s.v_cache, s.table, s.cu, s.kv, s.max_q,
                                         s.max_kv, scale=s.scale, window=c["window"], out=s.out,
                                         workspace=s.ws)
    return attention.prompt_attention(s.q, s.k, s.v, s.cu, s.max_q, causal=c["causal"],
                                      window=c["window"], scale=s.scale, out=s.out)


def _plan(s):
    P, B = s.c["page"], s.c["B"]
    ctx, new = s.ctx.long(), s.new.long()
    held, total = (ctx + P - 1) // P, (ctx + new + P - 1) // P
    before = (total - held).cumsum(0) - (total - held)
    cu = torch.zeros(B + 1, dtype=torch.int64, device="cuda")
    cu[1:] = new.cumsum(0)
    # pages come from the end of the free list, in the order of the requests
    w = torch.arange(s.W, device="cuda")[None]
    at = s.free_count.long() - 1 - (before[:, None] + w - held[:, None])
    taken = (w >= held[:, None]) & (w < total[:, None])
    s.table.copy_(torch.where(taken, s.free[at.clamp(0, s.pages - 1)], s.table))
    t = torch.arange(s.room, device="cuda")
    r = torch.searchsorted(cu[1:], t, right=True).clamp(max=B - 1)
    live = t < cu[-1]
    pos = torch.where(live, ctx[r] + t - cu[r], 0)
    slot = torch.where(live, s.table[r, pos // P].long() * P + pos % P, -1)
    left = s.free_count - (total - held).sum().int()
    return [cu.int(), (ctx + new).int(), pos.int(), slot.int(), left, torch.zeros_like(left), s.table]


def _append(s):
    c, dt = s.c, TYPES[s.c["dtype"]]
    h, d, P = c["rot"] // 2, c["d"], c["page"]
    angle = s.pos.double()[:, None, None] * s.freq  # 64 bits: positions times frequencies reach far
    cos, sin = angle.cos().float(), angle.sin().float()

    def rotate(x):
        x = x.float()
        if c["inter"]:
            a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
        else:
            a, b = x[..., :h], x[..., h:2 * h]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
        return torch.cat([y, x[..., 2 * h:]], dim=-1).to(dt)

    s.q_out.copy_(rotate(s.q))
    page, at = s.slots.long() // P, s.slots.long() % P
    s.k_cache[page, :, :, at] = rotate(s.k).view(s.T, c["hkv"], d // 8, 8)
    s.v_cache[page, :, at // 8, :, at % 8] = s.v.to(dt)
    return [s.q_out, s.k_cache, s.v_cache]


def _rows(s):
    """Row numbers of the padded form [B, max_q], and (request, row) of every
    token."""
    i = torch.arange(s.max_q, device="cuda")
    at = (s.cu[:-1, None] + i).clamp(max=s.T - 1).long()
    t = torch.arange(s.T, device="cuda")
    r = torch.searchsorted(s.cu[1:].long(), t, right=True)
    return at, r, t - s.cu[r]


def _softmax_v(s, k, v, first):
    """Attention of the padded queries on k, v [B, hkv, L, d] in 32 bits; the
    query of row i of a request is at position first + i."""
    c = s.c
    B, L, G = c["B"], k.shape[2], c["hq"] // c["hkv"]
    at, r, row = _rows(s)
    q = s.q[at].float().view(B, s.max_q, c["hkv"], G, c["d"]).permute(0, 2, 3, 1, 4)
    q = q.reshape(B * c["hkv"], G * s.max_q, c["d"])
    x = torch.bmm(q, k.reshape(B * c["hkv"], L, c["d"]).transpose(1, 2).contiguous()) * s.scale
    x = x.view(B, c["hkv"], G, s.max_q, L)
    j = torch.arange(L, device="cuda")
    p = (first[:, None] + torch.arange(s.max_q, device="cuda"))[:, :, None]
    seen = (j < s.kv[:, None, None]).expand(B, s.max_q, L)
    if c["op"] == "paged" or c["causal"]:
        seen = seen & (j <= p)
    if c["window"]:
        seen = seen & (j > p - c["window"])
    x.masked_fill_(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    x.sub_(top).exp_()
    o = torch.bmm(x.view(B * c["hkv"], G * s.max_q, L), v.reshape(B * c["hkv"], L, c["d"]))
    total = x.sum(-1).view(B * c["hkv"], G * s.max_q, 1)
    o = torch.where(total > 0, o / total, 0.0)
    o = o.view(B, c["hq"], s.max_q, c["d"])
    s.out.copy_(o[r, :, row])
    return s.out


def _paged(s):
    c, P = s.c, s.c["page"]
    W = -(-s.max_kv // P)
    page = s.table[:, :W].long()
    k = s.k_cache[page].float().permute(0, 2, 1, 4, 3, 5)  # B, hkv, W, P, d / 8, 8
    v = s.v_cache[page].float().permute(0, 2, 1, 3, 5, 4)  # B, hkv, W, P / 8, 8, d
    shape = (c["B"], c["hkv"], W * P, c["d"])
    return _softmax_v(s, k.reshape(shape), v.reshape(shape), s.kv - (s.cu[1:] - s.cu[:-1]))


def _prompt(s):
    at, _, _ = _rows(s)
    k, v = (x[at].float().transpose(1, 2) for x in (s.k, s.v))
    return _softmax_v(s, k, v, torch.zeros_like(s.kv))


# ------------------------------------------------------------ the definition
def exact(c, seed):
    """The outputs in 64 bits, request by request and head by head."""
    s = prepare(c, seed)
    ctx, new = _lengths(c)
    if c["op"] == "plan":
        return None
    if c["op"] == "append":
        return _exact_append(s)
    out = torch.zeros(s.T, c["hq"], c["d"], dtype=torch.float64, device="cuda")
    G, t0 = c["hq"] // c["hkv"], 0
    for b in range(c["B"]):
        L, n = ctx[b] + new[b], new[b]
        for h in range(c["hkv"]):
            if c["op"] == "prompt":
                k, v = s.k[t0:t0 + n, h].double(), s.v[t0:t0 + n, h].double()
            else:
                where = torch.arange(L, device="cuda")
                page, at = s.table[b].long()[where // c["page"]], where % c["page"]
                k = s.k_cache[page, h, :, at].double().reshape(L, c["d"])
                v = s.v_cache[page, h, at // 8, :, at % 8].double()
            for i in range(0, n, 2048):
                m = min(2048, n - i)
                mine = torch.arange(ctx[b] + i, ctx[b] + i + m, device="cuda")[:, None]
                keys = torch.arange(L, device="cuda")[None]
                hide = torch.zeros(m, L, dtype=torch.bool, device="cuda")
                if c["op"] == "paged" or c["causal"]:
                    hide |= keys > mine
                if c["window"]:
                    hide |= keys <= mine - c["window"]
                for e in range(h * G, (h + 1) * G):
                    x = s.q[t0 + i:t0 + i + m, e].double() @ k.T * s.scale
                    x[hide] = -math.inf
                    x = (x - x.max(1, keepdim=True).values).exp()
                    out[t0 + i:t0 + i + m, e] = (x @ v) / x.sum(1, keepdim=True)
        t0 += n
    return out


def _exact_append(s):
    c, P = s.c, s.c["page"]
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
    # slots of the cache, token by token in memory order, then back to pages
    k = s.k_cache.double().permute(0, 3, 1, 2, 4).reshape(-1, c["hkv"], c["d"])
    v = s.v_cache.double().permute(0, 2, 4, 1, 3).reshape(-1, c["hkv"], c["d"])
    k[s.slots.long()] = got[1]
    v[s.slots.long()] = s.v.double()
    k = k.view(-1, P, c["hkv"], c["d"] // 8, 8).permute(0, 2, 3, 1, 4).contiguous()
    v = v.view(-1, P // 8, 8, c["hkv"], c["d"]).permute(0, 3, 1, 4, 2).contiguous()
    return [got[0], k, v]
