"""Plain forms of what a step does with drafted tokens (include/ifx_drafts.h),
request by request in Python and 64 bits; shared by the drafts' and the 8-bit
cache's tests."""
import random

import torch

from tests.attn_ref import U


def tree(rng, n, reach=4):
    """Parents of a random tree of n nodes, the root first."""
    return [-1] + [rng.randint(max(0, j - reach), j - 1) for j in range(1, n)]


def ways(parents):
    """For each node the nodes on its way to the root, itself among them."""
    got = []
    for i, p in enumerate(parents):
        got.append((got[p] if 0 <= p < i else set()) | {i})
    return got


def seen_by_tree(masks, ctx, n, L):
    """[n, L] of bool: what the rows see, masks: sets of nodes or integers."""
    seen = torch.zeros(n, L, dtype=torch.bool)
    for i, m in enumerate(masks):
        seen[i, :max(ctx, 0)] = True
        for j in range(min(n, 64)):
            on = j in m if isinstance(m, set) else m >> j & 1
            if on and 0 <= ctx + j < L:
                seen[i, ctx + j] = True
    return seen


def attend_seen(q, k, v, seen, scale, weigh=None):
    """softmax(scale q k^T) v of q [n, Hq, D] over k, v [L, Hkv, D] where seen
    [n, L]; a row that sees nothing is 0.  Returns (out, bound) as
    tests.attn_ref.attend does, with the same terms; `weigh`: half a step of
    what the probabilities are rounded to, q's type if None."""
    dt = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    seen = seen.to(q.device)
    n, Hq, D = q.shape
    L, Hkv = k.shape[0], k.shape[1]
    G = Hq // Hkv
    out = torch.zeros(n, Hq, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    if L == 0:
        return out, bound
    some = seen.any(1)
    u = U[dt] if weigh is None else weigh
    for h in range(Hq):
        kh, vh = k[:, h // G], v[:, h // G]
        s = torch.where(seen, scale * (q[:, h] @ kh.T), -torch.inf)
        p = torch.where(seen, torch.softmax(s, 1), 0.0)
        bad = ~torch.isfinite(vh).all(1)
        o = p @ torch.where(bad[:, None], 0.0, vh)
        for x in bad.nonzero().flatten().tolist():
            o = torch.where(seen[:, x:x + 1], o + p[:, x:x + 1] * vh[x], o)
        out[:, h] = torch.where(some[:, None], o, 0.0)
        mag = q[:, h].abs() @ torch.nan_to_num(kh, 0, 0, 0).abs().T * scale
        mag = torch.where(seen, mag, 0.0).amax(1, keepdim=True)
        fine = torch.nan_to_num(vh, 0, 0, 0).abs()
        e = u + 2 * (D + 8) * 2.0 ** -23 * mag + 2 * (L + 16) * 2.0 ** -23
        bound[:, h] = e * (p.nan_to_num(0) @ fine)
        if u == U[torch.float16]:
            bound[:, h] += L * 2.0 ** -31 * fine.amax()
    return out, bound


def walk(parents, tokens, p, accept_u, sample_u, q=None):
    """(path, token drawn) of one request: p, q [n][V] lists of lists of floats
    (None: drafts without probabilities); parents None: a chain."""
    n, V = len(tokens), len(p[0])
    fine = lambda x: x if x > 0 else 0.0  # noqa: E731  NaN and negative values are 0
    parents = list(range(-1, n - 1)) if parents is None else parents
    path = [0]
    while True:
        i = path[-1]
        row = [fine(x) for x in p[i]]
        children = [j for j in range(i + 1, n) if parents[j] == i]
        to, w = None, list(row)
        if q is not None:
            if children:
                x = tokens[i + 1]
                other = [fine(y) for y in q[i]]
                if 0 <= x < V and accept_u[i] * other[x] < row[x]:
                    to = i + 1
                w = [max(a - b, 0.0) for a, b in zip(row, other)]
        else:
            part, met = 0.0, set()
            for j in children:
                x = tokens[j]
                if x in met:
                    continue
                met.add(x)
                if not 0 <= x < V:
                    continue
                part += row[x]
                w[x] = 0.0
                if to is None and accept_u[i] < part:
                    to = j
        if to is None:
            break
        path.append(to)
    if not sum(w) > 0:
        w = row
    if not sum(w) > 0:
        return path, -1
    at, goal, last = 0.0, max(sample_u, 0.0) * sum(w), -1
    for v, x in enumerate(w):
        at += x
        last = v if x > 0 else last
        if at > goal:
            return path, v
    return path, last


def verify(parents, tokens, cu, p, accept_u, sample_u, q=None, max_q=64):
    """accepted, path, emitted as lists; parents, tokens, p, q: rows of all requests."""
    accepted, paths, emitted = [], [], []
    for b in range(len(cu) - 1):
        rows = cu[b + 1] - cu[b]
        n = min(rows, max_q)
        if rows <= 0:
            accepted.append(-1)
            continue
        s = slice(cu[b], cu[b] + n)
        path, token = walk(None if parents is None else parents[s], tokens[s], p[s], accept_u[s],
                           sample_u[b], None if q is None else q[s])
        accepted.append(len(path) - 1)
        paths += path + [-1] * (rows - len(path))
        emitted += [tokens[cu[b] + j] for j in path[1:]] + [token] + [-1] * (rows - len(path))
    return accepted, paths, emitted


def keep(ctx, n, path, accepted):
    """[(from, to)] tokens of one request."""
    moves = min(accepted, n - 1)
    return [(ctx + path[i], ctx + i) for i in range(1, moves + 1) if path[i] > i]


def rand_lengths(rng, B, hi):
    return [rng.choice([0, 1, rng.randint(1, hi), hi]) for _ in range(B)]


__all__ = ["tree", "ways", "seen_by_tree", "attend_seen", "walk", "verify", "keep", "rand_lengths", "random"]
