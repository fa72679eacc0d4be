"""Plain 64-bit forms of the attention operators (include/ifx_attention.h) and
the bounds that their kernels' roundings obey; shared by the attention tests."""
import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}


def gather_cache(k_cache, v_cache, pages, n):
    """K, V [n, Hkv, D] (float64) of a request whose table row is `pages`."""
    P = k_cache.shape[3]
    j = torch.arange(n, device=k_cache.device)
    page, at = pages.long()[j // P], j % P
    k = k_cache[page, :, :, at].double().flatten(2)
    v = v_cache[page, :, at // 8, :, at % 8].double()
    return k, v


def put_cache(k_cache, v_cache, pages, k, v):
    """Writes k, v [n, Hkv, D] as the first n tokens of the table row `pages`."""
    n, P = k.shape[0], k_cache.shape[3]
    j = torch.arange(n, device=k_cache.device)
    page, at = pages.long()[j // P], j % P
    k_cache[page, :, :, at] = k.to(k_cache.dtype).unflatten(2, (-1, 8))
    v_cache[page, :, at // 8, :, at % 8] = v.to(v_cache.dtype)


def attend(q, k, v, first, scale, causal=True, window=0):
    """softmax(scale q k^T) v for q [n, Hq, D] at positions first + i and k, v
    [L, Hkv, D]; only what a row sees enters it, a row that sees nothing is 0.
    Returns (out, bound): how far a kernel may be off before its output
    rounding, from
      - the probabilities' rounding to q's type, half a step each: u A with
        A = sum p |v| / sum p;
      - fp16: probabilities under 2^-24, scaled by 2^6 at least against a sum of
        1 or more: 2^-31 a key;
      - fp32 scores: D products and their sum, (D + 4) 2^-23 sum |q k| scale,
        and the rounding of the exponent's argument, in natural units; the
        error of p relative to p is that, twice over as it enters the sum too;
      - fp32 sums over the keys: L 2^-23 A for the values and for the weights."""
    dt = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    n, Hq, D = q.shape
    L, Hkv = k.shape[0], k.shape[1]
    G = Hq // Hkv
    out = torch.zeros(n, Hq, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    pos = first + torch.arange(n, device=q.device)[:, None]
    j = torch.arange(L, device=q.device)[None]
    seen = (j <= pos) if causal else torch.ones(n, L, dtype=torch.bool, device=q.device)
    if window:
        seen = seen & (j > pos - window)
    some = seen.any(1)
    for h in range(Hq):
        kh, vh = k[:, h // G], v[:, h // G]
        s = scale * (q[:, h] @ kh.T)
        s = torch.where(seen, s, -math.inf)
        p = torch.softmax(s, 1)
        p = torch.where(seen, p, 0.0)
        # unseen keys have no influence, whatever they hold
        bad = ~torch.isfinite(vh).all(1)
        o = p @ torch.where(bad[:, None], 0.0, vh)
        for x in bad.nonzero().flatten().tolist():
            o = torch.where(seen[:, x:x + 1], o + p[:, x:x + 1] * vh[x], o)
        out[:, h] = torch.where(some[:, None], o, 0.0)
        mag = (q[:, h].abs() @ torch.nan_to_num(kh, 0, 0, 0).abs().T * scale)
        mag = torch.where(seen, mag, 0.0).amax(1, keepdim=True)
        A = p.nan_to_num(0) @ torch.nan_to_num(vh, 0, 0, 0).abs()
        top = torch.nan_to_num(vh, 0, 0, 0).abs().amax()
        e = U[dt] + 2 * (D + 8) * 2.0 ** -23 * mag + 2 * (L + 16) * 2.0 ** -23
        bound[:, h] = e * A + (L * 2.0 ** -31 * top if dt == torch.float16 else 0.0)
    return out, bound


def check(got, ref, bound, what=""):
    """got (any type) against ref within the bound and one rounding of got's
    type; infinities and NaN in the same places."""
    fine = torch.isfinite(ref)
    g = got.double()
    assert torch.equal(fine, torch.isfinite(g)), f"{what}: non-finite values elsewhere"
    assert torch.equal(torch.isnan(ref), torch.isnan(g)), f"{what}: NaN elsewhere"
    tol = bound + U[got.dtype] * (ref.abs() + bound) + TINY[got.dtype]
    off = torch.where(fine, (g - ref).abs() - tol, 0.0)
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 0, (f"{what}: off by up to {float(torch.where(fine, (g - ref).abs(), 0.0).max()):.3g}, "
                        f"{worst:.3g} over its bound at {int(off.argmax())}")
