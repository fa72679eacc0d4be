"""The 8-bit cache's definition (include/ifx_attention_q8.h) in 64 bits; shared
by its tests."""
import math

import torch


def bf16_not_below(x):
    """The smallest bfloat16 that is no less than x >= 0 (float64), as float64."""
    f = x.float()
    f = torch.where(f.double() < x, torch.nextafter(f, torch.full_like(f, math.inf)), f)
    return ((f.view(torch.int32) + 0xFFFF) & ~0xFFFF).view(torch.float32).double()


def quantise(x):
    """Codes (float64) and scales [..., 1] of rows x (float64)."""
    fine = torch.isfinite(x).all(-1, keepdim=True)
    y = torch.where(fine, x, 0.0)
    s = bf16_not_below(y.abs().amax(-1, keepdim=True) / 127)
    codes = torch.where(s > 0, torch.round(y / torch.where(s > 0, s, 1.0)), 0.0)
    return codes, torch.where(fine, s, math.nan)


def rotate(x, pos, freq, interleaved):
    """Rows [T, H, D] rotated in 64 bits."""
    x = x.double()
    if freq is None:
        return x
    h = freq.numel()
    # as turns, so that positions far out keep their angle's bits
    angle = pos.double()[:, None, None] * freq
    cos, sin = angle.cos(), angle.sin()
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
        y[..., 0:2 * h:2], y[..., 1:2 * h:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :h], x[..., h:2 * h]
        y[..., :h], y[..., h:2 * h] = a * cos - b * sin, b * cos + a * sin
    return y


def put(cache, slots, k, ks, v, vs):
    """Writes codes and scales [N, Hkv, D], [N, Hkv, 1] at slots."""
    P, D = cache.k.shape[3], k.shape[2]
    page, at = slots.long() // P, slots.long() % P
    cache.k[page, :, :, at] = k.to(torch.int8).unflatten(2, (D // 16, 16))
    cache.v[page, :, at // 16, :, at % 16] = v.to(torch.int8)
    cache.scales[page, :, at] = torch.cat([ks, vs], -1).to(torch.bfloat16)


def get(cache, slots):
    """Values (float64) [N, Hkv, D] of K and V, and V's scales [N, Hkv]."""
    P = cache.k.shape[3]
    page, at = slots.long() // P, slots.long() % P
    s = cache.scales[page, :, at].double()
    k = cache.k[page, :, :, at].flatten(2).double() * s[..., :1]
    v = cache.v[page, :, at // 16, :, at % 16].double() * s[..., 1:]
    return k, v, s[..., 1]
