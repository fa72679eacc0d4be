"""K's codes in the 8-bit cache against angles that are reduced exactly: positions
times frequencies as rational numbers, less whole turns, before anything is rounded."""
import math
import random
from fractions import Fraction

import pytest

from tests import q8_ref
from tests.test_gpu_attention import gen, i32
from tests.test_gpu_attention_q8 import dev  # noqa: F401
from tests.test_gpu_parity import note

pytestmark = pytest.mark.gpu

# pi to 50 digits
PI = Fraction(314159265358979323846264338327950288419716939937510, 10 ** 50)


def turned(pos, freq):
    """cos and sin [T, h] (float64) of pos * freq, off by less than 2^-52."""
    import torch
    cos, sin = [], []
    for p in pos:
        row = [float((Fraction(p) * Fraction(f)) % (2 * PI)) for f in freq]
        cos.append([math.cos(x) for x in row])
        sin.append([math.sin(x) for x in row])
    return torch.tensor(cos, dtype=torch.float64), torch.tensor(sin, dtype=torch.float64)


@pytest.mark.parametrize("far", [1000, 100000, 1 << 24])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,Hq,Hkv", [(96, 1, 2), (304, 8, 8)])  # one token a workgroup, eight
def test_codes_of_k(dev, far, inter, T, Hq, Hkv):  # noqa: F811
    import torch
    from inferflux_amd import attention_q8 as q8
    note(f"append q8 angles far={far} {inter} T={T}")
    D, P = 128, 16
    rng = random.Random(far)
    pos = [rng.randrange(far) for _ in range(T - 1)] + [far]
    freq = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    g = gen(dev, far)
    q, k, v = (torch.randn(T, h, D, generator=g, device=dev) for h in (Hq, Hkv, Hkv))
    c = q8.kv_cache(T // P, Hkv, D, P, device=dev)
    q8.rope_append(q, k, v, i32(pos, dev), torch.arange(T, device=dev).int(), c, freq.to(dev), interleaved=inter)
    cos, sin = (x[:, None] for x in turned(pos, freq.tolist()))
    x = k.double().cpu()
    y = torch.empty_like(x)
    a, b = (x[..., 0::2], x[..., 1::2]) if inter else (x[..., :D // 2], x[..., D // 2:])
    ya, yb = a * cos - b * sin, b * cos + a * sin
    if inter:
        y[..., 0::2], y[..., 1::2] = ya, yb
    else:
        y[..., :D // 2], y[..., D // 2:] = ya, yb
    codes, scales = q8_ref.quantise(y)
    at = torch.arange(T)
    got_s = c.scales.cpu()[at // P, :, at % P, :1].double()
    got = c.k.cpu()[at // P, :, :, at % P].flatten(2).double()
    # The kernel forms turns = position * frequency / 2 pi: 1 / 2 pi to half a step and two
    # products, 3 x 2^-53 of far / 2 pi turns, which is as much of far in the angle, and
    # moves a value by up to that times its pair's length; beside it sine, cosine, products
    # and sum, some 2^-50 of the length.  The reference's own is 2^-50 of it too.
    length = (a * a + b * b).sqrt()
    length = torch.stack((length, length), -1).flatten(-2) if inter else torch.cat((length, length), -1)
    off = length * (3 * far * 2.0 ** -53 + 2.0 ** -49)
    # scales: the smallest bf16 that is no less than the largest value's 127th, which could
    # fall on either side of a bf16 only within `off` of it
    top = y.abs().amax(-1, keepdim=True)
    near = off.amax(-1, keepdim=True)
    sure = q8_ref.bf16_not_below((top - near) / 127) == q8_ref.bf16_not_below((top + near) / 127)
    assert sure.all() and torch.equal(got_s, scales)
    # a code may only differ where the value lies within `off` of a border, and by one
    quotient = y / scales
    border = (quotient - (quotient.floor() + 0.5)).abs() * scales
    assert ((got - codes).abs() <= (border <= off)).all()
