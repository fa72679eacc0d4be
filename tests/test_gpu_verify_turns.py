"""Verification where a request's chunk of the row is looked through in several
turns: the token of an early turn stays the one drawn when later turns hold nothing."""
import random

import pytest

from tests.test_gpu_drafts import dev, run_verify  # noqa: F401
from tests.test_gpu_parity import note

pytestmark = pytest.mark.gpu

TURN = 4096  # values of a row that a workgroup looks at in one turn


@pytest.mark.parametrize("B,dtype", [(512, "f32"), (1025, "bf16")])  # two chunks of a row, one
@pytest.mark.parametrize("turns", [(0,), (0, 2), (1,), (0, 1, 2)])
def test_turns_that_hold_nothing(dev, B, dtype, turns):  # noqa: F811
    """Equal weights in some turns, numbers at their sums, next to them, and 1: then no
    sum passes and the last weight's token is drawn."""
    import torch
    note(f"verify turns B={B} {dtype} {turns}")
    rng, V = random.Random(B + len(turns)), 3 * TURN + 5
    at = sorted({t * TURN + x for t in turns for x in (0, 15, 16, 17, 1023, 1024, 4095)})
    p = torch.zeros(B, V, device=dev)
    p[:, at] = 0.03125
    su = [rng.choice([1.0, 1 - 2.0 ** -24, 0.0, rng.randrange(len(at)) / len(at) + rng.choice([0, 2.0 ** -20])])
          for _ in range(B)]
    run_verify(dev, [1] * B, [-1] * B, [rng.choice(at) for _ in range(B)], p, [0.5] * B, su, dtype=dtype)


def test_no_requests(dev):  # noqa: F811
    """cu_q of one value or none is refused as other bad arguments are."""
    import torch
    from inferflux_amd import attention as at, drafts
    ws = at.workspace(dev)
    for T in (0, 3):
        for n in (0, 1):
            with pytest.raises(ValueError):
                drafts.verify(torch.zeros(T, dtype=torch.int32, device=dev), torch.zeros(n, dtype=torch.int32, device=dev),
                              torch.ones(T, 5, device=dev), torch.zeros(T, device=dev), torch.zeros(0, device=dev), 4,
                              workspace=ws)
