"""What the kernels of beam search hold in 32 bits, and the forms that only large calls reach (see test_beams_gpu.py for the rest)."""
import math

import pytest
import torch

from deliverance_amd.kernels import ops
from test_beams_gpu import DEV, attend, beams_case, quick

pytestmark = pytest.mark.gpu


@quick
@pytest.mark.parametrize("length,shared", [(3, 0), (65, 64), (113, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_keep_their_32_bits(length, shared, dtype):
    """The first key has the score 0 and the value 0, the others by turns the scores -x and -x - d and the values 1 and -1: the result is a
    small difference of weights about e^-x.  Scores are exact, a 32-bit weight is off by 2^-23 of itself (its exponential and the product before
    it); that is the slack, beside half a step of the result.  (16 bits a weight leave the result off by some 2^-19.)"""
    c = beams_case(1, 3, 2, 1, 16, 16, dtype, [length] * 3, [shared], seed=3)
    x = torch.tensor([77.0, 81.0, 85.0, 91.0, 99.0, 111.0]) / 256                          # of (beam, head); exact in bfloat16
    d = torch.tensor([1.0, 1.125, 1.25, 1.375, 1.5, 1.625]) * 2.0 ** -12
    q = torch.zeros(6, 16)
    q[:, 5], q[:, 6] = 4 * x, 4 * d                                                        # (scores are scaled by 1 / 4)
    c["q"] = q.view(3, 32).to(dtype).to(DEV)
    cache = torch.zeros_like(c["cache"].cpu())
    cache[:, 0, :, :, 5] = -1
    cache[:, 0, :, 0::2, 6] = -1
    v = cache[:, 1].view(-1, 1, 16, 16)
    v[..., 0::2], v[..., 1::2] = -1, 1
    for first in c["table"][:, 0].tolist():
        cache[first, 0, :, 0], v[first, :, :, 0] = 0, 0
    c["cache"] = cache.to(DEV)
    w1, w2 = torch.exp(-x.double()), torch.exp(-x.double() - d.double())
    n1, n2 = length // 2, (length - 1) // 2                # keys 1, 3, ..; keys 2, 4, ..
    want = ((n1 * w1 - n2 * w2) / (1 + n1 * w1 + n2 * w2)).view(3, 2).repeat_interleave(16, 1)
    got = attend(c).cpu().double()
    near = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -22
    assert bool(((got - want).abs() <= near).all()), ((got - want).abs() / near).max()
