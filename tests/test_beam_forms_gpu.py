"""What the kernels of beam search hold in 32 bits, and the forms that only large calls reach (see test_beams_gpu.py for the rest)."""
import math

import pytest
import torch

from deliverance_amd.kernels import ops
from test_beams_gpu import DEV, attend, beams_case, check_attention, check_select, quick

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


# Calls that reach what smaller ones do not: four loads of logits a wavefront (from 16,384 loads on) with long and with short segments, four segments' keys a
# thread (from 2,049 segments a group on), segments past the kept ones (from 4,097), segments numbered by a division (from 65,536).
@pytest.mark.parametrize("groups,beams,vocab,keep", [(32, 8, 131071, 16), (1, 8, 140000, 128), (600, 1, 7000, 12), (1, 64, 262145, 40), (3, 5, 262143, 10)])
def test_choices_among_many_logits(groups, beams, vocab, keep):
    g = torch.Generator().manual_seed(groups + vocab)
    logits = torch.randn(groups * beams, vocab, generator=g) * 3
    logits[:, 17::29] = -math.inf
    scores = -20 * torch.rand(groups * beams, generator=g)
    if beams > 2:
        scores[beams - 1::beams] = -math.inf
    check_select(logits.to(DEV), scores.to(DEV), beams, keep)


def test_equal_entries_among_many_logits():
    """The first ones in the order of beams and tokens, through the divisions too."""
    logits = torch.full((64, 262145), 0.5)
    logits[1:, 5::2] = 1.5
    check_select(logits.to(DEV), torch.full((64,), -2.0, device=DEV), 64, 128)


# Four wavefronts a workgroup: with more workgroups than compute units, and over many chunks, at every head size that has both forms.
FOUR_WAVES = [(9, 4, 32, 32, 128, 16, [140 + i % 3 for i in range(36)], [128] * 9), (9, 4, 32, 32, 32, 32, [100 + i % 5 for i in range(36)], [96] * 9),
              (10, 3, 28, 28, 64, 16, [90] * 30, [80] * 10), (9, 4, 30, 30, 80, 16, [70] * 36, [64] * 9),
              (1, 2, 2, 1, 128, 64, [3200, 3199], [3136]), (1, 3, 2, 2, 32, 16, [3164, 3149, 3137], [3136]), (1, 2, 1, 1, 64, 32, [3090, 3080], [1024]),
              (1, 2, 4, 2, 96, 16, [3105, 3105], [0])]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("groups,beams,heads,kv_heads,dim,page,lengths,shared", FOUR_WAVES)
def test_attention_of_beams_by_four_wavefronts(groups, beams, heads, kv_heads, dim, page, lengths, shared, dtype):
    c = beams_case(groups, beams, heads, kv_heads, dim, page, dtype, lengths, shared, seed=dim + beams)
    workgroups = groups * kv_heads * -(-beams * (heads // kv_heads) // 16)
    assert workgroups > 256 or c["table"].shape[1] * page // 64 >= 48
    check_attention(c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_groups_of_many_beams_over_windows(dtype):
    """Shared heads, windows that end inside shared pages and places without a beam, in one call."""
    c = beams_case(5, 6, 12, 3, 64, 16, dtype, [300 + 7 * (i // 6) if i % 6 != 4 else 0 for i in range(30)], [288] * 5, seed=8)
    for window in (1, 20, 64, 290):
        check_attention(c, window=window, splits=2)
