"""GPU: attention over a paged int8 cache and appending to it, at the edges: V scales that are zero for long stretches, scores that are not numbers, pages, ends and
lengths that lie outside, batches of long and short runs of rows.  Tolerances as derived in test_gpu_paged_attention.py.  On 128-row tiles the
reference that w = p v_scale is relative to may be up to 2^15 behind the row's largest w: fp16 rounds it to 2^-11 there as well, and the absolute term, 2^-25 of
the reference, is a smaller part of the largest w."""
import math

import pytest
import torch

import test_gpu_paged_attention as base
from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu


def far_below(s, low=80, most=150.0):
    """Every score far below zero: q's codes are positive and K's negative.  Returns the largest and the least exponent (log2) of a score."""
    s.q8.copy_(s.q8.abs().clamp(low, 127))
    s.kc.copy_(-s.kc.abs().clamp(low, 127))
    unit = most / (s.kc.shape[3] * low * low)
    s.qs.fill_(0.02)
    s.ks.copy_(torch.where(torch.isnan(s.ks), s.ks, torch.full_like(s.ks, unit * math.log(2) / (0.02 * s.scale))))
    return -most, -s.kc.shape[3] * 127 * 127 * unit


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("D,zeros", [(64, 64), (64, 200), (128, 64), (128, 250), (256, 130)])
def test_values_of_zero_ahead_of_scores_far_below(D, zeros, path, pkg):
    """A run of all-zero values (scale 0), then ordinary ones whose p, relative to 1, are below what fp32 holds."""
    s = base.Setup([100, 3, 70], [400, 303, 270], 8, 2, D, 16, 1, seed=zeros)
    s.path = path
    most, least = far_below(s)
    assert most < -140
    for i, n in enumerate(s.lens.tolist()):
        for key in range(min(zeros, n)):
            page, slot = int(s.table[i, key // 16]), key % 16
            s.vs[page, :, slot] = 0
            s.vc[page, :, slot] = 0
    # exponents up to `least` in magnitude: three roundings of a product and a difference, 4 * |least| * 2^-24; p by ln 2 times that, p / sum p by twice
    # as much
    more = 4 * -least * 2.0 ** -24 * math.log(2) * 2
    for causal in (True, False):
        o = s.check(pkg, causal, torch.bfloat16, more=more)
        assert (o[:100].abs().amax(-1) > 0).all()
