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


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("v_zero", [False, True])
@pytest.mark.parametrize("what", ["row", "chunks", "length"])
def test_scores_that_are_not_numbers(what, v_zero, path, pkg):
    """A query scale, or the K scales of a sequence's first tokens, are NaN: the rows that see them are, and so are their sums."""
    s = base.Setup([100, 3, 70], [400, 303, 70], 8, 2, 128, 16, 1, seed=7)
    s.path = path
    bad = torch.zeros(173, 8, dtype=torch.bool, device="cuda")
    if what == "row":
        bad[[0, 5, 101, 110, 172], 3] = True
        s.qs[bad] = float("nan")
    else:
        n = 64 if what == "chunks" else 400
        for i in (0, 2):
            for key in range(min(n, int(s.lens[i]))):
                s.ks[int(s.table[i, key // 16]), 1, key % 16] = float("nan")
        bad[:100, 4:] = True
        bad[103:, 4:] = True
    if v_zero:                               # zero V scales among them: the sums are made the general way
        for i in (0, 2):
            s.vs[int(s.table[i, 0]), :, 3:7] = 0
            s.vs[int(s.table[i, 0]), :, 0] = 0
    want, wlse, A, B = O.attention(s.q8, s.qs, s.kc, s.vc, s.ks, s.vs, s.table, s.lens, s.cu, True, s.scale)
    o, lse = s.call(pkg, return_lse=True)
    assert torch.equal(torch.isnan(wlse), bad) and torch.equal(torch.isnan(want).all(-1), bad)
    assert torch.equal(torch.isnan(lse), bad)
    assert torch.equal(torch.isnan(o), bad[..., None].expand_as(o))
    # The others to the rounding of any row.  (Not bit for bit what they are without their neighbours' NaN: on tiles the 32 rows of a warp look for new
    # references together, and w, relative to another one, is rounded elsewhere.)
    assert ((o.double() - want).abs() <= s.tolerance(want, A, B))[~bad].all()
    assert ((lse.double() - wlse).abs() <= 2.0 ** -16 * 64)[~bad].all()
    pkg.check_status()
