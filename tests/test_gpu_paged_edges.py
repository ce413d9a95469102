"""GPU: attention over a paged int8 cache and appending to it, at the edges: V scales that are zero for long stretches, scores that are not numbers, pages, ends and
lengths that lie outside, batches of long and short runs of rows.  Tolerances as derived in test_gpu_paged_attention.py.  On 128-row tiles the
reference that w = p v_scale is relative to may be up to 2^15 behind the row's largest w: fp16 rounds it to 2^-11 there as well, and the absolute term, 2^-25 of
the reference, is a smaller part of the largest w."""
import math

import pytest
import torch

import test_gpu_paged_append as append
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


def without(s, seq, columns):
    """The same rows over a cache in which the tokens of those columns of a sequence's table are not there."""
    t = base.Setup.__new__(base.Setup)
    t.__dict__.update(s.__dict__)
    t.table, t.lens = s.table.clone(), s.lens.clone()
    page, width = s.kc.shape[2], s.table.shape[1]
    keep = [c for c in range(width) if c not in columns]
    t.table[seq, :len(keep)] = s.table[seq, keep]
    t.lens[seq] -= page * len(columns)
    return t


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page,block", [(8, 1), (16, 4), (64, 64)])
@pytest.mark.parametrize("news,one,path", [([1, 1, 1], True, 1), ([1, 1, 1], False, 1), ([3, 2, 4], False, 1), ([70, 3, 130], False, 2), ([3, 1, 2], False, 2)])
def test_keys_of_pages_outside_the_cache_do_not_count(news, one, path, D, page, block, pkg):
    lens = [6 * page + 5 + news[0], 0, 11 * page + news[2]]
    s = base.Setup(news, lens, 8, 2, D, page, block, one=one, seed=page, garbage=False)
    s.path = path
    s.check(pkg)
    for seq, columns, to in ((0, [0], -1), (0, [3], s.kc.shape[0]), (2, [1, 2, 7], 1 << 30), (2, [10], -(1 << 31)), (0, list(range(6)), s.kc.shape[0])):
        want = without(s, seq, columns)
        was = s.table.clone()
        s.table[seq, columns] = to
        for causal in (True, False):
            got = s.call(pkg, causal, return_lse=True)
            with pytest.raises(pkg.IntfaError, match="outside its table"):
                pkg.check_status()
            want.check(pkg, causal, got=got)
        # nothing is taken from any page that is not in the tables
        others = torch.ones(s.kc.shape[0], dtype=torch.bool, device="cuda")
        others[s.table[(s.table >= 0) & (s.table < s.kc.shape[0])].long()] = False
        keep = [x.clone() for x in (s.kc, s.vc, s.ks, s.vs)]
        s.kc[others], s.vc[others], s.ks[others], s.vs[others] = 127, -127, float("nan"), float("inf")
        again = s.call(pkg, False, return_lse=True)
        assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])
        for x, y in zip((s.kc, s.vc, s.ks, s.vs), keep):
            x.copy_(y)
        with pytest.raises(pkg.IntfaError, match="outside its table"):
            pkg.check_status()
        s.table.copy_(was)


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("one", [True, False])
def test_a_sequence_without_a_page_in_the_cache(one, path, pkg):
    """Rows that see no key that is there: zero, and no sum."""
    s = base.Setup([1, 1], [100, 40], 8, 2, 128, 16, 1, one=one)
    s.path = path
    good = s.call(pkg)
    s.table[0] = -1
    o, lse = s.call(pkg, return_lse=True)
    assert (o[0] == 0).all() and (lse[0] == -math.inf).all() and torch.equal(o[1], good[1])
    with pytest.raises(pkg.IntfaError, match="outside its table"):
        pkg.check_status()


@pytest.mark.parametrize("path", [1, 2])
def test_values_of_zero_next_to_a_page_outside_the_cache(path, pkg):
    """Zero V scales, for which p is summed up by itself on tiles, in the chunk of a page that is not there: its keys count for nothing, the zeros' do."""
    s = base.Setup([40, 2], [170, 50], 8, 2, 128, 16, 1, garbage=False)
    s.path = path
    for col in (0, 2, 5):
        s.vs[int(s.table[0, col]), :, ::3] = 0
    want = without(s, 0, [1, 6])
    s.table[0, 1] = s.table[0, 6] = s.kc.shape[0]
    got = s.call(pkg, return_lse=True)
    with pytest.raises(pkg.IntfaError, match="outside its table"):
        pkg.check_status()
    want.check(pkg, got=got)


@pytest.mark.parametrize("block", [1, 8, 64])
@pytest.mark.parametrize("H,Hkv,D", [(2, 2, 64), (40, 8, 128), (3, 1, 256)])
@pytest.mark.parametrize("what", ["page", "width", "length", "rotation"])
def test_queries_of_refused_tokens_are_zero(what, H, Hkv, D, block, pkg):
    """With scale zero; the other sequences' as ever, and padding, which is left out."""
    s = append.Setup([5, 2, 60], [70, 2, 70], H, Hkv, D, 64, block)
    cs = pkg.rotary_table(100, D, device="cuda")
    refused = torch.zeros(67, dtype=torch.bool, device="cuda")
    if what == "page":                       # tokens 64 .. 69 of the last sequence
        s.table[2, 1] = s.kc.shape[0]
        refused[67 - 6:] = True
    elif what == "width":
        s.lens[0] = s.table.shape[1] * 64 + 5
        refused[:5] = True
    elif what == "length":
        s.lens[0] = -4
        refused[:5] = True
    else:
        cs = pkg.rotary_table(66, D, device="cuda")        # positions 65 .. 69 and 10 .. 69
        refused[1:5] = True
        refused[67 - 4:] = True
    pos = torch.cat([torch.arange(65, 70), torch.arange(2), torch.arange(10, 70)]).cuda()
    x = O.turn(s.q.float(), pkg.rotary_table(100, D, device="cuda")[pos][:, None], False)
    qs = O.scale_of(O.absmax(x))
    q8 = O.codes(x, qs[..., None])
    q8[refused], qs[refused] = 0, 0.0
    old = torch.full_like(q8, 77), torch.full_like(qs, 77.0)             # (what a new tensor is likely to hold)
    del old
    got = s.run(pkg, cs)
    with pytest.raises(pkg.IntfaError, match="outside its table"):
        pkg.check_status()
    assert torch.equal(got[0], q8) and torch.equal(got[1], qs)


@pytest.mark.parametrize("D,block", [(64, 32), (128, 16), (256, 8), (128, 64)])
def test_scales_that_grow_with_every_token(D, block, pkg):
    """Each token is larger than all before it, so that every append reads its block's scale, raises it and moves all older codes."""
    S, Hkv = 40, 3
    s = append.Setup([1] * S, [1 + i % 5 for i in range(S)], 0, Hkv, D, 64, block)
    s.table[s.table < 0] = 0
    for i in range(block + 3):
        s.k = (torch.randn(S, Hkv, D, device="cuda", generator=s.g) * 1.3 ** i).half()
        s.v = (torch.randn(S, Hkv, D, device="cuda", generator=s.g) * 1.3 ** (i % 9)).half()
        s.check(pkg, cu=None)
        s.lens += 1
        if int(s.lens.max()) > 64:             # (its only page is full)
            break


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("cu,valid", [([0, 160, 100], [0, 160, 160]), ([0, 100, 200], [0, 100, 100]), ([-4, 1, 160], [1, 1, 160]), ([100, 0, 160], [0, 0, 160]),
                                      ([160, 160, 160], None), ([0, 0, 160], None), ([-9, -3, 70], [70, 70, 70]), ([1 << 30, 0, 0], [0, 0, 0])])
def test_ends_that_cannot_be(cu, valid, path, pkg):
    """Reported; the rows of the sequences whose ends can be are written as ever, no others."""
    s = base.Setup([100, 60], [200, 200], 4, 2, 64, 16, 1, garbage=False)
    s.path = path
    s.cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
    whole = torch.full((170, 4, 64), 9.0, device="cuda", dtype=torch.float16)
    out = whole[5:165]
    _, lse = s.call(pkg, out=out, return_lse=True)
    if valid is None:
        assert pkg.check_status() == 0
    else:
        with pytest.raises(pkg.IntfaError, match="outside its table"):
            pkg.check_status()
        s.cu = torch.tensor(valid, dtype=torch.int32, device="cuda")
    want, wlse, A, B = O.attention(s.q8, s.qs, s.kc, s.vc, s.ks, s.vs, s.table, s.lens, s.cu, True, s.scale)
    rows = ~torch.isnan(wlse[:, 0])
    assert int(rows.sum()) == int(s.cu[2] - s.cu[0])
    assert ((out.double() - want).abs() <= s.tolerance(want, A, B))[rows].all()
    assert ((lse.double() - wlse).abs() <= 2.0 ** -16 * 64)[rows].all()
    assert (out[~rows] == 9).all() and (whole[:5] == 9).all() and (whole[165:] == 9).all()


@pytest.mark.parametrize("block", [1, 8])
@pytest.mark.parametrize("what", ["rotation", "ends"])
def test_append_writes_only_what_it_may(what, block, pkg):
    """Positions past the rotary table, and ends past the rows: with a scale a token the tokens that are inside are written, with longer blocks none of the
    run that is not inside as a whole; every other slot and scale stays."""
    s = append.Setup([3, 2], [3, 18], 2, 2, 64, 16, block)
    cs = pkg.rotary_table(64, 64, device="cuda")
    before = [x.clone() for x in s.state()]
    if what == "rotation":
        cs = pkg.rotary_table(1, 64, device="cuda")
        s.lens[1] = 0
        inside = [(0, 0)]                                    # (sequence, position): the first token
    else:
        s.cu[2], s.lens[1] = 9, 8                            # positions 2 .. 7, of which rows 3 and 4 are here
        inside = [(0, 0), (0, 1), (0, 2), (1, 2), (1, 3)]
    if block > 1:
        inside = [x for x in inside if what == "ends" and x[0] == 0]
    s.run(pkg, cs)
    with pytest.raises(pkg.IntfaError, match="outside its table"):
        pkg.check_status()
    slots = torch.zeros(s.kc.shape[0], 16, dtype=torch.bool, device="cuda")
    for seq, pos in inside:
        slots[int(s.table[seq, pos // 16]), pos % 16] = True
    scales = slots.view(-1, 16 // block, block).any(-1)
    for now, was, there in zip(s.state(), before, (slots, slots, scales, scales)):
        same = (now == was).flatten(3).all(-1) if now.dim() == 4 else now == was
        assert same.transpose(1, 2)[~there].all()
        assert not same.transpose(1, 2)[there].any() if now.dim() == 4 else True
    rows = [0, 1, 2, 3, 4] if what == "ends" else [0]
    x = s.v[rows[:len(inside)]].float()
    if block == 1:
        for i, (seq, pos) in enumerate(inside):
            page = int(s.table[seq, pos // 16])
            scale = O.scale_of(O.absmax(x[i]))
            assert torch.equal(s.vs[page, :, pos % 16], scale) and torch.equal(s.vc[page, :, pos % 16], O.codes(x[i], scale[:, None]))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("news,lens", [([1] * 15 + [300], [40 + 31 * i for i in range(15)] + [420]),          # a step: single tokens and a chunk of a prompt
                                       ([500] + [1] * 3, [500, 900, 1, 33]), ([1, 2, 0, 1, 700, 1, 5, 1], [800, 2, 5, 0, 900, 64, 5, 129]),
                                       ([1] * 60 + [90, 1], [1 + 17 * i for i in range(60)] + [90, 1])])
def test_single_tokens_and_chunks_in_one_call(news, lens, D, pkg):
    """Whatever path the rule on sizes takes: it is one of the two, bit for bit, and right."""
    s = base.Setup(news, lens, 8, 2, D, 16, 4, seed=D)
    for causal in (True, False):
        o = s.check(pkg, causal)
        both = []
        for s.path in (1, 2):
            both.append(s.check(pkg, causal))
        s.path = 0
        assert any(torch.equal(o, x) for x in both)


@pytest.mark.parametrize("D,rot", [(64, 20), (64, 2), (128, 100), (256, 66), (64, 32), (16, 6)])
@pytest.mark.parametrize("dtype,words", [(torch.float16, torch.int16), (torch.bfloat16, torch.int16), (torch.float32, torch.int32)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_channels_that_are_not_rotated_keep_their_bits(D, rot, dtype, words, interleaved, pkg):
    """Whatever they hold, and wherever the rotated part ends."""
    g = torch.Generator(device="cuda").manual_seed(rot)
    top = torch.iinfo(words)
    x = torch.randint(top.min, top.max, (5, 3, D), device="cuda", generator=g, dtype=words)          # NaN of all kinds among them
    x[..., rot::3] = top.max - x[..., rot::3].abs() % 100                                              # (these are)
    x = x.view(dtype)
    x[..., :rot] = torch.randn(5, 3, rot, device="cuda", generator=g).to(dtype)
    cs, pos = pkg.rotary_table(50, rot, device="cuda"), torch.arange(45, 50, device="cuda")
    y = pkg.rotary(x, None, cs, pos, interleaved=interleaved)
    assert torch.equal(y[..., rot:].view(words), x[..., rot:].view(words))
    assert torch.equal(y[..., :rot], O.turn(x[..., :rot].float(), cs[pos][:, None], interleaved).to(dtype))
