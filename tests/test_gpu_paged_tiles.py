"""GPU: attention over a paged int8 cache where sequences have many query rows (128-row tiles on the tensor cores), against 64 bits with
the tolerance of test_gpu_paged_attention.py.  One term more: the reference that w is relative to may be up to 2^8 behind the largest w,
which changes no relative rounding and makes the absolute one, 2^-25 of the largest, smaller."""
import pytest
import torch

import test_gpu_paged_attention as base

pytestmark = pytest.mark.gpu


class Setup(base.Setup):
    path = 2                              # 128-row tiles, also where the rule on sizes takes packed rows


def test_the_rule_takes_either_path(pkg):
    """Prompts on tiles, drafts and single tokens packed: what the rule gives is bit for bit what one of the two gives."""
    for news, lens, path in (([300, 500, 200], [300, 900, 201], 2), ([4, 3, 5], [400, 900, 201], 1), ([1, 1], [1, 700], 1)):
        s = Setup(news, lens, 32, 8, 128, 16, 1)
        want = s.call(pkg)
        s.path = path
        got = s.call(pkg)
        s.path = 0
        assert torch.equal(s.call(pkg), got)
        if path == 1:
            assert not torch.equal(want, got)          # (the two round differently)
    s = Setup([3], [30], 129, 1, 64, 16, 1)            # more query heads a K/V head than a tile has rows
    with pytest.raises(pkg.IntfaError, match="debug_path"):
        s.call(pkg)
    s.path = 0
    s.check(pkg)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("ratio,Hkv", [(1, 3), (4, 2), (5, 2), (8, 1), (48, 1), (128, 1)])
def test_prompts(D, causal, ratio, Hkv, pkg):
    news = [200, 1, 0, 129, 64, 300] if ratio < 48 else [9, 1, 0, 33, 5]
    Setup(news, [n + o for n, o in zip(news, [0, 5, 3, 0, 200, 77])], ratio * Hkv, Hkv, D, 16, 4, seed=ratio).check(pkg, causal, torch.bfloat16 if ratio == 5 else torch.float16)


@pytest.mark.parametrize("page,block", [(8, 1), (8, 8), (16, 2), (32, 32), (64, 1), (128, 16), (256, 1), (256, 256)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_pages(page, block, D, pkg):
    s = Setup([150, 70], [150, 427], 8, 2, D, page, block, seed=page, layout="tokens" if block == 2 else "heads")
    s.check(pkg)


@pytest.mark.parametrize("n", [33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383])
def test_lengths(n, pkg):
    for ratio, D in ((1, 64), (2, 64), (1, 128), (1, 256)):
        Setup([n, n + 1], [n, n + 130], 2 * ratio, 2, D, 32, 1, seed=n).check(pkg)


@pytest.mark.parametrize("S,n,length,H,Hkv,D", [(1, 40, 30000, 8, 1, 128), (1, 9, 5000, 8, 2, 64), (1, 256, 256, 1, 1, 128), (40, 30, 500, 8, 2, 64), (200, 33, 40, 2, 1, 128),
                                                (1, 2000, 2000, 16, 4, 128), (3, 700, 3001, 32, 8, 64), (600, 33, 33, 1, 1, 64), (2, 300, 9000, 8, 2, 256),
                                                (1, 700, 700, 6, 2, 256)])
def test_shares(S, n, length, H, Hkv, D, pkg):
    news = [max(1, n - 3 * s % 29) for s in range(S)]
    s = Setup(news, [length - 7 * i % 31 if length > n else m for i, m in enumerate(news)], H, Hkv, D, 64, 1, seed=S + n)
    a = s.check(pkg)
    assert torch.equal(a, s.call(pkg))


@pytest.mark.parametrize("spread", [3.0, 12.0, 40.0])
@pytest.mark.parametrize("block", [1, 16])
def test_value_scales_of_all_sizes(spread, block, pkg):
    """Sigma 40: factors of 1e60, held down to what fp32 and bf16 have."""
    s = Setup([100, 80], [500, 80], 8, 2, 128, 16, block, v_spread=spread)
    s.vs.clamp_(1e-30, 1e30)
    s.check(pkg, out_dtype=torch.bfloat16)


def test_scales_of_zero(pkg):
    s = Setup([100, 80, 40], [500, 80, 41], 4, 2, 128, 16, 1, garbage=False)
    s.vs[torch.rand_like(s.vs) < 0.3] = 0
    s.vs[s.table[0, :8].long()] = 0                  # the first chunk as a whole
    s.check(pkg)
    s.vs[s.table[2, :3].long()] = 0                  # a sequence as a whole
    s.check(pkg)
    s.ks.zero_()
    s.check(pkg)
    s.vs.mul_(1e-30)
    s.check(pkg, out_dtype=torch.bfloat16)


def test_rising_and_falling_scores(pkg):
    """The largest score in the last keys, in the first, and far apart."""
    for D in (128, 256):
        rising_and_falling(D, pkg)


def rising_and_falling(D, pkg):
    s = Setup([64, 40], [1200, 900], 4, 2, D, 16, 1, garbage=False)
    order = torch.linspace(0.2, 3, 1200, device="cuda")
    for slope in (order, order.flip(0)):
        for b in range(2):
            n = int(s.lens[b])
            pos = torch.arange(n, device="cuda")
            s.ks[s.table[b, :-(-n // 16)].long()] = 0.02
            s.ks[s.table[b].long()[pos // 16], :, pos % 16] = (0.02 * slope[:n])[:, None]
        # exponents up to 127 * 127 * D * 0.025 * 0.06 / sqrt(D) * 1.4427 = 35 sqrt(D), 558 at D = 256: 4 * 558 * 2^-24 * ln 2 * 2 = 1.9e-4
        s.check(pkg, more=2.0 ** -12)
    s.scale = -0.05
    s.check(pkg, more=2.0 ** -12)
    s.scale = 1.0
    s.check(pkg, more=2.0 ** -8)                     # sqrt(D) times as much: 8939, 3.0e-3


def test_nan_reaches_its_rows_only(pkg):
    s = Setup([100, 64], [300, 64], 4, 2, 64, 16, 1)
    want, _, A, B = base.O.attention(s.q8, s.qs, s.kc, s.vc, s.ks, s.vs, s.table, s.lens, s.cu, True, s.scale)
    s.ks[s.table[0, 2].long(), 1, 3] = float("nan")               # key 35 of all rows of the first sequence
    s.vs[s.table[1, 2].long(), 0, 0] = float("nan")               # key 32: seen from row 32 on
    s.vs[s.table[1, 3].long(), 1, 15] = float("inf")              # the last key
    o = s.call(pkg)
    bad = torch.zeros(164, 4, 1, dtype=torch.bool, device="cuda")
    bad[:100, 2:] = True
    bad[132:, :2] = True
    bad[163, 2:] = True
    assert torch.equal(torch.isfinite(o).all(-1, keepdim=True), ~bad)
    # The rows that do not see them may take another way through the same arithmetic (P relative to another reference), so they are as they
    # were up to the roundings of both: each is held to the exact values by itself.
    keep = ~bad.expand_as(o)
    assert ((o.double() - want).abs() <= s.tolerance(want, A, B))[keep].all()


def test_rows_that_see_nothing(pkg):
    s = Setup([90, 50, 40], [30, 0, 300], 4, 2, 128, 16, 1)
    o, lse = s.call(pkg, return_lse=True)
    assert (o[:60] == 0).all() and (o[90:140] == 0).all() and torch.isinf(lse[:60]).all() and torch.isinf(lse[90:140]).all()
    s.check(pkg)
    s.check(pkg, causal=False)


def test_rows_behind_the_last_sequence_stay(pkg):
    s = Setup([70, 50], [70, 99], 4, 2, 64, 16, 1)
    want, T = s.call(pkg), 120
    pad = lambda x: torch.cat([x, x[:9]])
    s.q8, s.qs = pad(s.q8), pad(s.qs)
    out = torch.full((T + 9, 4, 64), 9.0, device="cuda", dtype=torch.float16)
    s.call(pkg, out=out)
    assert torch.equal(out[:T], want) and (out[T:] == 9).all()


def test_query_and_output_views(pkg):
    s = Setup([100, 41], [200, 300], 6, 2, 128, 16, 1)
    wide = torch.zeros(141, 9, 256, dtype=torch.int8, device="cuda")
    wide[:, 2:8, 128:] = s.q8
    s.q8 = wide[:, 2:8, 128:]
    base_ = torch.full((141, 6, 256), 7.0, device="cuda", dtype=torch.float16)
    o, lse = s.call(pkg, out=base_[..., :128], return_lse=True)
    assert (base_[..., 128:] == 7).all()
    s.check(pkg, got=(o, lse))
    s.q8 = s.q8[:, :1].expand(141, 6, 128)                        # one head's rows for all
    s.check(pkg)


def test_bad_indices(pkg):
    s = Setup([100, 60], [100, 200], 4, 2, 64, 16, 1)
    good = s.call(pkg)
    assert pkg.check_status() == 0
    for bad in (s.kc.shape[0], -1, 1 << 30):
        was = s.table[0, 3].clone()
        s.table[0, 3] = bad
        o = s.call(pkg)
        with pytest.raises(pkg.IntfaError, match="outside its table"):
            pkg.check_status()
        assert torch.equal(o[100:], good[100:])
        s.table[0, 3] = was
    s.table[0] = 0
    s.lens[0] = s.table.shape[1] * 16 + 1
    o = s.call(pkg)
    with pytest.raises(pkg.IntfaError, match="outside its table"):
        pkg.check_status()
    assert torch.equal(o[100:], good[100:])
    s.table[:] = 0
    for cu in ([0, 160, 100], [0, 100, 200], [-4, 1, 160], [100, 0, 160], [160, 160, 160], [0, 0, 160]):
        s.cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
        s.lens[:] = 200
        s.call(pkg)
        try:
            pkg.check_status()
        except pkg.IntfaError:
            pass


def test_two_streams_at_once_and_a_replayed_graph(pkg):
    a, b = Setup([100, 300, 8], [900, 300, 500], 8, 2, 128, 16, 1), Setup([3, 160], [1000, 200], 8, 2, 64, 16, 4, seed=5)
    wa, wb = a.call(pkg), b.call(pkg)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (sa, sb):
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(10):
        for s, x, w in ((sa, a, wa), (sb, b, wb)):
            with torch.cuda.stream(s):
                got.append((x.call(pkg), w))
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for x, w in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [a.call(pkg) for _ in range(2)]
    cu, lens = a.cu.clone(), a.lens.clone()
    for news, ls in (([100, 300, 8], [900, 300, 500]), ([1, 407, 0], [33, 407, 0]), ([200, 8, 200], [200, 8, 511])):
        a.cu[1:] = torch.tensor(news, device="cuda").cumsum(0).int()
        a.lens.copy_(torch.tensor(ls, device="cuda"))
        a.table.clamp_(max=a.kc.shape[0] - 1)
        graph.replay()
        want = a.call(pkg)
        # (bit by bit: the longer ones run into pages whose scales are NaN)
        assert all(torch.equal(o.view(torch.int16), want.view(torch.int16)) for o in outs)
    pkg.check_status()


def test_after_and_before_the_other_kernels(pkg, oracle):
    """Calls of every kind behind one another on one stream, each as it is by itself."""
    a, b = Setup([100, 300, 8], [900, 300, 500], 8, 2, 128, 16, 1), Setup([1, 1], [700, 90], 8, 2, 128, 16, 1, seed=3)
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(1, 4, 512, 128, device="cuda", generator=g).half() for _ in range(3))
    calls = [lambda: a.call(pkg), lambda: pkg.int_flash_attention(q, k, v, True, 0.09), lambda: b.call(pkg),
             lambda: pkg.int_flash_attention(q, k, v, False, 0.09, variant="half"), lambda: a.call(pkg)]
    want = []
    for f in calls:
        want.append(f())
        torch.cuda.synchronize()
    for _ in range(5):
        got = [f() for f in calls]
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    pkg.check_status()
