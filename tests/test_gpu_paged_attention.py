"""GPU: attention over a paged int8 cache against 64 bits.

Tolerance, for a row with n keys, A = sum p |v| / sum p (per channel) and B = the largest p max|v| / sum p:
  w = p v_scale is rounded to fp16 relative to the row's largest w: 2^-11 of each w, or 2^-25 of the largest where that is more; a
      value is at most max|v|, so    2^-11 A + n 2^-25 B * 127/64  (v8 may be 127/64 times what the largest code stands for
      when codes of the largest w are at least 64)
  p in fp32: exponents up to 64 in magnitude, their rounding and that of the scores (a few of 2^-24 of each) and of exp2 (2^-22):   2^-16 A
  sums in fp32, 16 keys a step of the matrix product, and the same for the sum of p:   (n/8 + 64) 2^-24 A
  the output's type: half a step of o, or of its smallest numbers (2^-25)
"""
import pytest
import torch

from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu
EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Setup:
    def __init__(self, news, lens, H, Hkv, D, page, block, seed=0, layout="heads", v_spread=0.0, garbage=True, one=False):
        g = torch.Generator(device="cuda").manual_seed(seed)
        S, T = len(news), sum(news)
        rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
        counts = [-(-n // page) for n in lens]
        pages = sum(counts) + 5
        perm = torch.randperm(pages, generator=g, device="cuda").int()
        self.table = torch.full((S, max(max(counts), 1) + 1), 1 << 30, dtype=torch.int32, device="cuda")       # entries past the last are not read
        at = 0
        for s, c in enumerate(counts):
            self.table[s, :c] = perm[at:at + c]
            at += c
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.cu = None if one else torch.tensor([0] + news, device="cuda").cumsum(0).int()
        def cache():
            x = torch.randint(-127, 128, (pages, Hkv, page, D), device="cuda", generator=g, dtype=torch.int8)
            return x.transpose(1, 2).contiguous().transpose(1, 2) if layout == "tokens" else x
        self.kc, self.vc = cache(), cache()
        self.ks = torch.rand(pages, Hkv, page // block, device="cuda", generator=g) * 0.02 + 0.01
        self.vs = (torch.rand(pages, Hkv, page // block, device="cuda", generator=g) + 0.5) * torch.exp(v_spread * rand(pages, Hkv, page // block)) * 0.01
        if layout == "tokens":
            self.ks, self.vs = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (self.ks, self.vs))
        if garbage:                       # scales of blocks that hold no token
            used = torch.zeros(pages, page // block, dtype=torch.bool, device="cuda")
            for s, n in enumerate(lens):
                for i in range(0, n, block):
                    used[int(self.table[s, i // page]), i % page // block] = True
            for x, bad in ((self.ks, float("nan")), (self.vs, float("inf"))):
                x.copy_(torch.where(used[:, None], x, torch.full_like(x, bad)))
        self.q8 = torch.randint(-127, 128, (T, H, D), device="cuda", generator=g, dtype=torch.int8)
        self.qs = torch.rand(T, H, device="cuda", generator=g) * 0.02 + 0.005
        self.scale = D ** -0.5

    path = 0                              # (debug_path: the rule on sizes)

    def call(self, pkg, causal=True, **kw):
        return pkg.attention_int8_paged(*self.args(causal), debug_path=self.path, **kw)

    def args(self, causal=True):
        return (self.q8, self.kc, self.vc, self.qs, self.ks, self.vs, self.table, self.lens, self.cu, causal, self.scale)

    def tolerance(self, want, A, B, out_dtype=torch.float16, more=0.0, least=2.0 ** -25):
        n = int(self.lens.max())
        return (2.0 ** -11 + 2.0 ** -16 + more + (n / 8 + 64) * 2.0 ** -24) * A + n * 2.0 ** -25 * 2 * B[..., None] + EPS[out_dtype] * want.abs() + least

    def check(self, pkg, causal=True, out_dtype=torch.float16, got=None, more=0.0):
        o, lse = self.call(pkg, causal, out_dtype=out_dtype, return_lse=True) if got is None else got
        want, wlse, A, B = O.attention(self.q8, self.qs, self.kc, self.vc, self.ks, self.vs, self.table, self.lens, self.cu, causal, self.scale)
        tol = self.tolerance(want, A, B, out_dtype, more)
        assert o.dtype == out_dtype
        off = (o.double() - want).abs()
        assert (off <= tol).all(), (float((off / tol).max()), torch.nonzero(~(off <= tol))[:5].tolist())
        none = wlse == -float("inf")
        assert torch.equal(none, lse == -float("inf")) and (o[none] == 0).all()
        assert ((lse.double() - wlse)[~none].abs() <= 2.0 ** -16 * 64 + more).all()
        pkg.check_status()
        return o


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page,block", [(8, 1), (8, 8), (16, 4), (32, 1), (64, 64), (256, 1), (128, 16)])
@pytest.mark.parametrize("ratio", [1, 4, 9])
def test_decode(D, page, block, ratio, pkg):
    lens = [1, 31, 32, 33, 0, 7, 64, 100, 1000, 257, 96, 511]
    s = Setup([1] * len(lens), lens, 2 * ratio, 2, D, page, block, seed=page + ratio, one=True)
    s.check(pkg)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("ratio,news", [(1, [2, 1, 5, 0, 3, 8]), (4, [1, 2, 3, 0, 7, 40]), (3, [17, 100, 1, 0, 64, 33])])
@pytest.mark.parametrize("out_dtype", [torch.float16, torch.bfloat16])
def test_several_rows(D, causal, ratio, news, out_dtype, pkg):
    lens = [n + old for n, old in zip(news, [0, 1, 300, 50, 29, 0])]
    s = Setup(news, lens, 2 * ratio, 2, D, 16, 4, seed=D + ratio)
    s.path = 1
    s.check(pkg, causal, out_dtype)


@pytest.mark.parametrize("S,n,Hkv,ratio,D", [(1, 5000, 1, 1, 128), (1, 40000, 1, 8, 64), (1, 20001, 8, 4, 128), (2, 9999, 1, 16, 256), (1, 120, 1, 2, 128),
                                             (600, 40, 1, 1, 64), (300, 333, 2, 4, 128), (5, 2048, 16, 1, 64), (1, 1, 1, 1, 128)])
@pytest.mark.parametrize("one", [True, False])
def test_shares(S, n, Hkv, ratio, D, one, pkg):
    """Units cut into many parts, a few, none; many units to a share.  One row a sequence by itself, or because cu_seqlens says so."""
    lens = [max(1, n - 37 * s % n) for s in range(S)]
    s = Setup([1] * S, lens, Hkv * ratio, Hkv, D, 32, 8, one=one, seed=S)
    s.path = 1
    a = s.check(pkg)
    assert torch.equal(a, s.call(pkg))           # repeats itself


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("S,Hkv,ratio", [(1, 1, 1), (1, 8, 4), (2, 8, 1), (1, 2, 16), (1, 2, 40), (3, 3, 7), (1, 17, 2), (1, 16, 9), (5, 3, 2)])
def test_few_units(S, Hkv, ratio, D, pkg):
    """One row a sequence, up to 16 (sequence, K/V head, tile) units and a few more: lengths from none to more chunks than there are warps."""
    for n in (0, 1, 33, 64, 300, 2000, 9000):
        s = Setup([1] * S, [max(0, n - 31 * i) for i in range(S)], Hkv * ratio, Hkv, D, 16, 1, one=True, seed=n + S)
        o = s.check(pkg)
        assert torch.equal(o, s.call(pkg))


@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_layouts(layout, D, pkg):
    Setup([1, 3, 9], [77, 300, 9], 8, 4, D, 16, 4, layout=layout).check(pkg)


def test_query_and_output_views(pkg):
    s = Setup([1, 4], [200, 30], 6, 2, 128, 16, 1)
    wide = torch.zeros(5, 9, 256, dtype=torch.int8, device="cuda")
    wide[:, 2:8, 128:] = s.q8
    s.q8 = wide[:, 2:8, 128:]
    s.qs = s.qs.t().contiguous().t()
    base = torch.full((5, 6, 256), 7.0, device="cuda", dtype=torch.bfloat16)
    out = base[..., :128]
    o, lse = s.call(pkg, out=out, return_lse=True)
    assert o.data_ptr() == out.data_ptr() and (base[..., 128:] == 7).all()
    s.check(pkg, got=(o, lse), out_dtype=torch.bfloat16)


@pytest.mark.parametrize("spread", [3.0, 12.0])
@pytest.mark.parametrize("block", [1, 16])
def test_value_scales_of_all_sizes(spread, block, pkg):
    """exp(+-12 sigma): factors of 1e20 between the scales of one sequence, among them the largest on tokens that hardly count."""
    s = Setup([1, 1, 3], [500, 63, 200], 8, 2, 128, 16, block, v_spread=spread)
    s.check(pkg, out_dtype=torch.bfloat16)


def test_small_values(pkg):
    """Scales near fp16's smallest numbers and far below: the products are relative to the row's largest."""
    s = Setup([1, 1], [300, 40], 4, 2, 128, 16, 1, garbage=False)
    s.vs.mul_(1e-30)
    s.check(pkg, out_dtype=torch.bfloat16)
    o = s.call(pkg, out_dtype=torch.bfloat16)
    assert (o.float().abs() > 1e-32).float().mean() > 0.9
    s.vs.zero_()
    s.check(pkg)
    s.ks.zero_()                          # all scores equal
    s.check(pkg)


@pytest.mark.parametrize("path", [1, 2])
def test_value_scales_below_the_normal_numbers(path, pkg):
    """2^-146 .. 2^-122, as single ones and next to larger ones: the outputs are bf16 numbers.  No absolute term but half a step of its smallest."""
    s = Setup([3, 70], [200, 90], 4, 2, 128, 16, 1, garbage=False)
    s.path = path
    g = torch.Generator(device="cuda").manual_seed(3)
    exponents = torch.rand(s.vs.shape, device="cuda", generator=g).double() * 24 - 146
    small = torch.exp2(exponents).float()
    for vs in (small, torch.full_like(small, 2.0 ** -130), torch.where(torch.rand(s.vs.shape, device="cuda", generator=g) < 0.5, small, s.vs)):
        s.vs = vs
        o = s.call(pkg, out_dtype=torch.bfloat16)
        want, _, A, B = O.attention(*s.args()[:1], s.qs, s.kc, s.vc, s.ks, s.vs, s.table, s.lens, s.cu, True, s.scale)
        tol = s.tolerance(want, A, B, torch.bfloat16, least=2.0 ** -134)
        assert ((o.double() - want).abs() <= tol).all()
    pkg.check_status()


@pytest.mark.parametrize("path", [1, 2])
def test_sequences_that_share_pages(path, pkg):
    """A common prefix: the pages of one sequence in the tables of others."""
    s = Setup([4, 40, 1], [200, 200, 70], 8, 2, 128, 16, 4, garbage=False)
    s.path = path
    s.table[1, :9] = s.table[0, :9]
    s.table[2, :4] = s.table[0, :4]
    s.check(pkg)


@pytest.mark.parametrize("path", [1, 2])
def test_padding(path, pkg):
    """Rows of sequences without tokens may hold anything."""
    s = Setup([1, 1, 1, 1], [40, 0, 0, 7], 4, 2, 64, 16, 1, one=True)
    s.path = path
    s.table[1:3] = -1
    want = s.call(pkg)
    s.qs[1], s.qs[2] = float("nan"), float("inf")
    o, lse = s.call(pkg, return_lse=True)
    assert torch.equal(o, want) and (o[1:3] == 0).all() and (lse[1:3] == -float("inf")).all()
    assert pkg.check_status() == 0


def test_strides_of_dimensions_of_one(pkg):
    """What a dimension of size one gives as its stride has no meaning."""
    odd = lambda x, i: x.as_strided(x.shape, [7 if j == i else st for j, st in enumerate(x.stride())], x.storage_offset())
    s = Setup([1], [20], 1, 1, 64, 32, 1, one=True, garbage=False)
    want = s.call(pkg)
    page = int(s.table[0, 0])
    s.kc, s.vc, s.ks, s.vs = (odd(x[page:page + 1].contiguous(), 0) for x in (s.kc, s.vc, s.ks, s.vs))
    s.table[0, 0] = 0
    out = odd(odd(torch.empty_like(want), 0), 1)
    s.q8, s.qs = odd(odd(s.q8, 0), 1), odd(odd(s.qs, 0), 1)
    for path in (1, 2):
        s.path = path
        s.call(pkg, out=out)
        assert (out.float() - want.float()).abs().max() < 2e-3 * want.float().abs().max()
    k = torch.randn(1, 1, 64, device="cuda").half()
    ready, torn = [x.clone() for x in (s.kc, s.vc, s.ks, s.vs)], [s.kc, s.vc, s.ks, s.vs]
    a = pkg.append_int8_paged(k, k, *ready, s.table, s.lens, q=k)
    b = pkg.append_int8_paged(odd(odd(k, 0), 1), odd(k, 1), *torn, s.table, s.lens, q=odd(k, 0))
    assert all(torch.equal(x, y) for x, y in zip([*ready, *a], [*torn, *b]))
    cs = pkg.rotary_table(30, 64, device="cuda")
    assert torch.equal(pkg.rotary(odd(odd(k, 0), 1), odd(k, 1), cs, s.lens)[0], pkg.rotary(k, None, cs, s.lens))
    pkg.check_status()


def test_sharp_and_negative_scores(pkg):
    s = Setup([1, 2], [700, 90], 4, 2, 128, 16, 1)
    for scale in (-0.03, 0.0):
        s.scale = scale
        s.check(pkg)
    s.scale = 1.0
    # Scores up to 127 * 127 * 128 * 0.025 * 0.03 = 1549, exponents up to 2234: one key takes nearly all.  The exponent is a product rounded three
    # times and a difference, 4 * 2234 * 2^-24 in all, so p is off by ln 2 times that, 3.7e-4, and p / sum p by twice as much: below 2^-10.
    s.check(pkg, more=2.0 ** -10)


def test_nan_reaches_its_rows_only(pkg):
    s = Setup([1, 1, 2], [100, 64, 33], 4, 2, 64, 16, 1)
    clean = s.call(pkg)
    s.ks[s.table[0, 2].long(), 1, 3] = float("nan")
    s.vs[s.table[2, 2].long(), 0, 0] = float("nan")       # the last token: seen by the last row alone
    o = s.call(pkg)
    bad = torch.zeros(4, 4, 1, dtype=torch.bool, device="cuda")
    bad[0, 2:] = True
    bad[3, :2] = True
    assert torch.equal(torch.isnan(o), bad.expand_as(o))
    assert torch.equal(o[~bad.expand_as(o)], clean[~bad.expand_as(o)])


def test_rows_that_see_nothing(pkg):
    """Causal rows ahead of their sequence's first token, and sequences without tokens."""
    s = Setup([5, 2, 1], [3, 0, 40], 4, 2, 128, 16, 1)
    o, lse = s.call(pkg, return_lse=True)
    assert (o[:2] == 0).all() and (o[5:7] == 0).all() and torch.isinf(lse[:2]).all() and torch.isinf(lse[5:7]).all()
    s.check(pkg)
    s.check(pkg, causal=False)


@pytest.mark.parametrize("news", [[1, 1, 1], [3, 20, 9]])
def test_rows_behind_the_last_sequence_stay(news, pkg):
    s = Setup(news, [50, 60, 70], 4, 2, 64, 16, 1)
    want = s.call(pkg)
    T = sum(news)
    pad = lambda x: torch.cat([x, x[:2]])
    s.q8, s.qs = pad(s.q8), pad(s.qs)
    out = torch.full((T + 2, 4, 64), 9.0, device="cuda", dtype=torch.float16)
    s.call(pkg, out=out)
    assert torch.equal(out[:T], want) and (out[T:] == 9).all()
    s.cu[0] = 1                           # rows ahead of the first sequence, too
    out[:] = 9
    s.call(pkg, out=out)
    assert (out[0] == 9).all() and torch.equal(out[news[0]:T], want[news[0]:]) and (out[T:] == 9).all()
    assert pkg.check_status() == 0


def test_bad_indices(pkg):
    s = Setup([1, 1], [100, 40], 4, 2, 64, 16, 1)
    good = s.call(pkg)
    assert pkg.check_status() == 0
    for bad in (s.kc.shape[0], -1, 1 << 30):
        was = s.table[0, 3].clone()
        s.table[0, 3] = bad
        o = s.call(pkg)
        with pytest.raises(pkg.IntfaError, match="outside its table"):
            pkg.check_status()
        assert torch.equal(o[1], good[1])
        s.table[0, 3] = was
    s.lens[0] = s.table.shape[1] * 16 + 1
    s.table[0] = 0
    o = s.call(pkg)
    with pytest.raises(pkg.IntfaError, match="outside its table"):
        pkg.check_status()
    assert torch.equal(o[1], good[1])
    s.lens[0] = -3                        # no tokens
    assert (s.call(pkg)[0] == 0).all()
    with pytest.raises(pkg.IntfaError, match="outside its table"):
        pkg.check_status()
    # ends that run backwards or past the rows: nothing is read or written outside
    s.lens[:] = 20
    for path in (1, 2):
        s.path = path
        for cu in ([0, 2, 1], [0, 1, 9], [-4, 1, 2], [1, 0, 2]):
            s.cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
            s.call(pkg)
            with pytest.raises(pkg.IntfaError, match="outside its table"):
                pkg.check_status()
        s.cu = torch.tensor([2, 2, 2], dtype=torch.int32, device="cuda")
        s.call(pkg)
        assert pkg.check_status() == 0


def test_no_rows(pkg):
    s = Setup([0, 0], [5, 0], 4, 2, 64, 16, 1)
    o, lse = s.call(pkg, return_lse=True)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_two_streams_at_once_and_a_replayed_graph(pkg):
    a, b = Setup([1] * 4, [900, 33, 500, 8], 8, 2, 128, 16, 1, one=True), Setup([3, 60], [1000, 200], 8, 2, 128, 16, 4, seed=5)
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
    lens = a.lens.clone()
    for new in ([900, 33, 500, 8], [1, 20, 499, 0], [640, 33, 0, 8]):      # other lengths, other shares
        a.lens.copy_(torch.tensor(new, device="cuda"))
        graph.replay()
        want = a.call(pkg)
        assert all(torch.equal(o, want) for o in outs)
    a.lens.copy_(lens)
    graph.replay()
    assert all(torch.equal(o, wa) for o in outs)
    pkg.check_status()


def test_pages_past_32_bits(pkg):
    """A cache whose last page begins more than 2^32 bytes in."""
    D, page, Hkv = 128, 64, 4
    pages = (1 << 32) // (D * page * Hkv) + 10
    s = Setup([1], [150], 8, Hkv, D, page, 1)
    small_k, small_v, small_t = s.kc, s.vc, s.table.clone()
    ks, vs = s.ks, s.vs
    want = s.call(pkg)
    s.kc, s.vc = (torch.zeros(pages, Hkv, page, D, dtype=torch.int8, device="cuda") for _ in range(2))
    s.ks, s.vs = (torch.ones(pages, Hkv, page, device="cuda") for _ in range(2))
    for i in range(3):
        to, frm = pages - 1 - i, int(small_t[0, i])
        s.kc[to], s.vc[to], s.ks[to], s.vs[to] = small_k[frm], small_v[frm], ks[frm], vs[frm]
        s.table[0, i] = to
    assert torch.equal(s.call(pkg), want)
    k = torch.randn(1, Hkv, D, device="cuda").half()
    before = s.kc[:5].clone()
    pkg.append_int8_paged(k, k, s.kc, s.vc, s.ks, s.vs, s.table, s.lens)
    to = pages - 3
    scale = O.scale_of(O.absmax(k.float()))
    assert torch.equal(s.kc[to, :, 149 % page], O.codes(k.float(), scale[..., None])[0]) and torch.equal(s.ks[to, :, 149 % page], scale[0])
    assert torch.equal(s.kc[:5], before)
    pkg.check_status()


def test_prompts_and_steps_together(pkg):
    """As a program uses them: two prompts rotated, appended and attended to; then a step of each at a time, in one captured graph."""
    g = torch.Generator(device="cuda").manual_seed(2)
    H, Hkv, D, page = 8, 2, 128, 16
    cs = pkg.rotary_table(128, D, device="cuda")
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4).flip(1).contiguous()
    kc, vc = (torch.zeros(8, Hkv, page, D, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(8, Hkv, page, device="cuda") for _ in range(2))
    rand = lambda n, h: torch.randn(n, h, D, device="cuda", generator=g).half()
    prompts = [30, 7]
    xs = {n: rand(sum(prompts) + 2 * 5, h) for n, h in (("q", H), ("k", Hkv), ("v", Hkv))}
    history = [{n: [] for n in xs} for _ in prompts]

    def expect(lens, rows):
        """Float attention on everything so far: the last rows of each sequence."""
        out = []
        for s, n in enumerate(lens):
            k, v, q = (torch.cat(history[s][x]).double() for x in ("k", "v", "q"))
            pos = torch.arange(n, device="cuda")
            k, q = (O.turn(t, cs[pos].double()[:, None], False) for t in (k, q))
            x = torch.einsum("qhd,khd->hqk", q[-rows[s]:], k.repeat_interleave(H // Hkv, 1)) * D ** -0.5
            x = x.masked_fill(pos[None] > pos[-rows[s]:, None], -float("inf"))
            out.append(torch.einsum("hqk,khd->qhd", x.softmax(-1), v.repeat_interleave(H // Hkv, 1)))
        return torch.cat(out)

    def close(o, want):
        # int8 q, k and v: each value off by up to half of 1/127 of its row's largest (about 3 sigma here): 1.2 % of a sigma, so
        # scores by 0.012 * sqrt(2) sigma and outputs by 0.012 times sqrt(sum p^2) <= 1 and 1.7 % of |v| ~ 3; 6 sigma of both
        return float((o.double() - want).abs().max()) < 6 * (0.012 + 0.017 * 3 / 3)

    lens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 30, 37], dtype=torch.int32, device="cuda")
    step = lambda part, cu: pkg.attention_int8_paged(*(lambda qq: (qq[0], kc, vc, qq[1]))(pkg.append_int8_paged(
        part["k"], part["v"], kc, vc, ks, vs, table, lens, cu, q=part["q"], table=cs)), ks, vs, table, lens, cu, True, D ** -0.5)
    part = {n: x[:37] for n, x in xs.items()}
    o = step(part, cu)
    for s, (a, b) in enumerate(((0, 30), (30, 37))):
        for n in xs:
            history[s][n].append(xs[n][a:b])
    assert close(o, expect(prompts, prompts))
    static = {n: xs[n][37:39].clone() for n in xs}
    keep = [x.clone() for x in (kc, vc, ks, vs)]
    lens += 1
    step(static, None)                                                     # (warm-up ahead of the capture)
    for a, b in zip((kc, vc, ks, vs), keep):
        a.copy_(b)
    lens -= 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens += 1
        out = step(static, None)
    for i in range(5):
        for n in xs:
            static[n].copy_(xs[n][37 + 2 * i:39 + 2 * i])
            for s in range(2):
                history[s][n].append(xs[n][37 + 2 * i + s:38 + 2 * i + s])
        graph.replay()
        assert close(out, expect([30 + i + 1, 7 + i + 1], [1, 1]))
    pkg.check_status()
