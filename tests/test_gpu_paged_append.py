"""GPU: tokens appended to a paged int8 cache, against the same operations one by one (codes and scales bit for bit) and in 64 bits."""
import pytest
import torch

from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu


class Setup:
    """A cache of `pages` pages with the sequences' pages in no order; what no token was ever written to is garbage."""

    def __init__(self, news, lens, H, Hkv, D, page, block, dtype=torch.float16, seed=0, layout="heads", extra=5):
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        S, T = len(news), sum(news)
        self.page, self.block, self.Hkv, self.D, self.news = page, block, Hkv, D, news
        width = max(1, max(-(-n // page) for n in lens)) + 1
        used = sum(-(-n // page) for n in lens)
        pages = used + extra
        perm = torch.randperm(pages, generator=g, device="cuda").int()
        self.table = torch.full((S, width), -7, dtype=torch.int32, device="cuda")             # (not read)
        at = 0
        for s, n in enumerate(lens):
            c = -(-n // page)
            self.table[s, :c] = perm[at:at + c]
            at += c
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.cu = torch.tensor([0] + news, device="cuda").cumsum(0).int()
        rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
        self.q, self.k, self.v = rand(T, H, D).to(dtype) if H else None, rand(T, Hkv, D).to(dtype), rand(T, Hkv, D).to(dtype)
        def cache():
            x = torch.randint(-127, 128, (pages, Hkv, page, D), device="cuda", generator=g, dtype=torch.int8)
            if layout == "tokens":           # [pages, page, heads, D] in memory
                x = x.transpose(1, 2).contiguous().transpose(1, 2)
            if layout == "both":             # K and V of a page behind each other
                x = torch.stack([x, x], 1)[:, 0]
            return x
        self.kc, self.vc = cache(), cache()
        self.ks, self.vs = (torch.rand(pages, Hkv, page // block, device="cuda", generator=g) * 0.03 for _ in range(2))

    def state(self):
        return self.kc, self.vc, self.ks, self.vs

    def run(self, pkg, cs=None, interleaved=False, cu="cu"):
        return pkg.append_int8_paged(self.k, self.v, self.kc, self.vc, self.ks, self.vs, self.table, self.lens, self.cu if cu == "cu" else None, q=self.q,
                                     table=cs, interleaved=interleaved)

    def check(self, pkg, cs=None, interleaved=False, cu="cu"):
        want = O.append(self.k, self.v, self.kc, self.vc, self.ks, self.vs, self.table, self.lens, self.cu, self.q, cs, interleaved)
        got = self.run(pkg, cs, interleaved, cu)
        for a, b in zip(self.state(), want[:4]):
            assert torch.equal(a.view(torch.int32) if a.dtype == torch.float32 else a, b.view(torch.int32) if b.dtype == torch.float32 else b)
        if self.q is not None:
            assert torch.equal(got[0], want[4]) and torch.equal(got[1], want[5])
        else:
            assert got is None
        pkg.check_status()


@pytest.mark.parametrize("block", [1, 2, 8, 16, "page"])
@pytest.mark.parametrize("page", [8, 16, 64, 256])
@pytest.mark.parametrize("D,H,Hkv", [(64, 6, 3), (128, 8, 1), (256, 0, 2)])
def test_ragged_batches(page, block, D, H, Hkv, pkg):
    block = page if block == "page" else min(block, page)
    s = Setup([1, 5, 64, 0, 33, 17, 200], [1, 70, 64, 9, 300, 17, 203], H, Hkv, D, page, block, seed=page + D)
    s.check(pkg, pkg.rotary_table(400, D, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rot,interleaved", [(None, False), (128, False), (128, True), (64, False), (20, True), (20, False), (2, False)])
@pytest.mark.parametrize("block", [1, 4])
def test_rotations(dtype, rot, interleaved, block, pkg):
    s = Setup([3, 1, 9], [30, 1, 1009], 5, 2, 128, 32, block, dtype)
    s.check(pkg, None if rot is None else pkg.rotary_table(2000, rot, device="cuda"), interleaved)


@pytest.mark.parametrize("layout", ["tokens", "both"])
@pytest.mark.parametrize("block", [1, 16])
def test_layouts(layout, block, pkg):
    s = Setup([20, 1, 7], [33, 16, 7], 4, 4, 64, 16, block, layout=layout)
    s.check(pkg, pkg.rotary_table(64, 64, device="cuda"))


@pytest.mark.parametrize("block", [1, 32])
def test_one_token_a_sequence(block, pkg):
    s = Setup([1] * 70, [1 + 37 * i % 500 for i in range(70)], 32, 8, 128, 32, block)
    s.check(pkg, pkg.rotary_table(512, 128, device="cuda"), cu=None)


def test_many_sequences(pkg):
    """More than a warp finds its place among in one step, with empty ones between."""
    news = [(7 * i) % 4 for i in range(1500)]
    for block in (1, 8):
        Setup(news, [n + (5 * i) % 40 for i, n in enumerate(news)], 2, 1, 64, 8, block, seed=block).check(pkg)


def test_token_by_token_is_the_same_cache(pkg):
    """One scale a token: however the tokens are handed over.  A scale for a block: it grows with them and the codes stay within the
    roundings of its steps."""
    cs = pkg.rotary_table(100, 64, device="cuda")
    for block in (1, 16):
        whole = Setup([37], [37], 2, 2, 64, 16, block)
        steps = Setup([37], [37], 2, 2, 64, 16, block)
        whole.run(pkg, cs)
        for i in range(37):
            pkg.append_int8_paged(steps.k[i:i + 1], steps.v[i:i + 1], *steps.state(), steps.table, torch.full((1,), i + 1, dtype=torch.int32, device="cuda"),
                                  table=cs)
        for a, b in zip(whole.state()[2:], steps.state()[2:]):
            pages = whole.table[0, :3].long()
            assert torch.equal(a[pages][:, :, :1], b[pages][:, :, :1]) and torch.equal(a[pages[:2]], b[pages[:2]])
        for a, b in zip(whole.state()[:2], steps.state()[:2]):
            pages = whole.table[0, :2].long()
            if block == 1:
                assert torch.equal(a, b)
            else:       # each of at most 15 growths of the scale rounds once, by half a code at most, and the last scale is the largest
                assert ((a[pages].int() - b[pages].int()).abs() <= 8).all()
    pkg.check_status()


def test_values_in_64_bits(pkg):
    """A code stands for its value to half a step: |y - code * scale| <= scale / 2, with what fp32 adds (|y| <= 127.001 scale)."""
    s = Setup([100], [100], 4, 2, 128, 64, 64)
    cs = pkg.rotary_table(128, 128, device="cuda")
    q8, qs = s.run(pkg, cs)
    y = O.turn(s.k.double(), cs[:100, None].double(), False).transpose(0, 1)
    got = O.gather(s.kc, s.ks, s.table[0], 100)
    step = s.ks.double()[s.table[0, :2].long()].repeat_interleave(64, -1).transpose(0, 1).flatten(1)[:, :100, None]
    assert ((y - got).abs() <= step * (0.5 + 2.0 ** -15)).all()
    yq = O.turn(s.q.double(), cs[:100, None].double(), False)
    assert ((yq - q8.double() * qs.double()[..., None]).abs() <= qs.double()[..., None] * (0.5 + 2.0 ** -15)).all()
    assert (q8.abs().amax(-1) == 127).all()


@pytest.mark.parametrize("block", [1, 8])
def test_zeros_infinities_nan_and_small_numbers(block, pkg):
    s = Setup([16, 3], [20, 3], 2, 2, 64, 16, block, torch.bfloat16)
    s.k[0] = 0                              # scale 0, codes 0
    s.v[3, 0, 5] = float("inf")             # scale infinite: codes 0
    s.v[5, 1, 60] = float("nan")
    s.k[7, 0] *= 1e-38                      # a subnormal scale
    s.k[9, 1] *= 1e-36
    s.q[1, 1, 0] = float("-inf")
    s.check(pkg)
    # what is poisoned stays within its block of tokens and head
    bad = ~torch.isfinite(s.vs[s.table[0, :2].long()])
    assert int(bad.sum()) == 2
    again = Setup([2], [22], 0, 2, 64, 16, block, torch.bfloat16, seed=3)
    again.kc, again.vc, again.ks, again.vs, again.table = s.kc, s.vc, s.ks, s.vs, s.table[:1]
    again.check(pkg)


@pytest.mark.parametrize("block", [1, 4])
def test_what_is_left_as_it_was(block, pkg):
    """Rows behind the last sequence, sequences that are padding, and all slots that no new token goes to."""
    s = Setup([4, 2, 3], [9, 2, 3], 2, 2, 64, 8, block)
    s.lens[1] = 0                           # padding: its table row may be anything
    s.table[1] = 1 << 30
    pad = lambda x: torch.cat([x, torch.full_like(x[:5], 3.0)])
    s.q, s.k, s.v = pad(s.q), pad(s.k), pad(s.v)
    before = [x.clone() for x in s.state()]
    want = O.append(s.k, s.v, *before, s.table, s.lens, s.cu, s.q)
    got = s.run(pkg)
    assert all(torch.equal(a, b) for a, b in zip(s.state(), want))
    rows = [0, 1, 2, 3, 6, 7, 8]
    assert torch.equal(got[0][rows], want[4][rows]) and torch.equal(got[1][rows], want[5][rows])
    assert pkg.check_status() == 0


@pytest.mark.parametrize("block", [1, 8])
@pytest.mark.parametrize("what", ["page", "negative", "width", "length", "rotation", "ends"])
def test_bad_indices_write_nothing(what, block, pkg):
    s = Setup([3, 2], [3, 18], 2, 2, 64, 16, block)
    cs = pkg.rotary_table(64, 64, device="cuda")
    if what == "page":
        s.table[0, 0] = s.kc.shape[0]
    elif what == "negative":
        s.table[0, 0] = -1
    elif what == "width":
        s.lens[0] = s.table.shape[1] * 16 + 3
    elif what == "length":
        s.lens[0] = -5
    elif what == "rotation":
        cs = pkg.rotary_table(1, 64, device="cuda")
        s.lens[1] = 0
    pages = s.table[1, :2].long()
    if what == "ends":                      # more rows than there are: those of the second sequence are not all here
        s.cu[2] = 9
        s.lens[1] = 8
    before = [x.clone() for x in s.state()]
    pkg.check_status()
    s.run(pkg, cs)
    with pytest.raises(pkg.IntfaError, match="outside its table"):
        pkg.check_status()
    if what in ("page", "negative", "width", "length"):
        others = [i for i in range(s.kc.shape[0]) if i not in pages.tolist()]
        assert all(torch.equal(a[others], b[others]) for a, b in zip(s.state(), before))
        assert not torch.equal(s.kc, before[0])            # the second sequence was appended


def test_ends_that_run_backwards(pkg):
    s = Setup([3, 2], [3, 18], 2, 2, 64, 16, 8)
    for cu in ([0, 3, 1], [-2, 3, 5]):
        s.cu.copy_(torch.tensor(cu))
        s.run(pkg, None)
        with pytest.raises(pkg.IntfaError, match="outside its table"):
            pkg.check_status()


def test_a_replayed_graph_appends_the_next_tokens(pkg):
    s = Setup([1, 1, 1], [40, 9, 64], 4, 2, 64, 16, 1, extra=9)
    cs = pkg.rotary_table(128, 64, device="cuda")
    s.table[s.table < 0] = 0
    start = [x.clone() for x in s.state()]
    s.lens -= 3
    lens = s.lens.clone()
    pkg.append_int8_paged(s.k, s.v, *s.state(), s.table, s.lens, table=cs)
    for a, b in zip(s.state(), start):
        a.copy_(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q8, qs = pkg.append_int8_paged(s.k, s.v, *s.state(), s.table, s.lens, q=s.q, table=cs)
        s.lens += 1
    want = start
    for i in range(3):
        s.k.normal_()
        s.q.normal_()
        out = O.append(s.k, s.v, *want, s.table, lens + i, None, s.q, cs)
        want = out[:4]
        graph.replay()
        assert torch.equal(q8, out[4]) and torch.equal(qs, out[5])
    assert all(torch.equal(a, b) for a, b in zip(s.state(), want))
    assert torch.equal(s.lens, lens + 3)
    pkg.check_status()


def test_no_tokens(pkg):
    s = Setup([0, 0], [5, 0], 2, 2, 64, 16, 4)
    before = [x.clone() for x in s.state()]
    q8, qs = s.run(pkg)
    assert q8.shape == (0, 2, 64) and qs.shape == (0, 2)
    assert all(torch.equal(a, b) for a, b in zip(s.state(), before))
