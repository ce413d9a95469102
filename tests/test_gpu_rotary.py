"""GPU: rotary positions against the same expression in elementary fp32 operations (bit for bit) and in 64 bits, and as a gradient."""
import pytest
import torch

from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu
EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}       # half a step


def table_rows(cs, positions, packed):
    rows = cs[positions.long()]
    return rows[:, None] if packed else rows[:, None] if rows.dim() == 4 else rows[None, None]


@pytest.mark.parametrize("D,rot", [(16, 16), (16, 8), (32, 32), (64, 64), (64, 20), (64, 2), (128, 128), (128, 64), (128, 96), (256, 256), (256, 66)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved,inverse", [(False, False), (True, False), (False, True), (True, True)])
def test_against_the_formula(D, rot, dtype, interleaved, inverse, pkg):
    g = torch.Generator(device="cuda").manual_seed(D + rot)
    B, H, Hkv, N = 2, 5, 3, 7
    q, k = (torch.randn(B, h, N, D, device="cuda", generator=g).to(dtype) for h in (H, Hkv))
    cs = pkg.rotary_table(5000, rot, device="cuda")
    pos = torch.randint(0, 5000, (B, N), device="cuda", generator=g, dtype=torch.int32)
    got = pkg.rotary(q, k, cs, pos, interleaved=interleaved, inverse=inverse)
    rows = table_rows(cs, pos, False)
    for x, y in zip((q, k), got):
        assert y.dtype == dtype and y.shape == x.shape
        assert torch.equal(y, O.turn(x.float(), rows, interleaved, inverse).to(dtype))
        want = O.turn(x.double(), rows.double(), interleaved, inverse)
        # two products of at most |x|max each and their sum, each rounded to fp32; then to the type (a step of fp16's smallest numbers too)
        tol = 4 * 2.0 ** -24 * x.abs().max().double() + EPS[dtype] * want.abs() + 2.0 ** -25
        assert ((y.double() - want).abs() <= tol).all()
    one = pkg.rotary(q, None, cs, pos, interleaved=interleaved, inverse=inverse)
    assert torch.equal(one, got[0])
    pkg.check_status()


@pytest.mark.parametrize("T,H,Hkv,D", [(1, 1, 1, 64), (1, 32, 8, 128), (3, 1, 1, 16), (37, 7, 1, 256), (1000, 2, 2, 32), (513, 40, 8, 128), (5, 300, 2, 64)])
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_packed(T, H, Hkv, D, wide, pkg):
    g = torch.Generator(device="cuda").manual_seed(T)
    q, k = (torch.randn(T, h, D, device="cuda", generator=g).half() for h in (H, Hkv))
    cs = pkg.rotary_table(40000, D, device="cuda")
    pos = torch.randint(0, 40000, (T,), device="cuda", generator=g, dtype=wide)
    for x, y in zip((q, k), pkg.rotary(q, k, cs, pos)):
        assert torch.equal(y, O.turn(x.float(), cs[pos.long()][:, None], False).half())


def test_views(pkg):
    """Heads out of one fused projection, a transposed layout, broadcast batches, rows that are not aligned."""
    g = torch.Generator(device="cuda").manual_seed(1)
    cs, pos = pkg.rotary_table(100, 64, device="cuda"), torch.arange(9, device="cuda")
    qkv = torch.randn(9, 12, 64, device="cuda", generator=g).half()
    q, k = qkv[:, :6], qkv[:, 6:8]
    rows = cs[pos][:, None]
    for x, y in zip((q, k), pkg.rotary(q, k, cs, pos)):
        assert torch.equal(y, O.turn(x.float(), rows, False).half())
    bnhd = torch.randn(2, 9, 4, 64, device="cuda", generator=g).bfloat16().transpose(1, 2)
    same = torch.randn(1, 4, 9, 64, device="cuda", generator=g).half().expand(3, 4, 9, 64)
    odd = torch.randn(2 * 4 * 9 * 64 + 1, device="cuda", generator=g)[1:].view(2, 4, 9, 64)
    gap = torch.randn(2, 4, 9, 67, device="cuda", generator=g)[..., :64]
    for x in (bnhd, same, odd, gap):
        assert torch.equal(pkg.rotary(x, None, cs, pos), O.turn(x.float(), cs[pos][None, None], False).to(x.dtype))
    table = pkg.rotary_table(100, 64, device="cuda").transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(pkg.rotary(q, None, table, pos), pkg.rotary(q, None, cs, pos))


def test_no_rows(pkg):
    cs = pkg.rotary_table(10, 64, device="cuda")
    q = torch.zeros(0, 4, 64, device="cuda").half()
    a, b = pkg.rotary(q, q[:, :2], cs, torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert a.shape == (0, 4, 64) and b.shape == (0, 2, 64)
    assert pkg.rotary(torch.zeros(2, 4, 0, 64, device="cuda"), None, cs, torch.zeros(0, dtype=torch.int32, device="cuda")).shape == (2, 4, 0, 64)


def test_channels_that_are_not_rotated_are_copied(pkg):
    """Infinities and NaN among them stay where they are."""
    for interleaved in (False, True):
        x = torch.randn(3, 2, 64, device="cuda").half()
        x[0, 0, 40], x[1, 1, 33], x[2, 0, 32] = float("inf"), float("nan"), float("-inf")
        y = pkg.rotary(x, None, pkg.rotary_table(10, 32, device="cuda"), torch.arange(3, device="cuda"), interleaved=interleaved)
        assert torch.equal(y[..., 32:].view(torch.int16), x[..., 32:].view(torch.int16)) and torch.isfinite(y[..., :32]).all()


def test_inverse_is_the_gradient(pkg):
    """Against the formula's gradient by autograd in 64 bits, and against differences."""
    g = torch.Generator(device="cuda").manual_seed(7)
    cs, pos = pkg.rotary_table(3000, 48, scaling=("by_parts", 4.0, 1000), device="cuda"), torch.tensor([0, 1, 2999, 77], device="cuda")
    for interleaved in (False, True):
        x, up = (torch.randn(2, 3, 4, 64, device="cuda", generator=g) for _ in range(2))
        leaf = x.double().requires_grad_()
        half = cs.shape[1]
        z = leaf[..., :2 * half].unflatten(-1, (half, 2)) if interleaved else leaf[..., :2 * half].unflatten(-1, (2, half)).transpose(-1, -2)
        c, s = (t.double() for t in cs[pos].unbind(-1))
        turned = torch.stack([z[..., 0] * c - z[..., 1] * s, z[..., 1] * c + z[..., 0] * s], -1)
        y = torch.cat([turned.flatten(-2) if interleaved else turned.transpose(-1, -2).flatten(-2), leaf[..., 2 * half:]], -1)
        (grad,) = torch.autograd.grad((y * up.double()).sum(), leaf)
        got = pkg.rotary(up, None, cs, pos, interleaved=interleaved, inverse=True)
        tol = 8 * 2.0 ** -24 * up.abs().max().double()          # (cos and sin up to 1.14)
        assert ((got.double() - grad).abs() <= tol).all()
        # the map is linear: a difference along one direction is exact up to roundings of values below 6
        d = torch.randn(x.shape, device="cuda", generator=g)
        f = lambda t: (pkg.rotary(t, None, cs, pos, interleaved=interleaved).double() * up.double()).sum()
        slope, want = (f(x + d) - f(x - d)) / 2, (got.double() * d.double()).sum()
        assert abs(slope - want) <= x.numel() * 16 * 2.0 ** -24 * up.abs().max()


def test_a_position_outside_the_table(pkg):
    cs = pkg.rotary_table(10, 64, device="cuda")
    x = torch.randn(4, 3, 64, device="cuda").half()
    pkg.check_status()
    for bad in (10, -1):
        y = pkg.rotary(x, None, cs, torch.tensor([1, bad, 3, 9], device="cuda"))
        assert (y[1] == 0).all() and torch.equal(y[[0, 2, 3]], pkg.rotary(x[[0, 2, 3]], None, cs, torch.tensor([1, 3, 9], device="cuda")))
        with pytest.raises(pkg.IntfaError, match="outside its table"):
            pkg.check_status()
    assert pkg.check_status() == 0


def test_on_a_side_stream_and_in_a_graph(pkg):
    cs = pkg.rotary_table(100, 128, device="cuda")
    q, k = torch.randn(20, 8, 128, device="cuda").half(), torch.randn(20, 2, 128, device="cuda").half()
    pos = torch.arange(20, device="cuda")
    want = pkg.rotary(q, k, cs, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.rotary(q, k, cs, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = pkg.rotary(q, k, cs, pos)
    pos.add_(5)
    graph.replay()
    want = pkg.rotary(q, k, cs, pos)
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    pkg.check_status()
