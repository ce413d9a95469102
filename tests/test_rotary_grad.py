"""rotary where gradients are recorded: refused rather than cut from the graph in silence, and as the two halves of a torch.autograd.Function."""
import pytest
import torch


def args(**kw):
    return {**dict(q=torch.zeros(1, 2, 3, 64), k=torch.zeros(1, 1, 3, 64), table=torch.zeros(5, 32, 2), positions=torch.zeros(3, dtype=torch.int32)), **kw}


@pytest.mark.parametrize("name", ["q", "k", "table"])
def test_inputs_that_require_grad_are_refused(name, pkg):
    leaf = args()[name].clone().requires_grad_()
    for x in (leaf, leaf * 2):
        with pytest.raises(ValueError, match="autograd"):
            pkg.rotary(**args(**{name: x}))
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):       # (as far as the device)
            pkg.rotary(**args(**{name: x}))


class Turn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, pkg, q, k, table, positions):
        ctx.pkg = pkg
        ctx.save_for_backward(table, positions)
        return pkg.rotary(q, k, table, positions)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        dq, dk = ctx.pkg.rotary(dq, dk, *ctx.saved_tensors, inverse=True)
        return None, dq, dk, None, None


@pytest.mark.gpu
def test_as_an_autograd_function(pkg):
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k = (torch.randn(2, h, 9, 64, device="cuda", generator=g, requires_grad=True) for h in (5, 2))
    up = torch.randn(2, 5, 9, 64, device="cuda", generator=g)
    cs, pos = pkg.rotary_table(100, 64, device="cuda"), torch.arange(40, 49, device="cuda")
    with pytest.raises(ValueError, match="autograd"):
        pkg.rotary(q, k, cs, pos)
    a, b = Turn.apply(pkg, q, k, cs, pos)
    ((a * up).sum() + b.sum()).backward()
    with torch.no_grad():
        assert torch.equal(a, pkg.rotary(q, None, cs, pos))
        assert torch.equal(q.grad, pkg.rotary(up, None, cs, pos, inverse=True))
        assert torch.equal(k.grad, pkg.rotary(torch.ones_like(k), None, cs, pos, inverse=True))
    # the same by autograd through the formula in 64 bits; two products and their sum, each rounded to fp32
    x = q.detach().double().requires_grad_()
    c, s = (t.double() for t in cs[pos].unbind(-1))
    lo, hi = x[..., :32], x[..., 32:]
    (torch.cat([lo * c - hi * s, hi * c + lo * s], -1) * up.double()).sum().backward()
    assert ((q.grad.double() - x.grad).abs() <= 4 * 2.0 ** -24 * up.abs().max().double()).all()
    pkg.check_status()
