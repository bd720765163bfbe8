"""Higher derivatives through fused_rms_norm and fused_add_rms_norm: their
gradient has none, and says so, in the compiled binding and in the Python
statement that runs under graph capture."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-6


def _binding(x, res, w):
    import kernel_opt as ko
    return (ko.fused_rms_norm(x, w, EPS),) if res is None else ko.fused_add_rms_norm(x, res, w, EPS)


def _statement(x, res, w):
    from kernel_opt.norm import _FusedRmsNorm
    out = _FusedRmsNorm.apply(x, res, w, EPS)
    return (out,) if res is None else out


NORMS = pytest.mark.parametrize("norm", [_binding, _statement], ids=["binding", "statement"])


def _leaves():
    g = torch.Generator(device=DEV).manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).requires_grad_()  # noqa: E731
    return r(6, 40), r(6, 40), r(40)


@NORMS
@pytest.mark.parametrize("residual", [False, True], ids=["plain", "residual"])
@pytest.mark.parametrize("loss", [lambda y: y.sum(), lambda y: y.square().sum()],
                         ids=["constant_gradient", "varying_gradient"])
def test_second_derivatives_are_refused(norm, residual, loss):
    """Also where another path to the same leaf has one, which alone would be a
    wrong sum, and where the norm's own incoming gradient is a constant."""
    for which in (0, 2):  # x, weight
        x, res, w = _leaves()
        leaves = (x, res, w)
        y = norm(x.tanh(), res if residual else None, w)[0]
        total = loss(y) + x.pow(3).sum() + w.pow(3).sum()
        d, = torch.autograd.grad(total, leaves[which], create_graph=True)
        with pytest.raises(RuntimeError, match="no second derivative"):
            torch.autograd.grad(d.square().sum(), leaves[which], retain_graph=True)
        with pytest.raises(RuntimeError, match="no second derivative"):
            d.square().sum().backward()


@NORMS
def test_first_derivatives_under_create_graph(norm):
    x, res, w = _leaves()
    want = torch.autograd.grad(norm(x, res, w)[0].square().sum(), (x, res, w))
    got = torch.autograd.grad(norm(x, res, w)[0].square().sum(), (x, res, w), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    frozen, = torch.autograd.grad(norm(x, res.detach(), w.detach())[0].sum(), x, create_graph=True)
    assert torch.equal(frozen, torch.autograd.grad(norm(x, res, w)[0].sum(), x)[0])


@NORMS
def test_second_derivative_of_the_sum(norm):
    """h = x + residual is linear: what flows through it alone has one, 2 + 2
    of (x + residual)^2 along x and residual."""
    x, res, w = _leaves()
    h = norm(x, res, w)[1]
    dx, = torch.autograd.grad(h.square().sum(), x, create_graph=True)
    assert torch.equal(dx, 2 * h)
    ddx, ddr = torch.autograd.grad(dx.sum(), (x, res))
    assert (ddx == 2).all() and (ddr == 2).all()
