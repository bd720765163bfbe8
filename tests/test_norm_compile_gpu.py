"""The norms under torch.compile: traced without a graph break, forward and
backward equal to the eager calls; the operators that break the graph still
give their eager results there."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BACKEND = "aot_eager"
EPS = 1e-6


def _leaves(shape, dtype, seed=3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)  # noqa: E731
    return r(*shape), r(*shape), r(shape[-1])


def _plain(x, res, w):
    import kernel_opt as ko
    return (ko.fused_rms_norm(x * 2, w, EPS) * 0.5,)


def _added(x, res, w):
    import kernel_opt as ko
    y, h = ko.fused_add_rms_norm(x * 2, res, w, EPS)
    return y * 0.5, h + 1


def _only_h(x, res, w):
    import kernel_opt as ko
    return (ko.fused_add_rms_norm(x * 2, res, w, EPS)[1] * 3,)


def _only_y(x, res, w):
    import kernel_opt as ko
    return (ko.fused_add_rms_norm(x, res, w, EPS)[0],)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("fn", [_plain, _added, _only_h, _only_y],
                         ids=["plain", "added", "only_h", "only_y"])
@pytest.mark.parametrize("need", [(1, 1, 1), (1, 0, 0), (0, 0, 1)], ids=["all", "x", "weight"])
def test_fullgraph(fn, dtype, need):
    data = _leaves((3, 7, 264), dtype)
    sides = []
    for compiled in (False, True):
        leaves = [t.clone().requires_grad_(bool(n)) for t, n in zip(data, need)]
        torch._dynamo.reset()
        f = torch.compile(fn, backend=BACKEND, fullgraph=True, dynamic=False) if compiled else fn
        out = f(*leaves)
        asked = [t for t in leaves if t.requires_grad]
        loss = sum(o.float().square().sum() for o in out)
        grads = torch.autograd.grad(loss, asked, allow_unused=True) if loss.requires_grad else ()
        # An input that only an unused output depends on: no gradient, or zeros.
        sides.append([*out, *(torch.zeros_like(t) if d is None else d
                              for d, t in zip(grads, asked))])
    assert len(sides[0]) == len(sides[1]) or not sides[0][0].requires_grad
    assert all(torch.equal(a, b) for a, b in zip(*sides))


def test_fullgraph_with_varying_rows():
    torch._dynamo.reset()
    f = torch.compile(_added, backend=BACKEND, fullgraph=True, dynamic=True)
    for rows in (5, 9, 300):
        data = _leaves((rows, 136), torch.bfloat16, rows)
        a, b = ([t.clone().requires_grad_() for t in data] for _ in range(2))
        got, want = f(*a), _added(*b)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        for outs, leaves in ((got, a), (want, b)):
            sum(o.float().square().sum() for o in outs).backward()
        assert all(torch.equal(p.grad, q.grad) for p, q in zip(a, b))


def test_registered_ops():
    import kernel_opt.norm  # noqa: F401  (registers them)
    x, res, w = _leaves((4, 5, 96), torch.float32)
    op = torch.ops.kernel_opt.rms_norm.default
    for r in (None, res):
        leaves = [None if t is None else t.clone().requires_grad_() for t in (x, r, w)]
        torch.library.opcheck(op, (*leaves, EPS))
    leaves = [t.clone().requires_grad_() for t in (x, res, w)]
    y, h, rstd = op(*leaves, EPS)
    assert not rstd.requires_grad
    d, = torch.autograd.grad(y.square().sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivative here either
        torch.autograd.grad(d.square().sum(), leaves[0])


def test_refusals_while_tracing():
    x, res, w = _leaves((4, 64), torch.float32)
    for bad in ((x, res[:3], w), (x, res.half(), w), (x, res, w[:63])):
        torch._dynamo.reset()
        with pytest.raises(Exception, match="must"):
            torch.compile(_added, backend=BACKEND)(*bad)


def test_operators_that_break_the_graph():
    """They run eagerly between the compiled parts, with the same results."""
    import kernel_opt as ko
    x, res, w = _leaves((12, 256), torch.bfloat16)
    head, hs = ko.quantize_fp8(_leaves((300, 256), torch.float32)[0], block_rows=128)
    u = torch.rand(12, device=DEV)
    t = torch.zeros(12, dtype=torch.int64, device=DEV)

    def tail(x, res):
        q, s, h = ko.fused_add_rms_norm_fp8(x * 2, res, w)
        logits = ko.fp8_linear(q, s, head, hs) * 1
        return (logits, h, *ko.quantize_fp8(h * 2)[1:], *ko.fused_sample(logits, u, 0.7, top_k=9),
                *ko.sample_hidden(x, w, head, hs, u, residual=res, top_p=0.8),
                *ko.score_hidden(x, w, head, hs, t, residual=res))

    torch._dynamo.reset()
    want, got = tail(x, res), torch.compile(tail, backend=BACKEND)(x, res)
    assert len(want) == len(got) and all(torch.equal(a, b) for a, b in zip(want, got))
