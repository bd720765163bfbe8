"""Uses of the alternatives, the norms around a block and the product's epilogue
that a program makes now and then: inference mode, recomputed forwards, a graph
walked twice, one tensor in two places, two captured graphs in turn."""
from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ko():
    import kernel_opt
    return kernel_opt


def _block(seed=1, rows=40, dim=520, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)  # noqa: E731
    return r(rows, dim), r(rows, dim), 1 + 0.1 * r(dim), 1 + 0.1 * r(dim), r(dim)


def _same(a, b):
    assert len(a) == len(b) and all(torch.equal(p, q) for p, q in zip(a, b))


def test_inference_mode_and_recomputed_forward():
    ko = _ko()
    x, res, w, post, gate = _block()
    head, hs = ko.quantize_fp8(torch.randn(300, 520, device=DEV).narrow(1, 0, 512), block_rows=128)
    t = torch.arange(40, device=DEV)

    def run():
        y, h = ko.fused_block_norm(x, res, w, post_weight=post, gate=gate, checkpoint="fp8")
        q, s, _ = ko.fused_block_norm_fp8(x[:, :512], res[:, :512], w[:512])
        logits = ko.fp8_linear(q, s, head, hs, softcap=9.0)
        return (y, h, logits, *ko.fused_top_logprobs(logits, t, 5))

    want = run()
    with torch.inference_mode():
        _same(run(), want)
    with torch.no_grad():
        _same(run(), want)
    grads = []
    for kept in (None, "fp8"):
        for again in (False, True):
            leaves = [v.clone().requires_grad_() for v in (x, res, w, post, gate)]

            def part(x, res, w, post, gate):
                y, h = ko.fused_block_norm(x, res, w, post_weight=post, gate=gate,
                                           checkpoint=kept)
                out = ko.fused_top_logprobs(y[:, :500].contiguous(), t, 7)
                return out[0].sum() + out[1].sum() + out[5].sum() + h.float().sum()

            loss = checkpoint(part, *leaves, use_reentrant=False) if again else part(*leaves)
            grads.append(torch.autograd.grad(loss, leaves))
    _same(grads[0], grads[1])
    _same(grads[2], grads[3])


def test_a_graph_walked_twice_and_tensors_in_two_places():
    ko = _ko()
    x, res, w, post, gate = _block(2, dtype=torch.float32)
    leaves = [v.requires_grad_() for v in (x, w)]
    y, h = ko.fused_block_norm(x, x, w, post_weight=w, gate=w, scale=0.5)
    loss = y.square().sum() + h.sum()
    a = torch.autograd.grad(loss, leaves, retain_graph=True)
    _same(a, torch.autograd.grad(loss, leaves, retain_graph=True))
    parts = [x.detach().clone().requires_grad_() for _ in range(2)] + \
            [w.detach().clone().requires_grad_() for _ in range(3)]
    y, h = ko.fused_block_norm(parts[0], parts[1], parts[2], post_weight=parts[3], gate=parts[4],
                               scale=0.5)
    g = torch.autograd.grad(y.square().sum() + h.sum(), parts)
    # Sums of the same two and three float32 numbers, in one order or another.
    tol = 4 * 2.0 ** -24
    assert bool(((a[0] - (g[0] + g[1])).abs() <= tol * (g[0].abs() + g[1].abs())).all())
    assert bool(((a[1] - (g[2] + g[3] + g[4])).abs()
                 <= tol * (g[2].abs() + g[3].abs() + g[4].abs())).all())
    t = torch.arange(40, device=DEV)
    out = ko.fused_top_logprobs(x, t, 6)
    loss = out[0].sum() + out[5].square().sum()
    a = torch.autograd.grad(loss, x, retain_graph=True)
    _same(a, torch.autograd.grad(loss, x))


def test_two_captured_graphs_in_turn():
    """Rows in pieces (a workspace) and a norm's forward and backward: two graphs
    captured on one stream, replayed in turn and on two streams at once, with
    eager calls between."""
    ko = _ko()
    states = []
    s = torch.cuda.Stream()
    for i in range(2):
        x, res, w, post, gate = (v.requires_grad_() for v in _block(5 + i))
        logits = torch.randn(3, 70001, device=DEV)
        t = torch.tensor([5, 70000, 11], device=DEV)

        def call(x=x, res=res, w=w, post=post, gate=gate, logits=logits, t=t):
            y, h = ko.fused_block_norm(x, res, w, post_weight=post, gate=gate)
            grads = torch.autograd.grad((y, h), (x, res, w, post, gate), (res.detach(), x.detach()))
            return (*[v.detach() for v in (y, h)], *grads, *ko.fused_top_logprobs(logits, t, 9))

        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = call()
        states.append((g, out, call, (x, res, logits)))
    torch.cuda.synchronize()
    for rep in range(3):
        for g, out, call, ins in states:
            with torch.no_grad():
                for v in ins:
                    v.copy_(torch.randn(v.shape, device=DEV))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in states]
        for st, (g, *_rest) in zip(streams, states):
            with torch.cuda.stream(st):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for g, out, call, ins in states:
            _same(out, call())
