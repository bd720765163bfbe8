"""The norms around a block, log-probabilities with alternatives and the 8-bit
product's epilogue under torch.compile, in threads, and on other streams."""
from __future__ import annotations

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ko():
    import kernel_opt
    return kernel_opt


def _inputs(seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    x, res, gate = r(3, 4, 256), r(3, 4, 256), r(3, 1, 256)
    w, post = 1 + 0.1 * r(256), 1 + 0.1 * r(256)
    t = torch.randint(0, 300, (3, 4), generator=g, device=DEV)
    return x, res, gate, w, post, t, _ko().quantize_fp8(r(300, 256), block_rows=128), r(300)


def _run(x, res, gate, w, post, t, head, bias):
    ko = _ko()
    y, h = ko.fused_block_norm(x * 2, res, w, post_weight=post, gate=gate, scale=0.5,
                               checkpoint="fp8")
    q, s, h2 = ko.fused_block_norm_fp8(y.detach() * 1, h.detach(), w, scale=0.5)
    logits = ko.fp8_linear(q, s, *head, out_dtype=torch.float32, bias=bias, softcap=5.0)
    top = ko.fused_top_logprobs((y @ torch.ones(256, 50, device=DEV)) * 0.1, t % 50, 4, 0.7)
    return (y, h, h2, logits, *ko.fused_top_logprobs(logits, t, 7), *top,
            *ko.score_hidden(x, w, *head, t, bias=bias, softcap=5.0, alternatives=3))


def test_they_break_the_graph():
    """Under torch.compile they run eagerly between the compiled parts, with the
    same results and gradients."""
    args = _inputs()
    torch._dynamo.reset()
    want, got = _run(*args), torch.compile(_run, backend="aot_eager")(*args)
    assert len(want) == len(got) and all(torch.equal(a, b) for a, b in zip(want, got))
    grads = []
    for f in (_run, torch.compile(_run, backend="aot_eager")):
        x, res, gate, w, post = (a.clone().requires_grad_() for a in args[:5])
        out = f(x, res, gate, w.detach(), post, *args[5:])
        grads.append(torch.autograd.grad(out[0].square().sum() + out[11].sum() + out[16].sum(),
                                         (x, res, gate, post)))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_threads_and_streams_of_their_own():
    """Four threads, a stream each, forward and backward at once: the bits of
    one alone."""
    args = _inputs(4)

    def step():
        x, res, gate, w, post = (a.detach().clone().requires_grad_() for a in args[:5])
        y, h = _ko().fused_block_norm(x, res, w, post_weight=post, gate=gate)
        out = _ko().fused_top_logprobs(y @ torch.ones(256, 50, device=DEV), args[5] % 50, 4)
        loss = out[0].sum() + out[5].sum() + h.sum()
        return (y, h, *out, *torch.autograd.grad(loss, (x, res, gate, w, post)), *_run(*args))

    want = step()
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(3):
                got[i] = step()
        s.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
