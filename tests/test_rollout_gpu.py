"""The tail of a decode step as it is used: norm, 8-bit head and sampler, and
the scoring of what was sampled; the pieces against their composition, and the
composition against a plain one in 64 bits."""
from __future__ import annotations

import threading

import numpy as np
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from oracle import fp8_oracle, norm_oracle
from oracle.sample_oracle import sample_row

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ko():
    import kernel_opt
    return kernel_opt


def _model(tokens, dim, vocab, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    w = (3.0 * r(vocab, dim) * dim ** -0.5).to(torch.bfloat16)
    return (r(tokens, dim).to(torch.bfloat16), r(tokens, dim).to(torch.bfloat16),
            (1 + 0.1 * r(dim)).to(torch.bfloat16), w, torch.rand(tokens, generator=g, device=DEV))


@pytest.mark.parametrize("tokens", [1, 7, 200])
@pytest.mark.parametrize("with_residual", [False, True])
def test_sample_and_score(tokens, with_residual):
    ko = _ko()
    dim, vocab = 528, 9001
    x, res, nw, w, u = _model(tokens, dim, vocab, tokens)
    head, head_scale = ko.quantize_fp8(w, block_rows=128)
    kw = dict(residual=res) if with_residual else {}
    tok, logp, slp = ko.sample_hidden(x, nw, head, head_scale, u, 0.8, top_k=50, top_p=0.95, **kw)
    # The pieces.
    if with_residual:
        q, s, _ = ko.fused_add_rms_norm_fp8(x, res, nw)
    else:
        q, s = ko.fused_rms_norm_fp8(x, nw)
    logits = ko.fp8_linear(q, s, head, head_scale)
    for a, b in zip((tok, logp, slp), ko.fused_sample(logits, u, 0.8, top_k=50, top_p=0.95)):
        assert torch.equal(a, b)
    # The sampler on these logits, in 64 bits.
    xs = logits.float().cpu().numpy()
    for i in range(0, tokens, 9):
        t, lp, sl, _ = sample_row(xs[i], float(u[i]), 0.8, 50, 0.95)
        # 1.04e-10: a weight's bound, as test_sample_gpu derives it.
        assert int(tok[i]) == t and abs(float(slp[i]) - sl) <= 2.0 ** -24 * abs(sl) + 1.04e-10
    # The logits against a head that was never quantized: the codes of both
    # sides are off by at most 2^-4 of themselves (2^-10 448ths of a block's
    # largest for small ones), so a sum of `dim` products of sizes a b is off by
    # at most sum a b (2 2^-4 + 2^-8) and those, before a bf16 rounding.
    h = (x.double() + res.double()).to(torch.bfloat16) if with_residual else x
    y, _ = norm_oracle.forward(h.double().cpu().numpy(), nw.double().cpu().numpy(), 1e-6)
    wd = w.double().cpu().numpy()
    ey = np.abs(y) * 2.0 ** -4 + fp8_oracle.spread(fp8_oracle.block_amax(y, 1), 1, *y.shape) / 448 * 2.0 ** -9
    ew = np.abs(wd) * 2.0 ** -4 + fp8_oracle.spread(fp8_oracle.block_amax(wd, 128), 128, *wd.shape) / 448 * 2.0 ** -9
    ref = y @ wd.T
    bound = np.abs(y) @ ew.T + ey @ np.abs(wd).T + ey @ ew.T
    bound = 1.01 * bound + np.abs(ref) * 2.0 ** -8
    assert (np.abs(xs - ref) <= bound).all()
    # Scoring: the forward of the same logits, whatever the chunks.
    want = ko.fused_logprob_entropy_forward(logits, tok, 0.8)
    for chunk in (None, 1 if tokens < 10 else 64, 1000):
        got = ko.score_hidden(x, nw, head, head_scale, tok, 0.8, chunk_tokens=chunk, **kw)
        if chunk in (None, 1000):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            continue
        # A chunk's products may come from another kernel: bf16 logits a step
        # (2^-7 of themselves) apart move a logit and the logsumexp by as much.
        step = 2.0 ** -7 * float(logits.abs().max()) / 0.8
        assert (got[0] - want[0]).abs().max() <= 2 * step + 4e-5
        assert (got[2] - want[2]).abs().max() <= step + 4e-5
    assert (got[0] - logp).abs().max() <= 4e-5


def test_leading_shapes_and_no_tokens():
    ko = _ko()
    x, res, nw, w, u = _model(12, 256, 1000, 3)
    head, hs = ko.quantize_fp8(w, block_rows=128)
    a = ko.sample_hidden(x, nw, head, hs, u, residual=res)
    b = ko.sample_hidden(x.view(3, 4, 256), nw, head, hs, u.view(3, 4), residual=res.view(3, 4, 256))
    assert all(torch.equal(p, q.reshape(-1)) and q.shape == (3, 4) for p, q in zip(a, b))
    c = ko.score_hidden(x.view(3, 4, 256), nw, head, hs, b[0], residual=res.view(3, 4, 256))
    assert all(t.shape == (3, 4) for t in c)
    e = ko.sample_hidden(x[:0], nw, head, hs, u[:0])
    assert [t.numel() for t in e] == [0, 0, 0]
    assert [t.numel() for t in ko.score_hidden(x[:0], nw, head, hs, e[0])] == [0, 0, 0]


def test_norm_in_front_of_the_fused_grpo_step():
    """The training norm feeding fused_linear_grpo_step: gradients of the
    norm's inputs against the same step fed with a leaf, taken through the
    norm's formula in 64 bits."""
    ko = _ko()
    B, S, D, V = 2, 8, 128, 1000
    g = torch.Generator(device=DEV).manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    x, res = (r(B, S, D).requires_grad_() for _ in range(2))
    nw = (1 + 0.1 * r(D)).requires_grad_()
    w = (r(V, D) * D ** -0.5).requires_grad_()
    t = torch.randint(0, V, (B, S), generator=g, device=DEV)
    old, adv = torch.full((B, S), -7.0, device=DEV), r(B)
    y, h = ko.fused_add_rms_norm(x, res, nw)
    loss, _, _ = ko.fused_linear_grpo_step(y, w, t, old, adv)
    loss.backward()
    leaf = y.detach().requires_grad_()
    loss2, _, _ = ko.fused_linear_grpo_step(leaf, w.detach().requires_grad_(), t, old, adv)
    loss2.backward()
    dx, dw, size, dw_size = norm_oracle.backward(
        h.detach().double().cpu().numpy().reshape(-1, D), nw.detach().double().cpu().numpy(), 1e-6,
        leaf.grad.double().cpu().numpy().reshape(-1, D))
    tol = 200 * 2.0 ** -24  # the norm's roundings, as test_norm_gpu.py counts them
    assert torch.equal(x.grad, res.grad)
    assert (np.abs(x.grad.double().cpu().numpy().reshape(-1, D) - dx) <= tol * size).all()
    assert (np.abs(nw.grad.double().cpu().numpy() - dw) <= tol * dw_size).all()


def _tail(x, res, nw, head, head_scale, u):
    ko = _ko()
    y, h = ko.fused_add_rms_norm(x, res, nw)
    logits = ko.fp8_linear(*ko.fused_rms_norm_fp8(h, nw), head, head_scale)
    return (y, h, logits, *ko.fused_sample(logits, u, 0.9, top_p=0.9),
            *ko.sample_hidden(x, nw, head, head_scale, u, residual=res, top_k=20))


def test_threads_with_streams_of_their_own():
    """Four threads, a stream each, calling at once: the bits of one alone."""
    x, res, nw, w, u = _model(40, 512, 3001, 5)
    head, head_scale = _ko().quantize_fp8(w, block_rows=128)
    want = _tail(x, res, nw, head, head_scale, u)
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got[i] = _tail(x, res, nw, head, head_scale, u)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_inference_mode_autocast_and_checkpoint():
    x, res, nw, w, u = _model(30, 272, 900, 6)
    head, head_scale = _ko().quantize_fp8(w, block_rows=128)
    want = _tail(x, res, nw, head, head_scale, u)
    with torch.inference_mode():
        assert all(torch.equal(a, b)
                   for a, b in zip(_tail(x, res, nw, head, head_scale, u), want))
    with torch.autocast("cuda", dtype=torch.float16):
        assert all(torch.equal(a, b)
                   for a, b in zip(_tail(x, res, nw, head, head_scale, u), want))
    leaf = x.float().requires_grad_()
    weight = nw.float().requires_grad_()
    grads = []
    for again in (False, True):
        f = lambda t: _ko().fused_rms_norm(t, weight)  # noqa: E731
        y = checkpoint(f, leaf, use_reentrant=False) if again else f(leaf)
        grads.append(torch.autograd.grad(y.square().sum(), (leaf, weight)))
    assert all(torch.equal(a, b) for a, b in zip(*grads))
