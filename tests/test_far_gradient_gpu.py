"""Gradients of rows whose log-sum-exp lies so far out that it is the row's maximum
itself, masked as a whole with a finite fill, say: probabilities are shared by the
logits equal to it, and a gradient of 0 gives 0.  Every backward, against the
definition in float64."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_grpo_step_gpu import run_step

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24

FILLS = [(torch.float32, f) for f in (-1e9, -1e10, -1e30, torch.finfo(torch.float32).min, 1e30)] \
    + [(torch.bfloat16, f) for f in (-1e9, -1e12, -1e30, torch.finfo(torch.bfloat16).min, 3e38)]


def _rows(rows, vocab, dtype, fill, seed):
    """Rows of the fill, of it with one logit further down, with three above it."""
    g = torch.Generator().manual_seed(seed)
    x = torch.full((rows, vocab), fill).to(dtype)
    if rows > 1:
        x[1, vocab // 2] *= 0.5 if fill > 0 else 1.0
    if rows > 2 and fill < 0:
        x[2, [0, vocab // 3, vocab - 1]] *= 0.5
    t = torch.randint(0, vocab, (rows,), generator=g)
    t[-1] = 0
    return x, t


def _want(x, t, T, g_logp, g_ent, g_lse):
    """(gradient, magnitudes), float64; the logits' product with 1 / T as float32."""
    s = float(np.float32(1.0 / np.float32(1.0 if T is None else T)))
    y = (x.float() * np.float32(s)).double().numpy()
    top = y.max(1, keepdims=True)
    at = y == top
    p = at / at.sum(1, keepdims=True)
    d = p * (g_lse - g_logp)[:, None]  # where p > 0, ln p + entropy is 0
    hot = np.arange(x.size(1)) == t.numpy()[:, None]
    d = d + hot * g_logp[:, None]
    size = p * (np.abs(g_lse) + np.abs(g_logp) + 40 * np.abs(g_ent))[:, None] \
        + hot * np.abs(g_logp)[:, None]
    return s * d, s * size


def _check(d, x, t, T, g, name):
    """p = e^-entropy: the entropy's error, below 2^-15 where exponents up to 64 stood
    in the sums of some thousand terms, and the exponential's."""
    want, size = _want(x, t, T, *g)
    bound = size * 2.0 ** -14
    bound = bound + torch.finfo(x.dtype).eps / 2 * (np.abs(want) + bound) + 1e-38
    off = np.abs(d.double().cpu().numpy() - want)
    assert (off <= bound).all(), (name, float(off.max()), int(off.argmax()))


@pytest.mark.parametrize("rows,vocab", [(3, 704), (130, 9008), (3, 4097), (2, 152064)])
@pytest.mark.parametrize("dtype,fill", FILLS)
def test_gradients(dtype, fill, rows, vocab):
    import kernel_opt
    x, t = _rows(rows, vocab, dtype, fill, vocab)
    rng = np.random.RandomState(vocab)
    for T in (None, 1.7):
        print(f"far gradient {fill} {dtype} {rows} x {vocab} T={T}", flush=True)
        g = [rng.randn(rows).astype(np.float32).astype(np.float64) for _ in range(3)]
        gd = [torch.tensor(v, dtype=torch.float32, device=DEV) for v in g]
        leaf = x.to(DEV).requires_grad_()
        out = kernel_opt.fused_logprob_entropy(leaf, t.to(DEV), T)
        d, = torch.autograd.grad(out, leaf, gd, retain_graph=True)
        _check(d, x, t, T, g, "logprob")
        zero = torch.zeros_like(gd[0])
        d, = torch.autograd.grad(out, leaf, [zero] * 3)
        assert not d.any()
        out = kernel_opt.fused_top_logprobs(leaf, t.to(DEV), 3, T)
        d, = torch.autograd.grad(out[:3], leaf, gd, retain_graph=True)
        _check(d, x, t, T, g, "top")
        # Through the alternatives: the order's first are equal logits or the only
        # ones, and their gradients' sum goes to all.
        gt = torch.randn(rows, 3, generator=torch.Generator().manual_seed(1))
        d, = torch.autograd.grad(out[5], leaf, gt.to(DEV))
        want, size = _want(x, t, T, *[0.0 * v for v in g])
        s = float(np.float32(1.0 / np.float32(1.0 if T is None else T)))
        p, _ = _want(x, torch.full_like(t, -1), T, np.zeros(rows), np.zeros(rows), np.ones(rows))
        gt64, ids = gt.double().numpy(), out[4].cpu().numpy()
        want = -p * gt64.sum(1, keepdims=True)
        size = p * np.abs(gt64).sum(1, keepdims=True)
        for i in range(rows):
            want[i, ids[i]] += s * gt64[i]
            size[i, ids[i]] += s * np.abs(gt64[i])
        bound = size * 2.0 ** -14
        bound = bound + torch.finfo(dtype).eps / 2 * (np.abs(want) + bound) + 1e-38
        assert (np.abs(d.double().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("vocab", [704, 65536, 152064])
def test_grpo_step(vocab):
    """The step's gradient is klp_bwd's; a token without weight has none."""
    from kernel_opt import _C
    for dtype, fill in ((torch.bfloat16, torch.finfo(torch.bfloat16).min), (torch.bfloat16, -1e9),
                        (torch.float16, None), (torch.float32, -1e30)):
        if dtype == torch.float32 and vocab > 77824:
            continue
        for T in (None, 1.7):
            N = 12
            x = torch.randn(1, N, vocab, generator=torch.Generator().manual_seed(2)).to(dtype)
            if fill is not None:
                x[0, 3:9] = fill
            t = torch.arange(N).view(1, N)
            mask = torch.ones(1, N)
            mask[0, 4] = 0.0
            print(f"far step {fill} {dtype} {vocab} T={T}", flush=True)
            old = torch.zeros(1, N)
            logp, ent, lse, _, d = run_step(x, t, old, torch.ones(1), mask, None, "bnpo", 0.0, T)
            assert torch.isfinite(d).all() and not d[0, 4].any()
            if fill is None:
                continue
            # Token 3's own logit: g (1 - p), all others -g p, with p = 1 / vocab.
            s = float(np.float32(1.0 / np.float32(1.0 if T is None else T)))
            row = d[0, 3].double().cpu().numpy()
            g = row[3] / (1 - 1 / vocab)
            eps = torch.finfo(dtype).eps
            rest = np.delete(row, 3)
            assert g != 0 and abs(s) > 0
            assert (np.abs(rest + g / vocab) <= (2 * eps + 2.0 ** -14) * abs(g) / vocab
                    + (6e-8 if dtype == torch.float16 else 0)).all()
            # The unfused backward from the same statistics.
            gl = torch.zeros(1, N, device=DEV)
            gl[0, 3] = float(g / s)
            e = torch.empty(x.shape, dtype=dtype, device=DEV)
            _C.bwd_launch(x.to(DEV), t.to(DEV), lse, ent, gl, None, None, e, temperature=T)
            assert (np.abs(e[0, 3].double().cpu().numpy() - row) <= 4 * eps * np.abs(row)).all()


@pytest.mark.parametrize("impl", ["chunked", "mfma"])
def test_head_products(impl):
    """The head's backward over rows of far logits: each token picks a column of the
    weight."""
    import kernel_opt
    N, K, V = 24, 64, 4096
    for fill in (torch.finfo(torch.bfloat16).min, -1e10, -1e9):
        x = torch.randn(N, V, generator=torch.Generator().manual_seed(1)).bfloat16()
        x[:3] = fill
        weight = torch.zeros(V, K, dtype=torch.bfloat16)
        weight[:, :N] = x.t()
        hidden = torch.eye(N, K, dtype=torch.bfloat16, device=DEV)
        w = weight.to(DEV).requires_grad_()
        t = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(2))
        out = kernel_opt.fused_linear_logprob_entropy(hidden, w, t.to(DEV), impl=impl)
        g = torch.zeros(N, device=DEV)
        g[0] = 1.0
        # d weight[v, n] = d logits[n, v]
        dw, = torch.autograd.grad(out[0], w, g)
        d = dw.double().cpu().numpy()[:, :N].T
        want, size = _want(x, t, None, g.double().cpu().numpy(), np.zeros(N), np.zeros(N))
        eps = torch.finfo(torch.bfloat16).eps
        bound = eps * np.abs(want) + size * 2.0 ** -14  # logits' gradient and dw rounded
        assert (np.abs(d[0] - want[0]) <= bound[0]).all(), (impl, fill)
        assert not d[1:].any()


def test_products_with_1_over_T_that_overflow():
    """Uniform rows of the lowest value at a temperature below 1: their products are
    -inf, as is lse, while fused_top_logprobs knows the distribution."""
    import kernel_opt
    for dtype in (torch.float32, torch.bfloat16):
        for rows, vocab in ((3, 704), (130, 9008), (2, 152064)):
            print(f"overflow {dtype} {rows} x {vocab}", flush=True)
            x = torch.full((rows, vocab), torch.finfo(dtype).min).to(dtype)
            t = torch.arange(rows)
            leaf = x.to(DEV).requires_grad_()
            out = kernel_opt.fused_top_logprobs(leaf, t.to(DEV), 3, 0.7)
            assert torch.isneginf(out[2]).all()
            assert (out[0].double() + np.log(vocab)).abs().max() <= 2.0 ** -16
            g = torch.ones(rows, device=DEV)
            d, = torch.autograd.grad(out[0], leaf, g)
            s = float(np.float32(1.0 / np.float32(0.7)))
            want = s * ((np.arange(vocab) == t.numpy()[:, None]) - 1 / vocab)
            eps = torch.finfo(dtype).eps / 2
            off = np.abs(d.double().cpu().numpy() - want)
            assert (off <= (2.0 ** -14 + eps) * np.abs(want)).all()
