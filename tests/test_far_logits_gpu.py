"""Finite logits so large that the offset of a row's sums, RN(max log2(e)), is
rounded by more than an exponent: masks with a finite fill, uniform rows of it.
Every forward that keeps an online state, against the float64 oracle."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from klp_testutil import FWD_TOL
from test_chunk_gpu import run_chunked
from test_grpo_step_gpu import run_step
from test_shard_gpu import run_sharded

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
NAMES = ("logp", "entropy", "lse")


def _forwards(x, t, T):
    """{path: (logp, entropy, lse)} of [N, V] logits, V a multiple of 8."""
    import kernel_opt
    N, V = x.shape
    xd, td = x.to(DEV), t.to(DEV)
    out = {"forward": kernel_opt.fused_logprob_entropy_forward(xd, td, T),
           "shards": run_sharded(xd, td, 3, T)[0]}
    widths = [V // 3 // 8 * 8, V // 2 // 8 * 8]
    plan = [(0, widths[0]), (widths[0], widths[1]), (sum(widths), V - sum(widths))]
    out["chunks"] = run_chunked(xd, td, plan, T)[0]
    old = torch.zeros(1, N)
    step = run_step(x.view(1, N, V), t.view(1, N), old, torch.ones(1), torch.ones(1, N), None,
                    "bnpo", 0.0, T)
    out["step"] = [o.view(N) for o in step[:3]]
    return out


def _check(name, got, want, x, T):
    """The forward's tolerance; lse and what is subtracted from it rounded where
    they lie.  A maximum below 2^30 keeps its offset's rounding, up to 64, as an
    exponent until the end: ln z and t / z carry 64 ln 2 times a sum's error, and
    ln z is rounded by at most 2^-18 and as much in the logarithm."""
    tol = FWD_TOL[x.dtype]
    top = np.abs(x.double().numpy().max(1)) / (1.0 if T is None else T)
    part = np.minimum(top * 2.0 ** -24, 64.0)
    n = x.size(1) // 256 + 60
    tol = tol + 2 * part * n * U + np.minimum(top * 2.0 ** -24, 1.0) * 2.0 ** -17
    logp, ent, lse = (np.asarray(o.cpu().double()) for o in got)
    e_lp, e_ent, e_lse = want
    assert (np.abs(ent - e_ent) <= tol).all(), (name, ent[:3], e_ent[:3])
    assert (np.abs(lse - e_lse) <= tol + 3 * U * np.abs(e_lse)).all(), (name, lse[:3], e_lse[:3])
    assert (np.abs(logp - e_lp) <= tol + 3 * U * (np.abs(e_lse) + np.abs(e_lp))).all(), \
        (name, logp[:3], e_lp[:3])


FILLS = [(torch.float32, f) for f in (-1e9, -1e10, -1e11, -1e12, -1e20, -1e30)] \
    + [(torch.float32, torch.finfo(torch.float32).min)] \
    + [(torch.bfloat16, f) for f in (-1e9, -1e10, -1e12, -1e20, -1e30)] \
    + [(torch.bfloat16, torch.finfo(torch.bfloat16).min), (torch.float16, -65504.0)]


@pytest.mark.parametrize("rows,vocab", [(3, 704), (130, 9008), (1, 77824)])
@pytest.mark.parametrize("dtype,fill", FILLS)
def test_finite_fills(dtype, fill, rows, vocab, oracle):
    """Rows masked with it in part (any logits, all but some, the first ones) and
    wholly: those are uniform."""
    g = torch.Generator().manual_seed(vocab)
    full = torch.randn(rows, vocab, generator=g).to(dtype)
    for T in (None, 1.7):
        for keep in (0, 1, 19, vocab // 2, -200):
            at = torch.randperm(vocab, generator=g)[:keep] if keep >= 0 \
                else torch.arange(vocab + keep, vocab)
            x = torch.full_like(full, fill)
            x[:, at] = full[:, at]
            t = torch.randint(0, vocab, (rows,), generator=g)
            print(f"fill {fill} {dtype} {rows} x {vocab} keep={keep} T={T}", flush=True)
            want = oracle.forward(x, t.numpy(), temperature=T)
            for name, got in _forwards(x, t, T).items():
                _check(name, got, want, x, T)


@pytest.mark.parametrize("rows,vocab", [(5, 1001), (300, 5003), (2, 152061)])
def test_fills_at_the_edges_of_rows(rows, vocab, oracle):
    """Rows that begin and end between vectors, with fills in the elements that are
    read alone."""
    import kernel_opt
    g = torch.Generator().manual_seed(vocab)
    for dtype in (torch.float32, torch.bfloat16):
        for fill in (-1e10, -1e30, torch.finfo(dtype).min):
            x = torch.randn(rows, vocab, generator=g).to(dtype)
            x[:, :9] = fill
            x[:, -9:] = fill
            x[0] = fill
            x[1, 20:] = fill
            t = torch.randint(0, vocab, (rows,), generator=g)
            print(f"edges {fill} {dtype} {rows} x {vocab}", flush=True)
            got = kernel_opt.fused_logprob_entropy_forward(x.to(DEV), t.to(DEV))
            _check("edges", got, oracle.forward(x, t.numpy()), x, None)


def test_maxima_around_the_border(oracle):
    """Maxima just below and above the value where sums change their offset, in two
    threads' parts, of either sign."""
    near = [2.0 ** 30 + 64.0 * n for n in range(-4, 0)] + [2.0 ** 30 + 128.0 * n
                                                          for n in range(4)]
    n = len(near) ** 2
    x = torch.full((2 * n, 5000), -float("inf"))
    for i, a in enumerate(near):
        for j, b in enumerate(near):
            k = i * len(near) + j
            x[k, 7], x[k, 4900] = a, b
            x[n + k, 7], x[n + k, 4900] = -a, -b
    t = torch.full((2 * n,), 4900)
    want = oracle.forward(x, t.numpy())
    for name, got in _forwards(x, t, None).items():
        _check(name, got, want, x, None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_head_products(dtype, oracle):
    """Logits of a head whose rows are far for some tokens: each token picks a
    column of the weight, so that the products are the weight's values."""
    import kernel_opt
    N, K, V = 24, 64, 4099
    g = torch.Generator().manual_seed(1)
    fill = torch.finfo(dtype).min
    x = torch.randn(N, V, generator=g).to(dtype)
    x[0] = fill
    x[1, ::2] = fill
    x[2, :2000] = fill
    x[3, 100:] = fill
    if dtype == torch.bfloat16:
        x[4] = -1e10
        x[5, ::3] = -1e12
        x[6, 5:] = -1e20
        x[7] = -1e9
    weight = torch.zeros(V, K, dtype=dtype)
    weight[:, :N] = x.t()
    hidden = torch.eye(N, K, dtype=dtype)
    t = torch.randint(0, V, (N,), generator=g)
    want = oracle.forward(x, t.numpy())
    for impl in ("chunked", "mfma") if dtype == torch.bfloat16 else ("chunked",):
        got = kernel_opt.fused_linear_logprob_entropy_forward(hidden.to(DEV), weight.to(DEV),
                                                              t.to(DEV), impl=impl)
        _check(impl, got, want, x, None)
