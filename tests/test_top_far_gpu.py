"""fused_top_logprobs over finite logits so large that the offset of a row's sums,
max log2(e) / T, is rounded by more than an exponent: masks with a finite fill, tiny
temperatures; against the float64 oracle with the bounds of test_top_gpu."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import top_oracle
from test_top_gpu import U, _check_row, _sum_error, np64

pytestmark = pytest.mark.gpu
DEV = "cuda"
# A row in registers, rows of a workgroup, a row in pieces.
SHAPES = [(2, 700), (300, 9001), (1, 140001)]


def _run(x, t, k, T):
    import kernel_opt
    print(f"far {tuple(x.shape)} {x.dtype} {float(x.min())} T={T}", flush=True)
    return [o.cpu().numpy() for o in kernel_opt.fused_top_logprobs(x.to(DEV), t.to(DEV), k, T)]


@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("T", [1.46, 1.5, 2.0, 2.5, 2.9])
def test_rows_of_the_lowest_value_at_a_temperature(T, rows, vocab):
    """The offset does not overflow here, and its rounding is of any sign."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.full((rows, vocab), torch.finfo(torch.float32).min)
    t = torch.randint(0, vocab, (rows,), generator=g)
    out = _run(x, t, 20, T)
    for i in range(min(rows, 3)):
        _check_row([o[i] for o in out], np64(x[i]), int(t[i]), 20, T)


FILLS = [(torch.float32, f) for f in (-1e9, -1e10, -1e11, -1e12, -1e20, -1e30)] \
    + [(torch.bfloat16, f) for f in (-1e9, -1e10, -1e12, -1e20, -1e30)] \
    + [(torch.bfloat16, torch.finfo(torch.bfloat16).min), (torch.float16, -65504.0)]


@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("dtype,fill", FILLS)
def test_finite_fills(dtype, fill, rows, vocab):
    """Rows masked with it in part (any logits, all but some, the first ones) and
    wholly: those are uniform."""
    g = torch.Generator().manual_seed(vocab)
    full = torch.randn(rows, vocab, generator=g).to(dtype)
    for T in (1.0, 1.7):
        for keep in (0, 1, 19, vocab // 2, -200):
            at = torch.randperm(vocab, generator=g)[:keep] if keep >= 0 \
                else torch.arange(vocab + keep, vocab)
            x = torch.full_like(full, fill)
            x[:, at] = full[:, at]
            t = torch.randint(0, vocab, (rows,), generator=g)
            out = _run(x, t, 20, T)
            for i in range(min(rows, 3)):
                _check_uniform_or_row([o[i] for o in out], np64(x[i]), int(t[i]), 20, T, keep)


def _check_uniform_or_row(got, x, target, k, T, keep):
    """Below 2^31 the offset's rounding, up to 64, stays an exponent of z and t
    until the end: ln z and t / z then carry 64 ln 2 times a sum's error, and ln z is
    rounded where it lies, by at most 2^-18 and as much in the logarithm."""
    if keep != 0 or abs(x[0] / T) * 1.4427 >= 2.0 ** 31:
        _check_row(got, x, target, k, T)
        return
    lp, ent, lse, rank, ids, top = got
    want = top_oracle.forward_row(x, target, k, T)
    err, _ = _sum_error(x, float(np.float32(T)))
    off = 2 * 64 * np.log(2) * (err + 8 * U) + 2.0 ** -17
    assert rank == want[3] and (ids == want[4]).all()
    assert abs(lp - want[0]) <= off and abs(ent - want[1]) <= off
    assert abs(lse - want[2]) <= off + 4 * U * abs(want[2])
    assert (np.abs(top - want[5]) <= off).all()


@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_tiny_temperatures_and_large_logits(rows, vocab):
    """Weights of all but the largest logits vanish; equal largest ones share."""
    g = torch.Generator().manual_seed(vocab)
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn(rows, vocab, generator=g).to(dtype)
        t = torch.randint(0, vocab, (rows,), generator=g)
        x[:, vocab // 3], x[:, vocab // 2] = 17.0, 30.0
        x[:, -1] = 30.0
        t[0] = vocab - 1
        for scale, T in ((1.0, 1e-9), (1.0, 1e-30), (2.0 ** 70, 1.0), (2.0 ** 122, 3.0),
                         (-(2.0 ** 60), 1.0)):
            y = x * scale
            out = _run(y, t, 20, T)
            for i in range(min(rows, 3)):
                _check_row([o[i] for o in out], np64(y[i]), int(t[i]), 20, T)


def test_maxima_around_the_border():
    """Offsets just below and above the value where sums change their offset: every
    pair of neighbours as the row's two largest, in two threads' parts."""
    border = 2.0 ** 31 / 1.4426950408889634
    near = [float(np.float32(border) + 128.0 * n) for n in range(-4, 5)]
    x = torch.full((2 * len(near) ** 2, 5000), -float("inf"))
    t = torch.zeros(len(x), dtype=torch.int64)
    for i, a in enumerate(near):
        for j, b in enumerate(near):
            n = i * len(near) + j
            x[n, 7], x[n, 4900] = a, b
            x[len(near) ** 2 + n, 7], x[len(near) ** 2 + n, 4900] = -a, -b
            t[n] = 4900
    out = _run(x, t, 2, 1.0)
    for i in range(len(x)):
        got, row = [o[i] for o in out], np64(x[i])
        want = top_oracle.forward_row(row, int(t[i]), 2)
        assert got[3] == want[3] and (got[4] == want[4]).all()
        # One weight of 1, or two: ln z is 0 or ln 2, behind exponents up to 64.
        for a, b in ((got[0], want[0]), (got[1], want[1]), *zip(got[5], want[5])):
            if np.isfinite(b):
                assert abs(a - b) <= 2.0 ** -17 + 4 * U * abs(b)
            else:
                assert a == b
        assert abs(got[2] - want[2]) <= 4 * U * abs(want[2])


def test_extreme_rows():
    """Logits around 10^30, rows of one large value of either sign, one logit far
    above the others."""
    g = torch.Generator().manual_seed(5)
    for vocab in (1000, 9001, 140001):
        x = torch.randn(4, vocab, generator=g) * 2.0
        x[0] *= 1e30
        x[1] = 3e38
        x[2] = -3e38
        x[2, 17] = -1e38
        x[3] = 10.0 ** (torch.rand(vocab, generator=g) * 43 - 5)
        x[3] *= torch.where(torch.rand(vocab, generator=g) < 0.5, -1.0, 1.0)
        t = torch.tensor([5, 6, 17, vocab - 1])
        for k in (4, 64):
            out = _run(x, t, k, 1.0)
            for i in range(4):
                _check_row([o[i] for o in out], np64(x[i]), int(t[i]), k, 1.0)
