"""The sums behind fused_sample's log-probabilities: float64 for unfiltered and
top_p rows (also with a min_p), as the header promises, so that logp and
sample_logp are float32 roundings of numbers known to 10 digits.  On the CPU:
the check tells a float32 sum from those, and the oracle's own borders."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle.sample_oracle import sample_row

DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]
FILTERS = {"none": {}, "p": dict(top_p=0.9), "p_wide": dict(top_p=0.9999), "p_half": dict(top_p=0.5),
           "pm": dict(top_p=0.95, min_p=0.001)}


def _logits(rows, vocab, dtype, seed, scale):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * scale
    return x.to(dtype), torch.rand(rows, generator=g)


def _misses(b, n_kept, got):
    """Whether `got` is not the rounding of any number within d of b.  d: a
    weight, so a sum of them, is within 1.04e-10 of itself by the polynomial of
    2^y; the exponents' factor is cut to 42 bits, which moves a sum's logarithm
    by the mean |y| under its weights, ln(vocab) <= 18 at most, times 2^-42 and
    the token's y by |b| 2^-42 at most; up to 4096 kept weights are summed as
    whole numbers of 2^-44, of a sum of at least 1; float64 rounds below 2^-50."""
    d = 1.04e-10 + (18 + abs(b)) * 2.0 ** -42 + min(n_kept, 4096) * 2.0 ** -44 \
        + (1 + abs(b)) * 2.0 ** -50
    return not np.float32(b - d) <= got <= np.float32(b + d)


@pytest.mark.gpu
@pytest.mark.parametrize("filters", FILTERS.values(), ids=FILTERS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,vocab,scale", [(40, 50257, 1.5), (300, 3001, 3.0), (24, 152064, 1.0)])
def test_rounded_once(rows, vocab, scale, dtype, filters):
    import kernel_opt as ko
    print(f"{rows} x {vocab} {dtype} {filters}", flush=True)
    x, u = _logits(rows, vocab, dtype, rows + vocab, scale)
    for T in (1.0, 0.6):
        tok, logp, slp = (t.cpu() for t in ko.fused_sample(x.to(DEV), u.to(DEV), T, **filters))
        for i, row in enumerate(x.float().numpy()):
            t, lp, sl, kept = sample_row(row, float(u[i]), T, **filters)
            assert int(tok[i]) == t, (i, int(tok[i]), t)
            assert not _misses(lp, 0, float(logp[i])), (i, float(logp[i]), lp)
            assert not _misses(sl, kept.size, float(slp[i])), (i, float(slp[i]), sl)


def test_the_check_tells_a_float32_sum():
    """Weights of float32, added in float32 (numpy's pairwise sums, nearer than
    a kernel's would be, off by some 2^-24): results near -10 have steps of
    2^-20, so one row in 16 is then another float32, and one fails the check."""
    x, u = _logits(40, 50257, torch.float32, 40 + 50257, 1.5)
    off = 0
    for i, row in enumerate(x.numpy()):
        t, lp, _, kept = sample_row(row, float(u[i]))
        y = row - row.max()
        got = np.float32(float(y[t]) - math.log(float(np.exp(y).sum(dtype=np.float32))))
        off += _misses(lp, 0, float(got))
        exact = float(np.float32(lp))
        assert not _misses(lp, 0, exact)
    assert off >= 1


def test_oracle_borders_by_hand():
    """Powers of two, whose weights, sums and borders are exact: the token at a
    min_p's border stays (w >= min_p), and one at which top_p is reached exactly
    is the last kept."""
    x = np.array([-math.inf, 1.0, 3.0, 2.0, 0.0]) * math.log(2.0)  # weights 0 1/4 1 1/2 1/8
    w = np.exp(x - x.max())
    kept = lambda **kw: list(sample_row(x, 0.0, **kw)[3])  # noqa: E731
    assert kept(min_p=float(np.float32(0.25 * (1 - 1e-6)))) == [1, 2, 3]
    assert kept(min_p=float(np.float32(0.25 * (1 + 1e-6)))) == [2, 3]
    y = np.array([0.0, -1074.0])  # the second weight is 0 in float64, the first exactly 1
    assert list(sample_row(y, 0.5, min_p=1.0)[3]) == [0]
    flat = np.zeros(8)  # equal weights of exactly 1
    assert list(sample_row(flat, 0.5, min_p=1.0)[3]) == list(range(8))
    assert list(sample_row(flat, 0.5, top_p=0.5)[3]) == [0, 1, 2, 3]
    assert list(sample_row(flat, 0.5, top_p=0.5 + 2.0 ** -20)[3]) == [0, 1, 2, 3, 4]
    assert sample_row(flat, 0.5)[0] == 4 and sample_row(flat, 0.5 - 2.0 ** -20)[0] == 3
    assert abs(w.sum() - 1.875) < 1e-15
