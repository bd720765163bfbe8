"""fused_sample on the GPU: rows whose first logits are masked, at the
temperatures and offsets where weights relative to anything but the row's own
logits leave float64's exponents, against the float64 oracle
(oracle/sample_oracle.py)."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle.sample_oracle import sample_row

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]


def _ko():
    import kernel_opt
    return kernel_opt


def _check(x, u, got, temperature):
    """Tokens equal the oracle's, and both log-probabilities are the float32
    value next to a number at most d from the oracle's.  d: a weight is within
    1.04e-10 of itself by its polynomial; its exponent is y (1 + e), |e| <=
    2^-42 (16-bit logits' scale is cut to 42 bits), which moves the logarithm
    of a sum by at most ln(vocab) 2^-42 (the mean |y| under the row's own
    weights is at most ln(vocab), 18 here at most) and the token's own y by |y|
    2^-42 <= |b| 2^-42; float64's roundings are below 2^-50 of either."""
    tokens, logp, sample_logp = (t.cpu() for t in got)
    xs = x.float().cpu().numpy()
    for i in range(xs.shape[0]):
        tok, lp, slp, _ = sample_row(xs[i], float(u[i]), temperature)
        assert int(tokens[i]) == tok, (i, int(tokens[i]), tok)
        for a, b in ((float(logp[i]), lp), (float(sample_logp[i]), slp)):
            d = 1.04e-10 + (18 + abs(b)) * 2.0 ** -42 + (1 + abs(b)) * 2.0 ** -50
            assert np.float32(b - d) <= a <= np.float32(b + d), (i, a, b)


# (largest logit, temperature): quotients from -0.5 to -50000, past the ends of
# float64's exponents (-708), of the weights that count (-665) and of those
# before light tokens go (-624), around the -208 from which on they are taken
# relative to the row's largest; and above zero.
TOPS = [(-0.5, 1.0), (-2.0, 0.01), (-2.2, 0.01), (-207.0, 1.0), (-209.0, 1.0), (-7.0, 0.01), (-14.0, 0.02), (-10.0, 0.01), (-640.0, 1.0), (-6.3, 0.01),
        (-700.0, 1.0), (-5000.0, 1.0), (-50.0, 1e-3), (9.0, 0.01), (700.0, 1.0), (0.0, 0.005)]


@pytest.mark.parametrize("top,temperature", TOPS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_leading_logits_masked(dtype, top, temperature):
    """The first 63, 64, 65, 700 or all but a few logits are -inf.  The others
    lie within 500 temperatures of the largest, so that each has a weight, and
    a uniform of 0 draws the first of them."""
    print(f"masked prefix {dtype} {top} {temperature}", flush=True)
    V = 9001
    g = torch.Generator().manual_seed(17)
    x = top - min(20.0, 400.0 * temperature) * torch.rand(10, V, generator=g)
    for i, n in enumerate((63, 64, 65, 700, V - 3, V - 1, 64, 512, 4096, 8191)):
        x[i, :n] = -math.inf
    x[6, 64:] = torch.where(torch.rand(V - 64, generator=g) < 0.5, x[6, 64:], -math.inf)
    x = x.to(dtype)
    one = torch.ones(10, device=DEV)
    for u in (torch.zeros(10), torch.rand(10, generator=g), torch.full((10,), 1 - 2.0 ** -24)):
        for t, kw in ((temperature, {}), (temperature * one, {}), (temperature, dict(top_p=one)),
                      (temperature * one, dict(top_p=one, min_p=0 * one))):
            got = _ko().fused_sample(x.to(DEV), u.to(DEV), t, **kw)
            _check(x, u, got, temperature)
        # More rows than CUs: 512 threads a row.
        got = _ko().fused_sample(x.repeat(30, 1).to(DEV), u.repeat(30).to(DEV), temperature)
        _check(x, u, tuple(v[-10:] for v in got), temperature)


def test_a_constrained_decode_step():
    """The first 64 ids masked behind the 8-bit head, at a low temperature."""
    ko = _ko()
    g = torch.Generator(device=DEV).manual_seed(3)
    logits = -12.0 - 4.0 * torch.rand(33, 32000, generator=g, device=DEV)
    logits[:, :64] = -math.inf
    u = torch.rand(33, generator=g, device=DEV)
    tok, logp, slp = ko.fused_sample(logits, u, 0.01)
    assert (tok >= 64).all() and logp.isfinite().all() and torch.equal(logp, slp)
    _check(logits, u, (tok, logp, slp), 0.01)
