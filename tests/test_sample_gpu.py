"""fused_sample on the GPU against the float64 oracle (oracle/sample_oracle.py):
tokens are equal, log-probabilities within the rounding of their last step."""
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


def _logits(rows, vocab, dtype, seed, scale=1.5, peaks=20):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * scale
    if peaks:
        at = torch.randint(0, vocab, (rows, peaks), generator=g)
        x.scatter_add_(1, at, 3.0 + 5.0 * torch.rand(rows, peaks, generator=g))
    return x.to(dtype), torch.rand(rows, generator=g)


def _check(x, u, got, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Against the oracle, row by row.  logp and sample_logp: y and the two
    logarithms are float64 and the result is rounded to float32 once; a weight
    is within 1.04e-10 of itself: 2^f on |f| <= 1/512 by a quadratic whose
    error is that of interpolation at the zeros of the cubic Chebyshev
    polynomial, (ln 2 / 512)^3 / (3! 2^2) = 1.0339e-10 times at most 2^f <=
    1.0014, with 2^-44 for a weight's fixed point: 1.0354e-10, and a sum of
    weights, so its logarithm, is as near as its weights are.  With a
    filter that needs no float64 sum of the whole row, the sum behind logp is
    of float32 weights: argument within 2 2^-24 of its depth d (log2 units) and
    v_exp_f32 within 2^-23, so a share 2^-d of the sum is off by
    (2 d ln 2 + 2) 2^-24 of itself at most, and no weighted mean of that over a
    row exceeds that of equal shares: d <= log2(vocab) plus the filters' top."""
    tokens, logp, sample_logp = (t.cpu() for t in got)
    assert tokens.dtype == torch.int64 and logp.dtype == sample_logp.dtype == torch.float32
    xs = x.float().cpu().numpy()
    V = xs.shape[-1]

    def of(v, i):
        return v[i] if isinstance(v, (list, np.ndarray)) else v

    for i in range(xs.shape[0]):
        tok, lp, slp, kept = sample_row(xs[i], float(u[i]), of(temperature, i), of(top_k, i) or 0,
                                        of(top_p, i), of(min_p, i))
        assert int(tokens[i]) == tok, (i, int(tokens[i]), tok, kept.size)
        for name, a, b in (("logp", float(logp[i]), lp), ("sample_logp", float(sample_logp[i]), slp)):
            if not math.isfinite(b):
                assert a == b or (math.isnan(a) and math.isnan(b)), (name, i, a, b)
                continue
            tol = 2.0 ** -24 * abs(b) + 1.04e-10
            if name == "logp":
                tol += (2 * math.log(max(V, 2)) + 2) * 2.0 ** -24
            assert abs(a - b) <= tol, (name, i, a, b)


FILTERS = {
    "none": {}, "k": dict(top_k=50), "k1": dict(top_k=1), "k1500": dict(top_k=1500),
    "p": dict(top_p=0.9), "p0": dict(top_p=0.0), "p_wide": dict(top_p=0.9999),
    "m": dict(min_p=0.02), "m1": dict(min_p=1.0), "m_tiny": dict(min_p=1e-8),
    "kp": dict(top_k=40, top_p=0.8), "pm": dict(top_p=0.95, min_p=0.05),
    "km": dict(top_k=300, min_p=0.01), "kpm": dict(top_k=64, top_p=0.95, min_p=0.01),
}


@pytest.mark.parametrize("filters", FILTERS.values(), ids=FILTERS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,vocab", [(3, 1), (5, 7), (4, 513), (6, 5003), (3, 50257),
                                        (2, 152064)])
def test_filters(rows, vocab, dtype, filters):
    x, u = _logits(rows, vocab, dtype, rows + vocab)
    for T in (1.0, 0.6):
        got = _ko().fused_sample(x.to(DEV), u.to(DEV), T, **filters)
        _check(x, u, got, T, **filters)


@pytest.mark.parametrize("filters", FILTERS.values(), ids=FILTERS)
def test_flat_rows(filters):
    """No peaks: thousands of tokens stay in every filter (the list of
    candidates overflows), many of them equal in bf16."""
    for dtype in (torch.bfloat16, torch.float32):
        x, u = _logits(3, 20011, dtype, 77, scale=0.7, peaks=0)
        kw = dict(filters)
        got = _ko().fused_sample(x.to(DEV), u.to(DEV), 1.3, **kw)
        _check(x, u, got, 1.3, **kw)
        if "top_k" in kw:
            kw["top_k"] = 9000
            got = _ko().fused_sample(x.to(DEV), u.to(DEV), 1.3, **kw)
            _check(x, u, got, 1.3, **kw)


@pytest.mark.parametrize("filters", FILTERS.values(), ids=FILTERS)
@pytest.mark.parametrize("vocab", [1, 2, 64, 4096, 8192, 10000])
def test_equal_logits(vocab, filters):
    """Every logit equal (also the type's lowest value): ties go by index,
    running sums are exact, so every border is."""
    if "top_k" in filters and vocab > 3:
        filters = dict(filters, top_k=vocab - 3 if vocab < 5000 else 5000)
    for value, dtype in ((3.25, torch.bfloat16), (0.0, torch.float16),
                         (torch.finfo(torch.float32).min, torch.float32)):
        x = torch.full((6, vocab), value, dtype=dtype)
        u = torch.tensor([0.0, 0.25, 0.5, 0.3, 0.999, 1.0 - 2.0 ** -24])
        got = _ko().fused_sample(x.to(DEV), u.to(DEV), **filters)
        _check(x, u, got, **filters)


def test_ties_at_the_border():
    """Equal logits across a top-k or top-p border: the lowest indexes stay."""
    for dtype in DTYPES:
        x = torch.zeros(8, 12000, dtype=dtype)
        x[:, 5::7] = 2.0   # 1714 of them
        x[:, 11] = 4.0
        u = torch.linspace(0.0, 0.999, 8)
        for kw in (dict(top_k=3), dict(top_k=1000), dict(top_k=1715), dict(top_k=1716),
                   dict(top_k=6000), dict(top_p=0.25), dict(top_p=0.6), dict(top_k=1200, top_p=0.5),
                   dict(top_k=7000, top_p=0.97), dict(top_k=5000, min_p=0.2)):
            got = _ko().fused_sample(x.to(DEV), u.to(DEV), **kw)
            _check(x, u, got, **kw)


def test_masked_logits():
    """-inf logits, rows of nothing but them, +inf and NaN; minus zero; the
    lowest finite value next to ordinary ones; rows that outrange float64's
    exponents."""
    low = torch.finfo(torch.float32).min
    x = torch.randn(12, 3000, generator=torch.Generator().manual_seed(5))
    x[0] = -math.inf
    x[1, :2990] = -math.inf
    x[2, 5] = math.inf
    x[3, 7] = math.nan
    x[4, 1:] = -math.inf
    x[5, ::2] = low
    x[6] = low
    x[6, 17] = 0.0
    x[7] = 0.0
    x[7, ::2] = -0.0
    x[8] *= 3000.0
    x[9, 0] = -5000.0
    x[9, 1:] += 6000.0
    x[10, 0] = -math.inf
    x[11] = math.nan
    u = torch.rand(12, generator=torch.Generator().manual_seed(6))
    for kw in ({}, dict(top_k=5), dict(top_k=2999), dict(top_p=0.7), dict(min_p=0.1),
               dict(top_k=2000, top_p=0.9, min_p=0.001)):
        got = _ko().fused_sample(x.to(DEV), u.to(DEV), **kw)
        _check(x, u, got, **kw)


def test_uniform_borders():
    x, _ = _logits(8, 1000, torch.float32, 9)
    x[:, :3] = -math.inf
    x[:, 990:] = -math.inf
    u = torch.tensor([0.0, -0.5, 1.0, 7.0, math.nan, 1e-30, 1.0 - 2.0 ** -24, 0.5])
    for kw in ({}, dict(top_k=20), dict(top_p=0.5)):
        got = _ko().fused_sample(x.to(DEV), u.to(DEV), **kw)
        _check(x, u, got, **kw)


def test_greedy_and_extreme_temperatures():
    for dtype in DTYPES:
        x, u = _logits(5, 4001, dtype, 21)
        x[1, 100] = x[1, 50] = 20.0
        for T in (0.0, 1e-6, 1e-30, 50.0):
            got = _ko().fused_sample(x.to(DEV), u.to(DEV), T)
            _check(x, u, got, T)
            got = _ko().fused_sample(x.to(DEV), u.to(DEV), T, top_k=30, top_p=0.9, min_p=0.01)
            _check(x, u, got, T, 30, 0.9, 0.01)
    assert int(_ko().fused_sample(x.to(DEV), u.to(DEV), 0.0)[0][1]) == 50


def test_parameters_per_row():
    rows, V = 9, 6007
    x, u = _logits(rows, V, torch.bfloat16, 33)
    t = [1.0, 0.0, 0.5, 1.5, 0.9, -1.0, math.inf, math.nan, 1.0]
    k = [0, 5, -3, 40, 100000, 7, 7, 7, 2000]
    p = [0.9, 0.5, 1.0, 2.0, math.nan, 0.5, 0.5, 0.5, 0.99]
    m = [0.0, 0.1, -1.0, math.nan, 0.05, 0.0, 0.0, 0.0, 0.0]
    got = _ko().fused_sample(x.to(DEV), u.to(DEV), torch.tensor(t, device=DEV),
                             top_k=torch.tensor(k, device=DEV), top_p=torch.tensor(p, device=DEV),
                             min_p=torch.tensor(m, device=DEV))
    clean = lambda v, off: [off if isinstance(q, float) and math.isnan(q) else q for q in v]  # noqa: E731
    _check(x, u, got, t, k, clean(p, 1.0), clean(m, 0.0))
    # One parameter at a time as a tensor gives what the number gives.
    ones = torch.ones(rows, device=DEV)
    a = _ko().fused_sample(x.to(DEV), u.to(DEV), 0.7, top_k=30, top_p=0.9)
    b = _ko().fused_sample(x.to(DEV), u.to(DEV), 0.7 * ones, top_k=(30 * ones).long(),
                           top_p=(0.9 * ones).double())
    assert all(torch.equal(i, j) for i, j in zip(a, b))


def test_layouts():
    """The trainer's window, a row stride, odd offsets, leading dims, rows not
    at 16 bytes, no rows."""
    g = torch.Generator().manual_seed(8)
    for dtype in DTYPES:
        full = (torch.randn(2, 5, 1003, generator=g) * 3).to(dtype)
        for x in (full[:, :-1, :], full[:, :, 1:1000], full[:, 1:, 5:], full[0]):
            u = torch.rand(x.shape[:-1], generator=g)
            for kw in ({}, dict(top_k=20, top_p=0.9)):
                dev = full.to(DEV)
                y = dev.as_strided(x.shape, x.stride(), x.storage_offset())
                got = _ko().fused_sample(y, u.to(DEV), **kw)
                assert all(t.shape == u.shape for t in got)
                _check(x.reshape(-1, x.size(-1)), u.reshape(-1),
                       tuple(t.reshape(-1) for t in got), **kw)
    e = _ko().fused_sample(torch.empty(0, 10, device=DEV), torch.empty(0, device=DEV))
    assert [t.shape[0] for t in e] == [0, 0, 0]
    one = _ko().fused_sample(full[0, 0].to(DEV), torch.tensor(0.5, device=DEV))
    assert one[0].shape == ()


def test_logp_is_the_scored_one():
    """logp equals fused_logprob_entropy_forward's of the sampled token, at the
    same temperature, within both results' tolerances."""
    x, u = _logits(64, 32000, torch.bfloat16, 4)
    x, u = x.to(DEV), u.to(DEV)
    for T in (1.0, 0.7):
        tok, logp, slp = _ko().fused_sample(x, u, T, top_p=0.9)
        ref, _, _ = _ko().fused_logprob_entropy_forward(x, tok, T)
        assert (logp - ref).abs().max() <= 4e-5  # 2e-5 is the forward's bar
        assert (slp >= logp).all()


def test_frequencies():
    """A million draws' shares of each token against its probability: within 5
    standard deviations."""
    V, n = 50, 200000
    x = torch.randn(1, V, generator=torch.Generator().manual_seed(1))
    u = torch.rand(n, generator=torch.Generator().manual_seed(2))
    tok, _, _ = _ko().fused_sample(x.to(DEV).expand(n, V), u.to(DEV), top_k=20)
    share = torch.bincount(tok.cpu(), minlength=V).double() / n
    keep = torch.zeros(V).scatter_(0, x[0].topk(20).indices, 1.0)
    p = (x[0].double().exp() * keep)
    p /= p.sum()
    assert ((share - p).abs() <= 5 * (p * (1 - p) / n).sqrt() + 1e-12).all()


def test_repeatable_stream_and_graph():
    """The same bits on every call, on another stream, and from a captured
    graph replayed with new logits and numbers."""
    ko = _ko()
    kw = dict(top_k=100, top_p=0.9)
    x, u = _logits(40, 32000, torch.bfloat16, 12)
    x, u = x.to(DEV), u.to(DEV)
    want = ko.fused_sample(x, u, 0.8, **kw)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(want, ko.fused_sample(x, u, 0.8, **kw)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ko.fused_sample(x, u, 0.8, **kw)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = ko.fused_sample(x, u, 0.8, **kw)
        free = ko.fused_sample(x, u)
    for rep in range(3):
        nx, nu = _logits(40, 32000, torch.bfloat16, 100 + rep)
        x.copy_(nx)
        u.copy_(nu)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ko.fused_sample(x, u, 0.8, **kw)))
        assert all(torch.equal(a, b) for a, b in zip(free, ko.fused_sample(x, u)))


def test_refusals():
    ko = _ko()
    x = torch.zeros(4, 100, dtype=torch.bfloat16, device=DEV)
    u = torch.zeros(4, device=DEV)
    for bad in (u[:3], u.double(), u[None]):
        with pytest.raises(RuntimeError, match="uniform must be"):
            ko.fused_sample(x, bad)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        ko.fused_sample(x, u.cpu())
    with pytest.raises(RuntimeError, match="bf16, fp16, or fp32"):
        ko.fused_sample(x.double(), u)
    with pytest.raises(RuntimeError, match="contiguous"):
        ko.fused_sample(x[:, ::2], u)
    with pytest.raises(RuntimeError, match="vocab"):
        ko.fused_sample(x[:, :0], u)
    for t in (-1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            ko.fused_sample(x, u, t)
    with pytest.raises(ValueError, match="top_k"):
        ko.fused_sample(x, u, top_k=1.5)
    with pytest.raises(ValueError, match="top_p"):
        ko.fused_sample(x, u, top_p=1.5)
    with pytest.raises(ValueError, match="min_p"):
        ko.fused_sample(x, u, min_p=-0.5)
    for name in ("temperature", "top_k", "top_p", "min_p"):
        with pytest.raises(RuntimeError, match=f"{name} must be"):
            ko.fused_sample(x, u, **{name: u[:3]})
    with pytest.raises(RuntimeError, match="top_k must hold integers"):
        ko.fused_sample(x, u, top_k=u)


def test_logits_beyond_32_bits():
    """The last rows of more than 2^31 logits, and rows that share memory."""
    ko = _ko()
    rows, vocab = 16500, 131077
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.empty(rows, vocab, dtype=torch.bfloat16, device=DEV)
    x[:] = torch.randn(vocab, device=DEV, generator=g).to(torch.bfloat16)
    x[-3:] = torch.randn(3, vocab, device=DEV, generator=g).to(torch.bfloat16)
    u = torch.rand(rows, device=DEV, generator=g)
    for how in ({}, {"top_k": 40}, {"top_p": 0.5}, {"min_p": 0.1}):
        whole = ko.fused_sample(x, u, **how)
        last = ko.fused_sample(x[-3:], u[-3:], **how)
        assert torch.equal(whole[0][-3:], last[0])
        # 512 or 1024 threads add the weights in another order.
        for a, b in zip(whole[1:], last[1:]):
            assert ((a[-3:] - b).abs() <= 4 * 2.0 ** -24 * (1 + b.abs())).all()
    one = x[-1:].expand(9, vocab)
    a = ko.fused_sample(one, u[:9], top_p=0.9)
    b = ko.fused_sample(one.contiguous(), u[:9], top_p=0.9)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_nucleus_alone(dtype):
    """top_p without another filter: rows whose largest logit lies far above,
    or behind, those that the buckets start from, rows too spread or too far
    from zero for the buckets, masked rows, short and long nuclei."""
    V = 70001
    x, u = _logits(12, V, dtype, 61)
    f = x.float()
    f[1, 69000] += 40.0                       # a peak past the first logits of a wave's part
    f[2] += 900.0 if dtype != torch.float16 else 300.0
    f[3] = f[3] * 60.0                        # a spread of hundreds of factors of 2
    f[4, ::2] = -math.inf
    f[5, :60000] = -math.inf
    f[6] = f[6] * 0.01                        # nearly flat: a list that overflows
    f[7, 512:] = 0.0
    f[8, 100] = math.inf
    f[9, 65000] = math.nan
    f[10] = -math.inf
    f[11, 5000:9000] = 9.0                    # ties at the border
    x = f.to(dtype)
    for T, p in ((1.0, 0.9), (0.7, 0.5), (1.3, 0.99), (1.0, 0.999999), (1.0, 1e-6)):
        got = _ko().fused_sample(x.to(DEV), u.to(DEV), T, top_p=p)
        _check(x, u, got, T, 0, p)
    t = [1.0, 0.0, 0.5, 1.5, 0.9, -1.0, 1.0, 1e-3, 1.0, 1.0, 1.0, 2.0]
    p = [0.9, 0.5, 1.0, 2.0, math.nan, 0.5, 0.0, -1.0, 0.3, 0.3, 0.3, 0.7]
    got = _ko().fused_sample(x.to(DEV), u.to(DEV), torch.tensor(t, device=DEV),
                             top_p=torch.tensor(p, device=DEV))
    _check(x, u, got, t, [0] * 12, [1.0 if math.isnan(q) else q for q in p], [0.0] * 12)
    # 512 threads a row.
    many = x.repeat(25, 1).to(DEV)
    a = _ko().fused_sample(many, u.repeat(25).to(DEV), top_p=0.9)
    _check(x, u, tuple(v[-12:] for v in a), 1.0, 0, 0.9)


def test_greedy_with_a_nucleus():
    """A temperature of 0, one for all or a row's, next to a top_p."""
    x, u = _logits(6, 30011, torch.bfloat16, 91)
    x[2, 7] = x[2, 29000] = 25.0
    want = x.float().argmax(-1)
    for t in (0.0, torch.zeros(6, device=DEV)):
        for p in (None, 0.9, 1.0):
            tok, logp, slogp = _ko().fused_sample(x.to(DEV), u.to(DEV), t, top_p=p)
            assert torch.equal(tok.cpu(), want) and not slogp.any()
    _check(x, u, (tok, logp, slogp), 0.0)


@pytest.mark.parametrize("filters", [{}, {"top_p": 0.4}, {"top_k": 900}], ids=["none", "p", "k"])
def test_a_vocabulary_past_the_histograms_counts(filters):
    x, u = _logits(2, 2 ** 24 + 5, torch.bfloat16, 92)
    _check(x, u, _ko().fused_sample(x.to(DEV), u.to(DEV), **filters), **filters)
