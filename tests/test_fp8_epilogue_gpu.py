"""fp8_linear's bias, activations, soft cap and residual against the float64
oracle (oracle/fp8_oracle.py), and the runs they are part of."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp8_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]
ACTS = [None, "relu", "silu", "gelu_tanh", "softcap"]
C = (2.0 / np.pi) ** 0.5


def _ko():
    import kernel_opt
    return kernel_opt


def _codes(q):
    return q.contiguous().view(torch.uint8).cpu().numpy()


def _matrices(m, n, k, seed, size=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    ko = _ko()
    x = torch.randn(m, k, generator=g, device=DEV) * torch.exp(
        torch.randn(m, 1, generator=g, device=DEV))
    w = torch.randn(n, k, generator=g, device=DEV) * (size * k ** -0.5)
    return *ko.quantize_fp8(x), *ko.quantize_fp8(w, block_rows=128)


def _product(xq, xs, wq, ws):
    """The product in 64 bits, and the terms its errors scale with."""
    return fp8_oracle.linear(fp8_oracle.decode(_codes(xq)), xs.cpu().numpy(),
                             fp8_oracle.decode(_codes(wq)), ws.cpu().numpy())


def _act64(z, act, cap):
    """(value, bound of |derivative|, the activation's own relative error in
    float32, per element in units of 2^-23).

    Its own error: exponentials of a rounded argument x (|x| 2^-23 with the
    constant's share) by a function good to 2 steps, one addition, one quotient
    or reciprocal and product: |x| + 8 covers them; the tanh form's argument u
    has 4 roundings of its own, 8 |u| in the exponential of 2 u and 2 |u| from
    before.  The cap's (1 - e) / (1 + e) has the error of e, 4 steps + 2 |t|,
    over 1 - e >= 2 / 65 (|t| >= 1/64): 33 (4 + 2 / 64) + 8 < 150 for the
    hardware's functions, as for float32's tanh with room."""
    with np.errstate(over="ignore"):
        if act is None:
            return z, 1.0, 0.0
        if act == "relu":
            return np.maximum(z, 0.0), 1.0, 0.0
        if act == "silu":
            return z / (1.0 + np.exp(-z)), 1.1, np.abs(z) + 8
        if act == "gelu_tanh":
            u = C * (z + 0.044715 * z ** 3)
            return z / (1.0 + np.exp(-2.0 * u)), 1.13, 10 * np.abs(u) + 8
        return cap * np.tanh(z / cap), 1.0, 150.0


def _check(out, product, k, bias=None, act=None, cap=None, residual=None):
    """The float32 product is off by A = (128 + 2 blocks) 2^-23 of its terms, and
    for 16-bit outputs by what the e4m3 instruction cuts, 7 2^-13 of the largest
    term of each 8 (tests/test_fp8_gpu.py derives both).  Adding the bias rounds
    once; the activation takes that error times its slope and adds its own;
    2^-118 stands for what lies below float32's range in an exponential's
    reciprocal, times |v| < 2^8; the residual's sum rounds once, the output once."""
    p, size, dropped = product
    acc = (128 + 2 * -(-k // 128)) * 2.0 ** -23 * size
    if out.dtype != torch.float32:
        acc = acc + 7 * 2.0 ** -13 * dropped
    z = p
    if bias is not None:
        z = p + bias.double().cpu().numpy()
        acc = acc + 2.0 ** -24 * (np.abs(z) + acc)
    value, slope, own = _act64(z, act, cap)
    err = slope * acc + own * 2.0 ** -23 * (np.abs(value) + slope * acc)
    if act is not None:
        err = err + 2.0 ** -118
    if residual is not None:
        value = value + residual.double().cpu().numpy().reshape(value.shape)
        err = err + 2.0 ** -24 * (np.abs(value) + err)
    half = torch.finfo(out.dtype).eps / 2
    tiny = 2.0 ** -25 if out.dtype == torch.float16 else 2.0 ** -134
    bound = err + half * (np.abs(value) + err) + tiny
    got = out.double().cpu().numpy().reshape(value.shape)
    over = np.abs(got - value) > bound
    assert np.isfinite(got).all() and not over.any(), (
        act, int(over.sum()), np.argwhere(over)[:3].tolist(),
        float((np.abs(got - value) / bound).max()))


def _act_args(act, cap):
    return dict(softcap=cap) if act == "softcap" else dict(activation=act)


def _extras(m, n, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    bias = 2.0 * torch.randn(n, generator=g, device=DEV)
    residual = torch.randn(m, n, generator=g, device=DEV).to(dtype)
    return bias, residual


# Both split kernels' widths and the four tiles, at sizes around their sides.
SMALL = [(1, 1, 16), (3, 129, 144), (17, 257, 1024), (64, 65, 48), (129, 255, 16), (65, 3001, 128)]
LARGE = [(20, 65600, 144), (128, 20000, 272), (130, 25000, 144), (257, 30001, 144)]


@pytest.mark.parametrize("m,n,k", SMALL)
def test_epilogues(m, n, k):
    """Every activation with and without each of bias (float32 and the output's
    type) and residual."""
    xq, xs, wq, ws = _matrices(m, n, k, m + n + k, 3.0)
    product = _product(xq, xs, wq, ws)
    for dtype in DTYPES:
        bias, residual = _extras(m, n, dtype, n)
        for act in ACTS:
            print(f"{m} x {n} x {k} {dtype} {act}", flush=True)
            cap = 5.0 if act == "softcap" else None
            for b in (None, bias, bias.to(dtype)):
                for r in (None, residual):
                    out = _ko().fp8_linear(xq, xs, wq, ws, out_dtype=dtype, bias=b, residual=r,
                                           **_act_args(act, cap))
                    assert out.shape == (m, n) and out.dtype == dtype
                    _check(out, product, k, b, act, cap, r)


@pytest.mark.parametrize("m,n,k", LARGE)
def test_epilogues_of_tiles(m, n, k):
    xq, xs, wq, ws = _matrices(m, n, k, m + n + k)
    product = _product(xq, xs, wq, ws)
    for dtype, act in zip(DTYPES, ("silu", "softcap", "gelu_tanh")):
        print(f"{m} x {n} x {k} {dtype} {act}", flush=True)
        bias, residual = _extras(m, n, dtype, n)
        cap = 30.0 if act == "softcap" else None
        out = _ko().fp8_linear(xq, xs, wq, ws, out_dtype=dtype, bias=bias, residual=residual,
                               **_act_args(act, cap))
        _check(out, product, k, bias, act, cap, residual)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "softcap"])
@pytest.mark.parametrize("size", [1e-3, 100.0])
def test_far_and_near_values(dtype, act, size):
    """Tails where the exponential leaves float32 and the neighbourhood of 0,
    caps from far above to far below the values."""
    m, n, k = 40, 200, 144
    xq, xs, wq, ws = _matrices(m, n, k, 7, size)
    product = _product(xq, xs, wq, ws)
    for cap in (0.5, 30.0, 1e4) if act == "softcap" else (None,):
        out = _ko().fp8_linear(xq, xs, wq, ws, out_dtype=dtype, **_act_args(act, cap))
        _check(out, product, k, None, act, cap)
        if cap is not None:
            assert float(out.float().abs().max()) <= cap


@pytest.mark.parametrize("m,n,k", [(5, 300, 144), (70, 8196, 144), (260, 8197, 144)])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_nothing_added_changes_nothing(m, n, k, dtype):
    """A bias of zeros and a residual of zeros give the plain call's bits; a
    residual alone the sum's, and its layout does not enter."""
    ko = _ko()
    xq, xs, wq, ws = _matrices(m, n, k, 3)
    plain = ko.fp8_linear(xq, xs, wq, ws, out_dtype=dtype)
    zeros = torch.zeros(n, device=DEV)
    assert torch.equal(plain, ko.fp8_linear(xq, xs, wq, ws, out_dtype=dtype, bias=zeros))
    assert torch.equal(plain, ko.fp8_linear(xq, xs, wq, ws, out_dtype=dtype,
                                            residual=torch.zeros_like(plain)))
    bias, residual = _extras(m, n, dtype, 5)
    want = ko.fp8_linear(xq, xs, wq, ws, out_dtype=dtype, bias=bias, activation="silu",
                         residual=residual)
    wide = torch.full((m, n + 7), float("nan"), dtype=dtype, device=DEV)
    for off in (0, 1, 4):
        wide[:, off:off + n] = residual
        got = ko.fp8_linear(xq, xs, wq, ws, out_dtype=dtype, bias=bias, activation="silu",
                            residual=wide[:, off:off + n])
        assert torch.equal(got, want), off
        wide.fill_(float("nan"))
    for r in (residual.t().contiguous().t(), residual[:1].expand(m, n)):
        got = ko.fp8_linear(xq, xs, wq, ws, out_dtype=dtype, bias=bias, residual=r)
        ref = ko.fp8_linear(xq, xs, wq, ws, out_dtype=dtype, bias=bias, residual=r.contiguous())
        assert torch.equal(got, ref)
    b2 = torch.stack([bias, bias], 1)[:, 0]
    assert torch.equal(want, ko.fp8_linear(xq, xs, wq, ws, out_dtype=dtype, bias=b2,
                                           activation="silu", residual=residual))
    if m % 5 == 0:
        got = ko.fp8_linear(xq.view(5, -1, k), xs.view(5, m // 5, -1), wq, ws, out_dtype=dtype,
                            bias=bias, activation="silu", residual=residual.view(5, -1, n))
        assert got.shape == (5, m // 5, n) and torch.equal(got.view(m, n), want)


@pytest.mark.parametrize("m,n", [(3, 261), (70, 8197), (150, 25001)])
def test_residual_in_place_and_rows_only(m, n):
    """Through the C entry: the residual in the output's own memory, with a row
    stride above n; what lies behind the rows stays."""
    from kernel_opt._library import KLP_ACT_SILU, check_status, lib, ptr, stream_handle
    k = 144
    xq, xs, wq, ws = _matrices(m, n, k, 9)
    bias, residual = _extras(m, n, torch.bfloat16, 2)
    want = _ko().fp8_linear(xq, xs, wq, ws, bias=bias, activation="silu", residual=residual)
    buf = torch.full((m + 2, n + 5), -7.0, dtype=torch.bfloat16, device=DEV)
    buf[:m, :n] = residual
    check_status(lib.klp_fp8_linear_act(ptr(xq), k, ptr(xs), ptr(wq), k, ptr(ws), m, n, k,
                                        ptr(bias), 2, KLP_ACT_SILU, 0.0, ptr(buf), n + 5, 0,
                                        ptr(buf), n + 5, stream_handle(0)))
    assert torch.equal(buf[:m, :n], want)
    assert (buf[:m, n:] == -7.0).all() and (buf[m:] == -7.0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_infinities_and_nan(dtype):
    """An infinite bias saturates, a NaN stays, each in its own column; so for
    the residual's elements."""
    ko = _ko()
    m, n, k = 20, 300, 144
    xq, xs, wq, ws = _matrices(m, n, k, 4)
    inf = float("inf")
    bias = torch.zeros(n, device=DEV)
    bias[3], bias[7], bias[290] = inf, -inf, float("nan")
    for act in ACTS:
        kw = _act_args(act, 5.0)
        out = ko.fp8_linear(xq, xs, wq, ws, out_dtype=dtype, bias=bias, **kw)
        want = ko.fp8_linear(xq, xs, wq, ws, out_dtype=dtype, bias=torch.zeros(n, device=DEV), **kw)
        rest = torch.ones(n, dtype=torch.bool, device=DEV)
        rest[[3, 7, 290]] = False
        assert torch.equal(out[:, rest], want[:, rest])
        assert out[:, 290].isnan().all()
        assert (out[:, 3] == (5.0 if act == "softcap" else inf)).all()
        if act in (None, "softcap", "relu"):
            low = {None: -inf, "softcap": -5.0, "relu": 0.0}[act]
            assert (out[:, 7] == low).all()
        else:
            assert out[:, 7].isnan().all()  # -inf / (1 + inf)
    res = torch.zeros(m, n, dtype=dtype, device=DEV)
    res[2, 5], res[3, 6], res[4, 299] = inf, -inf, float("nan")
    out = ko.fp8_linear(xq, xs, wq, ws, out_dtype=dtype, activation="relu", residual=res)
    assert out[2, 5] == inf and out[3, 6] == -inf and out[4, 299].isnan()
    assert int((~out.isfinite()).sum()) == 3


def test_no_tokens_graph_and_stream():
    """Captured on a stream of its own and replayed with new values, with eager
    work in between; every replay equals the eager call."""
    ko = _ko()
    m, n, k = 130, 700, 528
    xq, xs, wq, ws = _matrices(m, n, k, 2)
    bias, residual = _extras(m, n, torch.bfloat16, 1)
    call = lambda: ko.fp8_linear(xq, xs, wq, ws, bias=bias, activation="gelu_tanh",  # noqa: E731
                                 residual=residual)
    empty = ko.fp8_linear(xq[:0], xs[:0], wq, ws, bias=bias, softcap=3.0, residual=residual[:0])
    assert empty.shape == (0, n)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = call()
    for rep in range(3):
        other = _matrices(m, n, k, 40 + rep)
        xq.view(torch.uint8).copy_(other[0].view(torch.uint8))
        xs.copy_(other[1])
        bias.mul_(-1.5)
        residual.neg_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())


def test_refusals():
    ko = _ko()
    q, s = ko.quantize_fp8(torch.randn(4, 256, device=DEV))
    w, ws = ko.quantize_fp8(torch.randn(300, 256, device=DEV), 128)
    bias, res = torch.zeros(300, device=DEV), torch.zeros(4, 300, device=DEV, dtype=torch.bfloat16)

    def refused(kind, text, **kw):
        with pytest.raises(kind, match=text):
            ko.fp8_linear(q, s, w, ws, **kw)

    refused(ValueError, "activation must be", activation="tanh")
    refused(ValueError, "exclude", activation="relu", softcap=3.0)
    for cap in (0.0, -1.0, float("inf"), float("nan"), 2.0 ** -101):
        refused(ValueError, "softcap", softcap=cap)
    refused(RuntimeError, "bias must be", bias=bias[:299])
    refused(RuntimeError, "bias must be", bias=bias[None])
    refused(RuntimeError, "bias must be", bias=bias.cpu())
    refused(RuntimeError, "float32 or of out_dtype", bias=bias.half())
    refused(RuntimeError, "residual must be", residual=res.float())
    refused(RuntimeError, "residual must be", residual=res[:3])
    refused(RuntimeError, "residual must be", residual=res[0])
    refused(RuntimeError, "residual must be", residual=res.cpu())
    refused(RuntimeError, "no gradient", bias=bias.clone().requires_grad_())
    refused(RuntimeError, "no gradient", residual=res.clone().requires_grad_())
    with torch.no_grad():
        ko.fp8_linear(q, s, w, ws, bias=bias.clone().requires_grad_())
        ko.fp8_linear(q, s, w, ws, bias=bias.to(torch.bfloat16), out_dtype=torch.bfloat16)


# ---------------------------------------------------------------------------
# As they are used.
# ---------------------------------------------------------------------------


def _head(vocab, dim, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = 3.0 * torch.randn(vocab, dim, generator=g, device=DEV) * dim ** -0.5
    return _ko().quantize_fp8(w.to(torch.bfloat16), block_rows=128)


@pytest.mark.parametrize("tokens", [1, 9, 200])
@pytest.mark.parametrize("with_residual", [False, True])
def test_a_capped_head_sampled_and_scored(tokens, with_residual):
    """sample_hidden and score_hidden with a bias, a cap and alternatives: the
    bits of their pieces, whatever leading shape and chunks."""
    ko = _ko()
    dim, vocab, k = 528, 9001, 5
    g = torch.Generator(device=DEV).manual_seed(tokens)
    x, res = (torch.randn(tokens, dim, generator=g, device=DEV).to(torch.bfloat16)
              for _ in range(2))
    nw = (1 + 0.1 * torch.randn(dim, generator=g, device=DEV)).to(torch.bfloat16)
    u = torch.rand(tokens, generator=g, device=DEV)
    bias = torch.randn(vocab, generator=g, device=DEV)
    head, head_scale = _head(vocab, dim, 3)
    kw = dict(residual=res) if with_residual else {}
    cap = dict(bias=bias, softcap=4.0)
    if with_residual:
        q, s, _ = ko.fused_add_rms_norm_fp8(x, res, nw)
    else:
        q, s = ko.fused_rms_norm_fp8(x, nw)
    logits = ko.fp8_linear(q, s, head, head_scale, **cap)
    assert float(logits.abs().max()) <= 4.0
    got = ko.sample_hidden(x, nw, head, head_scale, u, 0.8, top_k=50, **cap, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, ko.fused_sample(logits, u, 0.8, top_k=50)))
    tok = got[0]
    got = ko.score_hidden(x, nw, head, head_scale, tok, 0.8, **cap, **kw)
    want = ko.fused_logprob_entropy_forward(logits, tok, 0.8)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    want = ko.fused_top_logprobs(logits, tok, k, 0.8)
    for chunk in (None, 1000):
        got = ko.score_hidden(x, nw, head, head_scale, tok, 0.8, alternatives=k,
                              chunk_tokens=chunk, **cap, **kw)
        assert len(got) == 6 and all(torch.equal(a, b) for a, b in zip(got, want))
    if tokens == 9:
        kw = {a: b.view(3, 3, dim) for a, b in kw.items()}
        got = ko.score_hidden(x.view(3, 3, dim), nw, head, head_scale, tok.view(3, 3), 0.8,
                              alternatives=k, **cap, **kw)
        assert got[0].shape == (3, 3) and got[4].shape == (3, 3, k)
        assert all(torch.equal(a.flatten(), b.flatten()) for a, b in zip(got, want))
    got = ko.score_hidden(x[:0], nw, head, head_scale, tok[:0], alternatives=k)
    assert got[0].shape == (0,) and got[5].shape == (0, k)
    # A chunk of its own kernel: the same tokens' ranks lie within what a step of
    # a bf16 logit (2^-7 of at most 4) can swap.
    got = ko.score_hidden(x, nw, head, head_scale, tok, 0.8, alternatives=k, chunk_tokens=7,
                          **cap, **kw) if tokens == 200 else want
    step = 2.0 ** -7 * 4.0 / 0.8
    assert (got[0] - want[0]).abs().max() <= 2 * step + 4e-5
    assert (got[5] - want[5]).abs().max() <= 2 * step + 4e-5


def test_a_decode_step_through_two_blocks():
    """The norms around two blocks in 8 bits, an 8-bit MLP with its activation
    and residual in the products, the capped head and its alternatives: the run
    against the pieces' formulas on the same codes, in 64 bits."""
    ko = _ko()
    dim, wide, vocab, tokens, k = 256, 640, 3001, 6, 4
    g = torch.Generator(device=DEV).manual_seed(8)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    x, h = r(tokens, dim).to(torch.bfloat16), r(tokens, dim).to(torch.bfloat16)
    post = (1 + 0.1 * r(dim)).to(torch.bfloat16)
    w1, w2 = ((1 + 0.1 * r(dim)).to(torch.bfloat16) for _ in range(2))
    up = ko.quantize_fp8(r(wide, dim) * dim ** -0.5, block_rows=128)
    down = ko.quantize_fp8(r(dim, wide) * wide ** -0.5, block_rows=128)
    head = ko.quantize_fp8(3 * r(vocab, dim) * dim ** -0.5, block_rows=128)
    bias = r(wide)
    t = torch.randint(0, vocab, (tokens,), generator=g, device=DEV)

    q, s, h1 = ko.fused_block_norm_fp8(x, h, w1, post_weight=post, scale=0.5)
    mid = ko.fp8_linear(q, s, *up, bias=bias, activation="silu")
    _check(mid, _product(q, s, *up), dim, bias, "silu")
    mq, ms = ko.quantize_fp8(mid)
    out = ko.fp8_linear(mq, ms, *down, residual=h1)
    _check(out, _product(mq, ms, *down), wide, None, None, None, h1)
    q, s, h2 = ko.fused_block_norm_fp8(out, h1, w2, scale=0.5)
    logits = ko.fp8_linear(q, s, *head, softcap=6.0, out_dtype=torch.float32)
    _check(logits, _product(q, s, *head), dim, None, "softcap", 6.0)
    logp, ent, lse, rank, ids, top = ko.fused_top_logprobs(logits, t, k)
    ref = torch.log_softmax(logits.double().cpu(), -1)
    # Both are a difference of a logit (at most 6) and a logsumexp of at most
    # 6 + ln V < 15: a step of each in float32 and the sum's own error, 64 steps
    # of 1 with room.
    tol = 2.0 ** -24 * (6 + 15) + 64 * 2.0 ** -24
    assert (logp.cpu().double() - ref.gather(-1, t.cpu()[:, None])[:, 0]).abs().max() <= tol
    best = ref.topk(k)
    assert torch.equal(ids.cpu(), best.indices)
    assert (top.cpu().double() - best.values).abs().max() <= tol
    place = (ref > ref.gather(-1, t.cpu()[:, None])).sum(-1)
    assert torch.equal(rank.cpu().long(), place)
    # The same, captured whole and replayed with other states between eager runs.
    def run():
        q, s, h1 = ko.fused_block_norm_fp8(x, h, w1, post_weight=post, scale=0.5)
        mid = ko.fp8_linear(q, s, *up, bias=bias, activation="silu")
        out = ko.fp8_linear(*ko.quantize_fp8(mid), *down, residual=h1)
        q, s, h2 = ko.fused_block_norm_fp8(out, h1, w2, scale=0.5)
        logits = ko.fp8_linear(q, s, *head, softcap=6.0, out_dtype=torch.float32)
        return (h2, logits, *ko.fused_top_logprobs(logits, t, k))

    assert torch.equal(run()[2], logp)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        run()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        held = run()
    for _ in range(3):
        x.copy_(r(tokens, dim))
        h.copy_(r(tokens, dim))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, run()))


def test_a_training_step_through_two_blocks():
    """Two gated blocks' norms with 8-bit checkpoints off and on, a float32 head
    and fused_top_logprobs, all the way back: gradients against the same step in
    64 bits on the CPU."""
    ko = _ko()
    B, S, dim, vocab, k = 2, 5, 96, 257, 3
    g = torch.Generator(device=DEV).manual_seed(12)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    names = dict(x=r(B, S, dim), h=r(B, S, dim), gate=r(B, 1, dim), post=1 + 0.1 * r(dim),
                 w1=1 + 0.1 * r(dim), w2=1 + 0.1 * r(dim), mix=r(dim, dim) * dim ** -0.5,
                 head=3 * r(vocab, dim) * dim ** -0.5)
    t = torch.randint(0, vocab, (B, S), generator=g, device=DEV)
    gl, ge, gt = r(B, S), r(B, S), r(B, S, k)

    def rms(v, w):
        return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w

    def plain(p):
        h = p["h"] + 0.5 * p["gate"] * rms(p["x"], p["post"])
        z = torch.tanh(rms(h, p["w1"]) @ p["mix"])
        h = h + 0.5 * z
        return rms(h, p["w2"]) @ p["head"].t()

    def ours(p, checkpoint):
        y, h = ko.fused_block_norm(p["x"], p["h"], p["w1"], post_weight=p["post"],
                                   gate=p["gate"], scale=0.5, checkpoint=checkpoint)
        y, _ = ko.fused_block_norm(torch.tanh(y @ p["mix"]), h, p["w2"], scale=0.5)
        return y @ p["head"].t()

    ref = {n: v.double().cpu().requires_grad_() for n, v in names.items()}
    lp = torch.log_softmax(plain(ref) / 0.9, -1)
    ids = lp.topk(k).indices
    ent = -(lp.exp() * lp).sum(-1)
    ((lp.gather(-1, t.cpu()[..., None])[..., 0] * gl.cpu()).sum() + (ent * ge.cpu()).sum()
     + (lp.gather(-1, ids) * gt.cpu()).sum()).backward()
    for checkpoint in (None, "fp8"):
        leaf = {n: v.clone().requires_grad_() for n, v in names.items()}
        logp, ent2, _, _, ids2, top = ko.fused_top_logprobs(ours(leaf, checkpoint), t, k, 0.9)
        assert torch.equal(ids2.cpu(), ids)
        ((logp * gl).sum() + (ent2 * ge).sum() + (top * gt).sum()).backward()
        for n, v in leaf.items():
            want = ref[n].grad
            got = v.grad.double().cpu()
            size = float(want.abs().max())
            # Sums of at most 1000 float32 terms a factor, a dozen factors deep:
            # far within 2^-12 of a gradient's largest.  A checkpoint's values are
            # off by 2^-4 of themselves, enter the two norms' backwards only and
            # there three times each: 6 2^-4 of the same.
            tol = 2.0 ** -12 if checkpoint is None else 6 * 2.0 ** -4
            assert float((got - want).abs().max()) <= tol * size, (checkpoint, n)
