"""fused_rms_norm, fused_add_rms_norm and their e4m3 forms on the GPU, against
the float64 oracle (oracle/norm_oracle.py, oracle/fp8_oracle.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp8_oracle, norm_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]
EPS = 1e-6
U = 2.0 ** -24  # half a step of float32, relative

# Around every group shape (64 to 1024 threads, 1 to 8 chunks of 8), one
# element to the longest row.
SIZES = [(1, 1), (3, 7), (5, 128), (9, 511), (8, 512), (7, 513), (66, 1024), (5, 1601), (4, 2048),
         (3, 2049), (300, 3584), (2, 4097), (3, 8192), (2, 8200), (2, 16385), (2, 32769),
         (1, 65536)]


def _ko():
    import kernel_opt
    return kernel_opt


def _data(rows, dim, dtype, seed, weight_dtype=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = (r(rows, dim) * torch.exp(r(rows, 1))).to(dtype)
    res = (2.0 * r(rows, dim)).to(dtype)
    w = (1.0 + 0.3 * r(dim)).to(weight_dtype or dtype)
    return x, res, w, r(rows, dim).to(dtype), r(rows, dim).to(dtype)


def np64(t):
    return t.detach().cpu().double().numpy()


def _steps(dim):
    """Roundings behind a row's sum, in units of U: a thread adds at most 64
    products one after the other, a group merges 10 levels of partial sums."""
    return min(dim, 64) + 10


def _assert_y(y, h, w, dtype):
    """rstd: half of the sum's relative error, and the mean, eps, root and
    quotient round once each; y: two products and the final rounding."""
    ref, _ = norm_oracle.forward(np64(h), np64(w), EPS)
    rel = (_steps(h.shape[-1]) / 2 + 4 + 2) * U
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    bound = np.abs(ref) * (rel + half * (1 + rel)) + tiny
    assert (np.abs(np64(y) - ref) <= bound).all(), float((np.abs(np64(y) - ref) - bound).max())


def _assert_grads(dx, dw, h, w, gy, gh, dtype):
    """d_x: the dot's sum as the norm's, its terms two roundings each, and four
    more roundings on the way; relative to the terms' magnitudes.  d_weight: at
    most rows additions of terms with rstd's error, two roundings each."""
    rows, dim = h.shape
    dx_ref, dw_ref, size, dw_size = norm_oracle.backward(
        np64(h), np64(w), EPS, np64(gy), None if gh is None else np64(gh))
    srel = (_steps(dim) / 2 + 4) * U
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    acc = size * (3 * srel + (_steps(dim) + 8) * U)
    bound = acc + half * (np.abs(dx_ref) + acc) + tiny
    assert (np.abs(np64(dx) - dx_ref) <= bound).all()
    acc = dw_size * (srel + (rows + 20) * U)
    half = torch.finfo(dw.dtype).eps / 2
    tiny = 2.0 ** -25 if dw.dtype == torch.float16 else 0.0
    bound = acc + half * (np.abs(dw_ref) + acc) + tiny
    assert (np.abs(np64(dw) - dw_ref) <= bound).all()


@pytest.mark.parametrize("residual", [False, True], ids=["plain", "residual"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,dim", SIZES)
def test_forward_and_backward(rows, dim, dtype, residual):
    print(f"rms_norm {rows} x {dim} {dtype} residual={residual}", flush=True)
    x, res, w, gy, gh = _data(rows, dim, dtype, rows + dim)
    xs, ws = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    if not residual:
        y = _ko().fused_rms_norm(xs, ws, EPS)
        _assert_y(y, x, w, dtype)
        dx, dw = torch.autograd.grad(y, (xs, ws), gy.to(DEV))
        _assert_grads(dx, dw, x, w, gy, None, dtype)
        return
    rs = res.to(DEV).requires_grad_()
    y, h = _ko().fused_add_rms_norm(xs, rs, ws, EPS)
    want = (x.float() + res.float()).to(dtype)
    assert torch.equal(h.cpu(), want)
    _assert_y(y, want, w, dtype)
    dx, dr, dw = torch.autograd.grad((y, h), (xs, rs, ws), (gy.to(DEV), gh.to(DEV)))
    assert torch.equal(dx, dr)
    _assert_grads(dx, dw, want, w, gy, gh, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_float32_weight(dtype):
    x, res, w, gy, gh = _data(40, 3000, dtype, 5, torch.float32)
    xs, rs, ws = (t.to(DEV).requires_grad_() for t in (x, res, w))
    y, h = _ko().fused_add_rms_norm(xs, rs, ws, EPS)
    _assert_y(y, h, w, dtype)
    dx, _, dw = torch.autograd.grad((y, h), (xs, rs, ws), (gy.to(DEV), gh.to(DEV)))
    assert dw.dtype == torch.float32
    _assert_grads(dx, dw, h.detach().cpu(), w, gy, gh, dtype)


@pytest.mark.parametrize("rows", [1, 255, 4097])
def test_weight_gradient_over_many_rows(rows):
    x, _, w, gy, _ = _data(rows, 264, torch.float32, rows)
    xs, ws = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    y = _ko().fused_rms_norm(xs, ws, EPS)
    dx, dw = torch.autograd.grad(y, (xs, ws), gy.to(DEV))
    _assert_grads(dx, dw, x, w, gy, None, torch.float32)


@pytest.mark.parametrize("dim", [16392, 33001])
@pytest.mark.parametrize("weight_dtype", [torch.bfloat16, torch.float32], ids=["w16", "w32"])
def test_weight_gradient_over_many_wide_rows(dim, weight_dtype):
    """More rows than groups, so that a group adds rows to its share."""
    x, res, w, gy, gh = _data(523, dim, torch.bfloat16, dim, weight_dtype)
    xs, rs, ws = (t.to(DEV).requires_grad_() for t in (x, res, w))
    y, h = _ko().fused_add_rms_norm(xs, rs, ws, EPS)
    dx, dw = torch.autograd.grad((y, h), (xs, ws), (gy.to(DEV), gh.to(DEV)))
    _assert_grads(dx, dw, h.detach().cpu(), w, gy, gh, torch.bfloat16)
    only_x, = torch.autograd.grad(_ko().fused_add_rms_norm(xs, rs, ws.detach(), EPS), xs,
                                  (gy.to(DEV), gh.to(DEV)))
    assert torch.equal(only_x, dx)


def test_gradient_against_differences():
    """Central differences of <y, gy> + <h, gh> in float64 along random
    directions, with the oracle's forward; the kernel's gradient is float32."""
    x, res, w, gy, gh = _data(6, 50, torch.float32, 77)
    xs, rs, ws = (t.to(DEV).requires_grad_() for t in (x, res, w))
    y, h = _ko().fused_add_rms_norm(xs, rs, ws, EPS)
    dx, dr, dw = torch.autograd.grad((y, h), (xs, rs, ws), (gy.to(DEV), gh.to(DEV)))
    base = np64(x) + np64(res)

    def loss(hh, ww):
        return (norm_oracle.forward(hh, ww, EPS)[0] * np64(gy)).sum() + (hh * np64(gh)).sum()

    rng = np.random.RandomState(3)
    for _ in range(5):
        v, u = rng.randn(*base.shape), rng.randn(50)
        e = 1e-5
        num = (loss(base + e * v, np64(w) + e * u) - loss(base - e * v, np64(w) - e * u)) / (2 * e)
        ana = (np64(dx) * v).sum() + (np64(dw) * u).sum()
        scale = np.abs(np64(dx) * v).sum() + np.abs(np64(dw) * u).sum()
        # float32 gradients and inputs of a few hundred roundings, and e^2.
        assert abs(num - ana) <= scale * (400 * U + 1e-8)


def test_which_gradients():
    """Only those asked for; h's gradient alone; broadcast inputs."""
    ko = _ko()
    x, res, w, gy, gh = (t.to(DEV) for t in _data(12, 300, torch.float32, 8))
    full = [t.clone().requires_grad_() for t in (x, res, w)]
    y, h = ko.fused_add_rms_norm(*full[:2], full[2], EPS)
    dx, dr, dw = torch.autograd.grad((y, h), full, (gy, gh))
    for need in range(1, 8):
        t = [a.clone().requires_grad_(bool(need >> i & 1)) for i, a in enumerate((x, res, w))]
        y, h = ko.fused_add_rms_norm(t[0], t[1], t[2], EPS)
        if h.requires_grad:
            torch.autograd.backward((y, h), (gy, gh))
        else:
            y.backward(gy)
        for a, want in zip(t, (dx, dr, dw)):
            assert a.grad is None if not a.requires_grad else torch.equal(a.grad, want)
    t = [a.clone().requires_grad_() for a in (x, res, w)]
    _, h = ko.fused_add_rms_norm(t[0], t[1], t[2], EPS)
    h.backward(gh)
    assert torch.equal(t[0].grad, gh) and torch.equal(t[1].grad, gh)
    assert t[2].grad is None or not t[2].grad.any()
    # A row used by every token: its gradient is the sum of the rows'.
    row = x[:1].clone().requires_grad_()
    y, h = ko.fused_add_rms_norm(row.expand(12, 300), res, w, EPS)
    y.backward(gy)
    wide = x[:1].expand(12, 300).contiguous().requires_grad_()
    y2, _ = ko.fused_add_rms_norm(wide, res, w, EPS)
    y2.backward(gy)
    assert torch.equal(y, y2)
    # 12 rows added in two orders.
    off = (row.grad - wide.grad.sum(0, keepdim=True)).abs()
    assert (off <= 24 * U * wide.grad.abs().sum(0, keepdim=True)).all()


def test_layouts():
    """Leading dims, row strides, odd offsets, transposed inputs, no rows."""
    ko = _ko()
    g = torch.Generator().manual_seed(2)
    for dtype in DTYPES:
        base = torch.randn(3, 7, 403, generator=g).to(dtype).to(DEV)
        w = torch.randn(806, generator=g).to(dtype).to(DEV)
        for x in (base, base[:, 1:, 3:200], base[..., ::2], base.transpose(0, 1), base[0, 0]):
            d = x.size(-1)
            for wt in (w[:d], w[::2][:d]):
                res = torch.randn(x.shape, generator=g).to(dtype).to(DEV)
                y, h = ko.fused_add_rms_norm(x, res, wt, EPS)
                y2, h2 = ko.fused_add_rms_norm(x.contiguous(), res, wt.contiguous(), EPS)
                assert y.shape == x.shape and torch.equal(y, y2) and torch.equal(h, h2)
                q, s, h3 = ko.fused_add_rms_norm_fp8(x, res, wt, EPS)
                assert q.shape == x.shape and s.shape == (*x.shape[:-1], -(-d // 128))
                assert torch.equal(h, h3)
                leaf = x.detach().requires_grad_()
                torch.autograd.grad(ko.fused_rms_norm(leaf, wt, EPS).sum(), leaf)
        e = torch.empty(0, 16, dtype=dtype, device=DEV, requires_grad=True)
        ew = w[:16].detach().requires_grad_()
        y = ko.fused_rms_norm(e, ew, EPS)
        dx, dw = torch.autograd.grad(y, (e, ew), torch.empty_like(y))
        assert y.shape == (0, 16) and dx.shape == (0, 16) and not dw.any()
        assert ko.fused_rms_norm_fp8(e, ew, EPS)[1].shape == (0, 1)


def test_special_rows():
    """Zeros, the smallest and largest magnitudes, infinities and NaN: each in
    its own row."""
    x = torch.randn(8, 300, generator=torch.Generator().manual_seed(4))
    x[1] = 0.0
    x[2] *= 1e-30
    x[3, 5] = float("nan")
    x[4, 7] = float("inf")
    x[5] *= 1e15
    w = torch.ones(300)
    y = _ko().fused_rms_norm(x.to(DEV), w.to(DEV), EPS).cpu()
    ok = [0, 1, 2, 5, 6, 7]
    _assert_y(y[ok], x[ok], w, torch.float32)
    assert y[3].isnan().all() and y[4, 7].isnan() and (y[4, :7] == 0).all()
    q, s = _ko().fused_rms_norm_fp8(x.to(DEV), w.to(DEV), EPS)
    assert (s[1] == 1).all() and s[3].isnan().all() and not s[ok].isnan().any()


@pytest.mark.parametrize("residual", [False, True], ids=["plain", "residual"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,dim", [(1, 1), (5, 127), (9, 1000), (64, 3584), (3, 5003), (2, 20000)])
def test_fp8(rows, dim, dtype, residual):
    """Scales within the norm's float32 error, and every code's value within
    half an e4m3 step (2^-4 of itself, 2^-10 where steps are equal) and the
    same error of the exact quotient."""
    x, res, w, _, _ = _data(rows, dim, dtype, rows * dim)
    ko = _ko()
    if residual:
        q, s, h = ko.fused_add_rms_norm_fp8(x.to(DEV), res.to(DEV), w.to(DEV), EPS)
        assert torch.equal(h.cpu(), (x.float() + res.float()).to(dtype))
        h = h.cpu()
    else:
        q, s = ko.fused_rms_norm_fp8(x.to(DEV), w.to(DEV), EPS)
        h = x
    y, _ = norm_oracle.forward(np64(h), np64(w), EPS)
    amax = fp8_oracle.block_amax(y, 1)
    rel = (_steps(dim) / 2 + 4 + 2 + 2) * U
    ref = np.where(amax == 0, 1.0, amax / 448.0)
    assert (np.abs(np64(s) - ref) <= ref * rel).all()
    codes = fp8_oracle.decode(q.view(torch.uint8).cpu().numpy())
    exact = y / fp8_oracle.spread(ref, 1, rows, dim)
    bound = np.maximum(np.abs(exact) * 2.0 ** -4, 2.0 ** -10) + np.abs(exact) * 2 * rel
    assert (np.abs(codes - exact) <= bound).all()


def test_streams_repeats_and_graph():
    """The same bits on every call and stream; forward and backward captured in
    one graph and replayed with new inputs equal the eager calls."""
    ko = _ko()
    x, res, w, gy, gh = (t.to(DEV) for t in _data(600, 1024, torch.bfloat16, 6))
    leaves = [t.clone().requires_grad_() for t in (x, res, w)]

    def step():
        y, h = ko.fused_add_rms_norm(leaves[0], leaves[1], leaves[2], EPS)
        q, s, _ = ko.fused_add_rms_norm_fp8(leaves[0], leaves[1], leaves[2], EPS)
        grads = torch.autograd.grad((y, h), leaves, (gy, gh))
        return [t.detach().clone() for t in (y, h, q.view(torch.uint8), s, *grads)]

    want = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(want, step()))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = step()
    for rep in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn_like(x, dtype=torch.float32))
            gy.mul_(0.5)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))



def test_refusals():
    ko = _ko()
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV)
    w = torch.ones(64, dtype=torch.bfloat16, device=DEV)
    for f in (ko.fused_rms_norm, ko.fused_rms_norm_fp8):
        for bad, text in ((w[:63], "weight must be"), (w.cpu(), "weight must be"),
                          (w.half(), "weight must be float32"), (w[None], "weight must be")):
            with pytest.raises(RuntimeError, match=text):
                f(x, bad)
        with pytest.raises(RuntimeError, match="eps"):
            f(x, w, -1e-6)
        with pytest.raises(RuntimeError, match="eps"):
            f(x, w, float("nan"))
        with pytest.raises(RuntimeError, match="bf16, fp16, or fp32"):
            f(x.double(), w)
        with pytest.raises(RuntimeError, match="last dim"):
            f(torch.zeros(2, 65537, dtype=torch.bfloat16, device=DEV), w)
        with pytest.raises(RuntimeError, match="last dim"):
            f(torch.zeros(2, 0, dtype=torch.bfloat16, device=DEV), w[:0])
    for f in (ko.fused_add_rms_norm, ko.fused_add_rms_norm_fp8):
        for bad in (x[:3], x.half(), x.cpu(), x[:, :63]):
            with pytest.raises(RuntimeError, match="residual must have"):
                f(x, bad, w)


def test_rows_beyond_32_bits():
    """The last rows of 2^31 and more elements, and rows that share memory."""
    ko = _ko()
    g = torch.Generator(device=DEV).manual_seed(1)
    rows, dim = 2 ** 19 + 5, 4104
    x = torch.empty(rows, dim, dtype=torch.bfloat16, device=DEV)
    x[-3:] = torch.randn(3, dim, generator=g, device=DEV)
    w = torch.randn(dim, generator=g, device=DEV)
    y = ko.fused_rms_norm(x, w, EPS)
    assert torch.equal(y[-3:], ko.fused_rms_norm(x[-3:], w, EPS))
    del y
    q, s = ko.fused_rms_norm_fp8(x, w, EPS)
    q1, s1 = ko.fused_rms_norm_fp8(x[-3:], w, EPS)
    assert torch.equal(q[-3:].view(torch.uint8), q1.view(torch.uint8))
    assert torch.equal(s[-3:], s1)
    one = x[-1:].expand(9, dim)
    assert torch.equal(ko.fused_rms_norm(one, w, EPS), ko.fused_rms_norm(one.contiguous(), w, EPS))
