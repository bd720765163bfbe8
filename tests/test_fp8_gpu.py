"""e4m3 quantization and the product of quantized matrices on the GPU, against
the float64 oracle (oracle/fp8_oracle.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp8_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]


def _ko():
    import kernel_opt
    return kernel_opt


def _codes(q):
    return q.contiguous().view(torch.uint8).cpu().numpy()


def _assert_quantized(q, scales, v, block_rows):
    """The formula's float32 operations are exactly rounded on both sides: the
    same bits."""
    vals, ref = fp8_oracle.quantize(v.float().cpu().numpy(), block_rows)
    np.testing.assert_array_equal(scales.cpu().numpy(), ref)
    np.testing.assert_array_equal(fp8_oracle.decode(_codes(q)), vals)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 128), (3, 127), (130, 129), (257, 1000),
                                      (64, 3584), (128, 16), (5, 5003)])
def test_quantize(dtype, block_rows, rows, dim):
    g = torch.Generator().manual_seed(rows * 7 + dim)
    x = (torch.randn(rows, dim, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))).to(dtype)
    q, s = _ko().quantize_fp8(x.to(DEV), block_rows=block_rows)
    assert q.shape == x.shape and q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32
    _assert_quantized(q, s, x, block_rows)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_special_values(block_rows):
    """Zeros, one large element, the smallest magnitudes, infinities and NaN:
    each within its own blocks."""
    x = torch.zeros(256, 512)
    x[0, 0] = 1.0
    x[1, 130] = 3.0e38
    x[1, 131] = -448.0
    x[2, 256] = 1.0e-45
    x[2, 257] = -3.0e-38
    x[130, 5] = float("inf")
    x[131, 6] = 1.0
    x[132, 140] = float("nan")
    x[133, 300] = -0.0
    q, s = _ko().quantize_fp8(x.to(DEV), block_rows=block_rows)
    _assert_quantized(q, s, x, block_rows)
    stands = fp8_oracle.decode(_codes(q)) * fp8_oracle.spread(
        s.cpu().numpy(), block_rows, *x.shape)
    bad = np.isnan(stands).reshape(256 // block_rows, block_rows, 4, 128)
    want = np.zeros((256 // block_rows, 4), dtype=bool)
    want[130 // block_rows, 0] = want[132 // block_rows, 1] = True
    np.testing.assert_array_equal(bad.all(axis=(1, 3)), want)
    np.testing.assert_array_equal(bad.any(axis=(1, 3)), want)


def test_quantize_layouts():
    """Row strides, an odd offset, leading dims, transposed input, no rows."""
    ko = _ko()
    g = torch.Generator().manual_seed(3)
    base = torch.randn(4, 9, 301, generator=g, device="cpu").to(torch.bfloat16).to(DEV)
    for x in (base[:, 1:, :], base[:, :, 3:260], base.transpose(0, 1), base[..., ::2]):
        q, s = ko.quantize_fp8(x)
        assert q.shape == x.shape and s.shape == (*x.shape[:-1], -(-x.size(-1) // 128))
        _assert_quantized(q.reshape(-1, x.size(-1)), s.reshape(-1, s.size(-1)),
                          x.reshape(-1, x.size(-1)), 1)
    q, s = ko.quantize_fp8(base[0, :, 1:].t(), block_rows=128)
    _assert_quantized(q, s, base[0, :, 1:].t(), 128)
    q, s = ko.quantize_fp8(torch.empty(0, 300, device=DEV), block_rows=128)
    assert q.shape == (0, 300) and s.shape == (0, 3)


# ---------------------------------------------------------------------------


def _matrices(m, n, k, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    ko = _ko()
    x = torch.randn(m, k, generator=g, device=DEV) * torch.exp(
        torch.randn(m, 1, generator=g, device=DEV))
    w = torch.randn(n, k, generator=g, device=DEV) * k ** -0.5
    return *ko.quantize_fp8(x), *ko.quantize_fp8(w, block_rows=128)


def _bound(ref, size, dropped, k, dtype):
    """Per output.  A block's 128 products are exact in float32, their sum is
    off by at most a rounding an addition (2^-23, half a step or a truncation),
    the scales' product and the multiply-add to the accumulator round once a
    block each: (128 + 2 blocks) 2^-23 of the terms' magnitudes.  16-bit
    outputs come from the e4m3 instruction, which drops from each of 8 neighbouring products what lies below 2^-13 of 2^E, E the
    largest exponent sum of the 8: that product itself, 6 bits behind its
    leading one, loses nothing, the other 7 less than 2^-13 2^E <= 2^-13 of it
    each (`dropped`: the sum of the groups' largest products).  The output
    rounds once (an fp16 one to a step of at least 2^-24)."""
    blocks = -(-k // 128)
    acc = (128 + 2 * blocks) * 2.0 ** -23 * size
    if dtype != torch.float32:
        acc = acc + 7 * 2.0 ** -13 * dropped
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134
    return acc + half * (np.abs(ref) + acc) + tiny


def _check_linear(out, xq, xs, wq, ws):
    ref, size, dropped = fp8_oracle.linear(fp8_oracle.decode(_codes(xq)), xs.cpu().numpy(),
                                           fp8_oracle.decode(_codes(wq)), ws.cpu().numpy())
    got = out.double().cpu().numpy()
    bound = _bound(ref, size, dropped, xq.size(1), out.dtype)
    over = np.abs(got - ref) > bound
    assert np.isfinite(got).all() and not over.any(), (
        int(over.sum()), np.argwhere(over)[:3].tolist(), float(np.abs(got - ref).max()))


# Every kernel: small products split over K (16, 32 or 64 tokens at a time) and
# the four tiles (tokens x weight rows 64 x 128, 128 x 128, 128 x 256, and, but
# for float32 outputs, 256 x 256); token, row and K counts around their sides.
@pytest.mark.parametrize("m,n,k", [
    # split
    (1, 1, 16), (1, 512, 128), (3, 129, 144), (16, 1000, 272), (17, 257, 1024), (33, 640, 3584),
    (64, 65, 48), (129, 255, 16), (256, 256, 1040),
    # 64 x 128
    (1, 65536, 256), (20, 65600, 144), (64, 65537, 400), (65, 3001, 128), (300, 1537, 512),
    # 128 x 128
    (128, 20000, 272), (127, 17025, 656),
    # 128 x 256
    (130, 25000, 144), (255, 25090, 16),
    # 256 x 256
    (500, 30001, 144), (257, 40000, 400),
])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_linear(m, n, k, dtype):
    print(f"fp8_linear {m} x {n} x {k} {dtype}", flush=True)
    xq, xs, wq, ws = _matrices(m, n, k, m + n + k)
    out = _ko().fp8_linear(xq, xs, wq, ws, out_dtype=dtype)
    assert out.shape == (m, n) and out.dtype == dtype
    _check_linear(out, xq, xs, wq, ws)


@pytest.mark.parametrize("m,n", [(5, 300), (100, 8300), (300, 8300), (500, 30001)])
def test_linear_layouts(m, n):
    """Row strides above K on both sides, leading dims, scales in another
    order in memory; what lies behind the rows' K (NaN codes) never enters."""
    k = 208
    xq, xs, wq, ws = _matrices(m, n, k, 11)
    want = _ko().fp8_linear(xq, xs, wq, ws)
    xb = torch.full((m, k + 48), 0x7F, dtype=torch.uint8, device=DEV)
    wb = torch.full((n, k + 16), 0x7F, dtype=torch.uint8, device=DEV)
    xb[:, :k] = xq.view(torch.uint8)
    wb[:, :k] = wq.view(torch.uint8)
    x2 = xb.view(torch.float8_e4m3fn)[:, :k]
    w2 = wb.view(torch.float8_e4m3fn)[:, :k]
    got = _ko().fp8_linear(x2, xs.t().contiguous().t(), w2, ws.t().contiguous().t())
    assert torch.equal(got, want)
    if m % 4 == 0:
        got = _ko().fp8_linear(xq.view(4, m // 4, k), xs.view(4, m // 4, 2), wq, ws)
        assert got.shape == (4, m // 4, n) and torch.equal(got.view(m, n), want)


@pytest.mark.parametrize("m,n", [(1, 384), (64, 384), (96, 8320), (260, 8320)])
def test_linear_nan_and_zero_scales(m, n):
    """A NaN code or scale enters its outputs and no others; a scale of zero
    takes its block away."""
    k = 400
    xq, xs, wq, ws = _matrices(m, n, k, 5)
    xs, ws = xs.clone(), ws.clone()
    xs[0, 1] = 0.0
    ws[2, 3] = 0.0
    out = _ko().fp8_linear(xq, xs, wq, ws, out_dtype=torch.float32)
    _check_linear(out, xq, xs, wq, ws)
    wq.view(torch.uint8)[130, 7] = 0x7F
    ws[0, 0] = float("nan")
    bad = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    bad[:, 130] = True
    bad[:, :128] = True
    if m > 1:
        xq.view(torch.uint8)[m - 1, k - 1] = 0xFF
        bad[m - 1] = True
    out2 = _ko().fp8_linear(xq, xs, wq, ws, out_dtype=torch.float32)
    assert torch.equal(out2.isnan(), bad)
    assert torch.equal(out2[~bad], out[~bad])


def test_linear_writes_its_rows_only():
    """Through the C entry: an output with a row stride above n keeps what lies
    behind each row and behind the last one."""
    from kernel_opt._library import check_status, lib, ptr, stream_handle
    k = 144
    for m, n in ((3, 261), (70, 8197), (150, 8197), (150, 25001), (500, 30001)):
        xq, xs, wq, ws = _matrices(m, n, k, 9)
        want = _ko().fp8_linear(xq, xs, wq, ws)
        buf = torch.full((m + 2, n + 5), -7.0, dtype=torch.bfloat16, device=DEV)
        check_status(lib.klp_fp8_linear(ptr(xq), k, ptr(xs), ptr(wq), k, ptr(ws), m, n, k, 0,
                                        ptr(buf), n + 5, stream_handle(0)))
        assert torch.equal(buf[:m, :n], want)
        assert (buf[:m, n:] == -7.0).all() and (buf[m:] == -7.0).all()


def test_linear_no_tokens_and_repeatable():
    xq, xs, wq, ws = _matrices(300, 512, 512, 1)
    out = _ko().fp8_linear(xq[:0], xs[:0], wq, ws)
    assert out.shape == (0, 512)
    a = _ko().fp8_linear(xq, xs, wq, ws)
    assert all(torch.equal(a, _ko().fp8_linear(xq, xs, wq, ws)) for _ in range(3))
    # A token's outputs do not depend on its neighbours' count within a kernel.
    b = _ko().fp8_linear(xq[:200], xs[:200], wq, ws)
    assert torch.equal(a[:200], b)


def test_linear_graph_and_stream():
    """Captured on a stream of its own and replayed with new codes, with eager
    work in between; every replay equals the eager call."""
    m, n, k = 130, 700, 528
    xq, xs, wq, ws = _matrices(m, n, k, 2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _ko().fp8_linear(xq, xs, wq, ws)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = _ko().fp8_linear(xq, xs, wq, ws)
    for rep in range(3):
        other = _matrices(m, n, k, 40 + rep)
        xq.view(torch.uint8).copy_(other[0].view(torch.uint8))
        xs.copy_(other[1])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, _ko().fp8_linear(xq, xs, wq, ws))


def test_refusals():
    ko = _ko()
    x = torch.randn(4, 256, device=DEV)
    with pytest.raises(ValueError, match="block_rows"):
        ko.quantize_fp8(x, 64)
    with pytest.raises(RuntimeError, match="bf16, fp16, or fp32"):
        ko.quantize_fp8(x.double())
    with pytest.raises(RuntimeError, match=r"\[N, dim\]"):
        ko.quantize_fp8(x[None], 128)
    with pytest.raises(RuntimeError, match="dim >= 1"):
        ko.quantize_fp8(x[:, :0])
    q, s = ko.quantize_fp8(x)
    w, ws = ko.quantize_fp8(torch.randn(300, 256, device=DEV), 128)
    good = (q, s, w, ws)

    def refused(text, at=None, value=None, **kw):
        args = list(good)
        if at is not None:
            args[at] = value
        with pytest.raises(RuntimeError, match=text):
            ko.fp8_linear(*args, **kw)

    refused("GPU tensors", 1, s.cpu())
    refused("float8_e4m3fn", 0, x)
    refused("float8_e4m3fn", 2, w.view(torch.uint8))
    refused("scales must be float32", 3, ws.bfloat16())
    refused("out_dtype", out_dtype=torch.float64)
    refused("x must be", 0, q[:, :128])
    refused("x must be", 2, w[0])
    refused("x must be", 2, w[:0])
    refused("x_scale must be", 1, s[:3])
    refused("x_scale must be", 1, s[:, :1])
    refused("weight_scale must be", 3, ws[:2])
    refused("no gradient", 1, s.clone().requires_grad_())
    with torch.no_grad():
        ko.fp8_linear(q, s.clone().requires_grad_(), w, ws)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        ko.fp8_linear(q[:, :40], s[:, :1], w[:, :40], ws[:, :1])
    # Rows that do not start at multiples of 16 bytes.
    with pytest.raises(RuntimeError, match="16"):
        ko.fp8_linear(q[:, 8:136], s[:, :1], w[:, 8:136], ws[:, :1])
    odd = torch.zeros(4, 264, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)[:, :256]
    with pytest.raises(RuntimeError, match="multiples of 16"):
        ko.fp8_linear(odd, s, w, ws)


def test_linear_beyond_32_bits():
    """Weights and outputs of more than 2^32 bytes or 2^31 elements: the last
    rows and columns are those of the product of these alone; a row that is
    every row."""
    ko = _ko()
    g = torch.Generator(device=DEV).manual_seed(7)
    byte = lambda *sh: torch.randint(0, 0x70, sh, dtype=torch.uint8, device=DEV,  # noqa: E731
                                     generator=g).view(torch.float8_e4m3fn)
    n, k = 2 ** 18 + 128, 2 ** 14 + 16
    w = torch.zeros(n, k, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    w[-256:] = byte(256, k)
    nb = -(-k // 128)
    ws = torch.rand(-(-n // 128), nb, device=DEV, generator=g)
    for m in (3, 300):
        x, xs = byte(m, k), torch.rand(m, nb, device=DEV, generator=g)
        out = ko.fp8_linear(x, xs, w, ws)
        # Another count of outputs may take another kernel: K is then added in
        # another order, 130 blocks' sums of like size and all positive.
        ref = ko.fp8_linear(x, xs, w[-256:], ws[-2:]).float()
        tol = 2 * 2.0 ** -8 + 2 * 140 * 2.0 ** -24 + 7 * 2.0 ** -13
        assert ((out[:, -256:].float() - ref).abs() <= tol * ref).all()
    del w, out
    n, m, k = 152064, 15000, 128
    x, xs = byte(m, k), torch.rand(m, 1, device=DEV, generator=g)
    w, ws = byte(n, k), torch.rand(n // 128, 1, device=DEV, generator=g)
    out = ko.fp8_linear(x, xs, w, ws)
    assert out.numel() > 2 ** 31
    assert torch.equal(out[-300:], ko.fp8_linear(x[-300:], xs[-300:], w, ws))
    same = ko.fp8_linear(x[-1:].expand(70, k), xs[-1:].expand(70, 1), w, ws)
    assert torch.equal(same, out[-1:].expand(70, n))


def test_quantize_beyond_32_bits():
    ko = _ko()
    x = torch.zeros(2 ** 20 + 3, 2056, dtype=torch.bfloat16, device=DEV)
    x[-5:] = torch.randn(5, 2056, device=DEV)
    q, s = ko.quantize_fp8(x)
    q1, s1 = ko.quantize_fp8(x[-5:])
    assert torch.equal(q[-5:].view(torch.uint8), q1.view(torch.uint8))
    assert torch.equal(s[-5:], s1)
