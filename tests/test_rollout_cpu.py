"""The norm, 8-bit and sampling operators on the CPU: their C entry points and
Python functions refuse bad arguments with the documented status and message
before touching the GPU, the oracles agree with independent statements, and the
generated code of the product keeps its wait states.  No compute call is made."""
from __future__ import annotations

import ctypes
import re

import numpy as np
import pytest
import torch

import isa_listing
from mfma_hazards import hazards
from oracle import fp8_oracle, norm_oracle
from oracle.sample_oracle import sample_row

# Fake, suitably aligned addresses: every call below fails its checks (or meets
# the injected failure) before any pointer is followed.
P = ctypes.c_void_p(0x10000)
ODD = ctypes.c_void_p(0x10001)


def _lib():
    from kernel_opt import _library
    return _library


def _refused(rc, status, text):
    L = _lib()
    assert rc == getattr(L, status), (rc, L.last_error())
    assert text in L.last_error(), L.last_error()


def _norm(x=P, dtype=0, ld=64, res=None, ldr=0, w=P, wd=0, rows=4, dim=64, eps=1e-6, y=P, h=None,
          rstd=P):
    return _lib().lib.klp_rms_norm(x, dtype, ld, res, ldr, w, wd, rows, dim, eps, y, h, rstd, None)


def _norm8(x=P, dtype=0, ld=64, res=None, ldr=0, w=P, wd=0, rows=4, dim=64, eps=1e-6, q=P,
           scales=P, h=None):
    return _lib().lib.klp_rms_norm_fp8(x, dtype, ld, res, ldr, w, wd, rows, dim, eps, q, scales, h,
                                       None)


@pytest.mark.parametrize("call", [_norm, _norm8], ids=["norm", "norm8"])
def test_norm_refusals(call):
    _refused(call(dtype=9), "KLP_EDTYPE", "x dtype")
    _refused(call(wd=1), "KLP_EDTYPE", "weight must be float32")
    _refused(call(dim=0), "KLP_EINVAL", "dim must be in [1, 65536]")
    _refused(call(dim=65537), "KLP_EINVAL", "got 65537")
    _refused(call(rows=-1), "KLP_EINVAL", "rows")
    _refused(call(rows=2 ** 31), "KLP_EINVAL", "2^31-1")
    _refused(call(x=None), "KLP_EINVAL", "x must be non-null")
    _refused(call(x=ODD), "KLP_EINVAL", "aligned")
    _refused(call(w=None), "KLP_EINVAL", "weight must be non-null")
    _refused(call(wd=2, w=ctypes.c_void_p(0x10002)), "KLP_EINVAL", "weight")
    _refused(call(ld=-1), "KLP_EINVAL", "strides")
    _refused(call(res=P, h=None), "KLP_EINVAL", "h must be non-null")
    _refused(call(res=ODD, h=P), "KLP_EINVAL", "residual")
    for eps in (-1.0, float("nan"), float("inf")):
        _refused(call(eps=eps), "KLP_EINVAL", "eps")
    assert call(rows=0, x=None, w=None) == 0
    L = _lib()
    L.lib.klp_debug_fail_next_launches(1)
    try:
        _refused(call(), "KLP_ELAUNCH", "injected")
    finally:
        L.lib.klp_debug_fail_next_launches(0)


def test_norm_output_refusals():
    _refused(_norm(y=None), "KLP_EINVAL", "y must be")
    _refused(_norm(rstd=ctypes.c_void_p(0x10002)), "KLP_EINVAL", "rstd")
    _refused(_norm8(q=None), "KLP_EINVAL", "q must be")
    _refused(_norm8(scales=None), "KLP_EINVAL", "scales")


def test_launches_of_too_many_threads_are_refused():
    """2^32 threads or more: a row takes 64 to 1024 of the norm, a scale block
    16 or 256, 16 weight rows 256, 128 x 64 outputs 512, a sampled row 512."""
    L = _lib().lib
    for dim, threads in ((8, 64), (2049, 256), (5000, 512), (65536, 1024)):
        most = 2 ** 32 // threads
        _refused(_norm(rows=most, dim=dim, ld=dim), "KLP_EINVAL", "too many rows")
        _refused(_norm8(rows=most, dim=dim, ld=dim), "KLP_EINVAL", "too many rows")
        _refused(L.klp_rms_norm_bwd(P, 0, dim, P, 0, P, P, None, most, dim, P, None, None, 0, None),
                 "KLP_EINVAL", "too many rows")
    _refused(L.klp_quantize_fp8(P, 0, 128, 2 ** 28, 128, 1, P, P, None), "KLP_EINVAL", "too many")
    _refused(L.klp_quantize_fp8(P, 0, 128, 2 ** 22, 2 ** 16, 128, P, P, None), "KLP_EINVAL",
             "too many")
    for m, n in ((1, 2 ** 30), (2 ** 20, 2 ** 20)):
        _refused(L.klp_fp8_linear(P, 16, P, P, 16, P, m, n, 16, 0, P, n, None), "KLP_EINVAL",
                 "too many")
    _refused(L.klp_sample(P, 0, 2 ** 23, 8, 2 ** 23, 0, 8, P, 1.0, None, 0, None, 1.0, None, 0.0,
                          None, P, P, P, None), "KLP_EINVAL", "too many rows")


def test_norm_backward_refusals():
    L = _lib()
    need = L.lib.klp_rms_norm_bwd_workspace_bytes(100, 64)
    assert need >= 64 * 4 and need % 4 == 0
    assert L.lib.klp_rms_norm_bwd_workspace_bytes(0, 64) == 0
    assert L.lib.klp_rms_norm_bwd_workspace_bytes(4, 1 << 20) == 0

    def call(h=P, dtype=0, ld=64, w=P, wd=0, rstd=P, gy=P, gh=None, rows=100, dim=64, dx=P, dw=P,
             ws=P, ws_bytes=need):
        return L.lib.klp_rms_norm_bwd(h, dtype, ld, w, wd, rstd, gy, gh, rows, dim, dx, dw, ws,
                                      ws_bytes, None)

    _refused(call(rows=0), "KLP_EINVAL", "rows must be >= 1")
    _refused(call(rstd=None), "KLP_EINVAL", "rstd")
    _refused(call(gy=None), "KLP_EINVAL", "g_y")
    _refused(call(gh=ODD), "KLP_EINVAL", "gradients")
    _refused(call(dx=None), "KLP_EINVAL", "d_x")
    _refused(call(dw=ODD), "KLP_EINVAL", "d_weight")
    _refused(call(ws=None), "KLP_EWORKSPACE", "workspace")
    _refused(call(ws_bytes=need - 4), "KLP_EWORKSPACE", "need")
    _refused(call(ws=ctypes.c_void_p(0x10008)), "KLP_EWORKSPACE", "16-byte")
    _refused(call(dim=70000), "KLP_EINVAL", "dim")
    L.lib.klp_debug_fail_next_launches(1)
    try:  # without d_weight no workspace is asked for
        _refused(call(dw=None, ws=None, ws_bytes=0), "KLP_ELAUNCH", "injected")
    finally:
        L.lib.klp_debug_fail_next_launches(0)


def test_quantize_refusals():
    def call(x=P, dtype=0, ld=64, rows=4, dim=64, br=1, q=P, s=P):
        return _lib().lib.klp_quantize_fp8(x, dtype, ld, rows, dim, br, q, s, None)

    _refused(call(dtype=-1), "KLP_EDTYPE", "x dtype")
    _refused(call(br=64), "KLP_EINVAL", "block_rows must be 1 or 128, got 64")
    _refused(call(rows=-1), "KLP_EINVAL", "rows")
    _refused(call(dim=0), "KLP_EINVAL", "dim")
    _refused(call(x=None), "KLP_EINVAL", "x must be")
    _refused(call(x=ODD), "KLP_EINVAL", "aligned")
    _refused(call(ld=-2), "KLP_EINVAL", "stride")
    _refused(call(q=None), "KLP_EINVAL", "q must be")
    _refused(call(s=ODD), "KLP_EINVAL", "scales")
    _refused(call(rows=1 << 26, dim=1 << 14), "KLP_EINVAL", "too many scale blocks")
    _refused(call(rows=1 << 24, br=128), "KLP_EINVAL", "too many scale blocks")
    assert call(rows=0, x=None, q=None, s=None) == 0


def test_linear_refusals():
    def call(x=P, ldx=64, xs=P, w=P, ldw=64, ws=P, m=4, n=8, k=64, dt=0, out=P, ldo=8):
        return _lib().lib.klp_fp8_linear(x, ldx, xs, w, ldw, ws, m, n, k, dt, out, ldo, None)

    _refused(call(dt=3), "KLP_EDTYPE", "out dtype")
    _refused(call(n=0), "KLP_EINVAL", "n >= 1")
    _refused(call(m=-1), "KLP_EINVAL", "m must be")
    for k in (0, 8, 100):
        _refused(call(k=k), "KLP_EINVAL", f"k must be a positive multiple of 16, got {k}")
    _refused(call(x=ctypes.c_void_p(0x10008)), "KLP_EINVAL", "x is not 16-byte aligned")
    _refused(call(w=ctypes.c_void_p(0x10004)), "KLP_EINVAL", "w is not 16-byte aligned")
    _refused(call(ldx=72), "KLP_EINVAL", "multiples of 16")
    _refused(call(ldw=-16), "KLP_EINVAL", "stride")
    _refused(call(xs=None), "KLP_EINVAL", "x_scales")
    _refused(call(ws=ODD), "KLP_EINVAL", "w_scales")
    _refused(call(out=None), "KLP_EINVAL", "out must be")
    _refused(call(ldo=7), "KLP_EINVAL", "row stride >= n")
    _refused(call(m=(1 << 20) + 1), "KLP_EINVAL", "must not exceed")
    _refused(call(k=1 << 25), "KLP_EINVAL", "must not exceed")
    _refused(call(m=1 << 20, n=1 << 30, ldo=1 << 30), "KLP_EINVAL", "too many")
    assert call(m=0, x=None, out=None) == 0


def test_sample_refusals():
    def call(x=P, dtype=0, n=4, v=100, ri=4, so=0, si=100, u=P, t=1.0, ts=None, k=0, ks=None,
             p=1.0, ps=None, m=0.0, ms=None, tok=P, lp=P, sl=P):
        return _lib().lib.klp_sample(x, dtype, n, v, ri, so, si, u, t, ts, k, ks, p, ps, m, ms, tok,
                                     lp, sl, None)

    _refused(call(dtype=5), "KLP_EDTYPE", "logits dtype")
    _refused(call(v=0), "KLP_EINVAL", "vocab")
    _refused(call(v=(1 << 26) + 1), "KLP_EINVAL", "2^26")
    _refused(call(n=-1), "KLP_EINVAL", "n_rows")
    _refused(call(x=None), "KLP_EINVAL", "non-null")
    _refused(call(x=ODD), "KLP_EINVAL", "aligned")
    _refused(call(ri=0), "KLP_EINVAL", "rows_inner")
    _refused(call(si=-1), "KLP_EINVAL", "strides")
    _refused(call(u=None), "KLP_EINVAL", "uniform")
    _refused(call(tok=ctypes.c_void_p(0x10004)), "KLP_EINVAL", "tokens")
    _refused(call(lp=None), "KLP_EINVAL", "logp")
    _refused(call(sl=ODD), "KLP_EINVAL", "sample_logp")
    for t in (-1.0, float("nan"), float("inf")):
        _refused(call(t=t), "KLP_EINVAL", "temperature must be finite and >= 0")
    for name in ("ts", "ks", "ps", "ms"):
        _refused(call(**{name: ctypes.c_void_p(0x10002)}), "KLP_EINVAL", "per-row parameters")
    assert call(n=0, x=None, u=None, tok=None, lp=None, sl=None) == 0


def test_python_refuses_cpu_tensors_and_bad_values():
    import kernel_opt as ko
    x, w = torch.zeros(3, 32), torch.zeros(32)
    for f in (lambda: ko.fused_rms_norm(x, w), lambda: ko.fused_add_rms_norm(x, x, w),
              lambda: ko.fused_rms_norm_fp8(x, w), lambda: ko.quantize_fp8(x),
              lambda: ko.fp8_linear(x, x, x, x), lambda: ko.fused_sample(x, w[:3]),
              lambda: ko.sample_hidden(x, w, x, x, w[:3]),
              lambda: ko.score_hidden(x, w, x, x, torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            f()
    with pytest.raises(RuntimeError, match="int64"):
        ko.score_hidden(x, w, x, x, torch.zeros(3))
    with pytest.raises(RuntimeError, match="leading shape"):
        ko.score_hidden(x, w, x, x, torch.zeros(4, dtype=torch.int64))


def test_sample_parameters():
    from kernel_opt.sample import _parameter
    dev, f, i = torch.device("cpu"), torch.float32, torch.int32
    p = lambda v, dt, lo, hi: _parameter(v, "p", (3,), dev, dt, 7, lo, hi)  # noqa: E731
    assert p(None, f, 0, 1) == (7, None)
    assert p(0.5, f, 0, 1) == (0.5, None)
    assert p(4, i, 0, 9) == (4, None)
    for bad, dt in ((-0.1, f), (1.5, f), (float("nan"), f), (float("inf"), f), (2.5, i), (True, i),
                    (-1, i)):
        with pytest.raises(ValueError):
            p(bad, dt, 0, 1)
    with pytest.raises(RuntimeError, match="must be a number or"):
        p(torch.zeros(4), f, 0, 1)
    with pytest.raises(RuntimeError, match="integers"):
        p(torch.zeros(3), i, 0, 1)
    big = p(torch.tensor([5, -4, 1 << 40]), i, 0, 1)[1]
    assert big.dtype == i and big.tolist() == [5, 0, 2 ** 31 - 1]


def test_e4m3_oracle_agrees_with_torch():
    codes = torch.arange(256, dtype=torch.uint8)
    vals = codes.view(torch.float8_e4m3fn).float().numpy()
    np.testing.assert_array_equal(fp8_oracle.E4M3, vals.astype(np.float64))
    g = torch.Generator().manual_seed(0)
    x = torch.cat([torch.randn(20000, generator=g) * 100, torch.randn(20000, generator=g) * 1e-3,
                   torch.linspace(-448, 448, 4001), torch.tensor([0.0, 2.0 ** -10, 3 * 2.0 ** -10])])
    x = x.clamp(-448, 448)
    np.testing.assert_array_equal(fp8_oracle.round_e4m3(x.double().numpy()),
                                  x.to(torch.float8_e4m3fn).double().numpy())


def test_norm_oracle_against_autograd():
    g = torch.Generator().manual_seed(1)
    h, w, gy, gh = (torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True)
                    for s in ((5, 33), (33,), (5, 33), (5, 33)))
    y = h * (h.square().mean(1, keepdim=True) + 1e-6).rsqrt() * w
    dh, dw = torch.autograd.grad((y, h * 1), (h, w), (gy, gh))
    n = lambda t: t.detach().numpy()  # noqa: E731
    np.testing.assert_allclose(norm_oracle.forward(n(h), n(w), 1e-6)[0], n(y), rtol=1e-12)
    dx, dwo, _, _ = norm_oracle.backward(n(h), n(w), 1e-6, n(gy), n(gh))
    np.testing.assert_allclose(dx, n(dh), rtol=1e-9, atol=1e-12)
    np.testing.assert_allclose(dwo, n(dw), rtol=1e-9, atol=1e-12)


def test_sample_oracle_by_hand():
    x = np.log([0.1, 0.2, 0.4, 0.3])
    draw = lambda u, **kw: sample_row(x, u, **kw)  # noqa: E731
    assert [draw(u)[0] for u in (0.05, 0.15, 0.5, 0.8)] == [0, 1, 2, 3]
    assert list(draw(0.5, top_k=2)[3]) == [2, 3] and draw(0.5, top_k=2)[0] == 2
    assert list(draw(0.5, top_p=0.6)[3]) == [2, 3]
    assert list(draw(0.5, top_p=0.39)[3]) == [2]
    assert list(draw(0.5, min_p=0.5)[3]) == [1, 2, 3] or list(draw(0.5, min_p=0.5)[3]) == [2, 3]
    tok, lp, slp, _ = draw(0.9, top_k=2)
    assert tok == 3 and abs(lp - np.log(0.3)) < 1e-12 and abs(slp - np.log(3 / 7)) < 1e-12
    assert draw(0.9, temperature=0.0)[:3] == (2, pytest.approx(np.log(0.4)), 0.0)
    assert sample_row([1.0, 1.0, 1.0], 0.99, top_k=2)[0] == 1
    assert sample_row([-np.inf, -np.inf], 0.5)[0] == -1
    assert sample_row([0.0, np.nan], 0.5)[0] == -1
    assert sample_row([0.0, 1.0], 1.0)[0] == 1


@pytest.mark.skipif(not isa_listing.available(), reason="hipcc not available")
def test_product_kernels_have_wait_states():
    """The copies written in asm: 5 wait states from a VALU instruction that
    writes their scalars, 1 from writing M0, which nothing else uses."""
    listing = isa_listing.listing("klp_fp8_gemm.hip")
    assert len(re.findall(r"^\s+v_mfma_f32_16x16x128_f8f6f4", listing, re.M)) > 0
    assert len(re.findall(r"^\s+v_mfma_scale", listing, re.M)) == 0
    found = {k: [f for f in v if f[0].startswith("buffer_load_dword")]
             for k, v in hazards(listing).items()}  # the rest is the compiler's
    assert not any(found.values()), {k: v[:2] for k, v in found.items() if v}
    blocks = [b for b in re.findall(r";;#ASMSTART\n(.*?);;#ASMEND", listing, re.S)
              if "buffer_load_dword" in b]
    assert blocks and all("s_mov_b32 m0" in b for b in blocks)
    uses = [s for s in listing.splitlines() if re.search(r"\bm0\b", s.split(";")[0])]
    assert len(uses) == len(blocks)


@pytest.mark.skipif(not isa_listing.available(), reason="hipcc not available")
@pytest.mark.parametrize("source", ["klp_norm.hip", "klp_fp8.hip", "klp_fp8_gemm.hip",
                                    "klp_sample.hip"])
def test_no_packed_float_arithmetic(source):
    assert not re.search(r"^\s+v_pk_(add|mul|fma)_f32", isa_listing.listing(source), re.M)
