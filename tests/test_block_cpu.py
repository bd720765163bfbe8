"""The C entry points of the norms around a block refuse bad arguments before
touching the GPU; the oracle agrees with torch's autograd.  No compute call is
made."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import block_oracle, norm_oracle

P = ctypes.c_void_p(0x10000)
ODD = ctypes.c_void_p(0x10001)


def _lib():
    from kernel_opt import _library
    return _library


def _refused(rc, status, text):
    L = _lib()
    assert rc == getattr(L, status), (rc, L.last_error())
    assert text in L.last_error(), L.last_error()


def _fwd(x=P, dtype=0, ld=64, r=P, ldr=64, wp=None, w=P, wd=0, g=None, gd=0, per=1, scale=1.0,
         rows=4, dim=64, eps=1e-6, y=P, h=P, sx=None, sh=None, xq=None, xs=None, hq=None, hs=None):
    return _lib().lib.klp_block_norm(x, dtype, ld, r, ldr, wp, w, wd, g, gd, per, scale, rows, dim,
                                     eps, y, h, sx, sh, xq, xs, hq, hs, None)


def _fwd8(x=P, dtype=0, ld=64, r=P, ldr=64, wp=None, w=P, wd=0, g=None, gd=0, per=1, scale=1.0,
          rows=4, dim=64, eps=1e-6, q=P, s=P, h=P):
    return _lib().lib.klp_block_norm_fp8(x, dtype, ld, r, ldr, wp, w, wd, g, gd, per, scale, rows,
                                         dim, eps, q, s, h, None)


def _bwd(x=P, dtype=0, ld=64, xq=None, xs=None, h=P, hq=None, hs=None, wp=P, w=P, wd=0, g=P, gd=0,
         per=1, scale=1.0, sx=P, sh=P, gy=P, gh=P, rows=4, dim=64, dx=P, dr=P, dp=None, dw=None,
         dg=None, ws=None, n=0):
    return _lib().lib.klp_block_norm_bwd(x, dtype, ld, xq, xs, h, hq, hs, wp, w, wd, g, gd, per,
                                         scale, sx, sh, gy, gh, rows, dim, dx, dr, dp, dw, dg, ws,
                                         n, None)


@pytest.mark.parametrize("call", [_fwd, _fwd8, _bwd], ids=["norm", "norm8", "backward"])
def test_refusals(call):
    _refused(call(dtype=9), "KLP_EDTYPE", "x dtype")
    _refused(call(wd=1), "KLP_EDTYPE", "weights must be float32")
    _refused(call(g=P, gd=1), "KLP_EDTYPE", "gate must be float32")
    _refused(call(dim=0), "KLP_EINVAL", "dim must be in [1, 16384]")
    _refused(call(dim=16385, ld=16385), "KLP_EINVAL", "got 16385")
    _refused(call(rows=-1), "KLP_EINVAL", "rows")
    _refused(call(rows=2 ** 31), "KLP_EINVAL", "2^31-1")
    _refused(call(rows=2 ** 22), "KLP_EINVAL", "too many rows")
    _refused(call(g=P, per=0), "KLP_EINVAL", "rows_per_gate")
    _refused(call(g=ODD), "KLP_EINVAL", "gate is not aligned")
    for scale in (float("nan"), float("inf")):
        _refused(call(scale=scale), "KLP_EINVAL", "scale")
    _refused(call(x=None, wp=P), "KLP_EINVAL", "x must be non-null")
    _refused(call(x=ODD, wp=P), "KLP_EINVAL", "aligned")
    _refused(call(ld=-1, wp=P), "KLP_EINVAL", "stride")
    _refused(call(w=None), "KLP_EINVAL", "weight must be non-null")
    _refused(call(wp=ODD), "KLP_EINVAL", "aligned")
    _refused(call(h=None), "KLP_EINVAL", "h must be non-null")
    L = _lib()
    L.lib.klp_debug_fail_next_launches(1)
    try:
        _refused(call(), "KLP_ELAUNCH", "injected")
    finally:
        L.lib.klp_debug_fail_next_launches(0)


@pytest.mark.parametrize("call", [_fwd, _fwd8], ids=["norm", "norm8"])
def test_forward_refusals(call):
    _refused(call(r=None), "KLP_EINVAL", "residual must be non-null")
    _refused(call(ldr=-1), "KLP_EINVAL", "residual: row stride")
    for eps in (-1.0, float("nan"), float("inf")):
        _refused(call(eps=eps), "KLP_EINVAL", "eps")
    assert call(rows=0, x=None, r=None, w=None, h=None) == 0


def test_output_refusals():
    _refused(_fwd(y=None), "KLP_EINVAL", "y must be")
    _refused(_fwd(sx=ODD), "KLP_EINVAL", "rstd_x")
    _refused(_fwd(xq=P), "KLP_EINVAL", "checkpoint")
    _refused(_fwd(hs=P), "KLP_EINVAL", "checkpoint")
    _refused(_fwd8(q=None), "KLP_EINVAL", "q must be")
    _refused(_fwd8(s=None), "KLP_EINVAL", "scales")


def test_backward_refusals():
    L = _lib().lib
    _refused(_bwd(rows=0), "KLP_EINVAL", "rows must be >= 1")
    _refused(_bwd(gy=None, gh=None), "KLP_EINVAL", "one of g_y and g_h")
    _refused(_bwd(dx=ODD), "KLP_EINVAL", "gradients aligned")
    _refused(_bwd(sh=None), "KLP_EINVAL", "rstd_h")
    _refused(_bwd(sx=None), "KLP_EINVAL", "rstd_x")
    _refused(_bwd(hq=P), "KLP_EINVAL", "h_scales")
    _refused(_bwd(hq=P, hs=P), "KLP_EINVAL", "x_codes")
    _refused(_bwd(hq=P, hs=P, xq=P), "KLP_EINVAL", "x_scales")
    _refused(_bwd(dw=ODD), "KLP_EINVAL", "aligned")
    need = L.klp_block_norm_bwd_workspace_bytes(100, 64, 1, 1, 100)
    assert need >= 3 * 64 * 4 and need % 4 == 0
    assert L.klp_block_norm_bwd_workspace_bytes(100, 64, 0, 0, 1) * 3 == need
    assert L.klp_block_norm_bwd_workspace_bytes(0, 64, 1, 1, 1) == 0
    assert L.klp_block_norm_bwd_workspace_bytes(4, 1 << 20, 1, 1, 1) == 0
    for kw in (dict(dw=P), dict(dp=P), dict(dg=P)):
        _refused(_bwd(rows=100, per=100, **kw), "KLP_EWORKSPACE", "workspace")
        _refused(_bwd(rows=100, per=100, **kw, ws=P, n=need - 1), "KLP_EWORKSPACE", "need")
        _refused(_bwd(rows=100, per=100, **kw, ws=ODD, n=need), "KLP_EWORKSPACE", "16-byte")


def test_python_refuses_cpu_tensors():
    import kernel_opt
    x = torch.zeros(2, 8)
    for f in (kernel_opt.fused_block_norm, kernel_opt.fused_block_norm_fp8):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            f(x, x, torch.ones(8))


def test_rows_per_gate():
    from kernel_opt.block import _rows_per_gate
    x = torch.zeros(3, 5, 7, 8)
    for shape, rows in (((8,), 105), ((3, 1, 1, 8), 35), ((3, 5, 1, 8), 7), ((3, 5, 7, 8), 1),
                        ((1, 1, 1, 8), 105), ((1, 5, 1, 8), None), ((3, 1, 7, 8), None),
                        ((5, 7, 8), None), ((3, 2, 1, 8), None)):
        assert _rows_per_gate(x, torch.zeros(shape)) == rows, shape
    assert _rows_per_gate(torch.zeros(1, 4, 8), torch.zeros(1, 1, 8)) == 4
    assert _rows_per_gate(torch.zeros(8), torch.zeros(8)) == 1
    assert _rows_per_gate(torch.zeros(0, 4, 8), torch.zeros(0, 1, 8)) == 4


def test_oracle_against_autograd():
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, res, w, p, gate, gy, gh = r(6, 20), r(6, 20), r(20), r(20), r(6, 20), r(6, 20), r(6, 20)
    for post in (None, p):
        t = [v.clone().requires_grad_() for v in (x, res, w, p, gate)]
        z = t[0]
        if post is not None:
            z = z * torch.rsqrt(z.square().mean(1, keepdim=True) + 1e-5) * t[3]
        h = t[1] + 0.3 * t[4] * z
        y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + 1e-5) * t[2]
        want = torch.autograd.grad((y, h), t, (gy, gh), allow_unused=True)
        n = [v.numpy() for v in (x, res, w, gate, gy, gh)]
        pn = None if post is None else p.numpy()
        ho, _ = block_oracle.forward(n[0], n[1], pn, n[3], 0.3, 1e-5)
        assert np.allclose(ho, h.detach().numpy())
        assert np.allclose(norm_oracle.forward(ho, n[2], 1e-5)[0], y.detach().numpy())
        got = block_oracle.backward(n[0], ho, block_oracle.rstd(n[0], 1e-5),
                                    block_oracle.rstd(ho, 1e-5), n[2], pn, n[3], 0.3, n[4], n[5],
                                    (1e-7, 1e-6, 6e-8))
        for k, v in zip(("x", "residual", "weight", "post", "gate"), want):
            if v is not None and k in got:
                assert np.allclose(got[k][0], v.numpy()), k
                assert (got[k][1] > 0).all()
