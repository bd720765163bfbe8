"""Refusals of the 8-bit product's epilogue that need no GPU."""
from __future__ import annotations

import ctypes

P = ctypes.c_void_p(0x10000)
ODD = ctypes.c_void_p(0x10001)


def _call(bias=None, bdt=0, act=0, cap=0.0, res=None, ldr=8, dt=0, m=4, n=8, k=64, out=P, ldo=8):
    from kernel_opt._library import lib
    return lib.klp_fp8_linear_act(P, k, P, P, k, P, m, n, k, bias, bdt, act, cap, res, ldr, dt,
                                  out, ldo, None)


def _refused(code, text, **kw):
    from kernel_opt import _library as L
    rc = _call(**kw)
    assert rc == getattr(L, code), (rc, L.last_error())
    assert text in L.last_error(), L.last_error()


def test_refusals():
    _refused("KLP_EDTYPE", "out dtype", dt=3)
    _refused("KLP_EDTYPE", "bias must be float32 or of out's dtype", bias=P, bdt=1)
    _refused("KLP_EDTYPE", "bias must be float32 or of out's dtype", bias=P, bdt=0, dt=2)
    _refused("KLP_EDTYPE", "bias must be float32 or of out's dtype", bias=P, bdt=7)
    _refused("KLP_EINVAL", "bias is not aligned", bias=ODD)
    _refused("KLP_EINVAL", "bias is not aligned", bias=ctypes.c_void_p(0x10002), bdt=2)
    for act in (-1, 5):
        _refused("KLP_EINVAL", f"unknown activation {act}", act=act)
    for cap in (0.0, -1.0, float("inf"), float("nan"), 2.0 ** -101, 2.0 ** 101):
        _refused("KLP_EINVAL", "cap must be within", act=4, cap=cap)
    _refused("KLP_EINVAL", "residual", res=ODD)
    _refused("KLP_EINVAL", "residual", res=P, ldr=-1)
    # What the plain product refuses.
    _refused("KLP_EINVAL", "k must be a positive multiple of 16", k=24)
    _refused("KLP_EINVAL", "out must be", out=None)
    _refused("KLP_EINVAL", "must not exceed", m=(1 << 20) + 1)
    assert _call(m=0, out=None, act=4, cap=2.0, bias=P) == 0


def test_python_refuses_before_any_launch():
    import pytest
    import torch
    import kernel_opt as ko
    x = torch.zeros(3, 32)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        ko.fp8_linear(x, x, x, x, bias=x[0], softcap=3.0)
    with pytest.raises(RuntimeError):
        ko.score_hidden(x, x[0], x, x, torch.zeros(3, dtype=torch.int64), alternatives=3)
