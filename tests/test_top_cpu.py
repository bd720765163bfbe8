"""The C entry points of the log-probabilities with alternatives refuse bad
arguments with the documented status and message before touching the GPU, and
the oracle agrees with independent statements.  No compute call is made."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import top_oracle

P = ctypes.c_void_p(0x10000)
ODD = ctypes.c_void_p(0x10004)


def _lib():
    from kernel_opt import _library
    return _library


def _refused(rc, status, text):
    L = _lib()
    assert rc == getattr(L, status), (rc, L.last_error())
    assert text in L.last_error(), L.last_error()


def _fwd(x=P, dtype=0, n=4, v=64, inner=4, so=0, si=64, t=P, T=1.0, k=5, lp=P, ent=P, lse=P, rank=P,
         ids=P, top=P, ws=None, ws_bytes=0):
    return _lib().lib.klp_fwd_top(x, dtype, n, v, inner, so, si, t, T, k, lp, ent, lse, rank, ids,
                                  top, ws, ws_bytes, None)


def _bwd(x=P, dtype=0, n=4, v=64, inner=4, so=0, si=64, t=P, T=1.0, k=5, ids=P, lse=P, ent=P, gl=P,
         ge=None, gs=None, gt=P, d=P):
    return _lib().lib.klp_bwd_top(x, dtype, n, v, inner, so, si, t, T, k, ids, lse, ent, gl, ge, gs,
                                  gt, d, None)


@pytest.mark.parametrize("call", [_fwd, _bwd], ids=["forward", "backward"])
def test_refusals(call):
    _refused(call(dtype=7), "KLP_EDTYPE", "dtype")
    _refused(call(x=None), "KLP_EINVAL", "non-null")
    _refused(call(t=ODD), "KLP_EINVAL", "8-byte")
    _refused(call(v=0), "KLP_EINVAL", "vocab")
    _refused(call(v=2 ** 26 + 1, si=2 ** 26 + 1), "KLP_EINVAL", "2^26")
    _refused(call(n=2 ** 23), "KLP_EINVAL", "too many rows")
    for k in (0, 257, -3):
        _refused(call(k=k), "KLP_EINVAL", "k must be in [1, 256]")
    for T in (0.0, -1.0, float("nan"), float("inf")):
        _refused(call(T=T), "KLP_EINVAL", "temperature")
    _refused(call(ent=None), "KLP_EINVAL", "entropy")
    _refused(call(lse=ctypes.c_void_p(0x10002)), "KLP_EINVAL", "lse")
    _refused(call(ids=ODD), "KLP_EINVAL", "top_ids")
    assert call(n=0, x=None) == 0
    L = _lib()
    L.lib.klp_debug_fail_next_launches(1)
    try:
        _refused(call(), "KLP_ELAUNCH", "injected")
    finally:
        L.lib.klp_debug_fail_next_launches(0)


def test_output_refusals():
    _refused(_fwd(lp=None), "KLP_EINVAL", "logprob")
    _refused(_fwd(rank=None), "KLP_EINVAL", "rank")
    _refused(_fwd(top=None), "KLP_EINVAL", "top_logprob")
    _refused(_bwd(d=None), "KLP_EINVAL", "d_logits")
    _refused(_bwd(gt=ctypes.c_void_p(0x10002)), "KLP_EINVAL", "g_top")
    _refused(_bwd(ids=None), "KLP_EINVAL", "top_ids")


def test_workspace():
    L = _lib().lib
    need = L.klp_fwd_top_workspace_bytes(0, 2, 152064, 20)
    assert need > 8192
    assert L.klp_fwd_top_workspace_bytes(0, 4096, 152064, 20) == 0
    assert L.klp_fwd_top_workspace_bytes(0, 2, 512, 20) == 0
    for bad in ((9, 2, 152064, 20), (0, 0, 152064, 20), (0, 2, 0, 20), (0, 2, 152064, 0),
                (0, 2, 152064, 257)):
        assert L.klp_fwd_top_workspace_bytes(*bad) == 0
    big = dict(n=2, v=152064, inner=2, si=152064, k=20)
    _refused(_fwd(**big, ws=P, ws_bytes=need - 1), "KLP_EWORKSPACE", "need")
    _refused(_fwd(**big, ws=ODD, ws_bytes=need), "KLP_EWORKSPACE", "16-byte")
    # Every split's pieces have their keys, whatever k.
    for n in (1, 2, 7, 64, 128):
        for k in (1, 20, 64, 256):
            b = L.klp_fwd_top_workspace_bytes(2, n, 262144, k)
            assert b == 0 or (b - 8192) % (n * (16 + 8 * k)) == 0
            if b:
                splits = (b - 8192) // (n * (16 + 8 * k))
                assert splits >= 2 and splits * k <= 4096 and n * splits <= 256


def test_python_refuses_cpu_tensors():
    import kernel_opt
    with pytest.raises(RuntimeError, match="GPU tensors"):
        kernel_opt.fused_top_logprobs(torch.zeros(2, 4), torch.zeros(2, dtype=torch.int64), 1)


def test_oracle_against_torch():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 40, generator=g, dtype=torch.float64).requires_grad_()
    T = 0.75
    lsm = torch.log_softmax(x / T, 1)
    ent = -(lsm.exp() * lsm).sum(1)
    lse = torch.logsumexp(x / T, 1)
    top, ids = torch.topk(lsm, 6, dim=1)
    t = torch.tensor([3, 39, 0])
    grads = [torch.randn(3, generator=g, dtype=torch.float64) for _ in range(3)]
    gt = torch.randn(3, 6, generator=g, dtype=torch.float64)
    loss = (lsm.gather(1, t[:, None])[:, 0] * grads[0] + ent * grads[1] + lse * grads[2]).sum() \
        + (top * gt).sum()
    d, = torch.autograd.grad(loss, x)
    for i in range(3):
        row = x[i].detach().numpy()
        got = top_oracle.forward_row(row, int(t[i]), 6, T)
        assert np.allclose(got[0], lsm[i, t[i]].item()) and np.allclose(got[1], ent[i].item())
        assert np.allclose(got[2], lse[i].item()) and (got[4] == ids[i].numpy()).all()
        assert got[3] == int((lsm[i] > lsm[i, t[i]]).sum())
        assert np.allclose(got[5], top[i].detach().numpy())
        dx, size = top_oracle.backward_row(row, int(t[i]), got[4], T,
                                           *(float(v[i]) for v in grads), gt[i].numpy())
        assert np.allclose(dx, d[i].numpy()) and (size >= np.abs(dx) - 1e-12).all()


def test_oracle_by_hand():
    inf = float("inf")
    got = top_oracle.forward_row([0.0, 1.0, 1.0, -inf], 2, 4)
    assert got[3] == 1 and got[4].tolist() == [1, 2, 0, -1] and got[5][3] == -inf
    assert top_oracle.forward_row([0.0, 0.0], -100, 1)[3] == -1
    assert top_oracle.forward_row([-inf, -inf], 1, 1)[2:4] == (-inf, 1)
    assert np.isnan(top_oracle.forward_row([inf, 0.0], 1, 1)[0])
