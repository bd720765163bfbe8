"""fused_block_norm over rows that do not start at multiples of 16 bytes: the bits
of the same rows where they do, and every width around the kernels' shapes
against the oracle."""
from __future__ import annotations

import pytest
import torch

from test_block_gpu import (DEV, DTYPES, IDS, _check_grads, _check_h, _check_y, _data, _run)

pytestmark = pytest.mark.gpu


def _ko():
    import kernel_opt
    return kernel_opt


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("dim", [64, 520, 1024, 2040, 4096, 8192, 9000])
def test_the_bits_of_aligned_rows(dim, dtype):
    """The same values one element further in memory and with a row stride of
    their own; gradients of one output alone too."""
    ko = _ko()
    rows = 37
    g = torch.Generator(device=DEV).manual_seed(dim)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)  # noqa: E731
    x, res, gate = r(rows, dim), r(rows, dim), r(dim)
    w, post = 1 + 0.1 * r(dim), 1 + 0.1 * r(dim)

    def moved(t):
        wide = torch.full((*t.shape[:-1], dim + 3), float("nan"), dtype=t.dtype, device=DEV)
        wide[..., 1:dim + 1] = t
        return wide[..., 1:dim + 1]

    for wt in (dtype, torch.float32):
        for checkpoint in (None, "fp8"):
            for outs in ((0, 1), (0,), (1,)):
                print(f"moved {dim} {dtype} {wt} {checkpoint} {outs}", flush=True)
                got = []
                for f in (lambda t: t, moved):
                    leaves = [f(t).detach().requires_grad_()
                              for t in (x, res, w.to(wt), post.to(wt), gate.to(wt))]
                    o = ko.fused_block_norm(leaves[0], leaves[1], leaves[2], post_weight=leaves[3],
                                            gate=leaves[4], scale=0.7, checkpoint=checkpoint)
                    got.append((*[v.detach() for v in o],
                                *torch.autograd.grad([o[i] for i in outs], leaves,
                                                     [f((res, x)[i]) for i in outs])))
                assert all(torch.equal(a, b) for a, b in zip(*got))
        got = [ko.fused_block_norm_fp8(f(x), f(res), f(w.to(wt)), post_weight=f(post.to(wt)),
                                       gate=f(gate.to(wt))) for f in (lambda t: t, moved)]
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(*got))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("dim", [1, 7, 9, 511, 513, 519, 521, 1023, 1025, 2047, 2055, 4095, 4097,
                                 8191, 8193, 16383])
def test_widths(dim, dtype):
    for gate, kept in (("sequence", None), ("channel", "fp8")):
        print(f"width {dim} {dtype} {gate} {kept}", flush=True)
        d, gy, gh = _data(3, 5, dim, dtype, dim, gate, True)
        for one in (gy, None):
            y, h, grads = _run(d, one, gh, 0.7, kept)
            _check_h(h, d, 0.7, dim, dtype)
            _check_y(y, h, d["weight"], dtype)
            if one is not None:
                _check_grads(grads, d, h, 0.7, one, gh, dtype, kept)
