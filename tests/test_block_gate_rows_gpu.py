"""One gate for all rows through the C entries: any count of rows a gate from the
rows' own up, beyond 32 bits too."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("per_gate", [70, 71, 2 ** 32 - 1, 2 ** 32, 2 ** 32 + 3, 2 ** 63 - 1])
def test_one_gate_of_any_count(per_gate):
    import kernel_opt as ko
    from kernel_opt._library import check_status, lib, ptr, stream_handle
    rows, dim = 70, 200
    g = torch.Generator(device=DEV).manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    x, res, w, gate = (v.requires_grad_() for v in (r(rows, dim), r(rows, dim), r(dim), r(dim)))
    y, h = ko.fused_block_norm(x, res, w, gate=gate, scale=0.5)
    g_y, g_h = r(rows, dim), r(rows, dim)
    want = torch.autograd.grad((y, h), (x, res, w, gate), (g_y, g_h))
    y2, h2, dx, dr = (torch.full((rows, dim), -7.0, device=DEV) for _ in range(4))
    sx, sh = (torch.empty(rows, device=DEV) for _ in range(2))
    dw, dg = (torch.empty(dim, device=DEV) for _ in range(2))
    st = stream_handle(0)
    check_status(lib.klp_block_norm(ptr(x.detach()), 2, dim, ptr(res.detach()), dim, None,
                                    ptr(w.detach()), 2, ptr(gate.detach()), 2, per_gate, 0.5, rows,
                                    dim, 1e-6, ptr(y2), ptr(h2), ptr(sx), ptr(sh), None, None, None,
                                    None, st))
    assert torch.equal(y2, y) and torch.equal(h2, h)
    nbytes = lib.klp_block_norm_bwd_workspace_bytes(rows, dim, 0, 1, per_gate)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    check_status(lib.klp_block_norm_bwd(
        ptr(x.detach()), 2, dim, None, None, ptr(h2), None, None, None, ptr(w.detach()), 2,
        ptr(gate.detach()), 2, per_gate, 0.5, None, ptr(sh), ptr(g_y), ptr(g_h), rows, dim, ptr(dx),
        ptr(dr), None, ptr(dw), ptr(dg), ptr(ws), nbytes, st))
    assert all(torch.equal(a, b) for a, b in zip((dx, dr, dw, dg), want))
