"""fused_top_logprobs where a row fits its workgroup's registers (4096 logits),
and next to that size, against the float64 oracle."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_top_gpu import DEV, DTYPES, IDS, _check, _ko, _logits

pytestmark = pytest.mark.gpu

# Around the sizes at which a row takes one wave more, odd ends, fewer logits
# than alternatives.
SIZES = [1, 2, 15, 16, 17, 63, 64, 65, 255, 257, 511, 1000, 1023, 1024, 1025, 1031, 2047, 2048,
         2049, 4095, 4096, 4097, 4103, 8185, 8191, 8192, 8193, 8200]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("vocab", SIZES)
def test_sizes(vocab, dtype):
    x, t = _logits(5, vocab, dtype, vocab)
    for k in (1, 3, 20, 64, 65, 128, 256):
        print(f"short {vocab} k={k} {dtype}", flush=True)
        out = _ko().fused_top_logprobs(x.to(DEV), t.to(DEV), k, 0.9)
        _check(out, x, t, k, 0.9)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("vocab", [9, 700, 1025, 3001, 8190])
def test_alignments_and_strides(vocab, dtype):
    """Rows that start at every element of a 16-byte vector, and rows with gaps
    between them: the outputs of dense ones, but for the order of the sums."""
    ko = _ko()
    x, t = _logits(9, vocab, dtype, 7)
    for off in range(0, 16 // x.element_size()):
        buf = torch.full((9 * vocab + 64,), float("nan"), dtype=dtype, device=DEV)
        flat = buf[off:off + 9 * vocab].view(9, vocab)
        flat.copy_(x)
        print(f"offset {off} {vocab} {dtype}", flush=True)
        _check(ko.fused_top_logprobs(flat, t.to(DEV), 20), x, t, 20)
    wide = torch.full((3, 4, vocab), float("nan"), dtype=dtype, device=DEV)
    wide[:, :3].copy_(x.view(3, 3, vocab))
    out = ko.fused_top_logprobs(wide[:, :3], t.view(3, 3).to(DEV), 20)
    _check([o.reshape(9, *o.shape[2:]) for o in out], x, t, 20)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("vocab", [30, 1001, 2047, 4090, 8187])
def test_equal_masked_and_infinite(vocab, dtype):
    """Lists that overflow, rows of few finite logits, the target among the
    masked ones and in the row's last, partial vector; rows without a
    distribution."""
    ko = _ko()
    g = torch.Generator().manual_seed(vocab)
    low = torch.finfo(dtype).min
    base = torch.randn(vocab, generator=g)
    few = torch.full((vocab,), -float("inf"))
    few[::max(vocab // 10, 1)] = base[::max(vocab // 10, 1)]
    mask = torch.full((vocab,), low)
    mask[1] = 0.5
    rows = [torch.zeros(vocab), torch.randint(0, 3, (vocab,), generator=g).float(), few, mask,
            torch.arange(vocab) / vocab, -torch.arange(vocab) / vocab,
            torch.where(torch.arange(vocab) % 16 < 2, 5 + base, base - 30)]
    x = torch.stack([r.to(dtype) for r in rows])
    for at in (0, vocab // 2, vocab - 1, vocab - 3):
        t = torch.full((len(rows),), at)
        for k in (1, 20, 65, 256):
            print(f"short special {vocab} {dtype} target {at} k={k}", flush=True)
            _check(ko.fused_top_logprobs(x.to(DEV), t.to(DEV), k), x, t, k)
    bad = torch.stack([base, base, torch.full((vocab,), -float("inf")), base]).to(dtype)
    bad[0, vocab - 1] = float("nan")
    bad[1, vocab // 2] = float("inf")
    lp, ent, lse, rank, ids, top = ko.fused_top_logprobs(
        bad.to(DEV), torch.tensor([0, 1, 2, -100], device=DEV), 5)
    assert lp[:3].isnan().all() and ent[:3].isnan().all() and lse[:2].isnan().all()
    assert lse[2] == -float("inf") and (ids[:3] == -1).all() and top[:2].isnan().all()
    assert (rank[:2] == -1).all() and rank[3] == -1 and float(lp[3]) == -float(lse[3])


def test_many_rows_and_gradients():
    """More rows than run at once; the gradient of the listed alternatives sums
    to the softmax's, row by row."""
    ko = _ko()
    x, t = _logits(9000, 700, torch.bfloat16, 1)
    leaf = x.to(DEV).requires_grad_()
    out = ko.fused_top_logprobs(leaf, t.to(DEV), 20)
    pick = torch.arange(0, 9000, 997)
    _check([o[pick.to(DEV)] for o in out], x[pick], t[pick], 20)
    out[5].sum().backward()
    p = torch.softmax(x.double(), -1)
    want = -20 * p
    want.scatter_add_(1, out[4].cpu(), torch.ones(9000, 20, dtype=torch.float64))
    # A bf16 rounding of each element, and float32's of p and of the sum before.
    err = (leaf.grad.double().cpu() - want).abs()
    assert bool((err <= 2.0 ** -8 * want.abs() + 2.0 ** -16 * (20 * p + 1)).all())
    assert np.isfinite(float(err.max()))
