"""fused_top_logprobs over finite logits so large that the offset of a row's sums,
max log2(e) / T, is rounded by more than an exponent: masks with a finite fill, tiny
temperatures; against the float64 oracle with the bounds of test_top_gpu."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import top_oracle
from test_top_gpu import U, _check_row, _sum_error, np64

pytestmark = pytest.mark.gpu
DEV = "cuda"
# A row in registers, rows of a workgroup, a row in pieces.
SHAPES = [(2, 700), (300, 9001), (1, 140001)]


def _run(x, t, k, T):
    import kernel_opt
    print(f"far {tuple(x.shape)} {x.dtype} {float(x.min())} T={T}", flush=True)
    return [o.cpu().numpy() for o in kernel_opt.fused_top_logprobs(x.to(DEV), t.to(DEV), k, T)]


@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("T", [1.46, 1.5, 2.0, 2.5, 2.9])
def test_rows_of_the_lowest_value_at_a_temperature(T, rows, vocab):
    """The offset does not overflow here, and its rounding is of any sign."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.full((rows, vocab), torch.finfo(torch.float32).min)
    t = torch.randint(0, vocab, (rows,), generator=g)
    out = _run(x, t, 20, T)
    for i in range(min(rows, 3)):
        _check_row([o[i] for o in out], np64(x[i]), int(t[i]), 20, T)
