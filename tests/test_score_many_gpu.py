"""score_hidden over more tokens than one product of the 8-bit head takes (a
small vocabulary, so that all their logits fit the default chunk)."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
MOST = 2 ** 20  # rows of one fp8_linear


def test_score_more_tokens_than_a_product_takes():
    import kernel_opt as ko
    g = torch.Generator(device=DEV).manual_seed(2)
    n, dim, vocab = MOST + 5, 16, 24
    x = torch.randn(n, dim, generator=g, device=DEV).to(torch.bfloat16)
    nw = torch.ones(dim, device=DEV, dtype=torch.bfloat16)
    head, hs = ko.quantize_fp8(torch.randn(vocab, dim, generator=g, device=DEV), block_rows=128)
    t = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    parts = [ko.score_hidden(x[i:i + MOST], nw, head, hs, t[i:i + MOST]) for i in (0, MOST)]
    # The last few tokens' own product may add K in another order; one block of
    # 16 has the same sums however many tokens there are.
    for chunk in (None, n, 700001):
        got = ko.score_hidden(x, nw, head, hs, t, chunk_tokens=chunk)
        assert all(torch.equal(a, torch.cat(b)) for a, b in zip(got, zip(*parts)))


def test_a_product_says_how_many():
    import kernel_opt as ko
    q, s = ko.quantize_fp8(torch.zeros(MOST + 1, 16, device=DEV))
    w, ws = ko.quantize_fp8(torch.ones(8, 16, device=DEV), block_rows=128)
    with pytest.raises(RuntimeError, match="must not exceed"):
        ko.fp8_linear(q, s, w, ws)
    assert ko.fp8_linear(q[:MOST], s[:MOST], w, ws).shape == (MOST, 8)
