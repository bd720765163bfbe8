"""fused_sample's parameters given as numbers: every documented way to turn a
filter off gives what None gives, every other value outside its range raises."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs():
    g = torch.Generator(device=DEV).manual_seed(7)
    return (3 * torch.randn(20, 5003, generator=g, device=DEV),
            torch.rand(20, generator=g, device=DEV))


@pytest.mark.parametrize("other", [{}, dict(top_p=0.8), dict(min_p=0.05)], ids=["none", "p", "m"])
def test_off(other):
    from kernel_opt import fused_sample
    x, u = _inputs()
    want = fused_sample(x, u, 0.9, **other)
    for k in (0, -1, -7, -2 ** 31, -2 ** 40, 5003, 10 ** 6, 2 ** 31 - 1, 2 ** 31, 2 ** 40, -1.0):
        got = fused_sample(x, u, 0.9, top_k=k, **other)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k
    for off in (dict(top_p=1.0), dict(min_p=0.0)):
        if not off.keys() & other.keys():
            got = fused_sample(x, u, 0.9, **off, **other)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), off


def test_the_same_as_numbers_and_tensors():
    from kernel_opt import fused_sample
    x, u = _inputs()
    for k in (-3, 0, 1, 17, 5002, 5003, 2 ** 40):
        a = fused_sample(x, u, 0.7, top_k=k)
        b = fused_sample(x, u, 0.7, top_k=torch.full((20,), k, device=DEV))
        assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
        assert ((a[1] - b[1]).abs() <= 40 * 2.0 ** -24 * (1 + a[1].abs())).all()


@pytest.mark.parametrize("name,value", [
    ("top_k", math.inf), ("top_k", -math.inf), ("top_k", math.nan), ("top_k", True),
    ("top_k", 0.5), ("top_p", -0.1), ("top_p", 1.0001), ("top_p", math.nan), ("min_p", 1.5),
    ("min_p", -1e-9), ("min_p", math.inf), ("temperature", -1e-9), ("temperature", math.inf)])
def test_refused(name, value):
    from kernel_opt import fused_sample
    x, u = _inputs()
    with pytest.raises(ValueError, match=name):
        fused_sample(x, u, **{name: value})
