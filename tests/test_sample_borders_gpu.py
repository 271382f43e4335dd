"""Where sample_scores' border falls: temperatures so small that nothing but the largest score has weight, and ties that top-k cuts."""
import math

import pytest
import torch
from test_sample_gpu import _check, _scores


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 700, 5000, 40_000, 70_001, 150_000])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_temperatures_close_to_zero(N, dtype):
    """0 < T: the largest scores share the weight however small T is (T = 0: the first of them)"""
    x, u = _scores(5, N, 31, getattr(torch, dtype))
    x[0, N // 2:] = 6.5                                           # a tie of the largest
    x[4, N // 3] = math.inf
    for T in (5e-324, 1e-305, 1e-300, 1.0000000001e-300, 1e-299, 1e-45, 1e-38, 1e-12):
        _check(x, u, T=T)
    for f in (dict(k=3), dict(p=0.4), dict(m=0.5), dict(k=N // 2 + 1, p=0.7, m=1e-3)):
        _check(x, u, T=1e-305, **f)


TIE_FILTERS = [dict(p=0.9999), dict(p=0.99, T=3.0), dict(p=1 - 2.0 ** -40), dict(p=0.5), dict(p=0.9999, m=0.01)]


def _ties(N, dtype):
    """three values; a top-k that ends inside the first, the second and the third of them, at its first and at its last entry"""
    g = torch.Generator().manual_seed(N)
    kind = torch.randint(0, 3, (3, N), generator=g)
    kind[0] = 0                                                   # one value
    x = torch.tensor([1.5, 1.0, -0.5])[kind]
    u = torch.rand(3, 6, generator=g)
    u[:, 0], u[:, 1] = 0.0, 1 - 2.0 ** -24
    n = [(kind == v).sum(1) for v in range(3)]
    ks = [n[0] // 2, n[0] + n[1] // 2, n[0] + n[1] + n[2] // 3, n[0] + 1, torch.clamp(n[0] - 1, min=1), n[0]]
    return x.to(getattr(torch, dtype)), u, [k.to(torch.int32) for k in ks]


@pytest.mark.gpu
@pytest.mark.parametrize("N", [5, 64, 128, 129, 700, 4001, 20_000, 33_000, 70_001, 200_000])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_top_p_behind_a_top_k_that_cuts_a_tie(N, dtype):
    """of the ties that top-k left, top-p takes some, or leaves them all: those that top-k cut do not come back"""
    x, u, ks = _ties(N, dtype)
    for k in ks:
        for f in TIE_FILTERS:
            _check(x, u, k=torch.clamp(k, min=1), **f)
    for f in TIE_FILTERS:
        _check(x, u, k=max(1, N // 2), **f)
