"""Where sample_scores' border falls: temperatures so small that nothing but the largest score has weight."""
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
