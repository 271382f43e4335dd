"""Where sample_scores' border falls: temperatures so small that nothing but the largest score has weight, ties that top-k cuts, and top-p
borders deep in a light tail, where a sum that drops the low bits of its terms moves the border by whole entries."""
import math
from fractions import Fraction

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


def _border(N, gap, cut):
    """one score of 0, N - 1 of -gap, a top-p that cuts off about cut N of those: (p, how many of the N - 1 stay, the draw for u,
    u), counted in rationals.  j of them stay while 1 + (j - 1) w < p (1 + (N - 1) w); the draw for u is the index (the score of 0 is
    index 0) of the first entry behind u (1 + t w)"""
    w = Fraction(math.exp(-gap))                                   # (2^-53 of itself)
    p = float(1 - Fraction(cut) * N * w)
    u = 1 - 2.0 ** -24
    border = (Fraction(p) * (1 + (N - 1) * w) - 1) / w
    t = math.ceil(border)
    n = (Fraction(u) * (1 + t * w) - 1) / w
    # a weight is a multiple of 2^-57, rounded down, of a double: w is off by 2^-57 + 2^-51 w; sums, products and the total are doubles
    wrong = float((1 - Fraction(p)) / w) * (2.0 ** -57 / float(w) + 2.0 ** -51) + 2.0 ** -50 * N + 2.0 ** -51 / float(w)
    for v in (border, n):
        assert min(v - math.floor(v), math.ceil(v) - v) > wrong, (N, gap, cut, float(v), wrong)
    assert 0 < n < t < N
    return p, t, math.floor(n) + 1, u


TAILS = [(20_000, 20.5, 0.4), (32_000, 23.0, 0.3), (60_000, 22.5, 0.35), (200_000, 22.0, 0.6), (1_000_000, 20.0, 0.48), (1_000_000, 22.0, 0.36), (4_000_000, 20.0, 0.12),
         (3_000_001, 21.5, 0.3)]


def test_the_tails_borders_are_not_in_question():
    for c in TAILS:
        _border(*c)


@pytest.mark.gpu
@pytest.mark.parametrize("N,gap,cut", TAILS)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("with_k", [False, True])
def test_a_border_in_a_light_tail(N, gap, cut, dtype, with_k):
    """with_k: behind a top-k that takes off a few lighter entries"""
    from unirec_amd import ops
    p, t, index, u = _border(N, gap, cut)
    x = torch.full((2, N + (5 if with_k else 0)), -gap)            # (multiples of 1/2: exact in every type)
    x[:, 0] = 0.0
    x[:, N:] = -gap - 0.5
    x = x.to(getattr(torch, dtype)).cuda()
    i, logp = ops.sample_scores(x, torch.full((2, 1), u, device="cuda"), top_p=p, top_k=N if with_k else 0)
    assert i.flatten().tolist() == [index] * 2, (i, index, t)
    want = -gap - math.log1p(t * math.exp(-gap))
    assert (logp.double() - want).abs().max() <= 2.0 ** -23 * abs(want)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [128, 129, 3000, 32_768, 65_536, 300_000, 2_000_001])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_sums_of_many_whole_weights(N, dtype):
    """flat rows: N weights of 1 (2^57 each: more than 64 bits hold from 128 on), and a half of them one step lower"""
    g = torch.Generator().manual_seed(N)
    x = torch.full((3, N), 2.0)
    x[1, ::2] = 1.0
    x[2] = torch.where(torch.rand(N, generator=g) < 0.01, 2.0, 2.0 - 2.0 ** -8)
    u = torch.rand(3, 4, generator=g)
    u[:, 0], u[:, 1] = 0.0, 1 - 2.0 ** -24
    for f in (dict(p=0.5), dict(p=0.3), dict(p=0.75, T=0.5), dict(k=N - 1, p=0.625), dict(k=(N + 1) // 2, p=0.99, T=3.0)):
        _check(x.to(getattr(torch, dtype)), u, **f)


@pytest.mark.gpu
def test_a_top_k_beyond_32_bits():
    from unirec_amd import _lib, ops
    x, u = (t.cuda() for t in _scores(4, 300, 32))
    want = ops.sample_scores(x, u)
    for k in (300, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, 10 ** 30):
        got = ops.sample_scores(x, u, top_k=k)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), k
    for k in (-1, -2 ** 31, -2 ** 32 + 5):
        with pytest.raises(_lib.UnirecAmdError):
            ops.sample_scores(x, u, top_k=k)
