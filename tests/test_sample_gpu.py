"""Sampling from scores (unirec_amd.ops.sample_scores) against the definition in 64 bits: indices are equal, the log-probability is a 64-bit
value rounded once to fp32 (half a step, 2^-24 of it, and as much again where the double sums round differently)."""
import math

import numpy as np
import pytest
import torch


def _reference(x, u, T, k, p, m):
    """one row: x float64 [N], u [S] -> (index, log-probability)"""
    N = len(x)
    x = np.where(np.isnan(x), -np.inf, x) + 0.0
    out_i, out_l = np.full(len(u), -1, np.int64), np.full(len(u), -np.inf)
    top = x.max()
    if top == -np.inf:
        return out_i, out_l
    if not T > 0:
        out_i[:], out_l[:] = int(np.argmax(x)), 0.0
        return out_i, out_l
    with np.errstate(invalid="ignore"):
        z = np.where(x == np.inf, 0.0, -np.inf) if top == np.inf else (x - top) / T
    order = np.argsort(-z, kind="stable")
    order = order[z[order] > -np.inf]
    if k > 0:
        order = order[:k]
    w = np.exp(z[order])
    if p < 1:
        c = np.cumsum(w)
        stay = np.concatenate([[0.0], c[:-1]]) < p * c[-1]
        stay[0] = True
        order, w = order[stay], w[stay]
    if m > 0:
        order = order[w >= min(m, 1.0)]
    keep = np.sort(order)
    c = np.cumsum(np.exp(z[keep]))
    at = np.searchsorted(c, np.clip(u.astype(np.float64), 0, 1 - 2.0 ** -24) * c[-1], side="right")
    return keep[at], z[keep[at]] - np.log(c[-1])


def _check(scores, rand, T=1.0, k=0, p=1.0, m=0.0, ids=None, dev=None):
    from unirec_amd import ops
    dev = dev if dev is not None else scores.cuda()
    t = [v.cuda() if torch.is_tensor(v) else v for v in (T, k, p, m)]
    got_i, got_l = ops.sample_scores(dev, rand.cuda(), *t, ids=None if ids is None else ids.cuda())
    assert got_i.shape == rand.shape and got_i.dtype == torch.int64 and got_l.dtype == torch.float32
    x, u = scores.double().numpy(), rand.reshape(rand.shape[0], -1).numpy()
    got_i, got_l = got_i.cpu().reshape(u.shape), got_l.cpu().reshape(u.shape)
    for b in range(x.shape[0]):
        v = [float(a[b]) if torch.is_tensor(a) else a for a in (T, k, p, m)]
        i, lp = _reference(x[b], u[b], v[0], int(v[1]), v[2], v[3])
        if ids is not None:
            i = np.where(i >= 0, ids[b].numpy()[i], -1)
        assert (got_i[b].numpy() == i).all(), (b, v, got_i[b], i)
        fin = np.isfinite(lp)
        assert (got_l[b].numpy()[~fin] == lp[~fin]).all()
        assert (np.abs(got_l[b].double().numpy()[fin] - lp[fin]) <= 2.0 ** -23 * np.abs(lp[fin]) + 1e-12).all()
    return got_i, got_l


def _scores(B, N, seed, dtype=torch.float32, masked=0.05, spread=2.0):
    g = torch.Generator().manual_seed(seed * 7919 + B * 31 + N)
    x = torch.randn(B, N, generator=g) * spread
    x[torch.rand(B, N, generator=g) < masked] = -math.inf
    if B > 3:
        x[2] = -math.inf
    return x.to(dtype), torch.rand(B, 3, generator=g)


# ------------------------------------------------------------------------------------------------ refusals (CPU)
def test_refusals():
    from unirec_amd import _lib, ops
    x, u = _scores(3, 10, 0)
    with pytest.raises(_lib.UnirecAmdError, match="GPU tensor"):
        ops.sample_scores(x, u)
    with pytest.raises(_lib.UnirecAmdError):
        ops.sample_scores(x.double(), u)
    one = 1 << 20

    def call(t=0, n=8, ld=8, B=2, S=1, T=1.0, k=0, p=1.0, m=0.0, scores=one, ids=None, ld_ids=8, ws=one):
        return _lib.lib.ur_sample_scores(scores, t, n, ld, B, one, S, T, k, p, m, None, None, None, None, ids, ld_ids, one, one, ws, None)

    for bad in (dict(t=3), dict(n=0), dict(ld=7), dict(B=0), dict(S=0), dict(T=-1.0), dict(T=math.nan), dict(T=math.inf), dict(k=-1), dict(p=0.0),
                dict(p=math.nan), dict(m=-0.1), dict(m=1.5), dict(m=math.nan), dict(scores=None), dict(ids=one, ld_ids=3),
                dict(n=1 << 20, ld=1 << 20, ws=None)):
        assert call(**bad) == -1, bad
        assert b"ur_sample_scores" in _lib.lib.ur_last_error()
    assert _lib.lib.ur_sample_scores_workspace_bytes(0, 0, 4) < 0 and _lib.lib.ur_sample_scores_workspace_bytes(9, 100, 4) < 0
    assert _lib.lib.ur_sample_scores_workspace_bytes(0, 1000, 4) == 0 < _lib.lib.ur_sample_scores_workspace_bytes(0, 1 << 20, 4)


# ------------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
def test_refusals_on_tensors():
    from unirec_amd import _lib, ops
    x, u = (t.cuda() for t in _scores(4, 12, 0))
    for args, kw in (((x[0], u), {}), ((x.t(), u), {}), ((x, u[:3]), {}), ((x, u.double()), {}), ((x, u[:, :0]), {}), ((x[:, :0], u), {}),
                     ((x, u), dict(temperature=-1.0)), ((x, u), dict(top_p=0.0)), ((x, u), dict(ids=torch.zeros(4, 11, dtype=torch.int64, device="cuda"))),
                     ((x, u), dict(top_k=torch.zeros(4, device="cuda"))), ((x, u), dict(top_p=torch.ones(3, device="cuda"))), ((x.expand(4, 12)[:1].expand(4, 12), u), {})):
        with pytest.raises(_lib.UnirecAmdError):
            ops.sample_scores(*args, **kw)


FILTERS = [dict(), dict(T=0.6), dict(k=5), dict(p=0.8), dict(m=0.05), dict(T=1.4, k=40, p=0.9, m=0.01), dict(k=1), dict(p=1e-6), dict(m=1.0), dict(T=0.0),
           dict(k=100000), dict(T=1e-4), dict(T=50.0, p=0.5)]


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 2, 3, 31, 64, 65, 255, 256, 257, 1000, 1024, 1025, 4097])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_against_the_definition(N, dtype):
    x, u = _scores(6, N, 1, getattr(torch, dtype))
    for f in FILTERS:
        _check(x, u, **f)


@pytest.mark.gpu
@pytest.mark.parametrize("B,N", [(3, 16384), (2, 16385), (5, 32769), (2, 70_001), (300, 8200), (1, 1_200_003)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_long_rows(B, N, dtype):
    x, u = _scores(B, N, 2, getattr(torch, dtype))
    for f in (dict(T=0.8), dict(p=0.9), dict(k=777, p=0.95, T=1.3), dict(m=0.02), dict(k=N // 3), dict(T=0.7, p=0.5, m=1e-4), dict(T=0.0)):
        _check(x, u, **f)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [50, 1000, 20_000, 100_000])
def test_ties_stay_in_index_order(N):
    g = torch.Generator().manual_seed(N)
    x = torch.randint(-2, 3, (4, N), generator=g).float()         # five values, every border falls inside a tie
    x[1] = 1.25                                                   # one value
    x[2, ::2], x[2, 1::2] = 0.0, -0.0                             # two zeros, one score
    u = torch.rand(4, 5, generator=g)
    u[:, 0], u[:, 1] = 0.0, 1 - 2.0 ** -24
    for f in (dict(), dict(k=N // 2), dict(k=7), dict(p=0.5), dict(p=0.37), dict(k=N // 3, p=0.5), dict(m=0.3), dict(k=N // 2, p=0.75, m=0.1), dict(T=0.0), dict(T=1e30, p=0.5)):
        _check(x, u, **f)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [60, 5000, 40_000, 70_001])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_a_border_right_below_zero(N, dtype):
    """zeros of both signs are one tie, and all of them stay where the border lies below them"""
    g = torch.Generator().manual_seed(N)
    kind = torch.randint(0, 4, (2, N), generator=g)
    x = torch.tensor([1.0, 0.0, -0.0, -0.5]).to(getattr(torch, dtype))[kind]
    u = torch.rand(2, 40, generator=g)
    kept = (kind < 3).sum(1).to(torch.int32)
    _check(x, u, T=0.7, k=kept)
    _check(x, u, T=0.7, k=kept, p=0.999)                         # (the last of the zeros go)
    one, rest = (kind == 0).sum(1).double(), (kind == 3).sum(1).double()
    zero = N - one - rest
    w = [math.exp(-1 / 0.7), math.exp(-1.5 / 0.7)]
    p = (one + w[0] * zero + 0.3 * w[1]) / (one + w[0] * zero + w[1] * rest)
    _check(x, u, T=0.7, p=float(p[0]), m=0.0)
    _check(x, u, T=0.7, m=0.2)                                   # exp(-1 / 0.7) = 0.24 stays, exp(-1.5 / 0.7) = 0.12 goes


@pytest.mark.gpu
@pytest.mark.parametrize("N", [40, 3000, 50_000])
def test_infinities_nan_and_empty_rows(N):
    x, u = _scores(9, N, 3, masked=0.0)
    x[0] = -math.inf
    x[1] = math.nan
    x[2] = torch.randn(N)
    x[2, 3], x[2, 7] = math.inf, math.inf                         # among those two
    x[3, ::3] = math.nan
    x[4] = torch.finfo(torch.float32).min                         # masked by the type's lowest value, all of it: a flat row
    x[5, 1:] = torch.finfo(torch.float32).min
    x[6], x[6, N - 1] = -math.inf, -3.0e38                        # one entry, far down
    x[7, :] = torch.linspace(-1e-30, 1e-30, N)                    # denormal differences
    for f in (dict(), dict(k=2), dict(p=0.6), dict(m=0.2), dict(k=N // 2, p=0.9, m=0.001), dict(T=0.0), dict(T=3e38)):
        _check(x, u, **f)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [300, 60_000])
def test_a_value_for_every_row(N):
    x, u = _scores(8, N, 4)
    T = torch.tensor([1.0, 0.5, 2.0, 0.0, 1.0, -1.0, 1.3, 0.9])
    k = torch.tensor([0, 5, N // 2, 3, 1, 9, -4, N + 9], dtype=torch.int32)
    p = torch.tensor([1.0, 0.9, 0.5, 0.3, 0.8, 2.0, 0.0, 0.999])
    m = torch.tensor([0.0, 0.1, 0.0, 0.0, 1.0, 0.2, 0.0, 5.0])
    _check(x, u, T=T, k=k, p=p, m=m)
    _check(x, u, T=0.8, k=k)
    _check(x, u, T=T, p=0.7)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_strided_rows_ids_and_one_draw(dtype):
    wide, u = _scores(5, 700, 5, getattr(torch, dtype))
    dev = wide.cuda()
    for lo, hi in ((0, 333), (1, 334), (3, 700), (5, 6)):
        ids = torch.randint(1, 10_000, (5, hi - lo))
        _check(wide[:, lo:hi].contiguous(), u, T=0.9, k=50, p=0.9, ids=ids, dev=dev[:, lo:hi])
    _check(wide, u[:, 0].contiguous(), k=20)
    _check(wide, torch.rand(5, 70), p=0.9)                        # many draws of a row


@pytest.mark.gpu
def test_random_numbers_outside_their_range():
    x, _ = _scores(2, 500, 6)
    from unirec_amd import ops
    u = torch.tensor([[-1.0, 1.0, 7.0, math.nan], [0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 0.0]])
    i, lp = ops.sample_scores(x[:1].expand(2, 500).contiguous().cuda(), u.cuda(), top_k=50)
    assert torch.equal(i[0], i[1]) and torch.equal(lp[0], lp[1])


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """2.2e9 scores: the last rows lie behind element 2^31"""
    B, N = 2100, 1 << 20
    x = torch.zeros(B, N, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(1)
    tail = (torch.randn(3, N, generator=g) * 2).to(torch.bfloat16)
    x[-3:] = tail.cuda()
    u = torch.rand(B, 1, generator=g)
    from unirec_amd import ops
    i, _ = ops.sample_scores(x, u.cuda(), top_p=0.9)
    for b in range(3):
        want, _ = _reference(tail[b].double().numpy(), u[B - 3 + b].numpy(), 1.0, 0, 0.9, 0.0)
        assert int(i[B - 3 + b]) == int(want[0])
    n = math.ceil(0.9 * N)                                        # a flat row: the first n indices, u n of them before the answer
    flat = torch.floor(u[:-3].double() * n).long()
    assert torch.equal(i[:-3].cpu(), flat)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [900, 60_000])
def test_captured_and_replayed(N):
    from unirec_amd import ops
    sets = [[t.cuda() for t in _scores(6, N, 10 + k)] for k in range(3)]
    buf = [t.clone() for t in sets[0]]
    kw = dict(temperature=0.8, top_k=200, top_p=0.9, min_p=0.001)
    ops.sample_scores(*buf, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sample_scores(*buf, **kw)
    for k in (0, 1, 2, 1, 0):
        for a, b in zip(buf, sets[k]):
            a.copy_(b)
        graph.replay()
        want = ops.sample_scores(*sets[k], **kw)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), k


@pytest.mark.gpu
def test_torch_op():
    import unirec_amd.torch_ops  # noqa: F401
    from unirec_amd import ops
    x, u = (t.cuda() for t in _scores(4, 400, 12))
    a, b = ops.sample_scores(x, u, 0.8, 30, 0.9), torch.ops.unirec_amd.sample_scores(x, u, 0.8, 30, 0.9)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
