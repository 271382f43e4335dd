"""Distillation from a teacher's top logits (unirec_amd.ops.full_distill_fwd / full_distill_bwd) against the formulas in 64 bits.

The tolerances are arithmetic, element by element.  With eps = 2^-24 (half a step of fp32):
  a product of two split operands is off by at most 2^-21 of its size (two operands at 2^-23 each, the dropped low x low at 2^-22) plus a floor
  of 2^-36 of the largest |x| |y|, and its fp32 sum over D by D eps more: the log score is off by  ds = (2^-21 + (D + 8) eps) A / (tau T) + 8 eps |s|,
  A = sum |u| |E|;
  q = exp(s - lse) is then off by a factor 1 + dq,  dq = 2 ds + 16 eps (|log q| <= 100) + 2^-21 (its own split), and sums over n terms add n eps;
  the split weights have a floor of 2^-30 of the largest weight of a row (forward) or column (backward; a weight there is q - p)."""
import math

import pytest
import torch

EPS = 2.0 ** -24


def _inputs(B, N, d, K, seed=0, bias=False, dtype=torch.float32, scale_u=1.0, scale_e=1.0, empty=()):
    g = torch.Generator().manual_seed(seed * 1000003 + B * 7919 + N * 31 + d)
    U = torch.randn(B, d, generator=g) * (6.0 / math.sqrt(d)) * scale_u
    E = torch.randn(N, d, generator=g) * 0.3 * scale_e
    E[0] = 0.0
    ids = torch.randint(1, N, (B, K), generator=g) if N > 1 else torch.zeros(B, K, dtype=torch.int64)
    score = (torch.randn(B, K, generator=g) * 2 + 3).to(dtype)
    for b in range(0, B, 5):                                  # short lists
        n = int(torch.randint(1, K + 1, (1,), generator=g))
        ids[b, n:] = -1
        score[b, n:] = -math.inf
    for b in empty:
        ids[b] = -1
        score[b] = -math.inf
    ib = torch.randn(N, generator=g) * 0.4 if bias else None
    return U, E, ids, score, ib


def _reference(U, E, ids, score, ib, tau, clip, T):
    """the definition in 64 bits on the CPU -> dict with the values, the weights and the bounds' ingredients"""
    U, E = U.double(), E.double()
    B, N = U.shape[0], E.shape[0]
    raw = U @ E.t()
    A = (U.abs() @ E.abs().t()) / (tau * T)
    if ib is not None:
        raw = raw + ib.double()
    raw = raw / tau
    s = (raw.clamp(-clip, clip) if clip > 0 else raw) / T
    lse = torch.logsumexp(s, 1)
    q = torch.exp(s - lse[:, None])
    t = score.double() / T
    here = (ids >= 1) & (ids < N) & (t > -math.inf)
    P = torch.zeros(B, N, dtype=torch.float64)
    rows, ok = torch.zeros(B, dtype=torch.float64), torch.zeros(B, dtype=torch.bool)
    for b in range(B):
        k = torch.nonzero(here[b]).flatten()
        if len(k) == 0:
            continue
        ok[b] = True
        p = torch.softmax(t[b, k], 0)
        rows[b] = (p * (p.log() - s[b, ids[b, k]] + lse[b])).sum()
        P[b].index_add_(0, ids[b, k], p)
    C = max(1, int(ok.sum()))
    inside = (raw.abs() <= clip) if clip > 0 else torch.ones_like(raw, dtype=torch.bool)
    Q = q * ok[:, None] * inside
    P = P * inside
    g = T / (C * tau)
    dT = g * (Q - P).t() @ U
    dT[0] = 0
    return dict(raw=raw, s=s, A=A, q=q, lse=lse, loss=T * T * rows.sum() / C, C=int(ok.sum()), dU=g * (Q - P) @ E, dE=dT, dib=g * (Q - P).sum(0),
                Q=Q, P=P, g=g, ok=ok, T=T, tau=tau)


def _close(got, want, tol, what):
    bad = (got.double().cpu() - want).abs() > tol
    assert not bad.any(), (what, int(bad.sum()), float((got.double().cpu() - want).abs().max()), float(torch.as_tensor(tol).min()))


def _check(r, U, E, loss_out, lse, grads, d_loss=1.0):
    B, d = U.shape
    N, D = E.shape[0], max(32, 1 << (d - 1).bit_length())
    Ua, Ea = U.double().abs(), E.double().abs()
    ds = (2.0 ** -21 + (D + 8) * EPS) * r["A"] + 8 * EPS * r["s"].abs() + 2.0 ** -36 * d * float(Ua.max() * Ea.max()) / (r["tau"] * r["T"])
    dlse = (r["q"] * ds).sum(1) * 2 + 16 * EPS + 2 * EPS * r["lse"].abs()
    _close(lse, r["lse"], dlse, "lse")
    assert float(loss_out[1]) == r["C"]
    assert float(loss_out[2]) == 1.0
    T = r["T"]
    per_row = (r["P"] * ds).sum(1) + dlse + 40 * EPS * (1 + r["s"].abs().amax(1) + r["lse"].abs())
    _close(loss_out[0], r["loss"], T * T * float(per_row.max()) + 8 * EPS * abs(float(r["loss"])), "loss")
    if grads is None:
        return
    du, dt, dib = grads
    dq = 2 * ds + 2 * dlse[:, None] + 116 * EPS + 2.0 ** -20
    g = abs(r["g"] * d_loss)
    Qt = r["Q"] * (dq + N * EPS) + 2.0 ** -30 * r["Q"].amax(1, keepdim=True)
    Pt = r["P"] * (40 * EPS + 4 * EPS * 40)
    _close(du, r["dU"] * d_loss, g * ((Qt + Pt) @ Ea) + 4 * EPS * (r["dU"] * d_loss).abs() + 1e-37, "d_user")
    Qt = r["Q"] * (dq + B * EPS) + 2.0 ** -30 * torch.maximum(r["Q"], r["P"]).amax(0, keepdim=True)
    _close(dt, r["dE"] * d_loss, g * ((Qt + Pt).t() @ Ua) + 4 * EPS * (r["dE"] * d_loss).abs() + 1e-37, "d_table")
    assert (dt[0] == 0).all()
    if dib is not None:
        _close(dib, r["dib"] * d_loss, g * (Qt + Pt).sum(0) + 4 * EPS * (r["dib"] * d_loss).abs() + 1e-37, "d_item_bias")


def _run(U, E, ids, score, ib, tau, clip, T, d_loss=None, grad=True):
    from unirec_amd import ops
    dev = "cuda:0"
    U, E, ids, score = (x.to(dev) for x in (U, E, ids, score))
    ib = None if ib is None else ib.to(dev)
    kw = dict(item_bias=ib, tau=tau, score_clip=clip, temperature=T)
    loss_out, lse, sv = ops.full_distill_fwd(U, E, ids, score, need_grad=grad, **kw)
    if not grad:
        assert sv is None
        return loss_out, lse, None
    dl = None if d_loss is None else torch.tensor([d_loss], device=dev)
    return loss_out, lse, ops.full_distill_bwd(U, E, ids, lse, loss_out, sv, d_loss=dl, **kw)


# ------------------------------------------------------------------------------------------------ refusals (CPU)
def test_refusals():
    from unirec_amd import _lib, ops
    U, E, ids, score, _ = _inputs(3, 20, 16, 4)
    with pytest.raises(_lib.UnirecAmdError, match="GPU tensor"):
        ops.full_distill_fwd(U, E, ids, score)
    lib = _lib.lib
    assert lib.ur_full_distill_workspace_bytes(0, 16, 20, 4, 1) < 0
    assert lib.ur_full_distill_workspace_bytes(1 << 20, 16, 20, 1 << 12, 1) < 0          # B * K does not fit 31 bits
    assert lib.ur_full_distill_workspace_bytes(400, 64, 1682, 20, 1) > lib.ur_full_distill_workspace_bytes(400, 64, 1682, 20, 0) > 0
    one = 1 << 20                                                                         # never read: every call below is refused first

    def fwd(B=4, d=16, N=20, K=3, t=0, tau=1.0, T=1.0, U=one, ws=one):
        return lib.ur_full_distill_fwd(U, one, N, B, d, one, one, t, K, None, tau, -1.0, T, one, one, 1, ws, None)

    for bad, msg in ((dict(U=None), b"null pointer"), (dict(d=18), b"shape"), (dict(N=1), b"shape"), (dict(K=0), b"shape"), (dict(d=260), b"d=260"),
                     (dict(t=7), b"score_type"), (dict(tau=0.0), b"positive"), (dict(T=-1.0), b"positive"), (dict(T=math.nan), b"positive"),
                     (dict(T=math.inf), b"positive"), (dict(ws=None), b"null pointer")):
        assert fwd(**bad) in (-1, -3) and msg in lib.ur_last_error(), bad
    rc = lib.ur_full_distill_bwd(one, one, 20, 4, 16, 3, one, 1.0, -1.0, 1.0, one, None, one, one, None, one, None)
    assert rc == -1 and b"d_item_bias" in lib.ur_last_error()


# ------------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
def test_refusals_on_tensors():
    from unirec_amd import _lib, ops
    U, E, ids, score, ib = (x.cuda() for x in _inputs(4, 20, 16, 3, bias=True))
    for args, kw in (((U, E[:, :8].contiguous(), ids, score), {}), ((U, E, ids[:3], score[:3]), {}), ((U, E, ids, score[:, :2]), {}),
                     ((U, E, ids.int(), score), {}), ((U, E, ids, score.double()), {}), ((U, E, ids, score), dict(tau=0.0)),
                     ((U, E, ids, score), dict(temperature=-1.0)), ((U, E, ids, score), dict(item_bias=ib[:5])), ((U.t(), E, ids, score), {})):
        with pytest.raises(_lib.UnirecAmdError):
            ops.full_distill_fwd(*args, **kw)
    loss_out, lse, sv = ops.full_distill_fwd(U, E, ids, score, need_grad=False)
    with pytest.raises(_lib.UnirecAmdError, match="need_grad"):
        ops.full_distill_bwd(U, E, ids, lse, loss_out, sv)


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,d,K,bias,tau,T,dtype", [
    (1, 2, 4, 1, False, 1.0, 1.0, "float32"), (1, 700, 64, 5, False, 1.0, 1.0, "float32"), (5, 31, 16, 3, True, 0.7, 2.0, "float16"),
    (33, 33, 32, 40, False, 1.0, 1.0, "bfloat16"), (130, 1682, 64, 10, True, 0.5, 2.0, "float32"), (64, 5001, 48, 7, False, 1.3, 0.9, "float32"),
    (65, 5000, 128, 100, True, 1.0, 3.0, "bfloat16"), (300, 2049, 100, 20, False, 0.8, 1.0, "float16"), (7, 3001, 132, 9, True, 1.0, 1.0, "float32"),
    (40, 1025, 256, 300, False, 1.0, 1.5, "float32"), (513, 260, 36, 2, True, 1.0, 1.0, "float32"), (2, 40_003, 128, 3, False, 1.0, 1.0, "float32"),
    (200, 9000, 64, 50, False, 1.0, 4.0, "float32"), (32, 64, 8, 64, True, 2.0, 1.0, "float32")])
def test_against_the_formula(B, N, d, K, bias, tau, T, dtype):
    empty = (B // 2,) if B > 2 else ()
    U, E, ids, score, ib = _inputs(B, N, d, K, bias=bias, dtype=getattr(torch, dtype), empty=empty)
    r = _reference(U, E, ids, score, ib, tau, 0.0, T)
    loss_out, lse, grads = _run(U, E, ids, score, ib, tau, 0.0, T, d_loss=0.7)
    _check(r, U, E, loss_out, lse, grads, 0.7)
    loss2, lse2, _ = _run(U, E, ids, score, ib, tau, 0.0, T, grad=False)
    _check(r, U, E, loss2, lse2, None)


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,d,bias", [(1, 50, 16, False), (20, 300, 64, True), (70, 200, 128, False), (10, 90, 200, True)])
def test_clipped_scores(B, N, d, bias):
    """no score lies within rounding of the clip: which side of it one falls on is not in question"""
    U, E, ids, score, ib = _inputs(B, N, d, 5, seed=3, bias=bias)
    tau, T = 0.8, 1.5
    raw = _reference(U, E, ids, score, ib, tau, 0.0, T)["raw"].abs().flatten().sort().values
    mid = raw[len(raw) // 2: int(len(raw) * 0.95)]
    i = int((mid[1:] - mid[:-1]).argmax())
    clip = float((mid[i] + mid[i + 1]) / 2)
    assert float(mid[i + 1] - mid[i]) > 1e-4
    r = _reference(U, E, ids, score, ib, tau, clip, T)
    loss_out, lse, grads = _run(U, E, ids, score, ib, tau, clip, T)
    _check(r, U, E, loss_out, lse, grads)


@pytest.mark.gpu
@pytest.mark.parametrize("su,se", [(1e-4, 1e4), (1e6, 1e-6), (1e-3, 1.0), (1.0, 1e-5), (30.0, 1.0)])
def test_operands_of_other_magnitudes(su, se):
    """the group exponents carry tables of 1e-5 and of 1e4 alike; rows of very different size share a table"""
    U, E, ids, score, _ = _inputs(50, 400, 64, 8, seed=4, scale_u=su, scale_e=se)
    E[10:20] *= 1e-3
    E[50] *= 20.0
    U[3] = 0.0
    r = _reference(U, E, ids, score, None, 1.0, 0.0, 1.0)
    loss_out, lse, grads = _run(U, E, ids, score, None, 1.0, 0.0, 1.0)
    _check(r, U, E, loss_out, lse, grads)


@pytest.mark.gpu
def test_masks_duplicates_and_absent_entries():
    U, E, ids, score, _ = _inputs(12, 60, 32, 6, seed=5)
    ids[1] = 7                                     # the same item six times
    ids[2, 3] = 0                                  # the padding row
    score[3, 2] = math.nan                         # a score that is none
    score[4, 1:] = torch.finfo(torch.float32).min  # masked by the type's lowest value: present, without mass
    ids[5], score[5] = -1, -math.inf               # no list at all
    score[6] = -math.inf                           # items without scores
    ids[7, 0] = ids[7, 4]
    r = _reference(U, E, ids, torch.nan_to_num(score, nan=-math.inf, neginf=-math.inf), None, 1.0, 0.0, 1.0)
    r["P"] = torch.nan_to_num(r["P"])
    loss = _loss64(r, ids, score)
    loss_out, lse, grads = _run(U, E, ids, score, None, 1.0, 0.0, 1.0)
    r["loss"] = loss
    _check(r, U, E, loss_out, lse, grads)


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,d,K", [(3, 40, 16, 30), (40, 300, 64, 1500), (70, 5000, 128, 260), (33, 1_200_000, 32, 40), (33, 1_200_000, 32, 160)])
def test_lists_that_fall_on_few_items(B, N, d, K):
    """every user lists the same few items, some of them over and over: one block of items has all entries, a cell has many"""
    U, E, ids, score, ib = _inputs(B, N, d, K, seed=13, bias=True)
    ids = torch.where(ids > 0, ids % min(N - 1, 50) + 1, ids)
    if N > 10_000:                                              # lists' blocks are wider than a workgroup's items there
        ids = torch.where(ids > 0, ids + N - 60, ids)
    r = _reference(U, E, ids, score, ib, 1.0, 0.0, 1.5)
    a = _run(U, E, ids, score, ib, 1.0, 0.0, 1.5)
    _check(r, U, E, *a)
    b = _run(U, E, ids, score, ib, 1.0, 0.0, 1.5)
    assert torch.equal(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[2], b[2]))


@pytest.mark.gpu
def test_a_forward_serves_more_than_one_backward():
    from unirec_amd import ops
    U, E, ids, score, ib = (x.cuda() for x in _inputs(50, 700, 64, 9, seed=14, bias=True))
    loss_out, lse, sv = ops.full_distill_fwd(U, E, ids, score, item_bias=ib)
    a = ops.full_distill_bwd(U, E, ids, lse, loss_out, sv, item_bias=ib)
    b = ops.full_distill_bwd(U, E, ids, lse, loss_out, sv, item_bias=ib, d_loss=torch.tensor([2.0], device="cuda"))
    assert all(torch.equal(2 * x, y) for x, y in zip(a, b))


def _loss64(r, ids, score):
    """the loss with entries of no mass counted as p log p = 0"""
    tot = 0.0
    for b in range(ids.shape[0]):
        t = torch.where((ids[b] >= 1) & (score[b].double() > -math.inf), score[b].double() / r["T"], -math.inf)
        if not (t > -math.inf).any():
            continue
        p = torch.softmax(t, 0)
        for k in range(len(t)):
            if p[k] > 0:
                tot += p[k] * (p[k].log() - r["s"][b, ids[b, k]] + r["lse"][b])
    return torch.as_tensor(r["T"] ** 2 * tot / max(1, r["C"]))


@pytest.mark.gpu
def test_no_row_has_a_teacher():
    U, E, ids, score, _ = _inputs(5, 40, 16, 3)
    ids[:], score[:] = -1, -math.inf
    loss_out, lse, (du, dt, _) = _run(U, E, ids, score, None, 1.0, 0.0, 1.0)
    assert loss_out[0] == 0 and loss_out[1] == 0 and loss_out[2] == 1
    assert (du == 0).all() and (dt == 0).all() and torch.isfinite(lse).all()


@pytest.mark.gpu
def test_an_item_masked_by_its_bias_and_a_nan_user():
    U, E, ids, score, ib = _inputs(40, 100, 32, 3, seed=6, bias=True)
    ids = ids.clamp(min=2)
    score = torch.nan_to_num(score, neginf=0.0)
    ib[1] = -math.inf                              # never in anybody's list: no weight, no gradient
    r = _reference(U, E, ids, score, ib, 1.0, 0.0, 1.0)
    for k in ("s", "A", "q", "Q"):
        r[k] = torch.nan_to_num(r[k], neginf=0.0)
    loss_out, lse, grads = _run(U, E, ids, score, ib, 1.0, 0.0, 1.0)
    _check(r, U, E, loss_out, lse, grads)
    assert (grads[1][1] == 0).all() and grads[2][1] == 0
    U[4, 3] = math.nan
    loss_out, lse, _ = _run(U, E, ids, score, ib, 1.0, 0.0, 1.0)
    assert math.isnan(float(loss_out[0])) and loss_out[2] == -1        # the optimizer skips such a step
    assert math.isnan(float(lse[4])) and torch.isfinite(lse[torch.arange(40) != 4]).all()


@pytest.mark.gpu
def test_an_id_outside_the_table_raises_the_guard():
    from unirec_amd import ops
    U, E, ids, score, _ = _inputs(6, 50, 16, 3, seed=8)
    ids[2, 1] = 50
    good = ids.clone()
    good[2, 1] = -1
    try:
        loss_out, lse, grads = _run(U, E, ids, score, None, 1.0, 0.0, 1.0)
        torch.cuda.synchronize()
        with pytest.raises(IndexError, match="50"):
            ops.id_guard_check()
        _check(_reference(U, E, good, score, None, 1.0, 0.0, 1.0), U, E, loss_out, lse, grads)
    finally:
        ops.id_guard_reset()


@pytest.mark.gpu
def test_gradient_against_differences():
    """d loss along a random direction of users, table and bias; loss differences of step h carry 2^-22 |loss| / h and h^2 of curvature"""
    U, E, ids, score, ib = _inputs(24, 300, 64, 6, seed=9, bias=True)
    g = torch.Generator().manual_seed(1)
    vU, vE, vb = torch.randn(U.shape, generator=g) * 0.05, torch.randn(E.shape, generator=g) * 0.05, torch.randn(ib.shape, generator=g)
    vE[0] = 0
    loss_out, _, (du, dt, dib) = _run(U, E, ids, score, ib, 0.9, 0.0, 1.7)
    slope = float((du.cpu().double() * vU).sum() + (dt.cpu().double() * vE).sum() + (dib.cpu().double() * vb).sum())
    h = 2.0 ** -5
    up = float(_run(U + h * vU, E + h * vE, ids, score, ib + h * vb, 0.9, 0.0, 1.7, grad=False)[0][0])
    down = float(_run(U - h * vU, E - h * vE, ids, score, ib - h * vb, 0.9, 0.0, 1.7, grad=False)[0][0])
    diff = (up - down) / (2 * h)
    ref = _reference(U, E, ids, score, ib, 0.9, 0.0, 1.7)
    step = [float(_reference((U + s * h * vU).double(), (E + s * h * vE).double(), ids, score, ib + s * h * vb, 0.9, 0.0, 1.7)["loss"]) for s in (1, -1)]
    curvature = abs((step[0] - step[1]) / (2 * h) - float((ref["dU"] * vU).sum() + (ref["dE"] * vE).sum() + (ref["dib"] * vb).sum()))
    assert abs(diff - slope) <= 1.01 * curvature + 2.0 ** -20 * abs(float(loss_out[0])) / h, (diff, slope)


@pytest.mark.gpu
def test_bits_do_not_depend_on_the_run_or_the_stream():
    U, E, ids, score, ib = _inputs(100, 3000, 64, 30, seed=10, bias=True)
    ids[:, 0] = 5                                  # one item in every list: its row is a long sum
    a = _run(U, E, ids, score, ib, 1.0, 0.0, 2.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = _run(U, E, ids, score, ib, 1.0, 0.0, 2.0)
    torch.cuda.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and all(torch.equal(x, y) for x, y in zip(a[2], b[2]))


@pytest.mark.gpu
def test_captured_and_replayed():
    """a step captured into a graph, replayed on other inputs with eager steps between: every replay equals the eager result"""
    from unirec_amd import ops
    dev = "cuda:0"
    sets = [[x.to(dev) for x in _inputs(70, 900, 64, 12, seed=20 + k)[:4]] for k in range(3)]
    buf = [x.clone() for x in sets[0]]

    def step(U, E, ids, score):
        loss_out, lse, sv = ops.full_distill_fwd(U, E, ids, score, tau=0.8, temperature=2.0)
        return (loss_out, lse) + ops.full_distill_bwd(U, E, ids, lse, loss_out, sv, tau=0.8, temperature=2.0)[:2]

    step(*buf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*buf)
    for k in (0, 1, 2, 1, 0):
        for x, y in zip(buf, sets[k]):
            x.copy_(y)
        graph.replay()
        want = step(*sets[k])
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want)), k


@pytest.mark.gpu
def test_table_offsets_beyond_32_bits():
    """18 M items of 128: element offsets of the table and of its gradient pass 2^31"""
    from unirec_amd import ops
    N, d, B, K = 18_000_000, 128, 6, 4
    g = torch.Generator(device="cuda").manual_seed(3)
    E = torch.randn(N, d, generator=g, device="cuda")
    E[0] = 0
    U = torch.randn(B, d, generator=g, device="cuda") * 0.2
    ids = torch.randint(N - 100_000, N, (B, K), generator=g, device="cuda")
    ids[0, 0] = N - 1
    score = torch.randn(B, K, generator=g, device="cuda")
    loss_out, lse, sv = ops.full_distill_fwd(U, E, ids, score)
    du, dt, _ = ops.full_distill_bwd(U, E, ids, lse, loss_out, sv)
    ref = torch.cat([torch.logsumexp(torch.stack([(U.double() @ E[i:i + 1_000_000].double().t()).logsumexp(1) for i in range(0, N, 1_000_000)]), 0)])
    # lse: |s| <= 20, so the score's bound of the file's head is 130 eps 20 + 8 eps 20
    tol = 2 * (2.0 ** -21 + 136 * EPS) * float((U.abs().sum(1) * 6).max()) + 32 * EPS * 20
    assert (lse.double() - ref).abs().max() <= tol
    lo = N - 100_000                                # the table's last rows, all of them
    s = U.double() @ E[lo:].double().t()
    q = torch.exp(s - ref[:, None])
    p = torch.softmax(score.double(), 1)
    grad = q.scatter_add(1, ids - lo, -p) / B
    want = grad.t() @ U.double()
    bound = (2 * tol + 2.0 ** -18) * (q.scatter_add(1, ids - lo, p) / B).t() @ U.double().abs() + 2.0 ** -28 * (q.scatter_add(1, ids - lo, p).amax(0) / B)[:, None] * U.double().abs().sum(0)
    assert ((dt[lo:].double() - want).abs() <= bound).all()
    mid = dt[N // 2: N // 2 + 1000]
    qm = torch.exp(U.double() @ E[N // 2: N // 2 + 1000].double().t() - ref[:, None]) / B
    bm = (2 * tol + 2.0 ** -18) * qm.t() @ U.double().abs() + 2.0 ** -28 * qm.amax(0)[:, None] * U.double().abs().sum(0)
    assert ((mid.double() - qm.t() @ U.double()).abs() <= bm).all()


@pytest.mark.gpu
def test_torch_ops():
    import unirec_amd.torch_ops  # noqa: F401
    U, E, ids, score, ib = _inputs(20, 200, 32, 5, seed=12, bias=True)
    a = _run(U, E, ids, score, ib, 0.9, 0.0, 1.5)
    U, E, ids, score, ib = (x.cuda() for x in (U, E, ids, score, ib))
    o = torch.ops.unirec_amd.full_distill_fwd(U, E, ids, score, ib, 0.9, -1.0, 1.5)
    g = torch.ops.unirec_amd.full_distill_bwd(U, E, ids, o[0], o[1], o[2], None, ib, 0.9, -1.0, 1.5)
    assert torch.equal(a[0], o[0]) and torch.equal(a[1], o[1]) and all(torch.equal(x, y) for x, y in zip(a[2], g))
