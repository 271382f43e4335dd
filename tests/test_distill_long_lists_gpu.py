"""Long teacher lists: an item listed twice is found among thousands, and lists that would hold the GPU for minutes are refused."""
import pytest
import torch
from test_distill_gpu import _check, _inputs, _reference, _run


def test_lists_too_long_are_refused():
    from unirec_amd import _lib
    lib, one = _lib.lib, 1 << 20                                  # (never read: every call is refused first)
    assert lib.ur_full_distill_workspace_bytes(2, 16, 1 << 20, 65537, 1) < 0 < lib.ur_full_distill_workspace_bytes(2, 16, 1 << 20, 65536, 1)
    assert lib.ur_full_distill_fwd(one, one, 1 << 20, 2, 16, one, one, 0, 65537, None, 1.0, -1.0, 1.0, one, one, 1, one, None) in (-1, -3)
    assert b"65537" in lib.ur_last_error()
    assert lib.ur_full_distill_bwd(one, one, 1 << 20, 2, 16, 65537, None, 1.0, -1.0, 1.0, one, None, one, one, None, one, None) in (-1, -3)


@pytest.mark.gpu
def test_lists_too_long_or_empty_are_refused_on_tensors():
    from unirec_amd import _lib, ops
    U, E, _, _, _ = (None if x is None else x.cuda() for x in _inputs(1, 50, 16, 3))
    for K in (0, 65537):
        with pytest.raises(_lib.UnirecAmdError, match="entries a list"):
            ops.full_distill_fwd(U, E, torch.ones(1, K, dtype=torch.int64, device="cuda"), torch.zeros(1, K, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,d,K", [(3, 20_000, 32, 5000), (2, 3000, 16, 9001)])
def test_long_lists(B, N, d, K):
    """(9 001 entries on 3 000 items: most are listed several times)"""
    U, E, ids, score, ib = _inputs(B, N, d, K, seed=81, bias=True)
    ids[0, 17] = ids[0, K - 3] = 5
    r = _reference(U, E, ids, score, ib, 1.0, 0.0, 1.0)
    # (_check's bound of a probability is 40 steps: the teacher's softmax over K entries adds up K of them, and the loss K terms)
    eps = 2.0 ** -24
    loss_out, lse, (du, dt, dib) = _run(U, E, ids, score, ib, 1.0, 0.0, 1.0)
    _check(r, U, E, loss_out, lse, None)
    A, lse_off = r["A"], 2.0 ** -20
    dq = 2 * ((2.0 ** -21 + 40 * eps) * A + 8 * eps * r["s"].abs()) + lse_off + N * eps
    Q = r["Q"] * dq + 2.0 ** -30 * r["Q"].amax(1, keepdim=True)
    P = r["P"] * (K + 200) * eps
    g = abs(r["g"])
    assert ((du.double().cpu() - r["dU"]).abs() <= g * ((Q + P) @ E.double().abs()) + 1e-30).all()
    assert ((dt.double().cpu() - r["dE"]).abs() <= g * ((Q + P).t() @ U.double().abs()) + 1e-30 + 2.0 ** -30 * g * torch.maximum(r["Q"], r["P"]).amax(0)[:, None]
            * U.double().abs().sum(0)).all()
    assert ((dib.double().cpu() - r["dib"]).abs() <= g * (Q + P).sum(0) + 1e-30 + 2.0 ** -30 * g * B * torch.maximum(r["Q"], r["P"]).amax(0)).all()
