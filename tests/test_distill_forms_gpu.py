"""The forms of the distillation kernels that a user count, a width and a catalogue choose between them (waves of a workgroup in the forward and in
the backward, padded width), each with clipped and with unclipped scores.  Scores are multiples of 1 / 16 and the clip lies 1 / 32 off them: which side
of it one falls on is not in question."""
import pytest
import torch
from test_distill_gpu import _check, _inputs, _reference, _run


def _grid(B, N, d, K, bias):
    U, E, ids, score, _ = _inputs(B, N, d, K, seed=71, empty=(B // 3,))
    g = torch.Generator().manual_seed(B * 7 + N + d)
    U = torch.randint(-3, 4, (B, d), generator=g) / 4.0
    E = torch.randint(-3, 4, (N, d), generator=g) / 8.0
    E[0] = 0
    return U, E, ids, score, torch.randint(-8, 9, (N,), generator=g) / 32.0 if bias else None


@pytest.mark.gpu
@pytest.mark.parametrize("clipped", [True, False])
@pytest.mark.parametrize("B,N,d,K,bias", [
    (200, 9000, 64, 20, True), (200, 9000, 128, 20, False), (260, 8300, 100, 12, True), (129, 8193, 36, 5, False),   # eight waves, four waves back
    (200, 700, 64, 20, False), (140, 600, 128, 9, True),                                                             # eight, one
    (128, 9000, 64, 20, False), (40, 12_000, 128, 6, True), (3, 8200, 64, 3, False),                                 # four, four
    (40, 9001, 256, 30, True), (300, 8500, 200, 10, False), (17, 500, 256, 5, True),                                 # width 256: four, four; one
    (200, 9000, 32, 8, True), (20, 9000, 16, 4, False), (33, 100, 28, 4, True)])                                     # width 32: four, four; one
def test_every_form(B, N, d, K, bias, clipped):
    U, E, ids, score, ib = _grid(B, N, d, K, bias)
    tau, T, clip = 0.5, 1.5, 2.0 + 1 / 32 if clipped else 0.0
    r = _reference(U, E, ids, score, ib, tau, clip, T)
    if clipped:
        out = float((r["raw"].abs() > clip).double().mean())
        assert 0.01 < out < 0.9 and float((r["raw"].abs() - clip).abs().min()) >= 1 / 32 - 1e-9
    loss_out, lse, grads = _run(U, E, ids, score, ib, tau, clip, T, d_loss=1.3)
    _check(r, U, E, loss_out, lse, grads, 1.3)
    loss2, lse2, _ = _run(U, E, ids, score, ib, tau, clip, T, grad=False)
    _check(r, U, E, loss2, lse2, None)
