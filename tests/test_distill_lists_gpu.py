"""Teacher lists that crowd: on items next to each other (the popular end of a catalogue sorted by popularity), and on items whose ids leave the
same remainder, which share one list of the table's gradient and do not fit its room at once."""
import pytest
import torch
from test_distill_gpu import _check, _inputs, _reference, _run


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,d,K", [(70, 40_000, 64, 64), (33, 400_000, 32, 160), (64, 9000, 128, 70), (40, 20_000, 200, 90)])
@pytest.mark.parametrize("step", [1, 37, 64, 256, 512, 4096])
def test_crowded_lists(B, N, d, K, step):
    U, E, ids, score, ib = _inputs(B, N, d, K, seed=41, bias=True)
    g = torch.Generator().manual_seed(B + step)
    room = (N - 1) // step                                       # items 1, 1 + step, ..: three crowds of them, far apart where there is room
    at = torch.cat([torch.arange(0, 90), torch.arange(room // 3, room // 3 + 40), torch.arange(room - 70, room)]).clamp(0, room - 1).unique()
    pick = torch.stack([at[torch.randint(0, len(at), (K,), generator=g)] if len(at) < K else at[torch.randperm(len(at), generator=g)[:K]] for _ in range(B)])
    ids = torch.where(ids > 0, 1 + step * pick, ids)
    r = _reference(U, E, ids, score, ib, 1.0, 0.0, 1.5)
    a = _run(U, E, ids, score, ib, 1.0, 0.0, 1.5)
    _check(r, U, E, *a)
    b = _run(U, E, ids, score, ib, 1.0, 0.0, 1.5)
    assert torch.equal(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[2], b[2]))
