"""torch.ops.unirec_amd.full_distill_fwd for the loss alone."""
import pytest
import torch
from test_distill_gpu import _inputs, _run


@pytest.mark.gpu
def test_the_loss_alone():
    import unirec_amd.torch_ops  # noqa: F401
    from unirec_amd import _lib
    U, E, ids, score, ib = _inputs(20, 200, 32, 5, seed=61, bias=True)
    want = _run(U, E, ids, score, ib, 0.9, 0.0, 1.5, grad=False)
    U, E, ids, score, ib = (x.cuda() for x in (U, E, ids, score, ib))
    op = torch.ops.unirec_amd.full_distill_fwd
    loss_out, lse, ws = op(U, E, ids, score, ib, 0.9, -1.0, 1.5, False)
    assert torch.equal(loss_out, want[0]) and torch.equal(lse, want[1]) and ws.numel() == 0 and ws.dtype == torch.uint8
    with pytest.raises(_lib.UnirecAmdError, match="ws"):
        torch.ops.unirec_amd.full_distill_bwd(U, E, ids, loss_out, lse, ws, None, ib, 0.9, -1.0, 1.5)
    fn = torch.compile(lambda u, n: op(u, E, ids, score, ib, 0.9, -1.0, 1.5, n)[0][0] * 2, backend="eager", fullgraph=True)
    assert torch.equal(fn(U, False), 2 * want[0][0]) and torch.equal(fn(U, True), 2 * want[0][0])
