"""What a distillation's forward leaves for its backward: refused where the two calls do not belong together, safe on another stream than the
forward's."""
import pytest
import torch
from test_distill_gpu import _inputs


def _forward(bias=True, **kw):
    from unirec_amd import ops
    U, E, ids, score, ib = (x.cuda() for x in _inputs(40, 900, 64, 9, seed=51, bias=True))
    return (U, E, ids, score, ib), ops.full_distill_fwd(U, E, ids, score, item_bias=ib if bias else None, **kw)


@pytest.mark.gpu
def test_a_backward_with_other_arguments_is_refused():
    from unirec_amd import _lib, ops
    for with_bias in (True, False):
        (U, E, ids, score, ib), (loss_out, lse, sv) = _forward(with_bias, tau=0.8, temperature=2.0)
        kw = dict(item_bias=ib if with_bias else None, tau=0.8, temperature=2.0)
        a = ops.full_distill_bwd(U, E, ids, lse, loss_out, sv, **kw)
        b = ops.full_distill_bwd(U, E, ids, lse, loss_out, sv, score_clip=0, d_loss=torch.ones(1, device="cuda"), **kw)   # (no clip, 1: the same)
        assert all(x is y or torch.equal(x, y) for x, y in zip(a, b))
        for other in (dict(item_bias=None if with_bias else ib), dict(tau=1.0), dict(temperature=1.0), dict(score_clip=3.0)):
            with pytest.raises(_lib.UnirecAmdError, match="its full_distill_fwd had"):
                ops.full_distill_bwd(U, E, ids, lse, loss_out, sv, **{**kw, **other})
        for args in ((U, E, ids, lse.double(), loss_out, sv), (U, E, ids, lse[:5], loss_out, sv), (U, E, ids, lse, loss_out.cpu(), sv), (U, E, ids.int(), lse, loss_out, sv),
                     (U, E, ids[:, :4].contiguous(), lse, loss_out, sv), (U, E, ids.flatten(), lse, loss_out, sv), (U, E, ids, lse, loss_out, None)):
            with pytest.raises(_lib.UnirecAmdError):
                ops.full_distill_bwd(*args, **kw)
        for n in (0, 2):                                          # (an empty tensor's address is null, which is d_loss = 1)
            with pytest.raises(_lib.UnirecAmdError, match="d_loss"):
                ops.full_distill_bwd(U, E, ids, lse, loss_out, sv, d_loss=torch.ones(n, device="cuda"), **kw)


@pytest.mark.gpu
def test_a_backward_on_another_stream_keeps_what_it_reads():
    """the results of the forward are dropped while the backward, on another stream, has not begun: their memory is not given out on the first"""
    from unirec_amd import ops
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(first):
        (U, E, ids, score, ib), (loss_out, lse, sv) = _forward()
        want = ops.full_distill_bwd(U, E, ids, lse, loss_out, sv, item_bias=ib)
    torch.cuda.synchronize()
    size = sv.ws.numel()
    with torch.cuda.stream(second):
        torch.cuda._sleep(100_000_000)                            # some 50 ms
        got = ops.full_distill_bwd(U, E, ids, lse, loss_out, sv, item_bias=ib)
        del sv
    with torch.cuda.stream(first):
        over = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    del over
    assert all(torch.equal(x, y) for x, y in zip(got, want))
