"""A distillation loss under no_grad (a validation loss of a model in training mode) takes the loss alone."""
import pytest
import torch
from test_distill_model_gpu import _batch, _model


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["MF", "SASRec"])
def test_the_loss_alone_under_no_grad(name, monkeypatch):
    from unirec_amd import ops
    N = 1200
    m, b = _model(name, N, 1, has_item_bias=True).train(), _batch(20, N, 2)
    score, ids = _model("MF", N, 3, loss_type="bpr").eval().topk(b, 20)
    asked, fwd = [], ops.full_distill_fwd

    def watched(*a, need_grad=True, **kw):
        asked.append(need_grad)
        return fwd(*a, need_grad=need_grad, **kw)
    monkeypatch.setattr(ops, "full_distill_fwd", watched)
    kw = dict(b, teacher_id=ids, teacher_score=score)
    with torch.no_grad():
        alone = m(**kw)[0]
    loss = m(**kw)[0]
    loss.backward()
    fused = m.forward_backward(**kw)
    assert asked == [False, True, True]
    # (the same sums from another instantiation, which may contract its products differently: 16 steps of 2^-24)
    assert abs(alone.item() - loss.item()) <= 2.0 ** -20 * abs(loss.item()) and fused.item() == loss.item()
