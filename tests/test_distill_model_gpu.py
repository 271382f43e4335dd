"""loss_type='distill' and BaseRecommender.sample: a teacher's top list, a student trained on it, items drawn from the student."""
import math
import types

import numpy as np
import pytest
import torch

T = 1.7


def _cfg(name, N, **kw):
    from unirec_amd.utils.argument_parser import parse_arguments
    return parse_arguments({**dict(model=name, n_users=60, n_items=N, device="cuda:0", loss_type="distill", embedding_size=32, hidden_size=32, inner_size=64,
                                   n_heads=4, n_layers=1, max_seq_len=12, seed=2, init_std=0.3, has_user_emb=name == "MF", hidden_dropout_prob=0.0,
                                   attn_dropout_prob=0.0, tau=0.6, distill_temperature=T), **kw})


def _model(name, N, seed, **kw):
    from unirec_amd.utils.general import get_class_instance
    torch.manual_seed(seed)
    return get_class_instance(name, "unirec_amd/model")(_cfg(name, N, **kw))


def _batch(B, N, seed):
    rng = np.random.default_rng(seed)
    seq = rng.integers(1, N, (B, 12)).astype(np.int32)
    for b in range(B):
        seq[b, : rng.integers(0, 12)] = 0
    return {k: torch.from_numpy(v).cuda() for k, v in dict(user_id=rng.integers(1, 60, B), item_id=rng.integers(1, N, B), item_seq=seq,
                                                           item_seq_len=(seq > 0).sum(1)).items()}


def _loss64(U, E, ib, ids, score, tau):
    """the definition, in the type of its arguments; differentiable"""
    s = (U @ E.t() + (0.0 if ib is None else ib)) / (tau * T)
    t = torch.softmax(score.double() / T, 1)
    hit = torch.gather(s, 1, ids.clamp_min(0))
    part = torch.where(t > 0, t * (torch.log(t.clamp_min(1e-300)) - hit + torch.logsumexp(s, 1, keepdim=True)), torch.zeros_like(t))
    return T * T * part.sum() / len(U)


# ------------------------------------------------------------------------------------------------ refusals (CPU)
def test_refusals():
    from unirec_amd.facility.distributed import ShardedSparseDenseAdam
    from unirec_amd.facility.trainer import Trainer
    from unirec_amd.model.base.recommender import BaseRecommender
    one = torch.zeros(2, 3)
    for a in ((None, None), (one, None), (None, one)):
        with pytest.raises(ValueError, match="teacher_id"):
            BaseRecommender._teacher_list(*a)
    with pytest.raises(NotImplementedError, match="one GPU"):
        ShardedSparseDenseAdam(types.SimpleNamespace(loss_type="distill"), 0, 2)
    tr = Trainer.__new__(Trainer)
    tr.model = types.SimpleNamespace(loss_type="bpr", n_items=10)
    teacher = types.SimpleNamespace(n_items=10)
    with pytest.raises(ValueError, match="labels"):
        tr.set_teacher(teacher, 5)
    tr.model.loss_type = "distill"
    for t, k in ((teacher, 0), (teacher, 1025), (types.SimpleNamespace(n_items=11), 5), (tr.model, 5)):
        with pytest.raises(ValueError, match="set_teacher"):
            tr.set_teacher(t, k)
    tr.set_teacher(teacher, 5)
    assert tr.teacher is teacher and tr.teacher_k == 5


# ------------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
def test_model_refusals():
    m = _model("MF", 300, 0).train()
    b = _batch(4, 300, 0)
    with pytest.raises(ValueError, match="teacher_id"):
        m.forward_backward(**b)
    lists = dict(teacher_id=torch.ones(4, 2, dtype=torch.int64, device="cuda"), teacher_score=torch.ones(4, 2, device="cuda"))
    with pytest.raises(NotImplementedError, match="materialised"):
        m(**b, **lists, return_loss_only=False)
    with pytest.raises(NotImplementedError, match="user-bias"):
        _model("MF", 300, 0, has_user_bias=True, score_clip_value=4.0)
    with pytest.raises(ValueError, match="distill_temperature"):
        _model("MF", 300, 0, distill_temperature=0.0)
    from unirec_amd.facility.trainer import Trainer
    with pytest.raises(ValueError, match="no teacher"):
        Trainer(_cfg("MF", 300), m).train_step(b)


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("name,B,N,bias,dtype", [("MF", 37, 2001, True, torch.float32), ("SASRec", 10, 1503, False, torch.bfloat16)])
def test_gradients_of_a_step(name, B, N, bias, dtype, fused):
    """one step of the model: loss and every gradient that the formula gives, from the user vectors on.  The operator's own bounds are a few
    1e-6 of the largest entry at these sizes (6 significant digits of a product over 32, sums over N): 2e-5 of it is ample"""
    m = _model(name, N, 1, has_user_bias=bias, has_item_bias=bias)
    b = _batch(B, N, 3)
    teacher = _model("MF", N, 4, loss_type="bpr").eval()
    score, ids = teacher.topk(b, 20)
    score = score.to(dtype)
    m.eval()
    with torch.no_grad():
        U = m.forward_user_emb(**{k: b[k] for k in ("user_id", "item_seq", "item_seq_len")}).double().cpu().requires_grad_()
    E = m.item_embedding.weight.detach().double().cpu().requires_grad_()
    ib = m.item_bias.detach().double().cpu().requires_grad_() if bias else None
    want = _loss64(U, E, ib, ids.cpu(), score.cpu(), 0.6)
    want.backward()
    m.train()
    if fused:
        loss = m.forward_backward(**b, teacher_id=ids, teacher_score=score)
    else:
        loss, scores, _, _ = m(**b, teacher_id=ids, teacher_score=score)
        assert scores is None
        loss.backward()
    assert abs(loss.item() - want.item()) <= 2e-5 * abs(want.item())
    got = m.dense_table_grads["item_embedding"].double().cpu()
    dE = E.grad.clone()
    dE[0] = 0                                                    # the padding row
    assert (got - dE).abs().max() <= 2e-5 * dE.abs().max()
    if bias:
        assert (m.item_bias.grad.double().cpu() - ib.grad).abs().max() <= 2e-5 * ib.grad.abs().max()
        assert float(m.user_bias.grad.abs().max()) == 0.0
    if name == "MF":
        (g,) = [g for g in m.sparse_grads if g["table"] == "user_embedding"]
        assert torch.equal(g["ids_a"].cpu().long(), b["user_id"].cpu())
        assert (g["rows"].double().cpu() - U.grad).abs().max() <= 2e-5 * U.grad.abs().max()
    else:
        assert m.dense_flat.grad is not None and torch.isfinite(m.dense_flat.grad).all()


@pytest.mark.gpu
def test_steps_follow_dense_adam():
    """the Trainer's step with a teacher, against torch's Adam in 64 bits on both tables"""
    from unirec_amd.facility.trainer import Trainer
    N = 800
    m, teacher = _model("MF", N, 5, learning_rate=1e-3), _model("MF", N, 6, loss_type="bpr").train()
    U, E = (t.weight.detach().double().cpu().requires_grad_() for t in (m.user_embedding, m.item_embedding))
    opt = torch.optim.Adam([U, E], lr=1e-3, eps=1e-8)
    tr = Trainer(m.config, m)
    tr.set_teacher(teacher, 30)
    batches = [_batch(24, N, s) for s in range(5)]
    for i, b in enumerate(batches):
        loss = tr.train_step(b, batches[i + 1] if i + 1 < len(batches) else None)
        assert not teacher.training
        score, ids = teacher.topk(b, 30)
        opt.zero_grad()
        want = _loss64(U[b["user_id"].cpu()], E, None, ids.cpu(), score.cpu(), 0.6)
        want.backward()
        E.grad[0] = 0
        opt.step()
        assert abs(loss.item() - want.item()) <= 1e-4 * abs(want.item()), i
    tr.optimizer.flush()
    # (Adam divides by sqrt(v): where a gradient is close to zero its sign decides a whole step of 1e-3, so the tables are compared in the mean)
    for t, ref in ((m.user_embedding, U), (m.item_embedding, E)):
        assert (t.weight.detach().double().cpu() - ref.detach()).abs().mean() <= 2e-6
    given = dict(batches[0], teacher_id=ids, teacher_score=score)   # a batch that brings its own list
    tr.teacher = None
    assert math.isfinite(float(tr.train_step(given)))


@pytest.mark.gpu
def test_teacher_student_and_draws():
    """the whole run: a teacher's lists, a student's steps on them, items drawn from the student"""
    from unirec_amd.facility.trainer import Trainer
    from test_sample_gpu import _reference
    N, B, k = 1203, 50, 64
    teacher, m = _model("MF", N, 7, loss_type="bpr").eval(), _model("SASRec", N, 8, has_item_bias=True)
    tr = Trainer(m.config, m)
    tr.set_teacher(teacher, 25)
    batches = [_batch(B, N, 20 + s) for s in range(3)]
    for i, b in enumerate(batches):
        assert math.isfinite(float(tr.train_step(b, batches[i + 1] if i < 2 else None)))
    tr.optimizer.flush()
    m.eval()
    b = batches[0]
    hist = b["item_seq"].long()
    rand = torch.rand(B, 6, generator=torch.Generator().manual_seed(1))
    temp = torch.linspace(0.0, 2.0, B)
    got, logp = m.sample(b, rand.cuda(), k=k, temperature=temp.cuda(), top_p=0.9, min_p=0.02, user_hist=hist)
    assert got.shape == (B, 6) and logp.shape == (B, 6)
    score, ids = m.topk(b, k, user_hist=hist)
    x, ids = score.double().cpu().numpy(), ids.cpu().numpy()
    for r in range(B):
        i, lp = _reference(x[r], rand[r].numpy(), float(temp[r]), 0, 0.9, 0.02)
        assert (got[r].cpu().numpy() == ids[r][i]).all()
        assert np.abs(logp[r].double().cpu().numpy() - lp).max() <= 2.0 ** -23 * np.abs(lp).max() + 1e-12
        assert not set(got[r].tolist()) & set(hist[r].tolist())
    best, zero = m.sample(b, rand[:, 0].contiguous().cuda(), k=k, temperature=0.0)
    assert torch.equal(best, m.topk(b, 1)[1][:, 0]) and float(zero.abs().max()) == 0.0
