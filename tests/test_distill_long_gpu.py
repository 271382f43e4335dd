"""A student that has nearly learnt its teacher's list, over a long catalogue: what is left of the gradient comes from a tail of a million items that
weigh next to nothing each."""
import math

import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,apart", [(4000, 1_000_001, 50_000), (500, 8_000_001, 400_000)])
@pytest.mark.parametrize("same", [True, False])
def test_a_light_tail_keeps_its_weight(B, N, apart, same):
    """20 items that the teacher lists, alike, and N - 20 whose scores lie 21.5 below (users of 0: the scores are the bias alone, and exact).
    d_user = (sum_n q E - mean of the 20) / B.  A sum in fp32 may lose what is added in pieces below 2^-25 of it, here all of the tail that stands in a
    partial sum with one of the 20: 20 runs of 8 192 items at most, 20 x 8 192 q |E|.  Everything else is rounding of the 20 themselves, 16 steps of
    2^-24 of the largest"""
    from unirec_amd import ops
    d, gap = 64, 21.5
    g = torch.Generator(device="cuda").manual_seed(N)
    E = torch.full((N, d), 0.3, device="cuda")
    if not same:
        E += torch.randn(N, d, generator=g, device="cuda") * 0.2
    heads = torch.arange(500, N, apart, device="cuda")
    E[heads] = torch.randn(len(heads), d, generator=g, device="cuda") * 0.3
    E[0] = 0
    bias = torch.full((N,), -gap, device="cuda")
    bias[heads] = 0
    ids = heads.repeat(B, 1).contiguous()
    kw = dict(item_bias=bias)
    loss_out, lse, sv = ops.full_distill_fwd(torch.zeros(B, d, device="cuda"), E, ids, torch.zeros(ids.shape, device="cuda"), **kw)
    du, _, _ = ops.full_distill_bwd(torch.zeros(B, d, device="cuda"), E, ids, lse, loss_out, sv, **kw)
    K, w = len(heads), math.exp(-gap)
    W = K + (N - K) * w
    rest = E.double().sum(0) - E[heads].double().sum(0)
    want = (E[heads].double().sum(0) / W + rest * w / W - E[heads].double().mean(0)) / B
    lost = K * 8192 * w / W * 0.3 * (1 if same else 1.2)         # (not same: 8 192 embeddings' mean is 0.3 +- 0.2 / 90, and the sum's own rounding)
    bound = (lost + 16 * 2.0 ** -24 * float(E[heads].abs().max())) / B
    assert float((du.double() - want).abs().max()) <= bound
    assert float(want.abs().max()) > 3 * bound                   # (the tail is what is looked at)
    assert abs(float(lse[0]) - math.log(W)) <= 4 * 2.0 ** -24 * math.log(W) + K * 8192 * w / W + 2.0 ** -20
