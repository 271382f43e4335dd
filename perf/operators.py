"""Distillation from a teacher's top logits over the whole catalogue (forward, and forward with backward), and sampling from scores with
temperature, top-k, top-p and min-p: the calls of unirec_amd.ops beside their plain forms."""
import math

import torch

own = False
DEV = "cuda:0"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _distill(name, B, N, d, K, train, bias=False, clip=0.0, tau=1.0, T=1.0, teacher="float32"):
    c = dict(op="distill", B=B, N=N, d=d, K=K, train=train, bias=bias, clip=clip, tau=tau, T=T, teacher=teacher)
    return dict(c, name=name) if name else c


def _sample(name, B, N, S, dtype, T=1.0, top_k=0, top_p=1.0, min_p=0.0):
    c = dict(op="sample", B=B, N=N, S=S, dtype=dtype, T=T, top_k=top_k, top_p=top_p, min_p=min_p)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a handful of users against the ML-100K-shaped catalogue: launch latency
        _distill("distill-step-small", 16, 1682, 64, 10, True),
        # the MF configuration's batch and catalogue, biases as that model has them
        _distill("distill-step-ml100k", 400, 1682, 64, 20, True, bias=True, tau=0.5, T=2.0),
        # the 60 K-item SASRec configuration, a teacher list of 50 stored in bfloat16
        _distill("distill-step-60k", 512, 60_000, 64, 50, True, teacher="bfloat16"),
        # odd sizes, clipped scores, a narrow model
        _distill("distill-step-odd", 333, 20_011, 48, 7, True, bias=True, clip=3.0, tau=0.7, T=1.5),
        # the 2 M-item configuration's batch: the table and its gradient are 2 GB
        _distill("distill-step-2m", 128, 2_000_000, 128, 100, True),
        # the largest: a wide batch over a million items
        _distill("distill-step-1m", 512, 1_000_000, 128, 100, True, T=2.0),
        # the loss alone, as a validation pass takes it
        _distill("distill-loss-1m", 512, 1_000_000, 128, 100, False, T=2.0),
        # one user's slate out of a retrieved list: latency
        _sample("sample-one-user", 1, 1000, 10, "float32", T=0.8, top_k=50, top_p=0.95),
        # a batch of users, slates of ten out of retrieved lists of 1000
        _sample("sample-retrieved", 512, 1000, 10, "float32", T=0.9, top_p=0.9),
        # scores of the whole 60 K catalogue in bfloat16, every filter on
        _sample("sample-60k-bf16", 256, 60_000, 4, "bfloat16", T=1.2, top_k=1000, top_p=0.95, min_p=0.01),
        # plain temperature sampling over a million items
        _sample("sample-1m-temperature", 64, 1_000_000, 4, "float32", T=1.0),
        # nucleus sampling over a million items
        _sample("sample-1m-nucleus", 64, 1_000_000, 1, "float32", T=0.7, top_p=0.9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        d = rng.choice([16, 32, 48, 64, 96, 100, 128, 128])
        N = _log(rng, 50, 1_000_000)
        B = max(1, min(_log(rng, 1, 1024), 512_000_000 // N))
        return _distill(None, B, N, d, min(_log(rng, 1, 100), N // 2), rng.random() < 0.75, rng.random() < 0.4, rng.choice([0.0, 0.0, 0.0, 4.0]),
                        round(rng.uniform(0.5, 1.5), 2), round(rng.uniform(0.8, 4.0), 2), rng.choice(sorted(TYPES)))
    N = _log(rng, 20, 1_000_000)
    B = max(1, min(_log(rng, 1, 512), 64_000_000 // N))
    return _sample(None, B, N, _log(rng, 1, 16), rng.choice(sorted(TYPES)), round(rng.uniform(0.3, 2.0), 2),
                   rng.choice([0, _log(rng, 1, min(N, 5000))]), rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                   rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.2), 3)]))


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    B, N = case["B"], case["N"]
    if case["op"] == "sample":
        # the scores of a trained model (a few units wide), items of the history masked out, and a user with nothing left to show
        x = randn(B, N) * 2.0
        x.masked_fill_(torch.rand(B, N, generator=g, device=DEV) < 0.02, -math.inf)
        if B >= 8:
            x[B // 2] = -math.inf
        return dict(case=case, scores=x.to(TYPES[case["dtype"]]), rand=torch.rand(B, case["S"], generator=g, device=DEV))
    d, K = case["d"], case["K"]
    table = randn(N, d) * 0.25
    table[0] = 0.0                                                        # the padding row
    user = randn(B, d) * (8.0 / math.sqrt(d))
    # the teacher's list: distinct items in no order of their own, scores descending; some lists are short, one is empty
    start = torch.randint(0, N - 1, (B, 1), generator=g, device=DEV)
    step = torch.arange(K, device=DEV) * max(1, (N - 1) // (K + 1))
    ids = (start + step) % (N - 1) + 1
    score = (randn(B, K) * 2.0 + 5.0).sort(dim=1, descending=True).values
    short = torch.where(torch.rand(B, 1, generator=g, device=DEV) < 0.1, torch.randint(1, K + 1, (B, 1), generator=g, device=DEV), K)
    if B >= 8:
        short[B // 3] = 0
    absent = torch.arange(K, device=DEV) >= short
    ids = ids.masked_fill(absent, -1)
    score = score.masked_fill(absent, -math.inf).to(TYPES[case["teacher"]])
    bias = randn(N) * 0.3 if case["bias"] else None
    return dict(case=case, user=user, table=table, bias=bias, ids=ids, score=score)


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_distill(case, user, table, bias, ids, score):
    tau, T, clip, B = case["tau"], case["T"], case["clip"], case["B"]
    s = user @ table.t()
    if bias is not None:
        s = s + bias
    s = s / tau
    inside = None
    if clip > 0:
        inside = (s <= clip) & (s >= -clip)
        s = torch.clamp(s, -clip, clip)
    s = s / T
    m = s.amax(dim=1, keepdim=True)
    e = torch.exp(s - m)
    total = e.sum(dim=1, keepdim=True)
    lse = m + torch.log(total)
    t = score.float() / T
    here = (ids >= 1) & (t > -math.inf)
    t = torch.where(here, t, -math.inf)
    some = here.any(dim=1, keepdim=True)
    top = torch.where(some, t.amax(dim=1, keepdim=True), 0.0)
    w = torch.exp(t - top)
    mass = torch.where(some, w.sum(dim=1, keepdim=True), 1.0)
    p = w / mass
    logp = torch.where(here, t - top - torch.log(mass), 0.0)
    at = ids.clamp(min=0)
    term = p * (logp - s.gather(1, at) + lse)
    count = some.sum().clamp(min=1)
    loss = T * T * torch.where(here, term, 0.0).sum() / count
    lse = lse.squeeze(1)
    if not case["train"]:
        return dict(loss=loss, lse=lse)
    q = torch.where(some, e / total, 0.0)
    q.scatter_add_(1, at, torch.where(here, -p, 0.0))
    if inside is not None:
        q = torch.where(inside, q, 0.0)
    q = q * (T / (count * tau))
    d_table = q.t() @ user
    d_table[0] = 0.0
    # the sum over the catalogue is long: partial sums of 4096 items each, added afterwards
    n, whole = 4096, q.shape[1] // 4096 * 4096
    d_user = q[:, whole:] @ table[whole:]
    if whole:
        d_user = d_user + torch.bmm(q[:, :whole].reshape(B, -1, n).transpose(0, 1), table[:whole].view(-1, n, table.shape[1])).sum(dim=0)
    out = dict(loss=loss, lse=lse, d_user=d_user, d_table=d_table)
    if bias is not None:
        out["d_item_bias"] = q.sum(dim=0)
    return out


def _plain_sample(case, scores, rand):
    T, top_k, top_p, min_p = case["T"], case["top_k"], case["top_p"], case["min_p"]
    B, N = scores.shape
    x = scores.double()                                                   # sums next to a border: 64 bits
    m = x.amax(dim=1, keepdim=True)
    some = m > -math.inf
    z = torch.where(some, (x - torch.where(some, m, 0.0)) / T, -math.inf)
    w = torch.exp(z)
    if top_k > 0 or top_p < 1.0:
        val, order = torch.sort(z, dim=1, descending=True, stable=True)
        first = torch.exp(val)
        if top_k > 0:
            first = torch.where(torch.arange(N, device=x.device) < top_k, first, 0.0)
        if top_p < 1.0:
            upto = torch.cumsum(first, dim=1)
            before = torch.cat([torch.zeros_like(upto[:, :1]), upto[:, :-1]], dim=1)
            first = torch.where(before < top_p * upto[:, -1:], first, 0.0)
        w = torch.zeros_like(w).scatter_(1, order, first)
    if min_p > 0.0:
        w = torch.where(w >= min_p, w, 0.0)
    upto = torch.cumsum(w, dim=1)
    total = upto[:, -1:]
    index = torch.searchsorted(upto, rand.double() * total, right=True)
    logp = (z.gather(1, index.clamp(max=N - 1)) - torch.log(total)).float()
    return dict(index=torch.where(some, index, -1), logp=torch.where(some, logp, -math.inf))


def run(state):
    case = state["case"]
    if case["op"] == "sample":
        if own:
            from unirec_amd import ops
            index, logp = ops.sample_scores(state["scores"], state["rand"], temperature=case["T"], top_k=case["top_k"], top_p=case["top_p"],
                                            min_p=case["min_p"])
            return dict(index=index, logp=logp)
        return _plain_sample(case, state["scores"], state["rand"])
    if own:
        from unirec_amd import ops
        kw = dict(item_bias=state["bias"], tau=case["tau"], score_clip=case["clip"], temperature=case["T"])
        loss_out, lse, saved = ops.full_distill_fwd(state["user"], state["table"], state["ids"], state["score"], need_grad=case["train"], **kw)
        if not case["train"]:
            return dict(loss=loss_out[0], lse=lse)
        d_user, d_table, d_bias = ops.full_distill_bwd(state["user"], state["table"], state["ids"], lse, loss_out, saved, **kw)
        out = dict(loss=loss_out[0], lse=lse, d_user=d_user, d_table=d_table)
        return dict(out, d_item_bias=d_bias) if d_bias is not None else out
    return _plain_distill(case, state["user"], state["table"], state["bias"], state["ids"], state["score"])


def work(case):
    B, N = case["B"], case["N"]
    if case["op"] == "sample":
        size = 4 if case["dtype"] == "float32" else 2
        return dict(bytes=B * N * size + B * case["S"] * 16, flops=2 * B * N)
    d, K = case["d"], case["K"]
    read = 4 * (N * d + B * d + (N if case["bias"] else 0)) + B * K * (8 + (4 if case["teacher"] == "float32" else 2)) + 4 * B
    if not case["train"]:
        return dict(bytes=read, flops=2 * B * N * d)
    return dict(bytes=read + 4 * (N * d + B * d + (N if case["bias"] else 0)), flops=6 * B * N * d)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _exact_sample(case, scores, rand):
    """row by row: the cut is found among the distinct values, ties by index; no weight is moved out of its place"""
    T, top_k, top_p, min_p = case["T"], case["top_k"], case["top_p"], case["min_p"]
    B, N = scores.shape
    index = torch.full((B, rand.shape[1]), -1, dtype=torch.int64, device=scores.device)
    logp = torch.full((B, rand.shape[1]), -math.inf, dtype=torch.float64, device=scores.device)
    for b in range(B):
        at = torch.nonzero(scores[b] > -math.inf).squeeze(1)
        if at.numel() == 0:
            continue
        z = scores[b][at].double()
        z = (z - z.max()) / T
        by = torch.argsort(-z, stable=True)
        if top_k > 0:
            by = by[:top_k]
        w = z[by].exp()
        if top_p < 1.0:
            run_sum = w.cumsum(0)
            by = by[: int(((run_sum - w) < top_p * run_sum[-1]).sum())]
        if min_p > 0.0:
            by = by[z[by].exp() >= min_p]
        by = by.sort().values
        c = z[by].exp().cumsum(0)
        pick = (c.unsqueeze(0) <= rand[b].double().unsqueeze(1) * c[-1]).sum(dim=1)
        index[b] = at[by[pick]]
        logp[b] = z[by[pick]] - c[-1].log()
    return dict(index=index, logp=logp)


def _exact_distill(case, user, table, bias, ids, score):
    """user block by user block, in 64 bits; the gradient of the scores is written out as softmax minus teacher"""
    tau, T, clip, B, N, d = (case[k] for k in ("tau", "T", "clip", "B", "N", "d"))
    U, E = user.double(), table.double()
    here = (ids >= 1) & (score.double() > -math.inf)
    count = max(1, int(here.any(dim=1).sum()))
    loss, lse, d_user = 0.0, [], []
    d_table = torch.zeros(N, d, dtype=torch.float64, device=user.device)
    d_bias = torch.zeros(N, dtype=torch.float64, device=user.device)
    block = max(1, min(B, 128_000_000 // N))
    for b0 in range(0, B, block):
        rows = slice(b0, min(B, b0 + block))
        raw = torch.mm(U[rows], E.t())
        if bias is not None:
            raw += bias.double()
        raw /= tau
        z = (raw.clamp(-clip, clip) if clip > 0 else raw) / T
        norm = torch.logsumexp(z, dim=1)
        lse.append(norm)
        teacher = torch.softmax(torch.where(here[rows], score[rows].double() / T, -1e300), dim=1) * here[rows]
        at = torch.where(here[rows], ids[rows], 0)
        log_ratio = torch.log(torch.where(teacher > 0, teacher, 1.0)) - z.gather(1, at) + norm.unsqueeze(1)
        loss = loss + (teacher * log_ratio).sum()
        if case["train"]:
            grad = torch.exp(z - norm.unsqueeze(1)) * here[rows].any(dim=1, keepdim=True)
            grad.scatter_add_(1, at, -teacher)
            if clip > 0:
                grad *= raw.abs() <= clip
            grad *= T / (count * tau)
            d_user.append(grad @ E)
            d_table += grad.t() @ U[rows]
            d_bias += grad.sum(dim=0)
    out = dict(loss=loss * T * T / count, lse=torch.cat(lse))
    if case["train"]:
        d_table[0] = 0.0
        out.update(d_user=torch.cat(d_user), d_table=d_table)
        if bias is not None:
            out["d_item_bias"] = d_bias
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(case, s["scores"], s["rand"])
    return _exact_distill(case, s["user"], s["table"], s["bias"], s["ids"], s["score"])
