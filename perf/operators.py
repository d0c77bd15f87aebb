"""What is timed of the operators around a distribution over the vocabulary that another model gives, or that a sampler cuts.

A teacher's top log-probabilities per token (``ops.top_logprobs``), the divergence of a student from them with its gradient
(``ops.distill_loss`` from logits, ``ops.lmhead_distill_loss`` from hidden states and the head), and one token per row under
temperature, top-k, top-p and min-p from given uniform numbers (``ops.sample_filtered``).

With ``own`` false ``run`` is their plain form in torch, with ``own`` true the calls that a user makes.  ``exact`` gives the same
outputs from the definitions in float64.
"""
import math
import random

import torch

own = False

DEV = "cuda"
VOCAB = 151936                      # the default policy's vocabulary
HIDDEN = 1536                       # and its hidden size
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # a served token with its twenty most probable alternatives: the smallest call
        {"name": "top_one_token", "op": "top", "rows": 1, "vocab": VOCAB, "k": 20, "dtype": "bf16", "temperature": 1.0, "shape": "peaked"},
        # the teacher's pass over the responses of a micro-step
        {"name": "top_micro_step", "op": "top", "rows": 2048, "vocab": VOCAB, "k": 64, "dtype": "bf16", "temperature": 1.0, "shape": "peaked"},
        # an odd vocabulary whose rows start at any alignment, many entries kept, logits in float
        {"name": "top_odd_vocab", "op": "top", "rows": 777, "vocab": 50021, "k": 200, "dtype": "fp32", "temperature": 0.7, "shape": "flat"},
        # the loss of a few tokens over a small vocabulary: latency
        {"name": "distill_few", "op": "distill", "rows": 48, "vocab": 32000, "k": 16, "dtype": "fp32", "temperature": 1.0, "beta": 0.0, "tail": True, "shape": "peaked"},
        # a micro-step's tokens over the whole vocabulary, forward and backward, mean over the tokens
        {"name": "distill_micro_step", "op": "distill", "rows": 2048, "vocab": VOCAB, "k": 64, "dtype": "bf16", "temperature": 1.0, "beta": 0.0, "tail": True, "shape": "peaked"},
        # the generalised divergence, odd vocabulary, float logits
        {"name": "distill_odd_vocab", "op": "distill", "rows": 1500, "vocab": 50021, "k": 100, "dtype": "fp32", "temperature": 2.0, "beta": 0.5, "tail": True, "shape": "flat"},
        # the same through the head, where no logits are handed over: a short response
        {"name": "head_short", "op": "head", "rows": 300, "vocab": VOCAB, "hidden": HIDDEN, "k": 64, "temperature": 1.0, "beta": 0.0, "tail": False},
        # and the responses of a micro-step: the largest
        {"name": "head_micro_step", "op": "head", "rows": 4011, "vocab": VOCAB, "hidden": HIDDEN, "k": 64, "temperature": 1.0, "beta": 1.0, "tail": True},
        # one sequence being served
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": VOCAB, "dtype": "bf16", "per_row": False, "temperature": 0.7, "top_k": 50, "top_p": 0.95, "min_p": 0.0, "shape": "peaked"},
        # a decode step of a full batch
        {"name": "sample_batch", "op": "sample", "rows": 1024, "vocab": VOCAB, "dtype": "bf16", "per_row": False, "temperature": 0.9, "top_k": 50, "top_p": 0.95, "min_p": 0.0, "shape": "peaked"},
        # requests of different users in one batch, each with filters of its own or none, float logits
        {"name": "sample_mixed", "op": "sample", "rows": 250, "vocab": 50021, "dtype": "fp32", "per_row": True, "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "shape": "peaked"},
        # a nucleus without other filters over an untrained policy's flat distribution: most tokens are kept
        {"name": "sample_flat_nucleus", "op": "sample", "rows": 256, "vocab": VOCAB, "dtype": "bf16", "per_row": False, "temperature": 1.0, "top_k": 0, "top_p": 0.95, "min_p": 0.0, "shape": "flat"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["top", "distill", "head", "sample"])
    vocab = rng.choice([VOCAB, rng.randint(1000, 151936), _log(rng, 1000, 151936)])
    c = {"op": op, "rows": _log(rng, 1, 2048), "vocab": vocab, "dtype": rng.choice(["bf16", "fp32"]), "shape": rng.choice(["peaked", "peaked", "flat"]),
         "temperature": rng.choice([1.0, round(rng.uniform(0.5, 2.0), 2)])}
    if op == "sample":
        c.update(rows=_log(rng, 1, 1024), per_row=rng.random() < 0.3, top_k=rng.choice([0, 0, _log(rng, 1, 400)]),
                 top_p=rng.choice([1.0, round(rng.uniform(0.5, 0.99), 3)]), min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.2), 3)]))
        return c
    c["k"] = _log(rng, 1, 256)
    if op != "top":
        c.update(beta=rng.choice([0.0, 0.0, 1.0, round(rng.uniform(0.1, 0.9), 2)]), tail=True)
        if c["beta"] == 0.0:
            c["tail"] = rng.random() < 0.5
    if op == "head":
        c.update(rows=_log(rng, 1, 4000), vocab=max(1000, vocab // 8 * 8), hidden=rng.choice([HIDDEN, 64 * rng.randint(4, 24)]))
        for key in ("dtype", "shape"):
            del c[key]
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------------------------
def _logits(g, rows, vocab, shape, dtype):
    """peaked: a trained model's row, some tens of likely tokens above a wide rest; flat: an untrained one's."""
    z = torch.randn(rows, vocab, generator=g, device=DEV) * (1.8 if shape == "peaked" else 0.6)
    if shape == "peaked":
        head = min(48, vocab)
        step = vocab // head
        at = torch.randint(0, step, (rows, head), generator=g, device=DEV) + step * torch.rand(rows, head, generator=g, device=DEV).argsort(-1)
        up = 16.0 * torch.rand(rows, head, generator=g, device=DEV) * torch.linspace(1.0, 0.3, head, device=DEV)
        z.scatter_(1, at, up + z.gather(1, at))
    return z.to(dtype)


def _teacher(g, z, k, noise):
    """top log-probabilities of a teacher that mostly agrees with the student's logits"""
    logp, idx = [], []
    for part in z.split(256):
        t = part.float() + noise * torch.randn(part.shape, generator=g, device=DEV)
        v, i = torch.log_softmax(t, -1).topk(k, -1)
        logp.append(v)
        idx.append(i.int())
    return torch.cat(logp), torch.cat(idx)


def _weights(g, rows):
    """mean over the tokens that count; a few are masked"""
    m = (torch.rand(rows, generator=g, device=DEV) > 0.1).float()
    m[0] = 1.0
    return m / m.sum()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    st = {"case": case}
    rows, vocab = case["rows"], case["vocab"]
    if case["op"] == "head":
        st["hidden"] = torch.randn(rows, case["hidden"], generator=g, device=DEV).to(torch.bfloat16)
        st["weight"] = (torch.randn(vocab, case["hidden"], generator=g, device=DEV) * (2.0 / math.sqrt(case["hidden"]))).to(torch.bfloat16)
        parts = [_teacher(g, (h @ st["weight"].t()), case["k"], 0.5) for h in st["hidden"].split(1024)]
        st["logp"], st["idx"] = torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
        st["weights"] = _weights(g, rows)
        return st
    st["logits"] = _logits(g, rows, vocab, case["shape"], TYPES[case["dtype"]])
    if case["op"] == "distill":
        st["logp"], st["idx"] = _teacher(g, st["logits"], case["k"], 0.5)
        st["weights"] = _weights(g, rows)
    if case["op"] == "sample":
        st["u"] = torch.rand(rows, generator=g, device=DEV)
        st["filters"] = {key: case[key] for key in ("temperature", "top_k", "top_p", "min_p")}
        if case["per_row"]:
            r = random.Random(seed)
            f = [{"temperature": r.choice([0.0, r.uniform(0.5, 1.5), r.uniform(0.5, 1.5)]), "top_k": r.choice([0, 0, r.randint(1, 300)]),
                  "top_p": r.choice([1.0, r.uniform(0.5, 0.98)]), "min_p": r.choice([0.0, 0.0, r.uniform(0.01, 0.2)])} for _ in range(rows)]
            st["filters"] = {key: torch.tensor([x[key] for x in f], device=DEV, dtype=torch.int32 if key == "top_k" else torch.float32) for key in f[0]}
    return st


# ---- plain forms -------------------------------------------------------------------------------------------------------------------
def _plain_top(logits, k, temperature):
    logp, idx = [], []
    for part in logits.split(256):
        z = part.float() / temperature
        m = z.amax(-1, keepdim=True)
        lse = m + (z - m).exp().sum(-1, keepdim=True).log()
        v, i = part.float().sort(dim=-1, descending=True, stable=True)
        v, i = v[:, :k] / temperature - lse, i[:, :k]
        logp.append(v)
        idx.append(torch.where(v == -math.inf, -1, i).int())
    return torch.cat(logp), torch.cat(idx)


def _plain_divergence(z, logp, idx, beta, tail):
    """token losses and dloss/dz of float logits that are divided by the temperature, in float64: a divergence is the small difference of large
    terms.  Entries of one row are distinct tokens."""
    z, logp = z.double(), logp.double()
    m = z.amax(-1, keepdim=True)
    e = (z - m).exp()
    total = e.sum(-1, keepdim=True)
    at = idx.long()
    inside = torch.zeros_like(z).scatter_(1, at, 1.0)
    q = e / total
    log_qk = z.gather(1, at) - m - total.log()
    p = logp.exp()
    if not tail:
        p = p / p.sum(-1, keepdim=True)
        return (p * (p.log() - log_qk)).sum(-1), q.scatter_add(1, at, -p)
    s = (e * (1.0 - inside)).sum(-1, keepdim=True) / total
    r = 1.0 - p.sum(-1, keepdim=True)
    r = torch.where(r > 2.0 ** -24, r, 0.0)
    if beta == 0.0:
        rest = torch.where(r > 0, r * (r / s).log(), 0.0)
        loss = (p * (logp - log_qk)).sum(-1) + rest.squeeze(-1)
        return loss, torch.where(inside > 0, q, q * (1.0 - r / s)).scatter_add(1, at, -p)
    qk = log_qk.exp()
    P, Q = torch.cat([p, r], -1), torch.cat([qk, s], -1)
    if beta == 1.0:
        D = torch.cat([log_qk - logp, s.log() - r.clamp_min(2.0 ** -24).log()], -1)
        loss = (Q * D).sum(-1)
    else:
        M = beta * P + (1.0 - beta) * Q
        D = (1.0 - beta) * (Q / M).log()
        loss = beta * torch.where(P > 0, P * (P / M).log(), 0.0).sum(-1) + (Q * D).sum(-1)
    mean = (Q * D).sum(-1, keepdim=True)
    dz = q * (D[:, -1:] - mean)
    return loss, dz.scatter(1, at, qk * (D[:, :-1] - mean))


def _plain_distill(st):
    c, losses, grads = st["case"], [], []
    for z, logp, idx, w in zip(st["logits"].split(256), st["logp"].split(256), st["idx"].split(256), st["weights"].split(256)):
        loss, dz = _plain_divergence(z.double() / c["temperature"], logp, idx, c["beta"], c["tail"])
        losses.append((loss * (w != 0)).float())
        grads.append((dz * (w / c["temperature"])[:, None]).to(z.dtype))
    token = torch.cat(losses)
    return (token.double() * st["weights"]).sum().float(), token, torch.cat(grads)


def _plain_head(st):
    c, w32 = st["case"], st["weight"].float()
    losses, dh, dw = [], [], torch.zeros_like(w32)
    for h, logp, idx, w in zip(st["hidden"].split(1024), st["logp"].split(1024), st["idx"].split(1024), st["weights"].split(1024)):
        h = h.float()
        loss, dz = _plain_divergence((h @ w32.t()).double() / c["temperature"], logp, idx, c["beta"], c["tail"])
        losses.append((loss * (w != 0)).float())
        dz = (dz * (w / c["temperature"])[:, None]).float()
        dh.append(dz @ w32)
        dw += dz.t() @ h
    token = torch.cat(losses)
    return (token.double() * st["weights"]).sum().float(), token, torch.cat(dh).to(st["hidden"].dtype), dw.to(st["weight"].dtype)


def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    rows, vocab = logits.shape
    row = lambda x: (x if torch.is_tensor(x) else torch.full((rows,), x, device=logits.device, dtype=torch.float64)).double()[:, None]  # noqa: E731
    temperature, top_k, top_p, min_p = row(temperature), row(top_k), row(top_p), row(min_p)
    tokens, logps = [], []
    rank = torch.arange(vocab, device=logits.device)
    for lo in range(0, rows, 64):
        hi = min(rows, lo + 64)
        T, K, P, M = temperature[lo:hi], top_k[lo:hi], top_p[lo:hi], min_p[lo:hi]
        z = logits[lo:hi].double()
        order = z.sort(dim=-1, descending=True, stable=True).indices
        best = order[:, :1]
        x = (z - z.gather(1, best)) / torch.where(T > 0, T, 1.0)
        w = x.exp().gather(1, order)
        keep = (w >= M) & ((rank < K) | (K <= 0))
        w = w * keep
        cum = w.cumsum(-1)
        keep &= (cum - w < P * cum[:, -1:]) | (P >= 1.0) | (rank == 0)
        kept = torch.zeros_like(keep).scatter_(1, order, keep)
        cum = (x.exp() * kept).cumsum(-1)
        token = (cum > u[lo:hi, None].double() * cum[:, -1:]).byte().argmax(-1, keepdim=True)
        logp = x.gather(1, token) - cum[:, -1:].log()
        tokens.append(torch.where(T > 0, token, best).int().squeeze(1))
        logps.append(torch.where(T > 0, logp, 0.0).float().squeeze(1))
    return torch.cat(tokens), torch.cat(logps)


# ---- one pass ----------------------------------------------------------------------------------------------------------------------
def run(state):
    c = state["case"]
    if own:
        return _own(state, c)
    with torch.no_grad():
        if c["op"] == "top":
            return _plain_top(state["logits"], c["k"], c["temperature"])
        if c["op"] == "distill":
            return _plain_distill(state)
        if c["op"] == "head":
            return _plain_head(state)
        return _plain_sample(state["logits"], state["u"], **state["filters"])


def _own(st, c):
    from nanorlhf_b200 import ops
    if c["op"] == "top":
        return ops.top_logprobs(st["logits"], c["k"], c["temperature"])
    if c["op"] == "sample":
        return ops.sample_filtered(st["logits"], st["u"], **st["filters"])
    if c["op"] == "distill":
        z = st["logits"].detach().requires_grad_()
        loss, token = ops.distill_loss(z, st["logp"], st["idx"], st["weights"], temperature=c["temperature"], beta=c["beta"], tail=c["tail"])
        loss.backward()
        return loss.detach(), token, z.grad
    h, w = st["hidden"].detach().requires_grad_(), st["weight"].detach().requires_grad_()
    loss, token = ops.lmhead_distill_loss(h, w, st["logp"], st["idx"], st["weights"], temperature=c["temperature"], beta=c["beta"], tail=c["tail"])
    loss.backward()
    return loss.detach(), token, h.grad, w.grad


def work(case):
    rows, vocab = case["rows"], case["vocab"]
    if case["op"] == "head":
        h = case["hidden"]
        return {"bytes": 2 * 2 * h * (rows + vocab) + rows * (8 * case["k"] + 8), "flops": 6 * rows * vocab * h}
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "top":
        return {"bytes": rows * (vocab * size + 8 * case["k"]), "flops": 4 * rows * vocab}
    if case["op"] == "distill":
        return {"bytes": rows * (2 * vocab * size + 8 * case["k"] + 8), "flops": 8 * rows * vocab}
    return {"bytes": rows * (vocab * size + 12), "flops": 2 * rows * vocab}


# ---- from the definitions, in float64 ----------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "top":
            return _exact_top(st["logits"], case)
        if case["op"] == "sample":
            return _exact_sample(st)
        return _exact_divergence(st, case)


def _exact_top(logits, case):
    logp, idx = [], []
    for z in logits.split(64):
        x = z.double()
        lp = torch.log_softmax(x / case["temperature"], -1)
        # descending values, then ascending indices: sort by index first, stably by value after
        order = torch.sort(-x, dim=-1, stable=True).indices[:, :case["k"]]
        v = lp.gather(1, order)
        logp.append(v)
        idx.append(order.masked_fill(torch.isneginf(v), -1).int())
    return torch.cat(logp), torch.cat(idx)


def _exact_divergence(st, case):
    """Losses by buckets as sums over a matrix of tokens; gradients by autograd of those in float64."""
    head = case["op"] == "head"
    rows, tau, beta = case["rows"], case["temperature"], case["beta"]
    token = torch.empty(rows, dtype=torch.float64, device=DEV)
    w64 = st["weight"].double() if head else None
    dw = torch.zeros_like(w64) if head else None
    grads = []
    step = 256 if head else 64
    for lo in range(0, rows, step):
        sl = slice(lo, min(rows, lo + step))
        x = (st["hidden"][sl].double() @ w64.t()) if head else st["logits"][sl].double()
        with torch.enable_grad():
            x.requires_grad_()
            lq = torch.log_softmax(x / tau, -1)
            at = st["idx"][sl].long()
            a = st["logp"][sl].double()
            lqk = lq.gather(1, at)
            if not case["tail"]:
                a = a - torch.logsumexp(a, -1, keepdim=True)
                per = (a.exp() * (a - lqk)).sum(-1)
            else:
                off = torch.ones_like(lq, dtype=torch.bool).scatter_(1, at, False)
                ls = torch.logsumexp(lq.masked_fill(~off, -math.inf), -1, keepdim=True)
                r = 1.0 - a.exp().sum(-1, keepdim=True)
                r = torch.where(r > 2.0 ** -24, r, torch.zeros_like(r))
                lP = torch.cat([a, r.clamp_min(2.0 ** -24).log()], -1)
                P = torch.cat([a.exp(), r], -1)
                lQ = torch.cat([lqk, ls], -1)
                if beta == 0.0:
                    per = (P * (lP - lQ)).sum(-1)
                elif beta == 1.0:
                    per = (lQ.exp() * (lQ - lP)).sum(-1)
                else:
                    lM = (beta * P + (1.0 - beta) * lQ.exp()).log()
                    per = beta * (P * (lP - lM)).sum(-1) + (1.0 - beta) * (lQ.exp() * (lQ - lM)).sum(-1)
            (dz,) = torch.autograd.grad((per * st["weights"][sl].double()).sum(), x)
        token[sl] = per.detach() * (st["weights"][sl] != 0)
        if head:
            grads.append(dz @ w64)
            dw += dz.t() @ st["hidden"][sl].double()
        else:
            grads.append(dz)
    loss = (token * st["weights"].double()).sum()
    return (loss, token, torch.cat(grads), dw) if head else (loss, token, torch.cat(grads))


def _exact_sample(st):
    rows = st["logits"].shape[0]
    f = {key: (v.tolist() if torch.is_tensor(v) else [v] * rows) for key, v in st["filters"].items()}
    tokens, logps = [], []
    for i, u in enumerate(st["u"].tolist()):
        z = st["logits"][i].double()
        if f["temperature"][i] == 0.0:
            tokens.append((z == z.max()).nonzero()[0])
            logps.append(torch.zeros(1, dtype=torch.float64, device=DEV))
            continue
        # the kept tokens are the first n of the order: shorten it filter by filter
        order = torch.sort(-z, stable=True).indices
        w = ((z[order] - z[order[0]]) / f["temperature"][i]).exp()
        if f["min_p"][i] > 0.0:
            order, w = order[w >= f["min_p"][i]], w[w >= f["min_p"][i]]
        if f["top_k"][i] > 0:
            order, w = order[:f["top_k"][i]], w[:f["top_k"][i]]
        if f["top_p"][i] < 1.0:
            n = 1 + int((w.cumsum(0)[:-1] < f["top_p"][i] * w.sum()).sum())
            order, w = order[:n], w[:n]
        by_index = order.sort().indices
        order, w = order[by_index], w[by_index]
        cum = w.cumsum(0)
        j = min(int(torch.searchsorted(cum, u * cum[-1], right=True)), w.numel() - 1)
        tokens.append(order[j:j + 1])
        logps.append((w[j] / cum[-1]).log()[None])
    return torch.cat(tokens).int(), torch.cat(logps)
