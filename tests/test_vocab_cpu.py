"""Top log-probabilities, the divergence from them and filtered sampling: their plain forms against loops over the definitions, and what is refused."""
import math

import pytest
import torch

from nanorlhf_b200 import ops
from nanorlhf_b200.ops import reference as ref

INF = math.inf


def _top(row, k, temperature):
    order = sorted(range(len(row)), key=lambda i: (-row[i], i))
    z = sum(math.exp((x - max(row)) / temperature) for x in row)
    return [((row[i] - max(row)) / temperature - math.log(z), i) for i in order[:k]]


def _kept(row, temperature, top_k, top_p, min_p):
    order = sorted((i for i in range(len(row)) if row[i] > -INF), key=lambda i: (-row[i], i))
    w = {i: math.exp((row[i] - row[order[0]]) / temperature) for i in order}
    order = [i for i in order if w[i] >= min_p]
    if top_k:
        order = order[:top_k]
    if top_p < 1.0:
        whole, n, mass = sum(w[i] for i in order), 0, 0.0
        while n == 0 or (n < len(order) and mass < top_p * whole):
            mass += w[order[n]]
            n += 1
        order = order[:n]
    return sorted(order), w


@pytest.mark.parametrize("temperature", [0.5, 1.0, 1.7])
def test_top_logprobs_by_the_definition(temperature):
    g = torch.Generator().manual_seed(1)
    z = (torch.randn(6, 40, generator=g) * 4).round() / 2          # many ties
    logp, idx = ops.top_logprobs(z, 13, temperature)
    for r in range(6):
        want = _top(z[r].tolist(), 13, temperature)
        assert idx[r].tolist() == [i for _, i in want]
        assert torch.allclose(logp[r].double(), torch.tensor([x for x, _ in want], dtype=torch.float64), atol=1e-6)


def test_top_logprobs_lists_no_token_without_mass():
    z = torch.full((2, 9), -INF)
    z[0, [7, 2]] = torch.tensor([1.0, 1.0])
    logp, idx = ops.top_logprobs(z, 4)
    assert idx.tolist() == [[2, 7, -1, -1], [-1] * 4]
    assert torch.allclose(logp[0, :2], torch.tensor(0.5).log()) and (logp[0, 2:] == -INF).all() and (logp[1] == -INF).all()


@pytest.mark.parametrize("temperature", [0.6, 1.0])
@pytest.mark.parametrize("top_k", [0, 1, 5])
@pytest.mark.parametrize("top_p", [0.3, 0.9, 1.0])
@pytest.mark.parametrize("min_p", [0.0, 0.05])
def test_sampling_by_the_definition(temperature, top_k, top_p, min_p):
    g = torch.Generator().manual_seed(2)
    z = (torch.randn(20, 31, generator=g) * 3).round() / 2
    z[3, ::2] = -INF
    u = torch.rand(20, generator=g)
    tok, logp = ops.sample_filtered(z, u, temperature, top_k, top_p, min_p)
    for r in range(20):
        kept, w = _kept(z[r].tolist(), temperature, top_k, top_p, min_p)
        whole, mass = sum(w[i] for i in kept), 0.0
        for i in kept:
            mass += w[i]
            if mass > u[r].item() * whole:
                break
        assert tok[r].item() == i
        assert abs(logp[r].item() - math.log(w[i] / whole)) < 1e-6


def test_sampling_frequencies():
    z = torch.tensor([[0.0, 1.0, 2.0, -1.0, 0.5]]).expand(4096, 5)
    tok, _ = ops.sample_filtered(z, (torch.arange(4096) + 0.5) / 4096, top_k=3)
    share = torch.bincount(tok, minlength=5) / 4096
    w = torch.tensor([0.0, 1.0, 2.0, -INF, 0.5]).exp()
    w[0] = 0.0
    assert (share - w / w.sum()).abs().max() < 2 / 4096           # the numbers are evenly spread: a share is off by a step at each end


def test_sampling_edges():
    z = torch.tensor([[1.0, 3.0, 3.0, math.nan], [-INF, math.nan, -INF, -INF], [INF, 0.0, INF, 1.0]])
    tok, logp = ops.sample_filtered(z, torch.tensor([0.999, 0.5, 0.6]))
    assert tok.tolist() == [2, -1, 2] and logp[1].item() == -INF and abs(logp[2].item() - math.log(0.5)) < 1e-6
    tok, logp = ops.sample_filtered(z, torch.tensor([0.999, 0.5, 0.6]), temperature=0.0)
    assert tok.tolist() == [1, -1, 0] and logp[0].item() == 0.0
    tok, _ = ops.sample_filtered(z[:1], torch.tensor([0.999]), top_p=0.0)
    assert tok.item() == 1
    each = torch.tensor([5.0, float("nan"), -1.0])                 # beyond the range: min_p as 1, then left out twice
    tok, _ = ops.sample_filtered(torch.zeros(3, 4), torch.tensor([0.0, 0.99, 0.99]), min_p=each)
    assert tok.tolist() == [0, 3, 3]


def _loss(row, logp, idx, temperature, beta, tail):
    """of one token, by buckets, in Python floats"""
    z = [x / temperature for x in row]
    lse = max(z) + math.log(sum(math.exp(x - max(z)) for x in z))
    P, K = {}, []
    for a, i in zip(logp, idx):
        if 0 <= i < len(row):
            P[i] = P.get(i, 0.0) + math.exp(a)
            K.append(i)
    K = sorted(set(K))
    if not tail:
        whole = sum(P.values())
        return sum(P[i] / whole * (math.log(P[i] / whole) - (z[i] - lse)) for i in K)
    p = [P[i] for i in K] + [max(0.0, 1.0 - sum(P.values()))]
    q = [math.exp(z[i] - lse) for i in K] + [sum(math.exp(z[i] - lse) for i in range(len(row)) if i not in K)]
    m = [beta * a + (1 - beta) * b for a, b in zip(p, q)]
    if beta == 0.0:
        return sum(a * math.log(a / b) for a, b in zip(p, q) if a > 0)
    if beta == 1.0:
        return sum(b * math.log(b / a) for a, b in zip(p, q) if b > 0)
    return beta * sum(a * math.log(a / c) for a, c in zip(p, m) if a > 0) + (1 - beta) * sum(b * math.log(b / c) for b, c in zip(q, m) if b > 0)


@pytest.mark.parametrize("beta,tail", [(0.0, True), (0.0, False), (1.0, True), (0.3, True)])
@pytest.mark.parametrize("temperature", [1.0, 1.6])
def test_distillation_by_the_definition(beta, tail, temperature):
    g = torch.Generator().manual_seed(3)
    z = torch.randn(5, 12, generator=g, dtype=torch.float64)
    logp, idx = ops.top_logprobs(z + 0.5 * torch.randn(5, 12, generator=g, dtype=torch.float64), 4)
    idx = idx.clone()
    idx[1, 2] = -1                                                 # not a token
    idx[2, 3] = idx[2, 0]                                          # one token twice
    w = torch.tensor([0.5, 0.0, 1.0, 2.0, 0.25])
    x = z.clone().requires_grad_()
    loss, token = ops.distill_loss(x, logp, idx, w, temperature, beta, tail)
    loss.backward()
    want = [_loss(z[r].tolist(), logp[r].tolist(), idx[r].tolist(), temperature, beta, tail) if w[r] else 0.0 for r in range(5)]
    assert torch.allclose(token.double(), torch.tensor(want, dtype=torch.float64), atol=1e-6)
    assert abs(loss.item() - sum(a * b for a, b in zip(want, w.tolist()))) < 1e-6
    # the gradient against differences: double arithmetic, step 1e-5, so that both the step's square and rounding stay below 1e-8
    h = 1e-5
    for r in (0, 1, 2):
        for v in range(12):
            up, dn = z[r].tolist(), z[r].tolist()
            up[v] += h
            dn[v] -= h
            d = (_loss(up, logp[r].tolist(), idx[r].tolist(), temperature, beta, tail) - _loss(dn, logp[r].tolist(), idx[r].tolist(), temperature, beta, tail)) / (2 * h)
            assert abs(x.grad[r, v].item() - w[r].item() * d) < 1e-7


def test_distillation_without_a_teacher_or_a_tail():
    z = torch.randn(3, 6, dtype=torch.float64, requires_grad=True)
    none = torch.full((3, 2), -1, dtype=torch.int32)
    for beta, tail in ((0.0, True), (0.0, False), (1.0, True), (0.5, True)):
        loss, token = ops.distill_loss(z, torch.zeros(3, 2), none, beta=beta, tail=tail)
        (g,) = torch.autograd.grad(loss, z)
        # the bucket's mass, the sum of all q, is 1 up to rounding, in which the gradient is of the size of that rounding too
        assert token.abs().max() < 1e-12 and g.abs().max() < 1e-12
    every = torch.arange(6, dtype=torch.int32).expand(3, 6)
    logp = torch.log_softmax(torch.randn(3, 6), -1)
    for beta in (0.0, 1.0, 0.5):                                   # no token outside the teacher's
        loss, token = ops.distill_loss(z, logp, every, beta=beta)
        assert torch.isfinite(token).all() and (token > 0).all()


def test_refusals():
    z, u = torch.zeros(3, 8), torch.zeros(3)
    for bad in (dict(k=0), dict(k=9), dict(k=2, temperature=0.0), dict(k=2, temperature=INF), dict(k=2, temperature=math.nan)):
        with pytest.raises(ValueError):
            ops.top_logprobs(z, **bad)
    with pytest.raises(ValueError):
        ops.top_logprobs(z[0], 2)
    logp, idx = ops.top_logprobs(z, 2)
    for args, kw in (((logp[:2], idx[:2]), {}), ((logp, idx[:, :1]), {}), ((logp, idx), dict(beta=1.5)), ((logp, idx), dict(beta=-0.1)),
                     ((logp, idx), dict(beta=0.5, tail=False)), ((logp, idx), dict(temperature=-1.0)), ((logp, idx, torch.ones(2)), {}),
                     ((logp[:, :0], idx[:, :0]), {}), ((logp, idx), dict(beta=math.nan))):
        with pytest.raises(ValueError):
            ops.distill_loss(z, *args, **kw)
        with pytest.raises(ValueError):
            ops.lmhead_distill_loss(torch.zeros(3, 4), torch.zeros(8, 4), *args, **kw)
    with pytest.raises(TypeError):
        ops.distill_loss(z, logp, idx.float())
    with pytest.raises(ValueError):
        ops.lmhead_distill_loss(torch.zeros(3, 4), torch.zeros(8, 5), logp, idx)
    with pytest.raises(ValueError):
        ops.lmhead_top_logprobs(torch.zeros(3, 4), torch.zeros(8, 4), 9)
    for kw in (dict(temperature=-1.0), dict(top_k=-1), dict(top_p=1.1), dict(top_p=-0.1), dict(min_p=2.0), dict(temperature=math.nan), dict(top_p=math.nan),
               dict(top_p=torch.ones(2)), dict(top_k=torch.ones(3)), dict(min_p=torch.ones(3, dtype=torch.float64))):
        with pytest.raises(ValueError):
            ops.sample_filtered(z, u, **kw)
    with pytest.raises(ValueError):
        ops.sample_filtered(z, u[:2])
    with pytest.raises(TypeError):
        ops.sample_filtered(z, u.double())


def test_empty_batches():
    assert [tuple(t.shape) for t in ops.top_logprobs(torch.zeros(0, 8), 3)] == [(0, 3), (0, 3)]
    assert [tuple(t.shape) for t in ops.sample_filtered(torch.zeros(0, 8), torch.zeros(0))] == [(0,), (0,)]
    z = torch.zeros(0, 8, requires_grad=True)
    loss, token = ops.distill_loss(z, torch.zeros(0, 2), torch.zeros(0, 2, dtype=torch.int32))
    loss.backward()
    assert loss.item() == 0.0 and token.numel() == 0 and z.grad.shape == (0, 8)


def test_row_ranges_cover_the_rows():
    from nanorlhf_b200.ops import native
    for rows in (0, 1, 255, 7065, 7066, 7067, 40000):
        got = native._row_ranges(rows, 151936)
        assert [s for s, _ in got] == [0] * bool(rows) + [e for _, e in got[:-1]] and (got[-1][1] if got else 0) == rows
        assert all(e > s and 4 * 151936 * (e - s) <= native.LOGITS_BYTES for s, e in got)
