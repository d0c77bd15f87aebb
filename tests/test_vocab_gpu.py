"""The kernels over rows of logits against float64: where rows start and end, ties, masked tokens, filters, gradients, streams, graphs, and their use together."""
import math

import pytest
import torch

from nanorlhf_b200 import ops
from nanorlhf_b200.ops import reference as ref

pytestmark = pytest.mark.gpu

INF = math.inf
BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _place(z, skew, pad):
    """the same rows `pad` elements further apart, the first `skew` elements into its buffer"""
    T, V = z.shape
    buf = torch.full((T * (V + pad) + skew,), math.nan, dtype=z.dtype, device=z.device)
    out = buf[skew:skew + T * (V + pad)].view(T, V + pad)[:, :V]
    out.copy_(z)
    return out


PATTERNS = ["normal", "peaked", "wide", "ties", "constant", "rising", "falling", "masked", "lowest", "zeros"]


def _logits(pattern, T, V, dtype, seed=0):
    g = _gen(seed * 1000 + V)
    z = torch.randn(T, V, generator=g, device=DEV)
    if pattern == "peaked":
        z = z * 2 + 14.0 * (torch.rand(T, V, generator=g, device=DEV) > 0.999)
    if pattern == "wide":
        z = z * 30.0
    if pattern == "ties":
        z = (z * 2).round()
    if pattern == "constant":
        z = torch.full_like(z, -3.25)
    if pattern == "rising":
        z = torch.arange(V, device=DEV).float().mul(20.0 / V).expand(T, V).clone()
    if pattern == "falling":
        z = torch.arange(V, device=DEV).float().mul(-20.0 / V).expand(T, V).clone()
    if pattern == "masked":                                # few tokens left, none in the first row, one in the last
        z = z.masked_fill(torch.rand(T, V, generator=g, device=DEV) > 0.01, -INF)
        z[0] = -INF
        z[-1] = -INF
        z[-1, V // 2] = 1.5
    if pattern == "lowest":                                # a mask by the type's lowest number
        z = z.masked_fill(torch.rand(T, V, generator=g, device=DEV) > 0.01, torch.finfo(dtype).min)
    if pattern == "zeros":
        z = torch.where(torch.rand(T, V, generator=g, device=DEV) > 0.5, 0.0, -0.0)
    return z.to(dtype)


SIZES = [(3, 1, 0, 0), (2, 2, 1, 0), (5, 7, 3, 2), (3, 33, 0, 1), (4, 1000, 2, 0), (3, 4099, 1, 3), (2, 32000, 0, 0), (2, 50021, 5, 0), (2, 151936, 0, 8)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("T,V,skew,pad", SIZES)
def test_top_logprobs(T, V, skew, pad, pattern, dtype):
    z = _place(_logits(pattern, T, V, dtype), skew, pad)
    for k in sorted({1, min(V, 20), min(V, 129), min(V, 1024)}):
        logp, idx = ops.top_logprobs(z, k, 0.9)
        want, at = ref.top_logprobs(z.double(), k, 0.9)
        assert torch.equal(idx, at)
        # rounding of the result, half a step; of the row's sum: terms to 3 steps of 2^-24 of their exponents, which in the mean of the mass are log2 V <= 18
        # at most, 2^-22 for 2^x, and the sum's own: 5e-6 together
        live = at >= 0
        assert torch.equal(logp[~live], want[~live])
        # (log-probabilities beyond float's range are -inf on both sides)
        assert ((logp == want) | ((logp - want).abs() <= 5e-6 + 2.0 ** -23 * want.abs()))[live].all()


def test_top_logprobs_of_nan_and_infinity():
    z = _logits("normal", 4, 3000, F32)
    z[0, 1234] = math.nan
    z[1, [5, 2999]] = INF
    logp, idx = ops.top_logprobs(z, 7)
    assert logp[0].isnan().all() and idx[1, :2].tolist() == [5, 2999] and torch.equal(logp[1, :2], torch.full((2,), 0.5, device=DEV).log())
    want, at = ops.top_logprobs(z[2:].clone(), 7)
    assert torch.equal(logp[2:], want) and torch.equal(idx[2:], at)


def _same_draws(z, u, **kw):
    tok, logp = ops.sample_filtered(z, u, **kw)
    want, lw = ref.sample_filtered(z, u, **kw)
    assert torch.equal(tok, want), (tok != want).nonzero()[:8]
    ok = want >= 0
    assert torch.equal(logp[~ok], lw[~ok])
    assert ((logp == lw) | ((logp - lw).abs() <= 2e-7 + 2.0 ** -23 * lw.abs()))[ok].all()          # both from float64, rounded once


FILTERS = [dict(), dict(top_k=1), dict(top_k=50), dict(top_k=2000), dict(top_p=0.9), dict(top_p=0.2), dict(top_p=0.999), dict(min_p=0.1), dict(min_p=1e-5),
           dict(top_k=50, top_p=0.95), dict(top_k=40, top_p=0.8, min_p=0.02), dict(temperature=0.0), dict(temperature=0.3, top_p=0.95), dict(temperature=3.0, top_k=700),
           dict(min_p=1.0), dict(top_p=0.0)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("V,skew,pad", [(1, 0, 0), (7, 3, 2), (1000, 1, 0), (32000, 0, 0), (50021, 2, 1), (151936, 0, 0)])
def test_sampling(V, skew, pad, pattern, dtype):
    T = 6
    z = _place(_logits(pattern, T, V, dtype), skew, pad)
    u = torch.rand(T, generator=_gen(V), device=DEV)
    u[0], u[1] = 0.0, 1.0 - 2.0 ** -24
    for kw in FILTERS:
        _same_draws(z, u, **kw)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,V", [(300, 4096), (700, 50021)])
def test_sampling_with_filters_of_every_row(B, V, dtype):
    g = _gen(B)
    z = _logits("peaked", B, V, dtype, seed=1)
    u = torch.rand(B, generator=g, device=DEV)
    r = lambda: torch.rand(B, generator=g, device=DEV)  # noqa: E731
    t = torch.where(r() < 0.2, 0.0, 0.4 + r())
    k = torch.where(r() < 0.4, 0, (r() * 300).int() + 1).int()
    p = torch.where(r() < 0.3, 1.0, 0.4 + 0.6 * r())
    m = torch.where(r() < 0.5, 0.0, 0.2 * r())
    _same_draws(z, u, temperature=t, top_k=k, top_p=p, min_p=m)
    k[3], p[4], m[5], t[6] = -5, 7.0, math.nan, math.nan           # beyond the range
    _same_draws(z, u, temperature=t, top_k=k, top_p=p, min_p=m)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B", [15, 30, 100, 200])          # four, two blocks a row and one
@pytest.mark.parametrize("pattern", ["normal", "peaked", "ties"])
def test_sampling_of_many_kept_tokens(pattern, B, dtype):
    """nuclei of most of the vocabulary, no filters, and more tokens above min_p than are sorted"""
    z = _logits(pattern, B, 80000, dtype, seed=2)
    u = torch.rand(B, generator=_gen(B), device=DEV)
    for kw in (dict(), dict(top_p=0.97), dict(temperature=1.5, top_p=0.6), dict(min_p=0.05), dict(min_p=0.01, top_p=0.9)):
        _same_draws(z, u, **kw)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B", [8, 100])
@pytest.mark.parametrize("lift", [-8.0, 8.0, -math.inf])
def test_nuclei_of_rows_whose_fourth_is_unlike_the_rest(lift, B, dtype):
    """512 vectors of 32 bytes out of every 2048 lie elsewhere than the others, or have no mass: threads' chunks and warps' ranges of very different masses"""
    V = 151936
    z = _logits("normal", B, V, dtype, seed=3)
    part = torch.arange(V, device=DEV) // (512 * 32 // z.element_size()) % 4 == 0
    z = torch.where(part, z + lift, z)
    u = torch.rand(B, generator=_gen(B), device=DEV)
    for kw in (dict(top_p=0.95), dict(top_p=0.5), dict(top_p=1e-3), dict(top_p=0.9999), dict(min_p=1e-4, top_p=0.9)):
        _same_draws(z, u, **kw)


@pytest.mark.parametrize("temperature", [1e-300, 1e-42, 1e-30, 1e30])
@pytest.mark.parametrize("pattern", ["normal", "ties"])
def test_temperatures_far_from_one(pattern, temperature):
    z = _logits(pattern, 4, 30000, F32)
    u = torch.rand(4, generator=_gen(3), device=DEV)
    for kw in (dict(), dict(top_p=0.9), dict(top_k=40), dict(top_k=40, top_p=0.3), dict(min_p=0.5)):
        _same_draws(z, u, temperature=temperature, **kw)
    if temperature >= 1e-42:
        _same_draws(z, u, temperature=torch.full((4,), temperature, device=DEV), top_p=torch.full((4,), 0.7, device=DEV))
    logp, idx = ops.top_logprobs(z, 9, temperature)
    want, at = ref.top_logprobs(z, 9, temperature)
    assert torch.equal(idx, at) and ((logp == want) | ((logp - want).abs() <= 5e-6 + 2.0 ** -23 * want.abs())).all()


def test_sampling_edges():
    z = torch.tensor([[1.0, 3.0, 3.0, math.nan], [-INF, math.nan, -INF, -INF], [INF, 0.0, INF, 1.0], [-2.0, -2.0, -INF, -2.0]], device=DEV)
    for u in ([0.999, 0.5, 0.6, 0.34], [0.0, 0.0, 0.0, 0.0], [0.2, 0.2, 0.2, 0.67]):
        for kw in FILTERS:
            _same_draws(z, torch.tensor(u, device=DEV), **kw)


@pytest.mark.parametrize("kw", [dict(top_p=0.95), dict(), dict(top_k=50, top_p=0.95)])
def test_sampling_frequencies(kw):
    """evenly spread numbers give every kept token its share, one row of logits for all of them"""
    n, V = 20000, 1031
    z = _logits("peaked", 1, V, F32).expand(n, V)
    tok, _ = ops.sample_filtered(z, (torch.arange(n, device=DEV) + 0.5) / n, 0.8, **kw)
    share = torch.bincount(tok, minlength=V) / n
    w = (z[0].double() / 0.8).softmax(0)
    order = w.argsort(descending=True)
    if "top_k" in kw:
        w[order[kw["top_k"]:]] = 0
        w /= w.sum()
    if "top_p" in kw:
        c = w[order].cumsum(0)
        w[order[c - w[order] >= kw["top_p"]]] = 0
        w /= w.sum()
    assert (share - w).abs().max() <= 2.0 / n


def _teacher(z, K, temperature=1.0, seed=5):
    t = z.float() + 0.5 * torch.randn(z.shape, generator=_gen(seed), device=DEV)
    return ops.top_logprobs(t, K, temperature)


BETAS = [(0.0, True), (0.0, False), (1.0, True), (0.4, True)]


def _rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-30)).item()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("beta,tail", BETAS)
@pytest.mark.parametrize("T,V,K,skew,pad", [(3, 1, 1, 0, 0), (4, 7, 3, 1, 2), (5, 1000, 16, 3, 0), (3, 4099, 64, 0, 1), (4, 50021, 100, 1, 0), (2, 151936, 64, 0, 0), (2, 32000, 1024, 0, 8)])
def test_distillation(T, V, K, skew, pad, beta, tail, dtype):
    z = _logits("peaked", T, V, dtype)
    logp, idx = _teacher(z, K, 1.3)
    idx = idx.clone()
    if K > 4:
        idx[1, 2], idx[0, 3] = -1, idx[0, 1]              # no token; one token twice
    w = torch.rand(T, generator=_gen(1), device=DEV)
    w[-1] = 0.0
    x = _place(z, skew, pad).requires_grad_()
    loss, token = ops.distill_loss(x, logp, idx, w, 1.3, beta, tail)
    (gx,) = torch.autograd.grad(loss, x)
    y = z.double().requires_grad_()
    want, tw = ref.distill_loss(y, logp, idx, w, 1.3, beta, tail)
    (gy,) = torch.autograd.grad(want, y)
    # the events' probabilities to 2e-6 of themselves (see the sum of the rows above); the loss moves with them by their share: of order one here
    assert ((token - tw).abs() <= 2e-6 * (1.0 + tw.abs())).all()
    assert abs(loss.item() - want.item()) <= 2e-6 * (1.0 + abs(want.item()))
    # each element half a step of its type, and float arithmetic to 5e-6
    assert gx.dtype == dtype and _rel(gx, gy) <= (2.0 ** -8 if dtype == BF16 else 0.0) + 5e-6
    assert (gx[-1] == 0).all()


@pytest.mark.parametrize("beta,tail", BETAS)
def test_distillation_gradient_by_differences(beta, tail):
    """of the kernel's own losses along a direction: central differences, float32 logits, step 2^-6: the third derivative's share is of order step^2 / 6, 4e-5,
    and rounding of the losses 2e-6 / 2^-5 at most, 6e-5"""
    T, V, h = 3, 500, 2.0 ** -6
    z = _logits("normal", T, V, F32)
    logp, idx = _teacher(z, 20)
    d = torch.randn(T, V, generator=_gen(9), device=DEV).sign()
    x = z.clone().requires_grad_()
    loss, _ = ops.distill_loss(x, logp, idx, beta=beta, tail=tail)
    loss.backward()
    up = ops.distill_loss(z + h * d, logp, idx, beta=beta, tail=tail)[1].double()
    dn = ops.distill_loss(z - h * d, logp, idx, beta=beta, tail=tail)[1].double()
    assert (((up - dn) / (2 * h)) / T - (x.grad.double() * d).sum(-1)).abs().max() <= 1.5e-4


@pytest.mark.parametrize("beta,tail", BETAS)
def test_distillation_where_the_student_is_sure(beta, tail):
    """all but 1e-9 of the student's mass on the teacher's tokens: the rest keeps its digits"""
    z = torch.randn(2, 5000, generator=_gen(3), device=DEV)
    z[:, :8] += 30.0
    idx = torch.arange(8, device=DEV, dtype=torch.int32).expand(2, 8).contiguous()
    logp = torch.log_softmax(torch.randn(2, 8, generator=_gen(4), device=DEV), -1) + math.log(0.9)
    x, y = z.clone().requires_grad_(), z.double().requires_grad_()
    loss, token = ops.distill_loss(x, logp, idx, beta=beta, tail=tail)
    want, tw = ref.distill_loss(y, logp, idx, None, 1.0, beta, tail)
    loss.backward()
    want.backward()
    assert ((token - tw).abs() <= 2e-6 * (1.0 + tw.abs())).all()
    assert _rel(x.grad, y.grad) <= 5e-6
    assert _rel(x.grad[:, 8:], y.grad[:, 8:]) <= 2e-5              # exponents of 30 / ln 2 = 43 here, three steps of 2^-24 of each: 8e-6, and the rest as above


def test_distillation_of_masked_rows_and_tokens():
    T, V = 6, 3000
    z = _logits("normal", T, V, F32)
    z[:, 100:2000] = -INF                                  # tokens that the student may not use
    logp, idx = _teacher(z[:, :100].contiguous(), 10)
    w = torch.tensor([1.0, 0.0, 2.0, 0.0, 1.0, 0.5], device=DEV)
    z[1] = math.nan                                        # rows that do not count
    z[3] = -INF
    idx[2] = -1                                            # no teacher
    x = z.clone().requires_grad_()
    loss, token = ops.distill_loss(x, logp, idx, w)
    loss.backward()
    assert torch.isfinite(loss) and torch.isfinite(x.grad).all() and (x.grad[[1, 3]] == 0).all() and (token[[1, 3]] == 0).all()
    assert abs(token[2].item()) < 1e-6 and x.grad[2].abs().max() < 1e-6 and (x.grad[:, 100:2000] == 0).all()
    y = z[[0, 4, 5]].double().requires_grad_()
    ref.distill_loss(y, logp[[0, 4, 5]], idx[[0, 4, 5]], w[[0, 4, 5]], 1.0, 0.0, True)[0].backward()
    assert _rel(x.grad[[0, 4, 5]], y.grad) <= 5e-6


def test_distillation_backward_twice_and_from_other_gradients():
    z = _logits("normal", 4, 2000, F32).requires_grad_()
    logp, idx = _teacher(z.detach(), 16)
    loss, _ = ops.distill_loss(z, logp, idx)
    (a,) = torch.autograd.grad(loss, z, retain_graph=True)
    (b,) = torch.autograd.grad(3.0 * loss, z, retain_graph=True)
    (c,) = torch.autograd.grad(loss, z)
    assert torch.equal(a, c) and torch.equal(b, 3.0 * a)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, z)
    s = torch.ones((), device=DEV, requires_grad=True)
    loss, _ = ops.distill_loss(z, logp, idx)
    (g,) = torch.autograd.grad(loss * s, z, create_graph=True)
    (gs,) = torch.autograd.grad((g * g).sum(), s)
    assert torch.allclose(gs, 2 * (a * a).sum())
    loss, _ = ops.distill_loss(z, logp, idx)
    loss.backward()
    (2.0 * ops.distill_loss(z, logp, idx)[0]).backward()
    assert torch.allclose(z.grad, 3.0 * a)
    with torch.no_grad():
        again, _ = ops.distill_loss(z, logp, idx)
    assert torch.equal(again, loss.detach())


@pytest.mark.parametrize("beta,tail", BETAS)
@pytest.mark.parametrize("T,V,H,K", [(1, 1000, 64, 5), (37, 4096, 256, 64), (300, 32000, 128, 20), (513, 8200, 72, 1)])
def test_head_distillation(T, V, H, K, beta, tail):
    g = _gen(T)
    h = torch.randn(T, H, generator=g, device=DEV).to(BF16).requires_grad_()
    w = (torch.randn(V, H, generator=g, device=DEV) * 2 / math.sqrt(H)).to(BF16).requires_grad_()
    logp, idx = _teacher((h @ w.t()).detach(), K)
    wt = torch.rand(T, generator=g, device=DEV) / T
    loss, token = ops.lmhead_distill_loss(h, w, logp, idx, wt, 0.9, beta, tail)
    loss.backward()
    h64, w64 = h.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    want, tw = ref.distill_loss(h64 @ w64.t(), logp, idx, wt, 0.9, beta, tail)
    want.backward()
    # float logits: sums of H products, 2^-23 of their terms' sizes (about 2) each at most and most cancel: 1e-5 of the events' probabilities
    assert ((token - tw).abs() <= 1e-5 * (1.0 + tw.abs())).all() and abs(loss.item() - want.item()) <= 1e-5 * (1.0 + abs(want.item()))
    # gradients: the logits' half a step of bf16, in sums, and the results' own
    assert _rel(h.grad, h64.grad) <= 2.0 ** -7 and _rel(w.grad, w64.grad) <= 2.0 ** -7


def test_head_in_ranges_of_rows(monkeypatch):
    from nanorlhf_b200.ops import native
    T, V, H, K = 700, 2048, 128, 8
    h = torch.randn(T, H, generator=_gen(1), device=DEV).to(BF16)
    w = (torch.randn(V, H, generator=_gen(2), device=DEV) * 0.2).to(BF16)
    logp, idx = ops.lmhead_top_logprobs(h, w, K)
    whole = [t.detach() for t in ops.lmhead_distill_loss(h, w, logp, idx)]

    def grads():
        a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
        out = ops.lmhead_distill_loss(a, b, logp, idx)
        (2.0 * out[0]).backward()
        return out[0].detach(), out[1], a.grad, b.grad

    one = grads()
    monkeypatch.setattr(native, "LOGITS_BYTES", 256 * 4 * V)
    assert len(native._row_ranges(T, V)) == 3
    some = grads()
    assert torch.equal(one[1], whole[1]) and torch.equal(one[1], some[1]) and torch.equal(one[0], some[0])
    assert torch.equal(one[2], some[2]) and _rel(some[3], one[3]) <= 2.0 ** -7       # sums of float parts, rounded once, against one sum
    assert all(torch.equal(a, b) for a, b in zip(ops.lmhead_top_logprobs(h, w, K), (logp, idx)))
    for need in ((True, False), (False, True)):
        a, b = h.clone().requires_grad_(need[0]), w.clone().requires_grad_(need[1])
        ops.lmhead_distill_loss(a, b, logp, idx)[0].backward()
        assert (a.grad is not None) == need[0] and (b.grad is not None) == need[1]


def test_head_of_other_types_and_sizes():
    h = torch.randn(9, 36, generator=_gen(1), device=DEV).requires_grad_()
    w = torch.randn(501, 36, generator=_gen(2), device=DEV).mul(0.3).requires_grad_()
    logp, idx = ops.lmhead_top_logprobs(h, w, 6)
    loss, _ = ops.lmhead_distill_loss(h, w, logp, idx, beta=1.0)
    loss.backward()
    assert h.grad is not None and w.grad is not None and loss.item() < 1e-5         # the teacher is the student


def test_refusals_on_the_device():
    z = torch.zeros(3, 8, device=DEV)
    logp, idx = ops.top_logprobs(z, 2)
    for bad in (z.half(), z.double(), z.int()):
        with pytest.raises(RuntimeError):
            ops.top_logprobs(bad, 2)
        with pytest.raises(RuntimeError):
            ops.sample_filtered(bad, torch.zeros(3, device=DEV))
        with pytest.raises(RuntimeError):
            ops.distill_loss(bad, logp, idx)
    for args in ((logp.cpu(), idx), (logp, idx.cpu()), (logp, idx, torch.ones(3))):
        with pytest.raises(RuntimeError):
            ops.distill_loss(z, *args)
    with pytest.raises(RuntimeError):
        ops.sample_filtered(z, torch.zeros(3))
    with pytest.raises(RuntimeError):
        ops.distill_loss(torch.zeros(1, (1 << 20) + 8, device=DEV), logp[:1], idx[:1])


def test_other_layouts():
    z = _logits("peaked", 40, 300, F32)
    t = z.t().contiguous().t()                             # elements of a row apart
    u = torch.rand(40, device=DEV)
    assert all(torch.equal(a, b) for a, b in zip(ops.top_logprobs(t, 9), ops.top_logprobs(z, 9)))
    assert all(torch.equal(a, b) for a, b in zip(ops.sample_filtered(t, u, top_k=7), ops.sample_filtered(z, u, top_k=7)))
    logp, idx = _teacher(z, 9)
    x, y = t.clone(memory_format=torch.preserve_format).requires_grad_(), z.clone().requires_grad_()
    ops.distill_loss(x, logp, idx.long())[0].backward()
    ops.distill_loss(y, logp.expand(40, 9), idx)[0].backward()
    assert torch.equal(x.grad, y.grad)
    wide = idx.long()
    wide[0, 0] += 1 << 33                                  # no token
    narrow = idx.clone()
    narrow[0, 0] = -1
    assert torch.equal(ops.distill_loss(z, logp, wide)[1], ops.distill_loss(z, logp, narrow)[1])


def test_empty_batches():
    assert [tuple(t.shape) for t in ops.top_logprobs(torch.zeros(0, 8, device=DEV), 3)] == [(0, 3), (0, 3)]
    assert [tuple(t.shape) for t in ops.sample_filtered(torch.zeros(0, 8, device=DEV), torch.zeros(0, device=DEV))] == [(0,), (0,)]
    z = torch.zeros(0, 8, device=DEV, requires_grad=True)
    none = torch.zeros(0, 2, device=DEV)
    loss, _ = ops.distill_loss(z, none, none.int())
    loss.backward()
    assert loss.item() == 0.0 and z.grad.shape == (0, 8)
    h, w = torch.zeros(0, 64, device=DEV, dtype=BF16, requires_grad=True), torch.zeros(16, 64, device=DEV, dtype=BF16, requires_grad=True)
    loss, _ = ops.lmhead_distill_loss(h, w, none, none.int())
    loss.backward()
    assert loss.item() == 0.0 and (w.grad == 0).all()


def test_results_repeat():
    z = _logits("peaked", 64, 32000, BF16)
    logp, idx = _teacher(z, 32)
    u = torch.rand(64, generator=_gen(2), device=DEV)

    def all_of_them():
        x = z.clone().requires_grad_()
        loss, token = ops.distill_loss(x, logp, idx, beta=0.5)
        loss.backward()
        return [loss.detach(), token, x.grad, *ops.top_logprobs(z, 100), *ops.sample_filtered(z, u, top_p=0.97), *ops.sample_filtered(z, u, 0.8, 40, 0.9, 0.01)]

    first = all_of_them()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, all_of_them()))


def test_two_streams_at_once():
    a, b = _logits("peaked", 200, 50021, F32, seed=1), _logits("peaked", 200, 50021, F32, seed=2)
    u = torch.rand(200, generator=_gen(2), device=DEV)

    def both(z):
        logp, idx = ops.top_logprobs(z, 32)
        x = (z * 0.9).requires_grad_()
        loss, _ = ops.distill_loss(x, logp, idx)
        loss.backward()
        return [logp, idx, loss.detach(), x.grad, *ops.sample_filtered(z, u, top_p=0.9)]

    want = both(a), both(b)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    got = [[], []]
    for _ in range(3):
        for i, (stream, z) in enumerate(((s, a), (t, b))):
            with torch.cuda.stream(stream):
                got[i] = both(z)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for i in range(2) for x, y in zip(want[i], got[i]))


def test_captured_and_replayed():
    T, V = 33, 5000
    z = _logits("peaked", T, V, F32, seed=1)
    u = torch.rand(T, generator=_gen(2), device=DEV)
    h = torch.randn(T, 64, generator=_gen(3), device=DEV).to(BF16)
    w = torch.randn(V, 64, generator=_gen(4), device=DEV).mul(0.2).to(BF16)

    def step():
        logp, idx = ops.top_logprobs(z * 1.1, 16)
        x, a, b = z.detach().clone().requires_grad_(), h.clone().requires_grad_(), w.clone().requires_grad_()
        loss, token = ops.distill_loss(x, logp, idx, beta=1.0)
        (gx,) = torch.autograd.grad(0.5 * loss, x)
        head, _ = ops.lmhead_distill_loss(a, b, logp, idx)
        ga, gb = torch.autograd.grad(2.0 * head, (a, b))
        return [logp, idx, token, gx, ga, gb, *ops.sample_filtered(z, u, 0.9, 20, 0.9)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 7):
        z.copy_(_logits("peaked", T, V, F32, seed=seed))
        u.copy_(torch.rand(T, generator=_gen(seed), device=DEV))
        for _ in range(2):
            graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_backward_captured_without_its_forward():
    """replays of such a graph must not multiply what an earlier one multiplied"""
    z = _logits("normal", 4, 2000, F32).requires_grad_()
    logp, idx = _teacher(z.detach(), 8)
    (want,) = torch.autograd.grad(0.5 * ops.distill_loss(z, logp, idx)[0], z)
    half = torch.full((), 0.5, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss, _ = ops.distill_loss(z, logp, idx)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            (g,) = torch.autograd.grad(loss, z, half)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        graph.replay()
    assert torch.equal(g, want)


@pytest.mark.parametrize("beta", [0.0, 0.5])
def test_traced_distillation_follows_its_inputs(beta):
    x, y = (_logits("normal", 5, 300, F32, seed=s) for s in (1, 2))
    logp, idx = _teacher(x, 9)
    f = lambda z: ops.distill_loss(z, logp, idx, beta=beta)  # noqa: E731
    traced = torch.jit.trace(f, x, check_trace=False)
    p, q = (y.clone().requires_grad_() for _ in range(2))
    got, want = traced(p), f(q)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    (2.0 * got[0]).backward()
    (2.0 * want[0]).backward()
    assert torch.equal(p.grad, q.grad)


def test_saved_gradients_may_be_packed_away():
    """hooks on saved tensors get the gradient that the forward has formed, and the backward takes what they give"""
    z = _logits("normal", 4, 500, F32)
    logp, idx = _teacher(z, 9)
    x, y = z.clone().requires_grad_(), z.clone().requires_grad_()
    with torch.autograd.graph.save_on_cpu():
        loss, _ = ops.distill_loss(x, logp, idx)
    (3.0 * loss).backward()
    (3.0 * ops.distill_loss(y, logp, idx)[0]).backward()
    assert torch.equal(x.grad, y.grad)


def test_rows_beyond_32_bit_offsets():
    """rows whose elements lie more than 2^31 apart in one buffer"""
    V = 1 << 16
    buf = torch.empty((1 << 15) + 9, V, dtype=BF16, device=DEV)
    z = buf[::1 << 15]                                     # two rows, 2^31 elements apart
    z.copy_(_logits("peaked", 2, V, BF16))
    u = torch.rand(2, device=DEV)
    assert all(torch.equal(a, b) for a, b in zip(ops.top_logprobs(z, 9), ops.top_logprobs(z.clone(), 9)))
    assert all(torch.equal(a, b) for a, b in zip(ops.sample_filtered(z, u, top_p=0.9), ops.sample_filtered(z.clone(), u, top_p=0.9)))
    logp, idx = _teacher(z.clone(), 8)
    assert torch.equal(ops.distill_loss(z, logp, idx)[1], ops.distill_loss(z.clone(), logp, idx)[1])


def test_one_distillation_step_as_it_is_used():
    """tokens are drawn, a teacher lists its alternatives, the student's head takes a step towards them: with the gradient that the definition gives"""
    B, V, H = 16, 4096, 128
    g = _gen(0)
    h = torch.randn(B, H, generator=g, device=DEV).to(BF16)
    student = (torch.randn(V, H, generator=g, device=DEV) * 0.2).to(BF16).requires_grad_()
    teacher = (student.detach().float() + 0.05 * torch.randn(V, H, generator=g, device=DEV)).to(BF16)
    logits = ops.linear(h, student.detach())
    tok, logp = ops.sample_filtered(logits, torch.rand(B, generator=g, device=DEV), 0.9, 50, 0.95)
    assert ((tok >= 0) & (tok < V)).all() and (logp <= 0).all()
    top, idx = ops.lmhead_top_logprobs(h, teacher, 32)
    weights = (tok != 7).float() / B
    loss, _ = ops.lmhead_distill_loss(h, student, top, idx, weights)
    loss.backward()
    w64 = student.detach().double().requires_grad_()
    want, _ = ref.distill_loss(h.double() @ w64.t(), top, idx, weights, 1.0, 0.0, True)
    want.backward()
    assert abs(loss.item() - want.item()) < 1e-5 and _rel(student.grad, w64.grad) <= 2.0 ** -7
