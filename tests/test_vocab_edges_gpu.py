"""Calls of the vocabulary operators at the ends of their ranges, against float64: what is sure, what has no mass left, what is not a number, what is held."""
import math

import pytest
import torch

from nanorlhf_b200 import ops
from nanorlhf_b200.ops import native
from nanorlhf_b200.ops import reference as ref

pytestmark = pytest.mark.gpu

INF = math.inf
BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda"
BETAS = [(0.0, True), (0.0, False), (1.0, True), (0.4, True)]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-30)).item()


def _same_draws(z, u, **kw):
    tok, logp = ops.sample_filtered(z, u, **kw)
    want, lw = ref.sample_filtered(z, u, **kw)
    assert torch.equal(tok, want), (tok != want).nonzero()[:8]
    # two roundings of float32, and 2e-7 where a mass's last bits move a sum
    assert ((logp == lw) | ((logp - lw).abs() <= 2e-7 + 2.0 ** -23 * lw.abs())).all()


# ---- one column ------------------------------------------------------------------------------------------------------------------
def _spoil():
    """the allocator's small blocks, which the next results lie in, hold no result of an earlier call"""
    x = [torch.full((128,), 0x7a7a7a7a, dtype=torch.int32, device=DEV) for _ in range(64)]
    torch.cuda.synchronize()
    del x


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [1, 3, 40])
def test_sampling_of_one_column_is_written(T, dtype):
    z = torch.linspace(-2.0, 2.0, T, device=DEV).to(dtype)[:, None].contiguous()
    u = torch.rand(T, generator=_gen(T), device=DEV)
    none = torch.full_like(z, -INF)
    for kw in (dict(temperature=0.0), dict(temperature=0.0, top_p=0.5), dict(temperature=0.0, min_p=0.3), dict(temperature=0.0, top_k=5), dict(top_k=1), dict(),
               dict(top_p=0.4), dict(min_p=0.2), dict(temperature=torch.zeros(T, device=DEV)), dict(temperature=0.0, top_p=torch.full((T,), 0.7, device=DEV))):
        _spoil()
        tok, logp = ops.sample_filtered(z, u, **kw)
        assert tok.tolist() == [0] * T and logp.tolist() == [0.0] * T, kw
        _spoil()
        tok, logp = ops.sample_filtered(none, u, **kw)
        assert tok.tolist() == [-1] * T and logp.tolist() == [-INF] * T, kw


# ---- a student that is sure --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("beta,tail", BETAS)
@pytest.mark.parametrize("gap,temperature", [(60.0, 0.6), (26.0, 0.25), (100.0, 1.0), (1e4, 1.0), (1e4, 0.3), (-100.0, 1.0), (-1e4, 0.5)])
@pytest.mark.parametrize("T,V", [(5, 1000), (3, 151936), (50, 151936)])          # one, four, two blocks a row
def test_distillation_where_the_rest_lies_far_below(T, V, gap, temperature, beta, tail, dtype):
    """the teacher's tokens `gap` above (or below) all others: what the rest has left, relative to the row's largest logit, is beyond float's range"""
    z = torch.randn(T, V, generator=_gen(3), device=DEV)
    at = torch.arange(8, device=DEV) * (V // 8) + 3
    z[:, at] += gap
    z = z.to(dtype)
    idx = at.int().expand(T, 8).contiguous()
    logp = torch.log_softmax(torch.randn(T, 8, generator=_gen(4), device=DEV), -1) + math.log(0.9)
    x, y = z.clone().requires_grad_(), z.double().requires_grad_()
    loss, token = ops.distill_loss(x, logp, idx, None, temperature, beta, tail)
    want, tw = ref.distill_loss(y, logp, idx, None, temperature, beta, tail)
    loss.backward()
    want.backward()
    # the rest's sum is off by 5e-6 of itself at most, of which the loss has a share below one; the result is rounded to float32, and so is the one it is held against
    assert torch.isfinite(token).all() and ((token - tw).abs() <= 5e-6 + 2.0 ** -23 * tw.abs()).all()
    assert abs(loss.item() - want.item()) <= 5e-6 + 2.0 ** -23 * abs(want.item())
    # gradients: half a step of their type, 5e-6 of the sum, and exponents of 10 bits where a row has its mass, three steps of 2^-24 of them: 2e-6
    tol = (2.0 ** -8 if dtype == BF16 else 0.0) + 1e-5
    # and where they are next to nothing, differences of logarithms up to 4e4 that are rounded to 2^-53 of themselves on either side: 1e-11 of the probabilities, which
    # sum to 1 (times 1 / (T temperature) <= 1)
    on = torch.zeros(V, dtype=torch.bool, device=DEV).index_fill_(0, at, True)
    for part in (on, ~on):
        gx, gy = x.grad[:, part].double(), y.grad[:, part]
        assert (gx - gy).norm() <= tol * gy.norm() + 1e-11


# ---- a teacher who lists all tokens ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("beta,tail", BETAS)
@pytest.mark.parametrize("T,V,K", [(300, 6, 6), (200, 1024, 1024), (100, 5000, 300), (40, 151936, 1000), (10, 151936, 7)])
def test_a_teacher_who_lists_all_that_the_student_may_use(T, V, K, beta, tail, dtype):
    """what rounding of its log-probabilities leaves of 1 is no mass that nobody has"""
    at = torch.randperm(V, generator=_gen(1), device=DEV)[:K]
    z, t = (torch.full((T, V), -INF, device=DEV).index_copy_(1, at, torch.randn(T, K, generator=_gen(s), device=DEV)) for s in (2, 3))
    logp, idx = ops.top_logprobs(t, K)
    assert (idx >= 0).all()
    x, y = z.to(dtype).clone().requires_grad_(), z.to(dtype).double().requires_grad_()
    loss, token = ops.distill_loss(x, logp, idx, None, 1.0, beta, tail)
    want, tw = ref.distill_loss(y, logp, idx, None, 1.0, beta, tail)
    loss.backward()
    want.backward()
    # no mass but the teacher's tokens', which is double: rounded to float32 on either side
    assert torch.isfinite(token).all() and ((token - tw).abs() <= 2.0 ** -23 * (1.0 + tw.abs())).all()
    assert torch.isfinite(x.grad).all() and _rel(x.grad, y.grad) <= (2.0 ** -8 if dtype == BF16 else 0.0) + 5e-6
    if beta == 0.0 and tail and K < V:                     # more than rounding: mass where the student has none
        assert (ops.distill_loss(x.detach(), logp - 1e-5, idx)[1] == INF).all()


# ---- what is not a number ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("beta,tail", BETAS)
@pytest.mark.parametrize("bad", [math.nan, INF])
@pytest.mark.parametrize("V", [500, 151936])
def test_gradients_of_a_row_that_is_not_a_number(V, bad, beta, tail, dtype):
    """are not numbers either, and those of the other rows are what they are without it"""
    z = torch.randn(4, V, generator=_gen(1), device=DEV)
    idx = torch.tensor([3, 40, 7], dtype=torch.int32, device=DEV).expand(4, 3).contiguous()
    logp = torch.full((4, 3), 0.25, device=DEV).log()
    z[1, 100] = bad                                        # off the teacher's tokens
    z[2, 40] = bad                                         # one of them
    x = z.to(dtype).requires_grad_()
    loss, token = ops.distill_loss(x, logp, idx, beta=beta, tail=tail)
    loss.backward()
    assert loss.isnan() and token[1:3].isnan().all() and x.grad[1:3].isnan().all()
    clean = z.detach().clone()
    clean[1:3] = 0.0
    y = clean.to(dtype).requires_grad_()
    loss, want = ops.distill_loss(y, logp, idx, beta=beta, tail=tail)
    loss.backward()
    assert torch.equal(token[[0, 3]], want[[0, 3]]) and torch.equal(x.grad[[0, 3]], y.grad[[0, 3]])


@pytest.mark.parametrize("beta,tail", BETAS)
def test_a_teacher_that_is_not_a_number_is_not_left_out(beta, tail):
    z = torch.randn(3, 700, generator=_gen(1), device=DEV, requires_grad=True)
    idx = torch.tensor([3, 40, 7, -1], dtype=torch.int32, device=DEV).expand(3, 4).contiguous()
    logp = torch.full((3, 4), 0.2, device=DEV).log()
    logp[1, 2] = math.nan
    logp[2, 3] = math.nan                                  # of no token: skipped
    loss, token = ops.distill_loss(z, logp, idx, beta=beta, tail=tail)
    loss.backward()
    assert loss.isnan() and token.isnan().tolist() == [False, True, False]
    assert z.grad[1].isnan().all() and torch.isfinite(z.grad[[0, 2]]).all()


# ---- min-p with a nucleus ----------------------------------------------------------------------------------------------------------
def _fastest(f, n=12):
    times = []
    for _ in range(n):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b))
    return min(times)


@pytest.mark.parametrize("rows,dtype", [(200, BF16), (60, F32), (20, BF16)])             # one, two, four blocks a row
@pytest.mark.parametrize("std,min_p", [(0.6, 0.02), (0.6, 0.05), (0.9, 0.01)])
def test_a_nucleus_behind_min_p_costs_what_a_nucleus_costs(std, min_p, rows, dtype):
    """thousands of tokens above min_p: where their nucleus ends is found by the ranges that find any other nucleus' end (0.2 ms; a row looked through for its border
    takes 1 ms), and is the definition's"""
    z = (torch.randn(rows, 151936, generator=_gen(7), device=DEV) * std).to(dtype)
    u = torch.rand(rows, generator=_gen(8), device=DEV)
    for p in (0.95, 0.7):
        _same_draws(z, u, min_p=min_p, top_p=p)
        plain, both = _fastest(lambda: ops.sample_filtered(z, u, top_p=p)), _fastest(lambda: ops.sample_filtered(z, u, top_p=p, min_p=min_p))
        assert both <= 2.5 * plain, (plain, both)


# ---- a log-probability beyond float32's quotients ----------------------------------------------------------------------------------
@pytest.mark.parametrize("kept", [2, 60, 100, 600])
@pytest.mark.parametrize("gap", [88.0, 100.0, 200.0, 600.0])
def test_log_probability_of_a_kept_token_of_little_mass(gap, kept):
    """a number of 0 draws the first kept token, however little it has"""
    z = torch.full((2, 3000), -1e30, device=DEV)
    z[0, 5], z[0, 10:9 + kept] = 0.0, gap
    z[1, 5], z[1, 10:9 + kept] = -gap, torch.linspace(0.0, 3.0, kept - 1, device=DEV)
    for kw in (dict(top_k=kept), dict(top_k=kept, min_p=1e-300), dict(min_p=1e-300), dict(top_k=kept, temperature=1.1)):
        _same_draws(z, torch.zeros(2, device=DEV), **kw)


# ---- uniform numbers ---------------------------------------------------------------------------------------------------------------
def test_uniform_numbers_stay_below_one():
    """of these rows, the first of seed 0 whose number is next to 1 (one in 3 * 10^7 is)"""
    ids = torch.tensor([40657998, 66330067, 84170650, 97987152, 137839096, 1068921965], dtype=torch.int32, device=DEV)
    assert native.row_uniforms(0, 0, ids).tolist() == [1.0 - 2.0 ** -24] * 6          # the largest float32 below 1
    assert torch.equal(native.row_uniforms(0, 0, ids + 1).lt(1.0 - 2.0 ** -20), torch.ones(6, dtype=torch.bool, device=DEV))


# ---- temperatures ------------------------------------------------------------------------------------------------------------------
def _rows(pattern, T, V, dtype):
    z = torch.randn(T, V, generator=_gen(V), device=DEV)
    if pattern == "masked":
        z = z.masked_fill(torch.rand(T, V, generator=_gen(2), device=DEV) > 0.5, -INF)
    return z.to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pattern", ["normal", "masked"])
@pytest.mark.parametrize("temperature", [1e44, 1e46, 1e100, 1e300])
@pytest.mark.parametrize("T,V", [(2, 151936), (60, 50021)])
def test_temperatures_whose_reciprocal_is_none_of_floats(T, V, temperature, pattern, dtype):
    """every token with mass is as probable as any other"""
    z = _rows(pattern, T, V, dtype)
    logp, idx = ops.top_logprobs(z, 9, temperature)
    want, at = ref.top_logprobs(z, 9, temperature)
    assert torch.equal(idx, at) and ((logp - want).abs() <= 5e-6 + 2.0 ** -23 * want.abs()).all()
    u = torch.rand(T, generator=_gen(5), device=DEV)
    for kw in (dict(), dict(top_p=0.5), dict(top_p=0.01), dict(top_k=40, top_p=0.3), dict(min_p=0.5, top_p=0.6)):
        _same_draws(z, u, temperature=temperature, **kw)
    if pattern == "normal":
        x, y = z.clone().requires_grad_(), z.double().requires_grad_()
        loss, token = ops.distill_loss(x, logp, idx, None, temperature)
        other, tw = ref.distill_loss(y, logp, idx, None, temperature, 0.0, True)
        loss.backward()
        other.backward()
        assert ((token - tw).abs() <= 5e-6).all() and (x.grad == 0).all()        # 1 / temperature of anything is below float32's least number


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pattern", ["normal", "masked"])
def test_an_infinite_temperature_of_a_row_is_the_largest(pattern, dtype):
    T, V = 20, 50021
    z = _rows(pattern, T, V, dtype)
    u = torch.rand(T, generator=_gen(6), device=DEV)
    hot = torch.ones(T, device=DEV)
    hot[::2] = INF
    for kw in (dict(), dict(top_p=0.5), dict(top_p=0.01), dict(top_k=40), dict(min_p=0.5, top_p=0.6)):
        _same_draws(z, u, temperature=hot, **kw)


# ---- what a head holds -------------------------------------------------------------------------------------------------------------
def _held(f):
    torch.cuda.synchronize()
    start = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = f()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - start, out


@pytest.mark.parametrize("dtype,H", [(BF16, 64), (F32, 64), (BF16, 36)])
def test_a_head_holds_no_more_than_it_says(dtype, H, monkeypatch):
    """the float logits of one range of rows and half as much of their gradients, beside inputs, results and a float sum of the weight's gradient"""
    T, V = 16384, 4000
    part = 4096 * 4 * V                                    # 66 MB; all rows' logits are 262
    monkeypatch.setattr(native, "LOGITS_BYTES", part)
    h = torch.randn(T, H, generator=_gen(1), device=DEV).to(dtype).requires_grad_()
    w = (torch.randn(V, H, generator=_gen(2), device=DEV) * 0.2).to(dtype).requires_grad_()
    top = torch.full((T, 8), 0.05, device=DEV).log()
    idx = torch.arange(8, dtype=torch.int32, device=DEV).expand(T, 8).contiguous() * 400
    ops.lmhead_distill_loss(h[:6000], w, top[:6000], idx[:6000])[0].backward()           # (workspaces that stay)
    h.grad = w.grad = None
    held, (loss, token) = _held(lambda: ops.lmhead_distill_loss(h, w, top, idx))
    # beside them: both gradients, the weight's as a float sum as well; operands in float where the type asks for it; allocations of 2 MiB at most for small things
    beside = h.nbytes + w.nbytes + 4 * w.numel() + 4 * (h.numel() + w.numel()) + (2 << 20)
    assert held <= 1.5 * part + beside, (held, part, beside)
    held, (logp, _) = _held(lambda: ops.lmhead_top_logprobs(h, w, 8))
    assert held <= part + 2 * 32 * T + 4 * (h.numel() + w.numel()) + (2 << 20), (held, part)
    loss.backward()
    # the whole in one range gives the same up to the order of float sums
    monkeypatch.setattr(native, "LOGITS_BYTES", 4 << 30)
    a, b = h.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    one, each = ops.lmhead_distill_loss(a, b, top, idx)
    one.backward()
    # float32 products of T, V and H terms, 2^-24 of their sizes each; gradients to half a step of their type in front of and behind the products
    tol = 2.0 ** -7 if dtype == BF16 else 1e-5
    assert abs(one.item() - loss.item()) <= 1e-6 and (each - token).abs().max() <= 1e-5 and _rel(h.grad, a.grad) <= tol and _rel(w.grad, b.grad) <= tol
    assert torch.allclose(logp, ops.lmhead_top_logprobs(h, w, 8)[0], rtol=0.0, atol=1e-5)


@pytest.mark.parametrize("beta,tail", BETAS)
@pytest.mark.parametrize("T,V,H,hd,wd", [(40, 1003, 64, BF16, BF16), (33, 512, 20, F32, F32), (33, 512, 64, F32, BF16), (600, 2001, 36, BF16, F32)])
def test_a_head_of_other_types_and_sizes(T, V, H, hd, wd, beta, tail, monkeypatch):
    monkeypatch.setattr(native, "LOGITS_BYTES", 256 * 4 * V)                             # 600 rows: three ranges
    h = torch.randn(T, H, generator=_gen(1), device=DEV).to(hd).requires_grad_()
    w = (torch.randn(V, H, generator=_gen(2), device=DEV) * 0.2).to(wd).requires_grad_()
    h64, w64 = h.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    top, idx = ops.top_logprobs((h64 @ w64.t()).detach().float() + 0.3, 9)
    wt = torch.rand(T, generator=_gen(3), device=DEV) / T
    loss, token = ops.lmhead_distill_loss(h, w, top, idx, wt, 0.8, beta, tail)
    (2.0 * loss).backward()
    want, tw = ref.distill_loss(h64 @ w64.t(), top, idx, wt, 0.8, beta, tail)
    (2.0 * want).backward()
    # float32 logits of H <= 64 products: 64 * 2^-24 of their terms, of which the sums are below 4: 1.5e-5 at the very most; gradients the same, and half a step of their type
    assert ((token - tw).abs() <= 1.5e-5 * (1.0 + tw.abs())).all() and abs(loss.item() - want.item()) <= 1.5e-5 * (1.0 + abs(want.item()))
    for a, b in ((h, h64), (w, w64)):
        assert a.grad.dtype == a.dtype and _rel(a.grad, b.grad) <= (2.0 ** -8 if a.dtype == BF16 else 0.0) + 1e-4


# ---- derivatives -------------------------------------------------------------------------------------------------------------------
def test_a_second_derivative_is_refused():
    z = torch.randn(4, 300, generator=_gen(1), device=DEV, requires_grad=True)
    logp, idx = ops.top_logprobs(z.detach() * 1.1, 8)
    s = torch.ones((), device=DEV, requires_grad=True)
    (want,) = torch.autograd.grad(ops.distill_loss(z, logp, idx)[0], z)
    loss, _ = ops.distill_loss(z, logp, idx)
    (g,) = torch.autograd.grad(loss * s, z, create_graph=True)
    assert torch.equal(g, want)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad((g * g).sum(), z, allow_unused=True, retain_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        ((g * g).sum() + (z * z).sum()).backward(retain_graph=True)
    (gs,) = torch.autograd.grad((g * g).sum(), s)          # of the factor there is one
    assert torch.allclose(gs, 2 * (want * want).sum())
    h = torch.randn(4, 64, generator=_gen(2), device=DEV).to(BF16).requires_grad_()
    w = torch.randn(304, 64, generator=_gen(3), device=DEV).to(BF16).requires_grad_()
    loss, _ = ops.lmhead_distill_loss(h, w, logp, idx)
    gh, gw = torch.autograd.grad(loss, (h, w), create_graph=True)
    for g, x in ((gh, h), (gw, w), (gh, w), (gw, h)):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(g.float().square().sum(), x, allow_unused=True, retain_graph=True)


# ---- logits a step of float32 apart at temperatures as small as that ---------------------------------------------------------------
@pytest.mark.parametrize("apart", [600.0, 689.0, 691.0, 707.0, 709.0, 730.0, 760.0, 1000.0, 1300.0, 1500.0])
@pytest.mark.parametrize("T", [3, 100])
def test_neighbouring_logits_at_their_own_temperature(T, apart):
    """the second largest logits are the next float32 number, `apart` temperatures below the largest: what they have is no share of a sum, and no garbage"""
    z = torch.randn(T, 40000, generator=_gen(1), device=DEV).clamp(max=2.0)
    top = torch.tensor(4.0, device=DEV)
    z[:, 100:200] = torch.nextafter(top, torch.zeros_like(top))
    z[:, [300, 9000]] = top
    step = 4.0 - z[0, 100].item()
    u = torch.linspace(1e-6, 1.0 - 2.0 ** -24, T, device=DEV)
    for kw in (dict(), dict(top_p=0.9), dict(top_p=0.4), dict(min_p=1e-300)):
        _same_draws(z, u, temperature=step / apart, **kw)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [3, 100])
def test_a_row_of_nothing_but_the_lowest_number(T, dtype):
    """a mask that leaves nothing: every token is as probable as any other, or as one that has twice its mass"""
    z = torch.full((T, 40000), torch.finfo(dtype).min, device=DEV, dtype=dtype)
    u = torch.rand(T, generator=_gen(2), device=DEV)
    for kw in (dict(), dict(top_p=0.7), dict(min_p=0.5), dict(top_k=9), dict(min_p=0.5, top_p=0.3), dict(temperature=1e30)):
        _same_draws(z, u, **kw)


# ---- probabilities at the end of double's range ------------------------------------------------------------------------------------
@pytest.mark.parametrize("beta", [0.01, 0.2, 0.5, 0.8, 0.99])
def test_divergences_of_probabilities_next_to_nothing(beta):
    """tokens of which neither teacher nor student gives more than the least numbers of double: their mixture may be rounded to 0"""
    V, far = 200, torch.arange(700.0, 760.0, 0.5, device=DEV)
    n = far.numel()
    z = torch.full((n, V), -2000.0, device=DEV)
    z[:, 0] = 0.0
    z[:, 7], z[:, 9], z[:, 150] = -far, -far.flip(0), -far  # 150 is not listed: all that others have
    idx = torch.tensor([0, 7, 9], dtype=torch.int32, device=DEV).expand(n, 3).contiguous()
    for p in (-far, torch.full_like(far, -INF), torch.full_like(far, -744.0)):
        logp = torch.stack([torch.zeros_like(p), p, p], -1)
        x, y = z.clone().requires_grad_(), z.double().requires_grad_()
        loss, token = ops.distill_loss(x, logp, idx, None, 1.0, beta)
        want, tw = ref.distill_loss(y, logp, idx, None, 1.0, beta, True)
        loss.backward()
        want.backward()
        # both sides sum numbers below e^-700; the mean is 0 within float32's least
        assert (token - tw).abs().max() <= 1e-38 and torch.isfinite(loss) and (x.grad - y.grad).abs().max() <= 1e-38


# ---- masks by a low number ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("beta,tail", BETAS)
@pytest.mark.parametrize("T,V,K", [(300, 700, 20), (10, 151936, 300), (50, 151936, 1024)])
def test_a_mask_by_a_low_number_is_one(T, V, K, beta, tail, dtype):
    """teacher and student share it: the loss is that of the tokens that are left, as by -infinity"""
    at = torch.randperm(V, generator=_gen(1), device=DEV)[:K]
    for low in (-1e4, torch.finfo(dtype).min):
        z, t = (torch.full((T, V), low, device=DEV).index_copy_(1, at, torch.randn(T, K, generator=_gen(s), device=DEV)) for s in (2, 3))
        z = z.to(dtype)
        logp, idx = ops.top_logprobs(t, K)
        x, y = z.clone().requires_grad_(), z.masked_fill(z == z.min(), -INF).requires_grad_()
        loss, token = ops.distill_loss(x, logp, idx, beta=beta, tail=tail)
        other, want = ops.distill_loss(y, logp, idx, beta=beta, tail=tail)
        loss.backward()
        other.backward()
        assert torch.equal(token, want) and torch.equal(loss, other) and torch.equal(x.grad, y.grad)
        ref_loss, tw = ref.distill_loss(z.double(), logp, idx, None, 1.0, beta, tail)
        assert ((token - tw).abs() <= 2.0 ** -23 * (1.0 + tw.abs())).all()


# ---- entries that sum to more than 1, and more of them than tokens -----------------------------------------------------------------
@pytest.mark.parametrize("beta,tail", BETAS)
@pytest.mark.parametrize("T,V,K", [(6, 2, 9), (5, 7, 1000), (4, 50, 333), (20, 5000, 64), (3, 151936, 1024)])
def test_entries_that_sum_to_more_than_one(T, V, K, beta, tail):
    """the gradient is the loss's own: entries of one token add up, whatever they add up to"""
    g = _gen(V)
    z = torch.randn(T, V, generator=g, device=DEV)
    idx = torch.randint(-1, V + 1, (T, K), generator=g, device=DEV).int()
    for more in (0.0, 0.4, -0.6):
        logp = torch.log_softmax(torch.randn(T, K, generator=g, device=DEV), -1) + more
        if V < K:
            idx[:, :V] = torch.arange(V, device=DEV)       # all tokens: only sums above 1 leave nothing to others, who are none
            logp = logp.clamp_min(-0.5)
        x, y = z.clone().requires_grad_(), z.double().requires_grad_()
        loss, token = ops.distill_loss(x, logp, idx, None, 0.9, beta, tail)
        want, tw = ref.distill_loss(y, logp, idx, None, 0.9, beta, tail)
        loss.backward()
        want.backward()
        # events to 5e-6 of themselves, of which there are as many as they sum up to
        whole = 1.0 + logp.double().exp().sum(-1)
        assert ((token - tw).abs() <= 5e-6 * whole * (1.0 + tw.abs())).all() and _rel(x.grad, y.grad) <= 1e-5
