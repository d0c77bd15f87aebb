"""Calls of the vocabulary operators at the ends of their ranges, in their plain forms."""
import math

import pytest
import torch

from nanorlhf_b200 import ops

INF = math.inf
BETAS = [(0.0, True), (0.0, False), (1.0, True), (0.4, True)]


@pytest.mark.parametrize("beta,tail", BETAS)
@pytest.mark.parametrize("K", [1, 2, 6, 300, 1024])
def test_a_teacher_who_lists_all_that_the_student_may_use(K, beta, tail):
    """what rounding of its log-probabilities leaves of 1 is no mass that nobody has"""
    T, V = 400, K + 50
    g = torch.Generator().manual_seed(K)
    teacher, z = torch.randn(T, K, generator=g), torch.randn(T, K, generator=g).double()
    logp, idx = ops.top_logprobs(teacher, K)
    listed = torch.log_softmax(teacher, -1)                        # another rounding
    every = torch.arange(K, dtype=torch.int32).expand(T, K)
    masked = torch.cat([z, torch.full((T, V - K), -INF, dtype=torch.float64)], -1)
    for a, i in ((logp, idx), (listed, every)):
        for x in (z, masked):
            x = x.clone().requires_grad_()
            loss, token = ops.distill_loss(x, a, i, beta=beta, tail=tail)
            loss.backward()
            assert torch.isfinite(token).all() and torch.isfinite(x.grad).all()
            # KL >= 0, of probabilities that sum to 1 within 2^-20
            assert (token >= -2.0 ** -20).all()
    if beta == 0.0 and tail:                                       # more than rounding: mass where the student has none
        assert (ops.distill_loss(masked, logp - 1e-5, idx)[1] == INF).all()


@pytest.mark.parametrize("beta,tail", BETAS)
@pytest.mark.parametrize("bad", [math.nan, INF])
def test_a_row_that_is_not_a_number_has_no_loss(bad, beta, tail):
    z = torch.randn(3, 40, generator=torch.Generator().manual_seed(1))
    idx = torch.tensor([3, 30, 7], dtype=torch.int32).expand(3, 3)
    logp = torch.full((3, 3), 0.25).log()
    z[1, 20] = bad                                                 # off the teacher's tokens
    z[2, 30] = bad                                                 # one of them
    x = z.requires_grad_()
    loss, token = ops.distill_loss(x, logp, idx, beta=beta, tail=tail)
    loss.backward()
    assert loss.isnan() and token.isnan().tolist() == [False, True, True] and x.grad[1:].isnan().all() and torch.isfinite(x.grad[0]).all()


@pytest.mark.parametrize("beta,tail", BETAS)
def test_a_teacher_that_is_not_a_number_is_not_left_out(beta, tail):
    z = torch.randn(3, 700, generator=torch.Generator().manual_seed(1), requires_grad=True)
    idx = torch.tensor([3, 40, 7, -1], dtype=torch.int32).expand(3, 4).contiguous()
    logp = torch.full((3, 4), 0.2).log()
    logp[1, 2] = math.nan
    logp[2, 3] = math.nan                                  # of no token: skipped
    loss, token = ops.distill_loss(z, logp, idx, beta=beta, tail=tail)
    loss.backward()
    assert loss.isnan() and token.isnan().tolist() == [False, True, False]
    assert z.grad[1].isnan().all() and torch.isfinite(z.grad[[0, 2]]).all()


def test_a_number_of_tokens_is_whole():
    z, u = torch.zeros(2, 8), torch.tensor([0.0, 0.99])
    for k in (2.5, torch.tensor(0.5)):                             # (one kept 3 tokens here and 2 on the device)
        with pytest.raises(ValueError):
            ops.sample_filtered(z, u, top_k=k)
    for k in (2, 2.0, torch.tensor(2)):
        assert ops.sample_filtered(z, u, top_k=k)[0].tolist() == [0, 1]
    from nanorlhf_b200.sampler.engine import generate
    with pytest.raises(ValueError, match="whole"):
        generate(1, None, None, [[1]], 1.0, 4, top_k=2.5)


@pytest.mark.parametrize("beta,tail", BETAS)
@pytest.mark.parametrize("low", [-1e4, torch.finfo(torch.bfloat16).min, torch.finfo(torch.float32).min])
def test_a_mask_by_a_low_number_is_one(low, beta, tail):
    """teacher and student share it: the loss is that of the tokens that are left, as by -infinity"""
    T, V, K = 100, 2000, 300
    g = torch.Generator().manual_seed(5)
    at = torch.arange(K) * 6
    z = torch.full((T, V), low).index_copy_(1, at, torch.randn(T, K, generator=g))
    logp, idx = torch.log_softmax(torch.randn(T, K, generator=g), -1), at.int().expand(T, K)
    x, y = z.double().requires_grad_(), z.masked_fill(z == low, -INF).double().requires_grad_()
    loss, token = ops.distill_loss(x, logp, idx, beta=beta, tail=tail)
    other, want = ops.distill_loss(y, logp, idx, beta=beta, tail=tail)
    loss.backward()
    other.backward()
    assert torch.equal(token, want) and (x.grad - y.grad).abs().max() < 1e-12


@pytest.mark.parametrize("low", [-1e4, -1e17, torch.finfo(torch.float32).min])
def test_tokens_of_equally_low_logits_share_a_gradient(low):
    """the teacher gives the others 0.1, the student next to nothing: the pull towards them is 0.1 altogether"""
    z = torch.full((2, 50), low)
    z[:, :3] = torch.tensor([1.0, 2.0, 0.5])
    x = z.requires_grad_()
    loss, _ = ops.distill_loss(x, torch.full((2, 3), 0.3).log(), torch.arange(3, dtype=torch.int32).expand(2, 3), torch.tensor([1.0, 2.0]))
    loss.backward()
    want = torch.tensor([[-0.1 / 47], [-0.2 / 47]]).expand(2, 47)
    assert torch.allclose(x.grad[:, 3:], want, rtol=1e-5, atol=0.0)         # 0.1 = 1 - 3 exp(log 0.3), of float32 logarithms: 1e-6 of it
