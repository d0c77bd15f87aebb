"""Calls of the vocabulary operators at the ends of their ranges, against float64: what is sure, what has no mass left, what is not a number, what is held."""
import math

import pytest
import torch

from nanorlhf_b200 import ops

pytestmark = pytest.mark.gpu

INF = math.inf
BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


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
