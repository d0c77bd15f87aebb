"""Attention over shared prefixes, decode attention over pages with scores and eviction, CPU forms: calls at the borders of what their documentation allows."""
import pytest
import torch

from groups_refusals import ints, packed, pool
from nanorlhf_b200 import ops


@pytest.mark.parametrize("groups", [0, 2])
def test_rows_without_any_sequence(groups):
    """they are behind the last one: 0, and so are their gradients"""
    q, k, v, dout, cu, _ = packed([[5]], 4, 2)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = ops.attention_shared_prefix(*leaves, cu[:1], ints(*[0] * (groups + 1)))
    for x in (out, *torch.autograd.grad(out, leaves, dout)):
        assert torch.equal(x, torch.zeros_like(x))


def test_share_prompts_is_refused_when_a_trainer_is_built():
    """... for models whose heads the kernels do not take; the CPU form takes all"""
    from nanorlhf_b200.models.lora import LoraConfig, get_peft_model
    from nanorlhf_b200.models.qwen2 import Qwen2Config, Qwen2ForCausalLM, Qwen2ForSequenceClassification
    from nanorlhf_b200.trainer.base import check_share_prompts
    made = lambda cls, dim: cls.from_config(Qwen2Config(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=1, num_attention_heads=2,  # noqa: E731
                                                        num_key_value_heads=1, head_dim=dim), torch.float32, "cpu", seed=1)
    narrow, wide = made(Qwen2ForCausalLM, 64), made(Qwen2ForCausalLM, 128)
    critic = Qwen2ForSequenceClassification.from_causal_lm(narrow)
    adapted = get_peft_model(made(Qwen2ForCausalLM, 64), LoraConfig(r=2, lora_alpha=4))
    for models in ((narrow, wide, None), (wide, narrow, None), (wide, wide, critic), (adapted, wide, None)):
        check_share_prompts(models, False)
        with pytest.raises(ValueError, match="share_prompts"):
            check_share_prompts(models, True)
    check_share_prompts((wide, wide, None), True)


def expanded_scores_are_refused(device):
    """... where they are written to: rows or heads that are one"""
    st = {n: None if x is None else x.to(device) for n, x in pool().items()}
    tables, context = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device=device), ints(40, 6).to(device)
    q = torch.ones(2, 4, 128, dtype=torch.bfloat16, device=device)
    call = lambda scores, into: ops.paged_decode_scored(q, st["k"], st["v"], tables, context, scores, out_scores=into)  # noqa: E731
    full = torch.rand(1, 2, 48, device=device).expand(2, -1, -1).contiguous()
    for x in (full[:1].expand(2, -1, -1), full[:, :1].expand(-1, 2, -1)):
        for scores, into in ((x, None), (full, x)):
            with pytest.raises(ValueError, match="expanded"):
                call(scores, into)
    # read, they may be
    want = call(full, torch.zeros_like(full))
    for a, b in zip(want, call(full[:1].expand(2, -1, -1), torch.zeros_like(full))):
        assert torch.equal(a, b)


def test_expanded_scores():
    expanded_scores_are_refused("cpu")


@pytest.mark.parametrize("kw", [{"keep": float("inf")}, {"keep": 8.5}, {"sinks": 1.5}, {"recent": 2.5}, {"recent": float("nan")}])
def test_evict_counts_in_whole_numbers(kw):
    st = pool()
    with pytest.raises(ValueError, match="whole number"):
        ops.kv_evict(st["k"], st["v"], torch.tensor([[0, 1, 2]], dtype=torch.int32), ints(40), torch.rand(1, 2, 40), **{"keep": 10, **kw})


@pytest.mark.parametrize("args", [(float("inf"), 4, None), (20.5, 4, None), (20, 1.5, None), (20, 4, 2.5), (20, 4, float("nan"))])
def test_a_bounded_cache_counts_in_whole_numbers(args):
    from nanorlhf_b200.sampler.engine import check_cache_options
    with pytest.raises(ValueError, match="whole number"):
        check_cache_options(False, *args)
    assert check_cache_options(False, 20.0, 4.0, None) == 5


def scales_of_packed_attention(device, dtype):
    """masked scores would not stay masked times 0 or less; small and large ones are taken"""
    q, k, v, _, cu, cg = (x.to(device) for x in packed([[3, 4]], 4, 2))
    q, k, v = (x.to(dtype) for x in (q, k, v))
    for bad in (0.0, -0.0, -0.1, 1e-40, 1e38, float("inf")):
        with pytest.raises(ValueError, match="scale"):
            ops.attention_shared_prefix(q, k, v, cu, cg, scale=bad)
    # so small that all scores are alike: means of the values up to a row (bf16: weights of 2^-8, the result's rounding)
    out = ops.attention_shared_prefix(q, k, v, cu, cg, scale=1e-37).float()
    seen = [list(range(i + 1)) for i in range(7)]
    for i, rows in enumerate(seen):
        want = v[rows].float().mean(0).repeat_interleave(2, 0)
        assert (out[i] - want).abs().max() <= (2 * 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -20) * v.float().abs().max()


def test_scales_of_packed_attention():
    scales_of_packed_attention("cpu", torch.float32)


def tables_of_shared_pages(device, wide=False, nobody=-1):
    """Rows behind the first, and ones that end inside what is shared: their tables need not name whole pages of it.  Entries that do not count are
    `nobody`; -1 is the page in front of the cache, of NaN."""
    for fp8 in (False, True):
        whole = {n: None if x is None else torch.cat([torch.full_like(x[:1], 0x7F if x.dtype == torch.uint8 else float("nan")), x]).to(device) for n, x in pool(fp8=fp8).items()}
        st = {n: None if x is None else x[1:] for n, x in whole.items()}                    # (page -1 lies in the same memory)
        full = torch.tensor([[0, 1, 2, 3], [0, 1, 4, 5], [0, 1, 2, 3], [0, 1, 2, 3], [0, 1, 2, 3], [0, 1, 6, 7]], dtype=torch.int32)
        context, cu, shared = ints(60, 64, 20, 0, 40, 41), ints(0, 6), ints(40)
        sparse = full.clone()
        sparse[1:, :2] = nobody
        sparse[2:5] = nobody                                                                 # they end inside
        sparse[5, 3] = nobody                                                                # 41 tokens: three pages
        if wide:
            full, sparse = (torch.cat([x, torch.full((6, 3000), -1, dtype=torch.int32)], 1) for x in (full, sparse))
        q = torch.randn(6, 12, 128, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).to(device)
        a, b = (ops.paged_decode_shared(q, st["k"], st["v"], t.to(device), context.to(device), cu.to(device), shared.to(device), k_scale=st["ks"], v_scale=st["vs"])
                for t in (full, sparse))
        assert torch.equal(a, b) and a.isfinite().all()


def test_tables_of_shared_pages():
    tables_of_shared_pages("cpu")
    tables_of_shared_pages("cpu", nobody=1_000_000)
