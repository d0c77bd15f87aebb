"""What calls the vocabulary operators on the device: both rollout engines' filters and a distillation step of a policy over its own rollout."""
import pytest
import torch

from test_nezavik_gpu import _model as _hybrid_model, _save, _tokens
from test_sampler_gpu import _models

from nanorlhf_b200 import ops
from nanorlhf_b200.ops import native

pytestmark = pytest.mark.gpu


def test_filters_of_the_paged_engine():
    from nanorlhf_b200.sampler.native_sampler import NativeSampler
    m = _models()
    prompts = [[1, 2, 3, 4, 5, 6, 7], [8, 9, 10]]
    eng = NativeSampler(m, kv_cache_gb=1.0, sync_every=8)
    eng.sync_weights()
    plain = eng.generate(prompts, 4, 0.9, 0.95, 20, None, 2047, 11)
    greedy = eng.generate(prompts, 4, 0.0, 1.0, 20, None, 2047, 11)
    # one token kept: the order's first, ties and all, which is what the arg-max takes
    assert torch.equal(eng.generate(prompts, 4, 1.5, 1.0, 20, None, 2047, 11, top_k=1), greedy)
    a = eng.generate(prompts, 4, 0.9, 0.95, 20, None, 2047, 11, top_k=30, min_p=0.01)
    b = eng.generate(prompts, 4, 0.9, 0.95, 20, None, 2047, 11, top_k=30, min_p=0.01)
    c = eng.generate(prompts, 4, 0.9, 0.95, 20, None, 2047, 12, top_k=30, min_p=0.01)
    assert torch.equal(a, b) and not torch.equal(a, c)
    assert torch.equal(eng.generate(prompts, 4, 0.9, 0.95, 20, None, 2047, 11), plain)          # the graph of other filters is not reused
    eager = NativeSampler(m, kv_cache_gb=1.0, sync_every=8, use_cuda_graph=False)
    eager.sync_weights()
    # the engines' batches are padded differently, so that products may round differently: rows agree in their first token at least
    assert torch.equal(eager.generate(prompts, 4, 0.9, 0.95, 1, None, 2047, 11, top_k=30, min_p=0.01)[:, 0], a[:, 0])


def test_filters_of_the_step_engine(tmp_path):
    from nanorlhf_b200.models.registry import load_model
    from nanorlhf_b200.sampler.engine import generate
    from nanorlhf_b200.utils.tokenizer import ByteTokenizer
    cfg, W = _hybrid_model("single_heads", seed=5)
    model = load_model(_save(tmp_path, cfg, W), torch_dtype=torch.bfloat16, device="cuda")
    tok = ByteTokenizer(vocab_size=cfg["vocab"])
    prompts = [_tokens(cfg, n, 80 + n) for n in (4, 9)]
    kw = dict(top_p=0.95, backend="native", eos_token_id=5)
    greedy = generate(3, model, tok, prompts, 0.0, 10, seed=7, **kw)
    assert torch.equal(generate(3, model, tok, prompts, 0.9, 10, seed=7, top_k=1, **kw), greedy)
    a, b = (generate(3, model, tok, prompts, 0.9, 10, seed=7, top_k=8, min_p=0.02, **kw) for _ in range(2))
    assert torch.equal(a, b)


def test_uniforms_are_functions_of_seed_row_and_step():
    ids = torch.arange(4000, dtype=torch.int32, device="cuda")
    steps = torch.zeros_like(ids)
    u = native.row_uniforms(5, 0, ids, steps)
    assert (u >= 0).all() and (u < 1).all()
    assert torch.equal(u[1000:1001], native.row_uniforms(5, 0, ids[1000:1001], steps[:1]))
    assert torch.equal(native.row_uniforms(5, 3, ids, steps), native.row_uniforms(5, 0, ids, steps + 3))
    assert not torch.equal(u, native.row_uniforms(6, 0, ids, steps)) and not torch.equal(u, native.row_uniforms(5, 1, ids, steps))
    # mean of 4000 uniform numbers: standard deviation 1 / sqrt(12 * 4000) = 0.0046, six of them
    assert abs(u.mean().item() - 0.5) < 0.028


def test_a_row_without_a_finite_logit_gives_token_zero():
    z = torch.full((2, 50), float("nan"), device="cuda")
    z[1] = torch.arange(50.0, device="cuda")
    ids = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert native.sample_tokens(z, 1.0, 1.0, 1, ids, ids, top_k=1).tolist() == [0, 49]


def test_distillation_step_of_a_policy_over_its_own_rollout():
    from nanorlhf_b200.models.qwen2 import Qwen2Config, Qwen2ForCausalLM, response_distill_loss, response_top_logprobs
    from nanorlhf_b200.sampler.engine import generate
    from nanorlhf_b200.utils.tokenizer import ByteTokenizer
    cfg = Qwen2Config(vocab_size=2048, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=1, head_dim=128,
                      tie_word_embeddings=True)
    student, teacher = (Qwen2ForCausalLM.from_config(cfg, torch.bfloat16, "cuda", seed=s) for s in (1, 2))
    tok = ByteTokenizer(vocab_size=2048)
    pad, ctx = tok.pad_token_id, 5
    out = generate(2, student, tok, [[1, 2, 3, 4, 5], [7, 8, 9, 11, 12]], 0.9, 8, top_p=0.95, top_k=50, seed=1, backend="native", eos_token_id=-1)
    qr = torch.cat([torch.tensor([[1, 2, 3, 4, 5], [7, 8, 9, 11, 12]], device="cuda").repeat_interleave(2, 0), out], 1)
    logp, idx = response_top_logprobs(teacher, qr, ctx, pad, 32)
    loss, token = response_distill_loss(student, qr, ctx, pad, logp, idx)
    loss.backward()
    grads = [p.grad for p in student.parameters()]
    assert torch.isfinite(loss) and loss.item() > 0 and all(g is not None and torch.isfinite(g).all() for g in grads)
    # the head's gradient against the same loss of materialised logits in float64
    from nanorlhf_b200.models.qwen2 import build_logprob_plan
    from nanorlhf_b200.ops import reference as ref
    plan = build_logprob_plan(qr, ctx, pad)
    hidden = student.hidden_states(plan["ids"], plan["cu"], plan["pos"], plan["max_seqlen"])[plan["src"]].detach()
    r, c = plan["r"], plan["c"]
    w = student.lm_head.weight.detach()
    h64 = hidden.double().requires_grad_()
    want, tw = ref.distill_loss(h64 @ w.double().t(), logp[r, c], idx[r, c], None, 1.0, 0.0, True)
    assert abs(loss.item() - want.item()) < 1e-5 * (1 + want.item()) and ((token[r, c] - tw).abs() <= 1e-5 * (1 + tw)).all()
    x = hidden.clone().requires_grad_()
    ops.lmhead_distill_loss(x, w, logp[r, c], idx[r, c])[0].backward()
    want.backward()
    assert ((x.grad.double() - h64.grad).norm() / h64.grad.norm()).item() <= 2.0 ** -7
