"""What calls the vocabulary operators on the CPU: the sampler's filters, a teacher's view of responses and the loss against it, the trainer's settings."""
import pytest
import torch

from nanorlhf_b200 import ops
from nanorlhf_b200.models.qwen2 import Qwen2Config, Qwen2ForCausalLM, build_logprob_plan, response_distill_loss, response_logprobs, response_top_logprobs
from nanorlhf_b200.sampler.engine import generate

PAD, CTX = 199, 6


class _Tok:
    pad_token_id, eos_token_id = PAD, None


def _model(seed):
    cfg = Qwen2Config(vocab_size=200, hidden_size=32, intermediate_size=64, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=1, head_dim=16,
                      tie_word_embeddings=True)
    return Qwen2ForCausalLM.from_config(cfg, torch.float32, seed=seed)


def _batch():
    g = torch.Generator().manual_seed(0)
    qr = torch.randint(0, 190, (3, CTX + 8), generator=g)
    qr[0, :3] = PAD                                        # a short query
    qr[1, CTX + 5:] = PAD                                  # a short response
    qr[2, CTX:] = PAD                                      # none
    return qr


def test_filters_of_the_sampler():
    m, prompts = _model(1), [[1, 2, 3], [4, 5, 6, 7]]
    greedy = generate(2, m, _Tok, prompts, 0.0, 6, top_p=1.0, seed=1)
    assert torch.equal(generate(2, m, _Tok, prompts, 1.3, 6, top_p=1.0, seed=1, top_k=1), greedy)
    assert torch.equal(generate(2, m, _Tok, prompts, 1.3, 6, top_p=1.0, seed=1, min_p=1.0), greedy)
    a, b, c = (generate(4, m, _Tok, prompts, 1.3, 6, top_p=0.9, seed=s, top_k=20, min_p=0.01) for s in (3, 3, 4))
    assert torch.equal(a, b) and not torch.equal(a, c)
    for kw in (dict(top_k=-1), dict(min_p=1.5), dict(min_p=-0.1)):
        with pytest.raises(ValueError):
            generate(1, m, _Tok, prompts, 1.0, 2, seed=1, **kw)


def test_sampled_tokens_are_among_the_k_first():
    m, prompts = _model(1), [[1, 2, 3], [4, 5, 6, 7]]
    out = generate(8, m, _Tok, prompts, 2.0, 1, top_p=1.0, seed=5, top_k=3)
    for i, p in enumerate(prompts):
        ids = torch.tensor(p)
        logits = m(ids, torch.tensor([0, len(p)], dtype=torch.int32), torch.arange(len(p)), len(p))[-1]
        assert set(out[8 * i:8 * i + 8, 0].tolist()) <= set(logits.topk(3).indices.tolist())


def test_teacher_and_student_over_responses():
    teacher, student, qr = _model(1), _model(2), _batch()
    logp, idx = response_top_logprobs(teacher, qr, CTX, PAD, 10, 0.9)
    assert logp.shape == idx.shape == (3, 8, 10)
    # the response's own tokens: where they are among the listed, their log-probability is that of response_logprobs
    own = response_logprobs(teacher, qr, CTX, PAD, 0.9)[0]
    hit = idx == qr[:, CTX:, None]
    assert torch.allclose(logp[hit], own[hit.any(-1)], atol=1e-5)
    plan = build_logprob_plan(qr, CTX, PAD)
    valid = torch.zeros(3, 8, dtype=torch.bool)
    valid[plan["r"], plan["c"]] = True
    assert (idx[~valid] == -1).all() and (logp[~valid] == -float("inf")).all() and (idx[valid] >= 0).all()

    w = torch.rand(3, 8)
    loss, token = response_distill_loss(student, qr, CTX, PAD, logp, idx, w, 0.9, 0.5)
    assert token.shape == (3, 8) and (token[~valid] == 0).all() and abs(loss.item() - (w * token).sum().item()) < 1e-6
    mean, token = response_distill_loss(student, qr, CTX, PAD, logp, idx, temperature=0.9)
    assert abs(mean.item() - token.sum().item() / valid.sum().item()) < 1e-6
    mean.backward()
    hidden = student.hidden_states(plan["ids"], plan["cu"], plan["pos"], plan["max_seqlen"])[plan["src"]]
    want, _ = ops.distill_loss(student.lm_head(hidden), logp[valid], idx[valid], temperature=0.9)
    got = student.model.layers[0].mlp.down_proj.weight.grad.clone()
    student.zero_grad()
    want.backward()
    assert torch.allclose(got, student.model.layers[0].mlp.down_proj.weight.grad, atol=1e-7)
    same, _ = response_distill_loss(teacher, qr, CTX, PAD, logp, idx, temperature=0.9)
    assert abs(same.item()) < 1e-6
    with pytest.raises(ValueError):
        response_distill_loss(student, qr, CTX, PAD, logp[:2], idx[:2])
    with pytest.raises(ValueError):
        response_distill_loss(student, qr, CTX, PAD, logp, idx, w[:, :3])


def test_settings():
    from nanorlhf_b200.config import RLConfig
    a = RLConfig()
    assert a.top_k == 0 and a.min_p == 0.0


@pytest.mark.parametrize("kw", [dict(top_k=40), dict(min_p=0.05)])
def test_trainer_does_not_score_with_the_nucleus_what_other_filters_cut(tmp_path, kw):
    from nanorlhf_b200.config import RLConfig
    from nanorlhf_b200.reward.api import LengthReward
    from nanorlhf_b200.trainer import ReinforceTrainer
    from nanorlhf_b200.utils.data import synthetic_hh_dataset
    from nanorlhf_b200.utils.tokenizer import ByteTokenizer

    tok = ByteTokenizer()
    cfg = Qwen2Config.tiny(vocab_size=tok.vocab_size)
    models = [Qwen2ForCausalLM.from_config(cfg, torch.float32, seed=1) for _ in range(2)]
    base = dict(output_dir=str(tmp_path), response_length=4, per_device_train_batch_size=2, gradient_accumulation_steps=2, num_mini_batches=2, total_episodes=8,
                learning_rate=1e-3, sampler="torch", report_to="none", **kw)
    data = synthetic_hh_dataset(tok, 8, max_prompt_tokens=8)
    ReinforceTrainer(RLConfig(**base), tok, *models, data, reward_func=LengthReward(3))
    with pytest.raises(ValueError, match="logprob_top_p_consistent"):
        ReinforceTrainer(RLConfig(**base, logprob_top_p_consistent=True), tok, *models, data, reward_func=LengthReward(3))
