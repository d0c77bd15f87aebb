"""What calls the operators of shared prompts and bounded caches on the CPU: log-probabilities, micro-steps, batches, the trainers, the options of generate."""
import pytest
import torch

from nanorlhf_b200.models.qwen2 import (Qwen2Config, Qwen2ForCausalLM, Qwen2ForSequenceClassification, build_logprob_plan, planned_response_logprobs,
                                        response_distill_loss, response_logprobs, response_top_logprobs)
from nanorlhf_b200.sampler.engine import generate
from nanorlhf_b200.utils.batching import create_prompt_batches
from tests.test_trainers_e2e import GRPOTrainer, PPOTrainer, RLOOTrainer, SparseGRPOTrainer, build

PAD, CTX = 199, 6
# two float32 runs that add up in another order: sums of at most 64 terms of order 1 are 64 * 2^-24 = 4e-6 apart, and a dozen of them follow one another
CLOSE = 5e-5


class _Tok:
    pad_token_id, eos_token_id = PAD, None


def _model(seed=1, cls=Qwen2ForCausalLM):
    cfg = Qwen2Config(vocab_size=200, hidden_size=32, intermediate_size=64, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=1, head_dim=16,
                      tie_word_embeddings=True)
    return cls.from_config(cfg, torch.float32, seed=seed)


def _batch(prompts):
    """row i answers query prompts[i]; query 1 is short, query 2 is a single token, query 3 is empty; one response is short, one empty"""
    g = torch.Generator().manual_seed(0)
    q = torch.randint(0, 190, (8, CTX), generator=g)
    q[1, :3] = PAD
    q[2, :CTX - 1] = PAD
    q[3] = PAD
    qr = torch.cat([q[torch.tensor(prompts)], torch.randint(0, 190, (len(prompts), 8), generator=g)], 1)
    qr[1, CTX + 5:] = PAD
    qr[2, CTX:] = PAD
    return qr


ROWS = [[0, 0, 0, 0], [0, 1, 0, 1, 4], [1, 1, 2, 2, 2, 5], [3, 3, 0, 3], [0, 1, 4, 5], [0, 0, 1]]


@pytest.mark.parametrize("prompts", ROWS, ids=str)
def test_shared_prompts_change_no_log_probability_and_no_gradient(prompts):
    m, critic, qr = _model(), _model(2, Qwen2ForSequenceClassification), _batch(prompts)
    weights = torch.randn(len(prompts), 8, generator=torch.Generator().manual_seed(1))
    got = []
    for share in (False, True):
        m.zero_grad(), critic.zero_grad()
        out = response_logprobs(m, qr, CTX, PAD, 0.9, want_entropy=True, value_model=critic, share_prompts=share)
        ((out[0] + out[2]) * weights).sum().backward()
        got.append((out, [p.grad.clone() for p in list(m.parameters()) + list(critic.parameters())]))
    for a, b in zip(*(g[0] for g in got)):
        assert (a - b).abs().max() <= CLOSE * max(1, a.abs().max())
    for a, b in zip(*(g[1] for g in got)):
        assert (a - b).abs().max() <= CLOSE * max(1, a.abs().max())


def test_what_is_packed_once():
    qr = _batch([0, 1, 0, 1, 4])
    plan, plain = build_logprob_plan(qr, CTX, PAD, True), build_logprob_plan(qr, CTX, PAD)
    assert plain["cu_groups"] is None and build_logprob_plan(_batch([0, 1, 4]), CTX, PAD, True)["cu_groups"] is None
    assert plan["ids"].numel() == plain["ids"].numel() - (CTX - 1) - 2           # but for the last column of either query
    assert sorted((plan["cu_groups"][1:] - plan["cu_groups"][:-1]).tolist()) == [1, 3, 3]
    assert plan["cu"].numel() == 1 + 7 and plan["cu"][-1] == plan["ids"].numel()
    assert torch.equal(plan["ids"], qr.view(-1)[plan["flat"]])
    slots = lambda p: sorted(zip(p["r"].tolist(), p["c"].tolist(), p["targets"].tolist()))                        # noqa: E731
    assert slots(plan) == slots(plain)
    assert build_logprob_plan(qr, 1, PAD, True)["cu_groups"] is None             # a query of one column has nothing in front of its last


@pytest.mark.parametrize("prompts", ROWS[:4], ids=str)
def test_padded_plan_of_groups(prompts):
    from nanorlhf_b200.trainer.graphed import GraphedMicroStep
    m, qr = _model(), _batch(prompts)
    B, plan = len(prompts), build_logprob_plan(qr, CTX, PAD, True)
    T, R = plan["ids"].numel(), plan["src"].numel()
    shapes = set()
    for more in (0, 9):
        padded = GraphedMicroStep._pad_plan(plan, B, PAD, T + more, R + more)
        a, b = (planned_response_logprobs(m, p, B, 8, 0.9, True, max_seqlen=14) for p in (plan, padded))
        assert torch.allclose(a[0], b[0], atol=CLOSE) and torch.allclose(a[1], b[1], atol=CLOSE)
        shapes.add((padded["cu"].numel(), padded["cu_groups"].numel()))
    assert shapes == {(B + B // 2 + 2, B + 1)}                                   # the rows alone say how large the tables are


def test_teacher_and_student_share_prompts():
    teacher, student, qr = _model(1), _model(2), _batch([0, 1, 0, 1, 4])
    top = [response_top_logprobs(teacher, qr, CTX, PAD, 5, 0.9, share_prompts=s) for s in (False, True)]
    assert torch.equal(top[0][1], top[1][1])
    real = top[0][1] >= 0
    assert (top[0][0][real] - top[1][0][real]).abs().max() <= CLOSE
    losses = [response_distill_loss(student, qr, CTX, PAD, *top[0], share_prompts=s) for s in (False, True)]
    assert (losses[0][1] - losses[1][1]).abs().max() <= CLOSE * max(1, losses[0][1].abs().max())


def test_gradient_checkpointing_of_groups():
    m, qr = _model(), _batch([0, 0, 1, 1])
    m.train()
    grads = []
    for on in (False, True):
        m.gradient_checkpointing_enable() if on else m.gradient_checkpointing_disable()
        m.zero_grad()
        response_logprobs(m, qr, CTX, PAD, 1.0, share_prompts=True)[0].sum().backward()
        grads.append([p.grad.clone() for p in m.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_batches_keep_prompts_together():
    lens, shared, prompts = [10, 12, 11, 30, 9, 13, 12], [6, 6, 6, 20, 5, 6, 5], [0, 0, 0, 1, 2, 0, 2]
    for budget in (1, 12, 20, 25, 40, 1000):
        batches = create_prompt_batches(lens, shared, prompts, budget)
        assert sorted(i for b in batches for i in b) == list(range(7))
        for b in batches:
            tokens = sum(lens[i] - shared[i] for i in b) + sum(max(shared[i] for i in b if prompts[i] == p) for p in {prompts[i] for i in b})
            assert tokens <= budget or len(b) == 1
    assert create_prompt_batches(lens, shared, prompts, 28) == [[4, 6], [0, 2, 1, 5], [3]]
    assert create_prompt_batches([], [], [], 5) == []


@pytest.mark.parametrize("cls,extra,kw", [
    (GRPOTrainer, {"grpo_sample_N": 4}, dict(train_samples_per_prompt=4)), (RLOOTrainer, {"rloo_sample_N": 4}, {}),
    (PPOTrainer, {"policy_learning_rate": 1e-3, "value_learning_rate": 2e-3}, {}), (SparseGRPOTrainer, {"grpo_sample_N": 4}, dict(train_samples_per_prompt=4)),
], ids=["grpo", "rloo", "ppo", "sparse"])
def test_algorithms_with_shared_prompts(cls, extra, kw, tmp_path):
    t = build(cls, tmp_path, extra, share_prompts=True, shared_decode=True, **kw)
    before = [p.detach().clone() for p in t.policy.parameters() if p.requires_grad]
    t.train()
    after = [p for p in t.policy.parameters() if p.requires_grad]
    assert t.state.global_step == 2 and any(not torch.equal(a, b) for a, b in zip(before, after)) and all(torch.isfinite(p).all() for p in after)


def test_log_probability_pass_of_a_trainer(tmp_path):
    t = build(GRPOTrainer, tmp_path, {"grpo_sample_N": 4})
    g = torch.Generator().manual_seed(3)
    q, r = torch.randint(5, 90, (3, 7), generator=g).repeat_interleave(4, 0), torch.randint(5, 90, (12, 10), generator=g)
    q[4:8, :2] = t.tokenizer.pad_token_id
    plain = t.logprob_pass(q, r)
    t.args.share_prompts = True
    for budget in (20, 60, t.args.token_budget_fwd):
        t.args.token_budget_fwd = budget
        for a, b in zip(plain[1:3], t.logprob_pass(q, r)[1:3]):
            assert (a - b).abs().max() <= CLOSE * max(1, a.abs().max())


def test_groups_of_batch_rows():
    from nanorlhf_b200.sampler.native_sampler import NativeSampler

    class Engine:
        PAGE = 16
    st = {"S": 12, "cu_groups": torch.zeros(13, dtype=torch.int32), "shared_lens": torch.zeros(12, dtype=torch.int32)}
    # of prompt 0 (33 tokens) three samples are left, of prompt 1 (40) one, of prompt 2 (9) four, of prompt 3 (16) two
    NativeSampler._share_pages(Engine, st, [0, 1, 3, 6, 8, 9, 10, 11, 12, 15], 4, [33, 40, 9, 16])
    assert st["cu_groups"].tolist() == [0, 3, 4, 8, 10] + [10] * 8
    assert st["shared_lens"].tolist() == [32, 0, 0, 16] + [0] * 8


def test_options_of_generate():
    m, prompts = _model(), [[1, 2, 3], [4, 5, 6, 7]]
    plain = generate(2, m, _Tok, prompts, 0.0, 6, seed=1)
    assert torch.equal(generate(2, m, _Tok, prompts, 0.0, 6, seed=1, shared_decode=True), plain)
    for kw in (dict(kv_budget=-1), dict(kv_budget=1.5), dict(kv_budget=3), dict(kv_budget=8, kv_recent=5), dict(kv_budget=8, kv_sinks=-1),
               dict(kv_budget=8, kv_recent=-1), dict(kv_budget=64, shared_decode=True), dict(kv_budget=64)):
        with pytest.raises(ValueError):
            generate(1, m, _Tok, prompts, 0.0, 2, seed=1, **kw)
