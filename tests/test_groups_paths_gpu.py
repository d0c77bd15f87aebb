"""What calls the operators of shared prompts and bounded caches on the GPU: the sampler, the log-probability passes and micro-steps of the trainers."""
import pytest
import torch

from tests.test_sampler_gpu import _models
from tests.test_trainers_gpu import _setup

pytestmark = pytest.mark.gpu

PAD = 2047


def _engine(fp8=False, graph=True, sync_every=8):
    from nanorlhf_b200.sampler.native_sampler import NativeSampler
    eng = NativeSampler(_models(), kv_cache_gb=1.0, sync_every=sync_every, use_cuda_graph=graph, kv_cache_dtype="fp8" if fp8 else "bf16")
    eng.sync_weights()
    return eng


def _prompts(lens=(5, 16, 17, 33, 64, 9, 31, 48)):
    g = torch.Generator().manual_seed(0)
    return [torch.randint(0, 2000, (L,), generator=g).tolist() for L in lens]


def _alike(a, b):
    """greedy rows agree until a near tie, which may tip either way"""
    assert a.shape == b.shape and torch.equal(a[:, 0], b[:, 0])
    assert (a == b).float().mean() > 0.9, (a == b).float().mean()


@pytest.mark.parametrize("graph", [True, False], ids=["graph", "eager"])
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_samples_over_shared_pages(fp8, graph):
    eng, prompts = _engine(fp8, graph), _prompts()
    plain = eng.generate(prompts, 4, 0.0, 1.0, 24, None, PAD, 1)
    shared = eng.generate(prompts, 4, 0.0, 1.0, 24, None, PAD, 1, shared_decode=True)
    _alike(plain, shared)
    assert torch.equal(eng.generate(prompts, 4, 0.0, 1.0, 24, None, PAD, 1), plain)            # (the graphs of one are not the other's)
    a, b, c = (eng.generate(prompts, 4, 0.9, 0.95, 24, None, PAD, s, shared_decode=True) for s in (3, 3, 4))
    assert torch.equal(a, b) and not torch.equal(a, c)
    assert torch.equal(eng.generate(prompts, 1, 0.0, 1.0, 24, None, PAD, 1, shared_decode=True), eng.generate(prompts, 1, 0.0, 1.0, 24, None, PAD, 1))


def test_groups_shrink_as_samples_finish():
    """rows leave at sync points, the batch is rebuilt, and what is left of a prompt still shares its pages"""
    eng, prompts = _engine(graph=False), _prompts((40, 65, 18, 33) * 12)            # (without graphs a batch is rebuilt whenever a row has finished)
    free = eng.generate(prompts, 4, 0.9, 0.95, 32, None, PAD, 11, shared_decode=True)
    eos = int(free[:, 4].mode().values)
    got = eng.generate(prompts, 4, 0.9, 0.95, 32, eos, PAD, 11, shared_decode=True)
    assert eng.stats["compactions"] > 0
    for row, whole in zip(got.tolist(), free.tolist()):
        end = row.index(eos) + 1 if eos in row else 32
        assert all(t == PAD for t in row[end:])
    _alike(got[(got != PAD).all(1)], free[(got != PAD).all(1)])


@pytest.mark.parametrize("graph", [True, False], ids=["graph", "eager"])
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_samples_over_a_bounded_cache(fp8, graph):
    eng, prompts = _engine(fp8, graph), _prompts()
    plain = eng.generate(prompts, 2, 0.0, 1.0, 40, None, PAD, 1)
    wide = eng.generate(prompts, 2, 0.0, 1.0, 40, None, PAD, 1, kv_budget=64 + 40 - 1)         # nothing to give up yet
    _alike(plain, wide)
    narrow = eng.generate(prompts, 2, 0.0, 1.0, 40, None, PAD, 1, kv_budget=24)
    assert torch.equal(narrow, eng.generate(prompts, 2, 0.0, 1.0, 40, None, PAD, 1, kv_budget=24))
    assert torch.equal(narrow[:, :9], wide[:, :9])                                             # up to the first eviction
    longest = torch.tensor([len(p) + 40 <= 24 + 8 for p in prompts]).repeat_interleave(2)
    assert not torch.equal(narrow[~longest], wide[~longest])                                   # 16 tokens and more of 64 have gone
    st = next(v for k, v in eng._state_pool.items() if v["mode"][0] == "scored" and v["scores0"].shape[2] < 104 + 16)
    assert int(st["ctx_lens"].max()) == 24 + 1 and int(st["positions"].max()) == 64 + 40 - 2


def test_a_bounded_cache_keeps_what_is_looked_at():
    """Keys that agree with every query are kept, whatever else goes: the operators as the sampler calls them, over three evictions."""
    from nanorlhf_b200 import ops
    g = torch.Generator().manual_seed(5)
    S, Hkv, D, budget, step = 3, 2, 128, 32, 16
    pages = 6
    k, v = (torch.randn(S * pages, Hkv, 16, D, generator=g).bfloat16().cuda() * 0.1 for _ in range(2))
    tables = torch.randperm(S * pages, generator=g).int().view(S, pages).cuda()
    lens, scores = torch.full((S,), 33, dtype=torch.int32, device="cuda"), torch.zeros(S, Hkv, 16 * pages, device="cuda")
    q = torch.randn(S, Hkv * 2, D, generator=g).bfloat16().cuda()
    special = [7, 19, 25]
    mean = q.view(S, Hkv, 2, D).float().mean(2)
    for s in range(S):
        for t in special:
            k[tables[s, t // 16].long(), :, t % 16] = mean[s].bfloat16()
            v[tables[s, t // 16].long(), :, t % 16] = float(t)
    kept = torch.arange(33, device="cuda").expand(S, Hkv, 33)
    for _ in range(3):
        for _ in range(step):
            ops.paged_decode_scored(q, k, v, tables, lens, scores)
            lens += 1
        lens -= 1
        index, kept_scores, lens = ops.kv_evict(k, v, tables, lens, scores, budget, 4, 8)
        scores[:, :, :budget] = kept_scores
        kept = torch.cat([kept, kept.new_full((S, Hkv, 64), 1000)], 2).gather(2, index.long())
        lens = lens + 1
        assert lens.tolist() == [budget + 1] * S
        assert all(t in kept[s, h].tolist() for t in [0, 1, 2, 3] + special for s in range(S) for h in range(Hkv))


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_the_token_that_is_fed_next_is_not_cached_yet(fp8):
    """it stands behind the kept ones whatever its place in the scores holds, and its place in the cache is free"""
    eng = _engine(fp8)
    eng.generate(_prompts((40,)), 1, 0.0, 1.0, 9, None, PAD, 1, kv_budget=47)
    st = next(v for v in eng._state_pool.values() if v["mode"][0] == "scored")
    st["ctx_lens"].fill_(1)
    st["ctx_lens"][0] = 41
    st["block_tables"][0, :3] = torch.tensor([2, 0, 1])
    for li in range(eng.cfg.num_hidden_layers):
        st[f"scores{li}"][0] = torch.arange(st[f"scores{li}"].shape[2], device="cuda").float()
        st[f"scores{li}"][0, :, 40] = -1.0
    k = eng.k_cache[0].clone()
    eng._evict(st, 16, 0, 0)
    assert st["ctx_lens"][0] == 17 and (st["ctx_lens"][1:] == 1).all()
    row = lambda x, t: x[st["block_tables"][0, t // 16].long(), :, t % 16]                               # noqa: E731
    for j in range(16):                                                                                  # tokens 24 to 39 of the forty
        assert torch.equal(row(eng.k_cache[0], j), row(k, 24 + j)) and (st["scores1"][0, :, j] == 24 + j).all()


def test_evicted_rows_are_moved_with_their_scores():
    """rows finish, others are admitted: a batch of few pages gives what one of many gives"""
    eng, prompts = _engine(), _prompts((40, 65, 18, 33) * 16)
    args = (prompts, 2, 0.9, 0.95, 40, None, PAD, 5)
    free = eng.generate(*args, kv_budget=48)
    eos = int(free[:, 12].mode().values)
    many = eng.generate(prompts, 2, 0.9, 0.95, 40, eos, PAD, 5, kv_budget=48)
    few = _engine()
    few.max_num_seqs = 40
    got = few.generate(prompts, 2, 0.9, 0.95, 40, eos, PAD, 5, kv_budget=48)
    assert torch.equal(many[:, 0], got[:, 0]) and (many == got).float().mean() > 0.9


def _lm(seed):
    from nanorlhf_b200.models.qwen2 import Qwen2Config, Qwen2ForCausalLM
    cfg = Qwen2Config(vocab_size=2048, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128)
    return Qwen2ForCausalLM.from_config(cfg, torch.bfloat16, "cuda", seed=seed)


def test_log_probabilities_of_shared_prompts():
    """bf16 activations round at other places; either is as far from the float32 model as the other"""
    from nanorlhf_b200.models.qwen2 import response_logprobs
    m, g = _lm(3), torch.Generator().manual_seed(1)
    q = torch.randint(0, 2000, (5, 70), generator=g)
    q[1, :30] = PAD
    qr = torch.cat([q[torch.tensor([0, 1, 0, 1, 2, 0, 3, 4, 4])], torch.randint(0, 2000, (9, 50), generator=g)], 1).cuda()
    qr[2, 70 + 20:] = PAD
    m32 = _lm(3).float().cpu()
    want = response_logprobs(m32, qr.cpu(), 70, PAD, 0.9)[0]
    plain, shared = (response_logprobs(m, qr, 70, PAD, 0.9, share_prompts=s)[0].detach().cpu() for s in (False, True))
    off, off_shared = (want - plain).abs(), (want - shared).abs()
    assert off_shared.mean() <= 1.25 * off.mean() and off_shared.max() <= 2 * off.max()
    from nanorlhf_b200.ops import native
    n = native.launches()
    response_logprobs(m, qr, 70, PAD, 0.9, share_prompts=True)
    assert native.launches() > n


@pytest.mark.parametrize("algo", ["grpo", "ppo"])
def test_graphed_micro_step_of_shared_prompts(tmp_path, algo):
    """replays over other numbers of groups give what eager micro-steps give"""
    from nanorlhf_b200.trainer import GRPOTrainer, PPOTrainer
    from nanorlhf_b200.trainer.graphed import GraphedMicroStep
    cls, extra = (PPOTrainer, {"policy_learning_rate": 1e-4, "value_learning_rate": 2e-4}) if algo == "ppo" else (GRPOTrainer, {"grpo_sample_N": 4})
    t = _setup(tmp_path, cls, extra, gradient_checkpointing=False, train_cuda_graph="on", share_prompts=True)
    dev, pad = t.device, t.tokenizer.pad_token_id
    B, ctx, T_r = 6, 40, 24
    gen = torch.Generator().manual_seed(0)

    def make(prompts, rlens):
        q = torch.randint(0, 4000, (6, ctx), generator=gen)
        qr = torch.full((B, ctx + T_r), pad, dtype=torch.long)
        pm = torch.ones(B, T_r, dtype=torch.bool)
        for b, (p, rl) in enumerate(zip(prompts, rlens)):
            qr[b, :ctx] = q[p]
            qr[b, ctx:ctx + rl] = torch.randint(0, 4000, (rl,), generator=gen)
            pm[b, :rl] = False
        f = lambda: (torch.randn(B, T_r, generator=gen) * 0.1 - 2.0).to(dev)                              # noqa: E731
        mb = {"query_responses": qr.to(dev), "padding_mask": pm.to(dev), "logprobs": f(), "ref_logprobs": f(), "advantages": f() + 2.0, "context_length": ctx}
        if algo == "ppo":
            mb.update(padding_mask_p1=pm.to(dev), values=f(), returns=f())
        return mb

    params = [p for p in t.model.parameters() if p.requires_grad]

    def run(step, mb):
        t.optimizer.zero_grad()
        vec = step(mb, ctx, pad).clone()
        return vec, torch.cat([p.grad.detach().float().reshape(-1) for p in params]).clone()

    t.model.train()
    g = GraphedMicroStep(t)
    one, two = make([0, 0, 1, 1, 1, 2], [24, 17, 20, 3, 9, 24]), make([0, 1, 1, 0, 2, 2], [20, 20, 12, 8, 13, 24])
    first = run(g, one)
    again, other = run(g, one), run(g, two)
    assert g.replays == 2 and g.eager == 1, (g.replays, g.eager)
    fresh = run(GraphedMicroStep(t), two)
    for a, b in ((first, again), (other, fresh)):
        assert torch.allclose(a[0], b[0], rtol=1e-4, atol=1e-5)
        assert (a[1] - b[1]).abs().max() <= 1e-3 * a[1].abs().max() + 1e-7 and a[1].abs().max() > 0


@pytest.mark.parametrize("kw", [dict(share_prompts=True, shared_decode=True), dict(share_prompts=True, kv_budget=32, kv_cache_dtype="bf16"),
                                dict(share_prompts=True, gradient_checkpointing=True, kv_budget=32)], ids=["shared", "bounded", "checkpointing"])
def test_a_trainer_with_both(kw, tmp_path):
    from nanorlhf_b200.trainer import GRPOTrainer
    t = _setup(tmp_path, GRPOTrainer, {"grpo_sample_N": 4}, train_samples_per_prompt=4, per_device_train_batch_size=4, total_episodes=32, **kw)
    t.train()
    assert t.state.global_step == 2 and all(torch.isfinite(p).all() for p in t.policy.parameters())
