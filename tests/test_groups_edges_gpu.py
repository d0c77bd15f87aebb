"""Attention over shared prefixes, decode attention over pages with scores and eviction: calls at the borders of what their documentation allows."""
import math

import pytest
import torch

import groups_oracle as oracle
from nanorlhf_b200 import ops
from nanorlhf_b200.ops import native
from tests.test_groups_gpu import DEV, SCALE, fill, gen, offsets, packed_inputs, pages_of, shared_batch, widen, within

pytestmark = pytest.mark.gpu


def offset(x):
    """the same numbers, contiguous, in a buffer of which they begin at the second element"""
    return torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(x.shape)


# ---- where inputs lie ----------------------------------------------------------------------------------------------------------------------
def test_packed_inputs_that_do_not_start_on_16_bytes():
    groups = [[33, 20, 70], [5]]
    q, k, v, dout, cu, cg = packed_inputs(groups, 4, 2, 101)
    # first what the kernels are handed, without a launch
    for x in native.ext().attn_groups_arguments(offset(q), offset(k), offset(v), cu, cg, None)[:3]:
        assert x.data_ptr() % 16 == 0
    results = []
    for place in (lambda x: x.contiguous(), offset):
        leaves = [place(x).detach().requires_grad_() for x in (q, k, v)]
        out = ops.attention_shared_prefix(*leaves, cu, cg)
        results.append((out.detach(), *torch.autograd.grad(out, leaves, place(dout))))
    assert all(x.data_ptr() % 16 for x in leaves)
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_packed_inputs_of_one_row_repeated():
    """expanded rows, and a gradient that is one (of a sum)"""
    groups = [[33, 20]]
    q, k, v, _, cu, cg = packed_inputs(groups, 4, 2, 102)
    q, k, v = (x[:1].expand(53, -1, -1) for x in (q, k, v))
    dout = torch.ones(1, 1, 1, dtype=torch.bfloat16, device=DEV).expand(53, 4, 128)
    for x in native.ext().attn_groups_arguments(q, k, v, cu, cg, None)[:3]:
        assert x.stride(0) > 0
    results = []
    for place in (lambda x: x.contiguous(), lambda x: x):
        leaves = [place(x).detach().requires_grad_() for x in (q, k, v)]
        out = ops.attention_shared_prefix(*leaves, cu, cg)
        results.append((out.detach(), *torch.autograd.grad(out, leaves, place(dout))))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("fp8", [False, True])
def test_decode_queries_that_do_not_start_on_16_bytes(fp8):
    st = shared_batch(103, [(100, [133, 101, 117]), (0, [33])], 2, fp8)
    q = torch.randn(4, 12, 128, generator=gen(103), device=DEV).to(torch.bfloat16)
    kw = {"k_scale": st["ks"], "v_scale": st["vs"]}
    args, rows = (st["k"], st["v"], st["tables"], st["context"]), []
    for x in (q, offset(q), q[:1].expand(4, -1, -1), q[:1].expand(4, -1, -1).contiguous()):
        scores = torch.zeros(4, 2, 133, device=DEV)
        out, _ = ops.paged_decode_scored(x, *args, scores, **kw)
        rows.append((ops.paged_decode_shared(x, *args, st["cu"], st["shared"], **kw), out, scores))
    bits = lambda x: x.view(torch.int16 if x.dtype == torch.bfloat16 else torch.int32)  # noqa: E731
    for i in (0, 2):
        for a, b in zip(rows[i], rows[i + 1]):
            assert torch.equal(bits(a), bits(b))              # (the scored rows' own copies of shared tokens are NaN)


@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("groups", [0, 2])
def test_rows_without_any_sequence(rows, groups):
    """they are behind the last one: 0, and so are their gradients"""
    q, k, v, dout, cu, _ = packed_inputs([[rows]], 4, 2, 104)
    cu, cg = cu[:1].contiguous(), torch.zeros(groups + 1, dtype=torch.int32, device=DEV)
    junk = torch.full((50, 1024, 128), float("nan"), device=DEV)             # what the allocator hands out next is not zero
    del junk
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = ops.attention_shared_prefix(*leaves, cu, cg)
    for x in (out, *torch.autograd.grad(out, leaves, dout)):
        assert torch.equal(x, torch.zeros_like(x))
    with torch.no_grad():
        assert torch.equal(ops.attention_shared_prefix(q, k, v, cu, cg), torch.zeros_like(q))


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_a_tangent_is_refused(which, recorded):
    """... and not lost; inputs without one go through"""
    import torch.autograd.forward_ad as fwd
    *qkv, _, cu, cg = packed_inputs([[4, 4]], 2, 1, 107)
    qkv = [x.contiguous().requires_grad_(recorded) for x in qkv]
    plain = ops.attention_shared_prefix(*qkv, cu, cg)
    with fwd.dual_level():
        assert torch.equal(ops.attention_shared_prefix(*qkv, cu, cg), plain)
        qkv[which] = fwd.make_dual(qkv[which], torch.ones_like(qkv[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.attention_shared_prefix(*qkv, cu, cg)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            ops.attention_shared_prefix(*qkv, cu, cg)


@pytest.mark.parametrize("recorded", [False, True])
def test_a_tangent_is_refused_by_plain_packed_attention(recorded):
    import torch.autograd.forward_ad as fwd
    *qkv, _, cu, _ = packed_inputs([[4], [5]], 2, 1, 108)
    qkv = [x.contiguous().requires_grad_(recorded) for x in qkv]
    plain = ops.attention_varlen(*qkv, cu, 5)
    with fwd.dual_level():
        assert torch.equal(ops.attention_varlen(*qkv, cu, 5), plain)
        with pytest.raises(RuntimeError):
            ops.attention_varlen(fwd.make_dual(qkv[0], torch.ones_like(qkv[0])), *qkv[1:], cu, 5)


# ---- shared pages --------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("groups", [[(200, [50, 0, 33, 64]), (70, [0, 0]), (64, [100])], [(200, [65 + i % 40 for i in range(40)])],
                                    [(40 + 100 * (i % 3), [(7 * i) % 60, i % 5]) for i in range(1100)]], ids=["short", "one", "many"])
def test_shared_tokens_behind_all_contexts_are_nobodys(groups, fp8, wide):
    """Rows that all end inside what they share: tables need not say anything of the pages behind, and places behind the longest row hold anything."""
    kv, heads, width = 2, 12, 13
    rows, blocks = [], 1
    for shared, ctxs in groups:
        n = (max(ctxs) + 15) // 16
        first = list(range(blocks, blocks + n))
        blocks += n
        for c in ctxs:
            whole = first[:shared // 16]
            own = max(0, (c + 15) // 16 - len(whole))
            rows.append((whole if c else []) + list(range(blocks, blocks + own)))
            blocks += own
        rows[len(rows) - len(ctxs)] = first                    # the first row's pages hold what anybody sees of the prefix
    st, g = pages_of(105, blocks, kv, fp8), gen(105)           # (page 0, of NaN, stands for what tables hold behind)
    at = 0
    for shared, ctxs in groups:
        fill(st, g, rows[at], 0, max(ctxs))
        for i, c in enumerate(ctxs):
            if i:
                fill(st, g, rows[at + i], shared, c)
        at += len(ctxs)
    st["tables"] = torch.tensor([r + [0] * (width - len(r)) for r in rows], dtype=torch.int32, device=DEV)
    st["context"] = torch.tensor([c for _, cs in groups for c in cs], dtype=torch.int32, device=DEV)
    cu, shared_lens = offsets([len(cs) for _, cs in groups]), torch.tensor([n for n, _ in groups], dtype=torch.int32, device=DEV)
    if wide:
        widen(st)
    q = torch.randn(len(rows), heads, 128, generator=gen(106), device=DEV).to(torch.bfloat16)
    out = ops.paged_decode_shared(q, st["k"], st["v"], st["tables"], st["context"], cu, shared_lens, k_scale=st["ks"], v_scale=st["vs"])
    row = 0
    for i, (shared, ctxs) in enumerate(groups):
        first = row
        for c in ctxs:
            if len(groups) < 10 or i % 37 < 2:
                n = min(shared, c)
                parts = zip(oracle.page_rows(st, st["tables"][first], n), (x[:, n:] for x in oracle.page_rows(st, st["tables"][row], c)))
                want, bound, _, _ = oracle.decode_row(q[row], *(torch.cat(x, 1) for x in parts), SCALE, fp8)
                within(out[row], want, bound, f"row {row}")
            row += 1


# ---- what is not a number ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
def test_a_query_that_is_not_a_number_has_no_result_that_is_one(fp8, wide):
    """One head of some rows, of one token and of many, behind a shared prefix and alone; the other heads and rows are as without it."""
    st = shared_batch(109, [(100, [133, 101, 117]), (0, [33, 1, 0, 2000])], 2, fp8)
    if wide:
        widen(st)
    q = torch.randn(7, 12, 128, generator=gen(109), device=DEV).to(torch.bfloat16)
    bad = q.clone()
    rows, heads = [0, 3, 4, 5, 6], [0, 5, 7, 8, 11]
    bad[rows, heads, 17] = float("nan")
    kw = {"k_scale": st["ks"], "v_scale": st["vs"]}
    args = (st["k"], st["v"], st["tables"], st["context"])
    good, out = (ops.paged_decode_shared(x, *args, st["cu"], st["shared"], **kw) for x in (q, bad))
    for r, h in zip(rows, heads):
        want = torch.zeros_like if r == 5 else lambda x: torch.full_like(x, float("nan"))           # (row 5 sees nothing)
        assert torch.equal(out[r, h].isnan(), want(out[r, h]).isnan()), (r, h)
        good[r, h] = out[r, h] = 0
    assert torch.equal(good, out)
    alone = [3, 4, 5, 6]                                                      # (the others' own pages do not hold what they share)
    args = (st["k"], st["v"], st["tables"][alone].contiguous(), st["context"][alone].contiguous())
    (good, sums), (out, spoilt) = (ops.paged_decode_scored(x[alone].contiguous(), *args, torch.zeros(4, 2, 2000, device=DEV), **kw) for x in (q, bad))
    for r, h in zip(range(4), heads[1:]):
        n = int(st["context"][alone[r]])
        assert out[r, h].isnan().all() or n == 0
        assert spoilt[r, h // 6, :n].isnan().all() and torch.equal(spoilt[r, 1 - h // 6], sums[r, 1 - h // 6]) and (spoilt[r, :, n:] == 0).all()
        good[r, h] = out[r, h] = 0
    assert torch.equal(good, out)


# ---- small values --------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("amax", [1e-2, 1e-6, 3e4])
@pytest.mark.parametrize("rows,shared", [(100, 0), (300, 0), (40, 1500)])
def test_tails_of_small_weights_over_fp8_values(rows, shared, amax):
    """A key in 97 has all the weight and a value of 0; the others' weights are 6e-6 of it, and the result is their sum.  Few and many rows, and a shared prefix."""
    n, kv, heads, group = 1570, 2, 12, 6
    pages = (n + 15) // 16
    k, v = torch.zeros(pages, kv, 16, 128, device=DEV), torch.rand(pages, kv, 16, 128, generator=gen(110), device=DEV) * amax
    at = torch.arange(5, n, 97, device=DEV)
    k[at // 16, :, at % 16], v[at // 16, :, at % 16] = 1.0, 0.0
    vs = (v.amax(-1) / 448.0).clamp_(min=amax / 448.0)
    st = {"k": (k * 448.0).to(torch.float8_e4m3fn).view(torch.uint8), "ks": torch.full((pages, kv, 16), 1.0 / 448.0, device=DEV), "vs": vs,
          "v": (v / vs[..., None]).to(torch.float8_e4m3fn).transpose(2, 3).contiguous().view(torch.uint8)}
    table = torch.arange(pages, dtype=torch.int32, device=DEV)
    st["tables"], st["context"] = table.expand(rows, -1).contiguous(), torch.tensor([n - i % 60 for i in range(rows)], dtype=torch.int32, device=DEV)
    if shared:
        widen(st)
    # a key's score: 12.02 = -log(6e-6) above the others'
    q = torch.full((rows, heads, 128), 12.02 * math.sqrt(128) / 128, device=DEV).to(torch.bfloat16)
    kw = {"k_scale": st["ks"], "v_scale": st["vs"]}
    cu, lens = offsets([rows]), torch.tensor([shared], dtype=torch.int32, device=DEV)
    args = (q, st["k"], st["v"], st["tables"], st["context"])
    outs = [ops.paged_decode_shared(*args, cu, lens, **kw), ops.paged_decode_scored(*args, torch.zeros(rows, kv, n, device=DEV), **kw)[0]]
    for r in range(0, rows, 13):
        c = int(st["context"][r])
        keys, values = oracle.page_rows(st, table, c)
        p = torch.softmax(q[r].double().view(kv, group, 128) @ keys.transpose(1, 2) * SCALE, -1)
        want = (p @ values).flatten(0, 1)
        # weights in f16: 2^-11 of each, and of the largest value 2^-37 for one that is denormal beside the run's largest; a score of 12 in float32
        bound = (oracle.F16 + oracle.F32) * (p @ values.abs()).flatten(0, 1) + c * 2.0 ** -37 * values.abs().max() * p.max()
        for out in outs:
            within(out[r], want, bound, f"row {r}")


# ---- a bounded cache's prefill -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("budget", [1, 100, 250, 32768])
def test_a_bounded_cache_computes_every_prompt_once(budget):
    """... however many samples it has, in however many chunks the prompts are computed; and chunks are no smaller for the samples"""
    from tests.test_groups_paths_gpu import PAD, _engine, _prompts
    eng, prompts, chunks = _engine(), _prompts((40, 65, 18, 33, 90, 7)), []
    whole = eng.generate(prompts, 8, 0.9, 0.95, 16, None, PAD, 3, kv_budget=30)
    prefill, tokens = eng._prefill, sum(map(len, prompts))
    assert eng.stats["prefill_tokens"] == tokens
    eng.prefill_token_budget = budget
    eng._prefill = lambda sched, groups, *a: (chunks.append(len(groups)), prefill(sched, groups, *a))[1]
    out = eng.generate(prompts, 8, 0.9, 0.95, 16, None, PAD, 3, kv_budget=30)
    assert eng.stats["prefill_tokens"] == 2 * tokens
    assert chunks == {1: [8] * 6, 100: [16, 24, 8], 250: [48], 32768: [48]}[budget]
    assert torch.equal(out[:, 0], whole[:, 0])


@pytest.mark.parametrize("algo", ["grpo", "ppo"])
def test_trainers_look_at_heads_when_they_are_built(algo, tmp_path, monkeypatch):
    from nanorlhf_b200.models.qwen2 import Qwen2Config
    from nanorlhf_b200.trainer import GRPOTrainer, PPOTrainer
    from tests.test_trainers_gpu import _setup
    cls, extra = (PPOTrainer, {"policy_learning_rate": 1e-4, "value_learning_rate": 2e-4}) if algo == "ppo" else (GRPOTrainer, {"grpo_sample_N": 4})
    _setup(tmp_path, cls, extra, share_prompts=True)
    monkeypatch.setattr(Qwen2Config, "__post_init__", lambda self: setattr(self, "head_dim", 64), raising=False)
    _setup(tmp_path, cls, extra)
    with pytest.raises(ValueError, match="share_prompts"):
        _setup(tmp_path, cls, extra, share_prompts=True)


def test_expanded_scores():
    from test_groups_edges_cpu import expanded_scores_are_refused
    expanded_scores_are_refused(DEV)


def test_scales_of_packed_attention():
    from test_groups_edges_cpu import scales_of_packed_attention
    scales_of_packed_attention(DEV, torch.bfloat16)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("scale", [0.0, -0.05, 3.0])
def test_scales_of_decode(scale, fp8):
    """there the mask comes behind the scale: none of these is refused"""
    groups = [(40, [50, 41, 77]), (0, [33, 0, 200])]
    st = shared_batch(111, groups, 2, fp8)
    q = torch.randn(6, 12, 128, generator=gen(111), device=DEV).to(torch.bfloat16)
    kw = {"k_scale": st["ks"], "v_scale": st["vs"], "scale": scale}
    args, sums = (st["k"], st["v"], st["tables"], st["context"]), torch.zeros(6, 2, 200, device=DEV)
    shared, scored = ops.paged_decode_shared(q, *args, st["cu"], st["shared"], **kw), ops.paged_decode_scored(q, *args, sums, **kw)[0]
    row = 0
    for n_shared, ctxs in groups:
        first = row
        for c in ctxs:
            n = min(n_shared, c)
            parts = zip(oracle.page_rows(st, st["tables"][first], n), (x[:, n:] for x in oracle.page_rows(st, st["tables"][row], c)))
            keys, values = (torch.cat(x, 1) for x in parts)
            want, bound, w, _ = oracle.decode_row(q[row], keys, values, scale, fp8)
            # scores up to 3 * 60 * sqrt(128) are off by 2^-24 of what they sum, 128 * 2^-24 at the worst, and so are their exponentials
            worst = 0.0 if c == 0 else (q[row].double().abs().view(2, 6, 128) @ keys.abs().transpose(1, 2)).amax() * abs(scale) * 128 * 2.0 ** -24
            bound = bound + (0.0 if c == 0 else worst * values.abs().amax())
            within(shared[row], want, bound, f"row {row}")
            if n_shared == 0:
                within(scored[row], want, bound, f"scored row {row}")
            row += 1


@pytest.mark.parametrize("wide", [False, True])
def test_tables_of_shared_pages(wide):
    from test_groups_edges_cpu import tables_of_shared_pages
    tables_of_shared_pages(DEV, wide)
