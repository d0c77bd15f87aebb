"""Attention over shared prefixes, decode attention over pages with scores and eviction: the CPU forms against float64, and what the calls refuse."""
import math

import pytest
import torch

import groups_oracle as oracle
from nanorlhf_b200 import ops

SCALE = 1.0 / math.sqrt(128)


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


def packed(groups, heads, kv, dim=128, dtype=torch.float32, spare=0):
    g = torch.Generator().manual_seed(1)
    T = sum(map(sum, groups)) + spare
    q, k, v, dout = (torch.randn(T, h, dim, generator=g).to(dtype) for h in (heads, kv, kv, heads))
    lens = [n for x in groups for n in x]
    return q, k, v, dout, ints(0, *torch.tensor(lens).cumsum(0).tolist()), ints(0, *torch.tensor([len(x) for x in groups]).cumsum(0).tolist())


@pytest.mark.parametrize("groups", [[[3, 4, 1]], [[0, 5, 0], [2]], [[20, 1], [0], [7, 3, 3, 3]]])
def test_shared_prefix(groups):
    q, k, v, dout, cu, cg = packed(groups, 4, 2, spare=2)
    want = oracle.packed(q, k, v, groups, SCALE, dout)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = ops.attention_shared_prefix(*leaves, cu, cg)
    # float32: a score of 128 products and its exponential, 2^-16 of each term
    for x, n in zip((out, *torch.autograd.grad(out, leaves, dout)), ("out", "dq", "dk", "dv")):
        assert (x.double() - want[n][0]).abs().max() < 1e-4 and torch.equal(x[-2:], torch.zeros_like(x[-2:])), n


def test_a_prefix_in_front_of_every_sample():
    """The same as whole sequences without sharing."""
    P, lens = 9, [4, 1, 6]
    q, k, v, _, cu, cg = packed([[P] + lens], 4, 2)
    out = ops.attention_shared_prefix(q, k, v, cu, cg)
    at = P
    for n in lens:
        rows = torch.cat([torch.arange(P), torch.arange(at, at + n)])
        whole = ops.attention_varlen(q[rows], k[rows], v[rows], ints(0, P + n))
        assert torch.allclose(out[at:at + n], whole[P:], atol=1e-5) and torch.allclose(out[:P], whole[:P], atol=1e-5)
        at += n


def pool(blocks=12, kv=2, fp8=False):
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(blocks, kv, 16, 128, generator=g) for _ in range(2))
    if not fp8:
        return {"k": k.to(torch.bfloat16), "v": v.to(torch.bfloat16), "ks": None, "vs": None}
    ks, vs = k.abs().amax(-1) / 448.0, v.abs().amax(-1) / 448.0
    return {"k": (k / ks[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), "ks": ks, "vs": vs,
            "v": (v / vs[..., None]).to(torch.float8_e4m3fn).transpose(2, 3).contiguous().view(torch.uint8)}


@pytest.mark.parametrize("fp8", [False, True])
def test_decode_over_shared_pages(fp8):
    st = pool(fp8=fp8)
    tables, context, cu, shared = torch.tensor([[0, 1, 2], [0, 1, 3], [0, 4, 5], [6, 7, 8]], dtype=torch.int32), ints(40, 33, 5, 17), ints(0, 3, 4), ints(32, 0)
    q = torch.randn(4, 12, 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    out = ops.paged_decode_shared(q, st["k"], st["v"], tables, context, cu, shared, k_scale=st["ks"], v_scale=st["vs"])
    for r, n in enumerate(context.tolist()):
        common = min(n, 32) if r < 3 else 0
        parts = zip(oracle.page_rows(st, tables[0], common), (x[:, common:] for x in oracle.page_rows(st, tables[r], n)))
        want = oracle.decode_row(q[r], *(torch.cat(x, 1) for x in parts), SCALE, fp8)[0]
        assert ((out[r].double() - want).abs() <= oracle.BF16 * want.abs() + 1e-4).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_decode_with_scores(fp8):
    st = pool(fp8=fp8)
    tables, context = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32), ints(40, 0)
    q = torch.randn(2, 4, 128, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    scores = torch.rand(2, 2, 45)
    before = scores.clone()
    out, new = ops.paged_decode_scored(q, st["k"], st["v"], tables, context, scores, 0.5, st["ks"], st["vs"])
    want, _, w, _ = oracle.decode_row(q[0], *oracle.page_rows(st, tables[0], 40), SCALE, fp8)
    assert new is scores and torch.equal(scores[:, :, 40:], before[:, :, 40:]) and torch.equal(scores[1], before[1]) and (out[1] == 0).all()
    assert ((out[0].double() - want).abs() <= oracle.BF16 * want.abs() + 1e-4).all()
    old = 0.5 * before[0, :, :39].double()
    assert (scores[0, :, :40].double() - torch.cat([old + w[:, :39], w[:, 39:]], 1)).abs().max() < 1e-5


@pytest.mark.parametrize("fp8", [False, True])
def test_evict(fp8):
    st = pool(fp8=fp8)
    tables, context = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32), ints(40, 6)
    scores = torch.rand(2, 2, 48)
    scores[0, 0, 7], scores[0, 0, 8:12], scores[0, 1] = float("nan"), 2.0, 0.0
    before = {n: None if st[n] is None else st[n].clone() for n in st}
    kept, kept_scores, lens = ops.kv_evict(st["k"], st["v"], tables, context, scores, 10, 2, 3, st["ks"], st["vs"])
    assert lens.tolist() == [10, 6] and kept[1].tolist() == [[0, 1, 2, 3, 4, 5, -1, -1, -1, -1]] * 2
    assert kept[0, 1].tolist() == [0, 1, 2, 3, 4, 5, 6, 37, 38, 39]                    # all alike: the first
    assert {8, 9, 10, 11} <= set(kept[0, 0].tolist()) and 7 not in kept[0, 0].tolist()
    rows = lambda s, h, t: [x[h, t] for x in oracle.page_rows(s, tables[0], 40)]  # noqa: E731
    for h in range(2):
        for j, t in enumerate(kept[0, h].tolist()):
            assert all(torch.equal(a, b) for a, b in zip(rows(st, h, j), rows(before, h, t))) and (kept_scores[0, h, j] == scores[0, h, t])
    assert all(torch.equal(a, b) for a, b in zip(oracle.page_rows(st, tables[1], 6), oracle.page_rows(before, tables[1], 6)))


def test_evict_into_other_pages_leaves_its_sources():
    st = pool()
    tables, to = torch.tensor([[0, 1, 2]], dtype=torch.int32), torch.tensor([[9]], dtype=torch.int32)
    before = st["k"].clone()
    kept, _, _ = ops.kv_evict(st["k"], st["v"], tables, ints(40), torch.rand(1, 2, 40), 8, out_tables=to)
    assert torch.equal(st["k"][:9], before[:9]) and torch.equal(st["k"][9, :, 8:], before[9, :, 8:])
    for h in range(2):
        t = kept[0, h].long()
        assert torch.equal(st["k"][9, h, :8], before[t // 16, h, t % 16])


def test_refusals():
    q, k, v, _, cu, cg = packed([[3, 4]], 4, 2)
    f = ops.attention_shared_prefix
    for bad in ((q[:, :3], k, v, cu, cg), (q, k[:-1], v[:-1], cu, cg), (q, k, v[:, :1], cu, cg), (q[0], k, v, cu, cg), (q, k, v, cu[None], cg), (q, k, v, cu, cg[:0])):
        with pytest.raises(ValueError):
            f(*bad)
    with pytest.raises(ValueError):
        f(q, k, v, cu, cg, scale=float("nan"))
    for bad in ((q.double(), k, v, cu, cg), (q, k, v, cu.long(), cg), (q, k, v, cu, cg.float())):
        with pytest.raises(TypeError):
            f(*bad)
    st, st8 = pool(), pool(fp8=True)
    tables, context, scores = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32), ints(40, 6), torch.rand(2, 2, 48)
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    groups = (ints(0, 2), ints(16))
    calls = {"shared": lambda q=q, k=st["k"], v=st["v"], t=tables, c=context, g=groups, **kw: ops.paged_decode_shared(q, k, v, t, c, *g, **kw),
             "scored": lambda q=q, k=st["k"], v=st["v"], t=tables, c=context, s=scores, **kw: ops.paged_decode_scored(q, k, v, t, c, s, **kw),
             "evict": lambda k=st["k"], v=st["v"], t=tables, c=context, s=scores, keep=10, **kw: ops.kv_evict(k, v, t, c, s, keep, **kw)}
    for call in calls.values():
        call()
        for kw in ({"k": st["k"][..., :8, :]}, {"v": st["v"][:3]}, {"t": tables[:1]}, {"t": tables[0]}, {"c": context[None]}, {"k_scale": st8["ks"]},
                   {"k": st8["k"], "v": st8["v"], "k_scale": st8["ks"][:3], "v_scale": st8["vs"]}):
            with pytest.raises(ValueError):
                call(**kw)
        for kw in ({"k": st8["k"], "v": st8["v"]}, {"k_scale": st8["ks"], "v_scale": st8["vs"]}, {"t": tables.long()}, {"c": context.float()}):
            with pytest.raises(TypeError):
                call(**kw)
    for name in ("shared", "scored"):
        for kw in ({"q": q[:1]}, {"q": q[:, :3]}, {"q": q[..., :64]}, {"q": torch.zeros(2, 18, 128)}, {"scale": math.inf}):
            with pytest.raises(ValueError):
                calls[name](**kw)
    for kw in ({"g": (ints(0, 1, 2), ints(16))}, {"max_group": 0}):
        with pytest.raises(ValueError):
            calls["shared"](**kw)
    with pytest.raises(TypeError):
        calls["shared"](g=(torch.tensor([0, 2]), ints(16)))
    for kw in ({"s": scores[:1]}, {"s": scores[:, :1]}, {"s": scores[0]}, {"decay": math.nan}, {"out_scores": scores[..., :47]}):
        with pytest.raises(ValueError):
            calls["scored"](**kw)
    for name in ("scored", "evict"):
        for s in (scores.double(), scores.transpose(1, 2).contiguous().transpose(1, 2)):
            with pytest.raises(TypeError):
                calls[name](s=s)
    for kw in ({"keep": 0}, {"keep": 3.5}, {"sinks": -1}, {"recent": 11}, {"sinks": 6, "recent": 5}, {"out_tables": tables[:1]}, {"out_tables": tables[0]},
               {"keep": 40, "out_tables": tables[:, :2]}):
        with pytest.raises(ValueError):
            calls["evict"](**kw)
    with pytest.raises(TypeError):
        calls["evict"](out_tables=tables.long())
