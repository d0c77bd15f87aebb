"""Attention over shared prefixes, decode attention over pages with scores and eviction: the CPU forms against float64, and what the calls refuse."""
import math

import pytest
import torch

import groups_oracle as oracle
from groups_refusals import ints, packed, pool, refused_calls
from nanorlhf_b200 import ops

SCALE = 1.0 / math.sqrt(128)


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
    refused_calls("cpu")
