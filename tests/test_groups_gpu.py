"""Attention over shared prefixes, decode attention over shared pages and with scores, eviction: against float64 and against plain loops."""
import math

import pytest
import torch

import groups_oracle as oracle
from groups_refusals import refused_calls
from nanorlhf_b200 import ops
from nanorlhf_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 1.0 / math.sqrt(128)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def offsets(lens):
    return torch.tensor([0] + lens, dtype=torch.int32, device=DEV).cumsum(0).int()


def within(got, want, bound, what, rounded=oracle.BF16):
    """|got - want| <= bound + the result's own rounding"""
    off = (got.double() - want).abs() - bound - rounded * want.abs() - 1e-30
    assert torch.isfinite(got).all(), what
    assert off.max().item() <= 0, f"{what}: {off.max().item()} beyond its bound at {off.argmax().item()}"


def test_refusals():
    refused_calls(DEV)
    q = torch.zeros(4, 2, 128, device=DEV)
    cu = torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    with pytest.raises(TypeError):
        ops.attention_shared_prefix(q, q, q, cu, cu)                                        # float32
    with pytest.raises(TypeError):
        ops.attention_shared_prefix(*(q[..., :64].to(torch.bfloat16),) * 3, cu, cu)         # another head size


# ---- packed groups -------------------------------------------------------------------------------------------------------------------------
GROUPS = {
    "one token each": [[1, 1, 1]],
    "empty prefix, empty samples": [[0, 5, 0, 130], [17, 0], [0]],
    "around a tile": [[127, 128, 129], [128, 127], [129, 1, 256]],
    "around two tiles": [[255, 257, 1], [256, 64, 65], [257, 3]],
    "long prefix, short samples": [[1100, 7, 1, 33, 64]],
    "short prefix, long samples": [[3, 700, 513]],
    "many": [[40 + i, 10 * i % 97, 31] for i in range(40)],
}


def packed_inputs(groups, heads, kv, seed, spare=0):
    g = gen(seed)
    T = sum(map(sum, groups)) + spare
    qkv = torch.randn(T, (heads + 2 * kv), 128, generator=g, device=DEV).to(torch.bfloat16)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]           # views of a projection
    dout = torch.randn(T, heads, 128, generator=g, device=DEV).to(torch.bfloat16)
    return q, k, v, dout, offsets([n for x in groups for n in x]), offsets([len(x) for x in groups])


@pytest.mark.parametrize("heads,kv", [(6, 1), (8, 8), (4, 2)])
@pytest.mark.parametrize("name", list(GROUPS))
def test_shared_prefix(name, heads, kv):
    groups = GROUPS[name]
    q, k, v, dout, cu, cg = packed_inputs(groups, heads, kv, 1)
    want = oracle.packed(q, k, v, groups, SCALE, dout)
    with torch.no_grad():
        plain = ops.attention_shared_prefix(q, k, v, cu, cg)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = ops.attention_shared_prefix(*leaves, cu, cg, max(map(max, groups)))
    assert torch.equal(out, plain)
    grads = torch.autograd.grad(out, leaves, dout)
    within(out, *want["out"], "out")
    for x, n in zip(grads, ("dq", "dk", "dv")):
        within(x, *want[n], n)


def test_shared_prefix_repeats_to_the_bit():
    q, k, v, dout, cu, cg = packed_inputs(GROUPS["many"], 12, 2, 2)
    def once():
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = ops.attention_shared_prefix(*leaves, cu, cg)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))
    for a, b in zip(once(), once()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("grouped", [True, False])
def test_groups_of_one_are_plain_sequences(grouped):
    """Sequences alone in their group, or in none: the results of attention_varlen and the values' gradients to the bit.  Its other gradients go by the rounded result."""
    lens = [5, 300, 0, 128, 700]
    q, k, v, dout, cu, cg = packed_inputs([[n] for n in lens], 12, 2, 3)
    if not grouped:
        cg = cg[:1].clone()
    results, want = [], oracle.packed(q, k, v, [[n] for n in lens], SCALE, dout)
    for f in (lambda *a: ops.attention_shared_prefix(*a, cu, cg), lambda *a: ops.attention_varlen(*a, cu, 700)):
        leaves = [x.detach().contiguous().requires_grad_() for x in (q, k, v)]
        out = f(*leaves)
        results.append((out.detach(), *torch.autograd.grad(out, leaves, dout)))
    (out, dq, dk, dv), plain = results
    assert torch.equal(out, plain[0]) and torch.equal(dv, plain[3])
    within(dq, *want["dq"], "dq")
    within(dk, *want["dk"], "dk")


def test_rows_behind_the_last_sequence_are_zero():
    groups = [[33, 20, 70], [5]]
    q, k, v, dout, cu, cg = packed_inputs(groups, 4, 1, 4, spare=140)
    want = oracle.packed(q, k, v, groups, SCALE, dout)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    junk = torch.full((50, 1024, 128), float("nan"), device=DEV)             # what the allocator hands out next is not zero
    del junk
    out = ops.attention_shared_prefix(*leaves, cu, cg)
    grads = torch.autograd.grad(out, leaves, dout)
    within(out, *want["out"], "out")
    for x, n in zip(grads, ("dq", "dk", "dv")):
        within(x, *want[n], n)


def test_shared_prefix_gradient_is_the_difference_quotient():
    """d out . w along a direction, against out at two points: bf16 results are rounded to 2^-8, the step is 2^-2 of unit vectors, so that what it moves is well above."""
    groups = [[70, 33, 140]]
    q, k, v, dout, cu, cg = packed_inputs(groups, 4, 2, 5)
    leaves = [x.float().to(torch.bfloat16).requires_grad_() for x in (q, k, v)]
    out = ops.attention_shared_prefix(*leaves, cu, cg)
    grads = torch.autograd.grad(out, leaves, dout)
    for i in range(3):
        d = torch.randn(leaves[i].shape, generator=gen(6 + i), device=DEV)
        h = 0.25 * d / d.norm() * math.sqrt(leaves[i].shape[0])
        at = lambda s: [x.detach().double() + (s * h if j == i else 0) for j, x in enumerate(leaves)]  # noqa: E731
        f = lambda s: (oracle.packed(*at(s), groups, SCALE)["out"][0] * dout.double()).sum()  # noqa: E731
        quotient = (f(0.01) - f(-0.01)).item() / 0.02
        mine, bound = (grads[i].double() * h).sum().item(), (oracle.packed(*at(0), groups, SCALE, dout)[("dq", "dk", "dv")[i]][1] * h.abs()).sum().item()
        # the bound of the sum, the gradient's own roundings, and the third derivative's part, which is below 1e-4 of the terms at a step of 0.01
        assert abs(mine - quotient) <= bound + ((oracle.BF16 + 1e-4) * (grads[i].double().abs() * h.abs()).sum().item())


def test_shared_prefix_in_a_graph_and_on_another_stream():
    groups = [[150, 40, 300], [64, 1]]
    q, k, v, dout, cu, cg = packed_inputs(groups, 12, 2, 7)
    leaves = [x.detach().contiguous().requires_grad_() for x in (q, k, v)]
    def step():
        out = ops.attention_shared_prefix(*leaves, cu, cg)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    q2, k2, v2, *_ = packed_inputs(groups, 12, 2, 8)
    with torch.no_grad():
        for x, y in zip(leaves, (q2, k2, v2)):
            x.copy_(y)
    graph.replay()
    want = oracle.packed(q2, k2, v2, groups, SCALE, dout)
    for x, n in zip(got, ("out", "dq", "dk", "dv")):
        within(x, *want[n], n)


def test_shared_prefix_second_derivative_is_refused():
    q, k, v, dout, cu, cg = packed_inputs([[4, 4]], 2, 1, 9)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    (dq,) = torch.autograd.grad(ops.attention_shared_prefix(*leaves, cu, cg), leaves[:1], dout, create_graph=True)
    with pytest.raises(RuntimeError):
        dq.float().sum().backward()


def test_shared_prefix_of_nothing():
    q, k, v = (torch.empty(0, h, 128, dtype=torch.bfloat16, device=DEV) for h in (4, 2, 2))
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert ops.attention_shared_prefix(q, k, v, zero, zero).shape == (0, 4, 128)


# ---- pages ---------------------------------------------------------------------------------------------------------------------------------
def pages_of(seed, blocks, kv, fp8, poison=True):
    """A pool of NaN (bytes and scales too); `fill` puts tokens there."""
    if not fp8:
        return {"k": torch.full((blocks, kv, 16, 128), float("nan"), dtype=torch.bfloat16, device=DEV), "ks": None, "vs": None,
                "v": torch.full((blocks, kv, 16, 128), float("nan"), dtype=torch.bfloat16, device=DEV)}
    nan = lambda *s: torch.full(s, float("nan"), device=DEV)  # noqa: E731
    return {"k": torch.full((blocks, kv, 16, 128), 0x7F, dtype=torch.uint8, device=DEV), "v": torch.full((blocks, kv, 128, 16), 0x7F, dtype=torch.uint8, device=DEV),
            "ks": nan(blocks, kv, 16), "vs": nan(blocks, kv, 16)}


def fill(st, g, table, lo, hi):
    """random keys and values for tokens [lo, hi) of a page table (a list)"""
    if hi <= lo:
        return
    t = torch.arange(lo, hi, device=DEV)
    page, off = torch.tensor(table, device=DEV)[t // 16], t % 16
    kv = st["k"].shape[1]
    k, v = (torch.randn(hi - lo, kv, 128, generator=g, device=DEV) for _ in range(2))
    if st["ks"] is None:
        st["k"][page, :, off], st["v"][page, :, off] = k.to(torch.bfloat16), v.to(torch.bfloat16)
        return
    ks, vs = k.abs().amax(-1) / 448.0, v.abs().amax(-1) / 448.0
    st["k"].view(torch.float8_e4m3fn)[page, :, off] = (k / ks[..., None]).to(torch.float8_e4m3fn)
    st["v"].view(torch.float8_e4m3fn)[page, :, :, off] = (v / vs[..., None]).to(torch.float8_e4m3fn)
    st["ks"][page, :, off], st["vs"][page, :, off] = ks, vs


def shared_batch(seed, groups, kv, fp8):
    """groups: [(shared tokens, [context, ...])].  Places of no token are NaN, and so are the copies of shared tokens in other rows' pages than the first's."""
    g, rows, blocks = gen(seed), [], 0
    for shared, ctxs in groups:
        whole = list(range(blocks, blocks + shared // 16))
        blocks += len(whole)
        for c in ctxs:
            n = max(0, (max(c, shared) + 15) // 16 - len(whole))
            rows.append(whole + list(range(blocks, blocks + n)))
            blocks += n
    width = max(1, max(map(len, rows)))
    st = pages_of(seed, blocks + 1, kv, fp8)
    i = 0
    for shared, ctxs in groups:
        for j, c in enumerate(ctxs):
            if j == 0:
                fill(st, g, rows[i], 0, shared)
            fill(st, g, rows[i], shared, c)
            i += 1
    st["tables"] = torch.tensor([r + [blocks] * (width - len(r)) for r in rows], dtype=torch.int32, device=DEV)
    st["context"] = torch.tensor([c for _, cs in groups for c in cs], dtype=torch.int32, device=DEV)
    st["cu"], st["shared"] = offsets([len(cs) for _, cs in groups]), torch.tensor([s for s, _ in groups], dtype=torch.int32, device=DEV)
    return st


BATCHES = {
    "a few": [(100, [133, 101, 117, 100])],
    "nothing shared": [(0, [1, 17, 0, 160]), (0, [33])],
    "inside pages": [(15, [16, 15, 40]), (17, [17, 33, 200]), (1, [1, 2])],
    "shorter than the prefix": [(70, [200, 0, 1, 64, 70, 71])],
    "many rows": [(333, [340 + 7 * i for i in range(37)]), (16, [16 + i for i in range(9)]), (64, [500])],
    "long": [(2500, [2600, 2501, 4000]), (64, [70, 65])],
}


def widen(st):
    """Page tables of 110 MB of pages and more: prefixes are attended to for all rows of a group, instead of by each row."""
    S, width = st["tables"].shape
    more = 110_000_000 // (S * st["k"].shape[1] * 4096) + 1
    st["tables"] = torch.cat([st["tables"], torch.full((S, more), st["k"].shape[0] - 1, dtype=torch.int32, device=DEV)], 1)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,kv", [(12, 2), (7, 1), (16, 2), (4, 4)])
@pytest.mark.parametrize("name", list(BATCHES))
def test_decode_over_shared_pages(name, heads, kv, fp8, wide):
    groups = BATCHES[name]
    st = shared_batch(11, groups, kv, fp8)
    if wide:
        widen(st)
    S = st["context"].numel()
    q = torch.randn(S, heads + 3, 128, generator=gen(12), device=DEV).to(torch.bfloat16)[:, :heads]
    kw = {"k_scale": st["ks"], "v_scale": st["vs"]}
    largest = max(len(c) for _, c in groups)
    outs = [ops.paged_decode_shared(q, st["k"], st["v"], st["tables"], st["context"], st["cu"], st["shared"], max_group=m, **kw)
            for m in (largest, None, 1)]
    row = 0
    for shared, ctxs in groups:
        first = row
        for c in ctxs:
            n = min(shared, c)
            parts = zip(oracle.page_rows(st, st["tables"][first], n), (x[:, n:] for x in oracle.page_rows(st, st["tables"][row], c)))
            want, bound, _, _ = oracle.decode_row(q[row], *(torch.cat(x, 1) for x in parts), SCALE, fp8)
            for out in outs:
                within(out[row], want, bound, f"row {row}")
            row += 1


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
def test_rows_of_no_group_are_plain(fp8, wide):
    """... and so are those of groups that do not follow one another."""
    st = shared_batch(13, [(48, [100, 77]), (0, [130, 5, 64])], 2, fp8)
    if wide:
        widen(st)
    q = torch.randn(5, 12, 128, generator=gen(14), device=DEV).to(torch.bfloat16)
    args = (q, st["k"], st["v"], st["tables"], st["context"])
    a = ops.paged_decode_shared(*args, st["cu"][:2].contiguous(), st["shared"][:1].contiguous(), max_group=2, k_scale=st["ks"], v_scale=st["vs"])
    b = ops.paged_decode_shared(*args, st["cu"], st["shared"], max_group=3, k_scale=st["ks"], v_scale=st["vs"])
    assert torch.equal(a[2:], b[2:])
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    c = ops.paged_decode_shared(*args, none, none[:0], k_scale=st["ks"], v_scale=st["vs"])
    d = ops.paged_decode_shared(*args, torch.tensor([-3, 7, 2], dtype=torch.int32, device=DEV), torch.tensor([48, 48], dtype=torch.int32, device=DEV), k_scale=st["ks"],
                                v_scale=st["vs"])
    assert torch.equal(a[2:], c[2:]) and torch.equal(c, d)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
def test_many_groups_and_long_prefixes(fp8, wide):
    """More groups and rows than decode_plan has threads, runs that meet several tiles, groups of more than one tile of query rows."""
    few = [(300 + 16 * i, [320 + 16 * i + j for j in range(33)]) for i in range(3)] + [(1500, [1501 + j for j in range(70)])]
    many = [(16 * (i % 5), [16 * (i % 5) + 1 + i % 3] * (1 + i % 2)) for i in range(1100)]
    for seed, groups in ((70, few), (71, many)):
        st = shared_batch(seed, groups, 2, fp8)
        if wide:
            widen(st)
        S = st["context"].numel()
        q = torch.randn(S, 12, 128, generator=gen(seed), device=DEV).to(torch.bfloat16)
        out = ops.paged_decode_shared(q, st["k"], st["v"], st["tables"], st["context"], st["cu"], st["shared"], max_group=70, k_scale=st["ks"], v_scale=st["vs"])
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


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("rows", [127, 128, 129])
def test_around_the_rows_for_which_every_block_plans(rows, fp8):
    groups = [(33, [34 + i % 40 for i in range(rows - 60)]), (0, [i % 5 for i in range(20)]), (100, [90 + i for i in range(40)])]
    st = shared_batch(75, groups, 2, fp8)
    q = torch.randn(rows, 12, 128, generator=gen(75), device=DEV).to(torch.bfloat16)
    out = ops.paged_decode_shared(q, st["k"], st["v"], st["tables"], st["context"], st["cu"], st["shared"], k_scale=st["ks"], v_scale=st["vs"])
    row = 0
    for shared, ctxs in groups:
        first = row
        for c in ctxs:
            n = min(shared, c)
            parts = zip(oracle.page_rows(st, st["tables"][first], n), (x[:, n:] for x in oracle.page_rows(st, st["tables"][row], c)))
            want, bound, _, _ = oracle.decode_row(q[row], *(torch.cat(x, 1) for x in parts), SCALE, fp8)
            within(out[row], want, bound, f"row {row}")
            row += 1


@pytest.mark.parametrize("fp8", [False, True])
def test_decode_over_shared_pages_in_two_graphs(fp8):
    """Two captured calls of other batches, replayed in turn and with other inputs."""
    calls = []
    for seed, name in ((15, "a few"), (16, "many rows"), (19, "long")):
        st = shared_batch(seed, BATCHES[name], 2, fp8)
        if seed > 15:
            widen(st)
        q = torch.randn(st["context"].numel(), 12, 128, generator=gen(seed), device=DEV).to(torch.bfloat16)
        f = lambda st=st, q=q: ops.paged_decode_shared(q, st["k"], st["v"], st["tables"], st["context"], st["cu"], st["shared"], max_group=37, k_scale=st["ks"],  # noqa: E731
                                                       v_scale=st["vs"])
        f()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        calls.append((graph, f, out, q))
    for seed in (17, 18):
        for _, _, _, q in calls:
            q.copy_(torch.randn(q.shape, generator=gen(seed), device=DEV))
        for graph, *_ in calls:
            graph.replay()
        for _, f, out, _ in calls:
            assert torch.equal(out, f())


# ---- scores ----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,kv", [(12, 2), (7, 1), (16, 2), (4, 4)])
@pytest.mark.parametrize("contexts", [[1], [0, 1, 2, 16, 17], [129, 33, 77], [600 + 13 * i for i in range(50)], [5000, 64], [7 * i % 90 for i in range(129)]],
                         ids=lambda c: f"{len(c)}x{max(c)}")
def test_decode_with_scores(contexts, heads, kv, fp8):
    st = shared_batch(21, [(0, [c]) for c in contexts], kv, fp8)
    S, L = len(contexts), max(contexts) + 3
    q = torch.randn(S, heads, 128, generator=gen(22), device=DEV).to(torch.bfloat16)
    before = torch.rand(kv, S, L, generator=gen(23), device=DEV).transpose(0, 1)              # other strides than a fresh tensor's
    for s, n in enumerate(contexts):
        if n:
            before[s, :, n - 1] = float("nan")                                                  # the newest token's place holds anything
    for decay, in_place in ((1.0, False), (0.75, True)):
        scores = before.clone()
        into = None if in_place else torch.full((S, kv, L), 7.0, device=DEV)
        out, new = ops.paged_decode_scored(q, st["k"], st["v"], st["tables"], st["context"], scores, decay, st["ks"], st["vs"], out_scores=into)
        assert new is (scores if in_place else into)
        for s, n in enumerate(contexts):
            want, bound, w, wb = oracle.decode_row(q[s], *oracle.page_rows(st, st["tables"][s], n), SCALE, fp8)
            within(out[s], want, bound, f"row {s}")
            assert torch.equal(new[s, :, n:], before[s, :, n:] if in_place else torch.full_like(new[s, :, n:], 7.0))
            if n:
                old = decay * before[s, :, :n - 1].double()
                within(new[s, :, :n], torch.cat([old + w[:, :-1], w[:, -1:]], 1), wb, f"scores of row {s}", 2.0 ** -23)


def test_scores_shorter_than_the_context():
    st = shared_batch(24, [(0, [100]), (0, [30])], 2, False)
    q = torch.randn(2, 12, 128, generator=gen(25), device=DEV).to(torch.bfloat16)
    full, part = torch.zeros(2, 2, 100, device=DEV), torch.zeros(2, 2, 41, device=DEV)
    a, _ = ops.paged_decode_scored(q, st["k"], st["v"], st["tables"], st["context"], full)
    b, _ = ops.paged_decode_scored(q, st["k"], st["v"], st["tables"], st["context"], part)
    assert torch.equal(a, b) and torch.equal(full[..., :41], part)


# ---- eviction --------------------------------------------------------------------------------------------------------------------------------
def evict_both(st, scores, keep, sinks, recent, out_tables=None):
    """The kernel's results and pages, and the plain loop's on the host."""
    names = ("k", "v", "ks", "vs")
    host = {n: None if st[n] is None else st[n].cpu().clone() for n in names}
    want = ref.kv_evict(host["k"], host["v"], st["tables"].cpu(), st["context"].cpu(), scores.cpu(), keep, sinks, recent, host["ks"], host["vs"],
                        None if out_tables is None else out_tables.cpu())
    got = ops.kv_evict(st["k"], st["v"], st["tables"], st["context"], scores, keep, sinks, recent, st["ks"], st["vs"], out_tables)
    bits = lambda x: x.cpu().view(torch.int16 if x.dtype == torch.bfloat16 else torch.int32 if x.dtype == torch.float32 else x.dtype)  # noqa: E731
    for a, b, n in zip(got, want, ("kept", "scores", "lens")):
        assert torch.equal(bits(a), bits(b)), n
    for n in names:
        if st[n] is not None:
            assert torch.equal(bits(st[n]), bits(host[n])), n
    return got


def random_scores(seed, S, kv, L):
    x = torch.randn(S, kv, L, generator=gen(seed), device=DEV).mul_(2.0).exp_()
    return torch.where(x < 0.3, 0.0, x)                        # many alike


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("contexts,keep,sinks,recent", [([300], 128, 4, 32), ([1, 0, 2, 17, 16], 1, 0, 0), ([40, 100, 99, 33], 33, 0, 33), ([500, 41, 1000, 700], 40, 40, 0),
                                                        ([3000, 2999, 1024], 1023, 16, 256), ([800] * 20, 777, 1, 0), ([64, 48], 100, 5, 5)])
def test_evict(contexts, keep, sinks, recent, fp8, apart):
    st = shared_batch(31, [(0, [c]) for c in contexts], 2, fp8)
    S, pages = len(contexts), (min(keep, max(contexts)) + 15) // 16
    to = None
    if apart:
        n = st["k"].shape[0]
        for name in ("k", "v", "ks", "vs"):
            if st[name] is not None:
                st[name] = torch.cat([st[name], st[name].new_full((S * pages, *st[name].shape[1:]), 3)])
        to = (n + torch.randperm(S * pages, generator=gen(32), device=DEV).view(S, pages)).int()
    evict_both(st, random_scores(33, S, 2, max(contexts)), keep, sinks, recent, to)


def test_evict_by_odd_scores():
    """NaN, infinities, both zeros, denormals, negatives; strides of a larger tensor."""
    odd = torch.tensor([float("nan"), float("inf"), float("-inf"), 0.0, -0.0, 1e-40, -1e-40, 1.0, -1.0, 3e38, -3e38], device=DEV)
    st = shared_batch(34, [(0, [c]) for c in (300, 301, 50)], 2, False)
    pick = torch.randint(0, odd.numel(), (3, 5, 310), generator=gen(35), device=DEV)
    evict_both(st, odd[pick][:, 1:3], 77, 3, 10)


def test_evict_all_alike_keeps_the_first():
    st = shared_batch(36, [(0, [200])], 1, True)
    kept, _, lens = evict_both(st, torch.zeros(1, 1, 200, device=DEV), 50, 0, 10)
    assert kept[0, 0].tolist() == list(range(40)) + list(range(190, 200)) and lens.tolist() == [50]


@pytest.mark.parametrize("contexts,keep", [([5000, 4200], 700), ([9001], 8000), ([20_011, 7, 12_345], 4097), ([50_001], 4097), ([330_000], 1000)])
def test_evict_by_several_blocks_a_row(contexts, keep):
    """Clusters of two to eight blocks, and more tokens than their shared memory holds; scores that tie across blocks."""
    fp8 = len(contexts) == 2
    st = shared_batch(37, [(0, [c]) for c in contexts], 1, fp8)
    evict_both(st, random_scores(38, len(contexts), 1, max(contexts)), keep, 16, 100)


@pytest.mark.parametrize("keep", [61, 700])
@pytest.mark.parametrize("apart", [False, True])
def test_evict_from_far_apart(apart, keep):
    """What is kept lies many pages apart: values of fp8 pages that wait for a page to be full, over spans without any; and by several blocks a row."""
    n = 4000
    st = shared_batch(39, [(0, [n])], 2, True)
    scores = torch.zeros(1, 2, n, device=DEV)
    scores[0, 0, 5::97], scores[0, 1, [3, 4, 1000, 3990]] = 1.0, 2.0
    to = None
    if apart:
        m = st["k"].shape[0]
        for name in ("k", "v", "ks", "vs"):
            st[name] = torch.cat([st[name], torch.zeros_like(st[name][:44])])
        to = torch.arange(m, m + 44, device=DEV).int()[None]
    evict_both(st, scores, keep, 0, 3, to)


@pytest.mark.parametrize("fp8", [False, True])
def test_decode_score_evict_decode(fp8):
    """As they are used together: decode steps that leave scores, an eviction in place, decode steps over what is left."""
    contexts, keep, steps = [150, 90, 260], 100, 4
    st = shared_batch(41, [(0, [c + 2 * steps]) for c in contexts], 2, fp8)           # the tokens of all steps lie there
    scores = torch.zeros(3, 2, 320, device=DEV)
    mine = torch.zeros(3, 2, 320, dtype=torch.float64, device=DEV)
    ctx, order = list(contexts), None
    full = [oracle.page_rows(st, st["tables"][s], contexts[s] + 2 * steps) for s in range(3)]      # every token by its first place
    place = [[list(range(n)) for _ in range(2)] for n in ctx]                                       # of every place the token there
    for step in range(2 * steps):
        q = torch.randn(3, 12, 128, generator=gen(50 + step), device=DEV).to(torch.bfloat16)
        st["context"] = torch.tensor(ctx, dtype=torch.int32, device=DEV)
        out, _ = ops.paged_decode_scored(q, st["k"], st["v"], st["tables"], st["context"], scores, 1.0, st["ks"], st["vs"])
        for s in range(3):
            keys, values = (torch.stack([x[h, place[s][h]] for h in range(2)]) for x in full[s])
            want, bound, w, _ = oracle.decode_row(q[s], keys, values, SCALE, fp8)
            within(out[s], want, bound, f"step {step}, row {s}")
            n = ctx[s]
            mine[s, :, n - 1] = 0
            mine[s, :, :n] += w
            assert (scores[s, :, :n].double() - mine[s, :, :n]).abs().max() < 1e-4
        if step == steps - 1:
            kept, kept_scores, lens = evict_both(st, scores, keep, 4, 20)
            for s in range(3):
                place[s] = [[place[s][h][t] for t in kept[s, h].tolist() if t >= 0] for h in range(2)]
            scores[:, :, :keep] = kept_scores
            mine[:, :, :keep] = kept_scores.double()
            ctx = lens.tolist()
        # the next token's place behind the last one
        grown = [c + 1 for c in ctx]
        for s in range(3):
            t = contexts[s] + step + 1 - 1
            to, off = int(st["tables"][s, ctx[s] // 16]), ctx[s] % 16
            src, src_off = int(st["tables"][s, t // 16]), t % 16
            if (to, off) != (src, src_off):
                st["k"][to, :, off] = st["k"][src, :, src_off].clone()
                if fp8:
                    st["v"][to, :, :, off] = st["v"][src, :, :, src_off].clone()
                    st["ks"][to, :, off], st["vs"][to, :, off] = st["ks"][src, :, src_off].clone(), st["vs"][src, :, src_off].clone()
                else:
                    st["v"][to, :, off] = st["v"][src, :, src_off].clone()
            for h in range(2):
                place[s][h].append(t)
        ctx = grown


def test_evict_in_a_graph():
    st = shared_batch(61, [(0, [300]), (0, [70])], 2, True)
    n = st["k"].shape[0]
    for name in ("k", "v", "ks", "vs"):
        st[name] = torch.cat([st[name], torch.zeros_like(st[name][:16])])
    to = (n + torch.arange(16, device=DEV).view(2, 8)).int()
    scores = random_scores(62, 2, 2, 300)
    f = lambda: ops.kv_evict(st["k"], st["v"], st["tables"], st["context"], scores, 128, 4, 32, st["ks"], st["vs"], to)  # noqa: E731
    f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept, kept_scores, lens = f()
    scores.copy_(random_scores(63, 2, 2, 300))
    graph.replay()
    want = ref.kv_evict(st["k"].cpu(), st["v"].cpu(), st["tables"].cpu(), st["context"].cpu(), scores.cpu(), 128, 4, 32, st["ks"].cpu(), st["vs"].cpu(), to.cpu())
    for a, b in zip((kept, kept_scores, lens), want):
        assert torch.equal(a.cpu(), b)
