"""What is timed of the operators around many samples of one prompt and a cache of bounded size.

Attention of packed groups, each a prefix and the samples that continue it, with its gradients (``ops.attention_shared_prefix``); the same for one new
token per sample over KV pages (``ops.paged_decode_shared``); decode attention that adds up what weight every cached token has got
(``ops.paged_decode_scored``); and the eviction of the tokens that got least (``ops.kv_evict``).

With ``own`` false ``run`` is their plain form in torch, with ``own`` true the calls that a user makes.  ``exact`` gives the same outputs from the
definitions in float64.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DIM = 128                           # the head size of the framework's attention kernels
PAGE = 16
HEADS = [(12, 2), (28, 4), (16, 2), (8, 8), (16, 4), (4, 1)]        # the policies' layouts, and others that the kernels take


def listed():
    return [
        # one prompt's few short samples: launches count
        {"name": "prefix_few", "op": "prefix", "groups": 1, "samples": 4, "prefix": 37, "response": 65, "heads": 12, "kv": 2, "grad": True},
        # a micro-step over all samples of some prompts, forward and backward
        {"name": "prefix_micro_step", "op": "prefix", "groups": 4, "samples": 4, "prefix": 731, "response": 1500, "heads": 12, "kv": 2, "grad": True},
        # scoring the samples of long prompts: no gradients
        {"name": "prefix_score_long", "op": "prefix", "groups": 2, "samples": 8, "prefix": 6001, "response": 700, "heads": 28, "kv": 4, "grad": False},
        # the tail of a rollout: one prompt's last samples
        {"name": "decode_few", "op": "decode", "groups": 1, "samples": 4, "prefix": 100, "response": 33, "heads": 12, "kv": 2, "pages": "bf16"},
        # a full rollout batch in the middle of its responses
        {"name": "decode_rollout", "op": "decode", "groups": 64, "samples": 8, "prefix": 517, "response": 1200, "heads": 12, "kv": 2, "pages": "bf16"},
        # many samples of long prompts, fp8 pages
        {"name": "decode_long_fp8", "op": "decode", "groups": 13, "samples": 16, "prefix": 4111, "response": 900, "heads": 28, "kv": 4, "pages": "fp8"},
        # a few rows with scores: the smallest call
        {"name": "scored_few", "op": "scored", "rows": 3, "context": 129, "heads": 12, "kv": 2, "pages": "bf16", "decay": 1.0},
        # a rollout batch with scores that fade
        {"name": "scored_rollout_fp8", "op": "scored", "rows": 509, "context": 1500, "heads": 12, "kv": 2, "pages": "fp8", "decay": 0.99},
        # few long contexts
        {"name": "scored_long", "op": "scored", "rows": 7, "context": 20011, "heads": 28, "kv": 4, "pages": "bf16", "decay": 1.0},
        # one row over its budget
        {"name": "evict_one", "op": "evict", "rows": 1, "context": 300, "keep": 128, "sinks": 4, "recent": 32, "kv": 2, "pages": "bf16"},
        # a rollout batch of which some rows are below their budget
        {"name": "evict_rollout_fp8", "op": "evict", "rows": 253, "context": 1400, "keep": 500, "sinks": 4, "recent": 64, "kv": 2, "pages": "fp8"},
        # few long contexts
        {"name": "evict_long", "op": "evict", "rows": 8, "context": 30011, "keep": 4096, "sinks": 16, "recent": 256, "kv": 4, "pages": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["prefix", "decode", "scored", "evict"])
    heads, kv = rng.choice(HEADS)
    if op == "prefix":
        while True:
            c = {"op": op, "groups": _log(rng, 1, 6), "samples": _log(rng, 1, 16), "prefix": _log(rng, 1, 6000), "response": _log(rng, 1, 1500),
                 "heads": heads, "kv": kv, "grad": rng.random() < 0.6}
            # not above the largest listed ones: their plain forms hold rows x keys scores, three times with gradients
            scores = heads * c["groups"] * (c["prefix"] ** 2 + c["samples"] * c["response"] * (c["prefix"] + c["response"]))
            if scores < (1.0e9 if c["grad"] else 4.5e9):
                return c
    pages = rng.choice(["bf16", "fp8"])
    if op == "decode":
        while True:
            c = {"op": op, "groups": _log(rng, 1, 64), "samples": _log(rng, 1, 32), "prefix": _log(rng, 16, 6000), "response": _log(rng, 1, 1500),
                 "heads": heads, "kv": kv, "pages": pages}
            if kv * c["groups"] * (c["prefix"] + c["samples"] * c["response"]) < 1.3e6 and heads * c["groups"] * c["samples"] * (c["prefix"] + c["response"]) < 3.0e7:
                return c
    if op == "scored":
        while True:
            c = {"op": op, "rows": _log(rng, 1, 512), "context": _log(rng, 1, 20000), "heads": heads, "kv": kv, "pages": pages,
                 "decay": rng.choice([1.0, round(rng.uniform(0.5, 1.0), 3)])}
            if kv * c["rows"] * c["context"] < 1.5e6 and heads * c["rows"] * c["context"] < 1.0e7:
                return c
    while True:
        c = {"op": op, "rows": _log(rng, 1, 256), "context": _log(rng, 1, 30000), "kv": kv, "pages": pages}
        c["keep"] = _log(rng, 1, max(1, c["context"]))
        c["sinks"] = rng.randint(0, min(16, c["keep"]))
        c["recent"] = rng.randint(0, min(256, c["keep"] - c["sinks"]))
        if kv * c["rows"] * c["context"] < 9.0e5:
            return c


# ---- lengths: by the case alone ------------------------------------------------------------------------------------------------------
def _lengths(case):
    """prefix: [[prefix, response, response, ...] per group]; decode: the same; scored, evict: [context per row].  The first is the largest."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["op"] in ("prefix", "decode"):
        out = []
        for g in range(case["groups"]):
            prefix = case["prefix"] if g == 0 else r.randint(max(1, case["prefix"] // 2), case["prefix"])
            out.append([prefix] + [case["response"] if g == i == 0 else r.randint(max(1, case["response"] // 4), case["response"]) for i in range(case["samples"])])
        return out
    return [case["context"] if i == 0 else r.randint(max(1, case["context"] // 4), case["context"]) for i in range(case["rows"])]


def _shared(prefix):
    """Tokens of a prompt that its samples share in whole pages."""
    return prefix // PAGE * PAGE


# ---- inputs ----------------------------------------------------------------------------------------------------------------------------
def _vectors(g, *shape):
    """Unit variance with the few large channels that keys and queries have."""
    x = torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)
    x[..., ::16] *= 2.0
    return x.to(torch.bfloat16)


def _cache(g, n_pages, kv, pages):
    """{"k", "v"} pages, with scales for fp8: e4m3 of the vectors by the largest of each, values transposed."""
    k, v = _vectors(g, n_pages, kv, PAGE, DIM), _vectors(g, n_pages, kv, PAGE, DIM)
    if pages == "bf16":
        return {"k": k, "v": v, "ks": None, "vs": None}
    ks, vs = k.abs().amax(-1).float() / 448.0, v.abs().amax(-1).float() / 448.0
    k8 = (k.float() / ks[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    v8 = (v.float() / vs[..., None]).to(torch.float8_e4m3fn).transpose(2, 3).contiguous().view(torch.uint8)
    return {"k": k8, "v": v8, "ks": ks, "vs": vs}


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _tables(perm, counts):
    """Rows of page numbers out of `perm`, counts[i] of them for row i, as wide as the largest."""
    width, at, rows = max(counts), 0, []
    for n in counts:
        rows.append(perm[at:at + n] + [0] * (width - n))
        at += n
    return rows


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    lens = _lengths(case)
    st = {"case": case}
    if case["op"] == "prefix":
        flat = [n for group in lens for n in group]
        T = sum(flat)
        st.update(q=_vectors(g, T, case["heads"], DIM), k=_vectors(g, T, case["kv"], DIM), v=_vectors(g, T, case["kv"], DIM), cu_seqlens=_int(_offsets(flat)),
                  cu_groups=_int(_offsets([len(group) for group in lens])), longest=max(flat), longest_prefix=max(x[0] for x in lens),
                  longest_response=max(max(x[1:]) for x in lens))
        if case["grad"]:
            st["dout"] = _vectors(g, T, case["heads"], DIM)
        return st
    shuffle = lambda n: torch.randperm(n, generator=g, device=DEV).tolist()  # noqa: E731
    if case["op"] == "decode":
        S = case["groups"] * case["samples"]
        own_counts = [(p + r + PAGE - 1) // PAGE - p // PAGE for p, *rs in lens for r in rs]
        shared = [x[0] // PAGE for x in lens]
        perm = shuffle(sum(own_counts) + sum(shared) + 1)
        table, at = [], 0
        for i, n in enumerate(shared):
            common, at = perm[at:at + n], at + n
            for c in own_counts[i * case["samples"]:(i + 1) * case["samples"]]:
                table.append(common + perm[at:at + c])
                at += c
        width = max(len(r) for r in table)
        st.update(_cache(g, len(perm), case["kv"], case["pages"]), q=_vectors(g, S, case["heads"], DIM), tables=_int([r + [perm[-1]] * (width - len(r)) for r in table]),
                  context=_int([x[0] + r for x in lens for r in x[1:]]), cu_groups=_int(_offsets([case["samples"]] * case["groups"])),
                  shared=_int([_shared(x[0]) for x in lens]), longest_shared=max(_shared(x[0]) for x in lens),
                  longest_rest=max(x[0] + r - _shared(x[0]) for x in lens for r in x[1:]))
        return st
    pages = [(n + PAGE - 1) // PAGE for n in lens]
    # what cached tokens have got so far: a few much, many next to nothing, some the same
    gain = torch.randn(len(lens), case["kv"], max(lens), generator=g, device=DEV).mul_(2.0).exp_()
    st["scores"] = torch.where(gain < 0.05, 0.0, gain)
    st["context"] = _int(lens)
    if case["op"] == "scored":
        st.update(_cache(g, sum(pages), case["kv"], case["pages"]), q=_vectors(g, len(lens), case["heads"], DIM), tables=_int(_tables(shuffle(sum(pages)), pages)),
                  new_scores=torch.zeros_like(st["scores"]))
        return st
    to = [(min(n, case["keep"]) + PAGE - 1) // PAGE for n in lens]
    st.update(_cache(g, sum(pages) + sum(to), case["kv"], case["pages"]), tables=_int(_tables(shuffle(sum(pages)), pages)), first=sum(pages),
              to=_int(_tables([sum(pages) + i for i in shuffle(sum(to))], to)))
    for name in ("k", "v", "ks", "vs"):
        if st[name] is not None:
            st[name][st["first"]:] = 0
    return st


# ---- plain forms -----------------------------------------------------------------------------------------------------------------------
def _softmax(s, seen):
    """Along the last axis over what is seen; 0 for a row that sees nothing."""
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    e = (s - torch.where(m == -math.inf, 0.0, m)).exp()
    return e / e.sum(-1, keepdim=True).clamp_min(1e-30)


def _attend(q, k, v, seen):
    """q [B, L, Hq, D], k and v [B, K, Hkv, D], seen [B, L, K]"""
    B, L, Hq, D = q.shape
    q = q.view(B, L, k.shape[2], -1, D)
    s = torch.einsum("blhgd,bkhd->bhglk", q, k) / math.sqrt(D)
    p = _softmax(s, seen[:, None, None])
    return torch.einsum("bhglk,bkhd->blhgd", p, v).reshape(B, L, Hq, D)


def _plain_prefix_forward(q, k, v, st):
    """Sequences padded to the longest: the prefixes, and the responses behind a copy of theirs."""
    c = st["case"]
    T = q.shape[0]
    cu, first = st["cu_seqlens"].long(), st["cu_groups"].long()[:-1]
    P, L, N = st["longest_prefix"], st["longest_response"], c["samples"]
    pre_at, pre_n = cu[first], cu[first + 1] - cu[first]
    pos = torch.arange(P, device=q.device)
    pre_idx = (pre_at[:, None] + pos).clamp(max=T - 1)
    pre_ok = pos < pre_n[:, None]
    own_seq = (first[:, None] + 1 + torch.arange(N, device=q.device)).reshape(-1)
    at, n = cu[own_seq], cu[own_seq + 1] - cu[own_seq]
    row = torch.arange(L, device=q.device)
    idx, ok = (at[:, None] + row).clamp(max=T - 1), row < n[:, None]
    o_pre = _attend(q[pre_idx], k[pre_idx], v[pre_idx], pre_ok[:, None, :] & (pos <= pos[:, None]))
    both = torch.cat([pre_idx.repeat_interleave(N, 0), idx], 1)
    seen = torch.cat([pre_ok.repeat_interleave(N, 0)[:, None, :].expand(-1, L, -1), ok[:, None, :] & (row <= row[:, None])], 2)
    o = _attend(q[idx], k[both], v[both], seen)
    # rows of the padding go to a row behind the last, which is cut off
    out = q.new_zeros(T + 1, *q.shape[1:])
    out = out.index_put((torch.where(pre_ok, pre_idx, T).reshape(-1),), o_pre.flatten(0, 1))
    return out.index_put((torch.where(ok, idx, T).reshape(-1),), o.flatten(0, 1))[:T]


def _plain_prefix(st):
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    if not st["case"]["grad"]:
        return {"out": _plain_prefix_forward(q, k, v, st).to(torch.bfloat16)}
    with torch.enable_grad():
        leaves = [x.requires_grad_() for x in (q, k, v)]
        out = _plain_prefix_forward(*leaves, st)
        grads = torch.autograd.grad(out, leaves, st["dout"].float())
    return {"out": out.detach().to(torch.bfloat16), **{n: x.to(torch.bfloat16) for n, x in zip(("dq", "dk", "dv"), grads)}}


def _read(st, page, off):
    """Keys and values [.., Hkv, D] in float of the tokens at (page, off)"""
    k, v = st["k"][page, :, off], st["v"]
    if st["ks"] is None:
        return k.float(), v[page, :, off].float()
    v = v[page, :, :, off]
    return (k.view(torch.float8_e4m3fn).float() * st["ks"][page, :, off][..., None],
            v.contiguous().view(torch.float8_e4m3fn).float() * st["vs"][page, :, off][..., None])


def _tokens(table, t):
    """(page, offset) of tokens t [B, n] of the rows of a page table"""
    return table.long().gather(1, (t // PAGE).clamp(max=table.shape[1] - 1)), t % PAGE


def _plain_decode(st):
    c = st["case"]
    G, N, Hkv = c["groups"], c["samples"], c["kv"]
    q = st["q"].float().view(G, N, Hkv, -1, DIM)
    shared, ctx = st["shared"].long(), st["context"].long()
    P, L = st["longest_shared"], st["longest_rest"]
    t = torch.arange(P, device=q.device).expand(G, -1)
    kp, vp = _read(st, *_tokens(st["tables"][st["cu_groups"].long()[:-1]], t))
    start = shared.repeat_interleave(N)
    t2 = start[:, None] + torch.arange(L, device=q.device)
    ks, vs = _read(st, *_tokens(st["tables"], t2))
    ks, vs = ks.view(G, N, L, Hkv, DIM), vs.view(G, N, L, Hkv, DIM)
    s = torch.cat([torch.einsum("bnhgd,bkhd->bnhgk", q, kp), torch.einsum("bnhgd,bnkhd->bnhgk", q, ks)], -1) / math.sqrt(DIM)
    seen = torch.cat([(t < shared[:, None])[:, None].expand(-1, N, -1), (t2 < ctx[:, None]).view(G, N, L)], -1)
    p = _softmax(s, seen[:, :, None, None])
    o = torch.einsum("bnhgk,bkhd->bnhgd", p[..., :P], vp) + torch.einsum("bnhgk,bnkhd->bnhgd", p[..., P:], vs)
    return {"out": o.reshape(G * N, -1, DIM).to(torch.bfloat16)}


def _plain_scored(st):
    c = st["case"]
    S, Hkv, L = st["scores"].shape
    q, ctx = st["q"].float().view(S, Hkv, -1, DIM), st["context"].long()
    t = torch.arange(L, device=q.device).expand(S, -1)
    k, v = _read(st, *_tokens(st["tables"], t))
    seen = t < ctx[:, None]
    p = _softmax(torch.einsum("shgd,skhd->shgk", q, k) / math.sqrt(DIM), seen[:, None, None])
    o = torch.einsum("shgk,skhd->shgd", p, v)
    old = torch.where((t < ctx[:, None] - 1)[:, None], st["scores"] * c["decay"], 0.0)         # the newest token has none yet
    st["new_scores"].copy_(torch.where(seen[:, None], old + p.sum(2), st["new_scores"]))
    return {"out": o.reshape(S, -1, DIM).to(torch.bfloat16), "scores": st["new_scores"]}


def _plain_evict(st):
    c, scores, n = st["case"], st["scores"], st["context"].long()
    S, Hkv, L = scores.shape
    keep = c["keep"]
    t = torch.arange(L, device=scores.device)
    here = t < n[:, None]
    safe = here & ((t < c["sinks"]) | (t >= n[:, None] - c["recent"]))
    value = torch.where(safe[:, None], math.inf, torch.where(here[:, None], scores, -math.inf))
    idx = value.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    idx = torch.nn.functional.pad(torch.where(idx < n[:, None, None], idx, L), (0, keep - idx.shape[-1]), value=L).sort(-1).values
    ok = idx < L
    at = torch.where(ok, idx, 0)
    src, off = st["tables"].long().gather(1, (at // PAGE).flatten(1)).view_as(at), at % PAGE
    h = torch.arange(Hkv, device=scores.device)[:, None]
    j = torch.arange(keep, device=scores.device).expand_as(at)
    to_page = (j // PAGE).clamp(max=st["to"].shape[1] - 1)
    to, to_off = st["to"].long().gather(1, to_page.flatten(1)).view_as(at), j % PAGE
    # places that nothing moves to take the row's first kept token a second time
    to, to_off = torch.where(ok, to, to[..., :1]), torch.where(ok, to_off, 0)
    src, off = torch.where(ok, src, src[..., :1]), torch.where(ok, off, off[..., :1])
    st["k"][to, h, to_off] = st["k"][src, h, off]
    if st["ks"] is None:
        st["v"][to, h, to_off] = st["v"][src, h, off]
    else:
        st["v"][to, h, :, to_off] = st["v"][src, h, :, off]
        st["ks"][to, h, to_off] = st["ks"][src, h, off]
        st["vs"][to, h, to_off] = st["vs"][src, h, off]
    return _evicted(st, torch.where(ok, idx, -1).int(), torch.where(ok, scores.gather(2, at), 0.0), n.clamp(max=keep).int())


def _evicted(st, kept, kept_scores, lens):
    out = {"kept": kept, "scores": kept_scores, "lens": lens, "k": st["k"][st["first"]:], "v": st["v"][st["first"]:]}
    if st["ks"] is not None:
        out.update(k=out["k"].view(torch.float8_e4m3fn), v=out["v"].view(torch.float8_e4m3fn), k_scale=st["ks"][st["first"]:], v_scale=st["vs"][st["first"]:])
    return out


# ---- one pass --------------------------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    with torch.no_grad():
        return {"prefix": _plain_prefix, "decode": _plain_decode, "scored": _plain_scored, "evict": _plain_evict}[op](state)


def _own(st, op):
    from nanorlhf_b200 import ops
    c = st["case"]
    if op == "prefix":
        if not c["grad"]:
            with torch.no_grad():
                return {"out": ops.attention_shared_prefix(st["q"], st["k"], st["v"], st["cu_seqlens"], st["cu_groups"], st["longest"])}
        q, k, v = (st[n].detach().requires_grad_() for n in ("q", "k", "v"))
        out = ops.attention_shared_prefix(q, k, v, st["cu_seqlens"], st["cu_groups"], st["longest"])
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), st["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if op == "decode":
        return {"out": ops.paged_decode_shared(st["q"], st["k"], st["v"], st["tables"], st["context"], st["cu_groups"], st["shared"], max_group=c["samples"],
                                               k_scale=st["ks"], v_scale=st["vs"])}
    if op == "scored":
        out, scores = ops.paged_decode_scored(st["q"], st["k"], st["v"], st["tables"], st["context"], st["scores"], decay=c["decay"], k_scale=st["ks"],
                                              v_scale=st["vs"], out_scores=st["new_scores"])
        return {"out": out, "scores": scores}
    kept, scores, lens = ops.kv_evict(st["k"], st["v"], st["tables"], st["context"], st["scores"], keep=c["keep"], sinks=c["sinks"], recent=c["recent"],
                                      k_scale=st["ks"], v_scale=st["vs"], out_tables=st["to"])
    return _evicted(st, kept, scores, lens)


def work(case):
    lens = _lengths(case)
    if case["op"] == "prefix":
        # pairs of a query and a key that it sees; 2 products forward, 5 backward; a triangle has n (n + 1) / 2
        pairs = sum(p * (p + 1) // 2 + sum(r * p + r * (r + 1) // 2 for r in rs) for p, *rs in lens)
        T = sum(sum(x) for x in lens)
        rows = 2 * DIM * T                                                          # bytes of one head
        # read q, k, v and written out; with gradients their own, and out's
        tensors = (4 * case["heads"] + 4 * case["kv"]) if case["grad"] else 2 * case["heads"] + 2 * case["kv"]
        return {"bytes": rows * tensors,
                "flops": 2 * DIM * case["heads"] * pairs * (7 if case["grad"] else 2)}
    token = case["kv"] * 2 * (2 * DIM if case["pages"] == "bf16" else DIM + 4)      # a token's keys and values
    if case["op"] == "decode":
        S = case["groups"] * case["samples"]
        read = sum(_shared(p) + sum(p + r - _shared(p) for r in rs) for p, *rs in lens)
        seen = sum(p + r for p, *rs in lens for r in rs)
        return {"bytes": read * token + 4 * DIM * S * case["heads"], "flops": 4 * DIM * case["heads"] * seen}
    if case["op"] == "scored":
        n = sum(lens)
        return {"bytes": n * (token + 8 * case["kv"]) + 4 * DIM * case["rows"] * case["heads"], "flops": 4 * DIM * case["heads"] * n}
    kept = sum(min(n, case["keep"]) for n in lens)
    return {"bytes": sum(lens) * 4 * case["kv"] + kept * (2 * token + 8 * case["kv"]), "flops": sum(lens) * case["kv"]}


# ---- from the definitions, in float64 --------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    lens = _lengths(case)
    with torch.no_grad():
        return {"prefix": _exact_prefix, "decode": _exact_decode, "scored": _exact_scored, "evict": _exact_evict}[case["op"]](st, case, lens)


def _rows64(q, k, v, mask, dout=None):
    """Attention of q [n, d] over k, v [m, d] by one mask; with dout its gradients from the formulas."""
    s = q @ k.t() / math.sqrt(DIM)
    if mask is not None:
        s = s.masked_fill(mask, -math.inf)
    p = torch.softmax(s, -1)
    o = p @ v
    if dout is None:
        return o
    ds = p * (dout @ v.t() - (dout * o).sum(-1, keepdim=True))
    return o, ds @ k / math.sqrt(DIM), ds.t() @ q / math.sqrt(DIM), p.t() @ dout


def _exact_prefix(st, case, lens):
    q, k, v = st["q"].double(), st["k"].double(), st["v"].double()
    share = case["heads"] // case["kv"]
    out = torch.zeros_like(q)
    grads = [torch.zeros_like(x) for x in (q, k, v)] if case["grad"] else None
    at = 0
    for prefix, *responses in lens:
        parts, begin = [(at, prefix, 0)], at + prefix
        for n in responses:
            parts.append((begin, n, prefix))
            begin += n
        for row0, n, extra in parts:
            rows = slice(row0, row0 + n)
            hidden = torch.cat([torch.zeros(n, extra, dtype=torch.bool, device=DEV), torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1)], 1)
            for h in range(case["heads"]):
                kh = h // share
                keys, values = (torch.cat([x[at:at + extra, kh], x[rows, kh]]) for x in (k, v))
                if grads is None:
                    out[rows, h] = _rows64(q[rows, h], keys, values, hidden)
                    continue
                out[rows, h], grads[0][rows, h], dk, dv = _rows64(q[rows, h], keys, values, hidden, st["dout"][rows, h].double())
                for into, d in ((grads[1], dk), (grads[2], dv)):
                    into[at:at + extra, kh] += d[:extra]
                    into[rows, kh] += d[extra:]
        at = begin
    return {"out": out} if grads is None else {"out": out, "dq": grads[0], "dk": grads[1], "dv": grads[2]}


def _row_cache(st, row, n):
    """Keys and values [Hkv, n, D] of one row in float64"""
    pages = st["tables"][row].long()[:(n + PAGE - 1) // PAGE]
    k, v = st["k"][pages], st["v"][pages]
    if st["ks"] is not None:
        k = k.view(torch.float8_e4m3fn).double() * st["ks"][pages].double()[..., None]
        v = v.view(torch.float8_e4m3fn).double().transpose(2, 3) * st["vs"][pages].double()[..., None]
    return tuple(x.double().transpose(0, 1).flatten(1, 2)[:, :n] for x in (k, v))


def _exact_rows(st, case, contexts):
    outs, weights = [], []
    for row, n in enumerate(contexts):
        k, v = _row_cache(st, row, n)
        q = st["q"][row].double().view(case["kv"], -1, DIM)
        p = torch.softmax(q @ k.transpose(1, 2) / math.sqrt(DIM), -1)
        outs.append((p @ v).reshape(-1, DIM))
        weights.append(p.sum(1))
    return torch.stack(outs), weights


def _exact_decode(st, case, lens):
    return {"out": _exact_rows(st, case, [p + r for p, *rs in lens for r in rs])[0]}


def _exact_scored(st, case, lens):
    out, weights = _exact_rows(st, case, lens)
    scores = torch.zeros(st["scores"].shape, dtype=torch.float64, device=DEV)
    for row, n in enumerate(lens):
        scores[row, :, :n] = weights[row]
        scores[row, :, :n - 1] += case["decay"] * st["scores"][row, :, :n - 1].double()
    return {"out": out, "scores": scores}


def _exact_evict(st, case, lens):
    """Row by row and head by head; what is moved has no other value in 64 bits."""
    keep, sinks, recent = case["keep"], case["sinks"], case["recent"]
    kept = torch.full((case["rows"], case["kv"], keep), -1, dtype=torch.int32, device=DEV)
    scores = torch.zeros(case["rows"], case["kv"], keep, dtype=torch.float64, device=DEV)
    for row, n in enumerate(lens):
        for h in range(case["kv"]):
            x = st["scores"][row, h, :n]
            if n <= keep:
                chosen = torch.arange(n, device=DEV)
            else:
                middle = torch.sort(-x[sinks:n - recent], stable=True).indices[:keep - sinks - recent] + sinks
                chosen = torch.cat([torch.arange(sinks, device=DEV), middle.sort().values, torch.arange(n - recent, n, device=DEV)])
            kept[row, h, :len(chosen)] = chosen.int()
            scores[row, h, :len(chosen)] = x[chosen].double()
    return {"kept": kept, "scores": scores, "lens": _int([min(n, keep) for n in lens]), "k": None, "v": None, "k_scale": None, "v_scale": None}
