"""Arguments of the calls around many samples of one prompt, and what they refuse."""
import math

import pytest
import torch

from nanorlhf_b200 import ops


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


def packed(groups, heads, kv, dim=128, dtype=torch.float32, spare=0):
    g = torch.Generator().manual_seed(1)
    T = sum(map(sum, groups)) + spare
    q, k, v, dout = (torch.randn(T, h, dim, generator=g).to(dtype) for h in (heads, kv, kv, heads))
    lens = [n for x in groups for n in x]
    return q, k, v, dout, ints(0, *torch.tensor(lens).cumsum(0).tolist()), ints(0, *torch.tensor([len(x) for x in groups]).cumsum(0).tolist())


def pool(blocks=12, kv=2, fp8=False):
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(blocks, kv, 16, 128, generator=g) for _ in range(2))
    if not fp8:
        return {"k": k.to(torch.bfloat16), "v": v.to(torch.bfloat16), "ks": None, "vs": None}
    ks, vs = k.abs().amax(-1) / 448.0, v.abs().amax(-1) / 448.0
    return {"k": (k / ks[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), "ks": ks, "vs": vs,
            "v": (v / vs[..., None]).to(torch.float8_e4m3fn).transpose(2, 3).contiguous().view(torch.uint8)}


def refused_calls(device):
    """Every call here is refused before anything is launched; the calls without a fault are not made on a GPU."""
    to = lambda x: x.to(device) if torch.is_tensor(x) else x  # noqa: E731
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    q, k, v, _, cu, cg = map(to, packed([[3, 4]], 4, 2, dtype=dtype))
    f = ops.attention_shared_prefix
    for bad in ((q[:, :3], k, v, cu, cg), (q, k[:-1], v[:-1], cu, cg), (q, k, v[:, :1], cu, cg), (q[0], k, v, cu, cg), (q, k, v, cu[None], cg), (q, k, v, cu, cg[:0])):
        with pytest.raises(ValueError):
            f(*bad)
    with pytest.raises(ValueError):
        f(q, k, v, cu, cg, scale=float("nan"))
    for bad in ((q.double(), k, v, cu, cg), (q, k, v, cu.long(), cg), (q, k, v, cu, cg.float()), (q, k.double(), v.double(), cu, cg)):
        with pytest.raises(TypeError):
            f(*bad)
    st, st8 = ({n: to(x) for n, x in pool(fp8=fp8).items()} for fp8 in (False, True))
    tables, context, scores = map(to, (torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32), ints(40, 6), torch.rand(2, 2, 48)))
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16, device=device)
    groups = (to(ints(0, 2)), to(ints(16)))
    calls = {"shared": lambda q=q, k=st["k"], v=st["v"], t=tables, c=context, g=groups, **kw: ops.paged_decode_shared(q, k, v, t, c, *g, **kw),
             "scored": lambda q=q, k=st["k"], v=st["v"], t=tables, c=context, s=scores, **kw: ops.paged_decode_scored(q, k, v, t, c, s, **kw),
             "evict": lambda k=st["k"], v=st["v"], t=tables, c=context, s=scores, keep=10, **kw: ops.kv_evict(k, v, t, c, s, keep, **kw)}
    for call in calls.values():
        if device == "cpu":
            call()
        for kw in ({"k": st["k"][..., :8, :]}, {"v": st["v"][:3]}, {"t": tables[:1]}, {"t": tables[0]}, {"c": context[None]}, {"k_scale": st8["ks"]},
                   {"k": st8["k"], "v": st8["v"], "k_scale": st8["ks"][:3], "v_scale": st8["vs"]}):
            with pytest.raises(ValueError):
                call(**kw)
        for kw in ({"k": st8["k"], "v": st8["v"]}, {"k_scale": st8["ks"], "v_scale": st8["vs"]}, {"t": tables.long()}, {"c": context.float()}):
            with pytest.raises(TypeError):
                call(**kw)
    for name in ("shared", "scored"):
        for kw in ({"q": q[:1]}, {"q": q[:, :3]}, {"q": q[..., :64]}, {"q": torch.zeros(2, 18, 128, device=device)}, {"scale": math.inf}):
            with pytest.raises(ValueError):
                calls[name](**kw)
    for kw in ({"g": (to(ints(0, 1, 2)), to(ints(16)))}, {"max_group": 0}):
        with pytest.raises(ValueError):
            calls["shared"](**kw)
    with pytest.raises(TypeError):
        calls["shared"](g=(to(torch.tensor([0, 2])), to(ints(16))))
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
