"""CUDA backend of the op layer: thin autograd wrappers over ``nanorlhf_b200/_C.so``.

``load()`` imports the in-tree extension (built by ``python -m nanorlhf_b200.csrc.build``).  It is
not JIT-compiled at import: the ``.so`` must travel with the source tree, and a
missing build on a machine with a GPU is a hard error (ops/__init__.py), never a silent PyTorch fallback.
"""
from __future__ import annotations

import math
import os
from typing import Optional

import torch
import torch.nn.functional as F

from . import reference as ref

_C = None
LAUNCHES = 0          # number of native kernel launches issued through this module (bench "gpu_launches")


def load():
    global _C
    if _C is None:
        from .. import _C as ext          # noqa: F401  (ImportError propagates with the real reason)
        _C = ext
    return _C


def ext():
    return load()


def _count(n: int = 1):
    global LAUNCHES
    LAUNCHES += n


def launches() -> int:
    return LAUNCHES


# --------------------------------------------------------------------------------------------
# GEMM
# --------------------------------------------------------------------------------------------
def add_layernorm(x, residual, weight, bias, eps):
    """LayerNorm(x + residual) in one pass (inference; reward model)."""
    _count()
    return ext().add_layernorm(x, residual, weight, bias, float(eps))


def gemm_bf16(a, b, bias=None, out=None, block_n: int = 0, act: int = 0):
    """a[M,K] @ b[N,K]^T (+bias) on the tcgen05 kernel; inputs must be bf16, K-contiguous."""
    _count()
    return ext().gemm_bf16(a, b, bias, out, block_n, act)


def linear(x, w, b=None, act: int = 0):
    """y = x W^T + b with forward / dgrad / wgrad on the general tcgen05 GEMM (ops/gemm.py)."""
    from . import gemm as _lin
    return _lin.linear(x, w, b, act)


# --------------------------------------------------------------------------------------------
# norms / rope / activation
# --------------------------------------------------------------------------------------------
class _RMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, eps):
        x2 = x.reshape(-1, x.shape[-1]).contiguous()
        need = x.requires_grad or w.requires_grad
        _count()
        y, _, rstd = ext().rmsnorm(x2, w, eps, None, need)
        if need:
            ctx.save_for_backward(x2, w, rstd)
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, gy):
        x2, w, rstd = ctx.saved_tensors
        g2 = gy.reshape(-1, gy.shape[-1]).contiguous()
        _count()
        gx = ext().rmsnorm_bwd(x2, w, g2, rstd).view(gy.shape)
        gw = None
        if ctx.needs_input_grad[1]:
            gw = (g2.float() * (x2.float() * rstd[:, None])).sum(0).to(w.dtype)
        return gx, gw, None


def rmsnorm(x, weight, eps):
    if x.dtype != torch.bfloat16:
        return ref.rmsnorm(x, weight, eps)
    return _RMSNormFn.apply(x, weight, eps)


def add_rmsnorm(x, residual, weight, eps):
    """Inference-only fused residual add + RMSNorm: returns (y, residual + x)."""
    _count()
    y, res, _ = ext().rmsnorm(x.contiguous(), weight, eps, residual.contiguous(), False)
    return y, res


class _RopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, cos, sin):
        ctx.save_for_backward(cos, sin)
        _count()
        return ext().rope(x, cos, sin, 1.0, False)

    @staticmethod
    def backward(ctx, gy):
        cos, sin = ctx.saved_tensors
        _count()
        return ext().rope(gy.contiguous(), cos, sin, -1.0, False), None, None


def apply_rope(x, cos, sin):
    if x.dtype != torch.bfloat16:
        return ref.apply_rope(x, cos, sin)
    if x.stride(-1) != 1 or x.stride(1) != x.shape[2]:
        x = x.contiguous()
    return _RopeFn.apply(x, cos.float().contiguous(), sin.float().contiguous())


class _SwigluFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu):
        g2 = gu.reshape(-1, gu.shape[-1]).contiguous()
        ctx.save_for_backward(g2)
        _count()
        return ext().swiglu(g2).view(*gu.shape[:-1], gu.shape[-1] // 2)

    @staticmethod
    def backward(ctx, go):
        (g2,) = ctx.saved_tensors
        _count()
        return ext().swiglu_bwd(g2, go.reshape(-1, go.shape[-1]).contiguous()).view(*go.shape[:-1], go.shape[-1] * 2)


def swiglu(gate_up):
    if gate_up.dtype != torch.bfloat16:
        return ref.swiglu(gate_up)
    return _SwigluFn.apply(gate_up)


class _SwigluPairFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up):
        g2 = gate.reshape(-1, gate.shape[-1]).contiguous()
        u2 = up.reshape(-1, up.shape[-1]).contiguous()
        ctx.save_for_backward(g2, u2)
        _count()
        return ext().swiglu_pair(g2, u2).view(gate.shape)

    @staticmethod
    def backward(ctx, go):
        g2, u2 = ctx.saved_tensors
        _count()
        dg, du = ext().swiglu_pair_bwd(g2, u2, go.reshape(-1, go.shape[-1]).contiguous())
        return dg.view(go.shape), du.view(go.shape)


def swiglu_pair(gate, up):
    if gate.dtype != torch.bfloat16:
        return (F.silu(gate.float()) * up.float()).to(gate.dtype)
    return _SwigluPairFn.apply(gate, up)


# --------------------------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------------------------
def attention_varlen(q, k, v, cu_seqlens, max_seqlen=None, causal=True, scale=None):
    from . import attention
    return attention.attention_varlen(q, k, v, cu_seqlens, max_seqlen, causal, scale)


# --------------------------------------------------------------------------------------------
# fused lm-head log-prob (K-LP)
# --------------------------------------------------------------------------------------------
class _LmHeadLogprobFn(torch.autograd.Function):
    """Forward: tcgen05 GEMM with an online-softmax epilogue, which for a backward also leaves the float32 logits where they take up to 4 GiB and plenty is free
    (``lmhead_logits_buffer``; no [T, V] tensor otherwise).
    Backward: dZ in bf16 from those logits, or from the same mainloop, which forms them again (one 8192-row chunk at a
    time); dH = dZ W (K-major x MN-major) and dW += dZ^T H (MN-major x MN-major, fp32 accumulate across chunks in the
    epilogue) run on the general tcgen05 GEMM -- W and H are consumed as stored, nothing is transposed."""

    CHUNK = 8192      # rows of dZ materialised at a time in backward (8192 x 152k bf16 = 2.5 GB)

    @staticmethod
    def forward(ctx, hidden, weight, targets, temperature, want_entropy, keep):
        h = hidden.contiguous()
        t32 = targets.to(torch.int32).contiguous()
        _count(2)
        z = ext().lmhead_logits_buffer(h, weight.shape[0]) if keep else None
        logp, ent, lse = ext().lmhead_logprob_fwd(h, weight, t32, 1.0 / temperature, 0, z)
        ctx.save_for_backward(h, weight, t32, lse, z)
        ctx.temperature = temperature
        ctx.mark_non_differentiable(ent)
        return logp, ent

    @staticmethod
    def backward(ctx, g_logp, _g_ent):
        h, weight, t32, lse, z = ctx.saved_tensors
        inv_t = 1.0 / ctx.temperature
        g = g_logp.float().contiguous()
        need_h, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        dh = torch.empty_like(h) if need_h else None
        T = h.shape[0]
        # one chunk: dW leaves the GEMM's float32 accumulators as bf16 at once, rounded once as before (6001 rows x 151 936: 10.3 -> 9.5 ms
        # for the head; the float32 sums were zeroed, read, written and converted, 3.3 GB in all)
        whole = T <= _LmHeadLogprobFn.CHUNK
        dw = torch.zeros(weight.shape, dtype=torch.float32, device=weight.device) if need_w and not whole else None
        from . import gemm as _lin
        for s in range(0, T, _LmHeadLogprobFn.CHUNK):
            e = min(T, s + _LmHeadLogprobFn.CHUNK)
            _count()
            if z is not None:
                dz = ext().logits_grad(z[s:e], t32[s:e], lse[s:e], g[s:e], inv_t)
            else:
                dz = ext().lmhead_dlogits(h[s:e], weight, t32[s:e], lse[s:e], g[s:e], inv_t)
            if need_h:
                _lin.gemm(dz, weight, b_mn=True, out=dh[s:e])
            if need_w and whole:
                dw = _lin.gemm(dz, h, a_mn=True, b_mn=True, split_k=0)
            elif need_w:
                _lin.gemm(dz, h[s:e], a_mn=True, b_mn=True, out_f32=dw, accumulate=True)
        return dh, (dw.to(weight.dtype) if need_w else None), None, None, None, None


def lmhead_logprob(hidden, weight, targets, temperature=1.0, want_entropy=True):
    if hidden.dtype != torch.bfloat16 or hidden.shape[0] == 0:
        logp, ent, _ = ref.lmhead_logprob(hidden, weight, targets, temperature, want_entropy=want_entropy)
        return logp, ent
    keep = torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad)
    return _LmHeadLogprobFn.apply(hidden, weight, targets, float(temperature), bool(want_entropy), keep)


# --------------------------------------------------------------------------------------------
# a teacher's top log-probabilities and the divergence from them
# --------------------------------------------------------------------------------------------
def _row_major(logits):
    return logits if logits.stride(1) == 1 or logits.shape[1] == 1 else logits.contiguous()


@torch.no_grad()
def top_logprobs(logits, k, temperature):
    _count()
    return ext().top_logprobs(_row_major(logits), k, 1.0 / temperature)


class _RecordedDistillFn(torch.autograd.Function):
    """The loss in a form that a tracer records as one operation (see ``_RecordedLossFn``)."""

    @staticmethod
    def forward(ctx, logits, top_logp, top_idx, weights, inv_temp, beta, tail):
        loss, token, grad = ext().distill_loss_parts(logits, top_logp, top_idx, weights, inv_temp, beta, tail, True, False, True)
        ctx.save_for_backward(grad)
        ctx.mark_non_differentiable(token)
        return loss, token

    @staticmethod
    def backward(ctx, g_loss, _g_token):
        return (ext().refuse_second(ctx.saved_tensors[0]) * g_loss,) + (None,) * 6


def distill_loss(logits, top_logp, top_idx, weights, temperature, beta, tail):
    _count(3 if logits.requires_grad and torch.is_grad_enabled() else 2)          # the rows, their sum and, later, a factor of the gradient
    if torch._C._get_tracing_state():
        return _RecordedDistillFn.apply(_row_major(logits), *ext().teacher_entries(top_logp, top_idx, weights, logits.shape[1]), 1.0 / temperature, beta, tail)
    return ext().distill_loss(logits, top_logp, top_idx, weights, 1.0 / temperature, beta, tail)


LOGITS_BYTES = 4 << 30      # float logits of a head that are held at a time


def _head_logits(h, weight, fused):
    """float logits of some rows"""
    from . import gemm as _lin
    if not fused:
        return F.linear(h.float(), weight.float())
    z = torch.empty(h.shape[0], weight.shape[0], dtype=torch.float32, device=h.device)
    _lin.gemm(h, weight, out_f32=z)
    return z


def _row_ranges(rows, columns):
    """as few equal ranges of rows as keep the float logits of one within LOGITS_BYTES"""
    most = max(256, LOGITS_BYTES // (4 * columns) // 256 * 256)
    n = max(1, -(-rows // most))
    step = max(1, -(-rows // n))
    return [(s, min(rows, s + step)) for s in range(0, rows, step)]


class _LmHeadDistillFn(torch.autograd.Function):
    """Logits, losses and the logits' gradients of a range of rows at a time, and with them at once the gradients of the hidden states and the head's, so that no
    logits are formed twice: three GEMMs in all, by torch in float32 for other types and sizes than the GEMM's.  The backward only multiplies by the loss's own gradient."""

    @staticmethod
    def forward(ctx, hidden, weight, top_logp, top_idx, weights, temperature, beta, tail, need_h, need_w):
        from . import gemm as _lin
        h, rows, V = hidden.contiguous(), hidden.shape[0], weight.shape[0]
        fused = _lin.supported(h, weight)
        if weights is None:
            weights = h.new_full((rows,), 1.0 / max(rows, 1), dtype=torch.float32)
        ranges = _row_ranges(rows, V if fused else V + V // 3 + 1)         # (their logits' gradients are float: both together take what the others' do)
        dh = torch.empty_like(h) if need_h else None
        once = fused and len(ranges) == 1                                 # dW leaves the GEMM rounded once
        dw = torch.zeros(weight.shape, dtype=torch.float32, device=weight.device) if need_w and not once else None
        tokens = []
        for s, e in ranges:
            z = _head_logits(h[s:e], weight, fused)
            _count()
            _, token, dz = ext().distill_loss_parts(z, top_logp[s:e], top_idx[s:e], weights[s:e], 1.0 / temperature, beta, tail,
                                                        need_h or need_w, fused, False)
            tokens.append(token)
            del z
            if need_h and fused:
                _lin.gemm(dz, weight, b_mn=True, out=dh[s:e])
            elif need_h:
                dh[s:e] = dz @ weight.float()
            if need_w and once:
                dw = _lin.gemm(dz, h, a_mn=True, b_mn=True, split_k=0)
            elif need_w and fused:
                _lin.gemm(dz, h[s:e], a_mn=True, b_mn=True, out_f32=dw, accumulate=True)
            elif need_w:
                dw.addmm_(dz.t(), h[s:e].float())
            del dz
        token = tokens[0] if len(tokens) == 1 else torch.cat(tokens) if tokens else h.new_empty(0, dtype=torch.float32)
        _count()
        loss = ext().weighted_sum(token, weights)
        ctx.save_for_backward(dh, None if dw is None else dw.to(weight.dtype))
        ctx.capture = ext().capture_id()
        ctx.mark_non_differentiable(token)
        return loss, token

    @staticmethod
    def backward(ctx, g_loss, _g_token):
        dh, dw = ctx.saved_tensors
        _count((dh is not None) + (dw is not None))
        return tuple(None if x is None else ext().scaled(x, g_loss, ctx.capture) for x in (dh, dw)) + (None,) * 8


def lmhead_distill_loss(hidden, weight, top_logp, top_idx, weights, temperature, beta, tail):
    top_logp, top_idx, weights = ext().teacher_entries(top_logp, top_idx, weights, weight.shape[0])
    grad = torch.is_grad_enabled()
    return _LmHeadDistillFn.apply(hidden, weight, top_logp, top_idx, weights, temperature, beta, tail, grad and hidden.requires_grad,
                                  grad and weight.requires_grad)


@torch.no_grad()
def lmhead_top_logprobs(hidden, weight, k, temperature):
    from . import gemm as _lin
    rows, V = hidden.shape[0], weight.shape[0]
    logp = torch.empty(rows, k, dtype=torch.float32, device=hidden.device)
    idx = torch.empty(rows, k, dtype=torch.int32, device=hidden.device)
    h = hidden.contiguous()
    for s, e in _row_ranges(rows, V):
        z = _head_logits(h[s:e], weight, _lin.supported(h, weight))
        logp[s:e], idx[s:e] = top_logprobs(z, k, temperature)
        del z
    return logp, idx


# --------------------------------------------------------------------------------------------
# RL kernels
# --------------------------------------------------------------------------------------------
def gae_scan(rewards, values, gamma, lam):
    _count()
    adv, ret = ext().gae_scan(rewards.float().contiguous(), None if values is None else values.float().contiguous(),
                              float(gamma), float(lam))
    return adv, ret


def _count_loss(x):
    _count(2 if x.requires_grad and torch.is_grad_enabled() else 1)          # forward and, later, backward


class _RecordedLossFn(torch.autograd.Function):
    """A loss in a form that a tracer records as one operation; it does not see autograd functions in C++ and would keep their results as constants."""

    @staticmethod
    def forward(ctx, parts, x, *rest):
        loss, grad, stats = parts(x.contiguous(), *[t.contiguous() if torch.is_tensor(t) else t for t in rest])
        ctx.save_for_backward(grad, stats[0].clone())
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    def backward(ctx, g_loss, _g_stats):
        grad, denom = ctx.saved_tensors
        return (None, grad * (g_loss / denom)) + (None,) * (len(ctx.needs_input_grad) - 2)


def _loss(name, x, *rest):
    _count_loss(x)
    if torch._C._get_tracing_state():
        loss, stats = _RecordedLossFn.apply(getattr(ext(), name + "_parts"), x.float(), *[t.float() if torch.is_tensor(t) and t.is_floating_point() else t for t in rest])
        return loss, stats.unbind()
    return getattr(ext(), name)(x, *rest)


def policy_loss_token(new_logp, old_logp, adv, mask, cliprange, ref_logp=None, kl_coef=0.0):
    loss, stats = _loss("policy_loss", new_logp, old_logp, adv, mask, ref_logp, float(cliprange), float(kl_coef))
    _, clipfrac, kl_masked, kl_all, ratio_all, ratio_masked, ref_all, ref_masked = stats
    out = {"clipfrac": clipfrac, "approxkl_masked": kl_masked, "approxkl_all": kl_all, "ratio_mean_all": ratio_all,
           "ratio_mean_masked": ratio_masked}
    if ref_logp is not None:
        out["refkl_all"], out["refkl_masked"] = ref_all, ref_masked
    return loss, out


def value_loss(vpred, values_old, returns, mask, cliprange_value):
    loss, stats = _loss("value_loss", vpred, values_old, returns, mask, float(cliprange_value))
    return loss, stats[1]


def adamw_flat(param, grad, m, v, lr, beta1, beta2, eps, wd, step, scale=1.0, master=None):
    _count()
    ext().adamw_flat(param, grad, m, v, lr, beta1, beta2, eps, wd, step, scale, master)


# --------------------------------------------------------------------------------------------
# sampler kernels
# --------------------------------------------------------------------------------------------
def sample(logits, temperature, top_p, seed, step, row_ids=None, row_steps=None, out=None, impl=0):
    _count()
    return ext().sample(logits, float(temperature), float(top_p), int(seed), int(step), row_ids, row_steps, out, int(impl))


def row_uniforms(seed, step, row_ids, row_steps=None):
    """float32 [rows] in [0, 1), functions of (seed, row_ids[i], step + row_steps[i]) alone."""
    _count()
    return ext().row_uniforms(int(seed), int(step), row_ids, row_steps)


@torch.no_grad()
def sample_filtered(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    _count()
    args = []
    for x, off in ((temperature, 1.0), (top_k, 0), (top_p, 1.0), (min_p, 0.0)):
        each = torch.is_tensor(x) and x.dim() > 0
        args += [x.contiguous(), off] if each else [None, type(off)(x)]
    return ext().sample_filtered(_row_major(logits), uniforms.contiguous(), *args)


def sample_tokens(logits, temperature, top_p, seed, row_ids, row_steps, top_k=0, min_p=0.0):
    """A token per row for the rollout engines, a function of (seed, row id, tokens generated): ``sample``, or with ``top_k`` / ``min_p`` ``sample_filtered``
    of one uniform number per row.  A row without a finite logit gives token 0."""
    if temperature == 0.0 or (top_k <= 0 and min_p <= 0.0):
        return sample(logits, temperature, top_p, seed, 0, row_ids, row_steps)
    tokens, _ = sample_filtered(logits, row_uniforms(seed, 0, row_ids, row_steps), float(temperature), int(top_k), float(top_p), float(min_p))
    return tokens.clamp_(min=0)


def kv_cache_write(k, v, k_cache, v_cache, slot_mapping, src_index=None):
    _count()
    ext().kv_cache_write(k, v, k_cache, v_cache, slot_mapping, src_index)


def paged_decode(q, k_cache, v_cache, block_tables, context_lens, scale=None, splits=1, out=None):
    _count()
    scale = scale if scale is not None else 1.0 / math.sqrt(q.shape[-1])
    return ext().paged_decode(q, k_cache, v_cache, block_tables, context_lens, float(scale), int(splits), out)


# --------------------------------------------------------------------------------------------
# many samples of one prompt, and a cache of bounded size
# --------------------------------------------------------------------------------------------
class _RecordedSharedPrefixFn(torch.autograd.Function):
    """The attention in a form that a tracer records as one operation (see ``_RecordedLossFn``)."""

    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, cu_groups, scale):
        o, rest, lse, table = ext().attn_groups_fwd(q, k, v, cu_seqlens, cu_groups, scale, True)
        ctx.save_for_backward(q, k, v, o, rest, lse, cu_seqlens, table)
        ctx.scale = scale
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        return (*ext().attn_groups_bwd(do, *ctx.saved_tensors, ctx.scale), None, None, None)


def attention_shared_prefix(q, k, v, cu_seqlens, cu_groups, scale):
    _count(4 if torch.is_grad_enabled() and q.requires_grad else 2)          # forward and, later, backward
    if torch._C._get_tracing_state():
        return _RecordedSharedPrefixFn.apply(*ext().attn_groups_arguments(q, k, v, cu_seqlens, cu_groups, scale))
    return ext().attention_shared_prefix(q, k, v, cu_seqlens, cu_groups, scale)


def paged_decode_shared(*args):
    _count(2)                                    # (a third one makes the plan of many rows)
    return ext().paged_decode_shared(*args)


def paged_decode_scored(*args):
    _count(2)
    return ext().paged_decode_scored(*args)


def kv_evict(*args):
    _count(2)
    return ext().kv_evict(*args)
