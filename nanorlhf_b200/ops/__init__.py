"""Op layer: every hot op of the engine behind one name, two backends.

* ``torch``  -- pure PyTorch (ops/reference.py): CPU plumbing backend and test oracle.
* ``cuda``   -- hand-written sm_100a kernels from ``nanorlhf_b200/csrc`` (ops/native.py).

On a CUDA tensor the native extension is *mandatory* unless ``NANORLHF_BACKEND=torch`` is set
explicitly: a missing ``.so`` raises instead of silently falling back (the round-end driver
records which ``.so`` files were loaded).
"""
from __future__ import annotations

import os

import torch

from . import reference as ref

_FORCED = os.environ.get("NANORLHF_BACKEND", "").lower()
_native = None
_native_err = None


def _nat():
    """Return the loaded native extension module, raising a clear error if it is unavailable."""
    global _native, _native_err
    if _native is None and _native_err is None:
        try:
            from . import native as _n
            _n.load()
            _native = _n
        except Exception as e:  # pragma: no cover - exercised on boxes without the build
            _native_err = e
    if _native is None:
        raise RuntimeError(
            "nanorlhf_b200 native extension is not available "
            f"({_native_err!r}). Build it with `python -m nanorlhf_b200.csrc.build` "
            "or set NANORLHF_BACKEND=torch to run the PyTorch reference ops.")
    return _native


def use_native(t: torch.Tensor) -> bool:
    if _FORCED == "torch":
        return False
    return t.is_cuda


def direct_calls() -> bool:
    """A kernel may be called without an autograd function around it: autograd is off and nothing traces or transforms the program.  A trace would
    keep such a call's result as a constant and forward-mode would lose the tangent, where the function is recorded or refuses."""
    return not (torch.is_grad_enabled() or torch._C._get_tracing_state() or torch._C._are_functorch_transforms_active()
                or torch.autograd.forward_ad._current_level >= 0)


def backend_name(t: torch.Tensor) -> str:
    return "cuda" if use_native(t) else "torch"


# ---- thin dispatchers (autograd-aware wrappers live in ops/native.py) -----------------------
def rmsnorm(x, weight, eps):
    if use_native(x):
        return _nat().rmsnorm(x, weight, eps)
    return ref.rmsnorm(x, weight, eps)


def add_rmsnorm(x, residual, weight, eps):
    if use_native(x):
        return _nat().add_rmsnorm(x, residual, weight, eps)
    return ref.add_rmsnorm(x, residual, weight, eps)


def apply_rope(x, cos, sin):
    if use_native(x):
        return _nat().apply_rope(x, cos, sin)
    return ref.apply_rope(x, cos, sin)


def swiglu(gate_up):
    if use_native(gate_up):
        return _nat().swiglu(gate_up)
    return ref.swiglu(gate_up)


def swiglu_pair(gate, up):
    """silu(gate) * up without concatenating the two projections."""
    if use_native(gate):
        return _nat().swiglu_pair(gate, up)
    return (torch.nn.functional.silu(gate.float()) * up.float()).to(gate.dtype)


def linear(x, weight, bias=None, act: int = 0):
    """``F.linear`` (+ optional fused exact GELU, ``act=1``) -- the general tcgen05 GEMM on CUDA bf16 (ops/gemm.py)."""
    if use_native(x):
        _nat()
        from . import gemm as _lin
        return _lin.linear(x, weight, bias, act)
    y = torch.nn.functional.linear(x, weight, bias)
    return torch.nn.functional.gelu(y) if act == 1 else y


def lora_linear(x, weight, bias, lora_a, lora_b, scaling: float):
    """``x W^T + b + scaling * (x A^T) B^T`` with a frozen ``W``; one dual-source-K GEMM per direction on CUDA bf16."""
    if use_native(x):
        _nat()
        from . import gemm as _lin
        if _lin.lora_supported(x, weight, lora_a, lora_b):
            return _lin.lora_linear(x, weight, bias, lora_a, lora_b, scaling)
    return ref.lora_linear(x, weight, bias, lora_a, lora_b, scaling)


def lora_linear_group(x, projs, scaling: float):
    """LoRA projections that share their input (q/k/v, gate/up): ``projs`` = [(W, bias, A, B), ...] -> list of outputs.
    One rank-r launch for all adapters on CUDA bf16 (ops/gemm.py); independent ``lora_linear`` calls elsewhere."""
    if use_native(x):
        _nat()
        from . import gemm as _lin
        if all(_lin.lora_supported(x, w, a, b) for w, _bias, a, b in projs) and len({a.shape[0] for _w, _b, a, _B in projs}) == 1:
            return _lin.lora_linear_group(x, projs, scaling)
    return [lora_linear(x, w, bias, a, b, scaling) for w, bias, a, b in projs]


def attention_varlen(q, k, v, cu_seqlens, max_seqlen=None, causal=True, scale=None):
    if use_native(q):
        return _nat().attention_varlen(q, k, v, cu_seqlens, max_seqlen, causal, scale)
    return ref.attention_varlen(q, k, v, cu_seqlens, causal=causal, scale=scale)


def lmhead_logprob(hidden, weight, targets, temperature=1.0, want_entropy=True):
    """Autograd-capable fused lm-head log-prob.  Returns (logp, entropy) both fp32 [T]."""
    if use_native(hidden):
        return _nat().lmhead_logprob(hidden, weight, targets, temperature, want_entropy)
    return _LmHeadLogprobTorch.apply(hidden, weight, targets, float(temperature), bool(want_entropy))


class _LmHeadLogprobTorch(torch.autograd.Function):
    """Chunked, recompute-in-backward log-prob head on the PyTorch backend."""

    @staticmethod
    def forward(ctx, hidden, weight, targets, temperature, want_entropy):
        logp, ent, lse = ref.lmhead_logprob(hidden, weight, targets, temperature, want_entropy=want_entropy)
        ctx.save_for_backward(hidden, weight, targets, lse)
        ctx.temperature = temperature
        ctx.mark_non_differentiable(ent)
        return logp, ent

    @staticmethod
    def backward(ctx, g_logp, _g_ent):
        hidden, weight, targets, lse = ctx.saved_tensors
        dh, dw = ref.lmhead_logprob_backward(hidden, weight, targets, lse, g_logp, ctx.temperature,
                                             need_weight_grad=ctx.needs_input_grad[1])
        return dh if ctx.needs_input_grad[0] else None, dw, None, None, None


# ---- a distribution over the vocabulary that another model gives, or that a sampler cuts -------------------------------------
def _check_temperature(what, temperature):
    if not 0.0 < float(temperature) < float("inf"):
        raise ValueError(f"{what}: temperature must be positive and finite, got {temperature}")


def top_logprobs(logits, k: int, temperature: float = 1.0):
    """Log-probabilities of the ``k`` most probable tokens of every row of ``logits`` [T, V] (bf16 or float32) under softmax(logits / temperature):
    (logp float32 [T, k], idx int32 [T, k]), most probable first, ties by the lower index.  Tokens without mass (logit -inf) are not listed: idx -1,
    logp -inf in their places.  1 <= k <= min(V, 1024).  No gradient; a row with a NaN has NaN log-probabilities."""
    _check_temperature("top_logprobs", temperature)
    if logits.dim() != 2 or not 1 <= int(k) <= min(logits.shape[1], 1024):
        raise ValueError(f"top_logprobs: logits [T, V] and 1 <= k <= min(V, 1024) are needed, got {tuple(logits.shape)} and k = {k}")
    if use_native(logits):
        return _nat().top_logprobs(logits, int(k), float(temperature))
    return ref.top_logprobs(logits, int(k), float(temperature))


def _check_teacher(what, rows, top_logp, top_idx, weights, temperature, beta, tail):
    _check_temperature(what, temperature)
    if top_logp.dim() != 2 or top_logp.shape != top_idx.shape or top_logp.shape[0] != rows or not 1 <= top_logp.shape[1] <= 1024:
        raise ValueError(f"{what}: top_logp and top_idx must be [{rows}, K] with 1 <= K <= 1024, got {tuple(top_logp.shape)} and {tuple(top_idx.shape)}")
    if top_idx.dtype not in (torch.int32, torch.int64) or not top_logp.is_floating_point():
        raise TypeError(f"{what}: top_logp must be a floating-point tensor and top_idx int32 or int64")
    if weights is not None and tuple(weights.shape) != (rows,):
        raise ValueError(f"{what}: weights must be [{rows}], got {tuple(weights.shape)}")
    if not 0.0 <= beta <= 1.0:
        raise ValueError(f"{what}: beta must be between 0 and 1, got {beta}")
    if not tail and beta != 0.0:
        raise ValueError(f"{what}: tail=False goes with beta = 0 only")


def distill_loss(logits, top_logp, top_idx, weights=None, temperature: float = 1.0, beta: float = 0.0, tail: bool = True):
    """Divergence of a student, ``logits`` [T, V], from a teacher of whom the log-probabilities ``top_logp`` of ``top_idx`` [T, K] are known
    (``top_logprobs``): (sum_t weights[t] * loss_t, loss_t float32 [T]).  The first has a gradient with respect to ``logits``, the second none.

    With q = softmax(logits / temperature), P and Q are the teacher's and the student's probabilities of the K tokens and of *all others together*:
    beta = 0: KL(P | Q); beta = 1: KL(Q | P); between: beta KL(P | M) + (1 - beta) KL(Q | M), M = beta P + (1 - beta) Q.  ``tail=False`` (beta = 0) scales
    the teacher's K probabilities to a sum of 1 instead, and compares them with q as it is.
    ``weights`` [T]: share of every token (a mask over its sum; None: 1 / T each); a row of weight 0 is not read, its loss and gradient are 0.  Put constant
    factors (gradient accumulation) in there: the gradient is formed in the forward, and a backward from 1 hands it on as it is.  A row with a NaN or +inf, or
    a token of the teacher's with a NaN, has NaN for its loss and no gradient that is a number.
    Entries of ``top_idx`` outside [0, V) are skipped, entries of one token add up; no entries and a tail: loss 0.  What the teacher leaves of 1 counts as 0 below
    2^-24, and below 2^-20 where the student gives all other tokens less than e^-745 of its best (with more than that, KL(P | Q) is infinite where it gives them nothing).  V <= 2^20 on CUDA, where a second derivative is refused."""
    if logits.dim() != 2:
        raise ValueError(f"distill_loss: logits must be [T, V], got {tuple(logits.shape)}")
    _check_teacher("distill_loss", logits.shape[0], top_logp, top_idx, weights, temperature, float(beta), tail)
    if use_native(logits):
        return _nat().distill_loss(logits, top_logp, top_idx, weights, float(temperature), float(beta), bool(tail))
    return ref.distill_loss(logits, top_logp, top_idx, weights, float(temperature), float(beta), bool(tail))


def lmhead_distill_loss(hidden, weight, top_logp, top_idx, weights=None, temperature: float = 1.0, beta: float = 0.0, tail: bool = True):
    """``distill_loss`` of the logits ``hidden @ weight.T`` ([T, H], [V, H], bf16), which are formed in float32 and never handed over; gradients with
    respect to ``hidden`` and ``weight``, formed in the forward.  T may be any: at most 4 GiB of logits and half as much of their gradients are held at a time.  Other types,
    and sizes that are no multiples of 8, are multiplied by torch in float32."""
    if hidden.dim() != 2 or weight.dim() != 2 or hidden.shape[1] != weight.shape[1]:
        raise ValueError(f"lmhead_distill_loss: hidden [T, H] and weight [V, H] are needed, got {tuple(hidden.shape)} and {tuple(weight.shape)}")
    _check_teacher("lmhead_distill_loss", hidden.shape[0], top_logp, top_idx, weights, temperature, float(beta), tail)
    if use_native(hidden):
        return _nat().lmhead_distill_loss(hidden, weight, top_logp, top_idx, weights, float(temperature), float(beta), bool(tail))
    return ref.distill_loss(hidden @ weight.t(), top_logp, top_idx, weights, float(temperature), float(beta), bool(tail))


def lmhead_top_logprobs(hidden, weight, k: int, temperature: float = 1.0):
    """``top_logprobs`` of the logits ``hidden @ weight.T``, which are formed in float32 (bf16 on CUDA) a few thousand rows at a time.  No gradient."""
    if hidden.dim() != 2 or weight.dim() != 2 or hidden.shape[1] != weight.shape[1]:
        raise ValueError(f"lmhead_top_logprobs: hidden [T, H] and weight [V, H] are needed, got {tuple(hidden.shape)} and {tuple(weight.shape)}")
    _check_temperature("lmhead_top_logprobs", temperature)
    if not 1 <= int(k) <= min(weight.shape[0], 1024):
        raise ValueError(f"lmhead_top_logprobs: 1 <= k <= min(V, 1024) is needed, got {k}")
    if use_native(hidden):
        return _nat().lmhead_top_logprobs(hidden, weight, int(k), float(temperature))
    with torch.no_grad():
        return ref.top_logprobs(hidden @ weight.t(), int(k), float(temperature))


def sample_filtered(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token per row of ``logits`` [B, V] (bf16 or float32) from given random numbers: (tokens int32 [B], logp float32 [B]).

    With w = exp((logit - largest) / temperature): tokens with w >= ``min_p`` are kept, of those the ``top_k`` first (largest logit first, ties by the lower
    index), of those the fewest first whose mass is at least ``top_p`` of theirs.  The token is the first kept one, by index, up to which the kept mass
    exceeds ``uniforms`` (float32 [B], in [0, 1)) times the whole; ``logp`` is its log-probability among the kept.  Masses are float64, so that the result is
    that of the definition.  Every filter is a number or a tensor [B] (float32; ``top_k`` int32); 0 / 1 / 0 leave top_k / top_p / min_p out, temperature 0
    takes the first token of the order (logp 0).  In tensors a value beyond its range counts as the nearest in it, NaN as left out (temperature: as 0).  Masses below
    e^-690 of the largest logit's may count as none.  NaN logits count as -inf; a row of nothing else has token -1, logp -inf."""
    if logits.dim() != 2 or tuple(uniforms.shape) != (logits.shape[0],):
        raise ValueError(f"sample_filtered: logits [B, V] and uniforms [B] are needed, got {tuple(logits.shape)} and {tuple(uniforms.shape)}")
    if uniforms.dtype != torch.float32:
        raise TypeError(f"sample_filtered: uniforms must be float32, got {uniforms.dtype}")
    for name, x, hi in (("temperature", temperature, float("inf")), ("top_k", top_k, float("inf")), ("top_p", top_p, 1.0), ("min_p", min_p, 1.0)):
        if torch.is_tensor(x) and x.dim() > 0:
            want = torch.int32 if name == "top_k" else torch.float32
            if tuple(x.shape) != (logits.shape[0],) or x.dtype != want:
                raise ValueError(f"sample_filtered: {name} must be a number or a {want} tensor [{logits.shape[0]}], got {x.dtype} {tuple(x.shape)}")
        elif not 0 <= x <= hi or x == float("inf") or (name == "top_k" and x != int(x)):
            raise ValueError(f"sample_filtered: {name} is out of range: {x}")
    if use_native(logits):
        return _nat().sample_filtered(logits, uniforms, temperature, top_k, top_p, min_p)
    return ref.sample_filtered(logits, uniforms, temperature, top_k, top_p, min_p)


def discounted_suffix_sum(rewards, gamma=1.0):
    if use_native(rewards):
        return _nat().gae_scan(rewards, None, gamma, 1.0)[0]
    return ref.discounted_suffix_sum(rewards, gamma)


def gae(rewards, values, gamma, lam):
    if use_native(rewards):
        return _nat().gae_scan(rewards, values, gamma, lam)
    return ref.gae(rewards, values, gamma, lam)


def policy_loss_token(new_logp, old_logp, adv, mask, cliprange, ref_logp=None, kl_coef=0.0):
    if use_native(new_logp):
        return _nat().policy_loss_token(new_logp, old_logp, adv, mask, cliprange, ref_logp, kl_coef)
    return ref.policy_loss_token(new_logp, old_logp, adv, mask, cliprange, ref_logp, kl_coef)


policy_loss_sequence = ref.policy_loss_sequence   # [B]-sized math; not a hot path
nll_loss = ref.nll_loss


def value_loss(vpred, values_old, returns, mask, cliprange_value):
    if use_native(vpred):
        return _nat().value_loss(vpred, values_old, returns, mask, cliprange_value)
    return ref.value_loss(vpred, values_old, returns, mask, cliprange_value)
