// Tensors in, launches out: attention over shared prefixes, decode attention with scores, eviction.
#include "bindings_groups.h"

#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <tuple>

#include "group_kernels.h"
#include "kernels.h"
#include "tma_host.h"

namespace {

inline cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }
inline void check(cudaError_t e, const char* what) { TORCH_CHECK(e == cudaSuccess, what, ": ", cudaGetErrorString(e)); }
inline int num_sms() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }
constexpr int64_t kIntMax = std::numeric_limits<int>::max();

// What is wrong with an argument raises what the checks of the CPU forms (ops/__init__.py) raise: ValueError for shapes and ranges, TypeError for types and devices.
void check_ints(const torch::Tensor& t, const torch::Tensor& beside, const char* what, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == torch::kInt32 && t.device() == beside.device(), what, ": ", name, " must be int32 on ", beside.device(), ", got ", t.scalar_type(),
                   " on ", t.device());
}
double scale_of(const c10::optional<double>& scale, const char* what) {
  TORCH_CHECK_VALUE(!scale.has_value() || std::isfinite(*scale), what, ": scale must be finite, got ", *scale);
  return scale.value_or(0.08838834764831845);                         // 1 / sqrt(128)
}
// A copy where the first element is not on 16 bytes: `contiguous` leaves a contiguous slice of a buffer where it is
torch::Tensor on_16(const torch::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone(at::MemoryFormat::Contiguous); }
// [rows, heads, 128] whose heads lie side by side and whose rows start on 16 bytes: a view of a projection stays one, rows that are one row repeated do not
torch::Tensor head_rows(const torch::Tensor& t) {
  if (t.numel() == 0) return t;
  const bool laid = t.stride(2) == 1 && (t.stride(1) == 128 || t.size(1) == 1) && (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) > 0));
  return on_16(laid ? t : t.contiguous());
}
int64_t row_stride(const torch::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1) * 128; }

// ---- packed groups ---------------------------------------------------------------------------------------------------------------------
void check_packed(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& cu_seqlens, const torch::Tensor& cu_groups,
                  const char* what) {
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(2) == q.size(2) && k.size(1) > 0 &&
                    q.size(1) % k.size(1) == 0, what, ": q [T, Hq, D] and k, v [T, Hkv, D] with Hq a multiple of Hkv are needed, got ", q.sizes(), ", ", k.sizes(), ", ",
                    v.sizes());
  TORCH_CHECK_TYPE(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type() && k.device() == q.device() && v.device() == q.device(), what,
                   ": q, k and v must have one type and device");
  TORCH_CHECK_VALUE(cu_seqlens.dim() == 1 && cu_groups.dim() == 1 && cu_seqlens.numel() >= 1 && cu_groups.numel() >= 1, what,
                    ": cu_seqlens [sequences + 1] and cu_groups [groups + 1] are needed, got ", cu_seqlens.sizes(), " and ", cu_groups.sizes());
  check_ints(cu_seqlens, q, what, "cu_seqlens");
  check_ints(cu_groups, q, what, "cu_groups");
  TORCH_CHECK_TYPE(q.is_cuda() && q.scalar_type() == torch::kBFloat16 && q.size(2) == 128, what, ": on CUDA bf16 and a head size of 128 are needed, got ", q.scalar_type(),
                   " and ", q.size(2));
  TORCH_CHECK_VALUE(q.size(0) * q.size(1) <= kIntMax, what, ": too many rows");
  // the kernels would leave a tangent behind, whether autograd records or not
  for (const torch::Tensor* t : {&q, &k, &v})
    TORCH_CHECK(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t->_fw_grad(0).defined(), what, ": there is no forward-mode derivative");
}
CUtensorMap map_of(const torch::Tensor& t, int box_rows) {
  return nrl::make_tma_2d(t.data_ptr(), t.size(0), static_cast<uint64_t>(t.size(1)) * 128, row_stride(t) * 2, box_rows, 64, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2);
}

// (out, what bf16 had no room for of it, lse [Hq, T], table of the sequences: for the backward, without which the second is not formed); q, k, v as head_rows gives them
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> attn_groups_fwd(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                                                                        const torch::Tensor& cu_seqlens, const torch::Tensor& cu_groups, double scale, bool train) {
  const char* what = "attention_shared_prefix";
  c10::cuda::CUDAGuard guard(q.device());
  const int T = q.size(0), Hq = q.size(1), Hkv = k.size(1), n = cu_seqlens.numel() - 1;
  torch::Tensor out = torch::empty({T, Hq, 128}, q.options()), lse = torch::empty({Hq, T}, q.options().dtype(torch::kFloat32));
  torch::Tensor table = torch::empty({n, 8}, cu_seqlens.options()), rest = train ? torch::empty({T, Hq, 128}, q.options().dtype(torch::kUInt8)) : torch::Tensor();
  if (T == 0) return {out, rest, lse, table};
  const CUtensorMap mq = map_of(q, 128), mk = map_of(k, 128), mv = map_of(v, 128);
  check(nrl_attn_group_table(cu_seqlens.data_ptr<int>(), cu_groups.data_ptr<int>(), table.data_ptr<int>(), n, cu_groups.numel() - 1, out.data_ptr(), T, Hq, cur_stream()),
        what);
  check(nrl_attn_groups_fwd_tc(&mq, &mk, &mv, out.data_ptr(), train ? rest.data_ptr() : nullptr, lse.data_ptr<float>(), out.stride(0), cu_seqlens.data_ptr<int>(), table.data_ptr<int>(), n, T, Hq, Hkv,
                               static_cast<float>(scale), num_sms(), cur_stream()), what);
  return {out, rest, lse, table};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> attn_groups_bwd(const torch::Tensor& grad, const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                                                                        const torch::Tensor& o, const torch::Tensor& rest, const torch::Tensor& lse,
                                                                        const torch::Tensor& cu_seqlens, const torch::Tensor& table, double scale) {
  const char* what = "attention_shared_prefix backward";
  const torch::Tensor dout = on_16(grad.contiguous());
  TORCH_CHECK(dout.sizes() == o.sizes() && dout.device() == q.device() && dout.scalar_type() == torch::kBFloat16, what, ": the gradient must be like the result");
  c10::cuda::CUDAGuard guard(q.device());
  const int T = q.size(0), Hq = q.size(1), Hkv = k.size(1), n = cu_seqlens.numel() - 1;
  torch::Tensor dq = torch::empty({T, Hq, 128}, q.options()), dk = torch::empty({T, Hkv, 128}, q.options()), dv = torch::empty({T, Hkv, 128}, q.options());
  if (T == 0) return {dq, dk, dv};
  torch::Tensor delta = torch::empty({Hq, T}, q.options().dtype(torch::kFloat32));
  const CUtensorMap maps[8] = {map_of(q, 64), map_of(dout, 64), map_of(k, 128), map_of(v, 128), map_of(q, 128), map_of(dout, 128), map_of(k, 64), map_of(v, 64)};
  check(nrl_attn_groups_bwd_tc(maps, o.data_ptr(), rest.data_ptr(), dout.data_ptr(), lse.data_ptr<float>(), delta.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                               o.stride(0), dq.stride(0), dk.stride(0), cu_seqlens.data_ptr<int>(), table.data_ptr<int>(), n, T, Hq, Hkv, static_cast<float>(scale),
                               cur_stream()), what);
  return {dq, dk, dv};
}

// A gradient of the running backward, where it may be differentiated again: refused, the kernels have no second derivative
torch::Tensor refuse_second(const torch::Tensor& grad) {
  const auto node = torch::autograd::get_current_node();
  if (!at::GradMode::is_enabled() || !node) return grad;
  torch::Tensor out = grad.detach();
  torch::autograd::edge_list inputs = node->next_edges();
  torch::autograd::create_gradient_edge(out, std::make_shared<torch::autograd::Error>("attention_shared_prefix: there is no second derivative", std::move(inputs)));
  return out;
}

// In C++, as the losses: of four samples of 65 tokens the kernels take 35 us and a Python function 110.
struct AttnGroupsFn : torch::autograd::Function<AttnGroupsFn> {
  static torch::Tensor forward(torch::autograd::AutogradContext* ctx, torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor cu_seqlens, torch::Tensor cu_groups,
                               double scale) {
    auto [out, rest, lse, table] = attn_groups_fwd(q, k, v, cu_seqlens, cu_groups, scale, true);
    ctx->save_for_backward({q, k, v, out, rest, lse, cu_seqlens, table});
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    const auto s = ctx->get_saved_variables();
    auto [dq, dk, dv] = attn_groups_bwd(g[0], s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], ctx->saved_data["scale"].toDouble());
    return {refuse_second(dq), refuse_second(dk), refuse_second(dv), {}, {}, {}};
  }
};

// q, k, v, cu_seqlens and cu_groups as the kernels take them, and the scale
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, double> packed_arguments(const torch::Tensor& q, const torch::Tensor& k,
                                                                                                               const torch::Tensor& v, const torch::Tensor& cu_seqlens,
                                                                                                               const torch::Tensor& cu_groups,
                                                                                                               const c10::optional<double>& scale) {
  const char* what = "attention_shared_prefix";
  check_packed(q, k, v, cu_seqlens, cu_groups, what);
  // masked scores are -inf in front of the scale: times 0 or less they would not stay it
  const double by = scale_of(scale, what);
  TORCH_CHECK_VALUE(by >= 1e-37 && by <= 1e37, what, ": scale must be positive, from 1e-37 to 1e37, got ", by);
  return {head_rows(q), head_rows(k), head_rows(v), cu_seqlens.contiguous(), cu_groups.contiguous(), by};
}
torch::Tensor attention_shared_prefix(const torch::Tensor& q_in, const torch::Tensor& k_in, const torch::Tensor& v_in, const torch::Tensor& cu_seqlens_in,
                                      const torch::Tensor& cu_groups_in, const c10::optional<double>& scale_in) {
  auto [q, k, v, cu_seqlens, cu_groups, scale] = packed_arguments(q_in, k_in, v_in, cu_seqlens_in, cu_groups_in, scale_in);
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad())) return AttnGroupsFn::apply(q, k, v, cu_seqlens, cu_groups, scale);
  return std::get<0>(attn_groups_fwd(q, k, v, cu_seqlens, cu_groups, scale, false));
}

// ---- pages -----------------------------------------------------------------------------------------------------------------------------
// k, v: bf16 [blocks, Hkv, 16, 128]; or uint8 (e4m3) of as many elements, values transposed, with scales [blocks, Hkv, 16]
void check_pages(const torch::Tensor& k, const torch::Tensor& v, const c10::optional<torch::Tensor>& ks, const c10::optional<torch::Tensor>& vs,
                 const torch::Tensor& tables, const torch::Tensor& context, const char* what) {
  TORCH_CHECK_VALUE(k.dim() == 4 && v.dim() == 4 && k.size(0) == v.size(0) && k.size(1) == v.size(1) && k.size(2) == 16 && k.size(3) == 128 && k.numel() == v.numel() &&
                    k.size(1) > 0, what, ": k_cache and v_cache must be [blocks, Hkv, 16, 128], got ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK_VALUE(ks.has_value() == vs.has_value(), what, ": k_scale and v_scale go together");
  TORCH_CHECK_TYPE(k.scalar_type() == v.scalar_type() && k.scalar_type() == (ks.has_value() ? torch::kUInt8 : torch::kBFloat16), what,
                   ": pages are bf16, or uint8 (e4m3) with scales, got ", k.scalar_type(), " and ", v.scalar_type());
  TORCH_CHECK_VALUE(k.is_contiguous() && v.is_contiguous() && reinterpret_cast<uintptr_t>(k.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(v.data_ptr()) % 16 == 0,
                    what, ": pages must be contiguous and start on 16 bytes");
  TORCH_CHECK_TYPE(k.is_cuda() && v.device() == k.device(), what, ": k_cache and v_cache must be on one device");
  for (const c10::optional<torch::Tensor>* s : {&ks, &vs}) {
    if (!s->has_value()) continue;
    TORCH_CHECK_VALUE((*s)->scalar_type() == torch::kFloat32 && (*s)->sizes() == k.sizes().slice(0, 3), what, ": scales must be float32 ", k.sizes().slice(0, 3), ", got ",
                      (*s)->scalar_type(), " ", (*s)->sizes());
    TORCH_CHECK_VALUE((*s)->device() == k.device() && (*s)->is_contiguous() && reinterpret_cast<uintptr_t>((*s)->data_ptr()) % 16 == 0, what,
                      ": scales must be contiguous, beside the pages and start on 16 bytes");
  }
  TORCH_CHECK_VALUE(context.dim() == 1 && tables.dim() == 2 && tables.size(0) == context.size(0) && tables.size(1) >= 1, what,
                    ": block_tables [rows, pages] and context_lens [rows] are needed, got ", tables.sizes(), " and ", context.sizes());
  check_ints(tables, k, what, "block_tables");
  check_ints(context, k, what, "context_lens");
  TORCH_CHECK_VALUE(tables.size(0) * tables.size(1) * k.size(1) <= kIntMax / 16 && tables.size(0) * k.size(1) <= kIntMax / 64 && tables.size(1) <= kIntMax / 512 && k.size(1) <= 256, what, ": too many rows, pages or heads");
}

// a decode call's arguments, its result and its scratch
struct Decode {
  torch::Tensor q, tables, context, out, scratch;
  nrl::DecodeCall c;
  Decode(const torch::Tensor& q_in, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& tables_in, const torch::Tensor& context_in,
         const c10::optional<torch::Tensor>& ks, const c10::optional<torch::Tensor>& vs, const c10::optional<double>& scale, const char* what) {
    check_pages(k, v, ks, vs, tables_in, context_in, what);
    const int64_t S = context_in.size(0), Hkv = k.size(1);
    TORCH_CHECK_VALUE(q_in.dim() == 3 && q_in.size(0) == S && q_in.size(2) == 128 && q_in.size(1) % Hkv == 0 && q_in.size(1) / Hkv <= 8, what, ": q must be [", S,
                      ", Hq, 128] with Hq a multiple, at most 8 times, of ", Hkv, ", got ", q_in.sizes());
    TORCH_CHECK_TYPE(q_in.scalar_type() == torch::kBFloat16 && q_in.device() == k.device(), what, ": q must be bf16 on ", k.device(), ", got ", q_in.scalar_type(), " on ",
                     q_in.device());
    q = head_rows(q_in);
    tables = tables_in.contiguous();
    context = context_in.contiguous();
    out = torch::empty({S, q.size(1), 128}, q.options());
    c.q = q.data_ptr();
    c.q_stride_s = row_stride(q);
    c.k_cache = k.data_ptr();
    c.v_cache = v.data_ptr();
    c.k_scale = ks.has_value() ? ks->data_ptr<float>() : nullptr;
    c.v_scale = vs.has_value() ? vs->data_ptr<float>() : nullptr;
    c.block_tables = tables.data_ptr<int>();
    c.context_lens = context.data_ptr<int>();
    c.out = out.data_ptr();
    c.S = S; c.Hq = q.size(1); c.Hkv = Hkv; c.D = 128; c.page = 16; c.max_blocks = tables.size(1);
    c.scale = static_cast<float>(scale_of(scale, what));
  }
  bool empty() const { return out.numel() == 0; }
  // `floats` of the call's own in front of the kernels' scratch
  float* take(int64_t floats, size_t bytes) {
    scratch = torch::empty({floats * 4 + static_cast<int64_t>(bytes)}, q.options().dtype(torch::kUInt8));
    return static_cast<float*>(scratch.data_ptr());
  }
};

torch::Tensor paged_decode_shared(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& tables, const torch::Tensor& context,
                                  const torch::Tensor& cu_groups_in, const torch::Tensor& shared_in, const c10::optional<int64_t>& max_group_in,
                                  const c10::optional<torch::Tensor>& ks, const c10::optional<torch::Tensor>& vs, const c10::optional<double>& scale) {
  const char* what = "paged_decode_shared";
  c10::cuda::CUDAGuard guard(k.device());
  Decode t(q, k, v, tables, context, ks, vs, scale, what);
  TORCH_CHECK_VALUE(shared_in.dim() == 1 && cu_groups_in.dim() == 1 && cu_groups_in.numel() == shared_in.numel() + 1, what,
                    ": cu_groups [groups + 1] and shared_lens [groups] are needed, got ", cu_groups_in.sizes(), " and ", shared_in.sizes());
  check_ints(cu_groups_in, k, what, "cu_groups");
  check_ints(shared_in, k, what, "shared_lens");
  TORCH_CHECK_VALUE(!max_group_in.has_value() || *max_group_in >= 1, what, ": max_group must be positive, got ", *max_group_in);
  if (t.empty()) return t.out;
  const torch::Tensor cu_groups = cu_groups_in.contiguous(), shared = shared_in.contiguous();
  const nrl::DecodeCall& c = t.c;
  const int64_t groups = shared.numel(), max_group = std::min<int64_t>(max_group_in.value_or(c.S), c.S);
  float* scratch = t.take(0, nrl_decode_scratch(&c, groups, max_group, num_sms()));
  check(nrl_paged_decode_shared(&c, cu_groups.data_ptr<int>(), shared.data_ptr<int>(), groups, max_group, scratch, num_sms(), cur_stream()), what);
  return t.out;
}

// scores [S, Hkv, tokens] float32, tokens side by side
void check_scores(const torch::Tensor& s, const torch::Tensor& k, int64_t rows, const char* what, const char* name) {
  TORCH_CHECK_VALUE(s.dim() == 3 && s.size(0) == rows && s.size(1) == k.size(1) && s.size(2) >= 1 && s.size(2) <= kIntMax, what, ": ", name, " must be [", rows, ", ", k.size(1),
                    ", tokens], got ", s.sizes());
  TORCH_CHECK_TYPE(s.scalar_type() == torch::kFloat32 && s.device() == k.device() && (s.stride(2) == 1 || s.size(2) == 1), what, ": ", name, " must be float32 on ",
                   k.device(), ", the tokens of a head side by side");
}

std::tuple<torch::Tensor, torch::Tensor> paged_decode_scored(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& tables,
                                                             const torch::Tensor& context, const torch::Tensor& scores, double decay,
                                                             const c10::optional<torch::Tensor>& ks, const c10::optional<torch::Tensor>& vs,
                                                             const c10::optional<double>& scale, const c10::optional<torch::Tensor>& out_scores) {
  const char* what = "paged_decode_scored";
  c10::cuda::CUDAGuard guard(k.device());
  Decode t(q, k, v, tables, context, ks, vs, scale, what);
  const nrl::DecodeCall& c = t.c;
  check_scores(scores, k, c.S, what, "scores");
  const torch::Tensor into = out_scores.value_or(scores);
  if (out_scores.has_value()) {
    check_scores(into, k, c.S, what, "out_scores");
    TORCH_CHECK_VALUE(into.sizes() == scores.sizes(), what, ": out_scores must be like scores, got ", into.sizes(), " and ", scores.sizes());
  }
  TORCH_CHECK_VALUE(at::has_internal_overlap(into) != at::MemOverlap::Yes, what, ": ", out_scores.has_value() ? "out_scores" : "scores",
                    " must not be expanded: they are written to");
  TORCH_CHECK_VALUE(std::isfinite(decay), what, ": decay must be finite, got ", decay);
  if (t.empty()) return {t.out, into};
  const int64_t raws = 16LL * c.max_blocks * c.S * c.Hq;
  float* raw = t.take(raws, nrl_decode_scratch(&c, 0, 0, num_sms()));
  check(nrl_paged_decode_scored(&c, scores.data_ptr<float>(), scores.stride(0), scores.stride(1), into.data_ptr<float>(), into.stride(0), into.stride(1), scores.size(2),
                                static_cast<float>(decay), raw, raw + raws, num_sms(), cur_stream()), what);
  return {t.out, into};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> kv_evict(torch::Tensor k, torch::Tensor v, const torch::Tensor& tables_in, const torch::Tensor& context_in,
                                                                 const torch::Tensor& scores, int64_t keep, int64_t sinks, int64_t recent,
                                                                 const c10::optional<torch::Tensor>& ks, const c10::optional<torch::Tensor>& vs,
                                                                 const c10::optional<torch::Tensor>& out_tables) {
  const char* what = "kv_evict";
  check_pages(k, v, ks, vs, tables_in, context_in, what);
  c10::cuda::CUDAGuard guard(k.device());
  const torch::Tensor tables = tables_in.contiguous(), context = context_in.contiguous();
  const int64_t S = tables.size(0), Hkv = k.size(1);
  check_scores(scores, k, S, what, "scores");
  TORCH_CHECK_VALUE(keep >= 1 && keep <= kIntMax / 2 && sinks >= 0 && recent >= 0 && sinks + recent <= keep, what,
                    ": keep must be positive and at least sinks + recent, got ", keep, ", ", sinks, " and ", recent);
  EvictCall c;
  // no token is looked for behind the scores or behind the tables
  c.max_tokens = std::min<int64_t>(scores.size(2), 16 * tables.size(1));
  torch::Tensor to;
  if (out_tables.has_value()) {
    TORCH_CHECK_VALUE(out_tables->dim() == 2 && out_tables->size(0) == S && 16 * out_tables->size(1) >= std::min<int64_t>(keep, c.max_tokens), what, ": out_tables must be [",
                      S, ", pages] with room for ", keep, " tokens, got ", out_tables->sizes());
    check_ints(*out_tables, k, what, "out_tables");
    to = out_tables->contiguous();
  }
  TORCH_CHECK_VALUE(k.size(0) * Hkv * 16 <= kIntMax && (std::min<int64_t>(keep, c.max_tokens) + 511) / 512 * Hkv <= 65535 && S <= kIntMax / 8, what, ": too many tokens");
  TORCH_CHECK_VALUE(c.max_tokens <= 8 * 48 * 1024, what, ": scores and tables of at most 393 216 tokens a row, got ", c.max_tokens);
  torch::Tensor kept = torch::empty({S, Hkv, keep}, tables.options()), kept_scores = torch::empty({S, Hkv, keep}, scores.options());
  torch::Tensor lens = torch::empty({S}, tables.options());
  // 512 bytes a row-head of counts, then the bits
  const torch::Tensor scratch = torch::empty({S * Hkv * (128 + (c.max_tokens + 31) / 32)}, tables.options());
  c.k_cache = k.data_ptr();
  c.v_cache = v.data_ptr();
  c.k_scale = ks.has_value() ? ks->data_ptr<float>() : nullptr;
  c.v_scale = vs.has_value() ? vs->data_ptr<float>() : nullptr;
  c.block_tables = tables.data_ptr<int>();
  c.context_lens = context.data_ptr<int>();
  c.out_tables = to.defined() ? to.data_ptr<int>() : nullptr;
  c.scores = scores.data_ptr<float>();
  c.score_row = scores.stride(0);
  c.score_head = scores.stride(1);
  c.kept = kept.data_ptr<int>();
  c.kept_scores = kept_scores.data_ptr<float>();
  c.new_lens = lens.data_ptr<int>();
  c.bits = reinterpret_cast<unsigned*>(scratch.data_ptr<int>()) + S * Hkv * 128;
  c.told = reinterpret_cast<uint4*>(scratch.data_ptr<int>());
  c.S = S; c.Hkv = Hkv; c.max_blocks = tables.size(1); c.out_blocks = to.defined() ? to.size(1) : 0;
  c.keep = keep; c.sinks = sinks; c.recent = recent;
  check(nrl_kv_evict(&c, num_sms(), cur_stream()), what);
  return {kept, kept_scores, lens};
}

}  // namespace

namespace nrl {

void bind_groups(pybind11::module_& m) {
  m.def("attention_shared_prefix", &attention_shared_prefix);
  m.def("attn_groups_arguments", &packed_arguments);
  m.def("attn_groups_fwd", &attn_groups_fwd);
  m.def("attn_groups_bwd", &attn_groups_bwd);
  m.def("paged_decode_shared", &paged_decode_shared);
  m.def("paged_decode_scored", &paged_decode_scored);
  m.def("kv_evict", &kv_evict);
}

}  // namespace nrl
