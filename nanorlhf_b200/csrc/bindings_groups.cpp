// Tensors in, launches out: attention over shared prefixes, decode attention with scores, eviction.
#include "bindings_groups.h"

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
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

// [rows, heads, 128] bf16 whose heads lie side by side and whose rows start on 16 bytes
void check_rows(const torch::Tensor& t, const char* what, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == torch::kBFloat16 && t.dim() == 3 && t.size(2) == 128, what, ": ", name, " must be a CUDA bf16 tensor [rows, heads, 128]");
  TORCH_CHECK((t.stride(2) == 1 && (t.stride(1) == 128 || t.size(1) == 1) && (t.size(0) <= 1 || t.stride(0) % 8 == 0) &&
               reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0) || t.numel() == 0,
              what, ": the heads of a row of ", name, " must lie side by side and rows start on 16 bytes");
}
int64_t row_stride(const torch::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1) * 128; }
void check_ints(const torch::Tensor& t, const torch::Tensor& beside, int64_t dims, const char* what, const char* name) {
  TORCH_CHECK(t.device() == beside.device() && t.scalar_type() == torch::kInt32 && t.dim() == dims && t.is_contiguous(), what, ": ", name,
              " must be a contiguous int32 tensor of ", dims, " dimension(s) on ", beside.device());
}

// ---- packed groups ---------------------------------------------------------------------------------------------------------------------
void check_packed(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const char* what) {
  check_rows(q, what, "q"); check_rows(k, what, "k"); check_rows(v, what, "v");
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.device() == q.device() && v.device() == q.device() && k.size(1) > 0 && q.size(1) % k.size(1) == 0, what,
              ": k and v must be [", q.size(0), ", kv heads, 128] beside q, the query heads a multiple of theirs");
  TORCH_CHECK(q.size(0) * q.size(1) <= kIntMax, what, ": too many rows");
}
CUtensorMap map_of(const torch::Tensor& t, int box_rows) {
  return nrl::make_tma_2d(t.data_ptr(), t.size(0), static_cast<uint64_t>(t.size(1)) * 128, row_stride(t) * 2, box_rows, 64, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2);
}

// (out, lse [Hq, T], table of the sequences for the backward)
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> attn_groups_fwd(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                                                                        const torch::Tensor& cu_seqlens, const torch::Tensor& cu_groups, double scale) {
  const char* what = "attention_shared_prefix";
  check_packed(q, k, v, what);
  check_ints(cu_seqlens, q, 1, what, "cu_seqlens");
  check_ints(cu_groups, q, 1, what, "cu_groups");
  TORCH_CHECK(cu_seqlens.numel() >= 1 && cu_groups.numel() >= 1, what, ": cu_seqlens and cu_groups begin with 0");
  c10::cuda::CUDAGuard guard(q.device());
  const int T = q.size(0), Hq = q.size(1), Hkv = k.size(1), n = cu_seqlens.numel() - 1;
  torch::Tensor out = torch::empty({T, Hq, 128}, q.options()), lse = torch::empty({Hq, T}, q.options().dtype(torch::kFloat32));
  torch::Tensor table = torch::empty({n, 8}, cu_seqlens.options());
  if (T == 0) return {out, lse, table};
  const CUtensorMap mq = map_of(q, 128), mk = map_of(k, 128), mv = map_of(v, 128);
  check(nrl_attn_group_table(cu_seqlens.data_ptr<int>(), cu_groups.data_ptr<int>(), table.data_ptr<int>(), n, cu_groups.numel() - 1, out.data_ptr(), T, Hq, cur_stream()),
        what);
  check(nrl_attn_groups_fwd_tc(&mq, &mk, &mv, out.data_ptr(), lse.data_ptr<float>(), out.stride(0), cu_seqlens.data_ptr<int>(), table.data_ptr<int>(), n, T, Hq, Hkv,
                               static_cast<float>(scale), num_sms(), cur_stream()), what);
  return {out, lse, table};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> attn_groups_bwd(const torch::Tensor& dout, const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                                                                        const torch::Tensor& o, const torch::Tensor& lse, const torch::Tensor& cu_seqlens,
                                                                        const torch::Tensor& table, double scale) {
  const char* what = "attention_shared_prefix backward";
  check_packed(q, k, v, what);
  check_rows(dout, what, "the gradient");
  TORCH_CHECK(o.is_contiguous() && dout.is_contiguous() && dout.sizes() == o.sizes() && o.sizes() == q.sizes() && dout.device() == q.device(), what,
              ": the gradient must be contiguous and like q");
  c10::cuda::CUDAGuard guard(q.device());
  const int T = q.size(0), Hq = q.size(1), Hkv = k.size(1), n = cu_seqlens.numel() - 1;
  torch::Tensor dq = torch::empty({T, Hq, 128}, q.options()), dk = torch::empty({T, Hkv, 128}, q.options()), dv = torch::empty({T, Hkv, 128}, q.options());
  if (T == 0) return {dq, dk, dv};
  torch::Tensor delta = torch::empty({Hq, T}, q.options().dtype(torch::kFloat32));
  const CUtensorMap maps[8] = {map_of(q, 64), map_of(dout, 64), map_of(k, 128), map_of(v, 128), map_of(q, 128), map_of(dout, 128), map_of(k, 64), map_of(v, 64)};
  check(nrl_attn_groups_bwd_tc(maps, o.data_ptr(), dout.data_ptr(), lse.data_ptr<float>(), delta.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                               o.stride(0), dq.stride(0), dk.stride(0), cu_seqlens.data_ptr<int>(), table.data_ptr<int>(), n, T, Hq, Hkv, static_cast<float>(scale),
                               cur_stream()), what);
  return {dq, dk, dv};
}

// ---- pages -----------------------------------------------------------------------------------------------------------------------------
struct Pages {
  bool fp8;
  int64_t blocks, kv;
};
// k, v: bf16 [blocks, Hkv, 16, 128]; or uint8 (e4m3) of as many elements, values transposed, with scales [blocks, Hkv, 16]
Pages check_pages(const torch::Tensor& k, const torch::Tensor& v, const c10::optional<torch::Tensor>& ks, const c10::optional<torch::Tensor>& vs, const char* what) {
  TORCH_CHECK(k.is_cuda() && k.dim() == 4 && k.size(2) == 16 && k.size(3) == 128 && k.is_contiguous(), what, ": k_cache must be a contiguous CUDA tensor [blocks, kv heads, 16, 128]");
  const bool fp8 = ks.has_value();
  TORCH_CHECK(fp8 == vs.has_value(), what, ": k_scale and v_scale go together");
  TORCH_CHECK(k.scalar_type() == (fp8 ? torch::kUInt8 : torch::kBFloat16), what, ": pages are bf16, or uint8 (e4m3) with scales");
  TORCH_CHECK(v.device() == k.device() && v.scalar_type() == k.scalar_type() && v.is_contiguous() && v.dim() == 4 && v.size(0) == k.size(0) && v.size(1) == k.size(1) &&
              v.size(2) * v.size(3) == 2048, what, ": v_cache must be like k_cache");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(k.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(v.data_ptr()) % 16 == 0, what, ": pages must start on 16 bytes");
  if (fp8) {
    for (const torch::Tensor* s : {&*ks, &*vs})
      TORCH_CHECK(s->device() == k.device() && s->scalar_type() == torch::kFloat32 && s->is_contiguous() && s->dim() == 3 && s->size(0) == k.size(0) &&
                  s->size(1) == k.size(1) && s->size(2) == 16 && reinterpret_cast<uintptr_t>(s->data_ptr()) % 16 == 0, what,
                  ": scales must be contiguous float32 tensors [blocks, kv heads, 16]");
  } else {
    TORCH_CHECK(v.size(2) == 16, what, ": v_cache must be like k_cache");
  }
  return {fp8, k.size(0), k.size(1)};
}

// the call and its result
struct DecodeTensors {
  torch::Tensor out;
  nrl::DecodeCall c;
};
DecodeTensors decode_call(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& tables, const torch::Tensor& context,
                          const c10::optional<torch::Tensor>& ks, const c10::optional<torch::Tensor>& vs, double scale, const char* what) {
  check_rows(q, what, "q");
  const Pages pages = check_pages(k, v, ks, vs, what);
  TORCH_CHECK(k.device() == q.device(), what, ": pages and q must be on one device");
  check_ints(tables, q, 2, what, "block_tables");
  check_ints(context, q, 1, what, "context_lens");
  const int64_t S = q.size(0), Hq = q.size(1);
  TORCH_CHECK(tables.size(0) == S && context.size(0) == S && tables.size(1) >= 1, what, ": block_tables [rows, pages] and context_lens [rows]");
  TORCH_CHECK(S * tables.size(1) * std::max<int64_t>(1, pages.kv) <= kIntMax / 16 && tables.size(1) <= kIntMax / 512, what, ": too many rows or pages");
  TORCH_CHECK(pages.kv > 0 && Hq % pages.kv == 0 && Hq / pages.kv <= 8 && pages.kv <= 256, what, ": the query heads must be a multiple, at most 8 times, of the kv heads");
  DecodeTensors t;
  t.out = torch::empty({S, Hq, 128}, q.options());
  nrl::DecodeCall& c = t.c;
  c.q = q.data_ptr();
  c.q_stride_s = row_stride(q);
  c.k_cache = k.data_ptr();
  c.v_cache = v.data_ptr();
  c.k_scale = pages.fp8 ? ks->data_ptr<float>() : nullptr;
  c.v_scale = pages.fp8 ? vs->data_ptr<float>() : nullptr;
  c.block_tables = tables.data_ptr<int>();
  c.context_lens = context.data_ptr<int>();
  c.out = t.out.data_ptr();
  c.S = S; c.Hq = Hq; c.Hkv = pages.kv; c.D = 128; c.page = 16; c.max_blocks = tables.size(1);
  c.scale = static_cast<float>(scale);
  return t;
}
torch::Tensor scratch_of(size_t bytes, const torch::Tensor& q) { return torch::empty({static_cast<int64_t>(bytes)}, q.options().dtype(torch::kUInt8)); }

torch::Tensor paged_decode_shared(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& tables, const torch::Tensor& context,
                                  const torch::Tensor& cu_groups, const torch::Tensor& shared, int64_t max_group, const c10::optional<torch::Tensor>& ks,
                                  const c10::optional<torch::Tensor>& vs, double scale) {
  const char* what = "paged_decode_shared";
  TORCH_CHECK(q.is_cuda(), what, ": q must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(q.device());
  const DecodeTensors t = decode_call(q, k, v, tables, context, ks, vs, scale, what);
  const nrl::DecodeCall& c = t.c;
  check_ints(cu_groups, q, 1, what, "cu_groups");
  check_ints(shared, q, 1, what, "shared_lens");
  const int64_t groups = shared.numel();
  TORCH_CHECK(cu_groups.numel() == groups + 1, what, ": cu_groups must be [groups + 1] and shared_lens [groups]");
  TORCH_CHECK(max_group >= 1, what, ": max_group must be positive");
  if (c.S == 0) return t.out;
  max_group = std::min<int64_t>(max_group, c.S);
  const int parts = groups > 0 ? nrl_decode_prefix_parts(groups, max_group, c.Hq, c.Hkv, c.max_blocks, num_sms()) : 0;
  const int64_t lines = static_cast<int64_t>(c.S) * c.Hkv * parts * 8;
  TORCH_CHECK(lines <= kIntMax, what, ": too many rows");
  const torch::Tensor prefix = torch::empty({lines * 130}, q.options().dtype(torch::kFloat32)), scratch = scratch_of(nrl_decode_flat_scratch(&c, num_sms()), q);
  float* prefix_o = parts > 0 ? prefix.data_ptr<float>() : nullptr;
  check(nrl_paged_decode_shared(&c, cu_groups.data_ptr<int>(), shared.data_ptr<int>(), groups, max_group, parts, prefix_o, prefix_o + lines * 128, scratch.data_ptr(),
                                num_sms(), cur_stream()), what);
  return t.out;
}

// scores [S, Hkv, tokens] float32, tokens side by side
void check_scores(const torch::Tensor& s, int64_t S, int64_t kv, const torch::Tensor& q, const char* what, const char* name) {
  TORCH_CHECK(s.device() == q.device() && s.scalar_type() == torch::kFloat32 && s.dim() == 3 && s.size(0) == S && s.size(1) == kv && s.size(2) >= 1 &&
              s.size(2) <= kIntMax && (s.stride(2) == 1 || s.size(2) == 1), what, ": ", name, " must be a float32 tensor [", S, ", ", kv, ", tokens], tokens side by side");
}

torch::Tensor paged_decode_scored(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& tables, const torch::Tensor& context,
                                  const torch::Tensor& scores, torch::Tensor out_scores, double decay, const c10::optional<torch::Tensor>& ks,
                                  const c10::optional<torch::Tensor>& vs, double scale) {
  const char* what = "paged_decode_scored";
  TORCH_CHECK(q.is_cuda(), what, ": q must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(q.device());
  const DecodeTensors t = decode_call(q, k, v, tables, context, ks, vs, scale, what);
  const nrl::DecodeCall& c = t.c;
  check_scores(scores, c.S, c.Hkv, q, what, "scores");
  check_scores(out_scores, c.S, c.Hkv, q, what, "out_scores");
  TORCH_CHECK(out_scores.size(2) == scores.size(2), what, ": out_scores must be like scores");
  if (c.S == 0) return t.out;
  const torch::Tensor raw = torch::empty({c.S, c.Hq, 16LL * c.max_blocks}, q.options().dtype(torch::kFloat32)), scratch = scratch_of(nrl_decode_flat_scratch(&c, num_sms()), q);
  check(nrl_paged_decode_scored(&c, scores.data_ptr<float>(), scores.stride(0), scores.stride(1), out_scores.data_ptr<float>(), out_scores.stride(0), out_scores.stride(1),
                                scores.size(2), static_cast<float>(decay), raw.data_ptr<float>(), scratch.data_ptr(), num_sms(), cur_stream()), what);
  return t.out;
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> kv_evict(torch::Tensor k, torch::Tensor v, const torch::Tensor& tables, const torch::Tensor& context,
                                                                 const torch::Tensor& scores, int64_t keep, int64_t sinks, int64_t recent,
                                                                 const c10::optional<torch::Tensor>& ks, const c10::optional<torch::Tensor>& vs,
                                                                 const c10::optional<torch::Tensor>& out_tables) {
  const char* what = "kv_evict";
  const Pages pages = check_pages(k, v, ks, vs, what);
  c10::cuda::CUDAGuard guard(k.device());
  check_ints(tables, k, 2, what, "block_tables");
  check_ints(context, k, 1, what, "context_lens");
  const int64_t S = tables.size(0);
  TORCH_CHECK(context.size(0) == S && tables.size(1) >= 1 && pages.kv > 0 && pages.kv <= 65535, what, ": block_tables [rows, pages] and context_lens [rows]");
  check_scores(scores, S, pages.kv, k, what, "scores");
  TORCH_CHECK(keep >= 1 && keep <= kIntMax / 2 && sinks >= 0 && recent >= 0 && sinks + recent <= keep, what, ": keep must be positive and at least sinks + recent");
  TORCH_CHECK(pages.blocks * pages.kv * 16 <= kIntMax && (std::min<int64_t>(keep, scores.size(2)) + 511) / 512 * pages.kv <= 65535, what, ": too many tokens");
  if (out_tables.has_value()) {
    check_ints(*out_tables, k, 2, what, "out_tables");
    TORCH_CHECK(out_tables->size(0) == S && out_tables->size(1) >= 1, what, ": out_tables must be [rows, pages]");
  }
  torch::Tensor kept = torch::empty({S, pages.kv, keep}, tables.options()), kept_scores = torch::empty({S, pages.kv, keep}, scores.options());
  torch::Tensor lens = torch::empty({S}, tables.options());
  EvictCall c;
  c.k_cache = k.data_ptr();
  c.v_cache = v.data_ptr();
  c.k_scale = pages.fp8 ? ks->data_ptr<float>() : nullptr;
  c.v_scale = pages.fp8 ? vs->data_ptr<float>() : nullptr;
  c.block_tables = tables.data_ptr<int>();
  c.context_lens = context.data_ptr<int>();
  c.out_tables = out_tables.has_value() ? out_tables->data_ptr<int>() : nullptr;
  c.scores = scores.data_ptr<float>();
  c.score_row = scores.stride(0);
  c.score_head = scores.stride(1);
  c.kept = kept.data_ptr<int>();
  c.kept_scores = kept_scores.data_ptr<float>();
  c.new_lens = lens.data_ptr<int>();
  c.S = S; c.Hkv = pages.kv; c.max_blocks = tables.size(1); c.out_blocks = out_tables.has_value() ? out_tables->size(1) : 0;
  // no token is looked for behind the scores or behind the tables
  c.max_tokens = std::min<int64_t>(scores.size(2), 16 * tables.size(1));
  c.keep = keep; c.sinks = sinks; c.recent = recent;
  const torch::Tensor bits = torch::empty({S, pages.kv, (c.max_tokens + 31) / 32}, tables.options());
  c.bits = reinterpret_cast<unsigned*>(bits.data_ptr<int>());
  check(nrl_kv_evict(&c, num_sms(), cur_stream()), what);
  return {kept, kept_scores, lens};
}

}  // namespace

namespace nrl {

void bind_groups(pybind11::module_& m) {
  m.def("attn_groups_fwd", &attn_groups_fwd);
  m.def("attn_groups_bwd", &attn_groups_bwd);
  m.def("paged_decode_shared", &paged_decode_shared);
  m.def("paged_decode_scored", &paged_decode_scored);
  m.def("kv_evict", &kv_evict);
}

}  // namespace nrl
