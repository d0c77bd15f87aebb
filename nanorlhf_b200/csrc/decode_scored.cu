// Decode attention that adds up what weight every cached token gets:
//
//   scores[s, h, t] = decay * scores[s, h, t] + sum over the G heads of kv head h of p[s, g, t]      (the newest token, t = context - 1: the sum alone)
//
// p = 2^(x - M) / L needs the row's maximum and sum over all keys, so the paged decode kernels (mode kDecodeScored) leave the scores x in scratch memory, 4 G bytes
// a token beside the 512 (bf16) or 264 (fp8) of its keys and values, and this kernel forms the weights from them; scratch that fits L2 is not read from memory again.
// Where the walk was cut into parts, their results are merged in the same launch.
#include "common.cuh"
#include "decode_merge.cuh"
#include "decode_modes.cuh"
#include "group_kernels.h"
#include "launch.h"

namespace nrl {

constexpr int kScoreChunk = 512;         // tokens a block

struct ScoreParams {
  MergeParams merge;
  const int* context_lens;
  const float* raw;                      // [S, Hkv, G, raw_len]
  const float* in;
  float* out;
  long raw_len, in_row, in_head, out_row, out_head;
  int max_tokens, merge_blocks;          // grid.y: merge_blocks of heads, then (kv head, chunk) pairs
  float decay;
};

__global__ void __launch_bounds__(kMergeD) decode_scored_kernel(const ScoreParams p) {
  pdl_wait();
  pdl_launch_dependents();
  if (blockIdx.y < static_cast<unsigned>(p.merge_blocks)) {
    merge_decode_parts(p.merge);
    return;
  }
  __shared__ float top[8], inv[8];
  const int seq = blockIdx.x, at = blockIdx.y - p.merge_blocks, kvh = at % p.merge.Hkv, t0 = at / p.merge.Hkv * kScoreChunk;
  const int ctx = min(p.context_lens[seq], static_cast<int>(p.raw_len)), n = min(min(ctx, p.max_tokens), t0 + kScoreChunk);
  if (t0 >= n) return;
  const long row = static_cast<long>(seq) * p.merge.Hkv + kvh;
  if (threadIdx.x < p.merge.G) {
    const float2* ml = reinterpret_cast<const float2*>(p.merge.part_ml) + row * p.merge.splits * 8 + threadIdx.x;
    float M = -INFINITY, L = 0.f;
    for (int s = 0; s < p.merge.splits; ++s) M = fmaxf(M, ml[s * 8].x);
    for (int s = 0; s < p.merge.splits; ++s) L += ml[s * 8].x == -INFINITY ? 0.f : ml[s * 8].y * exp2f(ml[s * 8].x - M);
    top[threadIdx.x] = M == -INFINITY ? 0.f : M;
    inv[threadIdx.x] = L > 0.f ? 1.f / L : 0.f;
  }
  __syncthreads();
  const float* raw = p.raw + row * p.merge.G * p.raw_len;
  const float* in = p.in + seq * p.in_row + kvh * p.in_head;
  float* out = p.out + seq * p.out_row + kvh * p.out_head;
  for (int t = t0 + threadIdx.x; t < n; t += kMergeD) {
    float w = 0.f;
    for (int r = 0; r < p.merge.G; ++r) w += exp2f(raw[r * p.raw_len + t] - top[r]) * inv[r];
    out[t] = t < ctx - 1 ? fmaf(p.decay, in[t], w) : w;
  }
}

}  // namespace nrl

using namespace nrl;

extern "C" cudaError_t nrl_paged_decode_scored(const DecodeCall* c, const float* scores_in, long in_row, long in_head, float* scores_out, long out_row, long out_head,
                                               int max_tokens, float decay, float* raw, cudaStream_t s) {
  if (c->S == 0) return cudaSuccess;
  DecodeExtra x = {};
  x.raw = raw;
  x.raw_len = 16L * c->max_blocks;
  const cudaError_t e = c->k_scale != nullptr ? paged_decode_scored_fp8(*c, x, s) : paged_decode_scored_bf16(*c, x, s);
  if (e != cudaSuccess) return e;
  ScoreParams p;
  p.merge = {c->part_o, c->part_ml, static_cast<__nv_bfloat16*>(c->out), c->Hq, c->Hkv, c->Hq / c->Hkv, c->splits};
  p.context_lens = c->context_lens;
  p.raw = raw; p.in = scores_in; p.out = scores_out;
  p.raw_len = x.raw_len; p.in_row = in_row; p.in_head = in_head; p.out_row = out_row; p.out_head = out_head;
  p.max_tokens = max_tokens < x.raw_len ? max_tokens : static_cast<int>(x.raw_len);
  p.merge_blocks = c->splits > 1 ? c->Hq : 0;
  p.decay = decay;
  const int chunks = (p.max_tokens + kScoreChunk - 1) / kScoreChunk;
  launch_dependent(decode_scored_kernel, dim3(c->S, p.merge_blocks + chunks * c->Hkv), kMergeD, 0, s, p);
  return cudaGetLastError();
}
