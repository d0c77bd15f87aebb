// Eviction from a paged KV cache: rows over their budget of `keep` tokens keep the first `sinks`, the last `recent` and, of the others, those with the
// largest scores (ties: the lower index), every kv head its own; what is kept moves together, in order, into the first `keep` places.
//
// kv_select: a block per (row, kv head).  The scores, as whole numbers whose order is theirs, wait in shared memory (in global memory above 48 K tokens); the smallest
// kept one is found digit by digit (11, 11 and 10 bits) from counts of the digits of what still ties with it, then every thread counts what is kept of a run of
// neighbouring tokens, the counts are summed over the block, and the indices are written in order.
// kv_move: a block per (row, kv head, slice of a token's keys or values).  Token j of what is kept comes from a place >= j, so that a block that reads a
// range of places before it writes them, ranges in order, may move in place; other slices' bytes are not touched.  Values of fp8 pages lie transposed: a thread
// has one element of all tokens, reads it sixteen tokens at a time and packs what is kept.
#include "common.cuh"
#include "group_kernels.h"
#include "launch.h"
#include "per_device.h"

namespace nrl {

constexpr int kSelThreads = 512;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelSmemTokens = 48 * 1024;
constexpr int kSelBins = 2048;

// larger scores have larger keys; -0 is 0, a NaN is below everything (0)
NRL_DEVICE uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

__global__ void __launch_bounds__(kSelThreads) kv_select_kernel(const EvictCall p, const int in_smem) {
  pdl_wait();
  pdl_launch_dependents();
  extern __shared__ uint32_t keys[];
  __shared__ uint32_t bins[kSelBins];
  __shared__ uint2 warp_sums[kSelWarps];
  __shared__ uint32_t found[2];                                       // a digit, and how many of it are kept
  const int seq = blockIdx.x, kvh = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = min(p.context_lens[seq], p.max_tokens);
  const long row = static_cast<long>(seq) * p.Hkv + kvh;
  int* kept = p.kept + row * p.keep;
  float* kept_scores = p.kept_scores + row * p.keep;
  const float* sc = p.scores + seq * p.score_row + kvh * p.score_head;
  if (kvh == 0 && tid == 0) p.new_lens[seq] = max(0, min(n, p.keep));
  if (n <= p.keep) {
    for (int j = tid; j < p.keep; j += kSelThreads) {
      kept[j] = j < n ? j : -1;
      kept_scores[j] = j < n ? sc[j] : 0.f;
    }
    return;
  }
  const int lo = p.sinks, hi = n - p.recent, m = hi - lo;             // candidates [lo, hi)
  uint32_t need = p.keep - p.sinks - p.recent;                        // < m
  auto key_at = [&](int i) { return in_smem ? keys[i] : order_key(sc[lo + i]); };
  if (in_smem) for (int i = tid; i < m; i += kSelThreads) keys[i] = order_key(sc[lo + i]);
  uint32_t prefix = 0, mask = 0;                                      // digits found so far
  if (need > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass == 2 ? 10 : 11;
      for (int i = tid; i < kSelBins; i += kSelThreads) bins[i] = 0;
      __syncthreads();
      for (int i = tid; i < m; i += kSelThreads) {
        const uint32_t k = key_at(i);
        if ((k & mask) == prefix) atomicAdd(&bins[(k >> shift) & ((1u << width) - 1)], 1u);
      }
      __syncthreads();
      // thread i sums bins [4 i, 4 i + 4) from the top; the digit is where the sum from the top reaches `need`
      uint32_t c[4], mine = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) mine += c[e] = bins[kSelBins - 1 - (tid * 4 + e)];
      uint32_t upto = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += v;
      }
      if (lane == 31) warp_sums[warp].x = upto;
      __syncthreads();
      for (int w = 0; w < warp; ++w) upto += warp_sums[w].x;
      uint32_t above = upto - mine;
      if (above < need && need <= upto) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (above < need && need <= above + c[e]) { found[0] = kSelBins - 1 - (tid * 4 + e); found[1] = need - above; }
          above += c[e];
        }
      }
      __syncthreads();
      prefix |= found[0] << shift;
      mask |= ((1u << width) - 1) << shift;
      need = found[1];
    }
  }
  // larger than `prefix`: kept; equal: the first `need`
  const int per = (m + kSelThreads - 1) / kSelThreads, i0 = min(m, tid * per), i1 = min(m, i0 + per);
  const bool none = p.keep == p.sinks + p.recent;
  __syncthreads();
  uint32_t more = 0, same = 0;
  for (int i = i0; i < i1; ++i) {
    const uint32_t k = key_at(i);
    more += k > prefix;
    same += k == prefix;
  }
  uint32_t more_upto = more, same_upto = same;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, more_upto, d), b = __shfl_up_sync(0xffffffffu, same_upto, d);
    if (lane >= d) { more_upto += a; same_upto += b; }
  }
  if (lane == 31) warp_sums[warp] = make_uint2(more_upto, same_upto);
  __syncthreads();
  uint32_t more_at = more_upto - more, same_at = same_upto - same;
  for (int w = 0; w < warp; ++w) { more_at += warp_sums[w].x; same_at += warp_sums[w].y; }
  if (!none) {
    for (int i = i0; i < i1; ++i) {
      const uint32_t k = key_at(i);
      if (k > prefix || (k == prefix && same_at < need)) {
        const uint32_t j = p.sinks + more_at + min(same_at, need);
        kept[j] = lo + i;
        kept_scores[j] = sc[lo + i];
      }
      more_at += k > prefix;
      same_at += k == prefix;
    }
  }
  for (int j = tid; j < p.sinks; j += kSelThreads) { kept[j] = j; kept_scores[j] = sc[j]; }
  for (int j = tid; j < p.recent; j += kSelThreads) { kept[p.keep - p.recent + j] = hi + j; kept_scores[p.keep - p.recent + j] = sc[hi + j]; }
}

// ---- tokens' rows: 16-byte pieces of keys (and of bf16 values), and their scales ---------------------------------------------------------------------
constexpr int kMoveThreads = 256;
constexpr int kMoveUnits = 8;             // pieces a thread holds
constexpr int kMovePieces = 4;            // pieces of a token that a block moves (64 bytes)

struct MoveParams {
  EvictCall e;
  const int* out_tables;
  int out_blocks, key_slices, value_slices;   // grid.z: slices of keys, then of values, then (fp8) values transposed and the scales
};

// where token t of a row lies: its place among all tokens of kv head `kvh`
NRL_DEVICE long token_place(const int* table, int t, int Hkv, int kvh) { return (static_cast<long>(table[t >> 4]) * Hkv + kvh) * 16 + (t & 15); }

template <class T, int PIECES>
NRL_DEVICE void move_rows(T* rows, int row_elems, int slice, const int* from, const int* to, const int* kept, int count, int Hkv, int kvh, bool in_place) {
  const int piece = threadIdx.x % PIECES, lane_tok = threadIdx.x / PIECES;
  constexpr int kTok = kMoveThreads / PIECES, kRange = kTok * kMoveUnits;
  T cur[kMoveUnits];
  long src[kMoveUnits], dst[kMoveUnits];
  for (int j0 = 0; j0 < count; j0 += kRange) {
#pragma unroll
    for (int u = 0; u < kMoveUnits; ++u) {
      const int j = j0 + u * kTok + lane_tok;
      const int t = j < count ? kept[j] : -1;
      dst[u] = -1;
      if (t < 0 || (in_place && t == j)) continue;
      src[u] = token_place(from, t, Hkv, kvh);
      dst[u] = token_place(to, j, Hkv, kvh);
    }
#pragma unroll
    for (int u = 0; u < kMoveUnits; ++u)
      if (dst[u] >= 0) cur[u] = rows[src[u] * row_elems + slice * PIECES + piece];
    __syncthreads();                      // all of this range is read before any of it is written
#pragma unroll
    for (int u = 0; u < kMoveUnits; ++u)
      if (dst[u] >= 0) rows[dst[u] * row_elems + slice * PIECES + piece] = cur[u];
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kMoveThreads) kv_move_kernel(const MoveParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int seq = blockIdx.x, kvh = blockIdx.y, tid = threadIdx.x;
  int z = blockIdx.z;
  const EvictCall& e = p.e;
  const bool in_place = e.out_tables == nullptr, fp8 = e.k_scale != nullptr;
  const int n = min(e.context_lens[seq], e.max_tokens), count = max(0, min(n, e.keep));
  if (in_place && n <= e.keep) return;
  const int* from = e.block_tables + static_cast<long>(seq) * e.max_blocks;
  const int* to = p.out_tables + static_cast<long>(seq) * p.out_blocks;
  const int* kept = e.kept + (static_cast<long>(seq) * e.Hkv + kvh) * e.keep;
  const int row_elems = fp8 ? 8 : 16;
  if (z < p.key_slices) return move_rows<uint4, kMovePieces>(static_cast<uint4*>(e.k_cache), row_elems, z, from, to, kept, count, e.Hkv, kvh, in_place);
  z -= p.key_slices;
  if (!fp8) return move_rows<uint4, kMovePieces>(static_cast<uint4*>(e.v_cache), row_elems, z, from, to, kept, count, e.Hkv, kvh, in_place);
  if (z == 1) return move_rows<float, 1>(e.k_scale, 1, 0, from, to, kept, count, e.Hkv, kvh, in_place);
  if (z == 2) return move_rows<float, 1>(e.v_scale, 1, 0, from, to, kept, count, e.Hkv, kvh, in_place);
  // values transposed: thread d of 128 packs element d of the kept tokens, page by page
  if (tid >= 128) return;
  const uint4* v = static_cast<const uint4*>(e.v_cache);
  uint4* out = static_cast<uint4*>(e.v_cache);
  uint32_t word[4] = {0, 0, 0, 0};
  int page = -1;
  uint4 cur = make_uint4(0, 0, 0, 0);
  for (int j = 0; j < count; ++j) {
    const int t = kept[j];
    if ((t >> 4) != page) {
      page = t >> 4;
      cur = v[(static_cast<long>(from[page]) * e.Hkv + kvh) * 128 + tid];
    }
    const int b = t & 15;
    const uint32_t w = b < 8 ? (b < 4 ? cur.x : cur.y) : (b < 12 ? cur.z : cur.w);
    const uint32_t byte = (w >> ((b & 3) * 8)) & 0xffu;
    const int c = j & 15;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((c >> 2) == i) word[i] |= byte << ((c & 3) * 8);
    if (c == 15 || j == count - 1) {
      const long at = (static_cast<long>(to[j >> 4]) * e.Hkv + kvh) * 128 + tid;
      if (c < 15) {                        // places behind the last stay as they were
        const uint4 old = out[at];
        const uint32_t ow[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = c + 1 - i * 4;                                  // bytes of this word that are new
          if (k < 4) word[i] = k <= 0 ? ow[i] : (word[i] & (0xffffffffu >> (32 - 8 * k))) | (ow[i] & (0xffffffffu << (8 * k)));
        }
      }
      out[at] = make_uint4(word[0], word[1], word[2], word[3]);
      word[0] = word[1] = word[2] = word[3] = 0;
    }
  }
}

}  // namespace nrl

using namespace nrl;

extern "C" cudaError_t nrl_kv_evict(const EvictCall* c, cudaStream_t s) {
  if (c->S == 0) return cudaSuccess;
  const int in_smem = c->max_tokens <= kSelSmemTokens;
  const int smem = in_smem ? c->max_tokens * 4 : 0;
  static PerDevice<bool> configured;
  cudaError_t e = allow_smem(configured, kv_select_kernel, kSelSmemTokens * 4);
  if (e != cudaSuccess) return e;
  launch_dependent(kv_select_kernel, dim3(c->S, c->Hkv), kSelThreads, smem, s, *c, in_smem);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  MoveParams p;
  p.e = *c;
  p.out_tables = c->out_tables != nullptr ? c->out_tables : c->block_tables;
  p.out_blocks = c->out_tables != nullptr ? c->out_blocks : c->max_blocks;
  const bool fp8 = c->k_scale != nullptr;
  p.key_slices = (fp8 ? 8 : 16) / kMovePieces;
  p.value_slices = fp8 ? 3 : 16 / kMovePieces;
  launch_dependent(kv_move_kernel, dim3(c->S, c->Hkv, p.key_slices + p.value_slices), kMoveThreads, 0, s, p);
  return cudaGetLastError();
}
