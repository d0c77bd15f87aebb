// Eviction from a paged KV cache: rows over their budget of `keep` tokens keep the first `sinks`, the last `recent` and, of the others, those with the
// largest scores (ties: the lower index), every kv head its own; what is kept moves together, in order, into the first `keep` places.
//
// kv_select: a cluster of blocks per (row, kv head), more blocks where there are few and their contexts long.  A block has a range of tokens; their scores, as whole
// numbers whose order is theirs, wait in shared memory.  The smallest kept one is found three bits at a time: a thread counts the eight digits of the keys that may still be it
// in the bytes of two words, warps, the block and (through memory) the cluster add up, until as many keys are at or above a digit as are to be kept.  Then the tokens are
// counted again, word by word of 32, and indices and a bit a token are written in order.  Bound by latency, up to eleven rounds of a barrier (and one of the cluster).
// (Counts of digits by atomics in shared memory meet: a score's highest bits are a few exponents, and 3750 tokens a block took 120 us with eight bits a round, 20 with eleven;
// seven votes a word and round 20.)
// kv_move: in place a block per (row, kv head, 64 bytes of a token's keys or values): token j of what is kept comes from a place >= j, so that a block that reads a range
// of places before it writes them, ranges in order and the next one on its way, may move it; other slices' bytes are not touched.  Where sources and targets are
// apart a block per (row, kv head, range of places, keys or values).
// In place from a budget and 64 tokens down to it, as the sampler evicts, nearly all that is kept moves: 253 rows of 1088 -> 1024 tokens, 2 kv heads, fp8 98 us and bf16 150
// (the bytes' floors 42 and 81), 8 of 4160 -> 4096, 4 heads, 73 and 45 (11 and 20); few long fp8 rows take longest, one block having all values of a row-head: 8 of
// 30 011 -> 4096 359 us, bf16 91.
// (All times here are of whole calls in graphs; one by one calls take up to 10 us more.)
// Values of fp8 pages lie transposed, and their blocks come first, for they take longest (in a launch in front of the others' 69 us, in one 60).  Sixteen pages at a
// time go through shared memory, rows of 16 bytes 20 apart (no bank conflicts), and a thread puts together an element's bytes of a whole page.
#include "common.cuh"
#include "group_kernels.h"
#include "launch.h"
#include "per_device.h"

#include <climits>

namespace nrl {

constexpr int kSelTokens = 48 * 1024;     // of a block, in shared memory; kSelCluster times as many of a row at the most (checked on the host)
constexpr int kSelCluster = 8;

// larger scores have larger keys; -0 is 0, a NaN is below everything (0)
NRL_DEVICE uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
// 0 from 32 places on
NRL_DEVICE uint32_t shl(uint32_t x, uint32_t by) {
  uint32_t r;
  asm("shl.b32 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(by));
  return r;
}
NRL_DEVICE void evict_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// WARPS: 4 for up to 2048 tokens a block, 8 for up to 3840, else 16: sums over more warps cost more than their share of the words saves (3752 tokens a block: 60 us of a
// call with 16 warps, 58 with 8, 69 with 4; 4096: 27 with 16, 29 with 8, 34 with 4)
template <int WARPS>
__global__ void __launch_bounds__(WARPS * 32) kv_select_kernel(const EvictCall p, const int cluster) {
  constexpr int kSelWarps = WARPS, kSelThreads = WARPS * 32;
  pdl_wait();
  pdl_launch_dependents();
  extern __shared__ uint32_t keys[];
  __shared__ __align__(16) uint4 warp_counts[2][kSelWarps];           // of two rounds in turn: eight counts of 16 bits
  __shared__ uint2 warp_sums[kSelWarps];
  const int seq = blockIdx.x / cluster, rank = blockIdx.x - seq * cluster, kvh = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = max(0, min(p.context_lens[seq], p.max_tokens));
  const long row = static_cast<long>(seq) * p.Hkv + kvh;
  int* kept = p.kept + row * p.keep;
  const float* sc = p.scores + seq * p.score_row + kvh * p.score_head;
  uint32_t* bits = p.bits + row * ((p.max_tokens + 31) / 32);
  // a cluster's blocks tell one another their counts, 32 bytes a block; of two rounds in turn: others may still read the last one's
  uint4* const told = p.told + row * (4 * kSelCluster);
  if (kvh == 0 && rank == 0 && tid == 0) p.new_lens[seq] = min(n, p.keep);
  if (n <= p.keep) {
    const int at = rank * kSelThreads + tid, step = cluster * kSelThreads;
    for (int j = at; j < p.keep; j += step) kept[j] = j < n ? j : -1;
    for (int w = at; w * 32 < n; w += step) bits[w] = n - w * 32 >= 32 ? 0xffffffffu : (1u << (n - w * 32)) - 1;
    return;
  }
  const int lo = p.sinks, hi = n - p.recent;                          // [lo, hi) may go
  const int words = (n + 31) / 32, per_block = (words + cluster - 1) / cluster, b0 = min(words, rank * per_block), b1 = min(words, b0 + per_block);
  const int t0 = b0 * 32, m0 = max(lo, t0), m1 = min(hi, b1 * 32);     // of this block
  const uint32_t wanted = p.keep - p.sinks - p.recent;
  const bool any = wanted > 0;
  // a warp has a range of neighbouring words of 32 tokens
  const int per = (b1 - b0 + kSelWarps - 1) / kSelWarps, w0 = min(b1, b0 + warp * per), w1 = min(b1, w0 + per);
  uint32_t least = 0;                                                 // `wanted` keys or more are at or above it
  bool exact = false;                                                 // no more than those
  if (any) {
#pragma unroll 8
    for (int w = w0; w < w1; ++w) {                                   // (a warp reads its own)
      const int t = w * 32 + lane;
      keys[t - t0] = t >= m0 && t < m1 ? order_key(sc[t]) : 0u;       // 0: may not go
    }
    uint32_t over = 0;                                                // keys behind the eight digits
#pragma unroll 1
    for (int round = 0; round < 11 && !exact; ++round) {
      const int shift = max(0, 29 - 3 * round);                       // (the last round has the last two bits; four more digits have been counted)
      uint32_t lo = 0, hi = 0;                                        // a lane has 96 words at the most
#pragma unroll 4
      for (int w = w0; w < w1; ++w) {
        const uint32_t d = 8 * min((keys[w * 32 + lane - t0] - least) >> shift, 8u);
        lo += shl(1u, d);
        hi += shl(1u, d - 32u);
      }
      uint4 c = make_uint4(lo & 0x00ff00ffu, (lo >> 8) & 0x00ff00ffu, hi & 0x00ff00ffu, (hi >> 8) & 0x00ff00ffu);       // digits 0 2, 1 3, 4 6, 5 7
      auto add = [&](uint4 x, int from) {
        for (int m = from; m > 0; m >>= 1) {
          x.x += __shfl_xor_sync(0xffffffffu, x.x, m); x.y += __shfl_xor_sync(0xffffffffu, x.y, m);
          x.z += __shfl_xor_sync(0xffffffffu, x.z, m); x.w += __shfl_xor_sync(0xffffffffu, x.w, m);
        }
        return x;
      };
      c = add(c, 16);
      if (lane == 0) warp_counts[round & 1][warp] = c;
      __syncthreads();
      c = add(lane < kSelWarps ? warp_counts[round & 1][lane] : make_uint4(0, 0, 0, 0), kSelWarps / 2);
      uint32_t n_of[8] = {c.x & 0xffffu, c.y & 0xffffu, c.x >> 16, c.y >> 16, c.z & 0xffffu, c.w & 0xffffu, c.z >> 16, c.w >> 16};
      if (cluster > 1) {
        uint4* const here = told + (round & 1) * 2 * kSelCluster;
        if (tid < 2) here[rank * 2 + tid] = tid == 0 ? make_uint4(n_of[0], n_of[1], n_of[2], n_of[3]) : make_uint4(n_of[4], n_of[5], n_of[6], n_of[7]);
        evict_cluster_sync();
        uint4 x = make_uint4(0, 0, 0, 0);                             // lane i + 8 j: half j of block i's
        if ((lane & 7) < cluster && lane < 16) x = __ldcg(here + (lane & 7) * 2 + (lane >> 3));
        x = add(x, kSelCluster / 2);
        const uint32_t mine[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int v = 0; v < 8; ++v) n_of[v] = __shfl_sync(0xffffffffu, mine[v & 3], (v >> 2) * 8);
      } else {
#pragma unroll
        for (int v = 0; v < 8; ++v) n_of[v] = __shfl_sync(0xffffffffu, n_of[v], 0);
      }
      // the highest digit that enough keys reach
      uint32_t best = 0, of_best = 0, behind = over, reach = over;
      bool found = false;
#pragma unroll
      for (int v = 7; v >= 0; --v) {
        const uint32_t with = reach + (v < 4 || round < 10 ? n_of[v] : 0u);
        if (!found && with >= wanted) { found = true; best = v; of_best = with; behind = reach; }
        reach = with;
      }
      least += best << shift;
      over = behind;
      exact = of_best == wanted && least > 0;
    }
  }
  if (exact) --least;                                                 // all above it (a candidate is above 0)
  // kept: the first, the last, keys above `least`, and of those equal to it as many as there is room for, the first ones
  auto look = [&](int word, uint32_t& more, uint32_t& same) {
    const int t = word * 32 + lane;
    const bool middle = any && t >= lo && t < hi;
    const uint32_t k = middle ? keys[t - t0] : 0u;
    more = __ballot_sync(0xffffffffu, t < n && (t < lo || t >= hi || (middle && k > least)));
    same = __ballot_sync(0xffffffffu, middle && k == least);
  };
  uint32_t more = 0, same = 0;
#pragma unroll 4
  for (int w = w0; w < w1; ++w) {
    uint32_t a, b;
    look(w, a, b);
    more += __popc(a);
    same += __popc(b);
  }
  if (lane == 0) warp_sums[warp] = make_uint2(more, same);
  __syncthreads();
  uint2 all = make_uint2(0, 0);
  for (int w = 0; w < kSelWarps; ++w) { all.x += warp_sums[w].x; all.y += warp_sums[w].y; }
  uint32_t need = p.keep;
  more = same = 0;
  if (cluster > 1) {
    evict_cluster_sync();                                             // (both rounds' counts have been read)
    if (tid == 0) told[rank] = make_uint4(all.x, all.y, 0, 0);
    evict_cluster_sync();
    for (int r = 0; r < cluster; ++r) {
      const uint4 v = __ldcg(told + r);
      need -= v.x;
      more += r < rank ? v.x : 0u;
      same += r < rank ? v.y : 0u;
    }
  } else {
    need -= all.x;
  }
  for (int w = 0; w < warp; ++w) { more += warp_sums[w].x; same += warp_sums[w].y; }
  const uint32_t under = (1u << lane) - 1;
#pragma unroll 4
  for (int w = w0; w < w1; ++w) {
    uint32_t a, b;
    look(w, a, b);
    const bool is = (a >> lane & 1) || ((b >> lane & 1) && same + __popc(b & under) < need);
    if (is) {
      const uint32_t j = more + __popc(a & under) + min(same + __popc(b & under), need);
      kept[j] = w * 32 + lane;
    }
    const uint32_t m = __ballot_sync(0xffffffffu, is);
    if (lane == 0) bits[w] = m;
    more += __popc(a);
    same += __popc(b);
  }
}

// ---- tokens' rows: 16-byte pieces of keys (and of bf16 values), and their scales ---------------------------------------------------------------------
constexpr int kMoveThreads = 256;
constexpr int kMoveUnits = 8;             // pieces a thread holds
// 16-byte pieces of a token that a block moves.  In place a block has all places of a row, and a slice of 64 bytes: more blocks.  Where sources and targets are apart it
// has whole rows and a range of places: of slices, indices were looked up once for each (253 fp8 rows 60.7 -> 57.2 us, 8 of 30 k bf16 tokens 70 -> 60).
__host__ __device__ constexpr int move_pieces(bool in_place, bool fp8) { return in_place ? 4 : fp8 ? 8 : 16; }
// Places of a block.  253 fp8 rows take 67 us with 128 (spans of transposed values meet too few), 57 with 256, 61 with 512.  Of fewer row-heads than fill the chip fewer:
// one span of transposed values follows another, and 2 rows of 24 k fp8 tokens, 628 kept, took 193 us with 512 places a block, 47 with 64.
__host__ __device__ constexpr int move_range(bool fp8) { return fp8 ? 256 : 128; }
constexpr int kMoveLeast = 64;
constexpr int kSpanPages = 16;            // of transposed values at a time: their tokens are as many as the threads
constexpr int kSpanRow = 5;               // words from an element's row to the next

struct MoveParams {
  EvictCall e;
  const int* out_tables;
  int out_blocks, key_slices, range;             // grid.y: kv heads x ranges of places; grid.z: slices of keys, then of values (fp8: the scales), then the scores
};

// where token t of a row lies: its place among all tokens (below 2^31: checked on the host)
NRL_DEVICE int token_place(const int* table, int t, int Hkv, int kvh) { return (table[t >> 4] * Hkv + kvh) * 16 + (t & 15); }

template <bool IN_PLACE, class T, int PIECES>
NRL_DEVICE void move_rows(T* rows, int row_elems, int slice, const int* from, const int* to, const int* kept, int j0, int j1, int Hkv, int kvh) {
  const int piece = threadIdx.x % PIECES, first = threadIdx.x / PIECES;
  constexpr int kTok = kMoveThreads / PIECES;
  T cur[kMoveUnits];
  int dst[kMoveUnits];
  T* mine = rows + slice * PIECES + piece;
  auto read = [&](int j_at) {
    int src[kMoveUnits];
#pragma unroll
    for (int u = 0; u < kMoveUnits; ++u) {
      const int j = j_at + u * kTok + first, t = j < j1 ? kept[j] : -1;
      const bool moves = t >= 0 && !(IN_PLACE && t == j);
      src[u] = moves ? token_place(from, t, Hkv, kvh) : -1;
      dst[u] = moves ? token_place(to, j, Hkv, kvh) : -1;
    }
#pragma unroll
    for (int u = 0; u < kMoveUnits; ++u)
      if (src[u] >= 0) cur[u] = mine[static_cast<long>(src[u]) * row_elems];
  };
  if (!IN_PLACE) {
    for (int j = j0; j < j1; j += kTok * kMoveUnits) {
      read(j);
#pragma unroll
      for (int u = 0; u < kMoveUnits; ++u)
        if (dst[u] >= 0) mine[static_cast<long>(dst[u]) * row_elems] = cur[u];
    }
    return;
  }
  read(j0);
  for (int j = j0; j < j1; j += kTok * kMoveUnits) {
    __syncthreads();                      // all of this range is read before any of it is written
    T val[kMoveUnits];
    int at[kMoveUnits];
#pragma unroll
    for (int u = 0; u < kMoveUnits; ++u) { val[u] = cur[u]; at[u] = dst[u]; }
    if (j + kTok * kMoveUnits < j1) read(j + kTok * kMoveUnits);
#pragma unroll
    for (int u = 0; u < kMoveUnits; ++u)
      if (at[u] >= 0) mine[static_cast<long>(at[u]) * row_elems] = val[u];
  }
}

// places [j0, j1) of the values of fp8 pages, j0 a multiple of 16
NRL_DEVICE void move_transposed(uint4* v, long step, const int* from, const int* to, const int* kept, const uint16_t* bits, int j0, int j1) {
  __shared__ uint32_t span[kSpanPages * 128 * kSpanRow];
  __shared__ uint32_t left[2][128 * kSpanRow];                        // places of a page that is not full yet: read by one span, written by it for the next
  __shared__ __align__(16) uint32_t place[kMoveThreads + 16];         // of the span's kept tokens, from the first place of their page on: the byte of element 0
  const int tid = threadIdx.x, d = tid & 127, warp_half = tid >> 7;
  __shared__ int ahead[2];                                            // the page of the first kept token behind the span, as far as the threads have looked
  const int last = kept[j1 - 1] >> 4;
  int page = kept[j0] >> 4, j = j0, turn = 0;
  uint4 cur[kMoveUnits];
  auto read = [&](int at) {
#pragma unroll
    for (int u = 0; u < kMoveUnits; ++u) {
      const int pg = at + u * 2 + warp_half;
      if (pg <= last && bits[pg] != 0) cur[u] = v[from[pg] * step + d];
    }
  };
  read(page);
  if (tid < 2) ahead[tid] = INT_MAX;
  __syncthreads();
  while (j < j1) {
    const int t = j + tid < j1 ? kept[j + tid] : -1;
    const bool here = t >= 0 && (t >> 4) < page + kSpanPages;
#pragma unroll
    for (int u = 0; u < kMoveUnits; ++u) {
      uint32_t* w = span + ((u * 2 + warp_half) * 128 + d) * kSpanRow;
      w[0] = cur[u].x; w[1] = cur[u].y; w[2] = cur[u].z; w[3] = cur[u].w;
    }
    if (here) place[(j & 15) + tid] = ((t >> 4) - page) * 128 * kSpanRow * 4 + (t & 15);
    const int warp_ahead = __reduce_min_sync(0xffffffffu, t >= 0 && !here ? t >> 4 : INT_MAX);
    if ((tid & 31) == 0 && warp_ahead != INT_MAX) atomicMin(&ahead[turn], warp_ahead);
    const int to_j = j + __syncthreads_count(here);                   // places [j, to_j) come from this span
    const int next = ahead[turn] != INT_MAX ? ahead[turn] : page + kSpanPages;         // (pages between that keep nothing are passed over)
    if (to_j < j1) read(next);
    const uint8_t* bytes = reinterpret_cast<const uint8_t*>(span) + d * kSpanRow * 4;
    for (int pg = (j >> 4) + warp_half; pg * 16 < to_j; pg += 2) {
      uint32_t word[4];
      const int k0 = max(0, j - pg * 16), k1 = min(16, to_j - pg * 16);          // places of this page that are put now
      const uint32_t* at = place + (pg - (j >> 4)) * 16;
      if (k0 == 0 && k1 == 16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 four = *reinterpret_cast<const uint4*>(at + 4 * i);
          const uint32_t a = bytes[four.x], b = bytes[four.y], c = bytes[four.z], e = bytes[four.w];
          word[i] = __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, e, 0x0040), 0x5410);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          word[i] = k0 > i * 4 ? left[turn][d * kSpanRow + i] : 0u;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int k = i * 4 + b;
            if (k >= k0 && k < k1) word[i] = (word[i] & ~(0xffu << (8 * b))) | (static_cast<uint32_t>(bytes[at[k]]) << (8 * b));
          }
        }
      }
      if (k1 == 16) {
        v[to[pg] * step + d] = make_uint4(word[0], word[1], word[2], word[3]);
      } else if (to_j < j1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) left[turn ^ 1][d * kSpanRow + i] = word[i];
      } else {                                                        // places behind the last stay as they were
        const uint4 old = v[to[pg] * step + d];
        const uint32_t ow[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = k1 - i * 4;                                   // bytes of this word that are new
          if (k < 4) word[i] = k <= 0 ? ow[i] : (word[i] & (0xffffffffu >> (32 - 8 * k))) | (ow[i] & (0xffffffffu << (8 * k)));
        }
        v[to[pg] * step + d] = make_uint4(word[0], word[1], word[2], word[3]);
      }
    }
    j = to_j;
    page = next;
    if (tid == 0) ahead[turn ^ 1] = INT_MAX;
    turn ^= 1;
    __syncthreads();                                                  // `left` is written, span and places are read
  }
}

struct MoveRow {
  const int *from, *to, *kept;
  long row;
  int kvh, j0, j1;                        // places [j0, j1) of a row-head
};
template <bool IN_PLACE>
NRL_DEVICE MoveRow move_row(const MoveParams& p) {
  const EvictCall& e = p.e;
  const int seq = blockIdx.x, kvh = blockIdx.y % e.Hkv, range = blockIdx.y / e.Hkv, n = min(e.context_lens[seq], e.max_tokens), count = max(0, min(n, e.keep));
  const long row = static_cast<long>(seq) * e.Hkv + kvh;
  const int j0 = IN_PLACE ? 0 : range * p.range, j1 = IN_PLACE ? (n > e.keep ? count : 0) : min(count, j0 + p.range);
  return {e.block_tables + static_cast<long>(seq) * e.max_blocks, p.out_tables + static_cast<long>(seq) * p.out_blocks, e.kept + row * e.keep, row, kvh, j0, j1};
}

// A block has, by z: the values of fp8 pages, which take longest; a slice of the keys; of bf16 values; fp8 scales; the scores of what is kept.
template <bool IN_PLACE, bool FP8>
__global__ void __launch_bounds__(kMoveThreads, IN_PLACE ? 2 : 4) kv_move_kernel(const MoveParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const EvictCall& e = p.e;
  const int z = static_cast<int>(blockIdx.z) - (FP8 ? 1 : 0), last = FP8 ? p.key_slices + 2 : 2 * p.key_slices;
  if (z == last) {
    const int kvh = blockIdx.y % e.Hkv;
    const long row = static_cast<long>(blockIdx.x) * e.Hkv + kvh;
    const int* kept = e.kept + row * e.keep;
    float* to = e.kept_scores + row * e.keep;
    const float* sc = e.scores + static_cast<long>(blockIdx.x) * e.score_row + kvh * e.score_head;
    const int j0 = IN_PLACE ? 0 : blockIdx.y / e.Hkv * p.range, j1 = IN_PLACE || (blockIdx.y / e.Hkv + 1) * e.Hkv == gridDim.y ? e.keep : min(e.keep, j0 + p.range);
#pragma unroll 4
    for (int j = j0 + threadIdx.x; j < j1; j += kMoveThreads) {
      const int t = kept[j];
      to[j] = t >= 0 ? sc[t] : 0.f;
    }
    return;
  }
  const MoveRow m = move_row<IN_PLACE>(p);
  if (m.j0 >= m.j1) return;
  if constexpr (FP8) {
    if (z < 0) {
      const uint16_t* bits = reinterpret_cast<const uint16_t*>(e.bits + m.row * ((e.max_tokens + 31) / 32));
      move_transposed(static_cast<uint4*>(e.v_cache) + static_cast<long>(m.kvh) * 128, static_cast<long>(e.Hkv) * 128, m.from, m.to, m.kept, bits, m.j0, m.j1);
      return;
    }
  }
  const bool keys = z < p.key_slices;
  if (FP8 && !keys)
    move_rows<IN_PLACE, float, 1>(z == p.key_slices ? e.k_scale : e.v_scale, 1, 0, m.from, m.to, m.kept, m.j0, m.j1, e.Hkv, m.kvh);
  else
    move_rows<IN_PLACE, uint4, move_pieces(IN_PLACE, FP8)>(static_cast<uint4*>(keys ? e.k_cache : e.v_cache), FP8 ? 8 : 16, keys ? z : z - p.key_slices, m.from, m.to, m.kept, m.j0, m.j1,
                                            e.Hkv, m.kvh);
}

}  // namespace nrl

using namespace nrl;

namespace {

template <int WARPS>
cudaError_t launch_select(const EvictCall& c, int cluster, int tokens, cudaStream_t s) {
  static PerDevice<bool> configured;
  const cudaError_t e = allow_smem(configured, kv_select_kernel<WARPS>, kSelTokens * 4);
  if (e != cudaSuccess) return e;
  const dim3 grid(c.S * cluster, c.Hkv);
  launch_dependent_clusters(kv_select_kernel<WARPS>, grid, WARPS * 32, tokens * 4, s, cluster, c, cluster);       // (one block a cluster: 60 us where a plain launch takes 64)
  return cudaGetLastError();
}

template <bool IN_PLACE>
cudaError_t launch_moves(MoveParams p, int num_sms, cudaStream_t s) {
  const EvictCall& c = p.e;
  const bool fp8 = c.k_scale != nullptr;
  const int places = c.keep < c.max_tokens ? c.keep : c.max_tokens;
  p.range = move_range(fp8);
  p.key_slices = (fp8 ? 8 : 16) / move_pieces(IN_PLACE, fp8);
  while (!IN_PLACE && p.range > kMoveLeast && static_cast<long>(c.S) * c.Hkv * ((places + p.range - 1) / p.range) < 2L * num_sms) p.range /= 2;
  while (static_cast<long>(c.Hkv) * ((places + p.range - 1) / p.range) > 65535) p.range *= 2;          // (a grid's second dimension)
  const int ranges = IN_PLACE ? 1 : (places + p.range - 1) / p.range;
  const dim3 grid(c.S, c.Hkv * ranges, (fp8 ? p.key_slices + 3 : 2 * p.key_slices) + 1);
  if (fp8) launch_dependent(kv_move_kernel<IN_PLACE, true>, grid, kMoveThreads, 0, s, p);
  else launch_dependent(kv_move_kernel<IN_PLACE, false>, grid, kMoveThreads, 0, s, p);
  return cudaGetLastError();
}

}  // namespace

extern "C" cudaError_t nrl_kv_evict(const EvictCall* c, int num_sms, cudaStream_t s) {
  if (c->S == 0) return cudaSuccess;
  // blocks a row-head: as many as find an SM, but 2048 tokens each at least; and as many as hold its scores
  int cluster = 1;
  while (cluster < kSelCluster && ((static_cast<long>(c->S) * c->Hkv * cluster * 2 <= 2L * num_sms && c->max_tokens >= cluster * 2 * 2048) ||
                                   c->max_tokens > static_cast<long>(cluster) * kSelTokens)) cluster *= 2;
  const int tokens = ((c->max_tokens + 31) / 32 + cluster - 1) / cluster * 32;
  if (tokens > kSelTokens) return cudaErrorInvalidValue;
  cudaError_t e = tokens <= 2048 ? launch_select<4>(*c, cluster, tokens, s) : tokens <= 3840 ? launch_select<8>(*c, cluster, tokens, s) : launch_select<16>(*c, cluster, tokens, s);
  if (e != cudaSuccess) return e;
  MoveParams p;
  p.e = *c;
  p.out_tables = c->out_tables != nullptr ? c->out_tables : c->block_tables;
  p.out_blocks = c->out_tables != nullptr ? c->out_blocks : c->max_blocks;
  return c->out_tables != nullptr ? launch_moves<false>(p, num_sms, s) : launch_moves<true>(p, num_sms, s);
}
