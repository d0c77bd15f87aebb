// Decode attention of rows that share their first tokens: the prefix's part.
//
// The query rows of a group (samples x G heads of a kv head) are tiles of up to 64; every key and value of the prefix is read from memory once for a tile.
// The prefixes' steps of 64 tokens, of all tiles one behind the other, are dealt to blocks in equal runs (decode_flat.cu: decode_plan); a run that meets a tile leaves a
// part of it, (maximum, sum, unnormalised result), which is decode_join's.
//
// Block = 4 warps of 16 rows; 4 pages a step through shared memory (cp.async, three stages), mma.sync m16n8k16.  fp8 pages are dequantised on the operand fragments as in
// attention_decode_fp8.cu.  Bound by the latency of a step (fp8, 96 rows: 2 warps a scheduler, of which one issues in 31 % of the cycles, the tensor pipe 25 %): so an
// fp8 warp holds the scores of two pages at a time and its queries in shared memory, in 168 registers, for three blocks an SM (32 x 2 x 2000 tokens of 96 rows 46 -> 41 us).
// Pages turned into f16 tiles once for the block, in place of once for every warp, took as long: what it saves in conversions it waits at one more barrier.
// On tcgen05, tiles of 128 rows against blocks of 128 keys with two streams of scores and a warpgroup each for their softmax, 13 groups x 4 kv heads x 4096 fp8
// tokens of 112 rows took 44 us and 64 x 2 x 390 bf16 tokens of 48 rows 21: a tile of few rows costs the tensor pipe as much as a full one, and fp8 pages' way
// through registers into its tiles competes with the softmax for issue slots.
#pragma once
#include "common.cuh"
#include "decode_runs.cuh"
#include "fp8_fragments.cuh"

namespace nrl {

constexpr int kPreWarps = kPrefixRows / 16;
constexpr int kPreStages = 3;
constexpr int kPreStep = kPrefixKeys / 16;        // pages a step

template <bool FP8>
struct PreSmem {
  static constexpr int kHalf = FP8 ? 2048 : 4096;                    // K or V of a page
  static constexpr int kPageSize = 2 * kHalf + (FP8 ? 128 : 0);      // K, V, k_scale[16], v_scale[16]
  static constexpr int kStage = kPreStep * kPageSize;
  static constexpr int kTotal = kPreStages * kStage + (FP8 ? kPrefixRows * 128 * 2 : 0);      // and the tile's queries
  static constexpr int kPages = FP8 ? 2 : 4;                         // whose scores a warp holds at a time
};

// Where a run stands: steps [step, step + n) of a tile
struct PreWalk {
  int g, h, tile, step, n;
  int first, rows;                                 // the group's first row; query rows of a kv head
  int shared, tiles, steps;                        // tokens that any row sees; the group's tiles and steps
  int left, at;                                    // steps of the run from this segment on; kv head x tiles + tile
  NRL_DEVICE PreWalk(const FlatParams& p, int run) {
    const int4 all = p.groups[p.n_groups], start = p.prefix_starts[run];               // all steps, steps a run
    left = min(all.y, all.x - run * all.y);
    at = start.y;
    if (left > 0) enter(p, start.x, start.z);
  }
  NRL_DEVICE void enter(const FlatParams& p, int group, int from) {
    const int4 x = p.groups[group];
    g = group; step = from;
    first = p.cu_groups[g];
    steps = x.y; shared = x.z; rows = x.w;
    tiles = prefix_tiles(rows);
    h = at / tiles; tile = at - h * tiles;
    n = min(left, steps - step);
  }
  NRL_DEVICE void next(const FlatParams& p) {
    left -= n;
    if (left <= 0) return;
    int group = g;
    if (++at == p.Hkv * tiles) {
      at = 0;
      do ++group; while (p.groups[group].y == 0);
    }
    enter(p, group, 0);
  }
};

NRL_DEVICE void pre_ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
NRL_DEVICE void pre_ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <bool FP8>
NRL_DEVICE void pre_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (FP8)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// run `run` of the prefixes, by a whole block
template <bool FP8>
NRL_DEVICE void decode_prefix_run(const FlatParams& p, uint8_t* smem, int run) {
  using L = PreSmem<FP8>;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;

  PreWalk in(p, run);                                                   // what is copied next: step in.step + in_j
  const int total = max(0, in.left);
  int in_j = 0, n_in = 0, id = 0;                                    // its page numbers, in the lanes
  auto look_up = [&]() {
    const int page = (in.step + in_j) * kPreStep + lane;
    id = in.left > 0 && lane < kPreStep && page * 16 < in.shared ? p.block_tables[static_cast<long>(in.first) * p.max_blocks + page] : 0;
  };
  look_up();
  auto issue = [&]() {
    if (n_in < total) {
      uint8_t* st = smem + (n_in % kPreStages) * L::kStage;
#pragma unroll
      for (int u = 0; u < kPreStep; ++u) {
        const long pg = static_cast<long>(__shfl_sync(0xffffffffu, id, u)) * p.Hkv + in.h;
        if (((in.step + in_j) * kPreStep + u) * 16 >= in.shared) break;
        const uint8_t *ksrc = p.k + pg * L::kHalf, *vsrc = p.v + pg * L::kHalf;
        uint8_t *kd = st + u * L::kPageSize, *vd = kd + L::kHalf;
        if (FP8) {
          cp_async_16(kd + (tid >> 3) * 128 + (((tid & 7) ^ k_sigma(tid >> 3)) << 4), ksrc + tid * 16);
          cp_async_16(vd + tid * 16, vsrc + tid * 16);
          if (tid < 8) cp_async_16(vd + L::kHalf + tid * 16, (tid < 4 ? p.ks : p.vs) + pg * 16 + (tid & 3) * 4);
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int chunk = tid + j * 128, at = (chunk >> 4) * 256 + (((chunk & 15) ^ ((chunk >> 4) & 7)) << 4);
            cp_async_16(kd + at, ksrc + chunk * 16);
            cp_async_16(vd + at, vsrc + chunk * 16);
          }
        }
      }
      ++n_in;
      if (++in_j == in.n) {
        in_j = 0;
        in.next(p);
      }
      look_up();
    }
    cp_async_commit();
  };
  issue();
  issue();

  int n_out = 0;
  for (PreWalk w(p, run); w.left > 0; w.next(p)) {
    const int shared = w.shared;
    // this thread's rows: g and g + 8 of the warp's sixteen
    int limit[2];
    bool real[2];
    const __nv_bfloat16* qrow[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = w.tile * kPrefixRows + warp * 16 + g + i * 8;
      real[i] = at < w.rows;
      const int seq = w.first + (real[i] ? at / p.G : 0), r = real[i] ? at % p.G : 0;
      limit[i] = real[i] ? min(shared, p.context_lens[seq]) : 0;
      qrow[i] = p.q + seq * p.q_stride_s + (w.h * p.G + r) * 128;
    }
    int all_see = real[1] ? min(limit[0], limit[1]) : real[0] ? limit[0] : shared;          // what all rows of the warp see
    all_see = __reduce_min_sync(0xffffffffu, all_see);
    const bool busy = w.tile * kPrefixRows + warp * 16 < w.rows;     // a warp without rows only copies
    uint32_t qf[FP8 ? 1 : 8][4];                                     // fp8: in shared memory, as the lanes hold them
    uint4* const q_frags = reinterpret_cast<uint4*>(smem + kPreStages * L::kStage) + warp * 256 + lane;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      uint32_t f[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (FP8) {
          const uint2 raw = *reinterpret_cast<const uint2*>(qrow[i] + (ks >> 2) * 64 + t4 * 16 + (ks & 3) * 4);
          const float2 a = unpack_bf16x2(raw.x), b = unpack_bf16x2(raw.y);
          f[i] = real[i] ? pack_f16x2(a.x, a.y) : 0u;
          f[2 + i] = real[i] ? pack_f16x2(b.x, b.y) : 0u;
        } else {
          f[i] = real[i] ? *reinterpret_cast<const uint32_t*>(qrow[i] + ks * 16 + t4 * 2) : 0u;
          f[2 + i] = real[i] ? *reinterpret_cast<const uint32_t*>(qrow[i] + ks * 16 + 8 + t4 * 2) : 0u;
        }
      }
      if (FP8) q_frags[ks * 32] = make_uint4(f[0], f[1], f[2], f[3]);
      else qf[FP8 ? 0 : ks][0] = f[0], qf[FP8 ? 0 : ks][1] = f[1], qf[FP8 ? 0 : ks][2] = f[2], qf[FP8 ? 0 : ks][3] = f[3];
    }
    float o[16][4];
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f}, factor = FP8 ? __uint_as_float(kMostFactor) : 1.f;          // (of weights, and of o)

    for (int step = w.step; step < w.step + w.n; ++step, ++n_out) {
      cp_async_wait<1>();
      __syncthreads();
      uint8_t* st = smem + (n_out % kPreStages) * L::kStage;
      const int key0 = step * kPrefixKeys;
      if (key0 + kPrefixKeys > shared) {
        // values (and scales) behind the prefix, whatever they are, meet weights of 0 as zeros; so do pages that were not fetched
        for (int u = 0; u < kPreStep; ++u) {
          uint8_t* vd = st + u * L::kPageSize + L::kHalf;
          const int n = max(0, min(16, shared - key0 - u * 16));
          if (FP8) {
            uint32_t* x = reinterpret_cast<uint32_t*>(vd + tid * 16);
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (n < c * 4 + 4) x[c] = n <= c * 4 ? 0u : x[c] & (0xffffffffu >> (32 - 8 * (n - c * 4)));
            if (tid < 16 && tid >= n) reinterpret_cast<float*>(vd + L::kHalf)[16 + tid] = 0.f;
          } else {
            for (int i = n * 16 + tid; i < 256; i += kPreWarps * 32) *reinterpret_cast<uint4*>(vd + i * 16) = make_uint4(0, 0, 0, 0);
          }
        }
        __syncthreads();
      }
      issue();                                                       // into the stage that all have left
      if (!busy) continue;
#pragma unroll 1
      for (int u0 = 0; u0 < kPreStep; u0 += L::kPages) {
      // ---- S = Q K^T ----
      float s[L::kPages * 2][4];
#pragma unroll
      for (int n = 0; n < 2 * L::kPages; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      if constexpr (FP8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint4 q[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) q[i] = q_frags[(4 * h + i) * 32];
#pragma unroll
          for (int u = 0; u < L::kPages; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int krow = ((g >> 1) << 2) + 2 * j + (g & 1);
              const uint4 w4 = lds128(smem_u32(st + (u0 + u) * L::kPageSize) + krow * 128 + (((4 * h + t4) ^ k_sigma(g)) << 4));
              const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t a[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
                pre_mma<true>(s[2 * u + j], a, e4m3x2_to_f16x2(w[i] & 0xFFFFu), e4m3x2_to_f16x2(w[i] >> 16));
              }
            }
        }
      } else {
#pragma unroll
        for (int u = 0; u < L::kPages; ++u) {
          const uint32_t kb = smem_u32(st + (u0 + u) * L::kPageSize);
          const int mrow = (lane & 7) + (lane >> 4) * 8, mcol = (lane >> 3) & 1;
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            uint32_t kf[4];
            pre_ldmatrix_x4(kf, kb + mrow * 256 + (((ks * 2 + mcol) ^ (mrow & 7)) << 4));
            pre_mma<false>(s[2 * u], qf[ks], kf[0], kf[1]);
            pre_mma<false>(s[2 * u + 1], qf[ks], kf[2], kf[3]);
          }
        }
      }
      // ---- scale, mask, online softmax on rows g and g + 8.  Key of column (u, j, e): bf16 16 u + 8 j + 2 t + e, fp8 16 u + 4 t + 2 j + e ----
      float vsc[L::kPages][4];
      float top[2] = {-INFINITY, -INFINITY};
      const bool whole = key0 + kPrefixKeys <= all_see;
#pragma unroll
      for (int u = 0; u < L::kPages; ++u) {
        float ksc[4] = {1.f, 1.f, 1.f, 1.f};
        if (FP8) {
          const uint32_t sb = smem_u32(st + (u0 + u) * L::kPageSize + 2 * L::kHalf);
          const uint4 kr = lds128(sb + t4 * 16), vr = lds128(sb + 64 + t4 * 16);
          ksc[0] = __uint_as_float(kr.x) * p.scale_log2; ksc[1] = __uint_as_float(kr.y) * p.scale_log2;
          ksc[2] = __uint_as_float(kr.z) * p.scale_log2; ksc[3] = __uint_as_float(kr.w) * p.scale_log2;
          vsc[u][0] = __uint_as_float(vr.x); vsc[u][1] = __uint_as_float(vr.y); vsc[u][2] = __uint_as_float(vr.z); vsc[u][3] = __uint_as_float(vr.w);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + (u0 + u) * 16 + (FP8 ? t4 * 4 + 2 * j + (e & 1) : j * 8 + t4 * 2 + (e & 1));
            float& x = s[2 * u + j][e];
            x *= FP8 ? ksc[2 * j + (e & 1)] : p.scale_log2;
            if (!whole && key >= limit[e >> 1]) x = -INFINITY;
            top[e >> 1] = fmaxf(top[e >> 1], x);
          }
      }
      float m_sub[2], corr[2], sum[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
        const float m_new = fmaxf(m_run[i], top[i]);
        m_sub[i] = m_new == -INFINITY ? 0.f : m_new;
        corr[i] = exp2f(m_run[i] - m_sub[i]);                          // 0 while nothing has been seen
        m_run[i] = m_new;
      }
      if constexpr (FP8) {
        float most = 0.f;
#pragma unroll
        for (int u = 0; u < L::kPages; ++u) most = fmaxf(most, fmaxf(fmaxf(vsc[u][0], vsc[u][1]), fmaxf(vsc[u][2], vsc[u][3])));
        const float before = inverse_factor(factor);
        factor = shrink_factor(factor, most);
#pragma unroll
        for (int u = 0; u < L::kPages; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) vsc[u][i] *= factor;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          l_run[i] *= corr[i];
          corr[i] *= factor * before;
        }
      }
      uint32_t pa[L::kPages][4];
#pragma unroll
      for (int u = 0; u < L::kPages; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float p0 = exp2f(s[2 * u + j][2 * i] - m_sub[i]), p1 = exp2f(s[2 * u + j][2 * i + 1] - m_sub[i]);
            sum[i] += p0 + p1;
            pa[u][2 * j + i] = FP8 ? pack_f16x2(p0 * vsc[u][2 * j], p1 * vsc[u][2 * j + 1]) : pack_bf16x2(p0, p1);
          }
#pragma unroll
      for (int i = 0; i < 2; ++i) l_run[i] = FP8 ? l_run[i] + sum[i] : l_run[i] * corr[i] + sum[i];
      if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) { o[i][0] *= corr[0]; o[i][1] *= corr[0]; o[i][2] *= corr[1]; o[i][3] *= corr[1]; }
      }
      // ---- O += P V ----
#pragma unroll
      for (int u = 0; u < L::kPages; ++u) {
        const uint32_t vb = smem_u32(st + (u0 + u) * L::kPageSize + L::kHalf);
        if (FP8) {
#pragma unroll
          for (int nd = 0; nd < 16; ++nd) {
            const uint32_t w = lds32(vb + (nd * 8 + g) * 16 + t4 * 4);
            pre_mma<true>(o[nd], pa[u], e4m3x2_to_f16x2(w & 0xFFFFu), e4m3x2_to_f16x2(w >> 16));
          }
        } else {
          const int mrow = (lane & 7) + ((lane >> 3) & 1) * 8, mcol = lane >> 4;
#pragma unroll
          for (int nd = 0; nd < 8; ++nd) {
            uint32_t vf[4];
            pre_ldmatrix_x4_trans(vf, vb + mrow * 256 + (((nd * 2 + mcol) ^ (mrow & 7)) << 4));
            pre_mma<false>(o[nd * 2], pa[u], vf[0], vf[1]);
            pre_mma<false>(o[nd * 2 + 1], pa[u], vf[2], vf[3]);
          }
        }
      }
      }
    }
    // ---- the part of every row; one without keys is (-inf, 0, 0) ----
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 1);
      l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 2);
      if (!real[i]) continue;
      const long at = prefix_part_row(p, w.first, w.h, w.rows, w.tile * kPrefixRows + warp * 16 + g + i * 8) + static_cast<long>(kPrefixRows) * run;
      float* dst = p.prefix_o + at * 128 + t4 * 2;
      const float f = FP8 ? inverse_factor(factor) : 1.f;
#pragma unroll
      for (int nd = 0; nd < 16; ++nd)
        *reinterpret_cast<float2*>(dst + nd * 8) = make_float2(o[nd][2 * i] * f, o[nd][2 * i + 1] * f);
      if (t4 == 0) *reinterpret_cast<float2*>(p.prefix_ml + at * 2) = make_float2(m_run[i], l_run[i]);
    }
  }
  cp_async_wait<0>();
}

}  // namespace nrl
