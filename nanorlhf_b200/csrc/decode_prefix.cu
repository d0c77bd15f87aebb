// Decode attention of rows that share their first tokens: the prefix once per group, the rest per row.
//
//   out = sum_parts 2^(m_p - M) O_p / sum_parts 2^(m_p - M) l_p,  a part being the (maximum, sum, unnormalised result) of some of the row's keys
//
// The prefix's parts are formed here: the query rows of a group (samples x G heads of a kv head) are up to 64 rows of a tile, every key and value of the prefix is
// read from memory once for all of them.  The rest of a row's tokens are decode_flat.cu's, which joins the parts.
//
// Block = 4 warps of 16 rows; 64 keys (4 pages) a step through shared memory (cp.async, three stages), mma.sync m16n8k16.  fp8 pages are dequantised on the
// operand fragments as in attention_decode_fp8.cu.
#include "common.cuh"
#include "fp8_fragments.cuh"
#include "group_kernels.h"
#include "launch.h"
#include "per_device.h"

namespace nrl {

constexpr int kPreWarps = 4;
constexpr int kPreRows = kPreWarps * 16;          // query rows of a block
constexpr int kPreStages = 3;
constexpr int kPreStep = 4;                       // pages a step
constexpr float kPreScale = 1024.f;               // of fp8 weights, which are f16 (2^10: small ones stay normal)

template <bool FP8>
struct PreSmem {
  static constexpr int kHalf = FP8 ? 2048 : 4096;                    // K or V of a page
  static constexpr int kPageSize = 2 * kHalf + (FP8 ? 128 : 0);      // K, V, k_scale[16], v_scale[16]
  static constexpr int kStage = kPreStep * kPageSize;
  static constexpr int kTotal = kPreStages * kStage;
};

struct PrefixParams {
  const __nv_bfloat16* q;
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int *block_tables, *context_lens, *cu_groups, *shared;
  float *part_o, *part_ml;
  long q_stride_s;
  int S, max_blocks, Hkv, G, prefix_parts, tiles;
  float scale_log2;
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

template <bool FP8>
__global__ void __launch_bounds__(kPreWarps * 32, 2) decode_prefix_kernel(const PrefixParams p) {
  pdl_wait();
  pdl_launch_dependents();
  using L = PreSmem<FP8>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int group = blockIdx.x, kvh = blockIdx.y, part = blockIdx.z / p.tiles;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int seq0 = p.cu_groups[group], n_rows = (min(p.cu_groups[group + 1], p.S) - seq0) * p.G;
  const int shared = min(p.shared[group], p.max_blocks * 16);
  if (shared <= 0) return;
  const int n_steps = (shared + 16 * kPreStep - 1) / (16 * kPreStep), per_part = (n_steps + p.prefix_parts - 1) / p.prefix_parts;
  const int step_lo = part * per_part, step_hi = min(n_steps, step_lo + per_part);
  const int n_pages = (shared + 15) / 16;
  const int* bt = p.block_tables + static_cast<long>(seq0) * p.max_blocks;

  int ids[kPreStep];                                                 // pages of the step that is copied next
  auto look_up = [&](int step) {
#pragma unroll
    for (int u = 0; u < kPreStep; ++u) ids[u] = step < step_hi && step * kPreStep + u < n_pages ? bt[step * kPreStep + u] : 0;
  };
  auto issue = [&](int step) {
    if (step < step_hi) {
      uint8_t* st = smem + ((step - step_lo) % kPreStages) * L::kStage;
#pragma unroll
      for (int u = 0; u < kPreStep; ++u) {
        if (step * kPreStep + u >= n_pages) break;
        const long pg = static_cast<long>(ids[u]) * p.Hkv + kvh;
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
    }
    cp_async_commit();
    look_up(step + 1);
  };

  // (one tile a block; more only where a group is larger than was said)
  for (int tile = blockIdx.z - part * p.tiles; tile * kPreRows < n_rows; tile += p.tiles) {
    // this thread's rows: g and g + 8 of the warp's sixteen
    int row[2], limit[2];
    bool real[2];
    const __nv_bfloat16* qrow[2];
  #pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = tile * kPreRows + warp * 16 + g + i * 8;
      real[i] = at < n_rows;
      const int seq = seq0 + (real[i] ? at / p.G : 0), r = real[i] ? at % p.G : 0;
      row[i] = (seq * p.Hkv + kvh) * p.prefix_parts * 8 + r;          // of the parts, without the part (S * Hkv * parts * 8 is below 2^31: checked on the host)
      limit[i] = real[i] ? min(shared, p.context_lens[seq]) : 0;
      qrow[i] = p.q + seq * p.q_stride_s + (kvh * p.G + r) * 128;
    }
    const bool busy = tile * kPreRows + warp * 16 < n_rows;            // a warp without rows only copies
    uint32_t qf[8][4];
  #pragma unroll
    for (int ks = 0; ks < 8; ++ks)
  #pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (FP8) {
          const uint2 raw = *reinterpret_cast<const uint2*>(qrow[i] + (ks >> 2) * 64 + t4 * 16 + (ks & 3) * 4);
          const float2 a = unpack_bf16x2(raw.x), b = unpack_bf16x2(raw.y);
          qf[ks][i] = real[i] ? pack_f16x2(a.x, a.y) : 0u;
          qf[ks][2 + i] = real[i] ? pack_f16x2(b.x, b.y) : 0u;
        } else {
          qf[ks][i] = real[i] ? *reinterpret_cast<const uint32_t*>(qrow[i] + ks * 16 + t4 * 2) : 0u;
          qf[ks][2 + i] = real[i] ? *reinterpret_cast<const uint32_t*>(qrow[i] + ks * 16 + 8 + t4 * 2) : 0u;
        }
      }

    float o[16][4];
  #pragma unroll
    for (int i = 0; i < 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};

    look_up(step_lo);
    issue(step_lo);
    issue(step_lo + 1);
    for (int step = step_lo; step < step_hi; ++step) {
      cp_async_wait<1>();
      __syncthreads();
      uint8_t* st = smem + ((step - step_lo) % kPreStages) * L::kStage;
      const int key0 = step * kPreStep * 16, pages = min(kPreStep, n_pages - step * kPreStep);
      if (pages < kPreStep || key0 + kPreStep * 16 > shared) {
        // values (and scales) behind the prefix, whatever they are, meet weights of 0 as zeros; so do pages that were not fetched
        for (int u = 0; u < kPreStep; ++u) {
          uint8_t* vd = st + u * L::kPageSize + L::kHalf;
          const int n = max(0, min(16, shared - key0 - u * 16));
          if (FP8) {
            uint32_t* w = reinterpret_cast<uint32_t*>(vd + tid * 16);
  #pragma unroll
            for (int c = 0; c < 4; ++c)
              if (n < c * 4 + 4) w[c] = n <= c * 4 ? 0u : w[c] & (0xffffffffu >> (32 - 8 * (n - c * 4)));
            if (tid < 16 && tid >= n) reinterpret_cast<float*>(vd + L::kHalf)[16 + tid] = 0.f;
          } else {
            for (int i = n * 16 + tid; i < 256; i += kPreWarps * 32) *reinterpret_cast<uint4*>(vd + i * 16) = make_uint4(0, 0, 0, 0);
          }
        }
        __syncthreads();
      }
      issue(step + 2);
      if (!busy) continue;
      // ---- S = Q K^T ----
      float s[kPreStep * 2][4];
  #pragma unroll
      for (int u = 0; u < kPreStep; ++u) {
        const uint32_t kb = smem_u32(st + u * L::kPageSize);
  #pragma unroll
        for (int j = 0; j < 2; ++j) s[2 * u + j][0] = s[2 * u + j][1] = s[2 * u + j][2] = s[2 * u + j][3] = 0.f;
        if (FP8) {
  #pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int krow = ((g >> 1) << 2) + 2 * j + (g & 1);
  #pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint4 w4 = lds128(kb + krow * 128 + (((4 * h + t4) ^ k_sigma(g)) << 4));
              const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
  #pragma unroll
              for (int i = 0; i < 4; ++i) pre_mma<true>(s[2 * u + j], qf[4 * h + i], e4m3x2_to_f16x2(w[i] & 0xFFFFu), e4m3x2_to_f16x2(w[i] >> 16));
            }
          }
        } else {
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
      float vsc[kPreStep][4];
      float top[2] = {-INFINITY, -INFINITY};
  #pragma unroll
      for (int u = 0; u < kPreStep; ++u) {
        float ksc[4] = {1.f, 1.f, 1.f, 1.f};
        if (FP8) {
          const uint32_t sb = smem_u32(st + u * L::kPageSize + 2 * L::kHalf);
          const uint4 kr = lds128(sb + t4 * 16), vr = lds128(sb + 64 + t4 * 16);
          ksc[0] = __uint_as_float(kr.x); ksc[1] = __uint_as_float(kr.y); ksc[2] = __uint_as_float(kr.z); ksc[3] = __uint_as_float(kr.w);
          vsc[u][0] = __uint_as_float(vr.x); vsc[u][1] = __uint_as_float(vr.y); vsc[u][2] = __uint_as_float(vr.z); vsc[u][3] = __uint_as_float(vr.w);
        }
  #pragma unroll
        for (int j = 0; j < 2; ++j)
  #pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + u * 16 + (FP8 ? t4 * 4 + 2 * j + (e & 1) : j * 8 + t4 * 2 + (e & 1));
            float& x = s[2 * u + j][e];
            x = key < limit[e >> 1] ? x * (ksc[2 * j + (e & 1)] * p.scale_log2) : -INFINITY;
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
      uint32_t pa[kPreStep][4];
  #pragma unroll
      for (int u = 0; u < kPreStep; ++u)
  #pragma unroll
        for (int j = 0; j < 2; ++j)
  #pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float p0 = exp2f(s[2 * u + j][2 * i] - m_sub[i]), p1 = exp2f(s[2 * u + j][2 * i + 1] - m_sub[i]);
            sum[i] += p0 + p1;
            pa[u][2 * j + i] = FP8 ? pack_f16x2(p0 * (vsc[u][2 * j] * kPreScale), p1 * (vsc[u][2 * j + 1] * kPreScale)) : pack_bf16x2(p0, p1);
          }
  #pragma unroll
      for (int i = 0; i < 2; ++i) l_run[i] = l_run[i] * corr[i] + sum[i];
  #pragma unroll
      for (int i = 0; i < 16; ++i) { o[i][0] *= corr[0]; o[i][1] *= corr[0]; o[i][2] *= corr[1]; o[i][3] *= corr[1]; }
      // ---- O += P V ----
  #pragma unroll
      for (int u = 0; u < kPreStep; ++u) {
        const uint32_t vb = smem_u32(st + u * L::kPageSize + L::kHalf);
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
    cp_async_wait<0>();
    // ---- the part of every row; one without keys is (-inf, 0, 0) ----
  #pragma unroll
    for (int i = 0; i < 2; ++i) {
      l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 1);
      l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 2);
      if (!real[i]) continue;
      const long base = row[i] + part * 8;
      float* dst = p.part_o + base * 128 + t4 * 2;
  #pragma unroll
      for (int nd = 0; nd < 16; ++nd)
        *reinterpret_cast<float2*>(dst + nd * 8) = make_float2(o[nd][2 * i] * (FP8 ? 1.f / kPreScale : 1.f), o[nd][2 * i + 1] * (FP8 ? 1.f / kPreScale : 1.f));
      if (t4 == 0) *reinterpret_cast<float2*>(p.part_ml + base * 2) = make_float2(m_run[i], l_run[i]);
    }
    __syncthreads();                                                 // the next tile's copies go where this one's were read
  }
}

namespace {

template <bool FP8>
cudaError_t launch_prefix(const PrefixParams& p, dim3 grid, cudaStream_t s) {
  static PerDevice<bool> configured;
  const cudaError_t e = allow_smem(configured, decode_prefix_kernel<FP8>, PreSmem<FP8>::kTotal);
  if (e != cudaSuccess) return e;
  launch_dependent(decode_prefix_kernel<FP8>, grid, kPreWarps * 32, PreSmem<FP8>::kTotal, s, p);
  return cudaGetLastError();
}

}  // namespace
}  // namespace nrl

using namespace nrl;

extern "C" int nrl_decode_prefix_parts(int n_groups, int max_group, int Hq, int Hkv, int max_blocks, int num_sms) {
  const long blocks = static_cast<long>(n_groups) * Hkv * ((static_cast<long>(max_group) * (Hq / Hkv) + kPreRows - 1) / kPreRows);
  const long want = blocks > 0 ? (2L * num_sms + blocks - 1) / blocks : 1, steps = (max_blocks + kPreStep - 1) / kPreStep;
  return static_cast<int>(want < 1 ? 1 : want > 16 ? (steps < 16 ? steps : 16) : (want < steps ? want : steps < 1 ? 1 : steps));
}

extern "C" cudaError_t nrl_decode_prefix(const DecodeCall* c, const int* cu_groups, const int* shared, int n_groups, int max_group, int prefix_parts, float* prefix_o,
                                         float* prefix_ml, cudaStream_t s) {
  PrefixParams p;
  p.q = static_cast<const __nv_bfloat16*>(c->q);
  p.k = static_cast<const uint8_t*>(c->k_cache);
  p.v = static_cast<const uint8_t*>(c->v_cache);
  p.ks = c->k_scale; p.vs = c->v_scale;
  p.block_tables = c->block_tables; p.context_lens = c->context_lens; p.cu_groups = cu_groups; p.shared = shared;
  p.part_o = prefix_o; p.part_ml = prefix_ml;
  p.q_stride_s = c->q_stride_s;
  p.S = c->S; p.max_blocks = c->max_blocks; p.Hkv = c->Hkv; p.G = c->Hq / c->Hkv;
  p.prefix_parts = prefix_parts;
  p.tiles = (max_group * p.G + kPreRows - 1) / kPreRows;
  p.scale_log2 = c->scale * 1.4426950408889634f;
  const dim3 grid(n_groups, c->Hkv, prefix_parts * p.tiles);
  return c->k_scale != nullptr ? launch_prefix<true>(p, grid, s) : launch_prefix<false>(p, grid, s);
}
