// Decode attention over the pages of rows whose contexts differ: behind a shared prefix (decode_prefix.cuh) and with scores.
//
//   out = sum_parts 2^(m_p - M) O_p / sum_parts 2^(m_p - M) l_p,  a part being the (maximum, sum, unnormalised result) of some of the row's keys
//   scores[s, h, t] = decay * scores[s, h, t] + sum over the G heads of kv head h of 2^(x - M) / L     (the newest token: the sum alone)
//
// The pages of all rows and kv heads, one behind the other, are dealt to the warps of the chip in equal runs: no block is longer than another, none starts
// again for every row, and few long contexts are cut as finely as many short ones.
//   decode_plan   (one block) adds up the rows' pages and finds where every warp's run begins; few rows without prefixes' runs do without it: every block of
//                 decode_flat makes the plan (4 rows of 330 tokens 10.1 -> 7.4 us)
//   decode_flat   the first blocks walk the prefixes (decode_prefix.cuh), then all of them the rows: a warp walks a run through its own ring of pages (cp.async);
//                 of every row that it meets it leaves a part.  Run w and row-head r meet in part w + r: along the runs one of the two grows by one at a time
//   decode_join   a warp a row and head joins the parts, the prefix's too, in their order; with scores, further blocks form the weights from the scores that the
//                 walk left in scratch memory (4 G bytes a token beside the 512 or 264 of its keys and values; what fits L2 is not read from memory again)
// The arithmetic is that of attention_decode.cu and attention_decode_fp8.cu, but for the factor of fp8 weights (fp8_fragments.cuh).  Bound by memory.
#include "common.cuh"
#include "decode_prefix.cuh"
#include "decode_runs.cuh"
#include "fp8_fragments.cuh"
#include "group_kernels.h"
#include "launch.h"
#include "per_device.h"

#include <type_traits>

namespace nrl {

constexpr int kFlatWarps = 4;
constexpr int kFlatD = 128;
constexpr int kPlanThreads = 1024;
constexpr int kNearRows = kFlatWarps * 32;
constexpr int kPrefixLeast = 2;                   // steps of the prefixes a run

template <bool FP8>
struct FlatSizes {
  static constexpr int kHalf = FP8 ? 2048 : 4096;                    // K or V of a page
  static constexpr int kStage = 2 * kHalf + (FP8 ? 128 : 0);         // K, V, k_scale[16], v_scale[16]
  static constexpr int kStages = FP8 ? 4 : 3;
  static constexpr int kBlocks = FP8 ? 3 : 2;                        // an SM
  static constexpr int kTotal = kFlatWarps * kStages * kStage;
  static_assert(kTotal >= PreSmem<FP8>::kTotal && kFlatWarps == kPreWarps);
};

// the last group that begins at or in front of a row; it has the row if it does not end there
NRL_DEVICE int group_search(const int* cu, int n, int row) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= row) lo = mid; else hi = mid;
  }
  return lo;
}

// the sum of `n` over the threads in front, and over all (a whole block)
NRL_DEVICE int plan_scan(int n, int* warp_sums, int& all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int upto = n;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += v;
  }
  if (lane == 31) warp_sums[warp] = upto;
  __syncthreads();
  const int mine = warp_sums[lane];
  int sums = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, sums, d);
    if (lane >= d) sums += v;
  }
  const int in_front = __shfl_sync(0xffffffffu, sums - mine, warp);
  all = __shfl_sync(0xffffffffu, sums, 31);
  __syncthreads();
  return in_front + upto - n;
}
// Where runs begin: in which owner's stretch, and there, as quotient and remainder by its divisor.  `from`: the first position of every owner (by index), `total` behind the last.
template <class From, class Divisor>
NRL_DEVICE void plan_starts(int4* starts, int owners, int total, int run, From from, Divisor divisor) {
  for (int w = threadIdx.x; w * run < total; w += kPlanThreads) {
    int lo = 0, hi = owners;                                         // the last owner that begins at or in front: one that has something
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (from(mid) <= w * run) lo = mid; else hi = mid;
    }
    const int at = w * run - from(lo), d = divisor(lo), q = at / d;
    starts[w] = make_int4(lo, q, at - q * d, 0);
  }
}

// Pages that a row walks itself.  A row that ends inside the shared tokens has none of its own: its table may say anything of the page where it ends.
NRL_DEVICE int flat_pages(const FlatParams& p, int ctx, int first) {
  return (ctx > first ? (ctx + 15) / 16 - first / 16 : 0) + (p.prefix_runs == 0 ? (first + 15) / 16 : 0);
}
// The plan of few rows and no prefixes' runs, by every block for itself, a thread a row: no kernel in front.
NRL_DEVICE const int4* plan_near(const FlatParams& p) {
  __shared__ struct { int4 rows[kNearRows + 1]; int group[kNearRows], sums[kNearRows / 32]; } near;
  const int s = threadIdx.x, warp = s >> 5, lane = s & 31, ctx = s < p.S ? flat_context(p, s) : 0;
  near.group[s] = 0;
  if (p.n_groups > 0) {
    __syncthreads();
    for (int g = s; g < p.n_groups; g += kNearRows) {
      const int a = p.cu_groups[g], b = p.cu_groups[g + 1];
      if (a >= 0 && b <= p.S && p.shared[g] > 0)
        for (int r = a; r < b; ++r) near.group[r] = g + 1;
    }
    __syncthreads();
  }
  const int prefix = near.group[s], first = prefix > 0 ? min(p.shared[prefix - 1], ctx) : 0, n = flat_pages(p, ctx, first);
  int upto = n;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += v;
  }
  if (lane == 31) near.sums[warp] = upto;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kNearRows / 32; ++w) {
    before += w < warp ? near.sums[w] : 0;
    all += near.sums[w];
  }
  const int4 row = make_int4(first, before + upto - n, n, prefix), total = make_int4(0, all, max(p.least, (all * p.Hkv + p.runs - 1) / p.runs), 0);
  near.rows[s] = row;
  if (s == 0) near.rows[kNearRows] = total;
  if (blockIdx.x == 0) {                                              // for decode_join
    if (s < p.S) p.rows[s] = row;
    if (s == 0) p.rows[p.S] = total;
  }
  __syncthreads();
  return near.rows;
}

// (all positions are below 2^27: checked on the host)
__global__ void __launch_bounds__(kPlanThreads) decode_plan_kernel(const FlatParams p) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ int warp_sums[32];
  __shared__ int cu_near[kPlanThreads + 1], from_near[kPlanThreads], longest_near[kPlanThreads];
  const int tid = threadIdx.x;
  const int* cu = p.cu_groups;
  // of every group the longest context: no page of the prefix behind it is anybody's, whatever the table says of it
  const bool prefixes = p.prefix_runs > 0, near = p.n_groups <= kPlanThreads;
  if (prefixes) {
    for (int g = tid; g < p.n_groups; g += kPlanThreads) (near ? longest_near[g] : p.groups[g].z) = 0;
    __syncthreads();
  }
  if (p.n_groups > 0 && p.n_groups <= kPlanThreads) {
    for (int i = tid; i <= p.n_groups; i += kPlanThreads) cu_near[i] = p.cu_groups[i];
    cu = cu_near;
    __syncthreads();
  }
  auto group_ok = [&](int g) { return cu[g] >= 0 && cu[g] < cu[g + 1] && cu[g + 1] <= p.S; };
  // ---- rows ----
  int before = 0, off, all;                                          // pages of the rows in front of this pass
  for (int s0 = 0; s0 < p.S; s0 += kPlanThreads) {
    const int s = s0 + tid;
    int first = 0, prefix = 0, n = 0;
    if (s < p.S) {
      const int ctx = flat_context(p, s);
      if (p.n_groups > 0) {
        const int g = group_search(cu, p.n_groups, s);
        if (cu[g] <= s && s < cu[g + 1] && group_ok(g)) {
          const int shared = p.shared[g];
          prefix = shared > 0 ? g + 1 : 0;
          first = max(0, min(shared, ctx));
          if (prefixes) atomicMax(near ? &longest_near[g] : &p.groups[g].z, ctx);
        }
      }
      n = flat_pages(p, ctx, first);
    }
    off = before + plan_scan(n, warp_sums, all);
    if (s < p.S) p.rows[s] = make_int4(first, off, n, prefix);
    from_near[tid] = off;
    before += all;
  }
  const int run = max(p.least, (before * p.Hkv + p.runs - 1) / p.runs);
  if (tid == 0) p.rows[p.S] = make_int4(0, before, run, 0);
  __syncthreads();                                                   // (a block sees its own writes)
  plan_starts(p.starts, p.S, before * p.Hkv, run, [&](int s) { return (p.S <= kPlanThreads ? from_near[s] : p.rows[s].y) * p.Hkv; }, [&](int s) { return p.rows[s].z; });
  if (p.prefix_runs == 0) return;
  // ---- prefixes ----
  const long own_work = static_cast<long>(before) * p.Hkv;
  before = 0;
  __syncthreads();
  for (int g0 = 0; g0 < p.n_groups; g0 += kPlanThreads) {
    const int g = g0 + tid;
    int rows = 0, steps = 0, tokens = 0;
    if (g < p.n_groups && group_ok(g)) {
      rows = (cu[g + 1] - cu[g]) * p.G;
      tokens = max(0, min(p.shared[g], near ? longest_near[g] : __ldcg(&p.groups[g].z)));
      steps = (tokens + kPrefixKeys - 1) / kPrefixKeys;
    }
    off = before + plan_scan(steps * prefix_tiles(rows) * p.Hkv, warp_sums, all);
    if (g < p.n_groups) p.groups[g] = make_int4(off, steps, tokens, rows);
    from_near[tid] = off;
    before += all;
  }
  // as many blocks as the prefixes' share of the work, one an SM at the least; they take rows' pages afterwards
  const long work = static_cast<long>(before) * p.step_cost;
  const long share = (p.blocks * work + own_work + work - 1) / max(1L, own_work + work), sms = p.num_sms;
  const long many = min(max(1L, (share + sms - 1) / sms) * sms, static_cast<long>(p.prefix_runs));
  const int prefix_run = max(kPrefixLeast, static_cast<int>((before + many - 1) / many));
  if (tid == 0) p.groups[p.n_groups] = make_int4(before, prefix_run, 0, 0);
  __syncthreads();
  plan_starts(p.prefix_starts, p.n_groups, before, prefix_run, [&](int g) { return p.n_groups <= kPlanThreads ? from_near[g] : p.groups[g].x; },
              [&](int g) { return p.groups[g].y; });
}

NRL_DEVICE void flat_ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
NRL_DEVICE void flat_ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
// rows 8..15 of the A tile are padding (G <= 8 query heads)
NRL_DEVICE void flat_mma_bf16(float (&d)[4], uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(0u), "r"(a2), "r"(0u), "r"(b0), "r"(b1));
}

// A place in the run: a row-head and a page of its own.
struct FlatAt {
  int s, h, page, pages;        // pages: that the row walks; page < pages
  int first, ctx;               // the row's first token of its own, its context
  int lead, lead_row;           // pages of a prefix that the row walks itself, in front, and the row whose they are
};
template <bool LEAD>
NRL_DEVICE void flat_row(const FlatParams& p, const int4* rows, FlatAt& a, int s) {
  const int4 row = rows[s];
  a.s = s;
  a.first = row.x;
  a.pages = row.z;
  a.ctx = flat_context(p, s);
  a.lead = LEAD && p.prefix_runs == 0 ? (a.first + 15) / 16 : 0;
  a.lead_row = a.lead > 0 ? p.cu_groups[row.w - 1] : 0;
}
template <bool LEAD>
NRL_DEVICE bool flat_next(const FlatParams& p, const int4* rows, FlatAt& a) {          // true: another row-head begins
  if (++a.page < a.pages) return false;
  a.page = 0;
  if (++a.h == p.Hkv) {
    a.h = 0;
    do flat_row<LEAD>(p, rows, a, a.s + 1); while (a.pages == 0 && a.s + 1 < p.S);
  }
  return true;
}
// the page table's entry of page i that the row walks
NRL_DEVICE long flat_entry(const FlatParams& p, const FlatAt& a, int i) {
  return i < a.lead ? static_cast<long>(a.lead_row) * p.max_blocks + i : static_cast<long>(a.s) * p.max_blocks + a.first / 16 + i - a.lead;
}

// NEAR: few rows, whose plan every block makes for itself; no prefixes' runs
template <bool FP8, bool SCORES, bool NEAR>
__global__ void __launch_bounds__(kFlatWarps * 32, FlatSizes<FP8>::kBlocks) decode_flat_kernel(const FlatParams p) {
  pdl_wait();
  pdl_launch_dependents();
  using Z = FlatSizes<FP8>;
  extern __shared__ __align__(128) uint8_t smem[];
  if constexpr (!SCORES && !NEAR) {
    if (static_cast<int>(blockIdx.x) < p.prefix_runs) {
      decode_prefix_run<FP8>(p, smem, blockIdx.x);
      __syncthreads();
    }
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int4* rows = p.rows;
  if constexpr (NEAR) rows = plan_near(p);
  const int4 total = rows[NEAR ? kNearRows : p.S];
  const int run = total.z, all = total.y * p.Hkv;
  // The next run that nobody has: blocks that have walked a prefix come late.  Of few rows, one a warp.
  for (bool more = true; more;) {
    int w = 0;
    if (NEAR) {
      w = blockIdx.x * kFlatWarps + warp;
      more = false;
    } else {
      if (lane == 0) w = atomicAdd(&p.rows[p.S].w, 1);
      w = __shfl_sync(0xffffffffu, w, 0);
    }
    const int count = w < p.runs ? min(run, all - w * run) : 0;
    if (count <= 0) break;
    FlatAt here, ahead;
    {
      int4 start;
      if (NEAR) {
        int lo = 0, hi = p.S;                                          // the last row that begins at or in front
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (rows[mid].y * p.Hkv <= w * run) lo = mid; else hi = mid;
        }
        const int at = w * run - rows[lo].y * p.Hkv, d = rows[lo].z;
        start = make_int4(lo, at / d, at % d, 0);
      } else {
        start = p.starts[w];
      }
      flat_row<!SCORES>(p, rows, here, start.x);
      here.h = start.y;
      here.page = start.z;
      ahead = here;
    }
    uint8_t* ring = smem + warp * Z::kStages * Z::kStage;

    // page numbers wait in the lanes, 32 of a row-head at a time
    int ids = 0, ids_from = -1, issued = 0;
    auto issue = [&]() {
      if (issued < count) {
        if (ids_from < 0 || ahead.page - ids_from >= 32) {
          ids_from = ahead.page;
          ids = ids_from + lane < ahead.pages ? p.block_tables[flat_entry(p, ahead, ids_from + lane)] : 0;
        }
        const long pg = static_cast<long>(__shfl_sync(0xffffffffu, ids, ahead.page - ids_from)) * p.Hkv + ahead.h;
        uint8_t *kd = ring + (issued % Z::kStages) * Z::kStage, *vd = kd + Z::kHalf;
        const uint8_t *ksrc = p.k + pg * Z::kHalf, *vsrc = p.v + pg * Z::kHalf;
        if (FP8) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int chunk = lane + j * 32, r = chunk >> 3, c = chunk & 7;
            cp_async_16(kd + r * 128 + ((c ^ k_sigma(r)) << 4), ksrc + chunk * 16);
            cp_async_16(vd + chunk * 16, vsrc + chunk * 16);
          }
          if (lane < 8) cp_async_16(vd + Z::kHalf + lane * 16, (lane < 4 ? p.ks : p.vs) + pg * 16 + (lane & 3) * 4);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int chunk = lane + j * 32, at = (chunk >> 4) * 256 + (((chunk & 15) ^ ((chunk >> 4) & 7)) << 4);
            cp_async_16(kd + at, ksrc + chunk * 16);
            cp_async_16(vd + at, vsrc + chunk * 16);
          }
        }
        if (++issued < count && flat_next<!SCORES>(p, rows, ahead)) ids_from = -1;
      }
      cp_async_commit();
    };
#pragma unroll 1
    for (int i = 0; i < (FP8 ? Z::kStages : Z::kStages - 1); ++i) issue();

    uint32_t qa0[8], qa2[8];                                           // row g: query head g of the kv head
    float o[16][4];
    float m_run = 0.f, l_run = 0.f, factor = 1.f;                    // of weights, and of what they have summed
    auto enter = [&]() {                                               // a row-head's queries, nothing seen
      const bool real = g < p.G;
      const __nv_bfloat16* qrow = p.q + here.s * p.q_stride_s + (here.h * p.G + (real ? g : 0)) * kFlatD;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        if (FP8) {
          const uint2 x = *reinterpret_cast<const uint2*>(qrow + (ks >> 2) * 64 + t4 * 16 + (ks & 3) * 4);
          const float2 a = unpack_bf16x2(x.x), b = unpack_bf16x2(x.y);
          qa0[ks] = real ? pack_f16x2(a.x, a.y) : 0u;
          qa2[ks] = real ? pack_f16x2(b.x, b.y) : 0u;
        } else {
          qa0[ks] = real ? *reinterpret_cast<const uint32_t*>(qrow + ks * 16 + t4 * 2) : 0u;
          qa2[ks] = real ? *reinterpret_cast<const uint32_t*>(qrow + ks * 16 + 8 + t4 * 2) : 0u;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      m_run = -INFINITY;
      l_run = 0.f;
      factor = FP8 ? __uint_as_float(kMostFactor) : 1.f;
    };
    auto leave = [&]() {                                               // its part
      const float f = FP8 ? inverse_factor(factor) : 1.f;
      float l = l_run;
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (g < p.G) {
        const long part = (static_cast<long>(w) + static_cast<long>(here.s) * p.Hkv + here.h) * 8 + g;
        float* dst = p.part_o + part * kFlatD + t4 * 2;
#pragma unroll
        for (int nd = 0; nd < 16; ++nd)
          *reinterpret_cast<float2*>(dst + nd * 8) = make_float2(o[nd][0] * f, o[nd][1] * f);
        if (t4 == 0) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(m_run, l);
      }
    };

    auto step = [&](auto number, int it) {                             // pages it and, of two, it + 1 of the run, both of this row-head: one rescaling of O
      constexpr int U = decltype(number)::value;
      cp_async_wait<FP8 ? Z::kStages - U : Z::kStages - 1>();
      __syncwarp();
      float s[U][2][4], vscale[U][4];
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint8_t* st = ring + ((it + u) % Z::kStages) * Z::kStage;
        const uint32_t kb = smem_u32(st);
        const int page = here.page + u;
        const bool lead = !SCORES && page < here.lead;
        const int tok0 = lead ? page * 16 : (here.first / 16 + page - here.lead) * 16;
#pragma unroll
        for (int j = 0; j < 2; ++j) s[u][j][0] = s[u][j][1] = s[u][j][2] = s[u][j][3] = 0.f;
        // ---- S = Q K^T.  Key of column (j, e): bf16 8 j + 2 t + e, fp8 4 t + 2 j + e ----
        if constexpr (FP8) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int krow = ((g >> 1) << 2) + 2 * j + (g & 1);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint4 w4 = lds128(kb + krow * 128 + (((4 * h + t4) ^ k_sigma(g)) << 4));
              const uint32_t x[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
              for (int i = 0; i < 4; ++i)
                mma_f16_16816(s[u][j], qa0[4 * h + i], qa2[4 * h + i], e4m3x2_to_f16x2(x[i] & 0xFFFFu), e4m3x2_to_f16x2(x[i] >> 16));
            }
          }
          const uint4 kr = lds128(kb + 2 * Z::kHalf + t4 * 16), vr = lds128(kb + 2 * Z::kHalf + 64 + t4 * 16);
          const float kscale[4] = {__uint_as_float(kr.x), __uint_as_float(kr.y), __uint_as_float(kr.z), __uint_as_float(kr.w)};
          vscale[u][0] = __uint_as_float(vr.x); vscale[u][1] = __uint_as_float(vr.y); vscale[u][2] = __uint_as_float(vr.z); vscale[u][3] = __uint_as_float(vr.w);
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) s[u][j][e] *= kscale[2 * j + e] * p.scale_log2;
        } else {
          const int mrow = (lane & 7) + (lane >> 4) * 8, mcol = (lane >> 3) & 1;
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            uint32_t kf[4];
            flat_ldmatrix_x4(kf, kb + mrow * 256 + (((ks * 2 + mcol) ^ (mrow & 7)) << 4));
            flat_mma_bf16(s[u][0], qa0[ks], qa2[ks], kf[0], kf[1]);
            flat_mma_bf16(s[u][1], qa0[ks], qa2[ks], kf[2], kf[3]);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) s[u][j][e] *= p.scale_log2;
        }
        // ---- mask; values and scales outside the row's own tokens, whatever they are, meet weights of 0 as zeros ----
        const int lo = lead ? 0 : here.first - tok0, hi = (lead ? here.first : here.ctx) - tok0;
        if (lo > 0 || hi < 16) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int t = FP8 ? t4 * 4 + 2 * j + e : j * 8 + t4 * 2 + e;
              if (t < lo || t >= hi) s[u][j][e] = -INFINITY;
              if (FP8 && (t < lo || t >= hi)) vscale[u][2 * j + e] = 0.f;
            }
          if (FP8) {
            fp8_clear_values(st + Z::kHalf, lo, hi, lane);
          } else {
            for (int i = lane; i < 256; i += 32)
              if ((i >> 4) < lo || (i >> 4) >= hi) *reinterpret_cast<uint4*>(st + Z::kHalf + i * 16) = make_uint4(0, 0, 0, 0);
            __syncwarp();
          }
        }
        if (SCORES && g < p.G) {
          float* raw = p.raw + ((static_cast<long>(here.s) * p.Hkv + here.h) * p.G + g) * (16L * p.max_blocks) + tok0;
          if (FP8) {
            *reinterpret_cast<float4*>(raw + t4 * 4) = make_float4(s[u][0][0], s[u][0][1], s[u][1][0], s[u][1][1]);
          } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) *reinterpret_cast<float2*>(raw + j * 8 + t4 * 2) = make_float2(s[u][j][0], s[u][j][1]);
          }
        }
        top = fmaxf(top, fmaxf(fmaxf(s[u][0][0], s[u][0][1]), fmaxf(s[u][1][0], s[u][1][1])));
      }
      // ---- online softmax on row g ----
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float m_new = fmaxf(m_run, top), m_sub = m_new == -INFINITY ? 0.f : m_new;
      const float corr = exp2f(m_run - m_sub);                         // 0 while nothing has been seen
      uint32_t pa[U][2];
      float sum = 0.f, corr_o = corr;
      if constexpr (FP8) {
        float most = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) most = fmaxf(most, fmaxf(fmaxf(vscale[u][0], vscale[u][1]), fmaxf(vscale[u][2], vscale[u][3])));
        const float before = inverse_factor(factor);
        factor = shrink_factor(factor, most);
        corr_o = corr * (factor * before);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float p0 = exp2f(s[u][j][0] - m_sub), p1 = exp2f(s[u][j][1] - m_sub);
          sum += p0 + p1;
          pa[u][j] = FP8 ? pack_f16x2(p0 * (vscale[u][2 * j] * factor), p1 * (vscale[u][2 * j + 1] * factor)) : pack_bf16x2(p0, p1);
        }
      l_run = l_run * corr + sum;
      m_run = m_new;
#pragma unroll
      for (int i = 0; i < 16; ++i) { o[i][0] *= corr_o; o[i][1] *= corr_o; }
      // ---- O += P V ----
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t vb = smem_u32(ring + ((it + u) % Z::kStages) * Z::kStage) + Z::kHalf;
        if constexpr (FP8) {
#pragma unroll
          for (int nd = 0; nd < 16; ++nd) {
            const uint32_t x = lds32(vb + (nd * 8 + g) * 16 + t4 * 4);
            mma_f16_16816(o[nd], pa[u][0], pa[u][1], e4m3x2_to_f16x2(x & 0xFFFFu), e4m3x2_to_f16x2(x >> 16));
          }
        } else {
          const int mrow = (lane & 7) + ((lane >> 3) & 1) * 8, mcol = lane >> 4;
#pragma unroll
          for (int nd = 0; nd < 8; ++nd) {
            uint32_t vf[4];
            flat_ldmatrix_x4_trans(vf, vb + mrow * 256 + (((nd * 2 + mcol) ^ (mrow & 7)) << 4));
            flat_mma_bf16(o[nd * 2], pa[u][0], pa[u][1], vf[0], vf[1]);
            flat_mma_bf16(o[nd * 2 + 1], pa[u][0], pa[u][1], vf[2], vf[3]);
          }
        }
      }
      __syncwarp();
    };

    enter();
    for (int it = 0; it < count;) {
      const bool two = FP8 && it + 1 < count && here.page + 1 < here.pages;
      if constexpr (FP8) {
        if (two) step(std::integral_constant<int, 2>{}, it);
        else step(std::integral_constant<int, 1>{}, it);
#pragma unroll 1
        for (int u = 0; u < (two ? 2 : 1); ++u) issue();
      } else {
        issue();
        step(std::integral_constant<int, 1>{}, it);
      }
      it += two ? 2 : 1;
      if (two) ++here.page;
      if (it == count) break;
      const FlatAt last = here;
      if (flat_next<!SCORES>(p, rows, here)) {
        const FlatAt now = here;
        here = last;
        leave();
        here = now;
        enter();
      }
    }
    leave();
    cp_async_wait<0>();
  }
}

// ---- parts to results, scores to weights ---------------------------------------------------------------------------------------------

constexpr int kJoinU = 4;                // parts in flight
constexpr int kJoinWarps = 8;

struct FlatParts {
  const float2* ml;                      // of the first part of a row
  const float4* o;
  int n;
};
// head r's parts of a row's own tokens
NRL_DEVICE FlatParts flat_parts(const FlatParams& p, int4 row, int s, int h, int r) {
  const int run = p.rows[p.S].z, a = row.y * p.Hkv + h * row.z, w0 = a / run;
  const long at = (static_cast<long>(w0) + static_cast<long>(s) * p.Hkv + h) * 8 + r;
  return {reinterpret_cast<const float2*>(p.part_ml) + at, reinterpret_cast<const float4*>(p.part_o) + at * 32, row.z > 0 ? (a + row.z - 1) / run - w0 + 1 : 0};
}
// and of the prefix's, one a run
NRL_DEVICE FlatParts prefix_parts(const FlatParams& p, int g, int s, int h, int r) {
  const int4 group = p.groups[g];
  const int first = p.cu_groups[g], row = (s - first) * p.G + r, run = p.groups[p.n_groups].y, a = group.x + (h * prefix_tiles(group.w) + row / kPrefixRows) * group.y, c0 = a / run;
  const long at = prefix_part_row(p, first, h, group.w, row) + static_cast<long>(kPrefixRows) * c0;
  return {reinterpret_cast<const float2*>(p.prefix_ml) + at, reinterpret_cast<const float4*>(p.prefix_o) + at * 32, group.y > 0 ? (a + group.y - 1) / run - c0 + 1 : 0};
}
// A part that has seen nothing has maximum -inf and sum 0; one that has seen nothing but NaN has sum NaN, as the maximum passes them over
NRL_DEVICE bool nothing_seen(float2 e) { return e.x == -INFINITY && e.y == 0.f; }
NRL_DEVICE void join_part(float2 e, float4 o, float& M, float& L, float4& acc) {
  if (nothing_seen(e)) return;
  const float top = fmaxf(M, e.x), a = exp2f(M - top), b = exp2f(e.x - top);          // 2^-inf = 0
  L = L * a + e.y * b;
  acc.x = acc.x * a + o.x * b; acc.y = acc.y * a + o.y * b; acc.z = acc.z * a + o.z * b; acc.w = acc.w * a + o.w * b;
  M = top;
}
// Parts `from`, `from` + STEP, ...; a lane has four elements; a row's parts lie 8 rows apart, a prefix's 64
template <bool PREFIX, int STEP>
NRL_DEVICE void join_parts(const FlatParts& x, int from, int lane, float& M, float& L, float4& acc) {
  for (int i0 = from; i0 < x.n; i0 += kJoinU * STEP) {
    float2 e[kJoinU];
    float4 o[kJoinU];
#pragma unroll
    for (int u = 0; u < kJoinU; ++u) {
      const bool ok = i0 + u * STEP < x.n;
      const long at = (i0 + u * STEP) * (PREFIX ? static_cast<long>(kPrefixRows) : 8L);
      e[u] = ok ? x.ml[at] : make_float2(-INFINITY, 0.f);
      o[u] = ok ? x.o[at * 32 + lane] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < kJoinU; ++u) join_part(e[u], o[u], M, L, acc);
  }
}
NRL_DEVICE void join_store(const FlatParams& p, int s, int head, int lane, float L, float4 acc) {
  const float f = L == 0.f ? 0.f : 1.f / L;
  uint2 v;
  v.x = pack_bf16x2(acc.x * f, acc.y * f);
  v.y = pack_bf16x2(acc.z * f, acc.w * f);
  *reinterpret_cast<uint2*>(p.out + (static_cast<long>(s) * p.Hq + head) * kFlatD + lane * 4) = v;
}

// Many rows: grid rows x (kv heads x, with scores, chunks of tokens), a warp a query head for the results, which the first chunk's blocks form.
// NEAR, few rows of many parts: rows x (query heads, whose parts are dealt to eight warps; then the chunks).  8 rows of 30 k tokens with scores 53 -> 47 us, 32 rows of
// 556 fp8 tokens 12.7 -> 10.8.
template <bool SCORES, bool NEAR>
__global__ void __launch_bounds__(kJoinWarps * 32) decode_join_kernel(const FlatParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int s = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (NEAR && static_cast<int>(blockIdx.y) < p.Hq) {
    __shared__ float2 part_ml[kJoinWarps];
    __shared__ float4 part_o[kJoinWarps][32];
    const int head = blockIdx.y;
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    join_parts<false, kJoinWarps>(flat_parts(p, p.rows[s], s, head / p.G, head % p.G), warp, lane, M, L, acc);
    if (lane == 0) part_ml[warp] = make_float2(M, L);
    part_o[warp][lane] = acc;
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int w = 1; w < kJoinWarps; ++w) join_part(part_ml[w], part_o[w][lane], M, L, acc);
    join_store(p, s, head, lane, L, acc);
    return;
  }
  const int y = blockIdx.y - (NEAR ? p.Hq : 0), h = y % p.Hkv, chunk = y / p.Hkv;
  const int ctx = flat_context(p, s), t0 = chunk * p.chunk, n = SCORES ? min(min(ctx, p.max_tokens), t0 + p.chunk) : 0;
  if ((NEAR || chunk > 0) && t0 >= n) return;
  const int4 row = p.rows[s];
  __shared__ float top[8], inv[8];
  if (warp < p.G) {
    const FlatParts own = flat_parts(p, row, s, h, warp);
    float M = -INFINITY, L = 0.f;
    if (!NEAR && chunk == 0) {
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      if (!SCORES && row.w > 0 && p.prefix_runs > 0) join_parts<true, 1>(prefix_parts(p, row.w - 1, s, h, warp), 0, lane, M, L, acc);
      join_parts<false, 1>(own, 0, lane, M, L, acc);
      join_store(p, s, h * p.G + warp, lane, L, acc);
    } else {
#pragma unroll 8
      for (int i = lane; i < own.n; i += 32) {
        const float2 e = own.ml[i * 8];
        if (nothing_seen(e)) continue;
        const float m = fmaxf(M, e.x);
        L = L * exp2f(M - m) + e.y * exp2f(e.x - m);
        M = m;
      }
      const float all = warp_max(M);
      L = warp_sum(L == 0.f ? 0.f : L * exp2f(M - all));
      M = all;
    }
    if (SCORES && lane == 0) {
      top[warp] = M == -INFINITY ? 0.f : M;
      inv[warp] = L == 0.f ? 0.f : 1.f / L;
    }
  }
  if (!SCORES) return;
  __syncthreads();
  const long len = 16L * p.max_blocks;
  const float* raw = p.raw + (static_cast<long>(s) * p.Hkv + h) * p.G * len;
  const float* in = p.scores_in + s * p.in_row + h * p.in_head;
  float* out = p.scores_out + s * p.out_row + h * p.out_head;
  // four tokens a thread (scratch rows are multiples of 16 long)
  for (int t = t0 + threadIdx.x * 4; t < n; t += blockDim.x * 4) {
    float4 x[8];
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < p.G) x[r] = *reinterpret_cast<const float4*>(raw + r * len + t);
    float w[4] = {0.f, 0.f, 0.f, 0.f}, old[4];
    const bool whole = t + 4 < ctx;       // none of them is the newest, all are there
    if (whole && p.wide && t + 4 <= n) {
      const float4 v = *reinterpret_cast<const float4*>(in + t);
      old[0] = v.x; old[1] = v.y; old[2] = v.z; old[3] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) old[i] = t + i < n && t + i < ctx - 1 ? in[t + i] : 0.f;
    }
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < p.G) {
        const float m = top[r], f = inv[r];
        w[0] += exp2f(x[r].x - m) * f; w[1] += exp2f(x[r].y - m) * f; w[2] += exp2f(x[r].z - m) * f; w[3] += exp2f(x[r].w - m) * f;
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = whole || t + i < ctx - 1 ? fmaf(p.decay, old[i], w[i]) : w[i];
    if (p.wide && t + 4 <= n) {
      *reinterpret_cast<float4*>(out + t) = make_float4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t + i < n) out[t + i] = w[i];
    }
  }
}

namespace {

cudaError_t launch_plan(const FlatParams& p, cudaStream_t s) {
  if (p.near) return cudaSuccess;
  launch_dependent(decode_plan_kernel, 1, kPlanThreads, 0, s, p);
  return cudaGetLastError();
}
template <bool FP8, bool SCORES, bool NEAR>
cudaError_t launch_walk(const FlatParams& p, cudaStream_t s) {
  static PerDevice<bool> configured;
  const cudaError_t e = allow_smem(configured, decode_flat_kernel<FP8, SCORES, NEAR>, FlatSizes<FP8>::kTotal);
  if (e != cudaSuccess) return e;
  launch_dependent(decode_flat_kernel<FP8, SCORES, NEAR>, p.blocks, kFlatWarps * 32, FlatSizes<FP8>::kTotal, s, p);
  return cudaGetLastError();
}

template <bool FP8, bool SCORES>
cudaError_t launch_flat(const FlatParams& p, cudaStream_t s) {
  return p.near ? launch_walk<FP8, SCORES, true>(p, s) : launch_walk<FP8, SCORES, false>(p, s);
}

template <bool SCORES>
cudaError_t launch_join(const FlatParams& p, int chunks, int threads, cudaStream_t s) {
  if (p.near) launch_dependent(decode_join_kernel<SCORES, true>, dim3(p.S, p.Hq + (SCORES ? p.Hkv * chunks : 0)), kJoinWarps * 32, 0, s, p);
  else launch_dependent(decode_join_kernel<SCORES, false>, dim3(p.S, p.Hkv * chunks), threads, 0, s, p);
  return cudaGetLastError();
}

// pieces of scratch, one behind the other, on 64 bytes
struct Pieces {
  uint8_t* at;
  size_t used = 0;
  template <class T>
  T* take(size_t n) {
    T* r = reinterpret_cast<T*>(at + used);
    used += (n * sizeof(T) + 63) / 64 * 64;
    return r;
  }
};

// Runs: as many as warps (prefixes: blocks) fit the chip, or as the longest contexts that the tables allow could fill.
// Where those contexts are few bytes, rows walk their prefixes themselves: with prefixes' runs, of whatever size, a call takes 17 us, in which others read 100 MB
// (16 groups of 8 rows, 100 + 100 bf16 tokens, 17 us with, 14 without; 16 of 4 rows, 1000 + 100, 20 and 17).
constexpr long kPrefixBytes = 100L << 20;
// A prefix's step of 64 tokens takes a block as long as this many pages of rows: blocks that begin with prefixes are as many SMs' worth as their share of the work.
// Rows of 12 heads, 2 kv heads, all on one block an SM, two, three: bf16 64 x 8 of 512 + 256 tokens 48, 51, 58 us, 32 x 16 of 2000 + 128 77, 61, 75;
// fp8 42, 42, 43 and 90, 67, 57; 13 x 16 of 28 heads, 4100 + 560 tokens 116, 86, 89.
constexpr int kStepCost = 5, kStepCostFp8 = 8;
struct FlatPlan { int runs, least, n_groups, prefix_runs, blocks; };
FlatPlan flat_plan(const DecodeCall* c, int n_groups, int max_group, int num_sms) {
  const long most = static_cast<long>(c->S) * c->Hkv * c->max_blocks;
  const int fit = num_sms * kFlatWarps * (c->k_scale != nullptr ? FlatSizes<true>::kBlocks : FlatSizes<false>::kBlocks), least = 2;
  const long runs = (most + least - 1) / least;
  FlatPlan plan = {static_cast<int>(runs < fit ? runs : fit), least, n_groups, 0, 0};
  if (n_groups > 0 && most * (c->k_scale != nullptr ? FlatSizes<true>::kStage : FlatSizes<false>::kStage) > kPrefixBytes) {
    const long tiles = (static_cast<long>(max_group) * (c->Hq / c->Hkv) + kPrefixRows - 1) / kPrefixRows;
    const long most_runs = (n_groups * tiles * c->Hkv * ((c->max_blocks * 16L + kPrefixKeys - 1) / kPrefixKeys) + kPrefixLeast - 1) / kPrefixLeast;
    const long prefix_fit = fit / kFlatWarps;
    plan.prefix_runs = static_cast<int>(most_runs < prefix_fit ? most_runs : prefix_fit);
  }
  plan.blocks = (plan.runs < fit ? plan.runs + kFlatWarps - 1 : fit) / kFlatWarps;
  if (plan.blocks < plan.prefix_runs) plan.blocks = plan.prefix_runs;
  return plan;
}
size_t lay_out(FlatParams& p, const DecodeCall* c, const FlatPlan& plan, void* scratch) {
  Pieces pieces = {static_cast<uint8_t*>(scratch)};
  const size_t parts = static_cast<size_t>(plan.runs) + static_cast<size_t>(c->S) * c->Hkv;
  p.rows = pieces.take<int4>(c->S + 1);
  p.starts = pieces.take<int4>(plan.runs);
  p.part_ml = pieces.take<float>(parts * 16);
  p.part_o = pieces.take<float>(parts * 8 * kFlatD);
  if (plan.prefix_runs > 0) {
    const size_t rows = static_cast<size_t>(c->S) * c->Hq + kPrefixRows * static_cast<size_t>(plan.prefix_runs);
    p.groups = pieces.take<int4>(plan.n_groups + 1);
    p.prefix_starts = pieces.take<int4>(plan.prefix_runs);
    p.prefix_ml = pieces.take<float>(rows * 2);
    p.prefix_o = pieces.take<float>(rows * kFlatD);
  }
  return pieces.used;
}
FlatParams flat_params(const DecodeCall* c, const FlatPlan& plan, void* scratch, int num_sms) {
  FlatParams p = {};
  lay_out(p, c, plan, scratch);
  p.q = static_cast<const __nv_bfloat16*>(c->q);
  p.k = static_cast<const uint8_t*>(c->k_cache);
  p.v = static_cast<const uint8_t*>(c->v_cache);
  p.ks = c->k_scale; p.vs = c->v_scale;
  p.block_tables = c->block_tables; p.context_lens = c->context_lens;
  p.out = static_cast<__nv_bfloat16*>(c->out);
  p.q_stride_s = c->q_stride_s;
  p.S = c->S; p.max_blocks = c->max_blocks; p.Hq = c->Hq; p.Hkv = c->Hkv; p.G = c->Hq / c->Hkv;
  p.runs = plan.runs; p.least = plan.least; p.n_groups = plan.n_groups; p.prefix_runs = plan.prefix_runs; p.blocks = plan.blocks; p.num_sms = num_sms;
  p.near = plan.prefix_runs == 0 && c->S <= kNearRows;
  p.step_cost = c->k_scale != nullptr ? kStepCostFp8 : kStepCost;
  p.scale_log2 = c->scale * 1.4426950408889634f;
  return p;
}

}  // namespace
}  // namespace nrl

using namespace nrl;

extern "C" size_t nrl_decode_scratch(const DecodeCall* c, int n_groups, int max_group, int num_sms) {
  FlatParams p = {};
  return lay_out(p, c, flat_plan(c, n_groups, max_group, num_sms), nullptr);
}

extern "C" cudaError_t nrl_paged_decode_shared(const DecodeCall* c, const int* cu_groups, const int* shared, int n_groups, int max_group, void* scratch, int num_sms,
                                               cudaStream_t s) {
  if (c->S == 0) return cudaSuccess;
  FlatParams p = flat_params(c, flat_plan(c, n_groups, max_group, num_sms), scratch, num_sms);
  p.cu_groups = cu_groups; p.shared = shared;
  cudaError_t e = launch_plan(p, s);
  if (e == cudaSuccess) e = c->k_scale != nullptr ? launch_flat<true, false>(p, s) : launch_flat<false, false>(p, s);
  if (e != cudaSuccess) return e;
  return launch_join<false>(p, 1, 32 * p.G, s);
}

extern "C" cudaError_t nrl_paged_decode_scored(const DecodeCall* c, const float* scores_in, long in_row, long in_head, float* scores_out, long out_row, long out_head,
                                               int max_tokens, float decay, float* raw, void* scratch, int num_sms, cudaStream_t s) {
  if (c->S == 0) return cudaSuccess;
  FlatParams p = flat_params(c, flat_plan(c, 0, 0, num_sms), scratch, num_sms);
  p.raw = raw; p.scores_in = scores_in; p.scores_out = scores_out;
  p.in_row = in_row; p.in_head = in_head; p.out_row = out_row; p.out_head = out_head;
  p.max_tokens = max_tokens < 16 * c->max_blocks ? max_tokens : 16 * c->max_blocks;
  p.decay = decay;
  cudaError_t e = launch_plan(p, s);
  if (e == cudaSuccess) e = c->k_scale != nullptr ? launch_flat<true, true>(p, s) : launch_flat<false, true>(p, s);
  if (e != cudaSuccess) return e;
  p.wide = (reinterpret_cast<uintptr_t>(scores_in) | reinterpret_cast<uintptr_t>(scores_out)) % 16 == 0 && (in_row | in_head | out_row | out_head) % 4 == 0;
  // tokens a block: rows' contexts whole where there are rows enough for the chip
  p.chunk = static_cast<long>(c->S) * c->Hkv >= 2L * num_sms ? 4096 : 1024;
  while ((p.max_tokens - 1) / p.chunk + 1 > 32768 / c->Hkv) p.chunk *= 2;                       // (a grid's second dimension ends at 65 535)
  return launch_join<true>(p, (p.max_tokens + p.chunk - 1) / p.chunk, 256, s);
}
