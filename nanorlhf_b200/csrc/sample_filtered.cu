// One token per row of logits under temperature, min-p, top-k and top-p, from a given uniform number:
//   w_i = exp((z_i - max z) / T);  keep w_i >= min_p;  of those the top_k first in (logit descending, index ascending);  of those the shortest prefix whose
//   mass is at least top_p of theirs;  token = the first kept i, by index, with sum_{j <= i, kept} w_j > u * (mass of the kept)
// and its log-probability among the kept.  Each filter keeps a prefix of the order.  T <= 0: the first of the order.
// Masses are double: a token changes with the last bits of a sum, and the same numbers are to give the same token wherever they are added up.
//
// What a filter leaves is mostly few tokens.  A row is read once, every thread keeping the maxima of its chunks; a bound that all kept tokens reach -- the
// top_k-th largest of the threads' maxima, or the largest logit + T ln min_p -- picks the chunks that are read again, and the candidates that they hold are sorted
// and filtered exactly.  A nucleus without other filters needs the mass of the whole row as well: the pass adds it up in float, and where what is known of its error
// leaves the nucleus' last token open, or the candidates do not reach it, the row is left to a second kernel, as are rows without filters.
//
// 1024 x 151 936 bf16, top-k 50 and top-p 0.95: 82 us, 3.8 TB/s, where a copy's rate would take 48: half of a row's time on an SM, which it shares with another, is the
// chain behind its reads (the wait for the last warp and the bound, candidates by two reads, sorting, filtering, drawing: 5000 cycles each at most), and 1024 rows are
// 3.5 rounds of 296 (2664 rows 185-193 us).  One row: 11.5 us by four blocks.
#include <curand_kernel.h>

#include <algorithm>

#include "common.cuh"
#include "logit_rows.cuh"
#include "per_device.h"
#include "vocab_rows.h"

namespace nrl {

struct RowFilter {
  double temp, inv_temp, top_p, min_p;
  int top_k;                                               // 0: none
  NRL_DEVICE RowFilter(const SampleFilters& f, long r, int V) {
    temp = f.temperature ? f.temperature[r] : f.temperature_all;
    top_p = f.top_p ? f.top_p[r] : f.top_p_all;
    min_p = f.min_p ? f.min_p[r] : f.min_p_all;
    top_k = f.top_k ? f.top_k[r] : f.top_k_all;
    if (top_k < 0 || top_k >= V) top_k = 0;
    if (!(temp > 0.0)) {                                   // the first of the order, which has log-probability 0 among itself; also of one column, or a call
      temp = 1.0;                                          // that is greedy altogether would leave its rows to a second kernel which it does not launch
      top_k = 1;
    }
    if (!(min_p > 0.0)) min_p = 0.0;
    if (min_p > 1.0) min_p = 1.0;
    if (!(top_p < 1.0)) top_p = 1.0;
    inv_temp = 1.0 / temp;
  }
  NRL_DEVICE double x(float z, float mx) const { return z == mx ? 0.0 : (static_cast<double>(z) - mx) * inv_temp; }
  NRL_DEVICE double mass(float z, float mx) const { return z == mx ? 1.0 : exp((static_cast<double>(z) - mx) * inv_temp); }
};

// The float sum of 2^x of a row is off by so much of itself at most, in units of 2^-24: 50 for a step's terms and for joining threads, warps and blocks; for every step of a
// thread, of 512 x 32 elements at least, 3 of its additions and 4 of 2^x where the reference moves; 4 of 2^x; 3 of every exponent, whose mean over the mass is
// log2 V <= 31, times ln 2.
NRL_DEVICE double sum_error(int V) { return (120.0 + V / 2300.0) * 0x1p-24; }

struct SampleShared {
  BorderShared border;
  RowList list;
  BoundShared bound;
  double scan[kRowWarps];
  float2 part[kRowWarps];                                  // maximum and sum of every warp
  int token;
};

constexpr int kBins = 32;                                  // ranges of logits a pass of the long way
struct LongShared {
  BorderShared border;
  RowList list;
  double scan[kRowWarps];
  double mass[kRowClusterMax][kRowWarps], whole[kRowClusterMax];         // kept for good and altogether, by ranges of the row
  double powers[128];
  double kept;                                             // what min_p keeps, by float sums
  float bins[kBins + 2];                                   // what lies above them, they, and what lies below
  float4 edges;                                            // where the next ranges begin, kept for good from, open from, enough
  unsigned short place[kCandidates];
  int base, token;
};
constexpr double kRangeSlack = 1e-5;                       // of the mass: what float sums may be off by when ranges are picked; double ones check them

// sums over the threads up to and with this one, and over all
NRL_DEVICE double block_scan(double v, double& all, double* red) {
  const int lane = static_cast<int>(lane_id()), warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 31) red[warp] = v;
  __syncthreads();
  double w = red[lane % kRowWarps];                        // every warp adds up the warps' sums, in one order
#pragma unroll
  for (int o = 1; o < kRowWarps; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane % kRowWarps >= o) w += y;
  }
  all = __shfl_sync(0xffffffffu, w, kRowWarps - 1);
  const double before = __shfl_sync(0xffffffffu, w, warp - 1);
  return warp > 0 ? before + v : v;
}

// The smallest key in [lo, top] whose mass is at least min_p -- the largest logit is in whatever min_p says -- by every lane of a warp: each tries one of 32 keys of a range,
// seven times.
NRL_DEVICE uint32_t least_key(const RowFilter& f, float mx, uint32_t lo0, uint32_t top) {
  uint64_t lo = lo0, hi = top;                             // in [lo, hi]
  while (lo < hi) {
    const uint64_t step = (hi - lo + 31) / 32, k = lo + lane_id() * step;
    const unsigned in = __ballot_sync(0xffffffffu, k >= hi || f.mass(key_logit(static_cast<uint32_t>(k)), mx) >= f.min_p);
    const int i = in ? __ffs(in) - 1 : 32;                 // the border lies behind the key of lane i - 1
    const uint64_t up = lo + static_cast<uint64_t>(i) * step;
    if (i == 0) return static_cast<uint32_t>(lo);
    lo = lo + static_cast<uint64_t>(i - 1) * step + 1;
    if (up < hi) hi = up;
  }
  return static_cast<uint32_t>(hi);
}

// By the border alone: found by ranges of keys, all in double, then the kept mass of every warp's range and a walk through the range that holds the drawn one.
// (A function of its own for every kernel: one that kernels of different register counts share ends ptxas 12.9.)
template <int KERNEL, typename T>
__device__ __noinline__ void sample_by_border(const LogitRow<T>& row, const RowFilter& f, float mx, double u, BorderShared& sh, double* masses, int* out_token,
                                              float* out_logp) {
  const int V = row.V, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t top = order_key(mx);
  auto mass = [&](float z) { return f.mass(z, mx); };
  auto one = [](float) { return 1.0; };
  uint32_t floor_key = mx == INFINITY ? top : kKeyNone + 1;
  if (f.min_p > 0.0) floor_key = least_key(f, mx, floor_key, top);
  Border b{floor_key, 0x7fffffff};
  auto total_of = [&](auto&& measure) {
    double m = 0.0;
    row.each([&](int e, float z) {
      if (b.has(order_key(clean(z)), e)) m += measure(z);
    });
    return block_sum(m, sh.red);
  };
  if (f.top_k > 0 && total_of(one) > f.top_k) b = find_border(row, floor_key, top, static_cast<double>(f.top_k), one, sh);
  if (f.top_p < 1.0) b = find_border(row, b.key, top, f.top_p > 0.0 ? f.top_p * total_of(mass) : 1e-300, mass, sh);
  // the kept mass of every warp's range, and the first range in which the drawn mass is passed
  double mine = 0.0;
  row.each([&](int e, float z) {
    if (b.has(order_key(clean(z)), e)) mine += mass(z);
  });
  mine = warp_sum(mine);
  if (lane == 0) masses[warp] = mine;
  __syncthreads();
  double total = 0.0;
  for (int w = 0; w < kRowWarps; ++w) total += masses[w];
  const double target = u * total;
  int owner = -1;
  double before = 0.0, base = 0.0;
  bool found = false;
  for (int w = 0; w < kRowWarps && !found; ++w)
    if (masses[w] > 0.0) {
      owner = w;
      before = base;
      base += masses[w];
      found = base > target;
    }
  if (warp != owner) return;
  const int per = (row.nvec + kRowWarps - 1) / kRowWarps, stop = min(row.nvec, (warp + 1) * per);
  int token = -1;
  for (int v0 = warp * per; v0 < stop; v0 += 32) {
    const int v = v0 + lane, e0 = v * LogitRow<T>::N - row.skew;
    float x[LogitRow<T>::N];
    double w[LogitRow<T>::N], sum = 0.0;
    int last = -1;
#pragma unroll
    for (int j = 0; j < LogitRow<T>::N; ++j) w[j] = 0.0;
    if (v < stop) {
      row.load(v, x);
#pragma unroll
      for (int j = 0; j < LogitRow<T>::N; ++j)
        if (e0 + j >= 0 && e0 + j < V && b.has(order_key(clean(x[j])), e0 + j)) {
          w[j] = mass(x[j]);
          if (w[j] > 0.0) last = e0 + j;
        }
    }
#pragma unroll
    for (int j = 0; j < LogitRow<T>::N; ++j) sum += w[j];
    double incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    double a = before + (incl - sum);
    int hit = -1;
#pragma unroll
    for (int j = 0; j < LogitRow<T>::N; ++j) {
      a += w[j];
      if (hit < 0 && w[j] > 0.0 && a > target) hit = e0 + j;
    }
    const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), any = __ballot_sync(0xffffffffu, last >= 0);
    if (any) token = __shfl_sync(0xffffffffu, last, 31 - __clz(any));        // where rounding lets no token pass: the last
    if (hits) {
      token = __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
      break;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) {
    const float z = row.at(token);
    *out_token = token;
    *out_logp = static_cast<float>(f.x(z, mx) - log(total));
  }
}

// w = e^((z - mx) / T) of a row, to a few steps of double, by a table and a short series (P. T. P. Tang, 1989): (z - mx) / T = (n + r) ln 2 / 128, n whole, |r| <= 1/2, so that
// w = 2^(n / 128) e^(r ln 2 / 128), the first from a table of 128 and an exponent, the second by five terms (the sixth is below 2e-15 of them).  Not for z below
// mx - 690 T, which has no such power of 2 (nor a share of a sum).
struct RowMass {
  double a, mx;                                            // n + r = (z - mx) a
  const double* powers;                                    // 2^(j / 128)
  static constexpr double kLn2 = 0.69314718055994530942;
  NRL_DEVICE RowMass(const RowFilter& f, float largest, const double* table) : a(f.inv_temp * (128.0 / kLn2)), mx(largest), powers(table) {}
  NRL_DEVICE double operator()(float z) const {
    constexpr double kMagic = 6755399441055744.0;          // 1.5 * 2^52: the sum's low bits are the whole number
    constexpr double kStep = kLn2 / 128;
    const double y = (static_cast<double>(z) - mx) * a, t = y + kMagic, r = y - (t - kMagic);
    const int n = __double2loint(t);
    double e = fma(r, kStep * kStep * kStep * kStep / 24, kStep * kStep * kStep / 6);
    e = fma(r, e, kStep * kStep / 2);
    e = fma(r, e, kStep);
    e = fma(r, e, 1.0);
    const double p = powers[n & 127];
    return e * __hiloint2double(__double2hiint(p) + ((n >> 7) << 20), __double2loint(p));
  }
};

// *addr += x in shared memory that no other thread uses
NRL_DEVICE void add_shared(uint32_t addr, float x) {
  float y;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(y) : "r"(addr) : "memory");
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(y + x) : "memory");
}

// ---- the long way -------------------------------------------------------------------------------------------------------------------------------
// Rows of which many tokens are kept: a nucleus of more than fit, or all.  The blocks of a cluster share a row.  (1) Where a nucleus ends is narrowed down by passes in
// float that add up the mass of 32 ranges of logits, every lane for itself in shared memory, until one range holds few tokens: two passes for the logits of an untrained
// model.  (2) One pass in double: what lies above that range, for every warp's range of the row, and altogether; the tokens inside are gathered.  (3) The first
// block sorts those, finds the last kept token, and walks through the range of the row that holds the drawn mass.  What does not work out (many tokens of one
// logit) is left to sample_by_border: then false.
// 256 x 151 936 bf16, top-p 0.95 of logits of deviation 0.6: 187 us (behind min-p 0.02 175, without filters 88), of which 30 the kernel in front; 19 instructions an element for each pass in float and 31 for the
// one in double fill the issue slots to 62 %; 108 SMs have two rows and 40 one.  A first look at a fourth of the row in place of the first pass, and vectors fetched
// one ahead, gave nothing.
template <typename T>
NRL_DEVICE bool sample_long(const LogitRow<T>& row, const RowFilter& f, float mx, double u, int rank, int blocks, uint32_t* s_hist, LongShared& sh,
                            RowMail* mail, int* out_token, float* out_logp) {
  constexpr int N = LogitRow<T>::N;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const RowShare share(row.nvec, rank, blocks, 1);
  const float c = log2_scale(f.inv_temp);
  if (tid < 128) sh.powers[tid] = exp2(tid / 128.0);
  const RowMass mass(f, mx, sh.powers);
  if (tid == 0) sh.list.n = sh.list.nhits = 0;
  uint32_t floor_key = kKeyNone + 1;                       // of the least logit that min_p keeps
  if (f.min_p > 0.0) floor_key = least_key(f, mx, floor_key, order_key(mx));
  // (rounded up: to nearest, the next float below mx would be in at up to 1380 temperatures, for which RowMass has no exponent)
  const float floor = fmaxf(key_logit(floor_key), __double2float_ru(mx - 690.0 * f.temp));
  const bool nucleus = f.top_p < 1.0;
  // kept for good: logits from `high` on; open: those from `low` on
  float high = floor, low = floor;
  __syncthreads();
  if (nucleus) {
    high = INFINITY;
    // what lies below V / (1 - p) times less than the largest is less than 1 - p of the whole; with min_p the ranges begin with what that keeps
    const double reach = f.temp * (log(static_cast<double>(row.V)) - log1p(-f.top_p)) + 1e-3;
    if (!(f.min_p > 0.0)) low = fmaxf(floor, static_cast<float>(mx - reach));
    float edge = mx;                                       // where the ranges begin
    uint32_t* const mine = s_hist + warp * (kBins + 2) * 32 + lane;
    bool enough = false;
#pragma unroll 1
    for (int pass = 0; pass < 6 && !enough; ++pass) {
#pragma unroll 8
      for (int i = 0; i < kBins + 2; ++i) mine[i * 32] = 0;
      // The number of a logit's range -- 0 above them, 1 .. kBins, kBins + 1 below -- is (edge + half a range - z) / (kBins + 1) ranges, held within 0 and 1, times kBins + 1 and
      // rounded, which the addition of 2^23 does; its bits shifted to a range's 128 bytes, less 2^23's, which leave 2^31 there.
      // With min_p the first ranges hold all that it keeps: what they sum up to is the whole, in later passes as well, whose bin below has tokens that count and others that
      // do not.  They reach a little lower, or the least logit kept would lie on the last one's edge and rounding would put its tokens on either side.
      const float least = f.min_p > 0.0 && pass == 0 ? low - (2e-6f * (edge - low) + 1e-6f * (fabsf(edge) + fabsf(low))) : low;
      const float per = 1.f / fmaxf((edge - least) * ((kBins + 1.f) / kBins), 1e-30f), zero = (edge + (edge - least) * (0.5f / kBins)) * per;
      const uint32_t bins = smem_u32(mine) - 0x80000000u;
      const uint64_t neg2 = pair_both(-mx), c2 = pair_both(c);
#pragma unroll 1
      for (int v = share.first + tid; v < share.end; v += kRowThreads) {
        RawVec a = row.raw(v);
        LogitRow<T>::drop_nan(a);
#pragma unroll
        for (int q = 0; q < N / 2; ++q) {
          const uint64_t z = LogitRow<T>::pair(a, q);
          const float2 x = pair_parts(z), e = pair_parts(pair_mul(pair_add(z, neg2), c2));
          add_shared(bins + (__float_as_uint(fmaf(__saturatef(fmaf(x.x, -per, zero)), kBins + 1.f, 8388608.f)) << 7), ex2(e.x));
          add_shared(bins + (__float_as_uint(fmaf(__saturatef(fmaf(x.y, -per, zero)), kBins + 1.f, 8388608.f)) << 7), ex2(e.y));
        }
      }
      __syncthreads();
#pragma unroll 1
      for (int b = warp; b < kBins + 2; b += kRowWarps) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) sum += __uint_as_float(s_hist[(w * (kBins + 2) + b) * 32 + lane]);
        sum = warp_sum(sum);
        if (lane == 0) (blocks > 1 ? mail->bins[rank] : sh.bins)[b] = sum;
      }
      __syncwarp();
      if (blocks > 1) {
        cluster_arrive();
        cluster_wait();
      } else {
        __syncthreads();
      }
      if (rank == 0 && warp == 0) {                        // a lane a range
        double m = 0.0, start = 0.0, rest = 0.0;
        for (int q = 0; q < blocks; ++q) {
          m += blocks > 1 ? __ldcg(&mail->bins[q][lane + 1]) : sh.bins[lane + 1];
          start += blocks > 1 ? __ldcg(&mail->bins[q][0]) : sh.bins[0];
          rest += f.min_p > 0.0 ? 0.0 : blocks > 1 ? __ldcg(&mail->bins[q][kBins + 1]) : sh.bins[kBins + 1];
        }
        double upto = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += y;
        }
        upto += start;
        double whole = __shfl_sync(0xffffffffu, upto, 31) + rest;
        if (f.min_p > 0.0) {
          if (pass > 0) whole = sh.kept;
          else if (lane == 0) sh.kept = whole;
        }
        // from the range in which the mass passes what the nucleus needs, less what float sums may be off by, to the one in which it passes that and as much more
        const unsigned past0 = __ballot_sync(0xffffffffu, upto >= whole * (f.top_p - kRangeSlack)), past1 = __ballot_sync(0xffffffffu, upto >= whole * (f.top_p + kRangeSlack));
        const int b0 = past0 ? __ffs(past0) - 1 : 31, b1 = past1 ? __ffs(past1) - 1 : 31;
        const double open = __shfl_sync(0xffffffffu, upto, b1) - __shfl_sync(0xffffffffu, upto - m, b0);
        const float width = (edge - least) / kBins, over = width / 1024 + 1e-6f * (fabsf(edge) + fabsf(low));        // for the edges' rounding
        const float e1 = b0 == 0 ? edge : edge - b0 * width + over, e0 = b1 == kBins - 1 ? low : edge - (b1 + 1) * width - over;
        const float next_high = b0 > 0 ? e1 : high, next_low = fmaxf(e0, low);
        const bool ok = open <= 1700.0 * ex2((next_low - mx) * c);        // tokens, by the least of their masses; those on the edges come on top
        if (lane == 0) (blocks > 1 ? mail->edges : sh.edges) = make_float4(e1, next_high, next_low, ok ? 1.f : 0.f);
        __syncwarp();
      }
      if (blocks > 1) {
        cluster_arrive();
        cluster_wait();
      } else {
        __syncthreads();
      }
      const float4 next = blocks > 1 ? __ldcg(&mail->edges) : sh.edges;
      edge = next.x;
      high = next.y;
      low = next.z;
      enough = next.w != 0.f;
    }
  }
  // ---- in double: every warp's range of the row ----
  double kept = 0.0, other = 0.0;
  const int per = (share.end - share.first + kRowWarps - 1) / kRowWarps, begin = min(share.end, share.first + warp * per), stop = min(share.end, begin + per);
#pragma unroll 1
  for (int v = begin + lane; v < stop; v += 32) {
    float x[N];
    row.load(v, x);
    unsigned open = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float z = x[j];                                // (NaN is not above anything)
      const double w = mass(z);
      if (z >= high) kept += w;
      else if (z >= floor) other += w;
      open |= (z >= low && z < high ? 1u : 0u) << j;
    }
    for (; open != 0; open &= open - 1) {
      const int e = v * N - row.skew + __ffs(open) - 1, at = atomicAdd(&sh.list.n, 1);
      if (at < kCandidates) sh.list.cand[at] = static_cast<uint64_t>(order_key(row.at(e))) << 32 | static_cast<uint32_t>(~e);
    }
  }
  const double all = block_sum(kept + other, sh.scan);
  kept = warp_sum(kept);
  if (lane == 0) sh.mass[rank][warp] = kept;
  if (tid == 0) sh.whole[rank] = all;
  __syncthreads();
  if (blocks > 1) {
    if (tid < kRowWarps) mail->mass[rank][tid] = sh.mass[rank][tid];
    if (tid == 0) mail->whole[rank] = all;
    send_candidates(sh.list, rank, make_float2(0.f, 0.f), 0, *mail);
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return true;
    if (tid < blocks * kRowWarps) sh.mass[tid / kRowWarps][tid % kRowWarps] = __ldcg(&mail->mass[tid / kRowWarps][tid % kRowWarps]);
    if (tid < blocks) sh.whole[tid] = __ldcg(&mail->whole[tid]);
    __syncthreads();
  }

  // ---- the last kept token ----
  int found = candidates_of(sh.list);
  if (blocks > 1) {
    uint4 part;
    found = join_candidates(sh.list, blocks, mail, part);
  }
  if (found > kCandidates) return false;
  double above = 0.0, whole = 0.0;
  for (int q = 0; q < blocks; ++q) {
    whole += sh.whole[q];
    for (int w = 0; w < kRowWarps; ++w) above += sh.mass[q][w];
  }
  Border last{floor_key, 0x7fffffff};
  int n = 0;
  if (nucleus) {
    const double limit = f.top_p * whole;
    last.key = 0xffffffffu;
    if (found > 0) sort_front(sh.list.cand, found, reinterpret_cast<uint64_t*>(s_hist), sh.list.counts);        // the ranges of logits are not needed any more
    if (above > 0.0 && above >= limit) return false;     // the border is above the range
    double done = above;
    double* const masses = reinterpret_cast<double*>(s_hist);
#pragma unroll 1
    for (int i0 = 0; i0 < found; i0 += kRowThreads) {
      const int i = i0 + tid;
      const double w = i < found ? mass(key_logit(static_cast<uint32_t>(sh.list.cand[i] >> 32))) : 0.0;
      if (i < found) masses[i] = w;
      double sum;
      const double before = done + block_scan(w, sum, sh.scan) - w;
      n += __syncthreads_count(i < found && (before < limit || (i == 0 && above == 0.0)));
      done += sum;
    }
    if (done < limit && low > floor) return false;       // or below it
    if (n > 0) {
      const uint64_t x = sh.list.cand[n - 1];
      last.key = static_cast<uint32_t>(x >> 32);
      last.cut = static_cast<int>(~static_cast<uint32_t>(x));
    }
    // kept candidates to their ranges of the row
    const int step = (row.nvec + blocks - 1) / blocks;
    for (int i = tid; i < n; i += kRowThreads) {
      const int v = (static_cast<int>(~static_cast<uint32_t>(sh.list.cand[i])) + row.skew) / N, q = v / step, first = q * step;
      const int share_per = (min(row.nvec, first + step) - first + kRowWarps - 1) / kRowWarps;
      sh.place[i] = static_cast<unsigned short>(q * kRowWarps + (v - first) / share_per);
    }
    __syncthreads();
    for (int q = warp; q < blocks * kRowWarps; q += kRowWarps) {
      double m = 0.0;
      for (int i = lane; i < n; i += 32) m += sh.place[i] == q ? masses[i] : 0.0;
      m = warp_sum(m);
      if (lane == 0) sh.mass[q / kRowWarps][q % kRowWarps] += m;
    }
    __syncthreads();
  }
  // ---- the range that holds the drawn mass, and the token in it ----
  double total = 0.0;
  for (int i = 0; i < blocks * kRowWarps; ++i) total += sh.mass[i / kRowWarps][i % kRowWarps];
  const double target = u * total;
  double base = 0.0, before = 0.0;
  int range = -1;
  for (int i = 0; i < blocks * kRowWarps; ++i) {
    const double m = sh.mass[i / kRowWarps][i % kRowWarps];
    if (!(m > 0.0)) continue;
    range = i;
    before = base;
    base += m;
    if (base > target) break;
  }
  if (range < 0) return false;
  const RowShare there(row.nvec, range / kRowWarps, blocks, 1);
  const int tper = (there.end - there.first + kRowWarps - 1) / kRowWarps, t0 = min(there.end, there.first + range % kRowWarps * tper), t1 = min(there.end, t0 + tper);
  if (tid == 0) {
    sh.token = -1;
    sh.base = 0x7fffffff;                                  // the first thread up to whose tokens the mass passes
  }
  int lead = -1;                                           // of this thread: its last kept token
  __syncthreads();
#pragma unroll 1
  for (int v0 = t0; v0 < t1; v0 += kRowThreads) {
    const int v = v0 + tid, e0 = v * N - row.skew;
    float x[N];
    double sum = 0.0;
    if (v < t1) {
      row.load(v, x);
#pragma unroll 1
      for (int j = 0; j < N; ++j) {
        const float z = clean(x[j]);
        if (e0 + j >= 0 && e0 + j < row.V && z >= floor && (z >= high || last.has(order_key(z), e0 + j))) {
          const double w = mass(z);
          sum += w;
          if (w > 0.0) lead = e0 + j;
        }
      }
    }
    double tile;
    const double upto = before + block_scan(sum, tile, sh.scan);
    if (sum > 0.0 && upto > target) atomicMin(&sh.base, tid);
    __syncthreads();
    if (sh.base == tid) {
      double a = upto - sum;
      int hit = lead;
#pragma unroll 1
      for (int j = 0; j < N; ++j) {
        const float z = clean(x[j]);
        if (e0 + j >= 0 && e0 + j < row.V && z >= floor && (z >= high || last.has(order_key(z), e0 + j))) {
          const double w = mass(z);
          a += w;
          if (w > 0.0 && a > target) {
            hit = e0 + j;
            break;
          }
        }
      }
      sh.token = hit;
    }
    before += tile;
    if (sh.base != 0x7fffffff) break;
  }
  if (sh.base == 0x7fffffff && lead >= 0) atomicMax(&sh.token, lead);      // rounding lets none pass: the range's last
  __syncthreads();
  if (tid == 0) {
    *out_token = sh.token;
    *out_logp = static_cast<float>(f.x(row.at(sh.token), mx) - log(total));
  }
  return true;
}

// rows whose largest logit the kernel in front has left in `top` (NaN: drawn already)
template <typename T>
__global__ void __launch_bounds__(kRowThreads, 2) sample_long_kernel(const T* __restrict__ logits, long row_stride, int V, const float* __restrict__ uniforms,
                                                                     SampleFilters filters, const float* __restrict__ top, int* __restrict__ tokens,
                                                                     float* __restrict__ logp, unsigned char* mails, size_t mail_bytes) {
  extern __shared__ __align__(16) uint32_t s_hist[];       // floats [warps][kBins + 2][32]
  __shared__ LongShared sh;
  const int rank = static_cast<int>(cluster_rank()), blocks = static_cast<int>(cluster_blocks());
  const long r = blockIdx.x / blocks;
  const float mx = top[r];
  if (mx != mx) return;
  const LogitRow<T> row(logits + r * row_stride, V);
  const RowFilter f(filters, r, V);
  if (!sample_long(row, f, mx, uniforms[r], rank, blocks, s_hist, sh, reinterpret_cast<RowMail*>(mails + r * mail_bytes), tokens + r, logp + r)) {
    __syncthreads();
    sample_by_border<1>(row, f, mx, uniforms[r], sh.border, sh.scan, tokens + r, logp + r);
  }
}

// Groups whose maxima bound the candidates of a nucleus: more of them reach further nuclei and cost more candidates.  us with 128 / 256 / 384, top-p 0.95: 1024 rows x 151 936 bf16
// whose nuclei have 69 tokens in the median and 20 000 at the ninth decile 352 / 379 / 397, few tokens 106 / 134 / 151; 300 rows of floats 161 / 172 / 177; one row 19 / 22.5 / 43.
constexpr int kNucleusGroups = 128;

// Over the sorted candidates: how many of them are kept; 0: it is not known (nucleus of a whole row whose mass `whole` is a float sum, or whose last token is
// not among the `sure` first, beyond which others may come between).  mass, upto: theirs, and the sums up to and with every one.
NRL_DEVICE int kept_of(const uint64_t* x, int found, int sure, const RowFilter& f, float mx, double whole, double off, double* mass, double* upto, SampleShared& sh) {
  const int tid = threadIdx.x, n1 = f.top_k > 0 && f.top_k < found ? f.top_k : found;
  double done = 0.0;
#pragma unroll 1
  for (int i0 = 0; i0 < n1; i0 += kRowThreads) {
    const int i = i0 + tid;
    double w = i < n1 ? f.mass(key_logit(static_cast<uint32_t>(x[i] >> 32)), mx) : 0.0, all;
    if (w < f.min_p) w = 0.0;
    const double sum = done + block_scan(w, all, sh.scan);
    if (i < n1) {
      mass[i] = w;
      upto[i] = sum;
    }
    done += all;
  }
  __syncthreads();
  double limit = f.top_p < 1.0 ? f.top_p * (whole > 0.0 ? whole : done) : 1e300, low = limit;
  if (whole > 0.0) {
    low *= 1.0 - off;
    limit *= 1.0 + off;
  }
  int n = 0;
  bool open = false;
#pragma unroll 1
  for (int i0 = 0; i0 < n1; i0 += kRowThreads) {
    const int i = i0 + tid;
    const bool some = i < n1 && mass[i] > 0.0;
    const double before = some && i > 0 ? upto[i - 1] : -1.0;
    open |= before >= low && before < limit;
    n += __syncthreads_count(some && before < low);
  }
  if (whole > 0.0 && (__syncthreads_or(open) || n >= sure)) return 0;        // the token behind the last kept has to be a candidate
  return n;
}

// from the n first candidates, which are sorted, by index; the log-probability from the logit: the quotient of a kept mass and the whole may be below float's range
template <typename T>
NRL_DEVICE void draw_of(const LogitRow<T>& row, uint64_t* x, int n, const RowFilter& f, float mx, const double* mass, double total, double u, SampleShared& sh, uint64_t* y,
                        int* out_token, float* out_logp) {
  const int tid = threadIdx.x;
  for (int i = tid; i < n; i += kRowThreads) x[i] = x[i] << 32 | static_cast<uint32_t>(i);        // (~index, place)
  sort_front(x, n, y, sh.list.counts);                               // (its first barrier is behind the swap)
  if (tid == 0) sh.token = 0x7fffffff;
  const double target = u * total;
  double done = 0.0;
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += kRowThreads) {
    const int i = i0 + tid;
    const double w = i < n ? mass[static_cast<uint32_t>(x[i])] : 0.0;
    double all;
    const double upto = done + block_scan(w, all, sh.scan);
    if (i < n && upto > target) atomicMin(&sh.token, i);
    done += all;
  }
  __syncthreads();
  if (tid == 0) {
    const int token = static_cast<int>(~static_cast<uint32_t>(x[min(sh.token, n - 1)] >> 32));
    *out_token = token;
    *out_logp = static_cast<float>(f.x(row.at(token), mx) - log(total));
  }
}

// Both in one warp, for up to 64 sorted candidates that hold all that is kept: 1024 x 151 936 with top-k 50 and top-p 0.95 87 us by
// the block and 80 by a warp, one row 12.4 / 11.3.
constexpr int kDrawWarp = 64;
NRL_DEVICE void draw_in_warp(const uint64_t* x, int n1, const RowFilter& f, float mx, double u, double* mass, int* out_token, float* out_logp) {
  const int lane = threadIdx.x & 31;
  double w[2], upto[2], before[2], done = 0.0;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int i = lane + t * 32;
    w[t] = i < n1 ? f.mass(key_logit(static_cast<uint32_t>(x[i] >> 32)), mx) : 0.0;
    if (w[t] < f.min_p) w[t] = 0.0;
    mass[i] = upto[t] = w[t];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, upto[t], o);
      if (lane >= o) upto[t] += y;
    }
    upto[t] += done;
    before[t] = __shfl_up_sync(0xffffffffu, upto[t], 1);
    if (lane == 0) before[t] = done;
    done = __shfl_sync(0xffffffffu, upto[t], 31);
  }
  const double limit = f.top_p < 1.0 ? f.top_p * done : 1e300;
  int n = 0;                                               // (the first is kept whatever top_p says)
#pragma unroll
  for (int t = 0; t < 2; ++t) n += __popc(__ballot_sync(0xffffffffu, w[t] > 0.0 && (before[t] < limit || (t == 0 && lane == 0))));
  const double total = __shfl_sync(0xffffffffu, n > 32 ? upto[1] : upto[0], (n - 1) & 31), target = u * total, log_total = log(total);
  __syncwarp();
  const uint32_t at0 = static_cast<uint32_t>(x[lane]), at1 = static_cast<uint32_t>(x[lane + 32]);        // ~index
  double a0 = 0.0, a1 = 0.0;                               // mass of the kept ones up to and with it, by index
#pragma unroll 4
  for (int j = 0; j < n; ++j) {
    const uint32_t at = static_cast<uint32_t>(x[j]);
    const double m = mass[j];
    a0 += at >= at0 ? m : 0.0;
    a1 += at >= at1 ? m : 0.0;
  }
  const bool in0 = lane < n, in1 = lane + 32 < n;
  const uint32_t first = __reduce_max_sync(0xffffffffu, max(in0 && a0 > target ? at0 : 0u, in1 && a1 > target ? at1 : 0u));
  const uint32_t last = __reduce_min_sync(0xffffffffu, min(in0 ? at0 : 0xffffffffu, in1 ? at1 : 0xffffffffu));
  const uint32_t token = first != 0u ? first : last;       // rounding lets none pass: the last
#pragma unroll
  for (int t = 0; t < 2; ++t)
    if ((t == 0 ? in0 && at0 == token : in1 && at1 == token)) {
      *out_token = static_cast<int>(~token);
      *out_logp = static_cast<float>(f.x(key_logit(static_cast<uint32_t>(x[lane + t * 32] >> 32)), mx) - log_total);
    }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads, 2) sample_filtered_kernel(const T* __restrict__ logits, long row_stride, int V,
                                                                         const float* __restrict__ uniforms, SampleFilters filters, int* __restrict__ tokens,
                                                                         float* __restrict__ logp, float* __restrict__ top, unsigned char* mails, size_t mail_bytes) {
  extern __shared__ __align__(16) float s_chunk[];         // [chunks][kRowThreads]
  static_assert(kRowChunks * kRowThreads * 4 >= 2 * kCandidates * 8, "masses and sums of the candidates in their place");
  __shared__ SampleShared sh;
  const int rank = static_cast<int>(cluster_rank()), blocks = static_cast<int>(cluster_blocks()), tid = threadIdx.x;
  const long r = blockIdx.x / blocks;
  if (tid == 0) sh.list.n = sh.list.nhits = 0;
  RowMail* const mail = reinterpret_cast<RowMail*>(mails + r * mail_bytes);        // of several blocks
  const LogitRow<T> row(logits + r * row_stride, V);
  const RowFilter f(filters, r, V);
  const RowShare share(row.nvec, rank, blocks, kFlight);
  const bool few = (f.top_k > 0 && f.top_k <= kTopMax) || f.min_p > 0.0;        // what is kept is a matter of the candidates alone
  const bool nucleus = !few && f.top_p < 1.0 && f.top_k == 0;
  const float c = log2_scale(f.inv_temp);
  float best, m = 0.f, s = 0.f;
  if (nucleus)
    row_pass<kFlight, true>(row, share, c, s_chunk, best, m, s, SkipNan<T>());
  else
    row_pass<kFlight, false>(row, share, c, s_chunk, best, m, s, SkipNone());
  // a thread's chunks in one group up to 256 tokens, in up to four above
  const int want = few ? (f.top_k > 0 && f.top_k <= kTopMax ? f.top_k : 0) : kNucleusGroups, groups = want <= 256 ? 1 : want <= 512 ? 2 : 4;
  uint32_t bound = kKeyNone + 1;
  put_state(nucleus ? m : best, s, c, sh.part);            // (without a nucleus the sum is 0)
  if (few || nucleus) {
    if (want > 0) {
      uint32_t keys[kGroupsMax];
      keys[0] = order_key(best);
      if (groups > 1)
#pragma unroll
        for (int g = 0; g < kGroupsMax; ++g) {
          float x = -INFINITY;
          for (int i = g; i < share.chunks; i += groups) x = fmaxf(x, s_chunk[i * kRowThreads + tid]);
          keys[g] = order_key(x);
        }
      bound = group_bound(keys, groups, want, sh.bound);
    }
    if (f.min_p > 0.0) {                                   // min_p of the block's largest logit or below: a little less than its border
      const float mb = block_max(best, reinterpret_cast<float*>(sh.scan));
      const double t = f.temp * log(f.min_p), z = mb + t - 1e-6 * (fabs(static_cast<double>(mb)) - t);
      if (z > -3e38 && z < 3e38) bound = max(bound, order_key(static_cast<float>(z)));
    }
    gather_candidates(row, share, s_chunk, bound, sh.list);
  } else {
    __syncthreads();
  }
  const float2 state = get_state(c, sh.part);
  float mx = state.x;
  double whole = state.y;
  uint32_t least = bound;
  int found = candidates_of(sh.list);
  if (blocks > 1) {
    send_candidates(sh.list, rank, state, bound, *mail);
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
    uint4 part;
    found = join_candidates(sh.list, blocks, mail, part);
    join_states(__uint_as_float(part.x), __uint_as_float(part.y), c, mx, whole);
    least = __reduce_max_sync(0xffffffffu, part.w);
  }
  const double u = uniforms[r];
  float open = __int_as_float(0x7fffffff);                 // NaN: drawn
  if (mx == -INFINITY || ((few || nucleus) && found == 0)) {        // nothing to draw from
    if (tid == 0) {
      tokens[r] = -1;
      logp[r] = -INFINITY;
    }
  } else if (mx == INFINITY || (few && found > kCandidates && f.top_k > 0) || (!few && f.top_k > 0)) {
    sample_by_border<0>(row, f, mx, u, sh.border, sh.scan, tokens + r, logp + r);
  } else if ((few || nucleus) && found <= kCandidates) {
    int sure = found;
    if (nucleus) {
      int n = 0;
      for (int i = tid; i < found; i += kRowThreads) n += static_cast<uint32_t>(sh.list.cand[i] >> 32) >= least ? 1 : 0;
      sure = static_cast<int>(block_sum(static_cast<double>(n), sh.border.red));
    }
    sort_front(sh.list.cand, found, reinterpret_cast<uint64_t*>(s_chunk), sh.list.counts);        // the maxima are not needed any more
    double* mass = reinterpret_cast<double*>(s_chunk);
    double* upto = mass + kCandidates;
    const int n1 = f.top_k > 0 ? min(f.top_k, found) : found;
    if (few && n1 <= kDrawWarp) {
      if (tid < 32) draw_in_warp(sh.list.cand, n1, f, mx, u, mass, tokens + r, logp + r);
    } else {
      const int n = kept_of(sh.list.cand, found, sure, f, mx, nucleus ? whole : 0.0, sum_error(V), mass, upto, sh);
      if (n > 0) draw_of(row, sh.list.cand, n, f, mx, mass, upto[n - 1], u, sh, reinterpret_cast<uint64_t*>(upto), tokens + r, logp + r);
      else open = mx;
    }
  } else {
    open = mx;
  }
  if (tid == 0 && top != nullptr) top[r] = open;
}

__global__ void row_uniforms_kernel(unsigned long long seed, unsigned long long step, const int* __restrict__ row_ids, const int* __restrict__ row_steps,
                                    int rows, float* __restrict__ out) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= rows) return;
  curandStatePhilox4_32_10_t st;
  curand_init(seed, static_cast<unsigned long long>(row_ids ? row_ids[i] : i), step + (row_steps ? static_cast<unsigned long long>(row_steps[i]) : 0ull), &st);
  out[i] = fminf(1.f - curand_uniform(&st), 0x1.fffffep-1f);        // (0, 1] -> [0, 1): the difference is rounded to 1 from 2^-25 down
}

// Filters of every row's own send a part of the rows on, which twice the blocks finish sooner: 250 x 50 021 floats, a third of them, 70 / 63.5 / 62 us in all with 1 / 2 / 4;
// where all rows come, 256 x 151 936, 194 / 229 / 284.  Of more than 1024 rows a third fill the SMs, and
// several blocks would want 19 KB of scratch a row.
template <typename T>
int long_blocks(int rows, int V, const SampleFilters& f) {
  const int blocks = row_blocks(rows, V, LogitRow<T>::N);
  const bool own = f.top_k != nullptr || f.top_p != nullptr || f.min_p != nullptr || f.temperature != nullptr;
  return own && rows <= 1024 ? std::min(2 * blocks, kRowClusterMax) : blocks;
}

template <typename T>
cudaError_t launch_sample(const void* logits, long row_stride, int rows, int V, const float* uniforms, const SampleFilters& f, int* tokens, float* logp,
                          float* top, void* scratch, cudaStream_t s) {
  static PerDevice<bool> done, done_long;
  if (const cudaError_t e = allow_smem(done, sample_filtered_kernel<T>, kRowChunks * kRowThreads * 4); e != cudaSuccess) return e;
  if (const cudaError_t e = allow_smem(done_long, sample_long_kernel<T>, (kBins + 2) * kRowThreads * 4); e != cudaSuccess) return e;
  const int blocks = row_blocks(rows, V, LogitRow<T>::N), more = long_blocks<T>(rows, V, f);
  unsigned char* const mails = static_cast<unsigned char*>(scratch);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * blocks);
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = kRowChunks * kRowThreads * 4;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const T* z = static_cast<const T*>(logits);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_filtered_kernel<T>, z, row_stride, V, uniforms, f, tokens, logp, top, mails, row_mail_bytes(blocks));
  if (e != cudaSuccess || top == nullptr) return e;
  cfg.dynamicSmemBytes = (kBins + 2) * kRowThreads * 4;
  attr[0].val.clusterDim.x = more;
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * more);
  return cudaLaunchKernelEx(&cfg, sample_long_kernel<T>, z, row_stride, V, uniforms, f, static_cast<const float*>(top), tokens, logp, mails,
                            row_mail_bytes(more));
}

}  // namespace nrl

using namespace nrl;

// Every row is settled by its candidates, or by its border in the first kernel: one top_k of 1 to kTopMax for all, or temperature 0.
extern "C" int nrl_sample_is_short(const SampleFilters* f, int V) {
  const bool greedy = f->temperature == nullptr && !(f->temperature_all > 0.0);
  return greedy || (f->top_k == nullptr && f->top_k_all > 0 && f->top_k_all <= kTopMax && f->top_k_all < V);
}

extern "C" size_t nrl_sample_scratch(int is_bf16, int rows, int V, const SampleFilters* f) {
  const int blocks = row_blocks(rows, V, is_bf16 ? LogitRow<__nv_bfloat16>::N : LogitRow<float>::N);
  const int more = nrl_sample_is_short(f, V) ? blocks : is_bf16 ? long_blocks<__nv_bfloat16>(rows, V, *f) : long_blocks<float>(rows, V, *f);
  return rows * row_mail_bytes(std::max(blocks, more));    // one after the other
}

extern "C" cudaError_t nrl_sample_filtered(const void* logits, int is_bf16, long row_stride, int rows, int V, const float* uniforms, const SampleFilters* f,
                                           int* tokens, float* logp, float* top, void* scratch, cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  if (top == nullptr && !nrl_sample_is_short(f, V)) return cudaErrorInvalidValue;
  return is_bf16 ? launch_sample<__nv_bfloat16>(logits, row_stride, rows, V, uniforms, *f, tokens, logp, top, scratch, s)
                 : launch_sample<float>(logits, row_stride, rows, V, uniforms, *f, tokens, logp, top, scratch, s);
}

extern "C" cudaError_t nrl_row_uniforms(unsigned long long seed, unsigned long long step, const int* row_ids, const int* row_steps, int rows, float* out,
                                        cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  row_uniforms_kernel<<<(rows + 127) / 128, 128, 0, s>>>(seed, step, row_ids, row_steps, rows, out);
  return cudaGetLastError();
}
