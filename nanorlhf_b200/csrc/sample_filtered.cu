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
#include <curand_kernel.h>

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
    if (!(temp > 0.0)) {                                   // the first of the order, which has log-probability 0 among itself
      temp = 1.0;
      top_k = 1;
    }
    if (top_k < 0 || top_k >= V) top_k = 0;
    if (!(min_p > 0.0)) min_p = 0.0;
    if (min_p > 1.0) min_p = 1.0;
    if (!(top_p < 1.0)) top_p = 1.0;
    inv_temp = 1.0 / temp;
  }
  NRL_DEVICE double x(float z, float mx) const { return z == mx ? 0.0 : (static_cast<double>(z) - mx) * inv_temp; }
  NRL_DEVICE double mass(float z, float mx) const { return z == mx ? 1.0 : exp((static_cast<double>(z) - mx) * inv_temp); }
};

struct SampleShared {
  BorderShared border;
  RowList list;
  BoundShared bound;
  double scan[kRowWarps];
  float2 part[kRowClusterMax][kRowWarps];                  // maximum and sum of every warp of the cluster
  uint32_t part_bound[kRowClusterMax];
  int base, token;
};

constexpr int kBins = 16;                                  // ranges of logits a pass of the long way
struct LongShared {
  BorderShared border;
  RowList list;
  double scan[kRowWarps];
  double mass[kRowClusterMax][kRowWarps], whole[kRowClusterMax];         // kept for good and altogether, by ranges of the row
  double powers[32];                                       // 2^(j / 32)
  float bins[2][kRowClusterMax][kBins + 2];                // and what lies above them and below
  unsigned short place[kCandidates];
  int base, token;
};

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
  double before = 0.0;
  all = 0.0;
#pragma unroll 1
  for (int w = 0; w < kRowWarps; ++w) {
    if (w == warp) before = all;
    all += red[w];
  }
  return before + v;
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
  if (f.min_p > 0.0) {                            // smallest key whose mass is min_p: every lane tries one of 32 keys of a range, seven times
    uint64_t lo = floor_key, hi = top;                     // in [lo, hi]; the largest logit is in whatever min_p says
    while (lo < hi) {
      const uint64_t step = (hi - lo + 31) / 32, k = lo + lane * step;
      const unsigned in = __ballot_sync(0xffffffffu, k >= hi || mass(key_logit(static_cast<uint32_t>(k))) >= f.min_p);
      const int i = in ? __ffs(in) - 1 : 32;               // the border lies behind the key of lane i - 1
      const uint64_t up = lo + static_cast<uint64_t>(i) * step;
      if (i == 0) { hi = lo; break; }
      lo = lo + static_cast<uint64_t>(i - 1) * step + 1;
      if (up < hi) hi = up;
    }
    floor_key = static_cast<uint32_t>(hi);
  }
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

// e^x, x <= 0, to a few steps of double, by a table and a short series (P. T. P. Tang, 1989): x = (32 i + j) ln 2 / 32 + f, |f| <= ln 2 / 64, and six
// terms of e^f (the seventh is below 3e-15 of them).  12 operations in double, which are what a long row's masses cost.
NRL_DEVICE double exp_mass(double x, const double* powers) {
  if (!(x > -700.0)) return 0.0;
  constexpr double kSteps = 46.16624130844683, kStep = 0x1.62e42fefa0000p-6, kStepLow = 5.145609244655338e-14, kMagic = 6755399441055744.0;       // 32 / ln 2, ln 2 / 32 in two parts, 1.5 * 2^52
  const double t = fma(x, kSteps, kMagic);
  const int n = __double2loint(t);
  double f = fma(t - kMagic, -kStep, x);
  f = fma(t - kMagic, -kStepLow, f);
  double e = fma(f, 1.0 / 120, 1.0 / 24);
  e = fma(f, e, 1.0 / 6);
  e = fma(f, e, 0.5);
  e = fma(f, e, 1.0);
  e = fma(f, e, 1.0);
  const double p = powers[n & 31];
  return e * __hiloint2double(__double2hiint(p) + ((n >> 5) << 20), __double2loint(p));
}

// ---- the long way -------------------------------------------------------------------------------------------------------------------------------
// Rows of which many tokens are kept: a nucleus of more than fit, or all.  The blocks of a cluster share a row.  (1) Where a nucleus ends is narrowed down by passes in
// float that add up the mass of 16 ranges of logits, lane by lane in shared memory, until one range holds few tokens.  (2) One pass in double: what lies above
// that range, for every warp's range of the row, and altogether; the tokens inside are gathered.  (3) The first block sorts those, finds the last kept token, and
// walks through the range of the row that holds the drawn mass.  What does not work out (many tokens of one logit, a border next to a range's edge) is left to
// sample_by_border: then false.
template <typename T>
NRL_DEVICE bool sample_long(const LogitRow<T>& row, const RowFilter& f, float mx, double u, int rank, int blocks, float* s_bins, LongShared& sh, int* out_token,
                            float* out_logp) {
  constexpr int N = LogitRow<T>::N;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const RowShare share(row.nvec, rank, blocks);
  const float c = static_cast<float>(f.inv_temp * 1.4426950408889634);
  if (tid < 32) sh.powers[tid] = exp2(tid / 32.0);
  if (tid == 0) sh.list.n = sh.list.nhits = sh.list.sent = 0;
  // the least logit that min_p keeps: every lane tries one of 32 keys of a range, seven times
  uint32_t floor_key = kKeyNone + 1;
  if (f.min_p > 0.0) {
    uint64_t lo = floor_key, hi = order_key(mx);            // in [lo, hi]; the largest logit is in whatever min_p says
    while (lo < hi) {
      const uint64_t step = (hi - lo + 31) / 32, k = lo + lane * step;
      const unsigned in = __ballot_sync(0xffffffffu, k >= hi || f.mass(key_logit(static_cast<uint32_t>(k)), mx) >= f.min_p);
      const int i = in ? __ffs(in) - 1 : 32;
      const uint64_t up = lo + static_cast<uint64_t>(i) * step;
      if (i == 0) { hi = lo; break; }
      lo = lo + static_cast<uint64_t>(i - 1) * step + 1;
      if (up < hi) hi = up;
    }
    floor_key = static_cast<uint32_t>(hi);
  }
  const float floor = key_logit(floor_key);
  const bool nucleus = f.top_p < 1.0;
  // kept for good: logits from `high` on; open: those from `low` on
  float high = floor, low = floor;
  __syncthreads();
  if (nucleus) {
    high = INFINITY;
    // what lies below V / (1 - p) times less than the largest is less than 1 - p of the whole
    const double reach = f.temp * (log(static_cast<double>(row.V)) - log1p(-f.top_p)) + 1e-3;
    low = fmaxf(floor, static_cast<float>(mx - reach));
    float edge = mx;                                       // where the ranges begin; above it only what earlier passes put there
    bool enough = false;
#pragma unroll 1
    for (int pass = 0; pass < 8 && !enough; ++pass) {
      for (int i = tid; i < kBins * kRowThreads; i += kRowThreads) s_bins[i] = 0.f;
      __syncthreads();
      const float scale = kBins / fmaxf(edge - low, 1e-30f);
      float above = 0.f, below = 0.f;
      float* mine = s_bins + warp * kBins * 32 + lane;
#pragma unroll 1
      for (int v = share.first + tid; v < share.end; v += kRowThreads) {
        float x[N];
        row.load(v, x);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float z = clean(x[j]);
          if (z < floor) continue;
          const float e = ex2((z - mx) * c);
          if (z >= high) above += e;
          else if (z < low) below += e;
          else {
            const int b = min(kBins - 1, max(0, static_cast<int>((edge - z) * scale)));
            mine[b * 32] += e;
          }
        }
      }
      __syncthreads();
      float sum = 0.f;                                     // a warp a bin
#pragma unroll 1
      for (int w = 0; w < kRowWarps; ++w) sum += s_bins[(w * kBins + warp) * 32 + lane];
      sum = warp_sum(sum);
      const double up = block_sum(static_cast<double>(above), sh.scan), rest = block_sum(static_cast<double>(below), sh.scan);
      static_assert(kBins == kRowWarps, "a warp a bin");
      float(&slot)[kRowClusterMax][kBins + 2] = sh.bins[pass & 1];
      if (lane < blocks) {
        st_block(in_block(&slot[rank][warp], lane), sum);
        if (warp == 0) {
          st_block(in_block(&slot[rank][kBins], lane), static_cast<float>(up));
          st_block(in_block(&slot[rank][kBins + 1], lane), static_cast<float>(rest));
        }
      }
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      double cum = 0.0, all = 0.0;
      for (int q = 0; q < blocks; ++q) {
        cum += slot[q][kBins];
        for (int b = 0; b < kBins + 2; ++b) all += slot[q][b];
      }
      const double target = f.top_p * all;
      int b = 0;
      double m = 0.0;
      for (;; ++b) {
        m = 0.0;
        for (int q = 0; q < blocks; ++q) m += slot[q][b];
        if (cum + m >= target || b == kBins - 1) break;
        cum += m;
      }
      const float width = (edge - low) / kBins, over = width / 16;
      const float e1 = b == 0 ? edge : edge - b * width + over, e0 = b == kBins - 1 ? low : edge - (b + 1) * width - over;
      if (b > 0) high = e1;                                // else as before: what lies above the edge is known
      edge = e1;
      low = fmaxf(e0, low);
      enough = m <= 1200.0 * ex2((low - mx) * c);
      __syncthreads();
    }
  }
  // ---- in double: every warp's range of the row ----
  double kept = 0.0, all = 0.0;
  const int per = (share.end - share.first + kRowWarps - 1) / kRowWarps, begin = min(share.end, share.first + warp * per), stop = min(share.end, begin + per);
#pragma unroll 1
  for (int v = begin + lane; v < stop; v += 32) {
    float x[N];
    row.load(v, x);
#pragma unroll 4
    for (int j = 0; j < N; ++j) {
      const float z = clean(x[j]);
      if (!(z >= floor)) continue;
      const double w = exp_mass(f.x(z, mx), sh.powers);
      all += w;
      if (z >= high) {
        kept += w;
      } else if (z >= low) {
        const int at = atomicAdd(&sh.list.n, 1);
        if (at < kCandidates) sh.list.cand[at] = static_cast<uint64_t>(order_key(z)) << 32 | static_cast<uint32_t>(~(v * N - row.skew + j));
      }
    }
  }
  kept = warp_sum(kept);
  all = block_sum(all, sh.scan);
  if (lane == 0) st_block(in_block(&sh.mass[rank][warp], 0), kept);
  if (tid == 0) st_block(in_block(&sh.whole[rank], 0), all);
  __syncthreads();
  if (rank != 0) send_candidates(sh.list, &sh.base);
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  if (rank != 0) return true;

  // ---- the last kept token ----
  const int found = join_candidates(sh.list);
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
    if (found > 0) sort_front(sh.list.cand, found);
    if (above > 0.0 && above >= limit) return false;     // the border is above the range
    double done = above, inside = 0.0;
#pragma unroll 1
    for (int i0 = 0; i0 < found; i0 += kRowThreads) {
      const int i = i0 + tid;
      const double w = i < found ? exp_mass(f.x(key_logit(static_cast<uint32_t>(sh.list.cand[i] >> 32)), mx), sh.powers) : 0.0;
      double sum;
      const double before = done + block_scan(w, sum, sh.scan) - w;
      const bool in = i < found && (before < limit || (i == 0 && above == 0.0));
      n += __syncthreads_count(in);
      double mine;
      block_scan(in ? w : 0.0, mine, sh.scan);
      inside += mine;
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
    if (tid < blocks * kRowWarps) {
      double m = sh.mass[tid / kRowWarps][tid % kRowWarps];
      for (int i = 0; i < n; ++i)
        if (sh.place[i] == tid) m += exp_mass(f.x(key_logit(static_cast<uint32_t>(sh.list.cand[i] >> 32)), mx), sh.powers);
      sh.mass[tid / kRowWarps][tid % kRowWarps] = m;
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
  const RowShare there(row.nvec, range / kRowWarps, blocks);
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
          const double w = exp_mass(f.x(z, mx), sh.powers);
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
          const double w = exp_mass(f.x(z, mx), sh.powers);
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
                                                                     float* __restrict__ logp) {
  extern __shared__ float s_bins[];                        // [warps][kBins][32]
  __shared__ LongShared sh;
  const int rank = static_cast<int>(cluster_rank()), blocks = static_cast<int>(cluster_blocks());
  const long r = blockIdx.x / blocks;
  const float mx = top[r];
  if (mx != mx) return;
  const LogitRow<T> row(logits + r * row_stride, V);
  const RowFilter f(filters, r, V);
  if (blocks > 1) {                                        // shared memory may be written by the others once it is known to run
    cluster_arrive();
    cluster_wait();
  }
  if (!sample_long(row, f, mx, uniforms[r], rank, blocks, s_bins, sh, tokens + r, logp + r)) {
    __syncthreads();
    sample_by_border<1>(row, f, mx, uniforms[r], sh.border, sh.scan, tokens + r, logp + r);
  }
}

// Float sums of 2^x are off by so much of themselves at most: 2^-22 for 2^x, three steps of 2^-24 of the exponents, whose mean over the mass is log2 V < 24 at most, and
// sums of at most 300 terms a thread in float.
constexpr double kSumError = 2e-5;
constexpr int kNucleusGroups = 128;                        // groups whose maxima bound the candidates of a nucleus

// Over the sorted candidates: how many of them are kept; 0: it is not known (nucleus of a whole row whose mass `whole` is only known to kSumError, or whose last token is
// not among the `sure` first, beyond which others may come between).
NRL_DEVICE int kept_of(const uint64_t* x, int found, int sure, const RowFilter& f, float mx, double whole, SampleShared& sh, double& total) {
  const int tid = threadIdx.x;
  double done = 0.0;
  int n = 0, n1 = found;
  bool open = false;
  total = 0.0;
  if (f.top_k > 0 && f.top_k < n1) n1 = f.top_k;
  const bool nucleus = f.top_p < 1.0;
  double limit = 1e300, low = 0.0;
  for (int pass = nucleus && whole == 0.0 ? 0 : 1; pass < 2; ++pass) {        // the first for the mass that the nucleus is a share of
    done = 0.0;
    n = 0;
    if (pass == 1 && nucleus) {
      limit = f.top_p * (whole > 0.0 ? whole : total);
      low = whole > 0.0 ? limit * (1.0 - kSumError) : limit;
      if (whole > 0.0) limit *= 1.0 + kSumError;
    }
    total = 0.0;
#pragma unroll 1
    for (int i0 = 0; i0 < n1; i0 += kRowThreads) {
      const int i = i0 + tid;
      double w = i < n1 ? f.mass(key_logit(static_cast<uint32_t>(x[i] >> 32)), mx) : 0.0;
      if (w < f.min_p) w = 0.0;
      double all;
      const double before = done + block_scan(w, all, sh.scan) - w;
      bool in = i < n1 && w > 0.0;
      if (pass == 1 && nucleus && i > 0) {
        if (in && before >= low && before < limit && whole > 0.0) open = true;
        in = in && before < low;
      }
      n += __syncthreads_count(in);
      double kept;
      block_scan(in ? w : 0.0, kept, sh.scan);
      total += kept;
      done += all;
    }
  }
  open = __syncthreads_or(open);
  if (whole > 0.0 && (open || n >= sure)) return 0;         // the token behind the last kept has to be a candidate
  return n;
}

// from the n first candidates, which are sorted, by index
NRL_DEVICE void draw_of(uint64_t* x, int n, const RowFilter& f, float mx, double u, double total, SampleShared& sh, int* out_token, float* out_logp) {
  const int tid = threadIdx.x;
  __syncthreads();
  for (int i = tid; i < n; i += kRowThreads) x[i] = x[i] << 32 | x[i] >> 32;        // (~index, key)
  sort_front(x, n);                                         // (its first barrier is behind the swap)
  if (tid == 0) sh.token = 0x7fffffff;
  const double target = u * total;
  double done = 0.0;
  int last = 0;
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += kRowThreads) {
    const int i = i0 + tid;
    const double w = i < n ? f.mass(key_logit(static_cast<uint32_t>(x[i])), mx) : 0.0;
    double all;
    const double upto = done + block_scan(w, all, sh.scan);
    if (i < n && w > 0.0 && upto > target) atomicMin(&sh.token, i);
    done += all;
    last = min(n, i0 + kRowThreads) - 1;
  }
  __syncthreads();
  if (tid == 0) {
    const uint64_t y = x[min(sh.token, last)];
    *out_token = static_cast<int>(~static_cast<uint32_t>(y >> 32));
    *out_logp = static_cast<float>(f.x(key_logit(static_cast<uint32_t>(y)), mx) - log(total));
  }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads, 3) sample_filtered_kernel(const T* __restrict__ logits, long row_stride, int V,
                                                                         const float* __restrict__ uniforms, SampleFilters filters, int* __restrict__ tokens,
                                                                         float* __restrict__ logp, float* __restrict__ top) {
  extern __shared__ float s_chunk[];                       // [chunks][kRowThreads]
  __shared__ SampleShared sh;
  const int rank = static_cast<int>(cluster_rank()), blocks = static_cast<int>(cluster_blocks()), tid = threadIdx.x, lane = tid & 31;
  const long r = blockIdx.x / blocks;
  if (tid == 0) sh.list.n = sh.list.nhits = sh.list.sent = 0;
  if (blocks > 1) cluster_arrive();                        // the first block's memory may be written once it is known to run
  const LogitRow<T> row(logits + r * row_stride, V);
  const RowFilter f(filters, r, V);
  const RowShare share(row.nvec, rank, blocks);
  const bool few = (f.top_k > 0 && f.top_k <= kTopMax) || f.min_p > 0.0;        // what is kept is a matter of the candidates alone
  const bool nucleus = !few && f.top_p < 1.0 && f.top_k == 0;
  const float c = static_cast<float>(f.inv_temp * 1.4426950408889634);
  float best, m = 0.f, s = 0.f;
  if (nucleus)
    row_pass<true>(row, share, c, s_chunk, best, m, s, [](int, RawVec& a) { LogitRow<T>::drop_nan(a); });
  else
    row_pass<false>(row, share, c, s_chunk, best, m, s, [](int, const RawVec&) {});
  // a thread's chunks in one group up to 256 tokens, in up to four above
  const int want = few ? (f.top_k > 0 && f.top_k <= kTopMax ? f.top_k : 0) : kNucleusGroups, groups = want <= 256 ? 1 : want <= 512 ? 2 : 4;
  uint32_t bound = kKeyNone + 1;
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
  }
  const float mw = warp_max(nucleus ? m : best);
  const float sw = nucleus ? warp_sum(s * ex2((m - mw) * c)) : 0.f;
  if (blocks > 1) cluster_wait();
  if (lane == 0) {
    const uint32_t there = in_block(&sh.part[rank][tid >> 5], 0);
    st_block(there, mw);
    st_block(there + 4, sw);
  }
  if (tid == 0) st_block(in_block(&sh.part_bound[rank], 0), __uint_as_float(bound));
  if (rank != 0) send_candidates(sh.list, &sh.base);
  __syncwarp();
  if (blocks > 1) {
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
  } else {
    __syncthreads();
  }

  float mx = -INFINITY;
  for (int i = lane; i < blocks * kRowWarps; i += 32) mx = fmaxf(mx, sh.part[i / kRowWarps][i % kRowWarps].x);
  mx = warp_max(mx);
  const int found = join_candidates(sh.list);
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
    double whole = 0.0;
    int sure = found;
    if (nucleus) {
      uint32_t least = 0;
      for (int i = lane; i < blocks * kRowWarps; i += 32) {
        const float2 p = sh.part[i / kRowWarps][i % kRowWarps];
        whole += p.y * ex2((p.x - mx) * c);
      }
      whole = warp_sum(whole);
      for (int i = 0; i < blocks; ++i) least = max(least, sh.part_bound[i]);
      int n = 0;
      for (int i = tid; i < found; i += kRowThreads) n += static_cast<uint32_t>(sh.list.cand[i] >> 32) >= least ? 1 : 0;
      sure = static_cast<int>(block_sum(static_cast<double>(n), sh.border.red));
    }
    sort_front(sh.list.cand, found);
    double total;
    const int n = kept_of(sh.list.cand, found, sure, f, mx, whole, sh, total);
    if (n > 0) draw_of(sh.list.cand, n, f, mx, u, total, sh, tokens + r, logp + r);
    else open = mx;
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
  out[i] = 1.f - curand_uniform(&st);                      // (0, 1] -> [0, 1)
}

template <typename T>
cudaError_t launch_sample(const void* logits, long row_stride, int rows, int V, const float* uniforms, const SampleFilters& f, int* tokens, float* logp,
                          float* top, cudaStream_t s) {
  static PerDevice<bool> done, done_long;
  if (const cudaError_t e = allow_smem(done, sample_filtered_kernel<T>, kRowChunks * kRowThreads * 4); e != cudaSuccess) return e;
  if (const cudaError_t e = allow_smem(done_long, sample_long_kernel<T>, kBins * kRowThreads * 4); e != cudaSuccess) return e;
  const int blocks = row_blocks(rows, V, LogitRow<T>::N);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * blocks);
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = row_chunks(V, LogitRow<T>::N, blocks) * kRowThreads * 4;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const T* z = static_cast<const T*>(logits);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_filtered_kernel<T>, z, row_stride, V, uniforms, f, tokens, logp, top);
  if (e != cudaSuccess || top == nullptr) return e;
  cfg.dynamicSmemBytes = kBins * kRowThreads * 4;
  return cudaLaunchKernelEx(&cfg, sample_long_kernel<T>, z, row_stride, V, uniforms, f, static_cast<const float*>(top), tokens, logp);
}

}  // namespace nrl

using namespace nrl;

// Every row is settled by its candidates, or by its border in the first kernel: one top_k of 1 to kTopMax for all, or temperature 0.
extern "C" int nrl_sample_is_short(const SampleFilters* f, int V) {
  const bool greedy = f->temperature == nullptr && !(f->temperature_all > 0.0);
  return greedy || (f->top_k == nullptr && f->top_k_all > 0 && f->top_k_all <= kTopMax && f->top_k_all < V);
}

extern "C" cudaError_t nrl_sample_filtered(const void* logits, int is_bf16, long row_stride, int rows, int V, const float* uniforms, const SampleFilters* f,
                                           int* tokens, float* logp, float* top, cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  if (top == nullptr && !nrl_sample_is_short(f, V)) return cudaErrorInvalidValue;
  return is_bf16 ? launch_sample<__nv_bfloat16>(logits, row_stride, rows, V, uniforms, *f, tokens, logp, top, s)
                 : launch_sample<float>(logits, row_stride, rows, V, uniforms, *f, tokens, logp, top, s);
}

extern "C" cudaError_t nrl_row_uniforms(unsigned long long seed, unsigned long long step, const int* row_ids, const int* row_steps, int rows, float* out,
                                        cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  row_uniforms_kernel<<<(rows + 127) / 128, 128, 0, s>>>(seed, step, row_ids, row_steps, rows, out);
  return cudaGetLastError();
}
