// Rows of logits [rows, V] as a block reads them: bf16 or float, any row stride, any alignment of a row's first element.
//
// The order of a row's tokens is (logit descending, index ascending).  Every filter of a sampler and every "k largest" keeps a prefix of it, which two
// numbers name: the key of its last logit, and how many of the tokens that have this very logit are in, the lowest indices first (Border).
#pragma once
#include "common.cuh"

namespace nrl {

constexpr int kRowThreads = 512, kRowWarps = kRowThreads / 32;

// Unsigned numbers in the order of the logits; the zeros are one value, NaN counts as -infinity.
NRL_DEVICE uint32_t order_key(float z) {
  const uint32_t b = __float_as_uint(z + 0.f);
  return b ^ (static_cast<uint32_t>(static_cast<int>(b) >> 31) | 0x80000000u);
}
NRL_DEVICE float key_logit(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }
constexpr uint32_t kKeyNone = 0x007fffffu;             // -infinity: no mass

NRL_DEVICE float clean(float z) { return z == z ? z : -INFINITY; }

// 32 bytes of logits as they lie in memory, and arithmetic on them in pairs
struct RawVec { uint32_t w[8]; };
NRL_DEVICE uint64_t pair_of(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
NRL_DEVICE uint64_t pair_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
NRL_DEVICE uint64_t pair_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
NRL_DEVICE float2 pair_parts(uint64_t a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
NRL_DEVICE uint64_t pair_both(float x) { return pair_of(__float_as_uint(x), __float_as_uint(x)); }
NRL_DEVICE float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// logits to exponents of 2; finite, so that 0 times it is 0, and above 0, so that -infinity times it is none, at any temperature (from 1e45 up, where it would be 0, a
// difference of float32 logits has an exponent below 1e-6)
NRL_DEVICE float log2_scale(double inv_temp) { return static_cast<float>(fmin(fmax(inv_temp * 1.4426950408889634, 0x1p-149), 3e38)); }

template <typename T>
struct LogitRow {
  static constexpr int N = 32 / sizeof(T);             // elements of a 32-byte vector
  const T* p;
  int V, skew, nvec;                                   // vector v holds the elements v * N - skew ...; the row starts `skew` elements into the first
  NRL_DEVICE LogitRow(const T* row, int v) : p(row), V(v) {
    skew = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 31) / sizeof(T));
    nvec = (V + skew + N - 1) / N;
  }
  NRL_DEVICE static float value(T x);
  NRL_DEVICE static uint32_t none();                   // a word of -infinity
  NRL_DEVICE static void put(RawVec& a, int j, T x);   // element j of a vector
  // elements outside the row are -infinity and are not read; LAST: nobody reads them again
  template <bool LAST = false>
  NRL_DEVICE RawVec raw(int v) const {
    RawVec a;
    const int e0 = v * N - skew;
    if (e0 >= 0 && e0 + N <= V) {
      if constexpr (LAST)
        asm volatile("ld.global.nc.L1::no_allocate.L2::evict_first.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(a.w[0]), "=r"(a.w[1]), "=r"(a.w[2]), "=r"(a.w[3]), "=r"(a.w[4]), "=r"(a.w[5]), "=r"(a.w[6]), "=r"(a.w[7])
                     : "l"(p + e0));
      else
        asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(a.w[0]), "=r"(a.w[1]), "=r"(a.w[2]), "=r"(a.w[3]), "=r"(a.w[4]), "=r"(a.w[5]), "=r"(a.w[6]), "=r"(a.w[7])
                     : "l"(p + e0));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) a.w[j] = none();
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (e0 + j >= 0 && e0 + j < V) put(a, j, p[e0 + j]);
    }
    return a;
  }
  NRL_DEVICE static RawVec no_vec() {
    RawVec a;
#pragma unroll
    for (int j = 0; j < 8; ++j) a.w[j] = none();
    return a;
  }
  NRL_DEVICE static void unpack(const RawVec& a, float (&x)[N]);
  NRL_DEVICE static float largest(const RawVec& a);    // NaN left aside
  NRL_DEVICE static uint64_t pair(const RawVec& a, int i);        // elements 2 i and 2 i + 1
  NRL_DEVICE static void drop_nan(RawVec& a);          // NaN become -infinity
  NRL_DEVICE void load(int v, float (&x)[N]) const { unpack(raw(v), x); }
  NRL_DEVICE float at(int e) const { return value(p[e]); }
  // every element of this warp's range: the warps have consecutive ranges of the row, their lanes interleaved vectors; f(index, logit)
  template <class F>
  NRL_DEVICE void each(F&& f) const {
    const int per = (nvec + kRowWarps - 1) / kRowWarps, warp = threadIdx.x >> 5, end = min(nvec, (warp + 1) * per);
    for (int v = warp * per + static_cast<int>(lane_id()); v < end; v += 32) {
      float x[N];
      load(v, x);
      const int e0 = v * N - skew;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (e0 + j >= 0 && e0 + j < V) f(e0 + j, x[j]);
    }
  }
};
template <>
NRL_DEVICE float LogitRow<float>::value(float x) { return x; }
template <>
NRL_DEVICE float LogitRow<__nv_bfloat16>::value(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
NRL_DEVICE uint32_t LogitRow<float>::none() { return 0xff800000u; }
template <>
NRL_DEVICE uint32_t LogitRow<__nv_bfloat16>::none() { return 0xff80ff80u; }
template <>
NRL_DEVICE void LogitRow<float>::put(RawVec& a, int j, float x) { a.w[j] = __float_as_uint(x); }
template <>
NRL_DEVICE void LogitRow<__nv_bfloat16>::put(RawVec& a, int j, __nv_bfloat16 x) {
  const uint32_t b = __bfloat16_as_ushort(x);
  a.w[j / 2] = j % 2 ? (a.w[j / 2] & 0xffffu) | b << 16 : (a.w[j / 2] & 0xffff0000u) | b;
}
template <>
NRL_DEVICE uint64_t LogitRow<float>::pair(const RawVec& a, int i) { return pair_of(a.w[2 * i], a.w[2 * i + 1]); }
template <>
NRL_DEVICE uint64_t LogitRow<__nv_bfloat16>::pair(const RawVec& a, int i) { return pair_of(a.w[i] << 16, a.w[i] & 0xffff0000u); }
template <>
NRL_DEVICE void LogitRow<float>::unpack(const RawVec& a, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(a.w[j]);
}
template <>
NRL_DEVICE void LogitRow<__nv_bfloat16>::unpack(const RawVec& a, float (&x)[16]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[2 * j] = __uint_as_float(a.w[j] << 16);
    x[2 * j + 1] = __uint_as_float(a.w[j] & 0xffff0000u);
  }
}
template <>
NRL_DEVICE float LogitRow<float>::largest(const RawVec& a) {
  float m = __uint_as_float(a.w[0]);
#pragma unroll
  for (int j = 1; j < 7; j += 2) asm("max.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(__uint_as_float(a.w[j])), "f"(__uint_as_float(a.w[j + 1])));
  return fmaxf(m, __uint_as_float(a.w[7]));
}
template <>
NRL_DEVICE float LogitRow<__nv_bfloat16>::largest(const RawVec& a) {
  __nv_bfloat162 m = *reinterpret_cast<const __nv_bfloat162*>(&a.w[0]);
#pragma unroll
  for (int j = 1; j < 8; ++j) m = __hmax2(m, *reinterpret_cast<const __nv_bfloat162*>(&a.w[j]));
  const float2 f = __bfloat1622float2(m);
  return fmaxf(f.x, f.y);
}

template <>
NRL_DEVICE void LogitRow<float>::drop_nan(RawVec& a) {
#pragma unroll
  for (int j = 0; j < 8; ++j) a.w[j] = __float_as_uint(fmaxf(__uint_as_float(a.w[j]), -INFINITY));
}
template <>
NRL_DEVICE void LogitRow<__nv_bfloat16>::drop_nan(RawVec& a) {
  const __nv_bfloat162 lowest = __halves2bfloat162(__ushort_as_bfloat16(0xff80u), __ushort_as_bfloat16(0xff80u));
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a.w[j]), lowest);
    a.w[j] = *reinterpret_cast<const uint32_t*>(&m);
  }
}

// Reductions over the block, in one order; every thread gets the result.  `red`: kRowWarps entries that nobody else uses until the next barrier.
template <typename T>
NRL_DEVICE T block_sum(T v, T* red) {
  v = warp_sum(v);
  __syncthreads();
  if (lane_id() == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  T t = red[0];
#pragma unroll
  for (int w = 1; w < kRowWarps; ++w) t += red[w];
  return t;
}
NRL_DEVICE float block_max(float v, float* red) {
  v = warp_max(v);
  __syncthreads();
  if (lane_id() == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = red[0];
#pragma unroll
  for (int w = 1; w < kRowWarps; ++w) t = fmaxf(t, red[w]);
  return t;
}

struct Border {
  uint32_t key;      // of the last logit that is in
  int cut;           // tokens of this key are in up to and with this index
  NRL_DEVICE bool has(uint32_t k, int index) const { return k > key || (k == key && index <= cut); }
};

struct BorderShared {
  double red[kRowWarps];
  double bins[8][kRowWarps];
  int ties[kRowWarps];
  int cut;
};

// The shortest prefix of the order, among tokens of keys >= lo, whose measure reaches `target` > 0; measure(logit) >= 0 is one number for one logit.
// Sums are doubles in one order.  Eight ranges of keys a pass over the row (up to 11 passes), then the last key's tokens are counted.
template <typename T, class M>
NRL_DEVICE Border find_border(const LogitRow<T>& row, uint32_t lo, uint32_t top, double target, M&& measure, BorderShared& sh) {
  uint64_t first = lo, end = static_cast<uint64_t>(top) + 1;       // the border's key is in [first, end)
  double above = 0.0;                                              // measure of the keys from `end` on
  const int warp = threadIdx.x >> 5;
  while (end - first > 1) {
    int shift = 61 - __clzll(static_cast<long long>(end - first - 1));        // the range's highest bits: at most eight bins
    if (shift < 0) shift = 0;
    double part[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    row.each([&](int, float z) {
      const uint64_t k = order_key(clean(z));
      if (k < first || k >= end) return;
      const int b = static_cast<int>((k - first) >> shift);
      const double m = measure(z);
#pragma unroll
      for (int i = 0; i < 8; ++i) part[i] += i == b ? m : 0.0;
    });
#pragma unroll
    for (int i = 0; i < 8; ++i) part[i] = warp_sum(part[i]);
    __syncthreads();
    if (lane_id() == 0)
#pragma unroll
      for (int i = 0; i < 8; ++i) sh.bins[i][warp] = part[i];
    __syncthreads();
    int b = 7;
    for (;; --b) {
      double m = 0.0;
      for (int w = 0; w < kRowWarps; ++w) m += sh.bins[b][w];
      if (above + m >= target || b == 0) break;
      above += m;
    }
    const uint64_t width = 1ull << shift;
    first += b * width;
    if (first + width < end) end = first + width;
  }
  // as many of the key's tokens as it takes, by index
  const uint32_t key = static_cast<uint32_t>(first);
  const double each = measure(key_logit(key));
  double want = each > 0.0 ? ceil((target - above) / each) : 1.0;
  if (each > 0.0 && want > 1.0 && above + (want - 1.0) * each >= target) want -= 1.0;
  int left = want < 1.0 ? 1 : want > 2147483647.0 ? 2147483647 : static_cast<int>(want);
  int mine = 0;
  row.each([&](int, float z) { mine += order_key(clean(z)) == key ? 1 : 0; });
  mine = warp_sum(mine);
  __syncthreads();
  if (lane_id() == 0) sh.ties[warp] = mine;
  if (threadIdx.x == 0) sh.cut = 0x7fffffff;
  __syncthreads();
  int owner = 0;
  for (; owner < kRowWarps && sh.ties[owner] < left; ++owner) left -= sh.ties[owner];
  if (owner == warp) {                                             // the range that holds the last of them
    const int per = (row.nvec + kRowWarps - 1) / kRowWarps, stop = min(row.nvec, (warp + 1) * per);
    for (int v0 = warp * per; v0 < stop && left > 0; v0 += 32) {
      const int v = v0 + static_cast<int>(lane_id());
      float x[LogitRow<T>::N];
      const int e0 = v * LogitRow<T>::N - row.skew;
      int n = 0;
      if (v < stop) {
        row.load(v, x);
#pragma unroll
        for (int j = 0; j < LogitRow<T>::N; ++j) n += e0 + j >= 0 && e0 + j < row.V && order_key(clean(x[j])) == key ? 1 : 0;
      }
      int incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (static_cast<int>(lane_id()) >= o) incl += y;
      }
      const int before = incl - n;
      if (before < left && incl >= left) {
        int seen = before;
#pragma unroll
        for (int j = 0; j < LogitRow<T>::N; ++j)
          if (e0 + j >= 0 && e0 + j < row.V && order_key(clean(x[j])) == key && ++seen == left) sh.cut = e0 + j;
      }
      left -= __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  __syncthreads();
  return {key, sh.cut};
}

// ---- a row shared by the blocks of a cluster, and read once ---------------------------------------------------------------------------------------
NRL_DEVICE uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
NRL_DEVICE uint32_t cluster_blocks() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
NRL_DEVICE void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
NRL_DEVICE void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Blocks of a cluster tell each other what they found through memory of the call's own, written before a barrier at which all arrive and read behind it, past the L1.
constexpr int kRowClusterMax = 4;
// Vectors of a thread in flight where two blocks share an SM (that what a block does behind its pass hides the other's reads needs many bytes under way).  us with 4, with 3 and
// three blocks, with 2 and three: top 64 of 2048 x 151 936 bf16 136 / 141 / 160, of 148 rows 16.4 / 18.7 / 22.9, sampling with top-k 50 of 1024 rows 86 / 92 / 99, top 200 of 777
// x 50 021 floats 58.3 / 61.1 / 57.9; with 6 and two blocks 157 / 18.8 / 88 / 64.
constexpr int kFlight = 4;
constexpr int kRowChunks = 16;                         // of a thread's vectors, each with a maximum of its own

// The vectors of this block: thread t has first + t, first + t + kRowThreads, ..., in `chunks` chunks of `len`.
struct RowShare {
  int first, end, len, chunks;
  NRL_DEVICE RowShare(int nvec, int rank, int blocks, int flight) {       // flight: vectors of a thread in flight
    const int per = (nvec + blocks - 1) / blocks;
    first = min(nvec, rank * per);
    end = min(nvec, first + per);
    const int steps = (end - first + kRowThreads - 1) / kRowThreads;
    len = (steps + kRowChunks * flight - 1) / (kRowChunks * flight) * flight;
    chunks = len > 0 ? (steps + len - 1) / len : 0;
  }
};
// Blocks of a row's cluster (host).  A row of its own block is fastest where the rows fill the SMs; of few rows the cluster shares the reading, until its barrier and
// the way through memory cost more.  us with 1 / 2 / 4 blocks of rows of 151 936, top 20 of bf16: 1 row 12.0 / 11.1 / 9.8, 32 rows 12.9 / 11.9 / 10.4, 64 rows 13.1 /
// 12.0 / 14.0, 100 rows 13.2 / 16.6 / 20.5; sampling with top-k 50 of floats: 1 row 16.9 / 14.4 / 12.9, 64 rows 17.7 / 15.2 / 16.6, of bf16, where the reads are the
// smaller part, 10.5 / 11.3 / 11.7 and 10.9 / 12.2 / 15.5; without filters 1 row of bf16 51 / 34 / 26, 64 rows 52 / 37 / 42.  Of 32 000 floats with 1 / 2, top 20: 1 row
// 6.8 / 7.6, 64 rows 7.1 / 8.2.
inline int row_blocks(long rows, int V, int vec) {
  constexpr int kSms = 148;
  const long nvec = V / vec;
  int blocks = rows < kSms / 4 ? 4 : rows <= kSms / 2 ? 2 : 1;
  while (blocks > 1 && nvec < 2048L * blocks) blocks /= 2;
  return blocks;
}

// One pass over the block's share: thread-wise maximum `best`, sum s of 2^((z - m) c), m = best or the lowest float, and the maximum of every chunk.  The sum's reference moves with the
// maximum, once for the FLIGHT vectors of a step.  z - m is formed before the multiplication: m c would round at the size of the logits.
// Elements may be taken out of maxima and sum by making them -infinity: skip(skip.marks(v), a) of vector v, its marks looked up while the vector is on its way.  chunk_max may
// be null.  SUM false: the maxima alone, of all elements.
struct SkipNone {
  NRL_DEVICE unsigned marks(int) const { return 0; }
  NRL_DEVICE void operator()(unsigned, RawVec&) const {}
};
template <typename T>
struct SkipNan {
  NRL_DEVICE unsigned marks(int) const { return 0; }
  NRL_DEVICE void operator()(unsigned, RawVec& a) const { LogitRow<T>::drop_nan(a); }
};
template <int FLIGHT, bool SUM = true, typename T, class S>
NRL_DEVICE void row_pass(const LogitRow<T>& row, const RowShare& sh, float c, float* chunk_max, float& best, float& m, float& s, const S& skip) {
  m = -3.402823466e38f;                                // finite, so that -infinity is 0 in the sum
  s = 0.f;
  best = -INFINITY;
  const uint64_t c2 = pair_both(c);
  for (int i = 0; i < sh.chunks; ++i) {
    float cm = -INFINITY;
    const int v0 = sh.first + i * sh.len * kRowThreads + static_cast<int>(threadIdx.x);
    for (int u = 0; u < sh.len; u += FLIGHT) {
      RawVec a[FLIGHT];
#pragma unroll
      for (int j = 0; j < FLIGHT; ++j) {
        const int v = v0 + (u + j) * kRowThreads;
        a[j] = v < sh.end ? row.raw(v) : LogitRow<T>::no_vec();
      }
      if constexpr (SUM) {
        unsigned marks[FLIGHT];
#pragma unroll
        for (int j = 0; j < FLIGHT; ++j) marks[j] = skip.marks(v0 + (u + j) * kRowThreads);
#pragma unroll
        for (int j = 0; j < FLIGHT; ++j) skip(marks[j], a[j]);
      }
      float l = LogitRow<T>::largest(a[0]);
#pragma unroll
      for (int j = 1; j < FLIGHT; ++j) l = fmaxf(l, LogitRow<T>::largest(a[j]));
      cm = fmaxf(cm, l);
      if constexpr (!SUM) continue;
      const float mn = fmaxf(m, l);
      const uint64_t neg = pair_both(-mn);
      uint64_t sum = 0;
#pragma unroll
      for (int j = 0; j < FLIGHT; ++j)
#pragma unroll
        for (int q = 0; q < LogitRow<T>::N / 2; ++q) {
          const float2 e = pair_parts(pair_mul(pair_add(LogitRow<T>::pair(a[j], q), neg), c2));
          sum = pair_add(sum, pair_of(__float_as_uint(ex2(e.x)), __float_as_uint(ex2(e.y))));
        }
      const float2 p = pair_parts(sum);
      s = s * ex2((m - mn) * c) + (p.x + p.y);
      m = mn;
    }
    best = fmaxf(best, cm);
    if (chunk_max != nullptr) chunk_max[i * kRowThreads + threadIdx.x] = cm;
  }
}

// The bound of a block's candidates: a key that at least `want` of the block's groups' maxima reach (`keys`: this thread's, `groups` of them) and few more, by
// a histogram of 256 equal ranges of keys between the least and the largest, and one of the range that holds the want-th where it holds many;
// kKeyNone + 1 where fewer groups have any mass.  600 cycles; bit by bit with counts of one warp 4000.
struct BoundShared {
  int bins[2][256];
  uint32_t lo[kRowWarps], hi[kRowWarps];
};
constexpr int kGroupsMax = 4;
// of `bins`, the highest b that has, with those above, at least `want` counts; every lane gets b, what lies above it and what it holds
NRL_DEVICE int highest_bin(const int* bins, int want, int& above, int& holds) {
  const int lane = static_cast<int>(lane_id());
  int n[8], sum = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += n[i] = bins[lane * 8 + i];
  int incl = sum;                                      // of this lane's bins and those above
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_down_sync(0xffffffffu, incl, o);
    if (lane + o < 32) incl += y;
  }
  const unsigned reach = __ballot_sync(0xffffffffu, incl >= want);
  const int owner = reach ? 31 - __clz(reach) : 0;
  int b = lane * 8 + 7, h = n[7], a = incl - sum;       // a: above bin b
#pragma unroll
  for (int i = 6; i >= 0; --i)
    if (a + h < want) {
      a += h;
      b = lane * 8 + i;
      h = n[i];
    }
  above = __shfl_sync(0xffffffffu, a, owner);
  holds = __shfl_sync(0xffffffffu, h, owner);
  return __shfl_sync(0xffffffffu, b, owner);
}
NRL_DEVICE uint32_t group_bound(const uint32_t (&keys)[kGroupsMax], int groups, int want, BoundShared& sh) {
  const int tid = threadIdx.x, lane = tid & 31;
  uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll
  for (int g = 0; g < kGroupsMax; ++g)
    if (g < groups && keys[g] > kKeyNone) {
      lo = min(lo, keys[g]);
      hi = max(hi, keys[g]);
    }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0) {
    sh.lo[tid >> 5] = lo;
    sh.hi[tid >> 5] = hi;
  }
  sh.bins[tid >> 8][tid & 255] = 0;
  static_assert(kRowThreads == 512, "a thread a bin");
  __syncthreads();
  lo = __reduce_min_sync(0xffffffffu, sh.lo[lane % kRowWarps]);
  hi = __reduce_max_sync(0xffffffffu, sh.hi[lane % kRowWarps]);
  if (hi == 0) return kKeyNone + 1;
  int bits = 32 - __clz(hi - lo);                      // keys differ from lo in so many bits at most
#pragma unroll 1
  for (int level = 0;; ++level) {
    const int shift = bits > 8 ? bits - 8 : 0;
#pragma unroll
    for (int g = 0; g < kGroupsMax; ++g)
      if (g < groups && keys[g] > kKeyNone && keys[g] >= lo && (bits == 32 || (keys[g] - lo) >> bits == 0)) atomicAdd(&sh.bins[level][(keys[g] - lo) >> shift], 1);
    __syncthreads();
    int above, holds;
    const int b = highest_bin(sh.bins[level], want, above, holds);
    if (above + holds < want) return kKeyNone + 1;
    lo += static_cast<uint32_t>(b) << shift;
    if (level == 1 || shift == 0 || holds <= 8 + want / 4) return lo;
    want -= above;
    bits = shift;
  }
}

// What a block has gathered of its share.
constexpr int kCandidates = 2048;
struct SortCounts {
  int start[kRowThreads + 1], next[kRowThreads];           // of 512 buckets
  uint32_t lo[kRowWarps], hi[kRowWarps];
  int sums[kRowWarps];
};
struct RowList {
  __align__(16) uint64_t cand[kCandidates];            // (key, ~index): unsigned numbers in the order
  union {
    unsigned short hits[kCandidates];
    SortCounts counts;                                 // (when the hits are not needed any more)
  };
  int n, nhits;
};
// x[j], out of registers
template <int N>
NRL_DEVICE float pick(const float (&x)[N], int j) {
  float z = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) z = i == j ? x[i] : z;
  return z;
}
// Into `list` all elements of the share whose keys reach `bound`: the chunks that have any (by their maxima) are read again, a vector a thread.  list.n and
// list.nhits are 0 before; above kCandidates they say that there is more than what the list holds.
template <typename T>
NRL_DEVICE void gather_candidates(const LogitRow<T>& row, const RowShare& share, const float* chunk_max, uint32_t bound, RowList& list) {
  const int tid = threadIdx.x, lane = tid & 31;
  unsigned mine = 0;
#pragma unroll 4
  for (int i = 0; i < share.chunks; ++i) mine |= (order_key(chunk_max[i * kRowThreads + tid]) >= bound ? 1u : 0u) << i;
  if (__any_sync(0xffffffffu, mine != 0)) {
    int incl = __popc(mine), base = 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) base = atomicAdd(&list.nhits, incl);
    base = __shfl_sync(0xffffffffu, base, 31) + incl - __popc(mine);
    for (; mine != 0; mine &= mine - 1, ++base)
      if (base < kCandidates) list.hits[base] = static_cast<unsigned short>((__ffs(mine) - 1) * kRowThreads + tid);
  }
  __syncthreads();
  const int vecs = min(list.nhits, kCandidates) * share.len;
  for (int i = tid; i < vecs; i += kRowThreads) {
    const int hit = list.hits[i / share.len], v = share.first + (hit / kRowThreads * share.len + i % share.len) * kRowThreads + hit % kRowThreads;
    if (v >= share.end) continue;
    const RawVec a = row.raw(v);
    if (order_key(LogitRow<T>::largest(a)) < bound) continue;
    float x[LogitRow<T>::N];
    LogitRow<T>::unpack(a, x);
    unsigned in = 0;
#pragma unroll
    for (int j = 0; j < LogitRow<T>::N; ++j) in |= (order_key(clean(x[j])) >= bound ? 1u : 0u) << j;
    for (int at = atomicAdd(&list.n, __popc(in)); in != 0 && at < kCandidates; in &= in - 1, ++at) {
      const int e = v * LogitRow<T>::N - row.skew + __ffs(in) - 1;
      list.cand[at] = static_cast<uint64_t>(order_key(pick(x, __ffs(in) - 1))) << 32 | static_cast<uint32_t>(~e);
    }
  }
  __syncthreads();
}

// A row's memory where several blocks share it; behind it the candidates of all blocks but the first, kCandidates each.
struct RowMail {
  uint4 part[kRowClusterMax];                          // a block's largest logit, its sum of 2^((z - m) c), how many candidates it brings, and their bound
  double whole[kRowClusterMax], mass[kRowClusterMax][kRowWarps];
  float4 edges;
  float bins[kRowClusterMax][36];
  NRL_DEVICE uint64_t* list(int rank) { return reinterpret_cast<uint64_t*>(this + 1) + (rank - 1) * kCandidates; }
};
static_assert(sizeof(RowMail) % 16 == 0, "lists on 16 bytes");
inline size_t row_mail_bytes(int blocks) { return blocks > 1 ? sizeof(RowMail) + static_cast<size_t>(blocks - 1) * kCandidates * 8 : 0; }

// In front of the barrier: what this block has, and its list for the first.
NRL_DEVICE void send_candidates(const RowList& list, int rank, float2 state, uint32_t bound, RowMail& mail) {
  const int n = list.nhits > kCandidates || list.n > kCandidates ? kCandidates + 1 : list.n;
  if (threadIdx.x == 0) mail.part[rank] = make_uint4(__float_as_uint(state.x), __float_as_uint(state.y), n, bound);
  if (rank == 0) return;
  uint64_t* to = mail.list(rank);
  for (int i = threadIdx.x; i < min(n, kCandidates); i += kRowThreads) to[i] = list.cand[i];
}
// Behind it, the first block: part[q] in lane q of every warp, all lists in its own; returns how many candidates there are, above kCandidates where they do not fit.
NRL_DEVICE int join_candidates(RowList& list, int blocks, RowMail* mail, uint4& part) {
  part = static_cast<int>(lane_id()) < blocks ? __ldcg(&mail->part[lane_id()]) : make_uint4(0xff800000u, 0, 0, 0);
  int n[kRowClusterMax];                               // up to and with a block's
#pragma unroll
  for (int q = 0; q < kRowClusterMax; ++q) n[q] = (q > 0 ? n[q - 1] : 0) + __shfl_sync(0xffffffffu, static_cast<int>(part.z), q);
  const int all = n[kRowClusterMax - 1];
  if (all > kCandidates) return all;
  for (int i = n[0] + threadIdx.x; i < all; i += kRowThreads) {        // of all blocks at once
    int q = 1, first = n[0];
#pragma unroll
    for (int p = 1; p < kRowClusterMax - 1; ++p)
      if (i >= n[p]) {
        q = p + 1;
        first = n[p];
      }
    list.cand[i] = __ldcg(reinterpret_cast<unsigned long long*>(mail->list(q) + (i - first)));
  }
  __syncthreads();
  return all;
}
NRL_DEVICE int candidates_of(const RowList& list) { return list.nhits > kCandidates ? kCandidates + 1 : list.n; }
// the row's largest logit and its sum of 2^((z - m) c), from those of its blocks
NRL_DEVICE void join_states(float m, float s, float c, float& largest, double& sum) {
  largest = warp_max(m);
  sum = warp_sum(static_cast<double>(s > 0.f ? s * ex2((m - largest) * c) : s));        // (a NaN stays one)
}

// The block's largest logit and sum of 2^((z - m) c) from its threads': put_state, a barrier, get_state, which every thread may call.  `part`: kRowWarps entries.
NRL_DEVICE void put_state(float m, float s, float c, float2* part) {
  const float mw = warp_max(m), sw = warp_sum(s * ex2((m - mw) * c));
  if (lane_id() == 0) part[threadIdx.x >> 5] = make_float2(mw, sw);
}
NRL_DEVICE float2 get_state(float c, const float2* part) {
  const float2 p = part[lane_id() % kRowWarps];
  const float mb = warp_max(p.x);
  return make_float2(mb, warp_sum(lane_id() < kRowWarps ? p.y * ex2((p.x - mb) * c) : 0.f));
}

// The place of a number among the n <= kRowThreads different ones x[0 .. n) in descending order, by counting those above it: `mine` of a number that some threads count
// together, up to eight each (55 numbers 2100 -> 1000 cycles); the first of them gets the place, the others n.  x lies on 16 bytes; x[n] .. x[n + 63] are overwritten.
NRL_DEVICE int place_of(uint64_t* x, int n, uint64_t& mine) {
  const int tid = threadIdx.x, lg = n <= kRowThreads / 8 ? 3 : n <= kRowThreads / 4 ? 2 : n <= kRowThreads / 2 ? 1 : 0, part = tid & ((1 << lg) - 1);
  if (tid < 64) x[n + tid] = 0;
  __syncthreads();
  mine = x[min(tid >> lg, n)];
  int above = 0;
  const int end = (tid & ~31) >> lg < n ? n : 0;           // (the warps that have none leave the others the time)
#pragma unroll 1
  for (int j = 2 * part; j < end; j += 8 << lg) {
    ulonglong2 y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = *reinterpret_cast<const ulonglong2*>(x + j + (2 * i << lg));
#pragma unroll
    for (int i = 0; i < 4; ++i) above += (y[i].x > mine ? 1 : 0) + (y[i].y > mine ? 1 : 0);
  }
  for (int o = 1; o < 1 << lg; o <<= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
  __syncthreads();
  return tid >> lg < n && part == 0 ? above : n;
}
// x[0 .. n) in descending order, n <= kCandidates, all different (the 32 high bits need not be); the 64 entries behind them may be overwritten; y: room for as many.  Up to one a thread, places are
// counted: by exchanges 7000 cycles.  More go to 512 buckets by equal ranges of their high bits first, and are counted
// within theirs: 1358 numbers of five logits 25 000 cycles, by exchanges 30 000, and 6000 where few are of one logit.
NRL_DEVICE void sort_front(uint64_t* x, int n, uint64_t* y, SortCounts& sc) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (n <= kRowThreads) {
    uint64_t mine;
    const int place = place_of(x, n, mine);
    if (place < n) x[place] = mine;
    __syncthreads();
    return;
  }
  __syncthreads();
  uint32_t lo = 0xffffffffu, hi = 0;
  for (int i = tid; i < n; i += kRowThreads) {
    lo = min(lo, static_cast<uint32_t>(x[i] >> 32));
    hi = max(hi, static_cast<uint32_t>(x[i] >> 32));
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0) {
    sc.lo[warp] = lo;
    sc.hi[warp] = hi;
  }
  sc.start[tid] = 0;
  __syncthreads();
  lo = __reduce_min_sync(0xffffffffu, sc.lo[lane % kRowWarps]);
  hi = __reduce_max_sync(0xffffffffu, sc.hi[lane % kRowWarps]);
  const int shift = max(0, 23 - __clz(hi - lo));           // 512 ranges at most, the highest numbers first
  static_assert(kRowThreads == 512, "a bucket a thread");
  auto bucket = [&](uint64_t v) { return static_cast<int>((hi - static_cast<uint32_t>(v >> 32)) >> shift); };
  for (int i = tid; i < n; i += kRowThreads) atomicAdd(&sc.start[bucket(x[i])], 1);
  __syncthreads();
  const int count = sc.start[tid];
  int incl = count;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int z = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += z;
  }
  if (lane == 31) sc.sums[warp] = incl;
  __syncthreads();
  int before = incl - count;
  for (int w = 0; w < warp; ++w) before += sc.sums[w];
  sc.start[tid] = sc.next[tid] = before;
  if (tid == 0) sc.start[kRowThreads] = n;
  __syncthreads();
  for (int i = tid; i < n; i += kRowThreads) y[atomicAdd(&sc.next[bucket(x[i])], 1)] = x[i];
  __syncthreads();
  for (int i = tid; i < n; i += kRowThreads) {
    const uint64_t mine = y[i];
    const int b = bucket(mine), end = sc.start[b + 1];
    int place = sc.start[b];
#pragma unroll 4
    for (int j = sc.start[b]; j < end; ++j) place += y[j] > mine ? 1 : 0;
    x[place] = mine;
  }
  __syncthreads();
}

// Candidates in their order: f(place, candidate) for the first n of them, behind a barrier.
template <class F>
NRL_DEVICE void in_order(uint64_t* x, int found, int n, uint64_t* y, SortCounts& sc, F&& f) {
  const int tid = threadIdx.x;
  if (found <= kRowThreads) {
    uint64_t mine;
    const int before = place_of(x, found, mine);
    if (before < n) f(before, mine);
    return;
  }
  sort_front(x, found, y, sc);
  for (int i = tid; i < n; i += kRowThreads) f(i, x[i]);
}

}  // namespace nrl
