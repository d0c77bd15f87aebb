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

template <typename T>
struct LogitRow {
  static constexpr int N = 16 / sizeof(T);             // elements of a 16-byte vector
  const T* p;
  int V, skew, nvec;                                   // vector v holds the elements v * N - skew ...; the row starts `skew` elements into the first
  NRL_DEVICE LogitRow(const T* row, int v) : p(row), V(v) {
    skew = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    nvec = (V + skew + N - 1) / N;
  }
  NRL_DEVICE static float value(T x);
  // elements outside the row are -infinity and are not read
  NRL_DEVICE void load(int v, float (&x)[N]) const {
    const int e0 = v * N - skew;
    if (e0 >= 0 && e0 + N <= V) {
      const uint4 a = ldg_nc_v4(p + e0);
      unpack(a, x);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = e0 + j >= 0 && e0 + j < V ? value(p[e0 + j]) : -INFINITY;
    }
  }
  NRL_DEVICE static void unpack(const uint4& a, float (&x)[N]);
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
NRL_DEVICE void LogitRow<float>::unpack(const uint4& a, float (&x)[4]) {
  x[0] = __uint_as_float(a.x); x[1] = __uint_as_float(a.y); x[2] = __uint_as_float(a.z); x[3] = __uint_as_float(a.w);
}
template <>
NRL_DEVICE void LogitRow<__nv_bfloat16>::unpack(const uint4& a, float (&x)[8]) {
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = __uint_as_float(w[j] << 16);
    x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
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

}  // namespace nrl
