// One token per row of logits under temperature, min-p, top-k and top-p, from a given uniform number:
//   w_i = exp((z_i - max z) / T);  keep w_i >= min_p;  of those the top_k first in (logit descending, index ascending);  of those the shortest prefix whose
//   mass is at least top_p of theirs;  token = the first kept i, by index, with sum_{j <= i, kept} w_j > u * (mass of the kept)
// and its log-probability among the kept.  Each filter keeps a prefix of the order, so what is kept is one Border.  T <= 0: the first of the order.
// Masses are double: a token changes with the last bits of a sum, and the same numbers are to give the same token wherever they are added up.
#include <curand_kernel.h>

#include "common.cuh"
#include "logit_rows.cuh"
#include "vocab_rows.h"

namespace nrl {

template <typename T>
__global__ void __launch_bounds__(kRowThreads) sample_filtered_kernel(const T* __restrict__ logits, long row_stride, int V,
                                                                      const float* __restrict__ uniforms, SampleFilters f, int* __restrict__ tokens,
                                                                      float* __restrict__ logp) {
  __shared__ BorderShared sh;
  __shared__ float redf[kRowWarps];
  __shared__ double s_mass[kRowWarps];
  const int r = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const LogitRow<T> row(logits + r * row_stride, V);
  const double temp = f.temperature ? f.temperature[r] : f.temperature_all, top_p = f.top_p ? f.top_p[r] : f.top_p_all,
               min_p = f.min_p ? f.min_p[r] : f.min_p_all;
  const int top_k = f.top_k ? f.top_k[r] : f.top_k_all;
  float mx = -INFINITY;
  row.each([&](int, float z) { mx = fmaxf(mx, z); });
  mx = block_max(mx, redf);
  if (mx == -INFINITY) {                                   // nothing to draw from
    if (threadIdx.x == 0) { tokens[r] = -1; logp[r] = -INFINITY; }
    return;
  }
  const uint32_t top = order_key(mx);
  const bool greedy = !(temp > 0.0);
  const double inv_temp = greedy ? 1.0 : 1.0 / temp;
  auto mass = [&](float z) { return z == mx ? 1.0 : exp((static_cast<double>(z) - mx) * inv_temp); };
  auto one = [](float) { return 1.0; };
  uint32_t floor_key = mx == INFINITY ? top : kKeyNone + 1;
  if (min_p > 0.0 && !greedy) {                            // smallest key whose mass is min_p: every lane tries one of 32 keys of a range, seven times
    uint64_t lo = floor_key, hi = top;                     // in [lo, hi]; the largest logit is in whatever min_p says
    while (lo < hi) {
      const uint64_t step = (hi - lo + 31) / 32, k = lo + lane * step;
      const unsigned in = __ballot_sync(0xffffffffu, k >= hi || mass(key_logit(static_cast<uint32_t>(k))) >= min_p);
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
  if (greedy) {
    b = find_border(row, top, top, 1.0, one, sh);
  } else {
    if (top_k > 0 && total_of(one) > top_k) b = find_border(row, floor_key, top, static_cast<double>(top_k), one, sh);
    if (top_p < 1.0) b = find_border(row, b.key, top, top_p > 0.0 ? top_p * total_of(mass) : 1e-300, mass, sh);
  }
  // the kept mass of every warp's range, and the first range in which the drawn mass is passed
  double mine = 0.0;
  row.each([&](int e, float z) {
    if (b.has(order_key(clean(z)), e)) mine += mass(z);
  });
  mine = warp_sum(mine);
  if (lane == 0) s_mass[warp] = mine;
  __syncthreads();
  double total = 0.0;
  for (int w = 0; w < kRowWarps; ++w) total += s_mass[w];
  const double target = static_cast<double>(uniforms[r]) * total;
  int owner = -1;
  double before = 0.0, base = 0.0;
  bool found = false;
  for (int w = 0; w < kRowWarps && !found; ++w)
    if (s_mass[w] > 0.0) {
      owner = w;
      before = base;
      base += s_mass[w];
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
    tokens[r] = token;
    const float z = row.at(token);
    logp[r] = greedy ? 0.f : static_cast<float>((z == mx ? 0.0 : (static_cast<double>(z) - mx) * inv_temp) - log(total));
  }
}

__global__ void row_uniforms_kernel(unsigned long long seed, unsigned long long step, const int* __restrict__ row_ids, const int* __restrict__ row_steps,
                                    int rows, float* __restrict__ out) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= rows) return;
  curandStatePhilox4_32_10_t st;
  curand_init(seed, static_cast<unsigned long long>(row_ids ? row_ids[i] : i), step + (row_steps ? static_cast<unsigned long long>(row_steps[i]) : 0ull), &st);
  out[i] = 1.f - curand_uniform(&st);                      // (0, 1] -> [0, 1)
}

}  // namespace nrl

using namespace nrl;

extern "C" cudaError_t nrl_sample_filtered(const void* logits, int is_bf16, long row_stride, int rows, int V, const float* uniforms, const SampleFilters* f,
                                           int* tokens, float* logp, cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  if (is_bf16)
    sample_filtered_kernel<<<rows, kRowThreads, 0, s>>>(static_cast<const __nv_bfloat16*>(logits), row_stride, V, uniforms, *f, tokens, logp);
  else
    sample_filtered_kernel<<<rows, kRowThreads, 0, s>>>(static_cast<const float*>(logits), row_stride, V, uniforms, *f, tokens, logp);
  return cudaGetLastError();
}

extern "C" cudaError_t nrl_row_uniforms(unsigned long long seed, unsigned long long step, const int* row_ids, const int* row_steps, int rows, float* out,
                                        cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  row_uniforms_kernel<<<(rows + 127) / 128, 128, 0, s>>>(seed, step, row_ids, row_steps, rows, out);
  return cudaGetLastError();
}
