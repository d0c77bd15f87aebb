// The k most probable tokens of every row of logits with their log-probabilities, as a teacher hands them to a student or a server to its user:
//   logp_j = z_j / tau - log sum_v exp(z_v / tau),   j = the k first tokens in (logit descending, index ascending)
// Tokens without mass (-infinity) are not listed: -1 and -infinity in their places.
#include "common.cuh"
#include "logit_rows.cuh"
#include "vocab_rows.h"

namespace nrl {

template <typename T>
__global__ void __launch_bounds__(kRowThreads) top_logprobs_kernel(const T* __restrict__ logits, long row_stride, int V, int k, double inv_temp,
                                                                   float* __restrict__ logp, int* __restrict__ idx) {
  extern __shared__ uint64_t s_top[];                    // (key, ~index): unsigned numbers in the order
  __shared__ BorderShared sh;
  __shared__ float red[kRowWarps];
  __shared__ int s_n;
  const LogitRow<T> row(logits + blockIdx.x * row_stride, V);
  float mx = -INFINITY;
  row.each([&](int, float z) { mx = fmaxf(mx, z); });
  mx = block_max(mx, red);
  double sum = 0.0, listed = 0.0;
  row.each([&](int, float z) {
    if (z != z) sum += z;
    if (order_key(clean(z)) > kKeyNone) {
      sum += z == mx ? 1.0 : exp((static_cast<double>(z) - mx) * inv_temp);
      listed += 1.0;
    }
  });
  sum = block_sum(sum, sh.red);
  listed = block_sum(listed, sh.red);
  const int n = min(k, static_cast<int>(listed));
  int size = 1;
  while (size < n) size *= 2;
  if (n > 0) {
    const Border b = find_border(row, kKeyNone + 1, order_key(mx), static_cast<double>(n), [](float) { return 1.0; }, sh);
    if (threadIdx.x == 0) s_n = 0;
    for (int i = threadIdx.x; i < size; i += kRowThreads) s_top[i] = 0;
    __syncthreads();
    row.each([&](int e, float z) {
      const uint32_t key = order_key(clean(z));
      if (b.has(key, e)) s_top[atomicAdd(&s_n, 1)] = static_cast<uint64_t>(key) << 32 | static_cast<uint32_t>(~e);
    });
    __syncthreads();
    for (int w = 2; w <= size; w *= 2)
      for (int d = w / 2; d > 0; d /= 2) {
        for (int i = threadIdx.x; i < size; i += kRowThreads) {
          const int j = i ^ d;
          if (j > i) {
            const uint64_t a = s_top[i], c = s_top[j];
            if ((a < c) == ((i & w) == 0)) { s_top[i] = c; s_top[j] = a; }
          }
        }
        __syncthreads();
      }
  }
  const double lz = log(sum);
  for (int i = threadIdx.x; i < k; i += kRowThreads) {
    const long o = static_cast<long>(blockIdx.x) * k + i;
    if (i < n) {
      const float z = key_logit(static_cast<uint32_t>(s_top[i] >> 32));
      logp[o] = static_cast<float>((z == mx ? 0.0 : (static_cast<double>(z) - mx) * inv_temp) - lz);
      idx[o] = static_cast<int>(~static_cast<uint32_t>(s_top[i]));
    } else {
      logp[o] = -INFINITY;
      idx[o] = -1;
    }
  }
}

}  // namespace nrl

using namespace nrl;

extern "C" cudaError_t nrl_top_logprobs(const void* logits, int is_bf16, long row_stride, int rows, int V, int k, double inv_temp, float* logp, int* idx,
                                        cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  int size = 1;
  while (size < k) size *= 2;
  if (is_bf16)
    top_logprobs_kernel<<<rows, kRowThreads, size * 8, s>>>(static_cast<const __nv_bfloat16*>(logits), row_stride, V, k, inv_temp, logp, idx);
  else
    top_logprobs_kernel<<<rows, kRowThreads, size * 8, s>>>(static_cast<const float*>(logits), row_stride, V, k, inv_temp, logp, idx);
  return cudaGetLastError();
}
