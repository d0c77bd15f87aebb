// Distillation from a teacher's top log-probabilities: the divergence between two distributions over a vocabulary of which the teacher's is known for K tokens.
//
// q = softmax(z / tau) is the student's.  Both are compared over K + 1 events: the teacher's tokens (p_k = exp(a_k), q_k) and one event for all others
// (r = 1 - sum p_k, s = sum of q off K).  With P, Q these K + 1 numbers and M = beta P + (1 - beta) Q the loss of a token is
//   beta = 0: KL(P | Q)     beta = 1: KL(Q | P)     between: beta KL(P | M) + (1 - beta) KL(Q | M)
// and with D_j = log(Q_j / P_j) (beta = 1) or (1 - beta) log(Q_j / M_j) its gradient is
//   dL/dz_v tau = q_v (D_event(v) - sum_j Q_j D_j)            (beta = 0: q_k - p_k for the teacher's tokens, q_v (1 - r / s) for the others)
// so that off K a row needs one factor.  Without the event for the others (tail = 0, beta = 0) the p_k are scaled to sum to 1, and q keeps the whole
// vocabulary: the factor is 1.
//
// A divergence is the small difference of large terms, so everything about the K + 1 events is in double.  s is summed over the tokens off K alone, which a
// bit map in shared memory knows: taken as 1 - sum q_k it would have no digits left where the student is sure.  r below 2^-24, which float32 log-probabilities
// cannot tell from 0, counts as 0, and as 2^-24 under a logarithm.
// An entry whose index is not a token (-1) is skipped; entries of one token add up.
#include "common.cuh"
#include "logit_rows.cuh"
#include "per_device.h"
#include "vocab_rows.h"

namespace nrl {

template <typename T, typename G>
__global__ void __launch_bounds__(kRowThreads) distill_kernel(const T* __restrict__ logits, long row_stride, int V, const float* __restrict__ top_logp,
                                                              const int* __restrict__ top_idx, int K, const float* __restrict__ weights, double inv_temp,
                                                              double beta, int tail, float* __restrict__ token_loss, G* __restrict__ grad) {
  extern __shared__ uint32_t s_map[];                      // a bit for every token: one of the teacher's
  __shared__ double red[kRowWarps];
  __shared__ float redf[kRowWarps];
  __shared__ int s_idx[kTopMax];                           // -1: not a token, or one that an earlier entry has
  __shared__ double s_p[kTopMax], s_q[kTopMax];
  const long r = blockIdx.x;
  const LogitRow<T> row(logits + r * row_stride, V);
  const double weight = weights ? static_cast<double>(weights[r]) : 1.0 / gridDim.x;
  G* out = grad ? grad + r * V : nullptr;
  if (weight == 0.0) {                                     // the row is not read
    if (threadIdx.x == 0) token_loss[r] = 0.f;
    if (out)
      for (int v = threadIdx.x; v < V; v += kRowThreads) out[v] = static_cast<G>(0.f);
    return;
  }
  for (int i = threadIdx.x; i < (V + 31) / 32; i += kRowThreads) s_map[i] = 0;
  for (int i = threadIdx.x; i < K; i += kRowThreads) {
    const int at = top_idx[r * K + i];
    s_idx[i] = at >= 0 && at < V ? at : -1;
  }
  __syncthreads();
  int twin[kTopMax / kRowThreads];
#pragma unroll
  for (int t = 0; t < kTopMax / kRowThreads; ++t) {
    const int i = threadIdx.x + t * kRowThreads;
    twin[t] = 0;
    if (i < K && s_idx[i] >= 0) {
      double p = 0.0;
      for (int j = 0; j < K; ++j)
        if (s_idx[j] == s_idx[i]) {
          p += exp(static_cast<double>(top_logp[r * K + j]));
          if (j < i) twin[t] = 1;
        }
      s_p[i] = p;
      atomicOr(&s_map[s_idx[i] >> 5], 1u << (s_idx[i] & 31));
    }
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < kTopMax / kRowThreads; ++t)
    if (twin[t]) s_idx[threadIdx.x + t * kRowThreads] = -1;

  float mx = -INFINITY;
  row.each([&](int, float z) { mx = fmaxf(mx, z); });
  mx = block_max(mx, redf);
  const float c = static_cast<float>(inv_temp * 1.4426950408889634);
  float rest = 0.f;
  row.each([&](int e, float z) {
    if (!(s_map[e >> 5] >> (e & 31) & 1)) rest += ex2((z - mx) * c);
  });
  double others = block_sum(static_cast<double>(rest), red);
  double top = 0.0, psum = 0.0;
  for (int i = threadIdx.x; i < K; i += kRowThreads)
    if (s_idx[i] >= 0) {
      const double q = exp((static_cast<double>(row.at(s_idx[i])) - mx) * inv_temp);
      s_q[i] = q;
      top += q;
      psum += s_p[i];
    }
  top = block_sum(top, red);
  psum = block_sum(psum, red);
  const double total = top + others, log_total = log(total), s = others / total;
  double rr = 1.0 - psum;
  if (!(rr > 5.9604644775390625e-8)) rr = 0.0;
  const double r_log = rr > 0.0 ? rr : 5.9604644775390625e-8;
  // losses, and D of every event
  double loss = 0.0, mean = 0.0;
  for (int i = threadIdx.x; i < K; i += kRowThreads) {
    if (s_idx[i] < 0) continue;
    const double log_q = (static_cast<double>(row.at(s_idx[i])) - mx) * inv_temp - log_total, q = s_q[i] / total;
    double p = s_p[i];
    if (!tail) p = psum > 0.0 ? p / psum : 0.0;
    if (beta == 0.0) {
      if (p > 0.0) loss += p * (log(p) - log_q);
      s_p[i] = q - p;                                      // the gradient's entry
    } else if (beta == 1.0) {
      const double d = q > 0.0 ? log_q - log(p) : 0.0;
      loss += q * d;
      mean += q * d;
      s_p[i] = d;
    } else {
      const double m = beta * p + (1.0 - beta) * q, d = q > 0.0 ? (1.0 - beta) * log(q / m) : 0.0;
      loss += (p > 0.0 ? beta * p * log(p / m) : 0.0) + q * d;
      mean += q * d;
      s_p[i] = d;
    }
    s_q[i] = q;
  }
  loss = block_sum(loss, red);
  mean = block_sum(mean, red);
  double off = 1.0;                                        // factor of q off K
  if (tail) {
    if (beta == 0.0) {
      if (rr > 0.0) loss += rr * (log(rr) - log(s));
      off = s > 0.0 ? 1.0 - rr / s : 0.0;
    } else if (beta == 1.0) {
      const double d = s > 0.0 ? log(s) - log(r_log) : 0.0;
      loss += s * d;
      mean += s * d;
      off = d - mean;
    } else {
      const double m = beta * rr + (1.0 - beta) * s, d = s > 0.0 ? (1.0 - beta) * log(s / m) : 0.0;
      loss += (rr > 0.0 ? beta * rr * log(rr / m) : 0.0) + s * d;
      mean += s * d;
      off = d - mean;
    }
  } else if (!(psum > 0.0)) {
    off = 0.0;                                             // no teacher
  }
  if (threadIdx.x == 0) token_loss[r] = static_cast<float>(loss);
  if (!out) return;
  const double g = weight * inv_temp;
  const float f = static_cast<float>(fmin(fmax(g * off / total, -3e38), 3e38));      // finite: 0 times it is 0
  row.each([&](int e, float z) {
    if (!(s_map[e >> 5] >> (e & 31) & 1)) out[e] = static_cast<G>(ex2((z - mx) * c) * f);
  });
  for (int i = threadIdx.x; i < K; i += kRowThreads) {
    if (s_idx[i] < 0) continue;
    const double u = beta == 0.0 ? (!tail && !(psum > 0.0) ? 0.0 : s_p[i]) : s_q[i] * (s_p[i] - mean);
    out[s_idx[i]] = static_cast<G>(static_cast<float>(g * u));
  }
}

// sum of weights * token_loss, in one order
__global__ void __launch_bounds__(kRowThreads) weighted_sum_kernel(const float* __restrict__ token_loss, const float* __restrict__ weights, int rows,
                                                                   float* __restrict__ loss) {
  __shared__ double red[kRowWarps];
  double t = 0.0;
  for (int i = threadIdx.x; i < rows; i += kRowThreads) {
    const double w = weights ? static_cast<double>(weights[i]) : 1.0 / rows;
    if (w != 0.0) t += w * token_loss[i];
  }
  t = block_sum(t, red);
  if (threadIdx.x == 0) loss[0] = static_cast<float>(t);
}

template <typename T>
__global__ void scale_kernel(T* __restrict__ x, long n, const float* __restrict__ g) {
  const float f = g[0];
  if (f == 1.f) return;
  for (long i = blockIdx.x * static_cast<long>(blockDim.x) + threadIdx.x; i < n; i += static_cast<long>(gridDim.x) * blockDim.x)
    x[i] = static_cast<T>(static_cast<float>(x[i]) * f);
}

template <typename T, typename G>
cudaError_t launch_distill(const void* logits, long row_stride, int rows, int V, const float* top_logp, const int* top_idx, int k, const float* weights,
                           double inv_temp, double beta, int tail, float* token_loss, void* grad, cudaStream_t s) {
  static PerDevice<bool> done;
  const int bytes = (V + 31) / 32 * 4;
  if (const cudaError_t e = allow_smem(done, distill_kernel<T, G>, kDistillVocabMax / 8); e != cudaSuccess) return e;
  distill_kernel<T, G><<<rows, kRowThreads, bytes, s>>>(static_cast<const T*>(logits), row_stride, V, top_logp, top_idx, k, weights, inv_temp, beta, tail,
                                                         token_loss, static_cast<G*>(grad));
  return cudaGetLastError();
}

}  // namespace nrl

using namespace nrl;

extern "C" cudaError_t nrl_distill_loss(const void* logits, int is_bf16, long row_stride, int rows, int V, const float* top_logp, const int* top_idx, int k,
                                        const float* weights, double inv_temp, double beta, int tail, float* token_loss, float* loss, void* grad,
                                        int grad_bf16, cudaStream_t s) {
  if (V > kDistillVocabMax || k > kTopMax || (is_bf16 && grad && !grad_bf16)) return cudaErrorInvalidValue;
  if (rows > 0) {
    const auto launch = is_bf16 ? launch_distill<__nv_bfloat16, __nv_bfloat16> : grad_bf16 ? launch_distill<float, __nv_bfloat16> : launch_distill<float, float>;
    const cudaError_t e = launch(logits, row_stride, rows, V, top_logp, top_idx, k, weights, inv_temp, beta, tail, token_loss, grad, s);
    if (e != cudaSuccess) return e;
  }
  return loss ? nrl_weighted_sum(token_loss, weights, rows, loss, s) : cudaSuccess;
}

extern "C" cudaError_t nrl_weighted_sum(const float* token_loss, const float* weights, int rows, float* loss, cudaStream_t s) {
  weighted_sum_kernel<<<1, kRowThreads, 0, s>>>(token_loss, weights, rows, loss);
  return cudaGetLastError();
}

extern "C" cudaError_t nrl_scale(void* x, int is_bf16, long n, const float* g, cudaStream_t s) {
  if (n == 0) return cudaSuccess;
  const long blocks = n / 512 + 1 < 1184 ? n / 512 + 1 : 1184;
  if (is_bf16)
    scale_kernel<<<static_cast<int>(blocks), 512, 0, s>>>(static_cast<__nv_bfloat16*>(x), n, g);
  else
    scale_kernel<<<static_cast<int>(blocks), 512, 0, s>>>(static_cast<float*>(x), n, g);
  return cudaGetLastError();
}
