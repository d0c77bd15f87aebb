// Distillation from a teacher's top log-probabilities: the divergence between two distributions over a vocabulary of which the teacher's is known for K tokens.
//
// q = softmax(z / tau) is the student's.  Both are compared over K + 1 events: the teacher's tokens (p_k = exp(a_k), q_k) and one event for all others
// (r = 1 - sum p_k, s = sum of q off K).  With P, Q these K + 1 numbers and M = beta P + (1 - beta) Q the loss of a token is
//   beta = 0: KL(P | Q)     beta = 1: KL(Q | P)     between: beta KL(P | M) + (1 - beta) KL(Q | M)
// and with D_j = log(Q_j / P_j) (beta = 1) or (1 - beta) log(Q_j / M_j) its gradient is
//   dL/dz_v tau = q_v (D_event(v) - sum_j Q_j D_j)            (beta = 0: W q_k - p_k for the teacher's tokens, q_v (W - r / s) for the others, W = sum p_k + r,
//                                                              which is 1 unless entries sum to more)
// so that off K a row needs one factor.  Without the event for the others (tail = 0, beta = 0) the p_k are scaled to sum to 1, and q keeps the whole
// vocabulary: the factor is 1.
//
// A divergence is the small difference of large terms, so everything about the K + 1 events is in double.  s is summed over the tokens off K alone, which a
// bit map in shared memory knows: taken as 1 - sum q_k it would have no digits left where the student is sure.  The sum is relative to the largest logit off K,
// m, since relative to the row's it would be 0 in float from 87 temperatures between the two on: s = S exp((m - max z) / tau) / total, of which the logarithm is
// taken in parts, and dL/dz_v tau = e_v (W exp((m - max z) / tau) / total - r / S) off K with e_v = exp((z_v - m) / tau).
// r below 2^-24, which float32 log-probabilities cannot tell from 0, counts as 0, and as 2^-24 under a logarithm.
// An entry whose index is not a token (-1) is skipped; entries of one token add up.
//
// Bytes bound it: logits read, gradients written; the second pass reads from L2 what the first has brought there, and forms the exponentials again, since a row of
// them would not fit beside two other rows.  2048 x 151 936 bf16, K = 64, forward and backward: 283 us, 4.4 TB/s, where a copy's rate would take 190; issue slots 67 %,
// special functions 57 %.  4011 rows of floats with gradients in bf16: 810-830 us, 4.5 TB/s, with beta 1 915.  Tried without gain: two blocks an SM, vectors fetched a step ahead in
// registers, the next row fetched into L2, rows that start one behind the other.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "logit_rows.cuh"
#include "per_device.h"
#include "vocab_rows.h"

namespace nrl {

// A row of gradients is written once and read by another kernel: it is the first to leave L2, where the logits wait for the second pass.
NRL_DEVICE void store_words(float* at, const uint32_t (&w)[8]) {
  asm volatile("st.global.L1::no_allocate.L2::evict_first.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
NRL_DEVICE void store_words(__nv_bfloat16* at, const uint32_t (&w)[8]) { store_words(reinterpret_cast<float*>(at), w); }
NRL_DEVICE void store_words(__nv_bfloat16* at, const uint32_t (&w)[4]) { __stcs(reinterpret_cast<uint4*>(at), make_uint4(w[0], w[1], w[2], w[3])); }
// N gradients in words, as elements e0 .. of a row: those inside it
template <typename G, int W>
NRL_DEVICE void store_grads(G* out, int e0, int V, const uint32_t (&w)[W]) {
  constexpr int N = W * 4 / sizeof(G);
  if (e0 >= 0 && e0 + N <= V && (reinterpret_cast<uintptr_t>(out + e0) & (4 * W - 1)) == 0) {
    store_words(out + e0, w);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (e0 + j >= 0 && e0 + j < V) {
        if constexpr (sizeof(G) == 4) out[e0 + j] = __uint_as_float(w[j]);
        else reinterpret_cast<unsigned short*>(out)[e0 + j] = static_cast<unsigned short>(w[j / 2] >> (16 * (j % 2)));
      }
  }
}

// Elements whose bits are set in a map of the vectors first .. end
template <int N>
struct SkipMapped {
  const uint32_t* map;
  int first, end;
  NRL_DEVICE unsigned marks(int v) const { return v < end ? reinterpret_cast<const std::conditional_t<N == 16, uint16_t, uint8_t>*>(map)[v - first] : 0; }
  NRL_DEVICE void operator()(unsigned bits, RawVec& a) const {
    if (bits == 0) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (N == 16) {
        if (bits >> (2 * j) & 1) a.w[j] = (a.w[j] & 0xffff0000u) | 0xff80u;
        if (bits >> (2 * j + 1) & 1) a.w[j] = (a.w[j] & 0xffffu) | 0xff800000u;
      } else {
        if (bits >> j & 1) a.w[j] = 0xff800000u;
      }
    }
  }
};

struct DistillShared {
  __align__(16) int idx[kTopMax];                          // -1: not a token
  float z[kTopMax], a[kTopMax];
  double p[kTopMax];                                       // of the token by all its entries; below 0: not a token, or an earlier entry has it
  double q[kTopMax];                                       // beta > 0: D of the token's event
  float2 part[kRowWarps];                                  // maximum and sum of every warp
  double red[2][kRowWarps];
  int twins;                                               // some token has several entries
  uint32_t top;                                            // key of the tokens' largest logit
};

NRL_DEVICE void block_sum_two(double& x, double& y, double (&red)[2][kRowWarps]) {
  x = warp_sum(x);
  y = warp_sum(y);
  __syncthreads();
  if (lane_id() == 0) {
    red[0][threadIdx.x >> 5] = x;
    red[1][threadIdx.x >> 5] = y;
  }
  __syncthreads();
  x = warp_sum(lane_id() < kRowWarps ? red[0][lane_id()] : 0.0);
  y = warp_sum(lane_id() < kRowWarps ? red[1][lane_id()] : 0.0);
}

// Vectors of a thread in flight in the first pass, where three blocks share an SM: us with 2 / 3, and with 4 and two blocks, of 2048 x 151 936 bf16 284 / 293-302 / 317, of 1500 x 50 021
// floats 154 / 157 / 172, of 2048 x 32 000 bf16 78 / 85 / 89.
constexpr int kDistillFlight = 2;

constexpr double kNoTail = 5.9604644775390625e-8;          // 2^-24
// What is left of 1 by K <= 1024 float32 log-probabilities that sum to 1: half a step of each, 2^-24 of sum p |log p| <= log 1024, and of the row's sum that they share
// 5e-7.  Where the student has no mass off K that a double holds -- all its tokens are listed, or teacher and student share a mask, by -infinity or by a number that is low
// enough -- that is nobody's, and no divergence, infinite or of the mask's size.
constexpr double kNobodys = 9.5367431640625e-7;            // 2^-20

// Blocks of a cluster share a row.  Beside the two passes, what a row costs is latency -- entries, barriers, double-precision logarithms -- so that is kept off
// the way from one pass to the other: with beta = 0 every warp finds the factor for itself behind the barrier, and the loss is left for the end.
template <typename T, typename G>
__global__ void __launch_bounds__(kRowThreads, 3) distill_kernel(const T* __restrict__ logits, long row_stride, int V, const float* __restrict__ top_logp,
                                                                 const int* __restrict__ top_idx, int K, const float* __restrict__ weights, double inv_temp,
                                                                 double beta, int tail, float* __restrict__ token_loss, G* __restrict__ grad, float2* parts) {
  constexpr int N = LogitRow<T>::N, W = N * sizeof(G) / 4;
  extern __shared__ __align__(16) uint32_t s_map[];        // a bit for every element of the share's vectors: one of the teacher's tokens
  __shared__ DistillShared sh;
  const int rank = static_cast<int>(cluster_rank()), blocks = static_cast<int>(cluster_blocks()), tid = threadIdx.x, lane = tid & 31;
  const long r = blockIdx.x / blocks, rows = gridDim.x / blocks;
  const LogitRow<T> row(logits + r * row_stride, V);
  const RowShare share(row.nvec, rank, blocks, kDistillFlight);
  // the row's own numbers on their way together
  static_assert(kTopMax == 2 * kRowThreads, "two entries a thread at most");
  int at[2];
  float a_mine[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int i = tid + t * kRowThreads;
    at[t] = i < K ? top_idx[r * K + i] : -1;
    a_mine[t] = i < K ? top_logp[r * K + i] : 0.f;
  }
  const float weight = weights ? weights[r] : 1.f;
  const int map_words = ((share.end - share.first) * N / 32 + 4) / 4 * 4;
  for (int i = tid * 4; i < map_words; i += kRowThreads * 4) *reinterpret_cast<uint4*>(s_map + i) = make_uint4(0, 0, 0, 0);
  G* out = grad ? grad + r * V : nullptr;
  if (weight == 0.f) {                                     // the row is not read
    if (tid == 0 && rank == 0) token_loss[r] = 0.f;
    const uint32_t none[W] = {};
    if (out)
      for (int v = share.first + tid; v < share.end; v += kRowThreads) store_grads(out, v * N - row.skew, V, none);
    return;
  }
  // ---- the teacher's entries, and where they lie in the share ----
  if (tid == 0) {
    sh.twins = 0;
    sh.top = kKeyNone;
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int i = tid + t * kRowThreads;
    if (i >= (K + 3) / 4 * 4) continue;
    if (at[t] < 0 || at[t] >= V) at[t] = -1;
    const int bit = at[t] + row.skew - share.first * N;
    sh.idx[i] = at[t];
    sh.a[i] = a_mine[t];
    if (at[t] >= 0 && bit >= 0 && bit < (share.end - share.first) * N) atomicOr(&s_map[bit >> 5], 1u << (bit & 31));
  }
  __syncthreads();

  // ---- off the teacher's tokens: the largest logit, and the mass relative to it ----
  const float c = log2_scale(inv_temp);
  float best, m, mass;
  row_pass<kDistillFlight>(row, share, c, static_cast<float*>(nullptr), best, m, mass, SkipMapped<N>{s_map, share.first, share.end});
  put_state(m, mass, c, sh.part);
  __syncthreads();
  const float2 state = get_state(c, sh.part);
  if (blocks > 1) {
    if (tid == 0) parts[r * blocks + rank] = state;
    __syncwarp();
    cluster_arrive();
  }
  for (int i = tid; i < K; i += kRowThreads) {             // probabilities of the teacher's tokens, while the other blocks come
    const int at = sh.idx[i];
    const T z = row.p[max(at, 0)];
    double p = -1.0;
    if (at >= 0) {
      int same = 0;
      for (int j = 0; j < K; j += 4) {                     // entries behind the last are -1
        const int4 x = *reinterpret_cast<const int4*>(&sh.idx[j]);
        same += (x.x == at) + (x.y == at) + (x.z == at) + (x.w == at);
      }
      p = exp(static_cast<double>(sh.a[i]));
      if (same > 1) {
        sh.twins = 1;
        for (int j = 0; j < K; ++j)
          if (sh.idx[j] == at && j != i) p = j < i || p < 0.0 ? -1.0 : p + exp(static_cast<double>(sh.a[j]));
      }
    }
    sh.p[i] = p;
    sh.z[i] = LogitRow<T>::value(z);
    if (at >= 0) atomicMax(&sh.top, order_key(clean(sh.z[i])));
  }
  __syncwarp();
  if (blocks > 1) cluster_wait();
  __syncthreads();
  float high = state.x;                                    // the largest off K
  double sum = state.y, psum = 0.0, top = 0.0;
  if (blocks > 1) {
    const float2 p = lane < blocks ? __ldcg(&parts[r * blocks + lane]) : make_float2(-INFINITY, 0.f);
    join_states(p.x, p.y, c, high, sum);
  }
  const float mx = fmaxf(high, key_logit(sh.top));         // the largest of all
  for (int i = lane; i < K; i += 32)
    if (!(sh.p[i] < 0.0)) {
      psum += sh.p[i];
      top += ex2((sh.z[i] - mx) * c);
    }
  psum = warp_sum(psum);
  top = warp_sum(top);
  if (psum != psum) sum = NAN;                             // a token of the teacher's that is not a number makes the row none
  const auto below = [&] { return high == mx ? 0.0 : (static_cast<double>(high) - mx) * inv_temp; };        // (formed where it is wanted: registers)
  const double shrink = beta == 0.0 ? ex2((high - mx) * c) : exp(below());        // (float beside the float sum of `top`; the loss forms its own)

  // ---- the K + 1 events ----
  double rr = 1.0 - psum, mean = 0.0, total = top + sum * shrink, off;         // off: factor of e_v off K
  if (!(rr > kNoTail) || (rr <= kNobodys && (sum == 0.0 || below() < -745.0))) rr = 0.0;
  const bool teacher = tail || psum != 0.0;
  if (beta == 0.0) {
    off = !teacher ? 0.0 : tail ? (psum + rr) * shrink / total : shrink / total;
    if (tail && sum != 0.0) off -= rr / sum;
  } else {
    double loss = 0.0, none = 0.0;
    top = 0.0;
    for (int i = tid; i < K; i += kRowThreads)
      if (sh.p[i] >= 0.0) top += exp((static_cast<double>(sh.z[i]) - mx) * inv_temp);
    block_sum_two(top, none, sh.red);
    total = top + sum * shrink;
    const double log_total = log(total), s = sum * shrink / total;
    for (int i = tid; i < K; i += kRowThreads) {
      const double p = sh.p[i];
      if (p < 0.0) continue;
      const double log_q = (static_cast<double>(sh.z[i]) - mx) * inv_temp - log_total, q = exp(log_q);
      double d = 0.0;
      if (beta == 1.0) {
        if (q > 0.0) d = log_q - log(p);
      } else {
        const double mid = beta * p + (1.0 - beta) * q;    // (0 where p and q are next to it: they count nothing)
        if (q > 0.0 && mid > 0.0) d = (1.0 - beta) * log(q / mid);
        if (p > 0.0 && mid > 0.0) loss += beta * p * log(p / mid);
      }
      loss += q * d;
      mean += q * d;
      sh.q[i] = d;
    }
    block_sum_two(loss, mean, sh.red);
    double d = 0.0;
    if (beta == 1.0) {
      if (s > 0.0) d = log(sum) + below() - log_total - log(rr > 0.0 ? rr : kNoTail);
    } else {
      const double mid = beta * rr + (1.0 - beta) * s;
      if (s > 0.0 && mid > 0.0) d = (1.0 - beta) * log(s / mid);
      if (rr > 0.0) loss += beta * rr * log(rr / mid);
    }
    loss += s * d;
    mean += s * d;
    off = (d - mean) * shrink / total;
    if (tid == 0 && rank == 0) token_loss[r] = static_cast<float>(loss);
  }

  // ---- the gradient: off K one factor a row; the teacher's tokens are put right behind the others ----
  if (out) {
    const double g = (weights ? static_cast<double>(weight) : 1.0 / rows) * inv_temp;
    const double y = g * off;
    const float f = y == y ? static_cast<float>(fmin(fmax(y, -3e38), 3e38)) : NAN;      // 0 times a finite one is 0; what is not a number makes the row none
    const uint64_t c2 = pair_both(c), neg = pair_both(-high), f2 = pair_both(f);
    // backwards: what the first pass read last is the likeliest to be in L2
#pragma unroll 1
    for (int v = share.first + (share.end - share.first - 1) / kRowThreads * kRowThreads + tid; v >= share.first; v -= kRowThreads) {
      if (v >= share.end) continue;
      const RawVec a = row.template raw<true>(v);
      uint32_t w[W];
#pragma unroll
      for (int q = 0; q < N / 2; ++q) {
        const float2 e = pair_parts(pair_mul(pair_add(LogitRow<T>::pair(a, q), neg), c2));
        const float2 y = pair_parts(pair_mul(pair_of(__float_as_uint(ex2(e.x)), __float_as_uint(ex2(e.y))), f2));
        if constexpr (sizeof(G) == 4) {
          w[2 * q] = __float_as_uint(y.x);
          w[2 * q + 1] = __float_as_uint(y.y);
        } else {
          w[q] = pack_bf16x2(y.x, y.y);
        }
      }
      store_grads(out, v * N - row.skew, V, w);
    }
    __syncthreads();
    for (int i = tid; i < K; i += kRowThreads) {
      const double p = sh.p[i];
      const int bit = sh.idx[i] + row.skew - share.first * N;
      if (p < 0.0 || bit < 0 || bit >= (share.end - share.first) * N) continue;
      const double q = ex2((sh.z[i] - mx) * c) / total;
      const double u = !teacher ? 0.0 : beta == 0.0 ? (tail ? q * (psum + rr) - p : q - p / psum) : q == 0.0 ? 0.0 : q * (sh.q[i] - mean);
      out[sh.idx[i]] = static_cast<G>(static_cast<float>(g * u));
    }
  }

  // ---- beta = 0: sum p (log p - log q) over the events, log q = x - log total ----
  if (beta != 0.0 || rank != 0) return;
  double mass_top = 0.0, loss = 0.0;
  for (int i = tid; i < K; i += kRowThreads) {
    const double p = sh.p[i];
    if (p < 0.0) continue;
    const double x = (static_cast<double>(sh.z[i]) - mx) * inv_temp;
    mass_top += exp(x);
    const double a = sh.a[i];                              // log p, unless other entries have the token too
    if (p > 0.0) loss += p * ((sh.twins ? log(p) : a) - x);
  }
  block_sum_two(mass_top, loss, sh.red);
  if (tid < 32) {                                          // three logarithms in one
    total = mass_top + sum * exp(below());
    const double l = log(lane == 0 ? total : lane == 1 ? (tail ? rr : psum) : sum);
    const double log_total = __shfl_sync(0xffffffffu, l, 0), log_r = __shfl_sync(0xffffffffu, l, 1), log_o = __shfl_sync(0xffffffffu, l, 2) + below();
    if (tail) {
      loss += psum * log_total;
      if (rr > 0.0) loss += rr * (log_r - log_o + log_total);
    } else {
      loss = psum != 0.0 ? loss / psum - log_r + log_total : 0.0;
    }
    if (lane == 0) token_loss[r] = static_cast<float>(loss);
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

template <typename T>
int distill_blocks(int rows, int V, bool with_grad) {
  // The second pass should find its rows in L2, which has 126 MB; three blocks on each of 148 SMs hold 444 rows at a time, or half or a quarter of them with two or four
  // blocks a row.  us with 1 / 2 / 4 of 2048 x 151 936 floats 575 / 555 / 528, bf16 290 / 284 / 363 (DRAM reads 1.47 / 1.07 / 1.00 of the logits), of 1500 x 50 021 floats
  // 154 / 181 / 266, of 2048 x 32 000 bf16 76 / 113 / 191.
  int blocks = row_blocks(rows, V, LogitRow<T>::N);
  const long held = std::min(rows, 444) * static_cast<long>(V) * sizeof(T);
  if (with_grad) blocks = std::max(blocks, held > 200L << 20 ? 4 : held > 100L << 20 ? 2 : 1);
  return blocks;
}

template <typename T, typename G>
cudaError_t launch_distill(const void* logits, long row_stride, int rows, int V, const float* top_logp, const int* top_idx, int k, const float* weights,
                           double inv_temp, double beta, int tail, float* token_loss, void* grad, void* parts, cudaStream_t s) {
  static PerDevice<bool> done;
  constexpr int N = LogitRow<T>::N;
  const int blocks = distill_blocks<T>(rows, V, grad != nullptr);
  const int vecs = ((V + 2 * N - 2) / N + blocks - 1) / blocks;
  if (const cudaError_t e = allow_smem(done, distill_kernel<T, G>, kDistillVocabMax / 8 + 128); e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * blocks);
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = (vecs * N / 32 + 4) / 4 * 16;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, distill_kernel<T, G>, static_cast<const T*>(logits), row_stride, V, top_logp, top_idx, k, weights, inv_temp, beta, tail,
                            token_loss, static_cast<G*>(grad), static_cast<float2*>(parts));
}

}  // namespace nrl

using namespace nrl;

extern "C" size_t nrl_distill_scratch(int is_bf16, int rows, int V, int with_grad) {
  const int blocks = is_bf16 ? distill_blocks<__nv_bfloat16>(rows, V, with_grad) : distill_blocks<float>(rows, V, with_grad);
  return blocks > 1 ? static_cast<size_t>(rows) * blocks * sizeof(float2) : 0;
}

extern "C" cudaError_t nrl_distill_loss(const void* logits, int is_bf16, long row_stride, int rows, int V, const float* top_logp, const int* top_idx, int k,
                                        const float* weights, double inv_temp, double beta, int tail, float* token_loss, float* loss, void* grad,
                                        int grad_bf16, void* scratch, cudaStream_t s) {
  if (V > kDistillVocabMax || k > kTopMax || (is_bf16 && grad && !grad_bf16)) return cudaErrorInvalidValue;
  if (rows > 0) {
    const auto launch = is_bf16 ? launch_distill<__nv_bfloat16, __nv_bfloat16> : grad_bf16 ? launch_distill<float, __nv_bfloat16> : launch_distill<float, float>;
    const cudaError_t e = launch(logits, row_stride, rows, V, top_logp, top_idx, k, weights, inv_temp, beta, tail, token_loss, grad, scratch, s);
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
