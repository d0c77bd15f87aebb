// The k most probable tokens of every row of logits with their log-probabilities, as a teacher hands them to a student or a server to its user:
//   logp_j = z_j / tau - log sum_v exp(z_v / tau),   j = the k first tokens in (logit descending, index ascending)
// Tokens without mass (-infinity) are not listed: -1 and -infinity in their places.
//
// A row is read once.  Beside the sum every thread keeps the maxima of its chunks.  The k-th largest of the block's threads' maxima is a bound that at least k
// tokens reach, and few more do (k of G groups: about G ln(G / (G - k)) tokens): the chunks whose maximum reaches it are read again, and what reaches it there
// are the candidates.  Every block of a row's cluster sends its own to the first, which ranks them.  Rows with more candidates than fit (many ties, a sorted
// vocabulary, a k next to the number of the chunks) and rows with an infinite logit are looked through for the border itself, eight ranges of keys a pass.
//
// 2048 x 151 936 bf16, k = 64: 135 us, 4.6 TB/s, where a copy's rate would take 95.  What keeps it from that is bytes under way: two blocks of an SM read four vectors a
// thread at a time, and while one waits for its last warp, finds the bound, reads the candidates (two reads, one behind the other) and ranks them -- 13 000 cycles of
// a row -- the other reads alone.  One row: 9.8 us by four blocks.
#include "common.cuh"
#include "logit_rows.cuh"
#include "per_device.h"
#include "vocab_rows.h"

namespace nrl {

struct TopShared {
  BorderShared border;
  RowList list;
  float2 part[kRowWarps];                                // maximum and sum of every warp
  BoundShared bound;
  float log_sum;
};

// by the border, with no use of what the pass found but NaN (in `sum`)
template <typename T>
__device__ __noinline__ void top_by_border(const LogitRow<T>& row, int k, double inv_temp, float mx, TopShared& sh, double& sum, int& n) {
  double add = 0.0, listed = 0.0;
  row.each([&](int, float z) {
    if (z != z) add += z;
    if (order_key(clean(z)) > kKeyNone) {
      add += z == mx ? 1.0 : exp((static_cast<double>(z) - mx) * inv_temp);
      listed += 1.0;
    }
  });
  sum = block_sum(add, sh.border.red);
  n = min(k, static_cast<int>(block_sum(listed, sh.border.red)));
  const Border b = find_border(row, kKeyNone + 1, order_key(mx), static_cast<double>(n), [](float) { return 1.0; }, sh.border);
  if (threadIdx.x == 0) sh.list.n = 0;
  __syncthreads();
  row.each([&](int e, float z) {
    const uint32_t key = order_key(clean(z));
    if (b.has(key, e)) sh.list.cand[atomicAdd(&sh.list.n, 1)] = static_cast<uint64_t>(key) << 32 | static_cast<uint32_t>(~e);
  });
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads, 2) top_logprobs_kernel(const T* __restrict__ logits, long row_stride, int V, int k, double inv_temp,
                                                                      float* __restrict__ logp, int* __restrict__ idx, unsigned char* mails, size_t mail_bytes) {
  extern __shared__ __align__(16) float s_chunk[];       // [chunks][kRowThreads]; then what sorting takes
  static_assert(kCandidates * 8 <= kRowChunks * kRowThreads * 4, "in the place of the maxima");
  __shared__ TopShared sh;
  const int rank = static_cast<int>(cluster_rank()), blocks = static_cast<int>(cluster_blocks()), tid = threadIdx.x;
  const long r = blockIdx.x / blocks;
  RowMail* const mail = reinterpret_cast<RowMail*>(mails + r * mail_bytes);        // of several blocks
  if (tid == 0) sh.list.n = sh.list.nhits = 0;
  const LogitRow<T> row(logits + r * row_stride, V);
  const RowShare share(row.nvec, rank, blocks, kFlight);
  const float c = log2_scale(inv_temp);
  float best, m, s;
  row_pass<kFlight>(row, share, c, s_chunk, best, m, s, SkipNone());
  // a thread's chunks in one group up to k = 256, in up to four above
  const int groups = k <= 256 ? 1 : k <= 512 ? 2 : 4;
  uint32_t keys[kGroupsMax];
  keys[0] = order_key(best);
  if (groups > 1)
#pragma unroll
    for (int g = 0; g < kGroupsMax; ++g) {
      float x = -INFINITY;
      for (int i = g; i < share.chunks; i += groups) x = fmaxf(x, s_chunk[i * kRowThreads + tid]);
      keys[g] = order_key(x);
    }
  put_state(m, s, c, sh.part);                           // where an infinite logit makes this NaN, the row is looked through again
  const uint32_t bound = group_bound(keys, groups, k, sh.bound);
  gather_candidates(row, share, s_chunk, bound, sh.list);
  const float2 state = get_state(c, sh.part);
  float top = state.x;
  double sum = state.y;
  int found = candidates_of(sh.list);
  if (blocks > 1) {
    send_candidates(sh.list, rank, state, bound, *mail);
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
    uint4 part;
    found = join_candidates(sh.list, blocks, mail, part);
    join_states(__uint_as_float(part.x), __uint_as_float(part.y), c, top, sum);
  }
  int n = min(k, found);
  bool infinite = false;
  for (int i = tid; i < found && i < kCandidates; i += kRowThreads) infinite |= sh.list.cand[i] >> 32 == 0xff800000u;
  if (found > kCandidates || __syncthreads_or(infinite)) {
    top_by_border(row, k, inv_temp, top, sh, sum, n);
    found = n;
    if (tid == 0) sh.log_sum = static_cast<float>(log(sum));
    __syncthreads();
  } else if (tid == kRowThreads - 1) {                   // while the others rank
    sh.log_sum = logf(static_cast<float>(sum));          // half a step of it: 5e-7; the double one takes as long as the ranking
  }
  in_order(sh.list.cand, found, n, reinterpret_cast<uint64_t*>(s_chunk), sh.list.counts, [&](int place, uint64_t x) {
    const float z = key_logit(static_cast<uint32_t>(x >> 32));
    logp[r * k + place] = static_cast<float>((z == top ? 0.0 : (static_cast<double>(z) - top) * inv_temp) - sh.log_sum);
    idx[r * k + place] = static_cast<int>(~static_cast<uint32_t>(x));
  });
  for (int i = n + tid; i < k; i += kRowThreads) {
    logp[r * k + i] = -INFINITY;
    idx[r * k + i] = -1;
  }
}

template <typename T>
int top_blocks(int rows, int V, int k) {
  int blocks = row_blocks(rows, V, LogitRow<T>::N);
  while (blocks > 1 && blocks * k * 3 / 2 > kCandidates) blocks /= 2;        // every block of a row brings about k candidates
  return blocks;
}

template <typename T>
cudaError_t launch_top(const void* logits, long row_stride, int rows, int V, int k, double inv_temp, float* logp, int* idx, void* mails, cudaStream_t s) {
  const int blocks = top_blocks<T>(rows, V, k);
  static PerDevice<bool> done;
  if (const cudaError_t e = allow_smem(done, top_logprobs_kernel<T>, kRowChunks * kRowThreads * 4); e != cudaSuccess) return e;
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
  return cudaLaunchKernelEx(&cfg, top_logprobs_kernel<T>, static_cast<const T*>(logits), row_stride, V, k, inv_temp, logp, idx, static_cast<unsigned char*>(mails),
                            row_mail_bytes(blocks));
}

}  // namespace nrl

using namespace nrl;

extern "C" size_t nrl_top_scratch(int is_bf16, int rows, int V, int k) {
  return rows * row_mail_bytes(is_bf16 ? top_blocks<__nv_bfloat16>(rows, V, k) : top_blocks<float>(rows, V, k));
}

extern "C" cudaError_t nrl_top_logprobs(const void* logits, int is_bf16, long row_stride, int rows, int V, int k, double inv_temp, float* logp, int* idx,
                                        void* scratch, cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  return is_bf16 ? launch_top<__nv_bfloat16>(logits, row_stride, rows, V, k, inv_temp, logp, idx, scratch, s)
                 : launch_top<float>(logits, row_stride, rows, V, k, inv_temp, logp, idx, scratch, s);
}
