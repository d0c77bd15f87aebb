// Packed groups for attention_fwd_tc.cu and attention_bwd_tc.cu: of every sequence where it lies and where the prefix that it continues.  Rows that no
// sequence has are cleared.  The first sequence of a group is its prefix; rows of the others see it as a whole, and their own sequence up to themselves.  As the sequences of
// a group lie one behind the other, the rows that see a prefix's keys are those behind them up to the end of the group.
#include "attention_tc.cuh"
#include "kernels.h"
#include "launch.h"

namespace nrl {

__global__ void attn_group_table_kernel(const int* __restrict__ cu, const int* __restrict__ cu_groups, int4* __restrict__ table, int num, int groups,
                                        uint4* out, int total, int chunks) {
  pdl_wait();
  pdl_launch_dependents();
  const int s = blockIdx.x * blockDim.x + threadIdx.x;
  // rows behind the last sequence, of `chunks` 16-byte pieces: 0
  for (long i = static_cast<long>(cu[num]) * chunks + s; i < static_cast<long>(total) * chunks; i += static_cast<long>(gridDim.x) * blockDim.x)
    out[i] = make_uint4(0, 0, 0, 0);
  if (s >= num) return;
  int lo = 0, hi = groups;                             // the last group that begins at or in front of s
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu_groups[mid] <= s) lo = mid; else hi = mid;
  }
  const int start = cu[s], len = max(0, cu[s + 1] - start);
  int4 a = make_int4(start, len, 0, 0);
  int seen_by = len;
  if (groups > 0) {
    const int first = cu_groups[lo], end = min(cu_groups[lo + 1], num);
    if (first == s && s < end) seen_by = max(len, cu[end] - start);
    else if (first >= 0 && first < s && s < end) {
      a.z = cu[first];
      a.w = max(0, cu[first + 1] - cu[first]);
    }
  }
  table[2 * s] = a;
  table[2 * s + 1] = make_int4(seen_by, 0, 0, 0);
}

}  // namespace nrl

using namespace nrl;

// table: [num_seqs, 8]; out [total, Hq, 128] bf16: its rows behind the last sequence are cleared
extern "C" cudaError_t nrl_attn_group_table(const int* cu, const int* cu_groups, int* table, int num_seqs, int num_groups, void* out, int total, int Hq,
                                            cudaStream_t s) {
  if (total == 0) return cudaSuccess;
  launch_dependent(attn_group_table_kernel, num_seqs / 128 + 8, 128, 0, s, cu, cu_groups, reinterpret_cast<int4*>(table), num_seqs, num_groups, static_cast<uint4*>(out),
                   total, Hq * 16);
  return cudaGetLastError();
}
