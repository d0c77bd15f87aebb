// Launch API of the kernels around many samples of one prompt and a cache of bounded size: decode attention behind a shared prefix and with scores
// (decode_flat.cu, decode_prefix.cuh), eviction (kv_evict.cu).  Pages have 16 tokens, heads 128 elements.
#pragma once
#include <cuda_runtime.h>

namespace nrl {

struct DecodeCall {
  const void* q;                          // [S, Hq, D] bf16, rows q_stride_s elements apart
  long q_stride_s;
  const void *k_cache, *v_cache;          // bf16 [blocks, Hkv, 16, D], or e4m3 and values transposed (attention_decode_fp8.cu) with
  const float *k_scale, *v_scale;         // their scales [blocks, Hkv, 16] (null: bf16)
  const int *block_tables, *context_lens; // [S, max_blocks], [S]
  void* out;                              // [S, Hq, D] bf16
  int S, Hq, Hkv, D, page, max_blocks;
  float scale;
};

}  // namespace nrl

extern "C" {
// bytes of `scratch` below, on 64, for one call at a time (scored: no groups)
size_t nrl_decode_scratch(const nrl::DecodeCall* c, int n_groups, int max_group, int num_sms);
// max_group: rows of a group at most; it bounds how many blocks the prefixes get, not what they do
cudaError_t nrl_paged_decode_shared(const nrl::DecodeCall* c, const int* cu_groups, const int* shared, int n_groups, int max_group, void* scratch, int num_sms,
                                    cudaStream_t s);
// scores_in, scores_out [S, Hkv, max_tokens], rows and heads their strides apart (they may be the same memory); raw: [S, Hkv, G, 16 max_blocks] floats of scratch
cudaError_t nrl_paged_decode_scored(const nrl::DecodeCall* c, const float* scores_in, long in_row, long in_head, float* scores_out, long out_row, long out_head,
                                    int max_tokens, float decay, float* raw, void* scratch, int num_sms, cudaStream_t s);

struct EvictCall {
  void *k_cache, *v_cache;                // as above, written in place
  float *k_scale, *v_scale;
  const int *block_tables, *context_lens; // [S, max_blocks], [S]
  const int* out_tables;                  // [S, out_blocks] (null: block_tables, in place)
  const float* scores;                    // [S, Hkv, max_tokens]
  long score_row, score_head;
  int* kept;                              // [S, Hkv, keep]
  float* kept_scores;                     // [S, Hkv, keep]
  int* new_lens;                          // [S]
  unsigned* bits;                         // [S, Hkv, ceil(max_tokens / 32)] of scratch: a bit a token that is kept
  uint4* told;                            // [S, Hkv, 32] of scratch: what the blocks of a row-head tell one another
  int S, Hkv, max_blocks, out_blocks, max_tokens, keep, sinks, recent;
};
cudaError_t nrl_kv_evict(const EvictCall* c, int num_sms, cudaStream_t s);
}
