// C launch API of the kernels over rows of logits (top_logits.cu, distill.cu, sample_filtered.cu).  Logits: bf16 or float [rows, V], elements of a row
// side by side, rows `row_stride` elements apart.
#pragma once
#include <cuda_runtime.h>

constexpr int kTopMax = 1024;             // entries of a row at most (k, teacher's entries)
constexpr int kDistillVocabMax = 1 << 20;

extern "C" {
// `scratch` below: so many bytes, on 16, for one call at a time
size_t nrl_top_scratch(int is_bf16, int rows, int V, int k);
size_t nrl_distill_scratch(int is_bf16, int rows, int V, int with_grad);
// logp, idx: [rows, k], k <= kTopMax
cudaError_t nrl_top_logprobs(const void* logits, int is_bf16, long row_stride, int rows, int V, int k, double inv_temp, float* logp, int* idx,
                             void* scratch, cudaStream_t s);
// token_loss [rows]; loss (null: not formed) [1] = sum of weights * token_loss; grad (null: none) [rows, V] of its own type; weights null: 1 / rows
cudaError_t nrl_distill_loss(const void* logits, int is_bf16, long row_stride, int rows, int V, const float* top_logp, const int* top_idx, int k,
                             const float* weights, double inv_temp, double beta, int tail, float* token_loss, float* loss, void* grad, int grad_bf16,
                             void* scratch, cudaStream_t s);
// loss[0] = sum of weights * token_loss (weights null: 1 / rows)
cudaError_t nrl_weighted_sum(const float* token_loss, const float* weights, int rows, float* loss, cudaStream_t s);
// x *= *g in place, or nothing where *g is 1
cudaError_t nrl_scale(void* x, int is_bf16, long n, const float* g, cudaStream_t s);
// a parameter's pointer (one value a row) or, where it is null, its value
struct SampleFilters {
  const float* temperature; const int* top_k; const float* top_p; const float* min_p;
  double temperature_all, top_p_all, min_p_all;
  int top_k_all;
};
size_t nrl_sample_scratch(int is_bf16, int rows, int V, const SampleFilters* f);
// top: [rows] of scratch; may be null where nrl_sample_is_short says so
cudaError_t nrl_sample_filtered(const void* logits, int is_bf16, long row_stride, int rows, int V, const float* uniforms, const SampleFilters* f,
                                int* tokens, float* logp, float* top, void* scratch, cudaStream_t s);
int nrl_sample_is_short(const SampleFilters* f, int V);
// uniforms[i] in [0, 1) of (seed, row_ids[i], step + row_steps[i])
cudaError_t nrl_row_uniforms(unsigned long long seed, unsigned long long step, const int* row_ids, const int* row_steps, int rows, float* out,
                             cudaStream_t s);
}
