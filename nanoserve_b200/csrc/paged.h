// Host-side declarations of the operators of batched serving: the paged cache's append, attention over it, and sampling.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

namespace b2 {

// b2_paged_cache as the kernels take it (checked by paged_cache_check).
struct PagedCache {
  __nv_bfloat16* k;
  __nv_bfloat16* v;
  long long page_stride, head_stride, token_stride;  // elements
  const int* table;
  long long table_stride;  // entries
  const int* lens;
  int n_pages, page, page_shift, Hk, D, width, B;
};

struct Sampling {
  const void* logits;
  long long stride;  // elements between rows
  int fp32, rows, V;
  const float* u;
  const float* temperature;  // null: the value beside it for every row
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  long long* tokens;
};

// Whether rows of `width` values may lie `stride` elements apart; where there is one row, its stride says nothing.
inline bool rows_fit(long long stride, long long width, int rows) { return rows == 1 || (stride >= width && stride % 8 == 0); }

// sm_count below 1: minus the error that the device gave, returned once the arguments are found right.
int paged_append_launch(const void* qkv, long long qkv_stride, const void* bias, const void* inv_freq, void* q_out,
                        long long q_stride, const PagedCache& c, const int* cu_tokens, int T, int Hq, int sm_count,
                        cudaStream_t s);
int paged_attention_launch(const void* q, long long q_stride, const PagedCache& c, const int* cu_tokens, int T,
                           int max_tokens, int Hq, int window, int sinks, float scale, void* out, long long out_stride,
                           void* workspace, size_t workspace_bytes, int sm_count, cudaStream_t s);
size_t paged_attention_workspace(int T, int B, int max_tokens, int Hq, int Hk, int D, int sm_count);
int shared_prefix_launch(const void* q, long long q_stride, const PagedCache& c, const int* prefix_table,
                         int prefix_width, const int* prefix_len, int Hq, float scale, void* out, long long out_stride,
                         void* workspace, size_t workspace_bytes, int sm_count, cudaStream_t s);
size_t shared_prefix_workspace(int B, int Hq, int Hk, int D, int sm_count);
int sample_launch(const Sampling& p, int sm_count, cudaStream_t s);

// Whether a wait of the kernels for few rows, or for many, ran out on device `dev`: added to *word, or cleared.  The caller has
// synchronised.
int few_rows_timed_out(int dev, bool clear, int* word);
int many_rows_timed_out(int dev, bool clear, int* word);

}  // namespace b2
