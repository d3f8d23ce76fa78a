// What the two kernels of attention over a paged cache, and the one that joins their parts, share.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include "paged.h"
#include "paged_rows.cuh"

namespace b2 {

// 2^x, to 2^-22 of it; -inf gives 0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct FewRows {
  const __nv_bfloat16* q;
  long long q_stride;
  __nv_bfloat16* out;
  long long out_stride;
  PagedCache c;
  const int* cu_tokens;
  Mask mask;
  int rep;           // query heads per KV head
  int n_cta;
  int parts_only;    // whole sequences are left as parts too (slots 2 n_cta + sequence and KV head)
  float scale_log2;  // scale / ln 2
  float* part;       // [slot][16][D], not divided by the sum
  float2* stat;      // [slot][16] maximum (in powers of two) and sum
  int* status;
};

// Tensor maps of K and V: boxes of 64 elements of min(page, block) tokens of one head of one page.
bool paged_tensor_maps(const PagedCache& c, int block, CUtensorMap* k, CUtensorMap* v);

}  // namespace b2
