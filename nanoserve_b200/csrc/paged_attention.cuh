// What the two kernels of attention over a paged cache, and the one that joins their parts, share.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include <atomic>

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
  int T, max_tokens; // rows of the call, most of a sequence: what cu_tokens says beyond them is left out
  int rep_all;       // query heads per KV head
  int rep;           // of these in a tile: all, or sixteen of more (one row per sequence then)
  int groups, heads; // tiles per KV head of a sequence; KV heads times that
  int n_cta;
  int late_wait;     // the kernel in front writes nothing that this one reads, and has seen what is in front of it complete:
                     // it is waited for at the end
  int parts_only;    // whole sequences are left as parts too (slots 2 n_cta + sequence and KV head)
  float scale_log2;  // scale / ln 2
  float* part;       // [slot][16][D], not divided by the sum
  float2* stat;      // [slot][16] maximum (in powers of two) and sum
  int* status;
};

// Tiles of 128 rows (token, query head) of a sequence and KV head.
struct ManyRows {
  const __nv_bfloat16* q;
  long long q_stride;
  __nv_bfloat16* out;
  long long out_stride;
  PagedCache c;
  const int* cu_tokens;
  Mask mask;
  int rep, T, max_tokens;
  int two;           // two tiles to a CTA
  int slots;         // tiles of 128 rows per KV head, at least as many as there are (even, with two)
  int splits;        // CTAs that share a tile's keys
  float scale_log2;
  float* part;       // [KV head][slot][split][128][D], not divided by the sum; null: one split, to out
  float2* stat;      // beside it: maximum (in powers of two) and sum
  int* status;
};
int many_rows_launch(const ManyRows& p, cudaStream_t s);
int join_many_launch(const ManyRows& p, cudaStream_t s);

// Dynamic shared memory beyond 48 KB is allowed a kernel once per device.
struct SharedMemoryOnce {
  std::atomic<unsigned long long> done{0};
  template <typename K>
  int allow(K* kernel, size_t bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (e != cudaSuccess || (done.load(std::memory_order_relaxed) & bit)) return (int)e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return (int)e;
  }
};

template <typename... Args>
int launch_pdl(void (*kernel)(Args...), dim3 grid, int block, size_t smem, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Tensor maps of K and V: boxes of 64 elements of min(page, block) tokens of one head of one page.
bool paged_tensor_maps(const PagedCache& c, int block, CUtensorMap* k, CUtensorMap* v);

}  // namespace b2
