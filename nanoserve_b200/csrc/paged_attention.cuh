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
};
int many_rows_launch(const ManyRows& p, cudaStream_t s);
int join_many_launch(const ManyRows& p, cudaStream_t s);

// Devices on which kernels of a source file have been launched: a bit each.
using Devices = std::atomic<unsigned long long>;

// Dynamic shared memory beyond 48 KB is allowed a kernel once per device, which is noted in `ran`.
struct SharedMemoryOnce {
  Devices done{0};
  template <typename K>
  int allow(K* kernel, size_t bytes, Devices* ran = nullptr) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (e != cudaSuccess || (done.load(std::memory_order_relaxed) & bit)) return (int)e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    if (e == cudaSuccess && ran) ran->fetch_or(bit, std::memory_order_release);
    return (int)e;
  }
};

// A word `timed_out` of a source file's device image, which its kernels set where a wait ran out.  It is there from the first launch
// on, captured or not, whether or not the library's state of the device is.  Added to *word; with `clear`, set to 0.
template <typename Word>
int timed_out_word(const Word& timed_out, const Devices& ran, int dev, bool clear, int* word) {
  if (dev < 0 || dev >= 64 || !(ran.load(std::memory_order_acquire) >> dev & 1)) return 0;  // (never loads a kernel's image)
  int here = 0;
  const cudaError_t e = clear ? cudaMemcpyToSymbol(timed_out, &here, sizeof here) : cudaMemcpyFromSymbol(&here, timed_out, sizeof here);
  *word |= here;
  return (int)e;
}

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

// Parts of a row joined by a warp, in the order of their keys: a lane holds D / 32 columns of the row.  They are added up in units of
// the power of two that the heaviest weighs (its reference and its sum's exponent): a part is then no more than twice the average of
// its values, whatever its sum in its own units (the kernel for many rows lets those grow).
struct Part {
  const float2* stat;  // maximum (in powers of two) and sum
  const float* sums;   // D to a row
  long long at;        // row
};
template <int D>
struct Row {
  static constexpr int E = D / 32;
  float l = 0.f, o[E] = {};
  static __device__ __forceinline__ float weighs(float2 stat) {
    return stat.y == 0.f ? -INFINITY : stat.x + (float)((int)(__float_as_uint(stat.y) >> 23) - 127);
  }
  template <typename F>
  __device__ __forceinline__ void join(int n, int lane, F part) {
    float m = -INFINITY;
    float2 kept[2];  // of the first 64 parts
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      kept[c] = make_float2(-INFINITY, 0.f);
      if (32 * c + lane < n) {
        const Part x = part(32 * c + lane);
        kept[c] = __ldcg(x.stat + x.at);
      }
    }
    for (int i = 64 + lane; i < n; i += 32) {
      const Part x = part(i);
      m = fmaxf(m, weighs(__ldcg(x.stat + x.at)));
    }
    m = fmaxf(m, fmaxf(weighs(kept[0]), weighs(kept[1])));
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    for (int i0 = 0; i0 < n; i0 += 32) {
      float2 st = i0 == 0 ? kept[0] : kept[1];
      if (i0 >= 64) {
        st = make_float2(-INFINITY, 0.f);
        if (i0 + lane < n) {
          const Part x = part(i0 + lane);
          st = __ldcg(x.stat + x.at);
        }
      }
      const float f = st.y == 0.f ? 0.f : ex2(st.x - m);
      l += f * st.y;
      const int here = min(32, n - i0);
      for (int i1 = 0; i1 < here; i1 += 8) {  // eight on their way at a time
        float x[8][E];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const Part y = part(i0 + min(i1 + i, here - 1));
          const float* src = y.sums + y.at * D + lane * E;
          if constexpr (E == 4) {
            const float4 z = __ldcg(reinterpret_cast<const float4*>(src));
            x[i][0] = z.x, x[i][1] = z.y, x[i][2] = z.z, x[i][3] = z.w;
          } else {
            const float2 z = __ldcg(reinterpret_cast<const float2*>(src));
            x[i][0] = z.x, x[i][1] = z.y;
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float g = __shfl_sync(0xffffffffu, f, (i1 + i) & 31);
          if (i1 + i < here && g != 0.f) {
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += g * x[i][e];
          }
        }
      }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
  }
  __device__ __forceinline__ void store(__nv_bfloat16* to, int lane) const {  // a sum of 0: the row sees nothing
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int e = 0; e < E; e += 2)
      *reinterpret_cast<__nv_bfloat162*>(to + lane * E + e) =
          __floats2bfloat162_rn(inv == 0.f ? 0.f : o[e] * inv, inv == 0.f ? 0.f : o[e + 1] * inv);
  }
};

// Tensor maps of K and V: boxes of 64 elements of min(page, block) tokens of one head of one page.
bool paged_tensor_maps(const PagedCache& c, int block, CUtensorMap* k, CUtensorMap* v);

}  // namespace b2
