// What the kernels over a paged cache share.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>

#include "paged.h"

namespace b2 {

inline bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

// (Everything that another kernel of the stream may have written is read through L2, __ldcg: under a programmatic launch the L1 may
// hold an older line.)

// The sequence that row t belongs to, its first row, its rows and its length (the whole warp asks, with one t); -1 behind the last
// sequence or in front of the first.  Without cu_tokens every sequence has one row.
__device__ __forceinline__ int sequence_of(const int* cu_tokens, const PagedCache& c, int t, int* first, int* n_new, int* len) {
  if (cu_tokens == nullptr) {
    *first = t;
    *n_new = 1;
    *len = t < c.B ? __ldcg(c.lens + t) : 0;
    return t < c.B ? t : -1;
  }
  const int lane = threadIdx.x & 31;
  for (int b0 = 0; b0 < c.B; b0 += 32) {
    int begin = 0, end = -1, n = 0;
    if (b0 + lane < c.B) {
      begin = __ldcg(cu_tokens + b0 + lane);
      end = __ldcg(cu_tokens + b0 + lane + 1);
      n = __ldcg(c.lens + b0 + lane);
    }
    const unsigned has = __ballot_sync(0xffffffffu, begin <= t && t < end);
    if (has != 0) {
      const int l = __ffs(has) - 1;
      *first = __shfl_sync(0xffffffffu, begin, l);
      *n_new = __shfl_sync(0xffffffffu, end, l) - *first;
      *len = __shfl_sync(0xffffffffu, n, l);
      return b0 + l;
    }
  }
  return -1;
}

// The page that holds token `col` * page of a table's sequence, -1 where there is none.
__device__ __forceinline__ int page_at(const PagedCache& c, const int* table, int width, int col) {
  if (col >= width) return -1;
  const int page = __ldcg(table + col);
  return page >= 0 && page < c.n_pages ? page : -1;
}

// sin and cos of position * f, the product and its reduction by whole turns in 64 bits.
__device__ __forceinline__ void rotation(int position, float f, float* sn, float* cs) {
  constexpr double kTurn = 6.283185307179586476925286766559;       // 2 pi to 64 bits,
  constexpr double kTurnRest = 2.4492935982947064e-16;             // and what is left of it
  const double a = (double)position * (double)f;
  const double n = rint(a * (1.0 / kTurn));
  sincosf((float)fma(-n, kTurnRest, fma(-n, kTurn, a)), sn, cs);
}

}  // namespace b2
