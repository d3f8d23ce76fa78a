// What the kernels over a paged cache share.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>

#include "paged.h"

namespace b2 {

inline bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

// Everything that another kernel of the stream may have written is read through L2: under a programmatic launch the L1 may
// hold an older line.
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&f)[8]) {
  const uint4 u = __ldcg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&f)[8]) {
  uint4 u;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = u;
}

// The sequence that row t belongs to and its first row (the whole warp asks, with one t); -1 behind the last sequence.
// Without cu_tokens every sequence has one row.
__device__ __forceinline__ int sequence_of(const int* cu_tokens, int B, int t, int* first) {
  *first = t;
  if (cu_tokens == nullptr) return t < B ? t : -1;
  const int lane = threadIdx.x & 31;
  int before = 0, start = 0;  // sequences that end at or before row t, and the end of the last of them
  for (int b0 = 0; b0 < B; b0 += 32) {
    const int end = b0 + lane < B ? __ldcg(cu_tokens + b0 + lane + 1) : 0x7fffffff;
    const unsigned done = __ballot_sync(0xffffffffu, end <= t);
    if (done != 0) start = __shfl_sync(0xffffffffu, end, 31 - __clz(done));
    before += __popc(done);
    if (done != 0xffffffffu) break;
  }
  if (before >= B) return -1;
  *first = before == 0 ? __ldcg(cu_tokens) : start;
  return t < *first ? -1 : before;
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
