// b2_paged_kv_append: what stands between a batch's q|k|v projection and its attention over a paged cache, in one pass over
// the rows: bias, rotate-half rotary embedding of q and k, q to its own buffer, k and v into the pages of their sequences.
//
//   x = qkv + bias;  (a, b) = (x[i], x[i + D/2]) -> (a cos - b sin, b cos + a sin),  angle = position * inv_freq[i]
//
// in 32 bits with one rounding to bf16 at the store.  The angle is formed and reduced to [-pi, pi] in 64 bits: in 32 bits the
// product alone is off by 2^-24 of itself, 0.004 radians at position 65536.
#include "paged.h"
#include "paged.cuh"
#include "w4_internal.h"

namespace b2 {
namespace {

constexpr int kMaxHalf = 128;  // D / 2

// One CTA per row.  Bound by memory; one thread moves eight (i, i + D/2) pairs of a head.
__global__ void __launch_bounds__(256) paged_append_kernel(const __nv_bfloat16* qkv, long long qkv_stride,
                                                           const __nv_bfloat16* bias, const float* inv_freq,
                                                           __nv_bfloat16* q_out, long long q_stride, PagedCache c,
                                                           const int* cu_tokens, int Hq) {
  __shared__ float s_cos[kMaxHalf], s_sin[kMaxHalf];
  const int t = blockIdx.x, D = c.D, heads = Hq + 2 * c.Hk;
  int first;
  const int b = sequence_of(cu_tokens, c.B, t, &first);
  if (b < 0) return;
  const int n_new = cu_tokens ? __ldcg(cu_tokens + b + 1) - first : 1;
  const int pos = __ldcg(c.lens + b) - n_new + (t - first);
  if (pos < 0) return;  // the sequence has no place for this row
  for (int i = threadIdx.x; i < D / 2; i += blockDim.x) rotation(pos, __ldcg(inv_freq + i), &s_sin[i], &s_cos[i]);
  const int col = pos >> c.page_shift;
  const int page = col < c.width ? __ldcg(c.table + b * c.table_stride + col) : -1;
  const bool stored = page >= 0 && page < c.n_pages;
  const long long at = (long long)page * c.page_stride + (long long)(pos & (c.page - 1)) * c.token_stride;
  __syncthreads();
  const int per_head = D / 16;
  for (int u = threadIdx.x; u < heads * per_head; u += blockDim.x) {
    const int h = u / per_head, e0 = (u - h * per_head) * 8;
    if (h >= Hq && !stored) continue;
    const __nv_bfloat16* src = qkv + t * qkv_stride + (long long)h * D;
    float lo[8], hi[8], f[8];
    load8(src + e0, lo);
    load8(src + D / 2 + e0, hi);
    if (bias != nullptr) {
      load8(bias + h * D + e0, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) lo[e] += f[e];
      load8(bias + h * D + D / 2 + e0, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) hi[e] += f[e];
    }
    if (h < Hq + c.Hk) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = lo[e], bb = hi[e], cs = s_cos[e0 + e], sn = s_sin[e0 + e];
        lo[e] = a * cs - bb * sn;
        hi[e] = bb * cs + a * sn;
      }
    }
    __nv_bfloat16* dst = h < Hq          ? q_out + t * q_stride + (long long)h * D
                         : h < Hq + c.Hk ? c.k + at + (h - Hq) * c.head_stride
                                         : c.v + at + (h - Hq - c.Hk) * c.head_stride;
    store8(dst + e0, lo);
    store8(dst + D / 2 + e0, hi);
  }
}

}  // namespace

int paged_append_launch(const void* qkv, long long qkv_stride, const void* bias, const void* inv_freq, void* q_out,
                        long long q_stride, const PagedCache& c, const int* cu_tokens, int T, int Hq, cudaStream_t s) {
  const int heads = Hq + 2 * c.Hk;
  if (T < 1 || Hq < 1 || (!cu_tokens && T != c.B)) return kErrBadShape;
  if (qkv_stride < (long long)heads * c.D || qkv_stride % 8 || q_stride < (long long)Hq * c.D || q_stride % 8)
    return kErrBadShape;
  if (!qkv || !inv_freq || !q_out || misaligned(qkv, 16) || misaligned(bias, 16) || misaligned(q_out, 16) ||
      misaligned(inv_freq, 4) || misaligned(cu_tokens, 4))
    return kErrBadPointer;
  paged_append_kernel<<<T, 256, 0, s>>>(static_cast<const __nv_bfloat16*>(qkv), qkv_stride,
                                        static_cast<const __nv_bfloat16*>(bias), static_cast<const float*>(inv_freq),
                                        static_cast<__nv_bfloat16*>(q_out), q_stride, c, cu_tokens, Hq);
  return (int)cudaGetLastError();
}

}  // namespace b2
