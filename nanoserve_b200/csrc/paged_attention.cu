// Attention over a paged cache: b2_paged_attention (new tokens against their sequences, causal, sliding window, first tokens
// that stay visible) and b2_shared_prefix_attention (one token per sequence, all behind a common prefix).
//
//   o = sum_j e^{s_j - m} v_j / sum_j e^{s_j - m},   s_j = scale * q . k_j,   over the keys j that the row sees,
//
// in one pass over the keys with the running maximum m, sum and weighted rows in 32 bits.  A row that sees nothing is zero.
#include <cfloat>

#include "paged.h"
#include "paged.cuh"
#include "w4_internal.h"

namespace b2 {
namespace {

// One warp per (row, query head); lanes split the head dimension.
template <int D>
struct RowState {
  static constexpr int E = D / 32;
  float q[E], acc[E], m = -FLT_MAX, l = 0.f;
  __device__ __forceinline__ void key(const __nv_bfloat16* k, const __nv_bfloat16* v, int lane) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e)
      s += q[e] * __bfloat162float(__ushort_as_bfloat16(__ldcg(reinterpret_cast<const unsigned short*>(k) + lane * E + e)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float mn = fmaxf(m, s), corr = __expf(m - mn), p = __expf(s - mn);
    l = l * corr + p;
#pragma unroll
    for (int e = 0; e < E; ++e)
      acc[e] = acc[e] * corr +
               p * __bfloat162float(__ushort_as_bfloat16(__ldcg(reinterpret_cast<const unsigned short*>(v) + lane * E + e)));
    m = mn;
  }
  __device__ void keys(const PagedCache& c, const int* table, int width, int kh, int j0, int j1, int lane) {
    for (int j = j0; j < j1; ++j) {
      const int col = j >> c.page_shift;
      if (col >= width) return;
      const int page = __ldcg(table + col);
      if (page < 0 || page >= c.n_pages) continue;
      const long long at = page * c.page_stride + kh * c.head_stride + (long long)(j & (c.page - 1)) * c.token_stride;
      key(c.k + at, c.v + at, lane);
    }
  }
};

template <int D>
__global__ void __launch_bounds__(128) attention_kernel(const __nv_bfloat16* q, long long q_stride, PagedCache c,
                                                        const int* cu_tokens, int T, int Hq, int window, int sinks,
                                                        float scale, __nv_bfloat16* out, long long out_stride,
                                                        const int* prefix_table, int prefix_width, const int* prefix_len) {
  const int lane = threadIdx.x & 31;
  const long long row = blockIdx.x * 4LL + (threadIdx.x >> 5);
  if (row >= (long long)T * Hq) return;
  const int t = (int)(row / Hq), h = (int)(row - (long long)t * Hq), kh = h / (Hq / c.Hk);
  int first;
  const int b = sequence_of(cu_tokens, c.B, t, &first);
  if (b < 0) return;
  RowState<D> r;
  constexpr int E = RowState<D>::E;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    r.q[e] = scale * __bfloat162float(q[t * q_stride + h * D + lane * E + e]);
    r.acc[e] = 0.f;
  }
  if (prefix_table) r.keys(c, prefix_table, prefix_width, kh, 0, __ldcg(prefix_len), lane);
  const int n_new = cu_tokens ? __ldcg(cu_tokens + b + 1) - first : 1;
  const int len = __ldcg(c.lens + b), pos = len - n_new + (t - first);
  const int lo = window > 0 ? max(0, pos - window + 1) : 0;
  const int* table = c.table + b * c.table_stride;
  r.keys(c, table, c.width, kh, 0, min(min(sinks, lo), pos + 1), lane);
  r.keys(c, table, c.width, kh, lo, pos + 1, lane);
#pragma unroll
  for (int e = 0; e < E; ++e)
    out[t * out_stride + h * D + lane * E + e] = __float2bfloat16(r.l > 0.f ? r.acc[e] / r.l : 0.f);
}

int check_rows(const void* q, long long q_stride, const PagedCache& c, int T, int Hq, const void* out, long long out_stride) {
  if (T < 1 || Hq < 1 || Hq % c.Hk || (c.D != 64 && c.D != 128)) return kErrBadShape;
  if (q_stride < (long long)Hq * c.D || q_stride % 8 || out_stride < (long long)Hq * c.D || out_stride % 8) return kErrBadShape;
  if (!q || !out || misaligned(q, 16) || misaligned(out, 16)) return kErrBadPointer;
  return 0;
}

int launch(const void* q, long long q_stride, const PagedCache& c, const int* cu_tokens, int T, int Hq, int window, int sinks,
           float scale, void* out, long long out_stride, const int* prefix_table, int prefix_width, const int* prefix_len,
           cudaStream_t s) {
  const unsigned grid = (unsigned)(((long long)T * Hq + 3) / 4);
  (c.D == 64 ? attention_kernel<64> : attention_kernel<128>)<<<grid, 128, 0, s>>>(
      static_cast<const __nv_bfloat16*>(q), q_stride, c, cu_tokens, T, Hq, window, sinks, scale,
      static_cast<__nv_bfloat16*>(out), out_stride, prefix_table, prefix_width, prefix_len);
  return (int)cudaGetLastError();
}

}  // namespace

size_t paged_attention_workspace(int, int, int, int, int, int, int) { return 0; }
size_t shared_prefix_workspace(int, int, int, int, int) { return 0; }

int paged_attention_launch(const void* q, long long q_stride, const PagedCache& c, const int* cu_tokens, int T,
                           int max_tokens, int Hq, int window, int sinks, float scale, void* out, long long out_stride,
                           void*, size_t, int sm_count, cudaStream_t s) {
  if (const int bad = check_rows(q, q_stride, c, T, Hq, out, out_stride)) return bad;
  if (max_tokens < 1 || window < 0 || sinks < 0 || (!cu_tokens && (T != c.B || max_tokens != 1))) return kErrBadShape;
  if (misaligned(cu_tokens, 4)) return kErrBadPointer;
  if (sm_count < 1) return -sm_count;
  return launch(q, q_stride, c, cu_tokens, T, Hq, window, sinks, scale, out, out_stride, nullptr, 0, nullptr, s);
}

int shared_prefix_launch(const void* q, long long q_stride, const PagedCache& c, const int* prefix_table,
                         int prefix_width, const int* prefix_len, int Hq, float scale, void* out, long long out_stride,
                         void*, size_t, int sm_count, cudaStream_t s) {
  if (const int bad = check_rows(q, q_stride, c, c.B, Hq, out, out_stride)) return bad;
  if (prefix_width < 0) return kErrBadShape;
  if ((long long)prefix_width * c.page > (1LL << 30)) return kErrTooLarge;
  if (!prefix_len || (prefix_width > 0 && !prefix_table) || misaligned(prefix_table, 4) || misaligned(prefix_len, 4))
    return kErrBadPointer;
  if (sm_count < 1) return -sm_count;
  return launch(q, q_stride, c, nullptr, c.B, Hq, 0, 0, scale, out, out_stride, prefix_table, prefix_width, prefix_len, s);
}

}  // namespace b2
