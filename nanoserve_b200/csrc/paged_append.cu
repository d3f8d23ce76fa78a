// b2_paged_kv_append: what stands between a batch's q|k|v projection and its attention over a paged cache, in one pass over
// the rows: bias, rotate-half rotary embedding of q and k, q to its own buffer, k and v into the pages of their sequences.
//
//   x = qkv + bias;  (a, b) = (x[i], x[i + D/2]) -> (a cos - b sin, b cos + a sin),  angle = position * inv_freq[i]
//
// in 32 bits with one rounding to bf16 at the store.  The angle is formed and reduced to [-pi, pi] in 64 bits: in 32 bits the
// product alone is off by 2^-24 of itself, 0.004 radians at position 65536.
//
// Bound by memory.  A thread moves eight (i, i + D/2) pairs of one head, two rows at a time, for rows the grid's length apart: while
// its loads are on their way, a thread makes an angle of the next rows and a warp finds where the rows behind those belong, so that
// nothing waits for the chain of row, sequence, page and angle (6665 rows of 28 / 4 heads of 128: 41 us with a CTA to a row and
// its loads behind the chain, 29 us so; 16 rows 3.3 and 2.6 us).  Of these 29 us the 123 MB are 19 at HBM's pace; the rest is that a
// row's loads live within one turn of the loop: issued at its top, used behind the next rows' angles (DRAM at 34 %).
#include <algorithm>

#include "paged_attention.cuh"
#include "ptx.cuh"
#include "w4_internal.h"

namespace b2 {
namespace {

constexpr int kMaxHalf = 128;  // D / 2
constexpr int kMostThreads = 320;  // three CTAs to an SM at up to 64 registers

struct Place {
  int pos;       // of the row in its sequence; negative: there is none, and nothing of the row is written
  int stored;    // its page is there
  long long at;  // where in the caches, without the head
};

__device__ __forceinline__ uint32_t word(const uint4& x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }
__device__ __forceinline__ float2 pair_of(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ uint32_t pack_pair(float2 x) {
  const __nv_bfloat162 y = __floats2bfloat162_rn(x.x, x.y);
  return *reinterpret_cast<const uint32_t*>(&y);
}

template <int R>
__global__ void __launch_bounds__(kMostThreads, 3) paged_append_kernel(const __nv_bfloat16* qkv, long long qkv_stride,
                                                                    const __nv_bfloat16* bias, const float* inv_freq,
                                                                    __nv_bfloat16* q_out, long long q_stride, PagedCache c,
                                                                    const int* cu_tokens, int T, int Hq) {
  __shared__ alignas(8) float s_cos[2][R][kMaxHalf], s_sin[2][R][kMaxHalf];
  __shared__ Place s_place[3][R];
  const int D = c.D, half = D / 2, per_head = D / 16, units = (Hq + 2 * c.Hk) * per_head, groups = (T + R - 1) / R;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int u = blockIdx.y * blockDim.x + threadIdx.x, h = u / per_head, e0 = (u - h * per_head) * 8;
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const float freq0 = (int)threadIdx.x < R * half ? __ldcg(inv_freq + threadIdx.x % half) : 0.f;  // of this thread's first angle
  auto load = [&](int g, uint4 (&x)[R][2]) {
    if (u >= units || g >= groups) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const __nv_bfloat16* src = qkv + (long long)min(g * R + r, T - 1) * qkv_stride + (long long)h * D + e0;
      x[r][0] = __ldcg(reinterpret_cast<const uint4*>(src));
      x[r][1] = __ldcg(reinterpret_cast<const uint4*>(src + half));
    }
  };
  auto find = [&](int g, int r, Place* to) {
    const int t = g * R + r;
    int first = 0, n_new = 1, len = 0;
    const int b = t < T ? sequence_of(cu_tokens, c, t, &first, &n_new, &len) : -1;
    Place at{-1, 0, 0};
    if (b >= 0) {
      at.pos = len - n_new + (t - first);
      const int page = at.pos < 0 ? -1 : page_at(c, c.table + b * c.table_stride, c.width, at.pos >> c.page_shift);
      at.stored = page >= 0;
      at.at = (long long)page * c.page_stride + (long long)(at.pos & (c.page - 1)) * c.token_stride;
    }
    if (lane == 0) to[r] = at;
  };
  auto turn = [&](const Place* of, int to) {
    for (int i = threadIdx.x; i < R * half; i += blockDim.x) {
      const int r = i / half, f = i - r * half;
      const float freq = i == (int)threadIdx.x ? freq0 : __ldcg(inv_freq + f);
      if (of[r].pos >= 0) rotation(of[r].pos, freq, &s_sin[to][r][f], &s_cos[to][r][f]);
    }
  };
  const int g0 = blockIdx.x, step = gridDim.x;
  uint4 x[R][2], add[2] = {};
  load(g0, x);
  if (bias != nullptr && u < units) {
    add[0] = __ldcg(reinterpret_cast<const uint4*>(bias + h * D + e0));
    add[1] = __ldcg(reinterpret_cast<const uint4*>(bias + h * D + half + e0));
  }
  if (warp < R) find(g0, warp, s_place[0]);
  if (warp >= R && warp < 2 * R) find(g0 + step, warp - R, s_place[1]);
  __syncthreads();
  turn(s_place[0], 0);
  __syncthreads();
  int now = 0, place = 0;
  for (int g = g0; g < groups; g += step) {
    if (g != g0) load(g, x);
    const int place1 = place == 2 ? 0 : place + 1, place2 = place1 == 2 ? 0 : place1 + 1;
    if (g + step < groups) {
      turn(s_place[place1], now ^ 1);
      const int last = (int)(blockDim.x >> 5) - 1 - warp;  // (the warps that are not the first to make angles)
      if (last < R) find(g + 2 * step, last, s_place[place2]);
    }
    if (u < units) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const Place at = s_place[place][r];
        if (at.pos < 0 || (h >= Hq && !at.stored)) continue;
        const bool turned = h < Hq + c.Hk;
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {  // two pairs at a time
          float2 a = pair_of(word(x[r][0], w)), b = pair_of(word(x[r][1], w));
          a = add_f32x2(a, pair_of(word(add[0], w)));
          b = add_f32x2(b, pair_of(word(add[1], w)));
          if (turned) {
            const float2 cs = *reinterpret_cast<const float2*>(&s_cos[now][r][e0 + 2 * w]);
            const float2 sn = *reinterpret_cast<const float2*>(&s_sin[now][r][e0 + 2 * w]);
            const float2 y = make_float2(a.x * cs.x - b.x * sn.x, a.y * cs.y - b.y * sn.y);
            b = make_float2(b.x * cs.x + a.x * sn.x, b.y * cs.y + a.y * sn.y);
            a = y;
          }
          lo[w] = pack_pair(a);
          hi[w] = pack_pair(b);
        }
        __nv_bfloat16* dst = h < Hq          ? q_out + (long long)(g * R + r) * q_stride + (long long)h * D
                             : h < Hq + c.Hk ? c.k + at.at + (h - Hq) * c.head_stride
                                             : c.v + at.at + (h - Hq - c.Hk) * c.head_stride;
        *reinterpret_cast<uint4*>(dst + e0) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        *reinterpret_cast<uint4*>(dst + half + e0) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      }
    }
    __syncthreads();
    now ^= 1;
    place = place1;
  }
}

}  // namespace

int paged_append_launch(const void* qkv, long long qkv_stride, const void* bias, const void* inv_freq, void* q_out,
                        long long q_stride, const PagedCache& c, const int* cu_tokens, int T, int Hq, int sm_count,
                        cudaStream_t s) {
  const long long heads = (long long)Hq + 2 * c.Hk;
  if (T < 1 || Hq < 1 || (!cu_tokens && T != c.B)) return kErrBadShape;
  if (!rows_fit(qkv_stride, heads * c.D, T) || !rows_fit(q_stride, (long long)Hq * c.D, T)) return kErrBadShape;
  if (!qkv || !inv_freq || !q_out || misaligned(qkv, 16) || misaligned(bias, 16) || misaligned(q_out, 16) ||
      misaligned(inv_freq, 4) || misaligned(cu_tokens, 4))
    return kErrBadPointer;
  if (heads * c.D > (1 << 24)) return kErrTooLarge;
  if (sm_count < 1) return -sm_count;
  // a unit to a thread; where there are more, they are cut into as few and as equal parts as fit
  const int units = (int)heads * (c.D / 16), parts = (units + kMostThreads - 1) / kMostThreads;
  const int threads = std::max(128, ((units + parts - 1) / parts + 31) / 32 * 32);
  const bool two = T >= 2 * sm_count;
  const int groups = two ? (T + 1) / 2 : T, resident = std::max(1, sm_count * std::max(1, 3 * kMostThreads / threads) / parts);
  return launch_pdl(two ? paged_append_kernel<2> : paged_append_kernel<1>, dim3(std::min(groups, resident), parts), threads, 0, s,
                    static_cast<const __nv_bfloat16*>(qkv), qkv_stride, static_cast<const __nv_bfloat16*>(bias),
                    static_cast<const float*>(inv_freq), static_cast<__nv_bfloat16*>(q_out), q_stride, c, cu_tokens, T, Hq);
}

}  // namespace b2
