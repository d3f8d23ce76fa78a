// Attention over a paged cache: b2_paged_attention (new tokens against their sequences, causal, sliding window, first tokens
// that stay visible) and b2_shared_prefix_attention (one token per sequence, all behind a common prefix).
//
//   o = sum_j e^{s_j - m} v_j / sum_j e^{s_j - m},   s_j = scale * q . k_j,   over the keys j that the row sees,
//
// in one pass over the keys with the running maximum m, sum and weighted rows in 32 bits; weights are rounded to bf16 for the
// second product, as tensor cores take them (the denominator adds up the unrounded ones).  A row that sees nothing is zero.
//
// Here: the kernel for few rows, whose time is that of reading the keys and values once, and what joins the parts of rows
// whose keys several CTAs shared.  paged_attention_tc.cu: the kernel for many rows.
//
// Few rows: the up to sixteen (token, query head) rows of a sequence that share a KV head are the M side of m16n8k16 products.
// Work is counted in blocks of 64 keys over all sequences and KV heads, and every CTA takes an equal run of them, wherever
// sequences begin and end: a batch of ragged lengths leaves no SM waiting for its longest member.  The lengths are on the
// device, so every CTA adds them up for itself.  One warp keeps TMA loads of the pages' rows in flight (a ring of 160 KB per SM);
// each of four warps takes sixteen keys of a block, with a maximum, sum and 16 x D of its own, joined at the end of a run.  Parts
// of rows whose keys several CTAs shared go through device memory to join_kernel.
//
// Bound by the start and the end of a launch, then by memory: a block of 64 keys of 128 takes an SM 1240 cycles from shared memory
// (at HBM's pace 32 KB take 1455), a launch some 7000 before the first block (lengths, tables, the first loads) and the join 2 to
// 4 us behind it.  28 / 4 heads of 128: 16 sequences of 500 to 32767 tokens in a window of 4096, 89 MB, 27 us (22 where the L2 still
// holds a part of them); the own keys of 64 sequences behind a prefix, 34 us for 143 MB, 4.2 TB/s.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "paged_attention.cuh"
#include "paged_rows.cuh"
#include "ptx.cuh"
#include "tensor_map.h"
#include "w4_internal.h"

namespace b2 {
namespace {

constexpr int kKeys = 64;       // keys per block
constexpr int kRows = 16;       // rows of a tile
constexpr int kWarps = 4;       // each takes sixteen keys of a block
constexpr int kThreads = 32 * (kWarps + 1);

__device__ int g_timed_out;  // a wait of this file's kernels ran out
Devices g_ran;

template <int D>
struct Geo {
  static constexpr int kTile = kKeys * D * 2;                 // K (or V) of a block
  static constexpr int kStage = 2 * kTile;
  static constexpr int kStages = D == 128 ? 5 : 10;
  static constexpr int kJoin = kStages * kStage;              // the warps' 16 x D sums, joined here
  static constexpr int kPitch = D + 4;                        // floats from row to row there: rows start in different banks
  static constexpr int kQ = kJoin + kWarps * kRows * kPitch * 4;  // two tiles of sixteen rows of q
  static constexpr int kQPitch = 2 * D + 16;                  // bytes, for the same reason
  static constexpr int kQTile = kRows * kQPitch;
  static constexpr int kBar = kQ + 2 * kQTile;
  static constexpr int kSmem = kBar + 1024 + 1024;            // barriers, statistics; room to align to 1024
};

// Equal runs of `total` blocks over n CTAs: where CTA c's begins, and the CTA whose run block u is in.
struct Runs {
  unsigned each, more;  // the first `more` CTAs have one block more than `each`
  __device__ __forceinline__ Runs(unsigned total, unsigned n) : each(total / n), more(total - each * n) {}
  __device__ __forceinline__ unsigned start(unsigned c) const { return c * each + min(c, more); }
  __device__ __forceinline__ unsigned owner(unsigned u) const {
    const unsigned longer = more * (each + 1);
    return u < longer ? u / (each + 1) : more + (u - longer) / each;
  }
};

// What the device says about a sequence.
struct Told {
  int first, rows, len;
};
__device__ __forceinline__ Told told(const FewRows& p, int b) {
  Told t;
  t.first = p.mask.flat ? b * p.mask.flat : p.cu_tokens ? __ldcg(p.cu_tokens + b) : b;
  t.rows = p.mask.flat ? p.mask.flat : p.cu_tokens ? __ldcg(p.cu_tokens + b + 1) - t.first : 1;
  t.len = __ldcg(p.c.lens + (p.mask.flat ? 0 : b));
  return t;
}
// A sequence's rows and what they see; at least one block, so that somebody writes the rows that see nothing.
__device__ __forceinline__ Visible sequence_rows(const FewRows& p, const Told& t) {
  Visible v;
  v.first = t.first;
  v.rows = t.rows;
  v.set<kKeys>(p.mask, t.len, p.c.width << p.c.page_shift);
  v.rows = v.first < 0 ? 0 : max(0, min(min(v.rows, p.max_tokens), p.T - v.first));
  v.count = v.rows == 0 ? 0 : max(1, v.count);
  return v;
}
// The first query head of tile h of a sequence, and its rows.
__device__ __forceinline__ int kv_head(const FewRows& p, int h) { return p.groups == 1 ? h : h / p.groups; }
__device__ __forceinline__ int group(const FewRows& p, int h) { return p.groups == 1 ? 0 : h % p.groups; }
__device__ __forceinline__ int first_head(const FewRows& p, int h) { return kv_head(p, h) * p.rep_all + group(p, h) * kRows; }
__device__ __forceinline__ int tile_rows(const FewRows& p, const Visible& v, int h) {
  return v.rows * min(p.rep, p.rep_all - group(p, h) * kRows);
}
__device__ __forceinline__ int token_of(const FewRows& p, int row) { return p.max_tokens == 1 ? 0 : row / p.rep; }
// The sequences as a warp sees them, 32 at a time, one to a lane.  What the device says of the first 32 is kept, and the blocks of
// the first 128.  The whole warp asks.
struct Sequences {
  static constexpr int kKept = 4;
  Told kept;
  unsigned kept_n[kKept];  // this lane's blocks of a KV head
  unsigned total;          // blocks of all sequences and KV heads
  __device__ __forceinline__ Sequences(const FewRows& p) {
    const int lane = threadIdx.x & 31;
    Told t[kKept];
#pragma unroll
    for (int c = 0; c < kKept; ++c)  // (all on their way before the first is looked at)
      if (32 * c + lane < p.c.B) t[c] = told(p, 32 * c + lane);
    unsigned sum = 0;
#pragma unroll
    for (int c = 0; c < kKept; ++c) {
      kept_n[c] = 0;
      if (32 * c >= p.c.B) continue;
      if (32 * c + lane < p.c.B) kept_n[c] = sequence_rows(p, t[c]).count;
      sum += __reduce_add_sync(0xffffffffu, kept_n[c]);
    }
    kept = t[0];
    for (int b0 = 32 * kKept; b0 < p.c.B; b0 += 32)
      sum += __reduce_add_sync(0xffffffffu, b0 + lane < p.c.B ? (unsigned)sequence_rows(p, told(p, b0 + lane)).count : 0u);
    total = sum * p.heads;
  }
  __device__ __forceinline__ Visible rows(const FewRows& p, int b) const {
    Told t;
    if (b < 32) {
      t.first = __shfl_sync(0xffffffffu, kept.first, b);
      t.rows = __shfl_sync(0xffffffffu, kept.rows, b);
      t.len = __shfl_sync(0xffffffffu, kept.len, b);
    } else {
      t = told(p, b);
    }
    return sequence_rows(p, t);
  }
  // Blocks of one KV head in front of the sequence that holds block `stop` of them all, which is returned, or in front of
  // sequence `upto`.
  __device__ __forceinline__ int add_up(const FewRows& p, unsigned stop, int upto, unsigned* before) const {
    const int lane = threadIdx.x & 31;
    unsigned sum = 0;
    int found = -1;
    auto chunk = [&](int b0, unsigned n) {
      unsigned x = b0 + lane < upto ? n : 0;
      n = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const unsigned beyond = __ballot_sync(0xffffffffu, (sum + x) * p.heads > stop);
      if (beyond != 0) {
        const int l = __ffs(beyond) - 1;
        sum += __shfl_sync(0xffffffffu, x - n, l);
        found = b0 + l;
      } else {
        sum += __shfl_sync(0xffffffffu, x, 31);
      }
    };
#pragma unroll
    for (int c = 0; c < kKept; ++c)
      if (found < 0 && 32 * c < upto) chunk(32 * c, kept_n[c]);
    for (int b0 = 32 * kKept; b0 < upto && found < 0; b0 += 32)
      chunk(b0, b0 + lane < upto ? sequence_rows(p, told(p, b0 + lane)).count : 0);
    *before = sum;
    return found < 0 ? upto : found;
  }
};

// Where a run stands: block i of sequence b and tile h of it.
struct Walk {
  int b, h, i;
  Visible v;
  __device__ __forceinline__ void start(const FewRows& p, const Sequences& all, unsigned u) {
    unsigned before;
    b = all.add_up(p, u, p.c.B, &before);
    v = all.rows(p, b);
    const int off = (int)(u - before * p.heads);
    h = off / v.count;
    i = off - h * v.count;
  }
  __device__ __forceinline__ void next(const FewRows& p, const Sequences& all) {
    if (++i < v.count) return;
    i = 0;
    if (++h < p.heads) return;
    h = 0;
    do v = all.rows(p, ++b);
    while (v.count == 0);  // (a run ends within the last sequence that has blocks)
  }
};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    few_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const FewRows p) {
  using geo = Geo<D>;
  constexpr int kHalves = D / 64;  // a row of D is 64 elements (128 swizzled bytes) at a time
  extern __shared__ unsigned char raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  unsigned char* gen = raw + (base - smem_u32(raw));
  const uint32_t bar_full = base + geo::kBar, bar_empty = bar_full + 8 * geo::kStages;
  const uint32_t bar_q = bar_empty + 8 * geo::kStages;  // [2] there, [2] free
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + geo::kBar + 16 * geo::kStages + 32);
  volatile unsigned* present = reinterpret_cast<volatile unsigned*>(gen + geo::kBar + 16 * geo::kStages + 40);  // [kStages]
  float* s_m = reinterpret_cast<float*>(gen + geo::kBar + 256 + 4 * 16);  // [kWarps][kRows] maxima, then sums
  float* s_l = s_m + kWarps * kRows;
  float* s_o = reinterpret_cast<float*>(gen + geo::kJoin);                // [kWarps][kRows][kPitch]
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

  if (tid == 0) {
    *abort_flag = 0;
    for (int s = 0; s < geo::kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, kWarps);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar_q + 8 * s, 1);
      mbar_init(bar_q + 16 + 8 * s, kWarps);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  __syncthreads();
  if (!p.late_wait) pdl_wait_prior_grid();
  pdl_launch_dependents();

  const Sequences all(p);
  const int n_cta = gridDim.x, cta = blockIdx.x;
  const Runs runs(all.total, n_cta);
  const unsigned u0 = runs.start(cta), u1 = runs.start(cta + 1);
  if (u0 >= u1) {
    if (p.late_wait) pdl_wait_prior_grid();
    return;
  }
  Walk w;
  w.start(p, all, u0);

  if (warp == kWarps) {
    // ------------------------------------------------------------ loads: one box of a page's rows per lane
    const int box_rows = min(p.c.page, kKeys), boxes = kKeys / box_rows;
    const int bx = lane % boxes, half = lane / boxes % kHalves, which = lane / (boxes * kHalves);
    const bool loads = which < 2;
    auto page_of = [&](const Walk& w) {
      const int key = w.v.block(w.i) * kKeys + bx * box_rows;
      return page_at(p.c, p.c.table + w.b * p.c.table_stride, p.c.width, key >> p.c.page_shift);
    };
    int page = page_of(w), s = 0;
    uint32_t ph = 0, items = 0;
    bool fresh = true;  // the run's, or a tile's, first block: its rows of q are brought too, one to a lane
    for (unsigned u = u0; u < u1; ++u) {
      Walk next = w;
      int page_next = 0;
      if (u + 1 < u1) {  // (the next block's table entries are on their way while this one's slot is waited for)
        next.next(p, all);
        page_next = page_of(next);
      }
      if (fresh) {
        const uint32_t slot = items & 1;
        const int rows = tile_rows(p, w.v, w.h), tok = token_of(p, lane);
        if (!__all_sync(0xffffffffu, mbar_wait(bar_q + 16 + 8 * slot, ((items >> 1) & 1) ^ 1, abort_flag))) break;
        if (lane == 0) mbar_arrive_expect_tx(bar_q + 8 * slot, rows * 2 * D);
        __syncwarp();
        if (lane < rows)
          bulk_g2s(base + geo::kQ + slot * geo::kQTile + lane * geo::kQPitch,
                   p.q + (long long)(w.v.first + tok) * p.q_stride + (first_head(p, w.h) + lane - tok * p.rep) * D, 2 * D,
                   bar_q + 8 * slot);
        ++items;
      }
      if (!__all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * s, ph ^ 1, abort_flag))) break;  // (no loads behind a wait that ran out)
      const unsigned there = __ballot_sync(0xffffffffu, page >= 0) & ((1u << boxes) - 1);
      if (lane == 0) {
        present[s] = there;
        mbar_arrive_expect_tx(bar_full + 8 * s, geo::kStage);
      }
      __syncwarp();
      if (loads) {
        const int key = w.v.block(w.i) * kKeys + bx * box_rows;
        // (a page that is not there: a coordinate behind the last one, for which the load brings zeros)
        tma_load_4d(base + s * geo::kStage + which * geo::kTile + half * (kKeys * 128) + bx * box_rows * 128,
                    which ? &tmap_v : &tmap_k, half * 64, key & (p.c.page - 1), kv_head(p, w.h), page < 0 ? p.c.n_pages : page,
                    bar_full + 8 * s);
      }
      fresh = next.b != w.b || next.h != w.h;
      w = next;
      page = page_next;
      if (++s == geo::kStages) { s = 0; ph ^= 1; }
    }
    return;
  }

  // -------------------------------------------------------------- products: sixteen keys of every block to a warp
  const int g = lane >> 2, quad = lane & 3;
  const int box_shift = p.c.page_shift < 6 ? p.c.page_shift - 4 : 2;  // granule of sixteen keys -> box of the block
  const int key_lane = 16 * warp + (lane >> 4) * 8 + (lane & 7);      // K: this lane's row for ldmatrix, chunk (lane >> 3) & 1
  const int val_lane = 16 * warp + ((lane >> 3) & 1) * 8 + (lane & 7);  // V, transposed: row; chunk lane >> 4
  int s = 0;
  uint32_t ph = 0, items = 0;
  unsigned u = u0;
  while (u < u1) {
    // ---- one sequence and KV head, or what of them this run holds
    const Visible v = w.v;
    const int b = w.b, h = w.h, head0 = first_head(p, h), rows = tile_rows(p, v, h);
    const int n_blocks = (int)min((unsigned)(v.count - w.i), u1 - u);
    const bool whole = n_blocks == v.count;
    uint32_t qf[D / 16][4];
    int pos[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) pos[r] = min(v.pmin + token_of(p, g + 8 * r), v.pmax);
    {
      const uint32_t slot = items & 1, tile = base + geo::kQ + slot * geo::kQTile;
      mbar_wait(bar_q + 8 * slot, (items >> 1) & 1, abort_flag);
      __syncwarp();
      // (rows that do not exist hold anything: a row of the product has nothing of the others)
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        ldmatrix4(tile + ((lane & 7) + ((lane >> 3) & 1) * 8) * geo::kQPitch + 32 * kk + (lane >> 4) * 16, qf[kk]);
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_q + 16 + 8 * slot);
      ++items;
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[D / 8][4];
#pragma unroll
    for (int t = 0; t < D / 8; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[t][e] = 0.f;

    for (int n = 0; n < n_blocks; ++n, ++u) {
      const int j0 = v.block(w.i + n) * kKeys + 16 * warp;
      mbar_wait(bar_full + 8 * s, ph, abort_flag);
      __syncwarp();
      const uint32_t sk = base + s * geo::kStage, sv = sk + geo::kTile;
      const bool there = (present[s] >> (warp >> box_shift)) & 1;
      float c[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[t][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t f[4];
        const int chunk = 2 * (kk & 3) + ((lane >> 3) & 1);
        ldmatrix4(sk + (kk >> 2) * (kKeys * 128) + key_lane * 128 + ((chunk ^ (key_lane & 7)) << 4), f);
        mma_16816_bf16(c[0], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], f[0], f[1]);
        mma_16816_bf16(c[1], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], f[2], f[3]);
      }
      const bool full = there && v.all(p.mask, j0, 16);
      uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;  // V's rows of this lane's fragments that some row sees
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[t][e] *= p.scale_log2;
      if (!full) {
        keep0 = keep1 = 0;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int j = j0 + 8 * t + 2 * quad + e;
            if (there && v.any(p.mask, j)) (t ? keep1 : keep0) |= 0xffffu << (16 * e);
#pragma unroll
            for (int r = 0; r < 2; ++r)
              if (!(there && v.sees(p.mask, j, pos[r]))) c[t][2 * r + e] = -INFINITY;
          }
        }
      }
      // ---- softmax: rows g and g + 8
      uint32_t a[4];
      bool moved = false;
      float corr[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float mx = fmaxf(fmaxf(c[0][2 * r], c[0][2 * r + 1]), fmaxf(c[1][2 * r], c[1][2 * r + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[r], mx), from = mn == -INFINITY ? 0.f : mn;
        corr[r] = ex2(m[r] - from);
        moved |= mn != m[r];
        m[r] = mn;
        float e[4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int x = 0; x < 2; ++x) e[2 * t + x] = ex2(c[t][2 * r + x] - from);
        l[r] = l[r] * corr[r] + (e[0] + e[1]) + (e[2] + e[3]);
        a[r] = pack_bf16(e[0], e[1]);
        a[2 + r] = pack_bf16(e[2], e[3]);
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int t = 0; t < D / 8; ++t) {
          o[t][0] *= corr[0];
          o[t][1] *= corr[0];
          o[t][2] *= corr[1];
          o[t][3] *= corr[1];
        }
      }
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        uint32_t f[4];
        const int chunk = 2 * (t & 3) + (lane >> 4);
        ldmatrix4_trans(sv + (t >> 2) * (kKeys * 128) + val_lane * 128 + ((chunk ^ (val_lane & 7)) << 4), f);
        if (!full) {  // what nobody sees may hold anything: 0 times an infinity is none
          f[0] &= keep0;
          f[2] &= keep0;
          f[1] &= keep1;
          f[3] &= keep1;
        }
        mma_16816_bf16(o[2 * t], a[0], a[1], a[2], a[3], f[0], f[1]);
        mma_16816_bf16(o[2 * t + 1], a[0], a[1], a[2], a[3], f[2], f[3]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_empty + 8 * s);
      if (++s == geo::kStages) { s = 0; ph ^= 1; }
    }

    // ---- the four warps' parts
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (quad == 0) {
        s_m[warp * kRows + g + 8 * r] = m[r];
        s_l[warp * kRows + g + 8 * r] = l[r];
      }
#pragma unroll
      for (int t = 0; t < D / 8; ++t)
        *reinterpret_cast<float2*>(s_o + (warp * kRows + g + 8 * r) * geo::kPitch + 8 * t + 2 * quad) =
            make_float2(o[t][2 * r], o[t][2 * r + 1]);
    }
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");
    const unsigned start = u - n_blocks;  // (a CTA has at most two parts: what its run begins with, and what it ends with)
    const long long slot = whole ? 2LL * n_cta + b * p.heads + h : 2LL * cta + (start == u0 ? 0 : 1);
    const bool final = whole && !p.parts_only;
    constexpr int kQuads = D / 4;
    for (int x = tid; x < rows * kQuads; x += 32 * kWarps) {
      const int row = x / kQuads, d = 4 * (x - row * kQuads);
      float mm = -INFINITY, ll = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) mm = fmaxf(mm, s_m[k * kRows + row]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const float f = s_m[k * kRows + row] == mm ? 1.f : ex2(s_m[k * kRows + row] - mm);
        ll += f * s_l[k * kRows + row];
        const float4 t = *reinterpret_cast<const float4*>(s_o + (k * kRows + row) * geo::kPitch + d);
        acc.x += f * t.x;
        acc.y += f * t.y;
        acc.z += f * t.z;
        acc.w += f * t.w;
      }
      if (final) {
        const int tok = token_of(p, row);
        const float inv = ll == 0.f ? 0.f : 1.f / ll;  // 0: the row sees nothing
        *reinterpret_cast<uint2*>(p.out + (long long)(v.first + tok) * p.out_stride + (head0 + row - tok * p.rep) * D + d) =
            make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
      } else {
        *reinterpret_cast<float4*>(p.part + (slot * kRows + row) * D + d) = acc;
        if (d == 0) p.stat[slot * kRows + row] = make_float2(mm, ll);
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");
    if (u < u1) {
      w.i += n_blocks - 1;
      w.next(p, all);
    }
  }
  if (tid == 0 && *abort_flag) g_timed_out = 1;
  if (*abort_flag)
    for (int i = 0; i < 64; ++i) __nanosleep(2000);  // copies in flight land before the shared memory is released
  if (p.late_wait) pdl_wait_prior_grid();
}

// ---------------------------------------------------------------- joining parts
// One CTA per tile of a sequence, a warp to a row.
struct JoinArgs {
  FewRows own;                    // the sequences' own keys
  int prefix_kind;                // 0: none, 1 and 3: the same kernel over the prefix, one tile or several, 2: the kernel for many rows
  FewRows prefix;
  const float* many_part;         // [tile, split][128][D]
  const float2* many_stat;        // [tile, split][128]
  int many_splits, many_tiles;
};

// The parts of tile h of sequence b, written by few_rows_kernel: n of them, part i in slot(i).
struct FewParts {
  int c0, n, n_cta;
  unsigned s, each, more;
  long long whole;
  __device__ __forceinline__ FewParts(const FewRows& p, const Sequences& all, const Visible& v, int b, int h)
      : n_cta(p.n_cta), whole(2LL * p.n_cta + b * p.heads + h) {
    unsigned before;
    all.add_up(p, 0xffffffffu, b, &before);
    const Runs runs(all.total, n_cta);
    each = runs.each;
    more = runs.more;
    s = before * p.heads + (unsigned)h * v.count;
    c0 = (int)runs.owner(s);
    n = (int)runs.owner(s + v.count - 1) - c0 + 1;
  }
  __device__ __forceinline__ long long slot(int i) const {
    if (n == 1) return whole;
    const unsigned c = c0 + i;
    return 2LL * c + (c * each + min(c, more) >= s ? 0 : 1);
  }
};

// KIND: prefix_kind.  (Its own code for each: a launch this short takes as long as its instructions take to come.)
template <int D, int KIND>
__global__ void __launch_bounds__(256) join_kernel(const JoinArgs a) {
  const FewRows& p = a.own;
  const int b = blockIdx.x / p.heads, h = blockIdx.x - b * p.heads, lane = threadIdx.x & 31;
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const Sequences all(p);
  const Visible v = all.rows(p, b);
  const int rows = tile_rows(p, v, h);
  if (rows == 0) return;
  const FewParts own(p, all, v, b, h);
  if (KIND == 0 && own.n == 1) return;  // written by its one CTA
  // the prefix's parts in front, then its own: which rows of which arrays
  int n_pre = 0;
  FewParts pre = own;
  if constexpr (KIND == 1 || KIND == 3) {
    const Sequences parts(a.prefix);
    const int g = KIND == 3 ? b / a.prefix.mask.flat : 0;
    pre = FewParts(a.prefix, parts, parts.rows(a.prefix, g), g, h);
    n_pre = pre.n;
  } else if constexpr (KIND == 2) {
    n_pre = a.many_splits;
  }
  for (int row = threadIdx.x >> 5; row < rows; row += 8) {
    // of the prefix's rows, or of those of a tile of them
    const int r = (KIND == 3 ? b % a.prefix.mask.flat : b) * p.rep_all + group(p, h) * kRows + row;
    const long long pre0 = ((long long)kv_head(p, h) * a.many_tiles + r / 128) * a.many_splits * 128 + r % 128;
    Row<D> out;
    out.join(
        n_pre + own.n, lane, [&](int i) {
          return KIND == 0 || i >= n_pre ? Part{p.stat, p.part, own.slot(i - n_pre) * kRows + row}
                 : KIND == 2             ? Part{a.many_stat, a.many_part, pre0 + i * 128}
                                         : Part{a.prefix.stat, a.prefix.part, pre.slot(i) * kRows + r};
        });
    const int tok = token_of(p, row);
    out.store(p.out + (long long)(v.first + tok) * p.out_stride + (first_head(p, h) + row - tok * p.rep) * D, lane);
  }
}

// ---------------------------------------------------------------- host
constexpr size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
size_t part_bytes(long long slots, int rows, int D) { return align256((size_t)slots * rows * D * 4) + align256((size_t)slots * rows * 8); }

template <int D>
int launch_few_of(const FewRows& p, cudaStream_t s) {
  CUtensorMap mk, mv;
  if (!paged_tensor_maps(p.c, kKeys, &mk, &mv)) return kErrBadShape;
  static SharedMemoryOnce once;
  if (const int rc = once.allow(few_rows_kernel<D>, Geo<D>::kSmem, &g_ran)) return rc;
  return launch_pdl(few_rows_kernel<D>, dim3(p.n_cta), kThreads, Geo<D>::kSmem, s, mk, mv, p);
}

int launch_few(const FewRows& p, cudaStream_t s) { return p.c.D == 64 ? launch_few_of<64>(p, s) : launch_few_of<128>(p, s); }

FewRows few_rows(const void* q, long long q_stride, const PagedCache& c, const int* cu_tokens, int rep, float scale_log2,
                 void* out, long long out_stride, void* parts, long long slots, int n_cta, int T, int max_tokens) {
  FewRows p{};
  p.T = T;
  p.max_tokens = std::min(max_tokens, std::max(1, kRows / rep));
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_stride = q_stride;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_stride = out_stride;
  p.c = c;
  p.cu_tokens = cu_tokens;
  p.rep_all = rep;
  p.rep = std::min(rep, kRows);
  p.groups = (rep + kRows - 1) / kRows;
  p.heads = c.Hk * p.groups;
  p.n_cta = n_cta;
  p.scale_log2 = scale_log2;
  p.part = static_cast<float*>(parts);
  p.stat = reinterpret_cast<float2*>(static_cast<char*>(parts) + align256((size_t)slots * kRows * c.D * 4));
  return p;
}

int join(const JoinArgs& a, int rows, cudaStream_t s) {
  static void (*const kernels[2][4])(JoinArgs) = {{join_kernel<64, 0>, join_kernel<64, 1>, join_kernel<64, 2>, join_kernel<64, 3>},
                                                  {join_kernel<128, 0>, join_kernel<128, 1>, join_kernel<128, 2>, join_kernel<128, 3>}};
  return launch_pdl(kernels[a.own.c.D == 128][a.prefix_kind], dim3((unsigned)(a.own.c.B * a.own.heads)), 32 * std::min(rows, 8), 0, s, a);
}

int check_rows(const void* q, long long q_stride, const PagedCache& c, int T, int Hq, float scale, const void* out,
               long long out_stride) {
  if (!(scale > 0.f) || scale > FLT_MAX / 2 || T < 1 || Hq < 1 || Hq % c.Hk || (c.D != 64 && c.D != 128)) return kErrBadShape;
  if (!rows_fit(q_stride, (long long)Hq * c.D, T) || !rows_fit(out_stride, (long long)Hq * c.D, T)) return kErrBadShape;
  if (!q || !out || misaligned(q, 16) || misaligned(out, 16)) return kErrBadPointer;
  // rows and blocks are counted in 31 bits
  if ((long long)T * Hq > 0x3fffffffLL || ((long long)c.width * c.page / kKeys + 2) * c.B * Hq > 0x7fffffffLL) return kErrTooLarge;
  return 0;
}

}  // namespace

bool paged_tensor_maps(const PagedCache& c, int block, CUtensorMap* k, CUtensorMap* v) {
  const uint64_t dims[4] = {(uint64_t)c.D, (uint64_t)c.page, (uint64_t)c.Hk, (uint64_t)c.n_pages};
  // (the stride of a dimension of one is never used, but has to be one that a map may have)
  const uint64_t strides[3] = {(uint64_t)c.token_stride, (uint64_t)(c.Hk > 1 ? c.head_stride : c.D),
                               (uint64_t)(c.n_pages > 1 ? c.page_stride : c.D)};
  const uint32_t box[2] = {64, (uint32_t)std::min(c.page, block)};
  return make_tensor_map_4d(k, c.k, dims, strides, box) && make_tensor_map_4d(v, c.v, dims, strides, box);
}

namespace {

// How the kernel for many rows cuts a call up: tiles of 128 rows, two to a CTA where sequences have more; CTAs that would leave
// SMs idle share the keys of a tile, down to two blocks of 128 each.  Where single tiles just fill the SMs, or over half of them,
// they are a CTA's each: it then works on two blocks of keys at a time, which two CTAs would have to join (three chunks of
// 280 to 468 tokens, 16 / 2 heads of 64: 22 us against 30 when it was chosen, 18.7 since).
struct ManyPlan {
  int two, slots, splits;
};
ManyPlan many_plan(long long rows, int B, long long most_rows, int Hk, long long most_keys, int sm_count) {
  ManyPlan m;
  long long tiles = 0, likely = 0;
  for (m.two = 0;; m.two = 1) {
    const int size = m.two ? 256 : 128;
    tiles = std::min(rows / size + B, B * ((most_rows + size - 1) / size));  // no fewer than there are
    likely = std::max<long long>(1, std::max((rows + size - 1) / size, tiles - B / 2));
    if (m.two || most_rows <= 128 || (likely * Hk <= sm_count && 2 * likely * Hk > sm_count)) break;
  }
  m.slots = (int)(m.two ? 2 * tiles : tiles);
  // (a step over a tile's blocks takes some 1.9 us, a part 0.15 us in the join: the sum is least where steps and parts balance)
  const long long balance = (long long)std::sqrt((m.two ? 12.0 : 6.0) * (double)(most_keys / 128));
  m.splits = (int)std::max<long long>(1, std::min({sm_count / (likely * Hk), (most_keys + 255) / 256, balance}));
  return m;
}
size_t many_bytes(const ManyPlan& m, int Hk, int D) { return part_bytes((long long)m.slots * Hk * m.splits, 128, D); }

ManyRows many_rows(const void* q, long long q_stride, const PagedCache& c, const int* cu_tokens, int rep, int T,
                   int max_tokens, const ManyPlan& m, float scale_log2, void* out, long long out_stride, void* parts) {
  ManyRows p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_stride = q_stride;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_stride = out_stride;
  p.c = c;
  p.cu_tokens = cu_tokens;
  p.rep = rep;
  p.T = T;
  p.max_tokens = max_tokens;
  p.two = m.two;
  p.slots = m.slots;
  p.splits = m.splits;
  p.scale_log2 = scale_log2;
  if (parts) {
    p.part = static_cast<float*>(parts);
    p.stat = reinterpret_cast<float2*>(static_cast<char*>(parts) +
                                       align256((size_t)m.slots * c.Hk * m.splits * 128 * c.D * 4));
  }
  return p;
}

// Whether a sequence's rows of a KV head are the few-row kernel's.  (One token of more than sixteen heads takes two tiles or more,
// each of which reads the keys.)
bool few(int max_tokens, int rep) { return max_tokens == 1 || (long long)max_tokens * rep <= kRows; }

constexpr long long kMostKeys = 1LL << 30;

}  // namespace

int few_rows_timed_out(int dev, bool clear, int* word) { return timed_out_word(g_timed_out, g_ran, dev, clear, word); }

size_t paged_attention_workspace(int T, int B, int max_tokens, int Hq, int Hk, int D, int sm_count) {
  max_tokens = std::min(max_tokens, T);
  const int rep = Hq / Hk;
  if (few(max_tokens, rep)) return part_bytes(2LL * sm_count, kRows, D);
  const ManyPlan m = many_plan((long long)T * rep, B, (long long)max_tokens * rep, Hk, kMostKeys, sm_count);
  return std::max<size_t>(256, m.splits > 1 ? many_bytes(m, Hk, D) : 0);
}
// The prefix through the kernel for few rows: sixteen rows' worth of whole sequences to a tile.  0: a sequence's rows do not fit.
long long prefix_tiles(int B, int rep) { return rep > kRows ? 0 : (B + kRows / rep - 1) / (kRows / rep); }

size_t shared_prefix_workspace(int B, int Hq, int Hk, int D, int sm_count) {
  const int rep = Hq / Hk;
  const size_t own = part_bytes(2LL * sm_count + (long long)B * Hk * ((rep + kRows - 1) / kRows), kRows, D);
  const long long tiles = prefix_tiles(B, rep);
  const size_t few = tiles ? part_bytes(2LL * sm_count + tiles * Hk, kRows, D) : 0;  // (which it will be, the prefix's length says)
  if (tiles == 1) return own + few;
  return own + std::max(few, many_bytes(many_plan((long long)B * rep, 1, (long long)B * rep, Hk, kMostKeys, sm_count), Hk, D));
}

int paged_attention_launch(const void* q, long long q_stride, const PagedCache& c, const int* cu_tokens, int T,
                           int max_tokens, int Hq, int window, int sinks, float scale, void* out, long long out_stride,
                           void* workspace, size_t workspace_bytes, int sm_count, cudaStream_t s) {
  if (const int bad = check_rows(q, q_stride, c, T, Hq, scale, out, out_stride)) return bad;
  if (max_tokens < 1 || window < 0 || sinks < 0 || (!cu_tokens && (T != c.B || max_tokens != 1))) return kErrBadShape;
  if (misaligned(cu_tokens, 4)) return kErrBadPointer;
  if (sm_count < 1) return -sm_count;
  if (!workspace || misaligned(workspace, 16)) return kErrBadPointer;
  max_tokens = std::min(max_tokens, T);
  if (workspace_bytes < paged_attention_workspace(T, c.B, max_tokens, Hq, c.Hk, c.D, sm_count)) return kErrWorkspace;
  if (window >= 1 << 30) window = 0;  // (positions are below that)
  const int rep = Hq / c.Hk;
  const Mask mask{window, std::min(sinks, 1 << 30), 0};
  const float scale_log2 = scale * 1.44269504088896340736f;
  if (few(max_tokens, rep)) {
    JoinArgs a{};
    a.own = few_rows(q, q_stride, c, cu_tokens, rep, scale_log2, out, out_stride, workspace, 2LL * sm_count, sm_count, T,
                     max_tokens);
    a.own.mask = mask;
    if (const int rc = launch_few(a.own, s)) return rc;
    return join(a, max_tokens * rep, s);
  }
  const ManyPlan m = many_plan((long long)T * rep, c.B, (long long)max_tokens * rep, c.Hk, (long long)c.width * c.page, sm_count);
  ManyRows p = many_rows(q, q_stride, c, cu_tokens, rep, T, max_tokens, m, scale_log2, out, out_stride,
                         m.splits > 1 ? workspace : nullptr);
  p.mask = mask;
  const int rc = many_rows_launch(p, s);
  return rc || m.splits == 1 ? rc : join_many_launch(p, s);
}

int shared_prefix_launch(const void* q, long long q_stride, const PagedCache& c, const int* prefix_table,
                         int prefix_width, const int* prefix_len, int Hq, float scale, void* out, long long out_stride,
                         void* workspace, size_t workspace_bytes, int sm_count, cudaStream_t s) {
  if (const int bad = check_rows(q, q_stride, c, c.B, Hq, scale, out, out_stride)) return bad;
  const int rep = Hq / c.Hk;
  if (prefix_width < 0) return kErrBadShape;
  // (its tiles' blocks are counted in 31 bits too; several tiles are few rows' work only where there are few)
  if ((long long)prefix_width * c.page > (1LL << 30) ||
      (prefix_tiles(c.B, rep) == 1 && ((long long)prefix_width * c.page / kKeys + 2) * c.Hk > 0x7fffffffLL))
    return kErrTooLarge;
  if (!prefix_len || (prefix_width > 0 && !prefix_table) || misaligned(prefix_table, 4) || misaligned(prefix_len, 4))
    return kErrBadPointer;
  if (sm_count < 1) return -sm_count;
  if (!workspace || misaligned(workspace, 16)) return kErrBadPointer;
  if (workspace_bytes < shared_prefix_workspace(c.B, Hq, c.Hk, c.D, sm_count)) return kErrWorkspace;
  const float scale_log2 = scale * 1.44269504088896340736f;
  const long long own_slots = 2LL * sm_count + (long long)c.B * c.Hk * ((rep + kRows - 1) / kRows);
  char* prefix_parts = static_cast<char*>(workspace) + part_bytes(own_slots, kRows, c.D);
  PagedCache pre = c;
  pre.table = prefix_table;
  pre.width = prefix_width;
  pre.lens = prefix_len;
  pre.B = 1;
  JoinArgs a{};
  int own_ctas = sm_count;
  // A tile reads all of the prefix, which several of them do where it is short and the sequences' own tables are: up to two blocks of
  // 64 keys to an SM in all, up to 128 rows, up to four blocks to an SM of own keys.  The kernel for many rows takes 13 us for whatever
  // it does (777 tokens, three sequences of 28 / 4 heads of 128: 13.2 us the three launches, 18.9 through that one; 500 tokens, 16
  // sequences of 300 and of 2000: 15.8 and 29.4 against 18.4 and 26.4).  Where both tables hold more blocks than there are SMs, the two
  // kernels divide these in that ratio, up to eight blocks to a CTA of the prefix's; else idle CTAs make room by themselves.
  const long long tiles = prefix_tiles(c.B, rep);
  const long long blocks = tiles * c.Hk * std::max(1LL, ((long long)prefix_width * c.page + kKeys - 1) / kKeys);
  const long long own_blocks = (long long)c.B * c.Hk * (((long long)c.width * c.page + kKeys - 1) / kKeys);
  const bool little = blocks <= 2LL * sm_count;
  if (tiles == 1 || (tiles > 1 && little && c.B * rep <= 128 && own_blocks <= 4LL * sm_count)) {
    a.prefix_kind = tiles == 1 ? 1 : 3;
    pre.B = (int)tiles;
    pre.table_stride = 0;
    int ctas = sm_count;
    if (little && blocks + own_blocks > sm_count) {
      const long long share = std::max(sm_count * blocks / (blocks + own_blocks), (blocks + 7) / 8);
      ctas = (int)std::max<long long>(1, std::min({share, blocks, sm_count - (sm_count + 7LL) / 8}));
      own_ctas = std::max(1, sm_count - ctas);
    }
    a.prefix = few_rows(q, q_stride, pre, nullptr, rep, scale_log2, out, out_stride, prefix_parts, 2LL * sm_count + tiles * c.Hk,
                        ctas, c.B, c.B);
    a.prefix.mask = Mask{0, 0, std::min(c.B, kRows / rep)};
    a.prefix.parts_only = 1;
    if (const int rc = launch_few(a.prefix, s)) return rc;
  } else {
    const long long rows = (long long)c.B * rep;
    const ManyPlan m = many_plan(rows, 1, rows, c.Hk, (long long)prefix_width * c.page, sm_count);
    ManyRows p = many_rows(q, q_stride, pre, nullptr, rep, c.B, c.B, m, scale_log2, out, out_stride, prefix_parts);
    p.mask = Mask{0, 0, c.B};
    if (const int rc = many_rows_launch(p, s)) return rc;
    a.prefix_kind = 2;
    a.many_part = p.part;
    a.many_stat = p.stat;
    a.many_splits = m.splits;
    a.many_tiles = m.slots;
    // Where the prefix leaves a third of the SMs or more, the own keys' kernel runs beside it, on those alone (8192 tokens, 16
    // sequences of up to 512: 23 us against 27.5 with CTAs for all SMs, half of which waited for the prefix's to end).
    const int left = sm_count - (m.two ? m.slots / 2 : m.slots) * c.Hk * m.splits;
    if (left * 3 >= sm_count) own_ctas = left;
  }
  a.own = few_rows(q, q_stride, c, nullptr, rep, scale_log2, out, out_stride, workspace, own_slots, own_ctas, c.B, 1);
  a.own.mask = Mask{0, 0, 0};
  a.own.parts_only = 1;
  a.own.late_wait = 1;
  if (const int rc = launch_few(a.own, s)) return rc;
  return join(a, rep, s);
}

}  // namespace b2
