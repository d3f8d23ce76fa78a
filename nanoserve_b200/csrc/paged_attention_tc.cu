// Attention over a paged cache, many rows (prompts, several new tokens, a batch behind a shared prefix): tcgen05.
//
// Rows (token, query head) of a sequence that share a KV head are the M side of both products, 128 to a tile:
//   S (128 x 128 keys, fp32 in tensor memory) = Q (shared memory) . K^T (shared memory)
//   P = 2^(S scale/ln2 - m), rounded to bf16, over S in tensor memory
//   O (128 x D, fp32 in tensor memory) += P (tensor memory) . V (shared memory, keys along the contraction as they lie)
// A CTA holds two tiles' worth of tensor memory (S and O twice, all 512 columns), so that the tensor core works on one while
// the other's softmax runs:
//   two tiles (TWO)  two neighbouring row tiles share every block of keys
//   one tile         up to 128 rows: the two halves take blocks of keys in turn, and are joined at the end
// warps 0-3 / 4-7   softmax of the first / second tile: one thread per row, 128 scores of it in registers
// warp 8            loads: a ring of tiles of 128 keys (K, V in the order in which they are used), a page's rows per box
// warp 9            issues the products; warps 10, 11 zero the values that no row sees
// The reference m of a row's weights is its maximum over the first block that it sees something of.  After that no maximum is
// taken: weights over 1 are as exact as others, in fp32 and in bf16 alike, and a block whose weights add up to over 2^10 raises m
// by the sum's exponent, for the next one; O is then rescaled in tensor memory, between the products that use it.  Where half a
// block adds up to over 2^24 (scores that jump), m is taken anew at once, and that half's weights too.  O stays under 2^10 |v| for
// every block and another 2^25 |v|: under 2^128 for |v| < 2^100 over 2^17 blocks, for |v| < 2^94 over the 2^23 that a table may hold.
// What bounds it: 128 x 128 scores of heads of 128 take the tensor core 1024 cycles (both products), and the 16 exponentials per
// cycle of an SM as long.  An eighth of the exponentials are therefore polynomials on the multiply-add pipes, pairs at a time, and
// the second product starts when half of the weights are there.  The products are issued by one thread without a branch between
// them: with a choice of the lane and a barrier of the warp around each group that warp alone took 2900 cycles per 256 rows x 128
// keys, where the products take 2048.  8192 new tokens in a window of 4096, 28 / 4 heads of 128: 333 us, 1080 TFLOP/s (a bf16 GEMM
// here: 1670), in a long row of calls 380 to 390, 930, at the clock that the board's power limit leaves.  The tensor pipe is busy for
// 53 % of it: what is left is the softmax's chain and its wait for the next scores (with nothing done between the products 242 us).
// Tried there: two threads to a row, so that rows of half the length leave room in registers, 388 us where one took 353; every
// second, third or fourth pair a polynomial 413, 358 and 357; the next block's scores in halves, beside the weights, 375 where 353
// (products of 64 columns read their operands twice); weights handed over as 96 and 32 keys 339 where 338.
// Every wait is bounded; a time-out is recorded in a word of this file's device image, which b2_device_status reads.
#include <algorithm>

#include "paged_attention.cuh"
#include "ptx.cuh"
#include "w4_common.cuh"
#include "w4_internal.h"

namespace b2 {
namespace {

constexpr int kKeys = 128;     // keys per block
constexpr int kLoadWarp = 8, kMmaWarp = 9;
constexpr int kThreads = 384;  // three warpgroups: registers are handed over in wholes of them
constexpr int kRegsSoftmax = 216, kRegsOther = 72;  // 2 * 216 + 72 = 3 * 168, what the launch gives
constexpr int kEvery = 8;      // every eighth pair of exponentials is a polynomial
constexpr int kPresent = 16;   // blocks whose presence bits are kept

__device__ int g_timed_out;  // a wait of this file's kernel ran out
Devices g_ran;

template <int D, bool TWO>
struct Geo {
  static constexpr int kTile = 128 * D * 2;                  // 128 rows of Q, K or V
  static constexpr int kQ = (TWO ? 2 : 1) * kTile;
  static constexpr int kBufs = std::min(12, (224 * 1024 - kQ) / kTile);
  static constexpr int kBar = kQ + kBufs * kTile;
  static constexpr int kSmem = kBar + 1024 + 1024;           // barriers; room to align to 1024
  static constexpr int kRowsPerCta = TWO ? 256 : 128;
};

// D[tmem] (+)= A[tmem] . B[smem]
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// V as it lies: rows of keys (the contraction) of 64 elements of D, 128-byte swizzle.  The next 64 elements lie a tile of 128
// rows further (leading offset), the next eight keys 1024 bytes (stride offset).
__device__ __forceinline__ uint64_t desc_v(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3FFFF) >> 4) | static_cast<uint64_t>((128 * 128) >> 4) << 16 |
         static_cast<uint64_t>(1024 >> 4) << 32 | static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 2^x, two at a time, to 2^-18: x = n + f with |f| <= 1/2 (n + 127 lands in the low bits of a sum with 1.5 * 2^23), a
// polynomial of fourth degree in f (least largest relative error), times 2^n.  0 from -127 down, infinity from 128 up; not a number
// stays that.
__device__ __forceinline__ float2 ex2_pair(float2 x) {
  constexpr float kMagic = 12582912.f + 127.f;
  asm("max.NaN.f32 %0, %0, %1;\n\tmin.NaN.f32 %0, %0, %2;" : "+f"(x.x) : "f"(-127.f), "f"(128.f));
  asm("max.NaN.f32 %0, %0, %1;\n\tmin.NaN.f32 %0, %0, %2;" : "+f"(x.y) : "f"(-127.f), "f"(128.f));
  auto both = [](float v) { return make_float2(v, v); };
  const float2 t = add_f32x2(x, both(kMagic)), n = add_f32x2(t, both(-kMagic));
  const float2 f = fma_f32x2(n, both(-1.f), x);
  float2 r = fma_f32x2(f, both(0.009570102207362652f), both(0.05591785907745361f));
  r = fma_f32x2(r, f, both(0.240247443318367f));
  r = fma_f32x2(r, f, both(0.6931217908859253f));
  r = fma_f32x2(r, f, both(0.9999992847442627f));
  return mul_f32x2(r, make_float2(__uint_as_float(__float_as_uint(t.x) << 23), __uint_as_float(__float_as_uint(t.y) << 23)));
}

// Ones in the bits below x.
__device__ __forceinline__ unsigned below(int x) { return x <= 0 ? 0u : x >= 32 ? ~0u : (1u << x) - 1; }

// Tile `t` of `size` rows, sequence after sequence: its rows and what they see.  The whole warp asks.
struct Tile {
  Visible v;     // rows: of the tile, counted in (token, head)
  int b, r0;     // sequence, and the tile's first row of it
  int p0;        // position of the sequence's first token in this call
  // False: there is no such tile.
  __device__ __forceinline__ bool find(const ManyRows& p, int size, int t) {
    const int lane = threadIdx.x & 31;
    int first = 0, n_new = p.mask.flat, len = 0, all = p.mask.flat * p.rep;
    if (p.mask.flat) {
      b = 0;
      r0 = t * size;
      len = __ldcg(p.c.lens);
      if (r0 >= all) return false;
    } else {
      int before = 0;
      b = -1;
      for (int b0 = 0; b0 < p.c.B && b < 0; b0 += 32) {
        int rows = 0;
        if (b0 + lane < p.c.B) {
          first = p.cu_tokens ? __ldcg(p.cu_tokens + b0 + lane) : b0 + lane;
          n_new = p.cu_tokens ? __ldcg(p.cu_tokens + b0 + lane + 1) - first : 1;
          len = __ldcg(p.c.lens + b0 + lane);
          rows = first < 0 ? 0 : max(0, min(min(n_new, p.max_tokens), p.T - first)) * p.rep;
        }
        const int n = (rows + size - 1) / size;
        int x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        const unsigned beyond = __ballot_sync(0xffffffffu, before + x > t);
        const int l = beyond != 0 ? __ffs(beyond) - 1 : 31;
        if (beyond != 0) {
          b = b0 + l;
          r0 = (t - before - __shfl_sync(0xffffffffu, x - n, l)) * size;
          first = __shfl_sync(0xffffffffu, first, l);
          n_new = __shfl_sync(0xffffffffu, n_new, l);
          len = __shfl_sync(0xffffffffu, len, l);
          all = __shfl_sync(0xffffffffu, rows, l);
        }
        before += __shfl_sync(0xffffffffu, x, 31);
      }
      if (b < 0) return false;
    }
    v.first = first;
    v.rows = n_new;
    v.set<kKeys>(p.mask, len, p.c.width << p.c.page_shift);
    p0 = v.pmin;
    v.rows = min(size, all - r0);
    if (!p.mask.flat) {
      v.pmax = p0 + (r0 + v.rows - 1) / p.rep;
      v.pmin = p0 + r0 / p.rep;
      v.span<kKeys>(p.mask);
    }
    return true;
  }
};

template <int D, bool TWO>
__global__ void __launch_bounds__(kThreads, 1)
    many_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const ManyRows p) {
  using geo = Geo<D, TWO>;
  constexpr int kHalves = D / 64;
  constexpr int kAhead = TWO ? 1 : 2;  // blocks whose scores are under way before the first weights are there
  extern __shared__ unsigned char raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  unsigned char* gen = raw + (base - smem_u32(raw));
  const uint32_t ring = base + geo::kQ;
  const uint32_t bar_full = base + geo::kBar, bar_empty = bar_full + 8 * geo::kBufs;
  // bar_p: [half of the weights][tile]
  const uint32_t bar_s = bar_empty + 8 * geo::kBufs, bar_p = bar_s + 16, bar_o = bar_p + 32, bar_h = bar_o + 16,
                 bar_q = bar_h + 16, bar_z = bar_q + 8, bar_y = bar_z + 8 * geo::kBufs;
  unsigned char* misc = gen + geo::kBar + 32 * geo::kBufs + 88;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(misc);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc + 4);
  volatile unsigned* present = reinterpret_cast<volatile unsigned*>(misc + 8);  // [kPresent]
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

  if (tid == 0) {
    *abort_flag = 0;
    for (int s = 0; s < geo::kBufs; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
      mbar_init(bar_y + 8 * s, 1);  // values with some that no row sees are on their way
      mbar_init(bar_z + 8 * s, 2);  // those are zeros
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(bar_s + 8 * t, 1);
      mbar_init(bar_p + 8 * t, 4);
      mbar_init(bar_p + 16 + 8 * t, 4);
      mbar_init(bar_o + 8 * t, 1);
      mbar_init(bar_h + 8 * t, 1);  // the second product's first half is done
    }
    mbar_init(bar_q, 8);
    fence_mbar_init();
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  pdl_wait_prior_grid();
  pdl_launch_dependents();  // (behind the wait: see FewRows::late_wait)

  // the longest tiles of a prompt are its last
  const int z = blockIdx.x % p.splits, h = blockIdx.x / p.splits % p.c.Hk;
  const int tile = gridDim.x / (p.splits * p.c.Hk) - 1 - blockIdx.x / (p.splits * p.c.Hk);
  Tile tl;
  const bool exists = tl.find(p, geo::kRowsPerCta, tile);
  const int b = tl.b, r0 = tl.r0;
  int i0 = 0, n = 0;
  if (exists) {
    i0 = (int)((long long)tl.v.count * z / p.splits);
    n = (int)((long long)tl.v.count * (z + 1) / p.splits) - i0;
  }
  const Visible& v = tl.v;
  // Whether some row sees each of a block's keys: blocks [seen0, seen1), and [0, sink1) of the first tokens'.
  const int skip = v.n_sink - v.from - i0;  // block b of the keys is this CTA's i = b + skip
  const int seen0 = max(v.n_sink - i0, (p.mask.window ? max(0, v.pmin - p.mask.window + kKeys) / kKeys : 0) + skip);
  const int seen1 = max(0, min(v.end, v.pmax + 1)) / kKeys + skip;
  const int sink1 = min(v.n_sink, p.mask.sinks / kKeys) - i0;
  auto whole_block = [&](int i) { return (i >= seen0 && i < seen1) || i < sink1; };

  if (warp >= kLoadWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (exists && warp == kLoadWarp) {
      // ------------------------------------------------------------ loads
      const int box_rows = min(p.c.page, kKeys), boxes = kKeys / box_rows;
      const int* table = p.c.table + b * p.c.table_stride;
      // loads 0 .. kAhead - 1: K of these blocks; then V of block i, K of block i + kAhead, in turn
      const int ahead = min(kAhead, n), total = 2 * n;
      auto what = [&](int x, int* block) {
        if (x < ahead) {
          *block = x;
          return 0;
        }
        const int y = x - ahead;
        if (y < 2 * (n - ahead)) {
          *block = (y >> 1) + ((y & 1) ? ahead : 0);
          return (y & 1) ? 0 : 1;
        }
        *block = n - ahead + (y - 2 * (n - ahead));  // V of the last blocks
        return 1;
      };
      // The pages of 32 / boxes blocks at a time, one to a lane: those of the values' block, of the next ones (the keys are up to two
      // blocks ahead), and the ones behind on their way.  One lane issues all boxes of a block: of lanes that issue one each, every one
      // took a round of its own (a block of four boxes 1150 cycles; three chunks 20.7 us against 18.7).
      const int log_boxes = 31 - __clz(boxes), log_per = 5 - log_boxes, mine = lane >> log_boxes, bx = lane & (boxes - 1);
      auto pages_of = [&](int group) {
        const int block = (group << log_per) + mine;
        return block < n ? page_at(p.c, table, p.c.width, (v.block(i0 + block) * kKeys + bx * box_rows) >> p.c.page_shift) : -1;
      };
      int group = 0, pages = pages_of(0), pages1 = pages_of(1), pages2 = pages_of(2), s = 0;
      uint32_t ph = 0;
      for (int x = 0; x < total; ++x) {
        int block;
        const int is_v = what(x, &block);
        if (is_v && block >> log_per > group) {
          ++group;
          pages = pages1, pages1 = pages2, pages2 = pages_of(group + 2);
        }
        const int held = block >> log_per == group ? pages : pages1, from = (block << log_boxes) & 31;
        const unsigned there = __ballot_sync(0xffffffffu, held >= 0) >> from & ((1u << boxes) - 1);
        int page[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) page[i] = __shfl_sync(0xffffffffu, held, from + i);
        if (!__all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * s, ph ^ 1, abort_flag))) break;  // (no loads behind a wait that ran out)
        if (lane == 0) {
          const uint32_t full = bar_full + 8 * s, to = ring + s * geo::kTile;
          if (!is_v) present[block % kPresent] = there;
          if (is_v && !whole_block(block)) mbar_arrive(bar_y + 8 * s);
          mbar_arrive_expect_tx(full, geo::kTile);
          const CUtensorMap* const map = is_v ? &tmap_v : &tmap_k;
          const int row = (v.block(i0 + block) * kKeys) & (p.c.page - 1);  // (pages of fewer rows: 0)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (i >= boxes) break;
#pragma unroll
            for (int half = 0; half < kHalves; ++half)
              tma_load_4d(to + half * (128 * 128) + i * box_rows * 128, map, half * 64, row, h, page[i] < 0 ? p.c.n_pages : page[i], full);
          }
        }
        __syncwarp();
        if (++s == geo::kBufs) { s = 0; ph ^= 1; }
      }
    } else if (exists && warp == kMmaWarp) {
      // ------------------------------------------------------------ products (one thread)
      constexpr uint32_t idesc_s = umma_idesc_bf16(128, 128);
      constexpr uint32_t idesc_o = umma_idesc_bf16(128, D) | (1u << 16);  // B along N as it lies
      if (elect_one()) {
        int s = 0;
        uint32_t ph = 0, ph_z = 0;
        auto scores = [&](int t, uint32_t buf) {
          const uint64_t dq = umma_desc_k128(base + (TWO ? t * geo::kTile : 0)), dk = umma_desc_k128(buf);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_f16_ss(tmem + 128 * t, dq + (kk >> 2) * ((128 * 128) >> 4) + 2 * (kk & 3),
                        dk + (kk >> 2) * ((128 * 128) >> 4) + 2 * (kk & 3), idesc_s, kk > 0);
          umma_commit(bar_s + 8 * t);
        };
        // (half of the keys)
        auto values = [&](int t, int half, uint32_t buf, bool first) {
          const uint64_t dv = desc_v(buf);
#pragma unroll
          for (int k4 = 0; k4 < kKeys / 32; ++k4) {
            const int kk = half * (kKeys / 32) + k4;
            umma_ts(tmem + 256 + 128 * t, tmem + 128 * t + 8 * kk, dv + kk * (2048 >> 4), idesc_o, !first || kk > 0);
          }
          if (half == 0) umma_commit(bar_h + 8 * t);
        };
        auto weights_of = [&](int t, int half, uint32_t parity) {
          mbar_wait(bar_p + 16 * half + 8 * t, parity, abort_flag);
          tc_fence_after_sync();
        };
        auto loaded = [&] {
          mbar_wait(bar_full + 8 * s, ph, abort_flag);
          tc_fence_after_sync();
          return ring + s * geo::kTile;
        };
        auto step = [&] {
          if (++s == geo::kBufs) { s = 0; ph ^= 1; }
        };
        // (a commit to bar_empty: the buffer is free once what was issued is done)
        if (n > 0) mbar_wait(bar_q, 0, abort_flag);
        for (int i = 0; i < min(kAhead, n); ++i) {
          const uint32_t buf = loaded();
          scores(TWO ? 0 : i, buf);
          if (TWO) scores(1, buf);
          umma_commit(bar_empty + 8 * s);
          step();
        }
        for (int i = 0; i < n; ++i) {
          const uint32_t buf_v = loaded();
          if (!whole_block(i)) {
            mbar_wait(bar_z + 8 * s, (ph_z >> s) & 1, abort_flag);
            ph_z ^= 1u << s;
          }
          const int s_v = s;
          step();
          if constexpr (TWO) {
            uint32_t buf_k = 0;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              weights_of(t, 0, i & 1);
              values(t, 0, buf_v, i == 0);
              if (t == 0 && i + 1 < n) buf_k = loaded();
              weights_of(t, 1, i & 1);
              values(t, 1, buf_v, false);
              if (t == 1) umma_commit(bar_empty + 8 * s_v);
              if (i + 1 < n)
                scores(t, buf_k);
              else
                umma_commit(bar_o + 8 * t);
            }
            if (i + 1 < n) {
              umma_commit(bar_empty + 8 * s);
              step();
            }
          } else {
            const int t = i & 1;
            weights_of(t, 0, (i >> 1) & 1);
            values(t, 0, buf_v, i < 2);
            uint32_t buf_k = 0;
            if (i + 2 < n) buf_k = loaded();
            weights_of(t, 1, (i >> 1) & 1);
            values(t, 1, buf_v, false);
            umma_commit(bar_empty + 8 * s_v);
            if (i + 2 < n) {
              scores(t, buf_k);
              umma_commit(bar_empty + 8 * s);
              step();
            } else {
              umma_commit(bar_o + 8 * t);
            }
          }
        }
      }
      __syncwarp();
    } else if (exists) {
      // ------------------------------------------------------------ zeros
      // Keys that no row sees may hold anything, and 0 times an infinity is none: their values become zeros.
      // (bar_y first: of a phase of bar_full that is further off than the next, a wait would not know.)
      uint32_t ph_y = 0;
      for (int i = 0; i < n; ++i) {
        if (whole_block(i)) continue;
        const int at = i < n - kAhead ? min(kAhead, n) + 2 * i : n + i, slot = at % geo::kBufs;  // of the loads (see there)
        mbar_wait(bar_y + 8 * slot, (ph_y >> slot) & 1, abort_flag);
        ph_y ^= 1u << slot;
        mbar_wait(bar_full + 8 * slot, (at / geo::kBufs) & 1, abort_flag);
        __syncwarp();
        const int j0 = v.block(i0 + i) * kKeys, thread = 32 * (warp - kMmaWarp - 1) + lane;
        auto clear = [&](int from, int to) {
          for (int x = from * (kHalves * 8) + thread; x < to * (kHalves * 8); x += 64)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                             ring + slot * geo::kTile + x / 8 % kHalves * (128 * 128) + x / (kHalves * 8) * 128 + (x & 7) * 16),
                         "r"(0)
                         : "memory");
        };
        clear(max(0, min(v.end, v.pmax + 1) - j0), kKeys);
        if (p.mask.window) clear(max(0, p.mask.sinks - j0), min(kKeys, v.pmin - p.mask.window + 1 - j0));
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_z + 8 * slot);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    if (exists) {
      // ------------------------------------------------------------ softmax: a row per thread
      const int t = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
      const int r = r0 + (TWO ? 128 * t : 0) + row, tok = r / p.rep, head = h * p.rep + r - tok * p.rep;
      const unsigned real = __ballot_sync(0xffffffffu, (TWO ? 128 * t : 0) + row < v.rows);  // of the warp's rows
      // Sixteen bytes to a lane, the lanes of a row beside one another: rows of global memory in whole sectors.
      constexpr int kPieces = D / 8, kRowsAtOnce = 32 / kPieces;  // of a row of bf16; rows per instruction
      const int piece = lane % kPieces, sub = lane / kPieces;
      {
        // Q (one tile: each half of the warps half of its rows); chunk c of sixteen bytes of row r lies at c ^ (r & 7)
        constexpr int kLoads = (TWO ? 32 : 16) / kRowsAtOnce;
        const long long off = (long long)(v.first + tok) * p.q_stride + head * D;
        uint4 x[kLoads];  // (all on their way before the first is stored)
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int rr = (TWO ? 0 : 16 * t) + i * kRowsAtOnce + sub;
          const long long at = __shfl_sync(0xffffffffu, off, rr);
          x[i] = (real >> rr) & 1 ? __ldcg(reinterpret_cast<const uint4*>(p.q + at) + piece) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int qrow = quad * 32 + (TWO ? 0 : 16 * t) + i * kRowsAtOnce + sub;
          sts128(base + (TWO ? t * geo::kTile : 0) + (piece >> 3) * (128 * 128) + qrow * 128 + (((piece & 7) ^ (qrow & 7)) << 4), x[i]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_q);
      }
      const int pos = p.mask.flat ? v.pmax : tl.p0 + tok;
      // The blocks that every row of this warp sees whole, as far as positions go: [whole0, whole1) of those behind the first tokens'.
      int whole0 = 0, whole1 = 0;
      {
        const int w0 = r0 + (TWO ? 128 * t : 0) + quad * 32;
        const int first = p.mask.flat ? v.pmin : tl.p0 + w0 / p.rep, last = p.mask.flat ? v.pmax : tl.p0 + (w0 + 31) / p.rep;
        const int lo = p.mask.window ? max(0, last - p.mask.window + 1) : 0;
        const int skip = v.n_sink - v.from - i0;  // block b of the keys is this CTA's i = b + skip
        whole0 = max(v.n_sink - i0, (lo + kKeys - 1) / kKeys + skip);
        whole1 = max(0, min(v.end, first + 1)) / kKeys + skip;
      }
      const int all_present = (1 << (kKeys / min(p.c.page, kKeys))) - 1;
      const uint32_t lanes = (uint32_t)quad * 32 << 16;
      const uint32_t t_s = tmem + lanes + 128 * t, t_o = tmem + lanes + 256 + 128 * t;
      const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
      // m: the reference in powers of two (-inf: nothing seen yet); l: the sum; up: powers by which the last block asks m to rise
      float m = -INFINITY, l = 0.f;
      int up = 0;
      auto rescale = [&](float corr) {
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          uint32_t o[16];
          tmem_ld_32x16(t_o + 16 * c, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
          tmem_st_32x16(t_o + 16 * c, o);
        }
        tmem_st_wait();
      };
      uint32_t parity = 0;  // of the tile's block
      for (int i = TWO ? 0 : t; i < n; i += TWO ? 1 : 2, parity ^= 1) {
        const bool whole = i >= whole0 && i < whole1;
        const bool some = __any_sync(0xffffffffu, up > 0 || m == -INFINITY);
        mbar_wait(bar_s + 8 * t, parity, abort_flag);
        __syncwarp();
        tc_fence_after_sync();
        float s[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32(t_s + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * c]));
        const unsigned there = present[i % kPresent];
        tmem_ld_wait();
        if (!whole || there != (unsigned)all_present) {
          // visible columns: first ones up to `few`, and those from `lo` to `hi`
          const int j0 = v.block(i0 + i) * kKeys, box_shift = min(p.c.page_shift, 7);
          const int hi = min(pos, v.end - 1) - j0;
          const int lo = p.mask.window ? pos - p.mask.window + 1 - j0 : 0;
          const int few = p.mask.window ? min(p.mask.sinks - j0, hi + 1) : 0;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            unsigned keep = (below(hi + 1 - 32 * c) & ~below(lo - 32 * c)) | below(few - 32 * c);
            keep &= ((there >> (32 * c >> box_shift)) & 1 ? 0xffffu : 0u) | ((there >> ((32 * c + 16) >> box_shift)) & 1 ? 0xffff0000u : 0u);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((keep >> e) & 1)) s[32 * c + e] = -INFINITY;
          }
        }
        auto largest = [&] {
          float top[4];  // (four chains)
#pragma unroll
          for (int c = 0; c < 4; ++c) top[c] = max3(s[c], s[4 + c], s[8 + c]);
#pragma unroll
          for (int c = 12; c < 124; c += 8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) top[e] = max3(top[e], s[c + e], s[c + 4 + e]);
          }
          return p.scale_log2 * fmaxf(max3(max3(top[0], s[124], s[125]), top[1], s[126]), max3(top[2], top[3], s[127]));
        };
        const bool first = i < (TWO ? 1 : 2);
        if (some) {
          if (!first && __any_sync(0xffffffffu, up > 0)) {
            const float corr = __uint_as_float((unsigned)(127 - up) << 23);
            l *= corr;
            m += (float)up;
            rescale(corr);
          }
          const float mx = largest();
          if (m == -INFINITY) m = mx;  // (what this row's O and l hold so far is zero)
        }
        float added = 0.f;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t w[32];
          float mine;
          auto weigh = [&] {
            const float neg = m == -INFINITY ? 0.f : -m;
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              float2 x = fma_f32x2(make_float2(s[64 * half + 2 * e], s[64 * half + 2 * e + 1]), scale2, make_float2(neg, neg));
              x = e % kEvery == kEvery - 1 ? ex2_pair(x) : make_float2(ex2(x.x), ex2(x.y));
              sum[e & 1] = add_f32x2(sum[e & 1], x);
              const __nv_bfloat162 y = __floats2bfloat162_rn(x.x, x.y);
              w[e] = *reinterpret_cast<const uint32_t*>(&y);
            }
            tmem_st_32x32(t_s + 32 * half, w);
            sum[0] = add_f32x2(sum[0], sum[1]);
            mine = sum[0].x + sum[0].y;
          };
          weigh();
          const bool large = !(mine < 16777216.f);  // 2^24, or not a number
          if (__any_sync(0xffffffffu, large)) {  // (rows that are not large keep their reference, and with it their bits)
            const float mx = largest(), mn = large ? fmaxf(m, mx) : m, corr = m == mn ? 1.f : ex2(m - mn);
            if (half == 1) {  // the first half's product has to be done before O is rescaled
              mbar_wait(bar_h + 8 * t, parity, abort_flag);
              __syncwarp();
              tc_fence_after_sync();
            }
            if (!first || half == 1) rescale(corr);
            l *= corr;
            added *= corr;
            m = mn;
            weigh();
          }
          added += mine;
          tmem_st_wait();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_p + 16 * half + 8 * t);
        }
        l += added;
        up = added > 1024.f && added < INFINITY ? (int)(__float_as_uint(added) >> 23) - 127 : 0;
      }
      // ------------------------------------------------------------ results
      if (n > (TWO ? 0 : t)) mbar_wait(bar_o + 8 * t, 0, abort_flag);
      __syncwarp();
      tc_fence_after_sync();
      float* other = reinterpret_cast<float*>(gen + geo::kQ);  // one tile: the second half's, [D + 2][128], where the ring was
      if constexpr (!TWO) {
        if (n > 1) mbar_wait(bar_o + 8 * (1 - t), 0, abort_flag);  // (both halves' products have left Q and the ring)
        __syncwarp();
        if (t == 1 && n > 1) {
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld_32x16(t_o + 16 * c, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) other[(16 * c + e) * 128 + row] = __uint_as_float(o[e]);
          }
          other[D * 128 + row] = m;
          other[(D + 1) * 128 + row] = l;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
      } else if (n == 0) {
        asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");  // (nobody stores Q any more where rows will leave)
      }
      if (TWO || t == 0) {
        float f0 = 1.f, f1 = 0.f;
        const bool two_parts = !TWO && n > 1;
        if (two_parts) {
          const float m1 = other[D * 128 + row], l1 = other[(D + 1) * 128 + row], mn = fmaxf(m, m1);
          f0 = m == mn ? 1.f : ex2(m - mn);
          f1 = m1 == mn ? 1.f : ex2(m1 - mn);
          l = f0 * l + f1 * l1;
          m = mn;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const long long slot = (((long long)h * p.slots + (TWO ? 2 * tile + t : tile)) * p.splits + z) * 128 + row;
        const bool parts = p.part != nullptr;
        if (parts && (real >> lane) & 1) p.stat[slot] = make_float2(m, l);
        // rows leave through the place where Q was, 2 D bytes of a row at a time, to be stored in whole sectors
        constexpr int kBytes = 2 * D;
        const uint32_t stage = base + (TWO ? t * geo::kTile : 0) + quad * 32 * kBytes;
        const long long off = parts ? slot * D : (long long)(v.first + tok) * p.out_stride + head * D;
        auto staged = [&](int at, uint32_t a, uint32_t bb, uint32_t c, uint32_t d) {
          sts128(stage + lane * kBytes + ((at ^ (lane & (kPieces - 1))) << 4), make_uint4(a, bb, c, d));
        };
        auto store = [&](char* to, int elem, int first_elem) {  // 2 D bytes of every row
          __syncwarp();
          constexpr int kBatch = 8;  // (reads first, then what waits for them)
#pragma unroll
          for (int i0 = 0; i0 < 32 / kRowsAtOnce; i0 += kBatch) {
            uint4 x[kBatch];
            long long at[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
              const int rr = (i0 + i) * kRowsAtOnce + sub;
              x[i] = lds128(stage + rr * kBytes + ((piece ^ (rr & (kPieces - 1))) << 4));
            }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) at[i] = __shfl_sync(0xffffffffu, off, (i0 + i) * kRowsAtOnce + sub);
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
              if ((real >> ((i0 + i) * kRowsAtOnce + sub)) & 1)
                *reinterpret_cast<uint4*>(to + (at[i] + first_elem) * elem + piece * 16) = x[i];
          }
          __syncwarp();
        };
        auto columns = [&](int c, float (&x)[16]) {  // sixteen of them
          uint32_t o[16];
          __syncwarp();
          if (n > 0) {
            tmem_ld_32x16(t_o + 16 * c, o);
            tmem_ld_wait();
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            x[e] = n > 0 ? __uint_as_float(o[e]) : 0.f;
            if (two_parts) x[e] = f0 * x[e] + f1 * other[(16 * c + e) * 128 + row];
          }
        };
        if (parts) {
          constexpr int kAtOnce = D / 32;  // sixteens of columns that 2 D bytes hold in fp32
#pragma unroll 1
          for (int c0 = 0; c0 < D / 16; c0 += kAtOnce) {
#pragma unroll
            for (int c = 0; c < kAtOnce; ++c) {
              float x[16];
              columns(c0 + c, x);
#pragma unroll
              for (int q = 0; q < 4; ++q)
                staged(c * 4 + q, __float_as_uint(x[4 * q]), __float_as_uint(x[4 * q + 1]), __float_as_uint(x[4 * q + 2]),
                       __float_as_uint(x[4 * q + 3]));
            }
            store(reinterpret_cast<char*>(p.part), 4, 16 * c0);
          }
        } else {
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            float x[16];
            columns(c, x);
            uint32_t y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const __nv_bfloat162 pair =
                  __floats2bfloat162_rn(inv == 0.f ? 0.f : x[2 * e] * inv, inv == 0.f ? 0.f : x[2 * e + 1] * inv);
              y[e] = *reinterpret_cast<const uint32_t*>(&pair);
            }
            staged(2 * c, y[0], y[1], y[2], y[3]);
            staged(2 * c + 1, y[4], y[5], y[6], y[7]);
          }
          store(reinterpret_cast<char*>(p.out), 2, 0);
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (tid == 0 && *abort_flag) g_timed_out = 1;
  if (*abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);  // copies and products in flight end before their memory is released
    __syncthreads();
  }
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

// Splits of the keys joined: sixteen rows of a tile of 128 to a CTA, four to a warp.
template <int D>
__global__ void __launch_bounds__(128) join_many_kernel(const ManyRows p) {
  const int lane = threadIdx.x & 31, h = blockIdx.x / p.slots, slot = blockIdx.x - h * p.slots;
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const int size = p.two ? 256 : 128, off = p.two ? 128 * (slot & 1) : 0, row0 = blockIdx.y * 16 + (threadIdx.x >> 5) * 4;
  Tile tl;
  if (!tl.find(p, size, p.two ? slot >> 1 : slot)) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + i, r = tl.r0 + off + row;
    if (off + row >= tl.v.rows) return;
    const long long at = ((long long)h * p.slots + slot) * p.splits * 128 + row;
    Row<D> out;
    out.join(p.splits, lane, [&](int z) { return Part{p.stat, p.part, at + z * 128}; });
    const int tok = r / p.rep;
    out.store(p.out + (long long)(tl.v.first + tok) * p.out_stride + (h * p.rep + r - tok * p.rep) * D, lane);
  }
}

template <int D, bool TWO>
int launch(const ManyRows& p, cudaStream_t s) {
  CUtensorMap mk, mv;
  if (!paged_tensor_maps(p.c, kKeys, &mk, &mv)) return kErrBadShape;
  using geo = Geo<D, TWO>;
  static SharedMemoryOnce once;
  if (const int rc = once.allow(many_rows_kernel<D, TWO>, geo::kSmem, &g_ran)) return rc;
  const int tiles = TWO ? p.slots / 2 : p.slots;
  return launch_pdl(many_rows_kernel<D, TWO>, dim3((unsigned)(tiles * p.c.Hk * p.splits)), kThreads, geo::kSmem, s, mk, mv, p);
}

}  // namespace

int many_rows_timed_out(int dev, bool clear, int* word) { return timed_out_word(g_timed_out, g_ran, dev, clear, word); }

int many_rows_launch(const ManyRows& p, cudaStream_t s) {
  if (p.c.D == 64) return p.two ? launch<64, true>(p, s) : launch<64, false>(p, s);
  return p.two ? launch<128, true>(p, s) : launch<128, false>(p, s);
}
int join_many_launch(const ManyRows& p, cudaStream_t s) {
  const dim3 grid((unsigned)(p.slots * p.c.Hk), 8);
  return launch_pdl(p.c.D == 64 ? join_many_kernel<64> : join_many_kernel<128>, grid, 128, 0, s, p);
}

}  // namespace b2
