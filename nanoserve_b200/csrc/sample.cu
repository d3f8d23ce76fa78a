// b2_sample: one token per row of logits l, drawn with a given random number u in [0, 1).
//
//   w_i = e^{(l_i - max l) / T}                                   (T <= 0: the largest logit, lowest index)
//   A   = the top_k largest of {i : w_i >= min_p}                 (equal logits: the lowest index first)
//   B   = the shortest prefix of A, in falling order, whose weight reaches top_p of A's
//   token = the first i of B, in the order of the vocabulary, with  sum_{j <= i, j in B} w_j > u * sum_{j in B} w_j
//
// Both borders and the draw are exact questions about sums over up to 2^18 terms, so weights are formed in 64 bits and added up
// as whole multiples of 2^-44: the sums do not depend on the order of the additions, and not on how a row is cut up.
//
// A row is read once: a cluster of C CTAs keeps it in shared memory as sortable keys.
//   1. the largest key; a histogram of the others' distance from it in 2048 equal steps up to 40 T (beyond, a weight is 0 here):
//      counts, one atomic an element, and without top_k a second one of how far in its bin a logit lies, in 256ths.  Every CTA adds
//      up a C-th of the bins over the cluster and sends the sums to all.
//   2. counts bound both borders: exactly the bin of the top_k-th logit, and, since weights within a bin are e^(-40/2048) or
//      nearer to one another (with the mean place in the bin known, 2^-14), bins between which the top_p border lies.
//   3. where no more than 1024 logits are in front of the borders' far end, they are gathered in one CTA, which goes on alone:
//      it sorts them, and prefix sums give both borders and the draw.
//   4. else the logits stay where they are.  The exact borders are found by radix selection (eight bits at a time) among the
//      few keys of the bins that the borders lie in, and the draw by prefix sums over all CTAs.
//
// Bound by the steps between barriers and by the shared memory's atomics and 64-bit weights, not by the logits' bytes: of 47 us for
// 16 rows of 152064 bf16 logits (5 MB, 0.75 us at HBM's pace), a row of way 4 takes 72000 cycles: loading 5000, the largest 4000,
// counting 7500, the borders' bins 6000, the pass over the weights 16000, the selections 13000, prefix sums and the draw the rest.  A
// row of way 3 takes 19 us.  By the rows drawn 46 to 59 us; 64 fp32 rows with settings of their own 63 to 71 us.
#include <algorithm>

#include "paged_attention.cuh"
#include "ptx.cuh"
#include "w4_internal.h"

namespace b2 {
namespace {

constexpr int kThreads = 1024;
constexpr int kBins = 2048;      // of the first histogram, of distances
constexpr int kDigit = 256;      // of the selections on keys
constexpr int kPowers = 1024;    // of the table of 2^(j / kPowers)
constexpr int kList = kThreads;  // logits that one CTA looks at alone, one to a thread
constexpr float kReach = 40.f;   // distances beyond it, in T, have a weight under 2^-57: none
constexpr int kMaxVocab = 1 << 18;
constexpr int kSliceBytes = 150 * 1024;
constexpr size_t kMaxSmem = 227 * 1024;
constexpr double kOne = 17592186044416.0;  // 2^44: a weight of 1
constexpr double kWhole = 6755399441055744.0;  // 1.5 * 2^52: a double added to it is rounded to a whole number, in its low bits

using u32 = unsigned;
using u64 = unsigned long long;

// Falling order of keys is falling order of logits; 0 is a logit that is not a number.
__device__ __forceinline__ u32 key_of(float x) {
  if (x != x) return 0;
  const u32 b = __float_as_uint(x == 0.f ? 0.f : x);  // -0 equals 0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float logit_of(u32 k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// Keys in shared memory: 32 bits, or for bf16 the upper 16 (the lower ones are all 0, or all 1 for negative logits).
template <typename L>
struct Keys;
template <>
struct Keys<float> {
  using Stored = u32;
  static constexpr int kBits = 32, kPerWord = 1;
  static __device__ __forceinline__ float load(const void* p, size_t i) { return __ldcg(static_cast<const float*>(p) + i); }
  static __device__ __forceinline__ u32 stored(u32 k) { return k; }
  static __device__ __forceinline__ float logit(u32 s) { return logit_of(s); }
};
template <>
struct Keys<__nv_bfloat16> {
  using Stored = unsigned short;
  static constexpr int kBits = 16, kPerWord = 2;
  static __device__ __forceinline__ float load(const void* p, size_t i) {
    return __uint_as_float((u32)__ldcg(static_cast<const unsigned short*>(p) + i) << 16);
  }
  static __device__ __forceinline__ u32 stored(u32 k) { return k >> 16; }
  static __device__ __forceinline__ float logit(u32 s) { return logit_of((s << 16) | ((s & 0x8000u) ? 0u : 0xffffu)); }
};

constexpr int kLimb = 15;  // a bin's weight in three sums of fifteen bits each: up to 2^17 elements leave them in 32 bits
struct alignas(16) Shared {
  // this CTA's, then (sums) the cluster's up to each bin, within the part of it one CTA adds up
  alignas(8) u32 count[kBins];
  alignas(8) u32 sums[kBins];
  u32 inside[kBins], insides[kBins];  // the same for how far in their bin the logits lie, in 256ths (each bin for itself)
  u32 limb[2][3][kDigit];          // a selection's bins (counts: the first alone), two in turn: peers may still read the other
  double power[kPowers];           // 2^44 2^(j / kPowers)
  u64 exchange[12];                // what this CTA tells the others, a place per question
  u64 scan[32], scanned[32];
  u64 found[6];
  u32 list_key[kList], list_at[kList];  // keys and their places in the vocabulary (or in this CTA's slice)
  u32 listed;
};

__device__ __forceinline__ u32 peer_u32(const u32* p, u32 rank) {
  u32 v;
  asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.u32 %0, [a];\n\t}"
               : "=r"(v) : "r"(smem_u32(p)), "r"(rank) : "memory");
  return v;
}
__device__ __forceinline__ void to_peer_u32(u32* p, u32 rank, u32 v) {
  asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\tst.shared::cluster.u32 [a], %2;\n\t}" ::"r"(smem_u32(p)),
               "r"(rank), "r"(v)
               : "memory");
}
__device__ __forceinline__ u64 peer_u64(const u64* p, u32 rank) {
  u64 v;
  asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.u64 %0, [a];\n\t}"
               : "=l"(v) : "r"(smem_u32(p)), "r"(rank) : "memory");
  return v;
}

// Sum of v over the threads in front of the calling one; total: over all.
template <typename T>
__device__ __forceinline__ T block_scan(T v, Shared& sh, T* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto inclusive = [&](T x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    return x;
  };
  const T x = inclusive(v);
  if (lane == 31) sh.scan[warp] = x;
  __syncthreads();
  if (warp == 0) sh.scanned[lane] = inclusive((T)sh.scan[lane]);
  __syncthreads();
  *total = (T)sh.scanned[31];
  return (warp > 0 ? (T)sh.scanned[warp - 1] : 0) + x - v;
}

template <typename L, int C>
__global__ void __launch_bounds__(kThreads) sample_kernel(const Sampling p, int chunk) {
  using K = Keys<L>;
  using Stored = typename K::Stored;
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  static_assert(sizeof(Shared) % 16 == 0, "the keys behind it are read sixteen bytes at a time");
  Stored* keys = reinterpret_cast<Stored*>(raw + sizeof(Shared));
  const int tid = threadIdx.x;
  const u32 rank = blockIdx.x % C;
  const int row = (int)(blockIdx.x / C);
  const int slice = kThreads * chunk, base = rank * slice;  // this CTA's logits: [base, base + slice)
  const int n = max(0, min(p.V - base, slice));
  int question = 0;
  auto meet = [&] {
    if constexpr (C > 1)
      cluster_barrier();
    else
      __syncthreads();
  };
  // Everybody's answer to the next question, added up; what the CTAs in front of this one said: before.
  auto heard = [&](int at, u64* before) {
    u64 told[C], sum = 0;
#pragma unroll
    for (u32 r = 0; r < (u32)C; ++r) told[r] = peer_u64(&sh.exchange[at], r);
    *before = 0;
#pragma unroll
    for (u32 r = 0; r < (u32)C; ++r) {
      if (r == rank) *before = sum;
      sum += told[r];
    }
    return sum;
  };
  auto ask = [&](u64 v, u64* before) {
    if (tid == 0) sh.exchange[question] = v;
    meet();
    return heard(question++, before);
  };

  // ---- 1. the row's slice as keys, and the largest
  for (int i = tid; i < kBins; i += kThreads) sh.count[i] = 0, sh.inside[i] = 0;
  if (tid == 0) sh.found[0] = 0, sh.listed = 0;
  const L* src = static_cast<const L*>(p.logits) + row * p.stride + base;
  u32 top = 0;
  constexpr int kVec = 16 / sizeof(L);
  const int vectors = (reinterpret_cast<uintptr_t>(src) & 15) == 0 ? n / kVec : 0;
  constexpr int kAhead = 4;  // loads of a thread on their way at a time; the table is made while the first are
  uint4 in[kAhead];
#pragma unroll
  for (int e = 0; e < kAhead; ++e)
    if (tid + e * kThreads < vectors) in[e] = __ldcg(reinterpret_cast<const uint4*>(src) + tid + e * kThreads);
  static_assert(kPowers == kThreads, "a thread per entry");
  sh.power[tid] = exp2(tid / (double)kPowers) * kOne;
  auto take = [&](const uint4& x, int i) {
    const u32 w[4] = {x.x, x.y, x.z, x.w};
    u32 out[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (K::kPerWord == 1) {
        out[e] = key_of(__uint_as_float(w[e]));
        top = max(top, out[e]);
      } else {
        const u32 lo = key_of(__uint_as_float(w[e] << 16)) >> 16, hi = key_of(__uint_as_float(w[e] & 0xffff0000u)) >> 16;
        out[e] = lo | hi << 16;
        top = max(top, max(lo, hi));
      }
    }
    reinterpret_cast<uint4*>(keys)[i] = make_uint4(out[0], out[1], out[2], out[3]);
  };
  for (int i0 = tid; i0 < vectors; i0 += kAhead * kThreads) {
#pragma unroll
    for (int e = 0; e < kAhead; ++e)
      if (i0 + e * kThreads < vectors) take(in[e], i0 + e * kThreads);
#pragma unroll
    for (int e = 0; e < kAhead; ++e)
      if (i0 + (kAhead + e) * kThreads < vectors)
        in[e] = __ldcg(reinterpret_cast<const uint4*>(src) + i0 + (kAhead + e) * kThreads);
  }
  for (int i = vectors * kVec + tid; i < slice; i += kThreads) {
    const u32 k = i < n ? key_of(K::load(src, i)) : 0;
    keys[i] = (Stored)K::stored(k);
    top = max(top, K::stored(k));
  }
  // the row's settings are on their way while the largest key is agreed on
  float T = p.temperature ? __ldcg(p.temperature + row) : p.temperature_all;
  int k = p.top_k ? __ldcg(p.top_k + row) : p.top_k_all;
  const float top_p = p.top_p ? __ldcg(p.top_p + row) : p.top_p_all;
  const float min_p = p.min_p ? __ldcg(p.min_p + row) : p.min_p_all;
  float u = __ldcg(p.u + row);
  top = __reduce_max_sync(0xffffffffu, top);
  __syncthreads();
  if ((tid & 31) == 0 && top) atomicMax(&sh.found[0], (u64)top);
  __syncthreads();
  if (tid == 0) sh.exchange[question] = sh.found[0];
  meet();
  top = 0;
#pragma unroll
  for (u32 r = 0; r < (u32)C; ++r) top = max(top, (u32)peer_u64(&sh.exchange[question], r));
  ++question;
  const float largest = K::logit(top);
  if (top == 0 || largest == __uint_as_float(0xff800000u)) {  // not a number, or nothing above minus infinity
    if (rank == 0 && tid == 0) p.tokens[row] = -1;
    meet();
    return;
  }

  if (!(T > 0.f)) k = 1, T = 1.f;
  T = fminf(T, 1e36f);  // (40 T has to be a number)
  if (k <= 0 || k > p.V) k = p.V;
  // (keys below this one have no weight, and minus infinity is below it)
  const u32 nothing = max(K::stored(key_of(largest - kReach * T)), K::stored(key_of(__uint_as_float(0xff800000u))) + 1);
  // The weight of a stored key in multiples of 2^-44.  2^(x / 1024) with x = whole + r, |r| <= 1/2: the whole part's low ten bits
  // from a table, the others into its exponent, and (r ln2 / 1024)^n / n! up to n = 3 (the next term is under 2^-50).  The last
  // product is added to 2^52, which rounds it to a whole number.
  // For keys that have a weight (from `nothing` on; of others it may be anything).  Where the largest logit is plus infinity only
  // its equals do.
  const bool finite = largest < __uint_as_float(0x7f800000u);
  const double per_T = finite ? kPowers * 1.4426950408889634074 / (double)T : 0.0, high = finite ? (double)largest : 0.0;
  auto weight = [&](u32 s) -> u64 {
    constexpr double a = 0.69314718055994530942 / kPowers;
    // fp32 to fp64 by its bits (a conversion takes as long as four products; numbers under 2^-126 become another such one)
    const u32 bits = __float_as_uint(K::logit(s));
    const double l = __hiloint2double((bits & 0x80000000u) | (((bits & 0x7fffffffu) >> 3) + (896u << 20)), bits << 29);
    const double x = (l - high) * per_T, t = x + kWhole, r = x - (t - kWhole);
    const int j = __double2loint(t);
    const double power = sh.power[j & (kPowers - 1)];
    const double scaled = __hiloint2double(__double2hiint(power) + ((j >> 10) << 20), __double2loint(power));
    const double v = fma(fma(fma(fma(a * a * a / 6.0, r, a * a / 2.0), r, a), r, 1.0), scaled, 4503599627370496.0);
    return (u64)__double_as_longlong(v) & ((1ull << 52) - 1);
  };

  // kept: keys above kf, and the first rf (in order of index) of those that equal it
  u32 kf = 0, rf = 0, equal = 0;  // equal: how many there are
  if (min_p > 0.f) {
    const double border = (double)largest + (double)T * log((double)fminf(min_p, 1.f));
    const u32 least = key_of(__double2float_ru(fmin(border, (double)largest)));
    // the smallest stored key that is no less than that
    const u32 s = K::kBits == 32 ? least : (least >> 16) + (K::logit(least >> 16) < logit_of(least) ? 1 : 0);
    if (s > 0) kf = min(s, top) - 1;
  }
  kf = max(kf, nothing - 1);  // (a logit without weight cannot be drawn, and counts for no border)

  const bool by_count = k < p.V, by_weight = !(top_p >= 1.f);
  // f(key) for every element of the slice, sixteen bytes to a read, in no order
  auto each = [&](auto f) {
    const uint4* v = reinterpret_cast<const uint4*>(keys);
    for (int i = tid; i < slice / kVec; i += kThreads) {
      const uint4 x = v[i];
      const u32 w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (K::kPerWord == 1) {
          f(w[e]);
        } else {
          f(w[e] & 0xffffu);
          f(w[e] >> 16);
        }
      }
    }
  };
  // f(four keys, place of the first in the slice) for this thread's elements, one behind the other
  const int words = chunk / K::kPerWord;
  auto in_order = [&](auto f) {
    const u32* mine = reinterpret_cast<const u32*>(keys) + tid * words;
    constexpr int kWords = 4 / K::kPerWord;
    for (int i = 0; i < words; i += kWords) {
      u32 s[4];
#pragma unroll
      for (int e = 0; e < kWords; ++e) {
        const u32 w = i + e < words ? mine[i + e] : 0;
        if constexpr (K::kPerWord == 1)
          s[e] = w;
        else
          s[2 * e] = w & 0xffffu, s[2 * e + 1] = w >> 16;
      }
      f(s, tid * chunk + i * K::kPerWord);
    }
  };
  // top_p of a weight, rounded up to a whole number, at least the first
  auto share = [&](u64 total) -> u64 {
    const double g = ceil((double)(top_p > 0.f ? top_p : 0.f) * (double)total);
    return g < 1.0 ? 1 : (u64)g > total ? total : (u64)g;
  };

  const float steps = kBins / (kReach * T);
  // falls with the key (each operation keeps the order); kBins and above: not counted
  auto distance = [&](u32 s) { return s == top ? 0.f : fminf((largest - K::logit(s)) * steps, (float)kBins); };
  auto bin_of = [&](u32 s) { return (int)distance(s); };
  // The smallest key of a bin up to b: a point to a lane.
  auto first_key = [&](int b) {
    u32 lo = 1, hi = top;
    while (lo < hi) {
      const u32 step = (hi - lo + 30) / 31, at = lo + min((u32)(tid & 31) * step, hi - lo);
      const int f = __ffs(__ballot_sync(0xffffffffu, bin_of(at) <= b)) - 1;
      hi = lo + min((u32)f * step, hi - lo);
      if (f > 0) lo += (f - 1) * step + 1;
    }
    return lo;
  };
  bool cut = false;  // top_k leaves some out:
  int bin_k = kBins - 1, bin_lo = 0, bin_hi = kBins - 1;  // the bin of the top_k-th, and those that hold the top_p border
  u32 front_k = 0;   // logits in front of bin_k

  if (by_count || by_weight) {
    // ---- 2. distances, counted
    const bool finer = by_weight && !by_count;
    each([&](u32 s) {
      if (s <= kf) return;
      const float x = distance(s);
      if (x >= (float)kBins) return;
      const int b = (int)x;
      atomicAdd(&sh.count[b], 1u);
      if (finer) atomicAdd(&sh.inside[b], (u32)((x - (float)b) * 256.f));
    });
    meet();
    constexpr int kPart = kBins / C;  // bins this CTA adds up, two to a thread (C = 1), or one
    {
      constexpr int kEach = kPart > kThreads ? kPart / kThreads : 1;
      u32 x[kEach], mine = 0, total;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        x[e] = 0;
        const int at = tid * kEach + e;
        if (at < kPart) {
          u32 y[C];
#pragma unroll
          for (u32 r = 0; r < (u32)C; ++r) y[r] = peer_u32(&sh.count[rank * kPart + at], r);
#pragma unroll
          for (u32 r = 0; r < (u32)C; ++r) x[e] += y[r];
        }
        mine += x[e];
      }
      u32 before = block_scan(mine, sh, &total);
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        before += x[e];
        const int at = rank * kPart + tid * kEach + e;
        if (tid * kEach + e < kPart) {
          u32 y = 0;
          if (finer) {
#pragma unroll
            for (u32 r = 0; r < (u32)C; ++r) y += peer_u32(&sh.inside[at], r);
          }
#pragma unroll
          for (u32 r = 0; r < (u32)C; ++r) {
            to_peer_u32(&sh.sums[at], r, before);
            if (finer) to_peer_u32(&sh.insides[at], r, y);
          }
        }
      }
    }
    meet();
    // every CTA has all sums now: this thread's two bins, and the logits up to each of them and in front
    const int b0 = 2 * tid;
    u32 base_count = 0, counted = 0;
#pragma unroll
    for (int r = 0; r < C; ++r) {
      const u32 x = sh.sums[(r + 1) * kPart - 1];
      if ((r + 1) * kPart <= b0) base_count += x;
      counted += x;
    }
    const u32 upto[2] = {base_count + sh.sums[b0], base_count + sh.sums[b0 + 1]};
    const u32 front[2] = {b0 % kPart ? base_count + sh.sums[b0 - 1] : base_count, upto[0]};
    cut = by_count && counted > (u32)k;
    const u32 left = cut ? (u32)k : counted;
    if (tid == 0) {
      sh.found[0] = kBins - 1, sh.found[1] = 0, sh.found[2] = counted;
      sh.found[3] = 0, sh.found[4] = kBins - 1, sh.found[5] = counted;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (cut && front[e] < left && upto[e] >= left) sh.found[0] = b0 + e, sh.found[1] = front[e], sh.found[2] = upto[e];
    __syncthreads();
    if (by_weight && !(cut && sh.found[2] <= kList)) {
      // The most and the least that the bins can weigh, in 2^-36.  A weight is e^(-w (bin + f)), f in [0, 1); with the mean of f
      // known, the average is at least e^-(w mean) and at most what the chord from f = 0 to 1 gives there: w^2 / 8 apart.
      constexpr float kWidth = kReach / kBins;
      u64 most[2], least[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const u32 n = min(upto[e], left) - min(front[e], left);
        const float near = __expf(-kWidth * (b0 + e)) * 68719476736.f * (float)n;
        const float mean = finer && n > 0 ? (float)sh.insides[b0 + e] / (256.f * (float)n) : 0.f;
        most[e] = (u64)(near * (1.f - mean * (1.f - __expf(-kWidth)))) + 1;
        least[e] = (u64)(near * __expf(-kWidth * (finer ? mean + 1.f / 256.f : 1.f)));
      }
      u64 total_most, total_least;
      u64 up = block_scan(most[0] + most[1], sh, &total_most), down = block_scan(least[0] + least[1], sh, &total_least);
      // the border is where the most that the bins can hold reaches top_p of the least, or further, and where the least reaches
      // top_p of the most, or nearer (5e-5: the rounding of distances and weights)
      const double share_p = (double)fmaxf(top_p, 0.f), lo = share_p * 0.99995 * (double)total_least,
                   hi = share_p * 1.00005 * (double)total_most;
      if (tid == 0 && hi <= 0.0) sh.found[4] = 0, sh.found[5] = upto[0];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if ((double)up < lo && (double)(up + most[e]) >= lo) sh.found[3] = b0 + e;
        if ((double)down < hi && (double)(down + least[e]) >= hi) sh.found[4] = b0 + e, sh.found[5] = upto[e];
        up += most[e];
        down += least[e];
      }
    }
    __syncthreads();
    bin_k = (int)sh.found[0];
    front_k = (u32)sh.found[1];
    bin_lo = (int)sh.found[3];
    bin_hi = (int)sh.found[4];
    const u32 n_work = (u32)sh.found[by_count ? 2 : 5];
    const int last_bin = by_count ? bin_k : bin_hi;

    if (n_work <= kList) {
      // ---- 3. the logits up to last_bin, gathered in the first CTA in the order of the vocabulary, and finished there
      if (by_weight && !by_count) {  // the whole's weight, exactly
        u64 mine = 0, total;
        each([&](u32 s) {
          const u64 v = weight(s);
          mine += s > kf ? v : 0;
        });
        block_scan(mine, sh, &total);
        if (tid == 0) sh.exchange[question] = total;
      }
      // (a thread's first few are kept in registers, so that one pass counts them and has them)
      constexpr int kFew = 4;
      u32 some = 0, mine_n, few_key[kFew], few_at[kFew];
      const u32 least = max(kf + 1, first_key(last_bin));
      auto wanted = [&](u32 x) { return x >= least; };
      in_order([&](const u32(&s)[4], int place) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (wanted(s[e])) {
#pragma unroll
            for (int f = 0; f < kFew; ++f)
              if (some == (u32)f) few_key[f] = s[e], few_at[f] = base + place + e;
            ++some;
          }
      });
      u32 at = block_scan(some, sh, &mine_n);
      if (some <= kFew) {
#pragma unroll
        for (int f = 0; f < kFew; ++f)
          if ((u32)f < some) sh.list_key[at + f] = few_key[f], sh.list_at[at + f] = few_at[f];
      } else {
        in_order([&](const u32(&s)[4], int place) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (wanted(s[e])) {
              sh.list_key[at] = s[e];
              sh.list_at[at++] = base + place + e;
            }
        });
      }
      if (tid == 0) sh.exchange[question + 1] = mine_n;
      meet();
      if (rank != 0) {
        meet();  // (the first CTA has read this one's list)
        return;
      }
      u64 unused;
      const u64 all_weight = by_weight && !by_count ? heard(question, &unused) : 0;
      int n_list = (int)mine_n;
      if constexpr (C > 1) {
        u32 end[C];
#pragma unroll
        for (u32 r = 0; r < (u32)C; ++r) end[r] = (u32)peer_u64(&sh.exchange[question + 1], r);
#pragma unroll
        for (u32 r = 1; r < (u32)C; ++r) end[r] += end[r - 1];
        n_list = (int)end[C - 1];
        if (tid >= (int)mine_n && tid < n_list) {
          u32 from = 0, first = 0;
#pragma unroll
          for (u32 r = 0; r < (u32)C - 1; ++r)
            if (tid >= (int)end[r]) from = r + 1, first = end[r];
          const u32 a = peer_u32(&sh.list_key[tid - first], from), b = peer_u32(&sh.list_at[tid - first], from);
          sh.list_key[tid] = a;
          sh.list_at[tid] = b;
        }
        meet();
      } else {
        __syncthreads();
      }
      // sorted: falling keys, equal ones by rising place
      u64* other = reinterpret_cast<u64*>(sh.count);  // [kThreads]
      u64 x = tid < n_list ? (u64)sh.list_key[tid] << 32 | (0xffffffffu - tid) : 0;
      int sorted = 32;  // threads that take part: the others hold zeros
      while (sorted < n_list) sorted *= 2;
      if (tid < sorted)
        for (int size = 2; size < 2 * n_list; size *= 2)
          for (int dist = size / 2; dist > 0; dist /= 2) {
            u64 y;
            if (dist < 32) {
              y = __shfl_xor_sync(0xffffffffu, x, dist);
            } else {
              other[tid] = x;
              asm volatile("bar.sync 1, %0;" ::"r"(sorted) : "memory");
              y = other[tid ^ dist];
              asm volatile("bar.sync 1, %0;" ::"r"(sorted) : "memory");
            }
            x = (((tid & size) == 0) == ((tid & dist) == 0)) == (x > y) ? x : y;
          }
      const int n_kept = by_count ? min(n_list, k) : n_list;
      u64 w = tid < n_kept ? weight((u32)(x >> 32)) : 0, total;
      const u64 before = block_scan(w, sh, &total);
      if (by_weight && before >= share(by_count ? total : all_weight)) w = 0;
      u64* of_place = reinterpret_cast<u64*>(sh.sums);  // [kThreads]
      if (tid < n_list) of_place[0xffffffffu - (u32)x] = w;
      __syncthreads();
      w = tid < n_list ? of_place[tid] : 0;
      const u64 from = block_scan(w, sh, &total);
      u = u > 0.f ? u : 0.f;
      u64 goal = (u64)((double)u * (double)total);
      if (goal >= total) goal = total - 1;
      if (from <= goal && from + w > goal) p.tokens[row] = (int)sh.list_at[tid];
      return;
    }
  }

  // ---- 4. more logits than that: they stay where they are
  // Radix selection, level after level, among the keys from `least` to below `sure` (above kf) in falling order: the key at which the
  // sum of `measure` reaches `goal` (1 or more), the sum in front of it, and the sum of all its equals.  False: it is not reached.
  int level = 0;
  auto select = [&](auto over, auto measure, u32 least, u32 sure, u64 goal, bool wide, u32* key, u64* front, u64* own) {
    u32 prefix = 0;
    u64 above = 0, held = 0;
    const u64 part = rf ? rf * measure(kf) : 0;  // the kept equals of kf are no elements of the histograms
    least = max(least, kf + 1);
    for (int left = K::kBits; left > 0; left -= 8) {
      const int shift = left - 8;
      u32(*limb)[kDigit] = sh.limb[level & 1];
      ++level;
      for (int i = tid; i < 3 * kDigit; i += kThreads) limb[0][i] = 0;
      __syncthreads();
      over([&](u32 s) {
        if (s < least || s >= sure || (left < K::kBits && (s >> left) != prefix)) return;
        const u64 v = measure(s);
        const u32 bin = (s >> shift) & (kDigit - 1);
        if (!wide) {
          atomicAdd(&limb[0][bin], (u32)v);
        } else {
          constexpr u32 kMask = (1u << kLimb) - 1;
          const u32 low = (u32)v & kMask, mid = (u32)(v >> kLimb) & kMask, up = (u32)(v >> (2 * kLimb));
          atomicAdd(&limb[0][bin], low);
          if (mid) atomicAdd(&limb[1][bin], mid);
          if (up) atomicAdd(&limb[2][bin], up);
        }
      });
      meet();
      // bins in falling order, one to a thread
      const int bin = kDigit - 1 - tid;
      u64 sum = 0;
      if (bin >= 0) {
#pragma unroll
        for (int w = 0; w < 3; ++w) {
          if (w > 0 && !wide) break;
          u32 a[C];
#pragma unroll
          for (u32 r = 0; r < (u32)C; ++r) a[r] = peer_u32(&limb[w][bin], r);
#pragma unroll
          for (u32 r = 0; r < (u32)C; ++r) sum += (u64)a[r] << (kLimb * w);
        }
        const u32 here = (left < K::kBits ? prefix << 8 : 0) | (u32)bin;
        if (rf && (kf >> shift) == here) sum += part;
      }
      u64 total;
      const u64 before = block_scan(sum, sh, &total);
      if (left == K::kBits && total < goal) return false;  // (the same in every CTA)
      const u64 want = goal - above;  // at least 1, and reached in this level
      if (before < want && before + sum >= want) {
        sh.found[0] = bin;
        sh.found[1] = before;
        sh.found[2] = sum;
      }
      __syncthreads();
      prefix = (left < K::kBits ? prefix << 8 : 0) | (u32)sh.found[0];
      above += sh.found[1];
      held = sh.found[2];
      __syncthreads();
    }
    *key = prefix;
    *front = above;
    *own = held;
    return true;
  };

  u32 key;
  u64 front, own;
  if (cut) {
    const u64 goal = k - front_k;
    if (select(each, [](u32) -> u64 { return 1; }, first_key(bin_k), bin_k > 0 ? first_key(bin_k - 1) : top + 1, goal, false,
               &key, &front, &own)) {
      kf = key;
      rf = (u32)(goal - front);
      equal = (u32)own;
    }
  }
  // One pass over the weights: all that is left, what is surely kept, a list of what the border decides about.
  const u32 least = by_weight ? first_key(bin_hi) : 0;
  const u32 sure = max(kf + 1, by_weight && bin_lo > 0 ? first_key(bin_lo - 1) : by_weight ? top + 1 : 0);
  const u32 low = max(least, rf ? kf : kf + 1);
  u32* owned_n = sh.sums;                           // [kThreads], by the thread whose chunk they are in: equals of the border
  u64* owned = reinterpret_cast<u64*>(sh.count);    // [kThreads] and weights that it keeps
  owned_n[tid] = 0;
  owned[tid] = 0;
  __syncthreads();
  u64 mine = 0, mine_sure = 0, total, before;
  in_order([&](const u32(&s)[4], int place) {
    bool some = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) some |= s[e] >= kf;
    if (!__any_sync(0xffffffffu, some)) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const u64 v = weight(s[e]);
      if (s[e] > kf) mine += v;
      if (s[e] >= sure)
        mine_sure += v;
      else if (s[e] >= low) {
        const u32 at = atomicAdd(&sh.listed, 1u);
        if (at < kList) sh.list_key[at] = s[e], sh.list_at[at] = place + e;
      }
    }
  });
  bool listed = true;  // no CTA's list is too short
  u64 total_sure = 0;
  if (by_weight || rf) {
    block_scan(mine, sh, &total);
    block_scan(mine_sure, sh, &total_sure);
    if (tid == 0) sh.exchange[question + 1] = total_sure, sh.exchange[question + 2] = sh.listed > kList;
    total = ask(total, &before);
    total_sure = heard(question++, &before);
    listed = heard(question++, &before) == 0;
  }
  const int n_list = (int)sh.listed;
  auto over = [&](auto f) {
    if (listed) {
      if (tid < n_list) f(sh.list_key[tid]);
    } else {
      each(f);
    }
  };
  if (by_weight) {
    const u64 reach = share(total + (rf ? rf * weight(kf) : 0));
    if (reach > total_sure && select(over, weight, least, sure, reach - total_sure, true, &key, &front, &own)) {
      const u64 w = weight(key);
      const u32 some = (u32)((reach - total_sure - front + w - 1) / w), all = (u32)(own / w);
      if (key != kf) equal = all;
      kf = key;
      rf = some;
    }
  }
  // fewer than all of the border's equals: those up to a place
  int last = 0x7fffffff;
  if (rf != 0 && rf < equal) {
    u32 equals = 0, sum;
    if (listed) {
      if (tid < n_list && sh.list_key[tid] == kf) atomicAdd(&owned_n[sh.list_at[tid] / chunk], 1u);
      __syncthreads();
      equals = owned_n[tid];
    } else {
      in_order([&](const u32(&s)[4], int) {
#pragma unroll
        for (int e = 0; e < 4; ++e) equals += s[e] == kf;
      });
    }
    const u32 at = block_scan(equals, sh, &sum);
    ask(sum, &before);
    if (tid == 0) sh.exchange[question] = 0;
    __syncthreads();
    if (before + at < rf && before + at + equals >= rf) {
      u32 need = rf - (u32)before - at;
      in_order([&](const u32(&s)[4], int place) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (s[e] == kf && --need == 0) sh.exchange[question] = (u64)(base + place + e) + 1;
      });
    }
    meet();
    u64 unused;
    last = (int)heard(question++, &unused) - 1;  // (one CTA's answer, and zeros)
  }
  // the draw, in the order of the vocabulary
  auto kept = [&](u32 s, int place) { return s > kf || (s == kf && rf != 0 && base + place <= last); };
  u64 mass = mine_sure;
  if (!by_weight && !rf) {
  } else if (listed) {
    if (tid < n_list && kept(sh.list_key[tid], (int)sh.list_at[tid]))
      atomicAdd(&owned[sh.list_at[tid] / chunk], weight(sh.list_key[tid]));
    __syncthreads();
    mass += owned[tid];
  } else {
    mass = 0;
    in_order([&](const u32(&s)[4], int place) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const u64 v = weight(s[e]);
        if (kept(s[e], place + e)) mass += v;
      }
    });
  }
  u64 at = block_scan(mass, sh, &total);
  const u64 sum = ask(total, &before);
  at += before;
  u = u > 0.f ? u : 0.f;
  u64 goal = (u64)((double)u * (double)sum);
  if (goal >= sum) goal = sum - 1;
  if (at <= goal && at + mass > goal) {
    in_order([&](const u32(&s)[4], int place) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (at > goal || !kept(s[e], place + e)) continue;
        at += weight(s[e]);
        if (at > goal) p.tokens[row] = base + place + e;
      }
    });
  }
  if constexpr (C > 1) {  // nobody leaves while another may read its memory
    __syncwarp();
    cluster_barrier();
  }
}

// Elements to a thread: an odd number of 32-bit words, so that the threads' chunks start in different banks.
template <typename L>
int chunk_of(int V, int C) {
  const int per = Keys<L>::kPerWord, words = (V + C * kThreads * per - 1) / (C * kThreads * per);
  return (words | 1) * per;
}

template <typename L, int C>
int launch_on(const Sampling& p, cudaStream_t s) {
  const int chunk = chunk_of<L>(p.V, C);
  const size_t smem = sizeof(Shared) + (size_t)kThreads * chunk * sizeof(typename Keys<L>::Stored);
  if (smem > kMaxSmem) return kErrTooLarge;
  // (the limit belongs to the kernel, not to the call: set to one call's size it would refuse another thread's launch)
  static SharedMemoryOnce once;
  if (const int rc = once.allow(sample_kernel<L, C>, kMaxSmem)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.rows * C));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, sample_kernel<L, C>, p, chunk);
}

template <typename L>
int launch(const Sampling& p, int sm_count, cudaStream_t s) {
  // As many CTAs to a row as the SMs take at once (one CTA fills one), down to 4096 logits each, and no fewer than a slice's shared
  // memory asks for.  Twice as many, in two waves, were slower wherever that is a choice, 1.15 to 2.4 times (us, this rule and those
  // in brackets, top-p alone / top-k 50 and top-p): 64 bf16 rows of 152064 66.4 / 34.0 (86.4 / 44.2), 70 67.2 / 34.0 (100.8 / 59.4);
  // 20 rows of 40000 29.1 / 16.0 (45.0 / 25.4); 100 fp32 rows of 12000 27.0 / 13.9 (43.0 / 27.9).
  const size_t row = (size_t)p.V * sizeof(typename Keys<L>::Stored);
  int C = 1;
  while (C < 8 && ((2 * p.rows * C <= sm_count && p.V / C > 4096) || row / C > kSliceBytes)) C *= 2;
  switch (C) {
    case 1: return launch_on<L, 1>(p, s);
    case 2: return launch_on<L, 2>(p, s);
    case 4: return launch_on<L, 4>(p, s);
    default: return launch_on<L, 8>(p, s);
  }
}

}  // namespace

int sample_launch(const Sampling& p, int sm_count, cudaStream_t s) {
  if (p.rows < 1 || p.V < 1 || p.stride < 0) return kErrBadShape;
  if (p.V > kMaxVocab || p.rows > (1 << 20)) return kErrTooLarge;
  if (!p.logits || !p.u || !p.tokens || misaligned(p.logits, p.fp32 ? 4 : 2) || misaligned(p.u, 4) || misaligned(p.tokens, 8) ||
      misaligned(p.temperature, 4) || misaligned(p.top_k, 4) || misaligned(p.top_p, 4) || misaligned(p.min_p, 4))
    return kErrBadPointer;
  if (sm_count < 1) return -sm_count;
  return p.fp32 ? launch<float>(p, sm_count, s) : launch<__nv_bfloat16>(p, sm_count, s);
}

}  // namespace b2
