// b2_sample: one token per row of logits l, drawn with a given random number u in [0, 1).
//
//   w_i = e^{(l_i - max l) / T}                                   (T <= 0: the largest logit, lowest index)
//   A   = the top_k largest of {i : w_i >= min_p}                 (equal logits: the lowest index first)
//   B   = the shortest prefix of A, in falling order, whose weight reaches top_p of A's
//   token = the first i of B, in the order of the vocabulary, with  sum_{j <= i, j in B} w_j > u * sum_{j in B} w_j
//
// Both borders and the draw are exact questions about sums over up to 2^18 terms, so weights are formed in 64 bits and added up
// as whole multiples of 2^-44: the sums do not depend on the order of the additions, and not on how a row is cut up.
// (In 32 bits one draw in a few hundred ended on a neighbouring token.)
//
// A row is read once: a cluster of C CTAs keeps it in shared memory as sortable keys.  The borders are found by radix
// selection on the keys (11 bits at a time; bf16 has 16, fp32 32): a histogram of counts for top_k and of weights for
// top_p per CTA, added up over the cluster through distributed shared memory by every CTA for itself.
#include <algorithm>

#include "paged.cuh"
#include "ptx.cuh"
#include "w4_internal.h"

namespace b2 {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxVocab = 1 << 18;
constexpr int kSliceBytes = 160 * 1024;
constexpr double kOne = 17592186044416.0;  // 2^44: a weight of 1

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

struct Shared {
  u32 lo[2][kBins], hi[2][kBins];  // a histogram (counts: lo alone), two in turn: peers may still read the other
  u64 exchange[8];                 // what this CTA tells the others, a place per question
  u64 scan[kWarps + 1];
  u64 found[3];
};

__device__ __forceinline__ uint4 peer_u4(const u32* p, u32 rank) {
  uint4 v;
  asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [a];\n\t}"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(smem_u32(p)), "r"(rank) : "memory");
  return v;
}
__device__ __forceinline__ u64 peer_u64(const u64* p, u32 rank) {
  u64 v;
  asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.u64 %0, [a];\n\t}"
               : "=l"(v) : "r"(smem_u32(p)), "r"(rank) : "memory");
  return v;
}

// Sum of v over the threads in front of the calling one; total: over all.
__device__ __forceinline__ u64 block_scan(u64 v, u64* scan, u64* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) scan[warp] = x;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const u64 y = scan[w];
    if (w < warp) before += y;
    all += y;
  }
  *total = all;
  return before + x - v;
}

template <typename L, int C>
__global__ void __launch_bounds__(kThreads) sample_kernel(const Sampling p, int chunk) {
  using K = Keys<L>;
  using Stored = typename K::Stored;
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  Stored* keys = reinterpret_cast<Stored*>(raw + sizeof(Shared));
  const int tid = threadIdx.x;
  const u32 rank = blockIdx.x % C;
  const int row = (int)(blockIdx.x / C);
  const int slice = kThreads * chunk, base = rank * slice;  // this CTA's logits: [base, base + slice), a chunk per thread
  const int n = max(0, min(p.V - base, slice));
  const Stored* mine = keys + tid * chunk;
  int question = 0;
  // Everybody's answer to the next question, added up (or the largest); what the CTAs in front of this one said: before.
  auto ask = [&](u64 v, u64* before) {
    if (tid == 0) sh.exchange[question] = v;
    cluster_barrier();
    u64 told[C], sum = 0;
#pragma unroll
    for (u32 r = 0; r < (u32)C; ++r) told[r] = peer_u64(&sh.exchange[question], r);
    *before = 0;
#pragma unroll
    for (u32 r = 0; r < (u32)C; ++r) {
      if (r == rank) *before = sum;
      sum += told[r];
    }
    ++question;
    return sum;
  };

  // ---- the row's slice as keys, and the largest
  const L* src = static_cast<const L*>(p.logits) + row * p.stride + base;
  u32 top = 0;
  constexpr int kVec = 16 / sizeof(L);
  const int vectors = (reinterpret_cast<uintptr_t>(src) & 15) == 0 ? n / kVec : 0;
  for (int i = tid; i < vectors; i += kThreads) {
    const uint4 x = __ldcg(reinterpret_cast<const uint4*>(src) + i);
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
  }
  for (int i = vectors * kVec + tid; i < slice; i += kThreads) {
    const u32 k = i < n ? key_of(K::load(src, i)) : 0;
    keys[i] = (Stored)K::stored(k);
    top = max(top, K::stored(k));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (tid == 0) sh.found[0] = 0;
  __syncthreads();
  if ((tid & 31) == 0) atomicMax(&sh.found[0], (u64)top);
  __syncthreads();
  if (tid == 0) sh.exchange[question] = sh.found[0];
  cluster_barrier();
  top = 0;
#pragma unroll
  for (u32 r = 0; r < (u32)C; ++r) top = max(top, (u32)peer_u64(&sh.exchange[question], r));
  ++question;
  const float largest = K::logit(top);
  if (largest == __uint_as_float(0xff800000u)) top = 0;  // nothing but minus infinity

  float T = p.temperature ? __ldcg(p.temperature + row) : p.temperature_all;
  int k = p.top_k ? __ldcg(p.top_k + row) : p.top_k_all;
  const float top_p = p.top_p ? __ldcg(p.top_p + row) : p.top_p_all;
  const float min_p = p.min_p ? __ldcg(p.min_p + row) : p.min_p_all;
  if (!(T > 0.f)) k = 1, T = 1.f;
  if (k <= 0 || k > p.V) k = p.V;
  const double per_T = 1.0 / (double)T;
  // (a weight of e^-31.5 is under half of 2^-44; keys below this one need not be asked)
  const u32 nothing = K::stored(key_of(largest - 40.f * T));
  // the weight of a stored key, in multiples of 2^-44
  auto weight = [&](u32 s) -> u64 {
    if (s == top) return (u64)kOne;
    if (s < nothing) return 0;
    const double x = ((double)K::logit(s) - (double)largest) * per_T;
    return x < -31.5 ? 0 : (u64)rint(exp(x) * kOne);  // (not finite: below, or nan, which compares false and converts to 0)
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

  // Radix selection, level after level, among the kept keys in falling order: the key at which the sum of `measure` reaches
  // `target(total)`, the sum in front of it, and the sum of all its equals.  False: it is not reached.
  int level = 0;
  auto select = [&](auto measure, auto target, bool wide, u32* key, u64* front, u64* own) {
    u32 prefix = 0;
    u64 goal = 0, above = 0, held = 0;
    const u64 part = rf ? rf * measure(kf) : 0;  // the kept equals of kf are no elements of the histograms
    int left = K::kBits;
    for (int l = 0; left > 0; ++l) {
      const int bits = min(left, 11), shift = left - bits;
      u32 *lo = sh.lo[level & 1], *hi = sh.hi[level & 1];
      ++level;
      for (int i = tid; i < kBins / 4; i += kThreads) {
        reinterpret_cast<uint4*>(lo)[i] = make_uint4(0, 0, 0, 0);
        reinterpret_cast<uint4*>(hi)[i] = make_uint4(0, 0, 0, 0);
      }
      __syncthreads();
      for (int i = 0; i < chunk; ++i) {
        const u32 s = mine[i];
        if (s <= kf || (l > 0 && (s >> left) != prefix)) continue;
        const u64 v = measure(s);
        if (v == 0) continue;
        const u32 bin = (s >> shift) & ((1u << bits) - 1), x = (u32)v;
        const u32 old = atomicAdd(&lo[bin], x);
        if (wide) {
          const u32 up = (u32)(v >> 32) + (old + x < old);
          if (up) atomicAdd(&hi[bin], up);
        }
      }
      cluster_barrier();
      // bins in falling order, four to a thread: bins top_bin - 3 .. top_bin
      constexpr int kEach = 4;
      static_assert(kBins == kEach * kThreads, "a thread reads its bins at once");
      const int top_bin = (1 << bits) - 1 - tid * kEach;
      u64 sum[kEach] = {}, mass = 0;
      if (top_bin > 0) {
        uint4 a[C], c[C];
#pragma unroll
        for (u32 r = 0; r < (u32)C; ++r) {
          a[r] = peer_u4(&lo[top_bin - 3], r);
          c[r] = wide ? peer_u4(&hi[top_bin - 3], r) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (u32 r = 0; r < (u32)C; ++r) {
          sum[0] += a[r].w + ((u64)c[r].w << 32);
          sum[1] += a[r].z + ((u64)c[r].z << 32);
          sum[2] += a[r].y + ((u64)c[r].y << 32);
          sum[3] += a[r].x + ((u64)c[r].x << 32);
        }
        if (rf) {
          const u32 first = (l > 0 ? prefix << bits : 0) | (u32)top_bin, at = first - (kf >> shift);
          if (at < kEach) {
#pragma unroll
            for (int e = 0; e < kEach; ++e)
              if (at == (u32)e) sum[e] += part;
          }
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) mass += sum[e];
      }
      u64 total;
      u64 before = block_scan(mass, sh.scan, &total);
      if (l == 0) {
        goal = target(total);
        if (total < goal || goal == 0) return false;  // (the same in every CTA)
      }
      const u64 want = goal - above;  // at least 1, and reached in this level
      if (before < want && before + mass >= want) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          if (before < want && before + sum[e] >= want) {
            sh.found[0] = top_bin - e;
            sh.found[1] = before;
            sh.found[2] = sum[e];
          }
          before += sum[e];
        }
      }
      __syncthreads();
      prefix = l > 0 ? (prefix << bits) | (u32)sh.found[0] : (u32)sh.found[0];
      above += sh.found[1];
      held = sh.found[2];
      left = shift;
      __syncthreads();
    }
    *key = prefix;
    *front = above;
    *own = held;
    return true;
  };

  u32 key;
  u64 front, own;
  if (top != 0 && k < p.V) {
    // (goal k: the k-th key in falling order)
    if (select([](u32) -> u64 { return 1; }, [&](u64 total) { return total < (u64)k ? 0 : (u64)k; }, false, &key, &front, &own)) {
      kf = key;
      rf = (u32)(k - front);
      equal = (u32)own;
    }
  }
  if (top != 0 && !(top_p >= 1.f)) {
    u64 reach = 0;
    auto goal = [&](u64 total) {
      const double g = ceil((double)(top_p > 0.f ? top_p : 0.f) * (double)total);
      return reach = g < 1.0 ? 1 : (u64)g > total ? total : (u64)g;
    };
    if (select(weight, goal, true, &key, &front, &own)) {
      const u64 w = weight(key);
      const u32 some = (u32)((reach - front + w - 1) / w), all = (u32)(own / w);
      if (key != kf) equal = all;
      kf = key;
      rf = some;
    }
  }
  // fewer than all of the border's equals: those up to an index
  int last = 0x7fffffff;
  if (rf != 0 && rf < equal) {
    u64 mine_n = 0, total, before;
    for (int i = 0; i < chunk; ++i) mine_n += mine[i] == kf;
    const u64 at = block_scan(mine_n, sh.scan, &total);
    ask(total, &before);
    if (tid == 0) sh.exchange[question] = 0;
    __syncthreads();
    if (before + at < rf && before + at + mine_n >= rf) {
      u64 need = rf - before - at;
      for (int i = 0; i < chunk; ++i)
        if (mine[i] == kf && --need == 0) sh.exchange[question] = (u64)(base + tid * chunk + i) + 1;
    }
    cluster_barrier();
    for (u32 r = 0; r < (u32)C; ++r) {
      const u64 e = peer_u64(&sh.exchange[question], r);
      if (e) last = (int)e - 1;
    }
    ++question;
  }
  // ---- the draw, in the order of the vocabulary
  const int first = base + tid * chunk;
  auto kept = [&](int i, u32 s) { return s > kf || (s == kf && rf != 0 && first + i <= last); };
  u64 mass = 0, total, before;
  for (int i = 0; i < chunk; ++i) {
    const u32 s = mine[i];
    if (kept(i, s)) mass += weight(s);
  }
  u64 at = block_scan(mass, sh.scan, &total);
  const u64 sum = ask(total, &before);
  at += before;
  float u = __ldcg(p.u + row);
  u = u > 0.f ? u : 0.f;
  u64 goal = (u64)((double)u * (double)sum);
  if (goal >= sum) goal = sum - 1;
  if (sum == 0) {
    if (rank == 0 && tid == 0) p.tokens[row] = -1;  // nothing to draw from
  } else if (at <= goal && at + mass > goal) {
    for (int i = 0; i < chunk; ++i) {
      const u32 s = mine[i];
      if (!kept(i, s)) continue;
      at += weight(s);
      if (at > goal) {
        p.tokens[row] = first + i;
        break;
      }
    }
  }
  cluster_barrier();  // nobody leaves while another may read its memory
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
  if (smem > 227 * 1024) return kErrTooLarge;
  cudaError_t e = cudaFuncSetAttribute(sample_kernel<L, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
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
int launch(const Sampling& p, cudaStream_t s) {
  const size_t row = (size_t)p.V * sizeof(typename Keys<L>::Stored);
  int C = 1;
  while (C < 8 && (p.rows * C < 148 || row / C > kSliceBytes)) C *= 2;
  switch (C) {
    case 1: return launch_on<L, 1>(p, s);
    case 2: return launch_on<L, 2>(p, s);
    case 4: return launch_on<L, 4>(p, s);
    default: return launch_on<L, 8>(p, s);
  }
}

}  // namespace

int sample_launch(const Sampling& p, cudaStream_t s) {
  if (p.rows < 1 || p.V < 1 || p.stride < 0) return kErrBadShape;
  if (p.V > kMaxVocab || p.rows > (1 << 20)) return kErrTooLarge;
  if (!p.logits || !p.u || !p.tokens || misaligned(p.logits, p.fp32 ? 4 : 2) || misaligned(p.u, 4) || misaligned(p.tokens, 8) ||
      misaligned(p.temperature, 4) || misaligned(p.top_k, 4) || misaligned(p.top_p, 4) || misaligned(p.min_p, 4))
    return kErrBadPointer;
  return p.fp32 ? launch<float>(p, s) : launch<__nv_bfloat16>(p, s);
}

}  // namespace b2
