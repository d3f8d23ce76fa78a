// Which keys the rows of a sequence see, as the attention kernels walk over them: blocks of KEYS keys, first those that hold
// first tokens that stay visible, then those from the first row's window on.
#pragma once
#include "paged.cuh"

namespace b2 {

struct Mask {
  int window, sinks;  // window 0: no window
  int flat;           // > 0: one sequence of that many rows, which see every key (a shared prefix)
};

struct Visible {
  int first, rows;   // first row of the call, number of rows (tokens)
  int end;           // keys behind the last one that has a page in the table
  int pmin, pmax;    // positions of the first and the last row
  int n_sink, from, count;  // blocks: n_sink from key 0 on, then those from block `from` on; count in all

  template <int KEYS>
  __device__ __forceinline__ void set(const Mask& m, int len, int width_keys) {
    end = max(0, min(len, width_keys));
    if (m.flat) {
      pmin = pmax = end - 1;
    } else {
      pmin = len - rows;
      pmax = len - 1;
    }
    span<KEYS>(m);
  }
  // The blocks that rows at positions pmin .. pmax see.
  template <int KEYS>
  __device__ __forceinline__ void span(const Mask& m) {
    const int last = min(end, pmax + 1);
    const int lo = m.window > 0 ? max(0, pmin - m.window + 1) : 0;
    from = lo / KEYS;
    n_sink = m.window > 0 ? min((max(0, min(m.sinks, last)) + KEYS - 1) / KEYS, from) : 0;
    count = n_sink + max(0, (last + KEYS - 1) / KEYS - from);
  }
  __device__ __forceinline__ int block(int i) const { return i < n_sink ? i : from + i - n_sink; }
  __device__ __forceinline__ bool sees(const Mask& m, int j, int p) const {
    return j < end && j <= p && (m.window == 0 || j > p - m.window || j < m.sinks);
  }
  // Whether some row sees key j; whether every row sees all keys j .. j + n - 1.
  __device__ __forceinline__ bool any(const Mask& m, int j) const {
    return j < end && j <= pmax && (m.window == 0 || j > pmin - m.window || j < m.sinks);
  }
  __device__ __forceinline__ bool all(const Mask& m, int j, int n) const {
    return j + n <= end && j + n - 1 <= pmin && (m.window == 0 || j > pmax - m.window || j + n <= m.sinks);
  }
};

}  // namespace b2
