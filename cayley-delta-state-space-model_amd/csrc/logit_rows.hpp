// Rows of logits as the operators on them read them: a row of V elements starts anywhere, so it is a head of single
// elements up to a 16-byte boundary, vectors of 16 bytes, and a tail.  Groups of W waves share a row, each wave with a
// run of the row's vectors in the row's order (the head is the first wave's, the tail the last one's).
#pragma once

#include "common.hpp"

namespace cdssm {
namespace rows {

// 16 bytes of a row as they lie in memory.
template <typename T>
struct Vec {
  static constexpr int E = 16 / T::bytes;
  uint4 u;
  __device__ __forceinline__ float get(int i) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (T::bytes == 2)
      return i & 1 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]);
    else
      return __uint_as_float(w[i]);
  }
  __device__ __forceinline__ void set(const float (&x)[E]) {
    if constexpr (T::bytes == 2)
      u = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
    else
      u = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};

// A wave's part of a row: single elements [0, head) and [tail, V), vectors [lo, hi) from element `first` on.
struct Part {
  int head, first, lo, hi, tail;
  // The element at which vector i starts.
  template <typename T>
  __device__ __forceinline__ int at(int i) const {
    return first + i * Vec<T>::E;
  }
  // Whether element i is this wave's.
  template <typename T>
  __device__ __forceinline__ bool has(int i, int V) const {
    return (i >= at<T>(lo) && i < at<T>(hi)) || i < head || (i >= tail && i < V);
  }
};

// Wave `w` of W of the row of V elements at p.
template <typename T, int W>
__device__ __forceinline__ Part part_of(const typename T::raw* p, int V, int w) {
  constexpr int E = Vec<T>::E;
  Part s;
  s.first = min(V, int(((16 - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / T::bytes));
  const int nv = (V - s.first) / E;
  const int per = (nv + W - 1) / W;
  s.lo = min(nv, w * per);
  s.hi = min(nv, s.lo + per);
  s.head = w == 0 ? s.first : 0;
  s.tail = w == W - 1 ? s.first + nv * E : V;
  return s;
}

// Entry i of a list of ids of 4 or 8 bytes; -1 for an id that 31 bits do not hold.
__device__ __forceinline__ int id_at(const void* ids, int bytes, int64_t i) {
  if (bytes == 4) return static_cast<const int*>(ids)[i];
  const int64_t v = static_cast<const int64_t*>(ids)[i];
  return v < 0 || v > 0x7fffffffLL ? -1 : int(v);
}

}  // namespace rows
}  // namespace cdssm
