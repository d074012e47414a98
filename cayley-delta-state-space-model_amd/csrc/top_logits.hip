// The k largest logits of every row with their ids, largest first, of equal ones the lowest id first: what a teacher's run
// keeps of its logits for distillation_loss, and the candidates of a decode step.
//
// A logit and its id make one whole number that orders them: the float's bits, turned so that they grow with the value, above
// the id's complement.  A wave goes through its part of a row in order with the k best so far in registers, sorted over the
// lanes, and passes over whatever is not above the last of them.  What is goes to a buffer in LDS, and 64 of
// those are sorted by exchanges between lanes and merged into the best.  So that few pass at the beginning, the first bound
// comes from the lanes' own maxima over the first vectors: at least k elements are no less than the k-th largest of those.  Where W
// waves share a row, at least k are no less than the least of their ceil(k / W)-th largest.
// No element's order in memory, and no number of equal ones, changes more than the time.
//
// Bound by memory where there are many rows: MI355X, 8192 x 50257 bf16, 32 kept 151 us (823 MB, 5.5 TB/s), 16384 x 32000 190
// (5.5 TB/s).  Few rows are one chain: launch, load, sort of the maxima, sort, four merges, 9.2 us for 64 x 32000.  Exchanges between
// lanes through the vector unit's permutations and swaps instead of LDS took 8192 x 50257 from 173 to 157, passing over a vector of
// every lane at once to 151.
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "logit_rows.hpp"

namespace cdssm {
namespace top {

using namespace rows;

constexpr int kMaxK = 2 * kWave;

// A wave's buffer: 63 that wait, and what a vector of every lane may add.
template <typename T>
constexpr int kBuffer = kWave * (1 + Vec<T>::E);

// Bits that grow with the value.  -0 counts as 0; every NaN counts as the largest value.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b ^ (uint32_t(int(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu)); }

__device__ __forceinline__ uint64_t key_of(float x, int i) { return uint64_t(order_of(x)) << 32 | uint32_t(~i); }

// x of lane ^ M, for the masks that a sorting network of 64 lanes takes, without LDS: permutations within rows of 16 lanes, swaps of
// rows and of halves of the wave.
template <int M>
__device__ __forceinline__ uint32_t from_lane_xor(uint32_t x, int lane) {
  const auto dpp = [](uint32_t v, auto c) {
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), decltype(c)::value, 0xF, 0xF, true));
  };
  using std::integral_constant;
  if constexpr (M == 1) return dpp(x, integral_constant<int, 0xB1>{});                    // quad_perm [1, 0, 3, 2]
  if constexpr (M == 2) return dpp(x, integral_constant<int, 0x4E>{});                    // quad_perm [2, 3, 0, 1]
  if constexpr (M == 3) return dpp(x, integral_constant<int, 0x1B>{});                    // quad_perm [3, 2, 1, 0]
  if constexpr (M == 7) return dpp(x, integral_constant<int, 0x141>{});                   // row_half_mirror
  if constexpr (M == 4) return from_lane_xor<3>(from_lane_xor<7>(x, lane), lane);
  if constexpr (M == 8) return dpp(x, integral_constant<int, 0x128>{});                   // row_ror 8
  if constexpr (M == 15) return dpp(x, integral_constant<int, 0x140>{});                  // row_mirror
  if constexpr (M == 16) {
    const auto s = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return lane & 16 ? s[0] : s[1];
  }
  if constexpr (M == 32) {
    const auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return lane & 32 ? s[0] : s[1];
  }
  if constexpr (M == 31) return from_lane_xor<16>(from_lane_xor<15>(x, lane), lane);
  if constexpr (M == 63) return from_lane_xor<32>(from_lane_xor<31>(x, lane), lane);
}
template <int M>
__device__ __forceinline__ uint64_t from_lane_xor(uint64_t x, int lane) {
  return uint64_t(from_lane_xor<M>(uint32_t(x >> 32), lane)) << 32 | from_lane_xor<M>(uint32_t(x), lane);
}
template <int M>
__device__ __forceinline__ float from_lane_xor(float x, int lane) {
  return __uint_as_float(from_lane_xor<M>(__float_as_uint(x), lane));
}

// Element e = 64 r + lane of a list of 64 R.  Steps of a sorting network: of lanes that differ in M, the one whose bit H is
// clear takes the larger.
template <int M, int H, typename V>
__device__ __forceinline__ V exchange(V x, int lane) {
  const V y = from_lane_xor<M>(x, lane);
  return (x > y) == ((lane & H) == 0) ? x : y;
}

// Sorts what falls and rises once over blocks of 2 J lanes, the larger first.
template <int J, typename V>
__device__ __forceinline__ V sort_bitonic(V x, int lane) {
  x = exchange<J, J>(x, lane);
  if constexpr (J > 1) x = sort_bitonic<J / 2>(x, lane);
  return x;
}

// Sorts the 64 lanes' values, largest in lane 0: blocks of N lanes, two halves that are sorted already.
template <int N = 2, typename V>
__device__ __forceinline__ V sort64(V x, int lane) {
  x = exchange<N - 1, N / 2>(x, lane);  // each with its mirror image: the larger ones in the first half
  if constexpr (N > 2) x = sort_bitonic<N / 4>(x, lane);
  if constexpr (N < kWave) x = sort64<2 * N>(x, lane);
  return x;
}

// The best 64 R of two lists, both sorted: the larger of each element and the other list's at the same place from behind
// are them, in an order that falls and rises once; log2 steps sort it.
template <int R>
__device__ __forceinline__ void merge(uint64_t (&best)[R], const uint64_t (&other)[R], int lane) {
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint64_t y = from_lane_xor<kWave - 1>(other[R - 1 - r], lane);
    if (y > best[r]) best[r] = y;
  }
  if constexpr (R == 2) {
    const uint64_t a = best[0], b = best[1];
    best[0] = a > b ? a : b;
    best[1] = a > b ? b : a;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) best[r] = sort_bitonic<kWave / 2>(best[r], lane);
}

// A wave's search.
template <int R>
struct Search {
  uint64_t best[R];
  uint64_t* buf;  // this wave's own
  int lane, k, n;
  float bound;    // elements not above it are passed over; NaN: none is

  __device__ __forceinline__ void init(uint64_t* b, int l, int kk) {
#pragma unroll
    for (int r = 0; r < R; ++r) best[r] = 0;
    buf = b;
    lane = l;
    k = kk;
    n = 0;
    bound = __uint_as_float(0x7fc00000u);
  }

  // Other lanes' entries of the buffer are read only behind their writes, and the other way round (LDS itself keeps a
  // wave's order).
  __device__ __forceinline__ void meet() const {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  // The last min(n, 64) of the buffer into the best.
  __device__ __forceinline__ void flush() {
    const int from = max(0, n - kWave);
    meet();
    uint64_t other[R] = {};
    other[0] = sort64(from + lane < n ? buf[from + lane] : 0, lane);
    meet();
    n = from;
    merge<R>(best, other, lane);
    const uint32_t last = __builtin_amdgcn_readlane(uint32_t(best[R - 1] >> 32), (k - 1) % kWave);
    if (last) bound = value_of(last);
  }

  __device__ __forceinline__ void add(float x, int i, bool there) {
    const bool in = there && !(x <= bound);
    const uint64_t m = __ballot(in);
    if (m == 0) return;
    if (in) buf[n + __popcll(m & ((uint64_t(1) << lane) - 1))] = key_of(x, i);
    n += __popcll(m);
  }
  __device__ __forceinline__ void drain() {
    while (n >= kWave) flush();
  }
};

// k-th largest of 64 R values, one a lane and register, or a little less.
template <int R>
__device__ __forceinline__ float lower_bound(const float (&m)[R], int k, int lane) {
  float b = INFINITY;
#pragma unroll
  for (int r = 0; r < R; ++r) b = fminf(b, __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sort64(m[r], lane)), (k + R - 1) / R - 1)));
  return b;
}

// The largest float below b (for 0: below -0 too); NaN for -inf.
__device__ __forceinline__ float below(float b) {
  const uint32_t o = order_of(b);
  return value_of(o - (o == 0x80000000u ? 2u : 1u));
}

// W waves to a row, W * Rows waves to a workgroup.
template <typename T, int R, int W, int Rows>
__global__ __launch_bounds__(kWave* W* Rows) void top_kernel(const typename T::raw* __restrict__ X, int64_t ld,
                                                             typename T::raw* __restrict__ values, int64_t* __restrict__ ids,
                                                             int64_t n_rows, int V, int k) {
  constexpr int E = Vec<T>::E, U = 4;  // vectors of a lane under way at once
  __shared__ uint64_t lds[W * Rows][kBuffer<T>];
  __shared__ float bounds[W];
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave), lane = int(threadIdx.x) % kWave;
  const int64_t t = int64_t(blockIdx.x) * Rows + wave / W;
  if (t >= n_rows) return;  // with Rows > 1 no workgroup meets at a barrier
  const int w = wave % W;
  const typename T::raw* row = X + t * ld;
  const Part s = part_of<T, W>(row, V, w);
  const uint4* vec = reinterpret_cast<const uint4*>(row + s.first);
  Search<R> f;
  f.init(lds[wave], lane, k);
  Vec<T> v[U];
  const auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kWave + lane;
      if (i < s.hi) v[u].u = vec[i];
    }
  };
  load(s.lo);
  const float head = lane < s.head ? T::load(row + lane) : 0.0f, tail = s.tail + lane < V ? T::load(row + s.tail + lane) : 0.0f;
  {
    float m[R];
#pragma unroll
    for (int r = 0; r < R; ++r) m[r] = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s.lo + u * kWave + lane < s.hi)
#pragma unroll
        for (int e = 0; e < E; ++e) m[u % R] = fmaxf(m[u % R], v[u].get(e));
    float b = lower_bound<R>(m, (k + W - 1) / W, lane);
    if constexpr (W > 1) {
      if (lane == 0) bounds[w] = b;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < W; ++i) b = fminf(b, bounds[i]);
    }
    f.bound = below(b);
  }
  if (s.head > 0) f.add(head, lane, lane < s.head);
  for (int i0 = s.lo; i0 < s.hi; i0 += U * kWave) {
    if (i0 > s.lo) load(i0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kWave + lane;
      const bool there = i < s.hi;
      bool any = false;
#pragma unroll
      for (int e = 0; e < E; ++e) any |= !(v[u].get(e) <= f.bound);
      if (__ballot(there && any) == 0) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) f.add(v[u].get(e), s.at<T>(i) + e, there);
      f.drain();
    }
  }
  if (s.tail < V) {
    const int i = s.tail + lane;
    f.add(tail, i, i < V);
  }
  while (f.n > 0) f.flush();
  if constexpr (W > 1) {
    // the waves' lists, two by two (the buffers of 64 R keys hold them)
#pragma unroll
    for (int d = 1; d < W; d *= 2) {
      __syncthreads();
      if (w % (2 * d) == d)
#pragma unroll
        for (int r = 0; r < R; ++r) lds[wave][r * kWave + lane] = f.best[r];
      __syncthreads();
      if (w % (2 * d) == 0) {
        uint64_t other[R];
#pragma unroll
        for (int r = 0; r < R; ++r) other[r] = lds[wave + d][r * kWave + lane];
        merge<R>(f.best, other, lane);
      }
    }
    if (w != 0) return;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int e = r * kWave + lane;
    if (e < k) {
      const int i = int(~uint32_t(f.best[r]));
      const uint32_t o = uint32_t(f.best[r] >> 32);
      ids[t * k + e] = i;
      if (o == 0xffffffffu || o == 0x80000000u)
        values[t * k + e] = row[i];  // which NaN, and the sign of 0, are not in the order
      else
        T::store(values + t * k + e, value_of(o));
    }
  }
}

template <typename T, int R>
static void launch(const void* X, int64_t ld, void* values, int64_t* ids, int64_t n, int64_t V, int64_t k, hipStream_t stream) {
  using raw = typename T::raw;
  const auto* x = static_cast<const raw*>(X);
  auto* v = static_cast<raw*>(values);
  auto go = [&](auto wc, auto rc) {
    constexpr int W = decltype(wc)::value, Rows = decltype(rc)::value;
    hipLaunchKernelGGL((top_kernel<T, R, W, Rows>), dim3(unsigned((n + Rows - 1) / Rows)), dim3(kWave * W * Rows), 0, stream, x,
                       ld, v, ids, n, int(V), int(k));
  };
  using std::integral_constant;
  // Some 8192 waves fill the device; a wave's part of a row is worth its search from 1024 elements on.  us with 1 / 2 / 4 / 8 / 16
  // waves to a row, bf16, 32 (50) of a row kept: 64 x 32000 41 / 25 / 15 / 9.7 / 9.2, 512 x 32000 45 / 29 / 17 / 12.2 / 14.3
  // (not its best by a sixth), 2048 x 32000 50 / 35 / 30 / 31 / 43, 8192 x 50257 151 / 172 / 156 / 163 / 219, 2048 x 300 fp32 5.3 / 6.0 / 8.7 / 16 / 33.
  int w = 1;
  while (w < 16 && 2 * w * n <= 8192 && V >= 2 * w * 1024) w *= 2;
  w == 16  ? go(integral_constant<int, 16>{}, integral_constant<int, 1>{})
  : w == 8 ? go(integral_constant<int, 8>{}, integral_constant<int, 1>{})
  : w == 4 ? go(integral_constant<int, 4>{}, integral_constant<int, 1>{})
  : w == 2 ? go(integral_constant<int, 2>{}, integral_constant<int, 1>{})
           : go(integral_constant<int, 1>{}, integral_constant<int, 4>{});
}

}  // namespace top
}  // namespace cdssm

using namespace cdssm;

// values, ids (T, k): the k largest of each row of logits (T, V; row stride ld) and where they stand, as described above.
extern "C" int cdssm_top_logits(int dtype, const void* logits, int64_t ld, void* values, int64_t* ids, int64_t T, int64_t V,
                                int64_t k, hipStream_t stream) {
  const char* op = "cdssm_top_logits";
  if (dtype != 0 && dtype != 1) {
    cdssm_host::set_error("%s: dtype must be 0 (fp32) or 1 (bf16), got %d", op, dtype);
    return CDSSM_EINVAL;
  }
  if (!logits || !values || !ids) {
    cdssm_host::set_error("%s: null pointer argument", op);
    return CDSSM_EINVAL;
  }
  if (T < 1 || T > (int64_t(1) << 24) || V < 1 || V > (int64_t(1) << 24) || k < 1 || k > top::kMaxK || k > V) {
    cdssm_host::set_error("%s: needs 1 <= T, V <= 2^24 and 1 <= k <= min(V, %d), got T %lld, V %lld, k %lld", op, top::kMaxK,
                          (long long)T, (long long)V, (long long)k);
    return CDSSM_EINVAL;
  }
  if (ld < V || ld > (int64_t(1) << 32) || reinterpret_cast<uintptr_t>(logits) % (dtype ? 2 : 4) ||
      reinterpret_cast<uintptr_t>(values) % (dtype ? 2 : 4) || reinterpret_cast<uintptr_t>(ids) % 8) {
    cdssm_host::set_error("%s: the row stride must be within V .. 2^32 and the tensors aligned to their elements", op);
    return CDSSM_EINVAL;
  }
  if (k <= kWave)
    dtype ? top::launch<BF16, 1>(logits, ld, values, ids, T, V, k, stream)
          : top::launch<F32, 1>(logits, ld, values, ids, T, V, k, stream);
  else
    dtype ? top::launch<BF16, 2>(logits, ld, values, ids, T, V, k, stream)
          : top::launch<F32, 2>(logits, ld, values, ids, T, V, k, stream);
  return cdssm_host::check_launch(op);
}
