// Token embedding: y[t] = scale W[ids[t]] (model.py:37-40), and the table's gradient
//   dW[v] = scale sum over t with ids[t] = v of dy[t]        (the padding row: 0)
// with the tokens sorted by id, so that every row of dW is summed by one wave in a fixed order (fp32) and written
// once, zeros included: no atomics, the same bits every time.
//
// Sort (token_sort.hpp): by the first workgroups of a training forward's launch, or in a launch of the backward's own.
// Sum: where an id fills whole chunks of kChunk sorted tokens, a wave per chunk sums those first (an id as frequent
// as 1 in 12 would else be one wave's long work); then a wave per row of dW and 64 vectors of columns.
//
// Bound by memory: MI355X, 16384 tokens of text-like frequency, 32000 x 1024 bf16: forward 12 us (67 MB, 5.4 TB/s), with the
// sort 18; chunks 6, rows 18 (99 MB, 5.5 TB/s).  In fp32, 9995 tokens, 50257 x 768: 13, 17; 7, 34.  The sort alone takes
// 10, a chain of waits (ids from L2, LDS counts, places), which in the forward hides behind the rows.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.hpp"
#include "token_sort.hpp"

namespace cdssm {
namespace emb {

using namespace token_sort;

constexpr int kChunk = 32;

// VEC elements next to each other, loaded and stored at once.
template <typename T, int VEC>
struct Vec {
  static constexpr int bytes = VEC * T::bytes;
  uint32_t u[bytes < 4 ? 1 : bytes / 4];
  __device__ __forceinline__ void load(const typename T::raw* p) {
    if constexpr (bytes == 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      u[0] = v.x; u[1] = v.y; u[2] = v.z; u[3] = v.w;
    } else if constexpr (bytes == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      u[0] = v.x; u[1] = v.y;
    } else if constexpr (bytes == 4) {
      u[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      u[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ void store(typename T::raw* p) const {
    if constexpr (bytes == 16)
      *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    else if constexpr (bytes == 8)
      *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
    else if constexpr (bytes == 4)
      *reinterpret_cast<uint32_t*>(p) = u[0];
    else
      *reinterpret_cast<uint16_t*>(p) = uint16_t(u[0]);
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (T::bytes == 2)
      return i & 1 ? bf16_hi(u[i / 2]) : bf16_lo(u[i / 2]);
    else
      return __uint_as_float(u[i]);
  }
  __device__ __forceinline__ void set(const float* x) {
    if constexpr (T::bytes == 2) {
      if constexpr (VEC == 1)
        u[0] = f32_to_bf16(x[0]);
      else
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) u[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) u[i] = __float_as_uint(x[i]);
    }
  }
};

// The wave's place in the launch, two-dimensional where one dimension would pass 2^32 threads; `before` workgroups do other work.
template <int Waves = 4>
__device__ __forceinline__ int64_t wave_place(int before = 0) {
  return (int64_t(blockIdx.y) * gridDim.x + blockIdx.x - before) * Waves + threadIdx.x / kWave;
}

// A wave's place as a scalar, so that what it looks up comes through scalar loads.
__device__ __forceinline__ int64_t scalar(int64_t x) { return int64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(x)))); }

// Wave w's part of the rows: a wave per token and 64 vectors of columns.  An id out of range gives a row of NaN and reads nothing.
template <typename T, typename I, int VEC>
__device__ __forceinline__ void gather(int64_t w, const I* __restrict__ ids, const typename T::raw* __restrict__ W, int64_t ldw,
                                       float scale, typename T::raw* __restrict__ y, int64_t n, int64_t V, int64_t C) {
  const int64_t per = (C + kWave * VEC - 1) / (kWave * VEC), t = scalar(w / per);
  if (t >= n) return;
  const int64_t c = ((w - t * per) * kWave + threadIdx.x % kWave) * VEC;
  if (c >= C) return;
  const int64_t id = int64_t(ids[t]);
  Vec<T, VEC> v;
  float x[VEC];
  if (id >= 0 && id < V) {
    v.load(W + id * ldw + c);
    if (scale != 1.0f) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = v.get(i) * scale;
      v.set(x);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = NAN;
    v.set(x);
  }
  v.store(y + t * C + c);
}

template <typename T, typename I, int VEC>
__global__ __launch_bounds__(256) void gather_kernel(const I* __restrict__ ids, const typename T::raw* __restrict__ W, int64_t ldw,
                                                     float scale, typename T::raw* __restrict__ y, int64_t n, int64_t V,
                                                     int64_t C) {
  gather<T, I, VEC>(wave_place(), ids, W, ldw, scale, y, n, V, C);
}

// Where the order's parts lie; with two levels `buckets` is not null, and the first leaves its order in `tokens`.
struct Order {
  int* order;
  int2* rows;
  int* tokens;
  int2* buckets;
  int bits;  // log2 of the workgroups of a single level, else of the buckets
};

// The first launch of a sort; workgroups from sorters() on have no part in it.
template <bool Two, typename I>
__device__ __forceinline__ void sort_first(const Order& o, const I* ids, int64_t T, int64_t V, int64_t padding) {
  if constexpr (Two)
    sort_buckets(ids, o.tokens, o.buckets, int(T), V, padding, o.bits);
  else
    sort(ids, o.order, o.rows, int(T), V, padding, o.bits);
}
template <bool Two>
__host__ __device__ __forceinline__ int sorters(const Order& o) {
  return Two ? 256 : 1 << o.bits;
}

template <bool Two, typename I>
__global__ __launch_bounds__(kSortThreads) void sort_kernel(const I* __restrict__ ids, Order o, int64_t T, int64_t V,
                                                            int64_t padding) {
  sort_first<Two>(o, ids, T, V, padding);
}

template <typename I>
__global__ __launch_bounds__(kSortThreads) void sort_bucket_kernel(const I* __restrict__ ids, Order o, int64_t V) {
  sort_bucket(ids, o.tokens, o.buckets, o.order, o.rows, V, o.bits);
}

// A training forward: the first workgroups sort the tokens for the backward while the others, which wait for memory, bring the
// rows.
template <bool Two, typename T, typename I, int VEC>
__global__ __launch_bounds__(kSortThreads, 8) void gather_sort_kernel(const I* __restrict__ ids, const typename T::raw* __restrict__ W,
                                                                   int64_t ldw, float scale, typename T::raw* __restrict__ y,
                                                                   Order o, int64_t n, int64_t V, int64_t C, int64_t padding) {
  const int first = sorters<Two>(o);
  if (blockIdx.y == 0 && blockIdx.x < unsigned(first))
    sort_first<Two>(o, ids, n, V, padding);
  else
    gather<T, I, VEC>(wave_place<kSortWaves>(first), ids, W, ldw, scale, y, n, V, C);
}

// acc += rows order[s .. e) of dy at column c, U under way at once.
template <typename T, int VEC, int U>
__device__ __forceinline__ void add_rows(float* acc, const typename T::raw* dy, int64_t ld, const int* order, int s, int e,
                                         int64_t c) {
  for (; s < e; s += U) {
    Vec<T, VEC> v[U];
    int t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) t[u] = order[s + u];  // behind the last token: what follows in the workspace
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s + u < e) v[u].load(dy + int64_t(t[u]) * ld + c);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s + u < e)
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += v[u].get(i);
  }
}

// Sums the chunks of the order that one id fills.
template <typename T, typename I, int VEC>
__global__ __launch_bounds__(256) void chunk_kernel(const I* __restrict__ ids, const int* __restrict__ order,
                                                    const int2* __restrict__ rows, const typename T::raw* __restrict__ dy,
                                                    int64_t ld, float* __restrict__ part, int64_t n, int64_t V, int64_t C,
                                                    int64_t padding) {
  const int64_t w = wave_place();
  const int64_t per = (C + kWave * VEC - 1) / (kWave * VEC), p = scalar(w / per);
  if (p >= n / kChunk) return;
  const int64_t c = ((w - p * per) * kWave + threadIdx.x % kWave) * VEC;
  const int s = int(p) * kChunk;
  // where tokens are left out the order's end holds anything: no row covers a chunk there
  const int t = order[s];
  if (t < 0 || t >= n) return;
  const int64_t id = valid_id(int64_t(ids[t]), V, padding);
  if (id < 0) return;
  const int2 r = rows[id];
  if (s < r.x || s + kChunk > r.x + r.y || c >= C) return;
  float acc[VEC] = {};
  add_rows<T, VEC, 16>(acc, dy, ld, order, s, s + kChunk, c);
#pragma unroll
  for (int i = 0; i < VEC; ++i) part[p * C + c + i] = acc[i];
}

// A wave per row of dW and 64 vectors of columns: a chain of waits (where its tokens start, which they are, their rows).  With a
// lane's several vectors in one wave it took twice as long.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void rows_kernel(const int* __restrict__ order, const int2* __restrict__ rows,
                                                   const typename T::raw* __restrict__ dy, int64_t ld,
                                                   const float* __restrict__ part, float scale,
                                                   typename T::raw* __restrict__ dW, int64_t V, int64_t C) {
  const int64_t w = wave_place();
  const int64_t per = (C + kWave * VEC - 1) / (kWave * VEC), v = scalar(w / per);
  if (v >= V) return;
  const int64_t c = ((w - v * per) * kWave + threadIdx.x % kWave) * VEC;
  if (c >= C) return;
  const int s = rows[v].x, e = s + rows[v].y;
  float acc[VEC] = {};
  const int c0 = (s + kChunk - 1) / kChunk, c1 = e / kChunk;  // the chunks that this id fills
  if (c0 < c1) {
    add_rows<T, VEC, 8>(acc, dy, ld, order, s, c0 * kChunk, c);
#pragma unroll 8
    for (int p = c0; p < c1; ++p)
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += part[int64_t(p) * C + c + i];
    add_rows<T, VEC, 8>(acc, dy, ld, order, c1 * kChunk, e, c);
  } else {
    add_rows<T, VEC, 8>(acc, dy, ld, order, s, e, c);
  }
  Vec<T, VEC> o;
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] *= scale;
  o.set(acc);
  o.store(dW + v * C + c);
}

static int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

static bool bad(const char* op, int dtype, int id_bytes, int64_t T, int64_t V, int64_t C) {
  if (dtype != 0 && dtype != 1) {
    cdssm_host::set_error("%s: dtype must be 0 (fp32) or 1 (bf16), got %d", op, dtype);
    return true;
  }
  if (id_bytes != 4 && id_bytes != 8) {
    cdssm_host::set_error("%s: ids must have 4 or 8 bytes each, got %d", op, id_bytes);
    return true;
  }
  if (T < 1 || V < 1 || C < 1 || T > (int64_t(1) << 28) || V > (int64_t(1) << 28) || C > (1 << 20) ||
      std::max(T, V) > (int64_t(1) << 32) / ((C + 63) / 64)) {
    cdssm_host::set_error("%s: needs 1 <= T, V <= 2^28 and C >= 1 with max(T, V) ceil(C / 64) <= 2^32 (T %lld, V %lld, C %lld)",
                          op, (long long)T, (long long)V, (long long)C);
    return true;
  }
  return false;
}

// Elements per access that columns, row strides and pointers allow: 16 bytes, 8, or one element.
template <typename T, typename F>
static void with_vec(int64_t C, int64_t ld, const void* p, const void* q, F&& f) {
  constexpr int n = 16 / T::bytes;
  const auto a = reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q);
  if (C % n == 0 && ld % n == 0 && a % 16 == 0)
    f(std::integral_constant<int, n>{});
  else if (C % (n / 2) == 0 && ld % (n / 2) == 0 && a % 8 == 0)
    f(std::integral_constant<int, n / 2>{});
  else
    f(std::integral_constant<int, 1>{});
}

static dim3 blocks(int64_t rows, int64_t C, int vec, int waves = 4, int64_t more = 0) {
  const int64_t n = (rows * ((C + kWave * vec - 1) / (kWave * vec)) + waves - 1) / waves + more;
  const int64_t most = (int64_t(1) << 24) / waves;
  return n <= most ? dim3(unsigned(n)) : dim3(unsigned(most), unsigned((n + most - 1) / most));
}

}  // namespace emb
}  // namespace cdssm

using namespace cdssm;
using namespace cdssm::emb;

// The order's parts: the tokens, where each id's start, and with two levels the first one's.
static Order order_at(void* p, int64_t T, int64_t V) {
  char* at = static_cast<char*>(p);
  const int64_t tokens = up256(4 * T), rows = up256(8 * V);
  Order o{reinterpret_cast<int*>(at), reinterpret_cast<int2*>(at + tokens), nullptr, nullptr, id_shift(V)};
  if (two_levels(T, V)) {
    o.tokens = reinterpret_cast<int*>(at + tokens + rows);
    o.buckets = reinterpret_cast<int2*>(at + 2 * tokens + rows);
    o.bits = bucket_bits(V);
  }
  return o;
}
static int64_t order_bytes(int64_t T, int64_t V) {
  return up256(4 * T) + up256(8 * V) + (two_levels(T, V) ? up256(4 * T) + (int64_t(8) << bucket_bits(V)) : 0);
}
// first(whether there are two levels), then the second.
template <typename I, typename F>
static void sort_levels(const I* ids, const Order& o, int64_t V, hipStream_t stream, F&& first) {
  if (!o.buckets) return first(std::false_type{});
  first(std::true_type{});
  hipLaunchKernelGGL((sort_bucket_kernel<I>), dim3(unsigned(bucket_groups(V))), dim3(kSortThreads), 0, stream, ids, o, V);
}

extern "C" int64_t cdssm_token_embedding_order_bytes(int64_t T, int64_t V) {
  if (bad("cdssm_token_embedding_order_bytes", 0, 8, T, V, 1)) return -1;
  return order_bytes(T, V);
}

extern "C" int cdssm_token_embedding_fwd(int dtype, int id_bytes, const void* ids, const void* W, int64_t ldw, float scale,
                                         int64_t padding_idx, void* y, void* order, int64_t T, int64_t V, int64_t C,
                                         hipStream_t stream) {
  const char* op = "cdssm_token_embedding_fwd";
  if (bad(op, dtype, id_bytes, T, V, C)) return CDSSM_EINVAL;
  if (!ids || !W || !y || ldw < C) {
    cdssm_host::set_error("%s: null pointer argument, or a row stride below C", op);
    return CDSSM_EINVAL;
  }
  auto run = [&](auto tag, auto itag) {
    using E = decltype(tag);
    using I = decltype(itag);
    using raw = typename E::raw;
    with_vec<E>(C, ldw, W, y, [&](auto vec) {
      constexpr int VEC = decltype(vec)::value;
      if (order) {
        const Order o = order_at(order, T, V);
        sort_levels(static_cast<const I*>(ids), o, V, stream, [&](auto two) {
          constexpr bool Two = decltype(two)::value;
          hipLaunchKernelGGL((gather_sort_kernel<Two, E, I, VEC>), blocks(T, C, VEC, kSortWaves, sorters<Two>(o)), dim3(kSortThreads), 0,
                             stream, static_cast<const I*>(ids), static_cast<const raw*>(W), ldw, scale, static_cast<raw*>(y), o, T, V,
                             C, padding_idx);
        });
        return;
      }
      hipLaunchKernelGGL((gather_kernel<E, I, VEC>), blocks(T, C, VEC), dim3(256), 0, stream, static_cast<const I*>(ids),
                         static_cast<const raw*>(W), ldw, scale, static_cast<raw*>(y), T, V, C);
    });
  };
  if (dtype == 1)
    id_bytes == 8 ? run(BF16{}, int64_t{}) : run(BF16{}, int32_t{});
  else
    id_bytes == 8 ? run(F32{}, int64_t{}) : run(F32{}, int32_t{});
  return cdssm_host::check_launch(op);
}

extern "C" int64_t cdssm_token_embedding_bwd_workspace_bytes(int64_t T, int64_t V, int64_t C) {
  if (bad("cdssm_token_embedding_bwd_workspace_bytes", 0, 8, T, V, C)) return -1;
  return up256(4 * (T / kChunk) * C) + order_bytes(T, V);
}

extern "C" int cdssm_token_embedding_bwd(int dtype, int id_bytes, const void* ids, const void* dy, int64_t lddy, float scale,
                                         int64_t padding_idx, const void* sorted, void* dW, void* workspace, int64_t T, int64_t V,
                                         int64_t C, hipStream_t stream) {
  const char* op = "cdssm_token_embedding_bwd";
  if (bad(op, dtype, id_bytes, T, V, C)) return CDSSM_EINVAL;
  if (!ids || !dy || !dW || (!workspace && (!sorted || T >= kChunk)) || lddy < C) {
    cdssm_host::set_error("%s: null pointer argument, or a row stride below C", op);
    return CDSSM_EINVAL;
  }
  float* part = static_cast<float*>(workspace);
  void* at = sorted ? const_cast<void*>(sorted) : static_cast<char*>(workspace) + up256(4 * (T / kChunk) * C);
  const Order o = order_at(at, T, V);
  auto run = [&](auto tag, auto itag) {
    using E = decltype(tag);
    using I = decltype(itag);
    using raw = typename E::raw;
    if (!sorted)
      sort_levels(static_cast<const I*>(ids), o, V, stream, [&](auto two) {
        constexpr bool Two = decltype(two)::value;
        hipLaunchKernelGGL((sort_kernel<Two, I>), dim3(unsigned(sorters<Two>(o))), dim3(kSortThreads), 0, stream,
                           static_cast<const I*>(ids), o, T, V, padding_idx);
      });
    with_vec<E>(C, lddy, dy, dW, [&](auto vec) {
      constexpr int VEC = decltype(vec)::value;
      if (T >= kChunk)
        hipLaunchKernelGGL((chunk_kernel<E, I, VEC>), blocks(T / kChunk, C, VEC), dim3(256), 0, stream,
                           static_cast<const I*>(ids), o.order, o.rows, static_cast<const raw*>(dy), lddy, part, T, V, C,
                           padding_idx);
      hipLaunchKernelGGL((rows_kernel<E, VEC>), blocks(V, C, VEC), dim3(256), 0, stream, o.order, o.rows,
                         static_cast<const raw*>(dy), lddy, part, scale, static_cast<raw*>(dW), V, C);
    });
  };
  if (dtype == 1)
    id_bytes == 8 ? run(BF16{}, int64_t{}) : run(BF16{}, int32_t{});
  else
    id_bytes == 8 ? run(F32{}, int64_t{}) : run(F32{}, int32_t{});
  return cdssm_host::check_launch(op);
}
