// The 2-norm over many gradients and their clipping by it (trainer.py:242-243, torch's clip_grad_norm_):
//   n = sqrt(sum_i |g_i|^2),  c = min(1, max_norm / (n + 1e-6)),  out_i = c g_i
// The tensors' addresses and sizes travel in the launches' arguments (kPer tensors each), so a call copies nothing to
// the device and can be captured.  Norm: workgroups walk the tensors in chunks and leave a partial sum each, at most
// kPartials in all; every workgroup of the scaling adds all partial sums itself in the same order, which saves a launch.  Squares are added
// in fp64: no gradient that fp32 holds overflows, and the order of the sum does not show.  The scaling walks the tensors
// backwards, from what the norm read last and the last-level cache may still hold.
//
// Bound by memory: MI355X, 163M bf16 gradients of 410 tensors (views of one bucket) into fp32: norm 96 us (3.4 TB/s while the
// last call's results drain; 59, 5.5 TB/s, by itself), scaling 177 (5.5 TB/s); 65M fp32 gradients of 50 tensors in place: norm
// 42 .. 64 (4.1 .. 6.2 TB/s), scaling 84 (6.2 TB/s, half of it from the last-level cache) where they are clipped.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>
#include <vector>

#include "common.hpp"

namespace cdssm {
namespace gn {

constexpr int kPer = 128;        // tensors per launch: 3.7 KB of arguments
constexpr int kThreads = 512;
constexpr int kChunk = 32768;    // elements a workgroup takes at a time: 8 vectors of 8 for a thread, all under way at once
constexpr int kPartials = 1024;  // two for each thread
constexpr int kScaleBlocks = 1024;

struct Table {
  const void* in[kPer];
  void* out[kPer];
  int64_t n[kPer];
  int first[kPer + 1];     // a tensor's first chunk
  uint8_t code[kPer];      // bit 0: bf16 in, bit 1: bf16 out
  int count;
};

__device__ __forceinline__ int find(const Table& t, int chunk) {
  int lo = 0, hi = t.count;  // first[lo] <= chunk < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= chunk)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__device__ __forceinline__ double block_sum(double x, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, kWave);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = x;
  __syncthreads();
  x = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / kWave; ++w) x += red[w];
  __syncthreads();
  return x;
}

// Eight elements as they lie in memory.
template <typename T>
struct Eight {
  uint4 u[T::bytes / 2];
  __device__ __forceinline__ void load(const typename T::raw* p) {
#pragma unroll
    for (int i = 0; i < T::bytes / 2; ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (T::bytes == 2) {
      const uint32_t w[4] = {u[0].x, u[0].y, u[0].z, u[0].w};
      return i & 1 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]);
    } else {
      const uint4 v = u[i / 4];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      return __uint_as_float(w[i % 4]);
    }
  }
};

// The range lo .. hi of a tensor: one(index, value) for single elements up to a 16-byte boundary and behind the last
// vector, eight(index, vector) for the vectors between, a thread's kUnder of which are under way at once.
constexpr int kUnder = kChunk / 8 / kThreads;
template <typename T, typename One, typename Vector>
__device__ __forceinline__ void walk(const typename T::raw* p, int64_t lo, int64_t hi, One&& one, Vector&& eight) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p + lo);
  const int64_t head = min(hi, lo + int64_t(((16 - (at & 15u)) & 15u) / T::bytes));
  const int nv = int((hi - head) / 8);
  const int64_t tail = head + nv * 8;
  Eight<T> v[kUnder];  // a range is a chunk at most
#pragma unroll
  for (int u = 0; u < kUnder; ++u) {
    const int i = u * kThreads + int(threadIdx.x);
    if (i < nv) v[u].load(p + head + i * 8);
  }
  const int64_t a = lo + threadIdx.x, b = tail + threadIdx.x;
  if (a < head) one(a, T::load(p + a));
  if (b < hi) one(b, T::load(p + b));
#pragma unroll
  for (int u = 0; u < kUnder; ++u) {
    const int i = u * kThreads + int(threadIdx.x);
    if (i < nv) eight(head + i * 8, v[u]);
  }
}

template <typename T>
__device__ __forceinline__ double sum_squares(const void* in, int64_t lo, int64_t hi) {
  double s = 0.0, s2 = 0.0;
  walk<T>(
      static_cast<const typename T::raw*>(in), lo, hi, [&](int64_t, float x) { s = fma(double(x), double(x), s); },
      [&](int64_t, const Eight<T>& v) {
#pragma unroll
        for (int u = 0; u < 8; u += 2) {
          const double x = v.get(u), y = v.get(u + 1);
          s = fma(x, x, s);
          s2 = fma(y, y, s2);
        }
      });
  return s + s2;
}

__global__ __launch_bounds__(kThreads) void squares_kernel(Table t, double* part) {
  __shared__ double red[kThreads / kWave];
  double s = 0.0;
  for (int c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
    const int k = find(t, c);
    const int64_t lo = int64_t(c - t.first[k]) * kChunk, hi = min(t.n[k], lo + kChunk);
    s += t.code[k] & 1 ? sum_squares<BF16>(t.in[k], lo, hi) : sum_squares<F32>(t.in[k], lo, hi);
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__device__ __forceinline__ double norm_of(const double* part, int n, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) s += part[i];
  return sqrt(block_sum(s, red));
}

__global__ __launch_bounds__(kThreads) void norm_kernel(const double* part, int n, float* norm) {
  __shared__ double red[kThreads / kWave];
  const double v = norm_of(part, n, red);
  if (threadIdx.x == 0) *norm = float(v);
}

template <typename TI, typename TO>
__device__ __forceinline__ void scale_range(const void* in, void* out, int64_t lo, int64_t hi, float c) {
  const auto* p = static_cast<const typename TI::raw*>(in);
  auto* q = static_cast<typename TO::raw*>(out);
  // vectors where both sides reach a 16-byte boundary at the same element
  const uintptr_t a = reinterpret_cast<uintptr_t>(p + lo), b = reinterpret_cast<uintptr_t>(q + lo);
  const int64_t head = int64_t(((16 - (a & 15u)) & 15u) / TI::bytes);
  if (((b + head * TO::bytes) & 15u) != 0) {
#pragma unroll 8
    for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads) TO::store(q + i, TI::load(p + i) * c);
    return;
  }
  walk<TI>(
      p, lo, hi, [&](int64_t i, float x) { TO::store(q + i, x * c); },
      [&](int64_t i, const Eight<TI>& v) {
        if constexpr (TO::bytes == 2) {
          *reinterpret_cast<uint4*>(q + i) =
              make_uint4(pack_bf16x2(v.get(0) * c, v.get(1) * c), pack_bf16x2(v.get(2) * c, v.get(3) * c),
                         pack_bf16x2(v.get(4) * c, v.get(5) * c), pack_bf16x2(v.get(6) * c, v.get(7) * c));
        } else {
          reinterpret_cast<float4*>(q + i)[0] = make_float4(v.get(0) * c, v.get(1) * c, v.get(2) * c, v.get(3) * c);
          reinterpret_cast<float4*>(q + i)[1] = make_float4(v.get(4) * c, v.get(5) * c, v.get(6) * c, v.get(7) * c);
        }
      });
}

__global__ __launch_bounds__(kThreads) void scale_kernel(Table t, const double* part, int n, float max_norm, float* norm) {
  __shared__ double red[kThreads / kWave];
  const double v = norm_of(part, n, red);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = float(v);
  const double r = double(max_norm) / (v + 1e-6);
  const float c = r > 1.0 ? 1.0f : float(r);  // NaN stays
  const int chunks = t.first[t.count];
  for (int b = blockIdx.x; b < chunks; b += gridDim.x) {
    const int i = chunks - 1 - b, k = find(t, i);
    if (c == 1.0f && t.in[k] == t.out[k]) continue;  // nothing to change
    const int64_t lo = int64_t(i - t.first[k]) * kChunk, hi = min(t.n[k], lo + kChunk);
    switch (t.code[k]) {
      case 0: scale_range<F32, F32>(t.in[k], t.out[k], lo, hi, c); break;
      case 1: scale_range<BF16, F32>(t.in[k], t.out[k], lo, hi, c); break;
      case 2: scale_range<F32, BF16>(t.in[k], t.out[k], lo, hi, c); break;
      default: scale_range<BF16, BF16>(t.in[k], t.out[k], lo, hi, c); break;
    }
  }
}

}  // namespace gn
}  // namespace cdssm

using namespace cdssm;
using namespace cdssm::gn;

constexpr int64_t kMostElements = int64_t(1) << 38;

// What lies behind n elements at p.
static const void* after(const void* p, int64_t n, bool bf16) { return static_cast<const char*>(p) + n * (bf16 ? 2 : 4); }

static int check_tensors(const char* op, int64_t count, const void* const* in, const int* in_dtype, void* const* out,
                         const int* out_dtype, const int64_t* n, const void* workspace) {
  if (count < 0 || (count && (!in || !in_dtype || !n || (out && !out_dtype))) || !workspace) {
    cdssm_host::set_error("%s: null pointer argument, or a negative count", op);
    return CDSSM_EINVAL;
  }
  for (int64_t i = 0; i < count; ++i) {
    if (n[i] < 0 || n[i] > kMostElements || (n[i] && (!in[i] || (out && !out[i])))) {
      cdssm_host::set_error("%s: tensor %lld: null pointer, or a size out of range", op, (long long)i);
      return CDSSM_EINVAL;
    }
    const int di = in_dtype[i], dn = out ? out_dtype[i] : 0;
    if ((di != 0 && di != 1) || (dn != 0 && dn != 1)) {
      cdssm_host::set_error("%s: tensor %lld: dtype must be 0 (fp32) or 1 (bf16)", op, (long long)i);
      return CDSSM_EINVAL;
    }
    if (reinterpret_cast<uintptr_t>(in[i]) % (di ? 2 : 4) || (out && reinterpret_cast<uintptr_t>(out[i]) % (dn ? 2 : 4))) {
      cdssm_host::set_error("%s: tensor %lld: not aligned to its elements", op, (long long)i);
      return CDSSM_EINVAL;
    }
  }
  return CDSSM_OK;
}

// The tensors that are not empty, kPer to a table (of 2^38 elements at most each: 2^30 chunks).  Neighbours in memory, as the
// views of a bucket are, count as one: fewer launches, each of which takes some 8 us to fill and empty the chip.
static std::vector<Table> make_tables(int64_t count, const void* const* in, const int* in_dtype, void* const* out,
                                      const int* out_dtype, const int64_t* n) {
  std::vector<Table> ts;
  for (int64_t i = 0; i < count; ++i) {
    if (!n[i]) continue;
    const uint8_t code = uint8_t(in_dtype[i] | (out ? out_dtype[i] << 1 : 0));
    if (!ts.empty()) {
      Table& t = ts.back();
      const int k = t.count - 1;
      if (t.code[k] == code && t.n[k] + n[i] <= kMostElements && after(t.in[k], t.n[k], code & 1) == in[i] &&
          (!out || after(t.out[k], t.n[k], code & 2) == out[i])) {
        t.n[k] += n[i];
        t.first[k + 1] = t.first[k] + int((t.n[k] + kChunk - 1) / kChunk);
        continue;
      }
    }
    const int64_t chunks = (n[i] + kChunk - 1) / kChunk;
    if (ts.empty() || ts.back().count == kPer) {
      ts.emplace_back();
      ts.back().count = 0;
      ts.back().first[0] = 0;
    }
    Table& t = ts.back();
    const int k = t.count++;
    t.in[k] = in[i];
    t.out[k] = out ? out[i] : nullptr;
    t.n[k] = n[i];
    t.code[k] = code;
    t.first[k + 1] = t.first[k] + int(chunks);
  }
  return ts;
}

// The same into ts; false, with the error set, where the host has no memory for them.
static bool tables_into(std::vector<Table>& ts, const char* op, int64_t count, const void* const* in, const int* in_dtype,
                        void* const* out, const int* out_dtype, const int64_t* n) {
  try {
    ts = make_tables(count, in, in_dtype, out, out_dtype, n);
    return true;
  } catch (const std::bad_alloc&) {
    cdssm_host::set_error("%s: no host memory for the launches' arguments of %lld tensors", op, (long long)count);
    return false;
  }
}

// Launches the sums of squares; the number of partial sums.
static int squares(const std::vector<Table>& ts, double* part, hipStream_t stream) {
  int used = 0;
  const int most = std::max(1, kPartials / std::max(1, int(ts.size())));
  for (const Table& t : ts) {
    const int blocks = std::min(t.first[t.count], most);
    hipLaunchKernelGGL(squares_kernel, dim3(unsigned(blocks)), dim3(gn::kThreads), 0, stream, t, part + used);
    used += blocks;
  }
  return used;
}

extern "C" int64_t cdssm_grad_norm_workspace_bytes(int64_t count) {
  if (count < 0) return -1;
  return 8 * (kPartials + count / kPer + 1);
}

extern "C" int cdssm_grad_norm(int64_t count, const void* const* in, const int* in_dtype, const int64_t* n, float* norm,
                               void* workspace, hipStream_t stream) {
  const char* op = "cdssm_grad_norm";
  if (const int st = check_tensors(op, count, in, in_dtype, nullptr, nullptr, n, workspace)) return st;
  if (!norm) {
    cdssm_host::set_error("%s: null pointer argument", op);
    return CDSSM_EINVAL;
  }
  auto* part = static_cast<double*>(workspace);
  std::vector<Table> ts;
  if (!tables_into(ts, op, count, in, in_dtype, nullptr, nullptr, n)) return CDSSM_EINVAL;
  const int used = squares(ts, part, stream);
  hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(gn::kThreads), 0, stream, part, used, norm);
  return cdssm_host::check_launch(op);
}

extern "C" int cdssm_clip_grads(int64_t count, const void* const* in, const int* in_dtype, void* const* out,
                                const int* out_dtype, const int64_t* n, float max_norm, float* norm, void* workspace,
                                hipStream_t stream) {
  const char* op = "cdssm_clip_grads";
  if (const int st = check_tensors(op, count, in, in_dtype, out, out_dtype, n, workspace)) return st;
  if (!norm || (count && (!out || !out_dtype)) || !(max_norm >= 0.0f)) {
    cdssm_host::set_error("%s: null pointer argument, or max_norm not a number of at least 0", op);
    return CDSSM_EINVAL;
  }
  auto* part = static_cast<double*>(workspace);
  std::vector<Table> ts;
  if (!tables_into(ts, op, count, in, in_dtype, out, out_dtype, n)) return CDSSM_EINVAL;
  const int used = squares(ts, part, stream);
  if (!used) {
    hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(gn::kThreads), 0, stream, part, 0, norm);
    return cdssm_host::check_launch(op);
  }
  for (size_t i = ts.size(); i-- > 0;) {
    const Table& t = ts[i];
    hipLaunchKernelGGL(scale_kernel, dim3(unsigned(std::min(t.first[t.count], kScaleBlocks))), dim3(gn::kThreads), 0, stream, t,
                       part, used, max_norm, i + 1 == ts.size() ? norm : nullptr);
  }
  return cdssm_host::check_launch(op);
}
