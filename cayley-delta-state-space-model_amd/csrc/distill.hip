// Distillation of a student from a teacher's top logits: with p = softmax(z / tau) over a token's K kept logits z, of the words
// i_1 .. i_K, and q = softmax(x / tau) over the student's logits x of all V words,
//   loss = tau^2 sum_k p_k (log p_k - log q_{i_k}),   dx_v = s tau (q_v - sum over k with i_k = v of p_k)
// (s: upstream gradient, / count for a mean).  A kept logit of -inf takes no part, whatever its id; a token without any
// takes none either: its loss and gradient are 0, its logits are not read.
//
// Forward: W waves go through a row once, every lane with a maximum and a sum of its own, which are joined at the end; the
// row's (m, 1 / sum) is kept.  Backward: the row is read again, q formed and written as the gradient, and the words of the list
// are written once more by the wave that wrote them before, their gradient formed whole (so a word that is listed twice is right).
// Both are bound by memory; a row is not kept on the chip between the two, which are calls of their own.  MI355X, 16384 x 32000 bf16,
// 32 kept: forward 182 us (1.05 GB, 5.8 TB/s), backward 390 (2.1 GB, 5.4 TB/s, where a large copy reaches 4.9); 8192 x 50257 bf16 142
// and 321, 4995 x 50257 fp32 166 and 391.
#include <hip/hip_runtime.h>

#include <cmath>

#include "common.hpp"
#include "logit_rows.hpp"

namespace cdssm {
namespace distill {

using namespace rows;

constexpr int kMaxK = 256, kPer = kMaxK / kWave;
constexpr float kLog2e = 1.44269504088896340736f;

struct Args {
  const void* x;  // (T, V) logits, row stride ld
  int64_t ld;
  const void *z, *ids;  // (T, K)
  int id_bytes;
  float inv_tau, scale, gscale;  // 1 / tau; log2 e / tau; tau
  int64_t T;
  int V, K;
};

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int j = kWave / 2; j > 0; j /= 2) x = fmaxf(x, __shfl_xor(x, j, kWave));
  return x;
}
__device__ __forceinline__ float wave_sum(float x) { return group_sum<kWave>(x); }

// The teacher's distribution over a token's list, entry k = 64 j + lane in a lane's j-th: p and log p, both 0 where the entry
// takes no part, and the word (-1 where it is out of range).  any: whether an entry takes part.
template <typename Z>
struct Teacher {
  float p[kPer], logp[kPer];
  int id[kPer];
  bool part[kPer], any;
  __device__ __forceinline__ void load(const Args& a, int64_t t, int lane) {
    const auto* z = static_cast<const typename Z::raw*>(a.z) + t * a.K;
    float m = -INFINITY;
    bool mine = false;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int k = j * kWave + lane;
      p[j] = -INFINITY;
      id[j] = -1;
      if (k < a.K) {
        p[j] = Z::load(z + k);
        id[j] = id_at(a.ids, a.id_bytes, t * a.K + k);
        if (id[j] >= a.V) id[j] = -1;
      }
      part[j] = !(p[j] == -INFINITY);
      mine |= part[j];
      m = fmaxf(m, p[j]);
    }
    any = __ballot(mine) != 0;
    m = wave_max(m);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      logp[j] = part[j] ? (p[j] - m) * a.inv_tau : 0.0f;
      // exp2f: down to the subnormal numbers, which the instruction alone gives as 0; a listed word's loss may be infinite
      p[j] = part[j] ? exp2f((p[j] - m) * a.scale) : 0.0f;
      sum += p[j];
    }
    sum = wave_sum(sum);
    const float inv = 1.0f / sum, log_sum = logf(sum);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      p[j] *= inv;
      logp[j] -= log_sum;
    }
  }
};

// A maximum and a sum of e^((x - m) / tau).
struct Soft {
  float m, s;
  // Takes in n values.  The maximum is taken out before the factor, whose product with large logits would be rounded.
  template <int N>
  __device__ __forceinline__ void add(const float (&x)[N], float scale) {
    float top = m;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, x[i]);
    const float base = top == -INFINITY ? 0.0f : top;
    s *= m == top ? 1.0f : __builtin_amdgcn_exp2f((m - top) * scale);
    m = top;
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      s0 += __builtin_amdgcn_exp2f((x[i] - base) * scale);
      if (i + 1 < N) s1 += __builtin_amdgcn_exp2f((x[i + 1] - base) * scale);
    }
    s += s0 + s1;
  }
  __device__ __forceinline__ void rebase(float top, float scale) {
    s *= m == top ? 1.0f : __builtin_amdgcn_exp2f((m - top) * scale);
    m = top;
  }
};

// The maximum and sum over a wave's part of a row.
template <typename T>
__device__ __forceinline__ Soft soft_of(const typename T::raw* row, const Part& s, int V, float scale, int lane) {
  constexpr int E = Vec<T>::E, U = 4;
  Soft f{-INFINITY, 0.0f};
  const uint4* vec = reinterpret_cast<const uint4*>(row + s.first);
  // single elements at the ends: at most 16, one a lane
  const int n_tail = V - s.tail, n_ends = s.head + n_tail;
  if (n_ends > 0) {
    const int i = lane < s.head ? lane : s.tail + lane - s.head;
    const float x[1] = {lane < n_ends ? T::load(row + i) : -INFINITY};
    f.add(x, scale);
  }
  int i = s.lo + lane;
  Vec<T> v[U];
  for (; i + (U - 1) * kWave < s.hi; i += U * kWave) {
#pragma unroll
    for (int u = 0; u < U; ++u) v[u].u = vec[i + u * kWave];
    float x[U * E];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) x[u * E + e] = v[u].get(e);
    f.add(x, scale);
  }
  for (; i < s.hi; i += kWave) {
    v[0].u = vec[i];
    float x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = v[0].get(e);
    f.add(x, scale);
  }
  const float top = wave_max(f.m);
  f.rebase(top, scale);
  f.s = wave_sum(f.s);
  return f;
}

// each: a token's loss; soft: (m, 1 / sum), the second 0 where the token takes no part.
template <typename T, typename Z, int W, int Rows>
__global__ __launch_bounds__(kWave* W* Rows) void fwd_kernel(Args a, float* __restrict__ each, float2* __restrict__ soft) {
  __shared__ Soft parts[W];
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave), lane = int(threadIdx.x) % kWave;
  const int64_t t = int64_t(blockIdx.x) * Rows + wave / W;
  if (t >= a.T) return;  // with Rows > 1 no workgroup meets at a barrier
  const int w = wave % W;
  Teacher<Z> z;
  z.load(a, t, lane);
  if (!z.any) {  // the same in every wave of the row
    if (w == 0 && lane == 0) {
      each[t] = 0.0f;
      soft[t] = make_float2(0.0f, 0.0f);
    }
    return;
  }
  const auto* row = static_cast<const typename T::raw*>(a.x) + t * a.ld;
  float at[kPer];
  if (w == 0)
#pragma unroll
    for (int j = 0; j < kPer; ++j) at[j] = z.id[j] >= 0 ? T::load(row + z.id[j]) : NAN;
  Soft f = soft_of<T>(row, part_of<T, W>(row, a.V, w), a.V, a.scale, lane);
  if constexpr (W > 1) {
    if (lane == 0) parts[w] = f;
    __syncthreads();
    if (w != 0) return;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < W; ++i) top = fmaxf(top, parts[i].m);
    f.s = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      Soft g = parts[i];
      g.rebase(top, a.scale);
      f.s += g.s;
    }
    f.m = top;
  }
  const float log_sum = logf(f.s);
  float loss = 0.0f;
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    // a probability that fp32 does not hold counts as 0, also where the student's is 0; a word out of range is NaN with any
    if (z.part[j] && (z.id[j] < 0 || !(z.p[j] == 0.0f))) loss += z.p[j] * (z.logp[j] - ((at[j] - f.m) * a.inv_tau - log_sum));
  loss = wave_sum(loss) * a.gscale * a.gscale;
  if (lane == 0) {
    each[t] = loss;
    soft[t] = make_float2(f.m, 1.0f / f.s);
  }
}

// The tokens' losses as one, and how many took part.
constexpr int kSumThreads = 1024;
__global__ __launch_bounds__(kSumThreads) void sum_kernel(const float* __restrict__ each, const float2* __restrict__ soft, int64_t T,
                                                          bool mean, float* __restrict__ loss, float* __restrict__ count) {
  __shared__ double sums[kSumThreads / kWave];
  __shared__ int counts[kSumThreads / kWave];
  double s = 0.0;
  int n = 0;
  constexpr int U = 16;  // of a thread under way at once
  for (int64_t t0 = threadIdx.x; t0 < T; t0 += U * kSumThreads) {
    float v[U], y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = t0 + u * kSumThreads;
      v[u] = each[min(t, T - 1)];  // no branches around the loads
      y[u] = soft[min(t, T - 1)].y;
    }
    __builtin_amdgcn_sched_barrier(0);  // all loads first
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool there = t0 + u * kSumThreads < T;
      s += double(there ? v[u] : 0.0f);
      n += there && y[u] != 0.0f;
    }
  }
#pragma unroll
  for (int j = kWave / 2; j > 0; j /= 2) {
    s += __shfl_xor(s, j, kWave);
    n += __shfl_xor(n, j, kWave);
  }
  if (threadIdx.x % kWave == 0) {
    sums[threadIdx.x / kWave] = s;
    counts[threadIdx.x / kWave] = n;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  s = 0.0;
  n = 0;
#pragma unroll
  for (int i = 0; i < kSumThreads / kWave; ++i) {
    s += sums[i];
    n += counts[i];
  }
  *loss = float(mean ? s / double(n) : s);
  *count = float(n);
}

// 16 bytes of memory, past the caches where Stream.
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
template <bool Stream>
__device__ __forceinline__ uint4 get16(const uint4* p) {
  if constexpr (Stream) return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p)));
  return *p;
}
template <bool Stream>
__device__ __forceinline__ void put16(uint4* p, uint4 v) {
  if constexpr (Stream)
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, v), reinterpret_cast<u32x4_t*>(p));
  else
    *p = v;
}

// The last rows first: the last-level cache may still hold what the forward read last.
// per_token: a gradient for each token, else one for all; count: divides it, or null.
template <typename T, typename Z, int W, int Rows, bool Stream>
__global__ __launch_bounds__(kWave* W* Rows) void bwd_kernel(Args a, const float* __restrict__ up, bool per_token,
                                                             const float* __restrict__ count, const float2* __restrict__ soft,
                                                             typename T::raw* __restrict__ grad, int64_t ldg) {
  constexpr int E = Vec<T>::E, U = 4;
  __shared__ float ps[Rows][kMaxK];
  __shared__ int is[Rows][kMaxK];
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave), lane = int(threadIdx.x) % kWave;
  const int64_t t = a.T - 1 - (int64_t(blockIdx.x) * Rows + wave / W);
  if (t < 0) return;  // with Rows > 1 no workgroup meets at a barrier
  const int w = wave % W, V = a.V;
  const auto* row = static_cast<const typename T::raw*>(a.x) + t * a.ld;
  auto* out = grad + t * ldg;
  Teacher<Z> z;
  z.load(a, t, lane);
  const Part s = part_of<T, W>(row, V, w);
  const uint4* vec = reinterpret_cast<const uint4*>(row + s.first);
  uint4* vout = reinterpret_cast<uint4*>(out + s.first);
  // whether the gradient's row reaches a 16-byte boundary where the logits' does
  const bool same = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
  float m = 0.0f, c = 0.0f;  // gradient = c e^((x - m) / tau) - r p
  float r = 0.0f;
  if (z.any) {
    const float2 f = soft[t];
    bool bad = false;
#pragma unroll
    for (int j = 0; j < kPer; ++j) bad |= z.part[j] && (z.id[j] < 0 || z.p[j] != z.p[j]);
    r = (per_token ? up[t] : up[0]) * a.gscale;
    if (count) r /= *count;
    if (__ballot(bad)) r = NAN;
    m = f.x;
    c = r * f.y;
    if (w == 0)
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int k = j * kWave + lane;
        if (k < a.K) {
          ps[wave / W][k] = z.p[j];
          is[wave / W][k] = z.part[j] ? z.id[j] : -1;
        }
      }
  }
  const auto g = [&](float x) { return c * __builtin_amdgcn_exp2f((x - m) * a.scale); };
  const int n_ends = s.head + V - s.tail;
  if (lane < n_ends) {
    const int i = lane < s.head ? lane : s.tail + lane - s.head;
    T::store(out + i, z.any ? g(T::load(row + i)) : 0.0f);
  }
  if (same) {
    int i = s.lo + lane;
    Vec<T> v[U];
    const auto put = [&](Vec<T>& u, int at) {
      float y[E];
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = g(u.get(e));
      u.set(y);
      put16<Stream>(vout + at, u.u);
    };
    if (!z.any) {
      for (; i < s.hi; i += kWave) put16<Stream>(vout + i, make_uint4(0, 0, 0, 0));
    } else {
      for (; i + (U - 1) * kWave < s.hi; i += U * kWave) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u].u = get16<Stream>(vec + i + u * kWave);
#pragma unroll
        for (int u = 0; u < U; ++u) put(v[u], i + u * kWave);
      }
      for (; i < s.hi; i += kWave) {
        v[0].u = get16<Stream>(vec + i);
        put(v[0], i);
      }
    }
  } else {
    const int hi = s.at<T>(s.hi);
#pragma unroll 8
    for (int i = s.at<T>(s.lo) + lane; i < hi; i += kWave) T::store(out + i, z.any ? g(T::load(row + i)) : 0.0f);
  }
  if (!z.any) return;  // the same in every wave of the row
  // the words of the list, by the wave that has written them already
  if constexpr (W > 1) {
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int id = z.part[j] ? z.id[j] : -1;
    if (id < 0 || !s.has<T>(id, V)) continue;
    float p = 0.0f;
    for (int k = 0; k < a.K; ++k) p += is[wave / W][k] == id ? ps[wave / W][k] : 0.0f;
    T::store(out + id, fmaf(-r, p, g(T::load(row + id))));
  }
}

// What the forward leaves for the backward.
struct State {
  float* count;
  float2* soft;
  float* each;
  int64_t bytes;
};
static State carve(void* ws, int64_t T) {
  char* p = static_cast<char*>(ws);
  return {reinterpret_cast<float*>(p), reinterpret_cast<float2*>(p + 256), reinterpret_cast<float*>(p + 256 + 8 * T),
          256 + 12 * T};
}

// f(element type, teacher's type, waves to a row, rows to a workgroup)
template <typename F>
static void choose(int dtype, int teacher_dtype, int64_t T, int64_t V, bool backward, F&& f) {
  using std::integral_constant;
  const auto waves = [&](auto x, auto z) {
    // 12 KB of a row, or more, to a wave of the forward, 4 KB of the backward, whose writes run better the nearer they lie
    // together; less only where few rows leave the device empty.  us, forward + backward as it is launched (past the caches from
    // 200 MB on), with 1 / 4 / 8 / 16 waves to a row: 16384 x 32000 bf16 192 + 424 / 182 + 389 / 197 + 391 / 333 + 453, 8192 x 50257
    // bf16 151 + 350 / 145 + 331 / 141 + 319 / 211 + 320, 4995 x 50257 fp32 182 + 423 / 173 + 411 / 171 + 399 / 166 + 393, 4096 x 131072
    // bf16 193 + 439 / 194 + 407 / 201 + 382 / 191 + 384, 16384 x 4000 bf16 40 + 66 / 43 + 66 / 67 + 95 / 117 + 190.
    const int64_t row = V * x.bytes, share = backward ? 4096 : 12288;
    int w = 1;
    while (w < 16 && (row >= 2 * w * share || (2 * w * T <= 2048 && row >= 2 * w * 1024))) w *= 2;
    w == 16  ? f(x, z, integral_constant<int, 16>{}, integral_constant<int, 1>{})
    : w == 8 ? f(x, z, integral_constant<int, 8>{}, integral_constant<int, 1>{})
    : w == 4 ? f(x, z, integral_constant<int, 4>{}, integral_constant<int, 1>{})
    : w == 2 ? f(x, z, integral_constant<int, 2>{}, integral_constant<int, 1>{})
             : f(x, z, integral_constant<int, 1>{}, integral_constant<int, 4>{});
  };
  const auto teacher = [&](auto x) { teacher_dtype ? waves(x, BF16{}) : waves(x, F32{}); };
  dtype ? teacher(BF16{}) : teacher(F32{});
}

static int check(const char* op, int dtype, int teacher_dtype, int id_bytes, const void* x, int64_t ld, const void* z, const void* ids,
                 float tau, int reduction, const void* ws, int64_t T, int64_t V, int64_t K) {
  if ((dtype != 0 && dtype != 1) || (teacher_dtype != 0 && teacher_dtype != 1)) {
    cdssm_host::set_error("%s: dtypes must be 0 (fp32) or 1 (bf16), got %d and %d", op, dtype, teacher_dtype);
    return CDSSM_EINVAL;
  }
  if (id_bytes != 4 && id_bytes != 8) {
    cdssm_host::set_error("%s: ids must have 4 or 8 bytes, got %d", op, id_bytes);
    return CDSSM_EINVAL;
  }
  if (reduction < 0 || reduction > 2) {
    cdssm_host::set_error("%s: reduction must be 0 (none), 1 (mean) or 2 (sum), got %d", op, reduction);
    return CDSSM_EINVAL;
  }
  if (!(tau >= 1e-4f && tau <= 1e4f)) {
    cdssm_host::set_error("%s: temperature must be within 1e-4 .. 1e4, got %g", op, double(tau));
    return CDSSM_EINVAL;
  }
  if (!x || !z || !ids || !ws) {
    cdssm_host::set_error("%s: null pointer argument", op);
    return CDSSM_EINVAL;
  }
  if (T < 1 || T > (int64_t(1) << 24) || V < 1 || V > (int64_t(1) << 24) || K < 1 || K > kMaxK) {
    cdssm_host::set_error("%s: needs 1 <= T, V <= 2^24 and 1 <= K <= %d, got T %lld, V %lld, K %lld", op, kMaxK, (long long)T,
                          (long long)V, (long long)K);
    return CDSSM_EINVAL;
  }
  if (ld < V || ld > (int64_t(1) << 32) || reinterpret_cast<uintptr_t>(x) % (dtype ? 2 : 4) ||
      reinterpret_cast<uintptr_t>(z) % (teacher_dtype ? 2 : 4) || reinterpret_cast<uintptr_t>(ids) % unsigned(id_bytes) ||
      reinterpret_cast<uintptr_t>(ws) % 8) {
    cdssm_host::set_error("%s: row strides must be within V .. 2^32, the tensors aligned to their elements and the workspace to 8 bytes", op);
    return CDSSM_EINVAL;
  }
  return CDSSM_OK;
}

static Args args_of(const void* x, int64_t ld, const void* z, const void* ids, int id_bytes, float tau, int64_t T, int64_t V,
                    int64_t K) {
  return {x, ld, z, ids, id_bytes, float(1.0 / double(tau)), float(1.4426950408889634 / double(tau)), tau, T, int(V), int(K)};
}

}  // namespace distill
}  // namespace cdssm

using namespace cdssm;

extern "C" int64_t cdssm_distillation_workspace_bytes(int64_t T) {
  if (T < 1 || T > (int64_t(1) << 24)) {
    cdssm_host::set_error("cdssm_distillation_workspace_bytes: needs 1 <= T <= 2^24, got %lld", (long long)T);
    return CDSSM_EINVAL;
  }
  return distill::carve(nullptr, T).bytes;
}

extern "C" int cdssm_distillation_fwd(int dtype, int teacher_dtype, int id_bytes, const void* logits, int64_t ld,
                                      const void* teacher_logits, const void* teacher_ids, float temperature, int reduction,
                                      float* loss, void* workspace, int64_t T, int64_t V, int64_t K, hipStream_t stream) {
  const char* op = "cdssm_distillation_fwd";
  if (const int st = distill::check(op, dtype, teacher_dtype, id_bytes, logits, ld, teacher_logits, teacher_ids, temperature,
                                    reduction, workspace, T, V, K))
    return st;
  if (!loss || reinterpret_cast<uintptr_t>(loss) % 4) {
    cdssm_host::set_error("%s: loss must not be null, and aligned to 4 bytes", op);
    return CDSSM_EINVAL;
  }
  const distill::State st = distill::carve(workspace, T);
  const distill::Args a = distill::args_of(logits, ld, teacher_logits, teacher_ids, id_bytes, temperature, T, V, K);
  float* each = reduction == 0 ? loss : st.each;
  distill::choose(dtype, teacher_dtype, T, V, false, [&](auto x, auto z, auto wc, auto rc) {
    constexpr int W = decltype(wc)::value, Rows = decltype(rc)::value;
    hipLaunchKernelGGL((distill::fwd_kernel<decltype(x), decltype(z), W, Rows>), dim3(unsigned((T + Rows - 1) / Rows)),
                       dim3(kWave * W * Rows), 0, stream, a, each, st.soft);
  });
  if (reduction != 0)
    hipLaunchKernelGGL(distill::sum_kernel, dim3(1), dim3(distill::kSumThreads), 0, stream, st.each, st.soft, T, reduction == 1,
                       loss, st.count);
  return cdssm_host::check_launch(op);
}

extern "C" int cdssm_distillation_bwd(int dtype, int teacher_dtype, int id_bytes, const void* logits, int64_t ld,
                                      const void* teacher_logits, const void* teacher_ids, float temperature, int reduction,
                                      const float* gloss, const void* fwd_workspace, void* grad, int64_t ldg, int64_t T, int64_t V,
                                      int64_t K, hipStream_t stream) {
  const char* op = "cdssm_distillation_bwd";
  if (const int st = distill::check(op, dtype, teacher_dtype, id_bytes, logits, ld, teacher_logits, teacher_ids, temperature,
                                    reduction, fwd_workspace, T, V, K))
    return st;
  if (!gloss || !grad || reinterpret_cast<uintptr_t>(gloss) % 4 || reinterpret_cast<uintptr_t>(grad) % (dtype ? 2 : 4) || ldg < V ||
      ldg > (int64_t(1) << 32)) {
    cdssm_host::set_error("%s: gloss and grad must not be null, and aligned to their elements, grad's row stride within V .. 2^32", op);
    return CDSSM_EINVAL;
  }
  const distill::State st = distill::carve(const_cast<void*>(fwd_workspace), T);
  const distill::Args a = distill::args_of(logits, ld, teacher_logits, teacher_ids, id_bytes, temperature, T, V, K);
  distill::choose(dtype, teacher_dtype, T, V, true, [&](auto x, auto z, auto wc, auto rc) {
    constexpr int W = decltype(wc)::value, Rows = decltype(rc)::value;
    using X = decltype(x);
    const auto go = [&](auto stream_past) {
      hipLaunchKernelGGL((distill::bwd_kernel<X, decltype(z), W, Rows, decltype(stream_past)::value>),
                         dim3(unsigned((T + Rows - 1) / Rows)), dim3(kWave * W * Rows), 0, stream, a, gloss, reduction == 0,
                         reduction == 1 ? st.count : nullptr, st.soft, static_cast<typename X::raw*>(grad), ldg);
    };
    // Logits that fill the last-level cache by themselves are not kept in it, nor is their gradient: 16384 x 32000 bf16 432 -> 391
    // us, 4096 x 32000 113 -> 103; but 2048 x 32000 (131 MB) 51 -> 56.
    T * V * X::bytes >= (int64_t(200) << 20) ? go(std::true_type{}) : go(std::false_type{});
  });
  return cdssm_host::check_launch(op);
}
