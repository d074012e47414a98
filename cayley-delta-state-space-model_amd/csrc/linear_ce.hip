// Softmax cross entropy of the language model's head, in pieces of the vocabulary, without keeping the logits:
//   l[t][v] = x[t] . W[v],  lse[t] = log sum_v exp l[t][v],  loss[t] = lse[t] - l[t][y_t]
//   g[t][v] = (exp(l - lse) - [v = y_t]) s_t,  dx = g W,  dW = g^T x     (s_t: upstream gradient, / count for a mean)
// (the training step's loss over the tied head, trainer.py:235-238 with model.py:51).
//
// Everything large is a matrix product on the matrix cores (mma_tiles.hpp).  Forward: a tile of logits is reduced in
// registers to its rows' maximum and sum of exponentials, and a second kernel joins the tiles.  Backward: per piece
// of the vocabulary the logits are formed again, turned into g and stored (at most kPieceBytes of it at a time), and
// one launch forms the piece's dW (complete) and adds its part of dx to fp32 sums.
//
// x is first packed: rows whose label is ignored are left out, the others lie next to each other, padded with zeros
// to whole tiles.  So ignored rows cost nothing, and whatever they hold (NaN too) enters nothing.
//
// fp32: x, W and g are split into three bf16 planes (8 bits of the significand each: all 24), and every product is
// the sum of six plane products.  The planes are rounded, so the second is at most 2^-8 of the number and the third 2^-17, of either
// sign: what is dropped is at most 2^-24 of the product (and a little: 2^-34), without a direction.  Six bf16 products are 2.7
// times as fast as one on the fp32 matrix instructions (peak rates).
//
// Forming the logits a second time is a quarter of all products; keeping them (or their exponentials) would take T V
// numbers, which is what this form is there to avoid.  Measured on MI355X, bf16, 16384 x 1024 tokens and 32000 words,
// loss and both gradients: 3.9 ms, of which packing 0.02, statistics 0.94 .. 1.05, the sums at the labels 0.04, per piece (of four) g
// 0.27 .. 0.31 and products 0.48 .. 0.52, joins and the last pass over dx 0.10: 1.1 PFLOP/s over the four products, where the library's
// largest product alone reaches 1.3 on the same card (and 1.07, 1.08, 0.80 at these three shapes).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <climits>

#include "common.hpp"
#include "mma_tiles.hpp"
#include "token_sort.hpp"

namespace cdssm {
namespace lce {

using namespace mma;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr double kLn2 = 0.69314718055994530942;
// What a piece's g may take.  Loss and gradients with 64 / 128 / 256 / 512 MB, ms: 16384 x 1024 x 32000 bf16 4.14 / 3.88 / 3.78 /
// 4.00 (from 512 MB on g no longer stays in the last-level cache between its two halves), 9995 x 768 x 50257 bf16 3.61 / 3.33 /
// 3.11 / 2.96, 2048 x 768 x 32000 fp32 2.25 / 2.36 / 2.37 / 2.28.
constexpr int64_t kPieceBytes = int64_t(256) << 20;
constexpr int kRowTile = 256, kPad = 64;  // packed rows fill whole tiles of either engine, their elements whole 128-byte lines
// Each workgroup of the packing counts the labels ahead of it: at most kPackGroups of them, so that a million labels are not
// read 32768 times.
constexpr int kPackRows = 32, kPackThreads = 512, kPackGroups = 1024, kTailGroups = kRowTile / kPackRows;
constexpr int kJoinGroups = 1024;  // each adds one to a counter in memory, some 20 ns
constexpr int kGroups = 256;    // persistent workgroups: one per CU
constexpr int kMinShare = 4;    // steps that are worth a workgroup
// Below so many tiles of 256 x 256 logits, too few for the CUs, bf16 takes tiles of 128.  Forward + backward with tiles of 256 and
// of 128, us: 7 x 1024 tokens, 2720 words (11 tiles) 34 + 84 and 25 + 45, 8088 x 512, 91 (32) 33 + 76 and 27 + 44, 16384 x 768,
// 97 (64) 46 + 104 and 38 + 74, 256 x 1024, 32000 (125) 40 + 144 and 48 + 166, 4096 x 1024, 2048 (128) 43 + 89 and 47 + 103.
constexpr int64_t kFewTiles = 96;

// The maximum is taken out before the factor log2 e: of logits beyond 10^9 the rounded product of the maximum is more than the
// exponent's range away from the exact one.
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

struct Header {
  int n_valid;        // rows whose label is not ignored
  unsigned arrived;   // workgroups of the join that have stored their sum
};

// The forward's state, which the backward reads.
struct State {
  Header* hdr;
  int *rowmap, *inv, *label;  // (Mp) row of a packed row; (T) packed row of a row or -1; (Mp) label or -1 where it is out of range
  float2* soft;               // (Mp) the largest logit m, and log2 sum_v e^(l - m)
  float* target;              // (Mp) the label's logit
  int* first;                 // (V) bf16: the first packed row with this label (once a backward has passed), INT_MAX for none
  double* sums;               // (kJoinGroups) the join's partial sums
  uint16_t *xp, *wp;          // packed x (planes, Mp, dp); packed W (planes, V, dp) or null
  float2* part;               // (tiles of V, Mp) a tile row's maximum and sum of e^(l - maximum)
  int64_t bytes;
};

__host__ __device__ inline int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

struct Shape {
  int64_t T, V, d, Mp, dp, planes, tile;
  bool pack_w;
};

static Shape make_shape(int dtype, const void* W, int64_t ldw, int64_t T, int64_t V, int64_t d) {
  Shape s{T, V, d, up(T, kRowTile), up(d, kPad), dtype == 0 ? 3 : 1, dtype == 0 || up(T, 256) / 256 * (up(V, 256) / 256) < kFewTiles ? 128 : 256, false};
  s.pack_w = dtype == 0 || d % kPad || ldw % 8 || (reinterpret_cast<uintptr_t>(W) & 15u);
  return s;
}

static State carve(const Shape& s, void* ws) {
  State st{};
  char* p = static_cast<char*>(ws);
  auto take = [&](int64_t bytes) {
    char* r = p;
    p += up(bytes, 256);
    return r;
  };
  st.hdr = reinterpret_cast<Header*>(take(sizeof(Header)));
  st.rowmap = reinterpret_cast<int*>(take(4 * s.Mp));
  st.inv = reinterpret_cast<int*>(take(4 * s.Mp));
  st.label = reinterpret_cast<int*>(take(4 * s.Mp));
  st.soft = reinterpret_cast<float2*>(take(8 * s.Mp));
  st.target = reinterpret_cast<float*>(take(4 * s.Mp));
  st.first = s.planes == 1 ? reinterpret_cast<int*>(take(4 * s.V)) : nullptr;
  st.sums = reinterpret_cast<double*>(take(8 * kJoinGroups));
  st.xp = reinterpret_cast<uint16_t*>(take(2 * s.planes * s.Mp * s.dp));
  st.wp = s.pack_w ? reinterpret_cast<uint16_t*>(take(2 * s.planes * s.V * s.dp)) : nullptr;
  st.part = reinterpret_cast<float2*>(take(8 * (up(s.V, s.tile) / s.tile) * s.Mp));
  st.bytes = p - static_cast<char*>(ws);
  return st;
}

// A value as the bf16 planes that stand for it, each in the high half of a word: one rounded value, or for fp32 three whose
// sum it is: the value rounded (cut off where that would be infinity), what that leaves rounded, and the rest, which has 7 bits at
// most.  Cut off instead, planes would leave products of up to 8 times as much out, all of the product's sign.
// Infinity and NaN stay in the first.
template <typename T>
struct Planes {
  static constexpr int n = T::bytes == 2 ? 1 : 3;
  uint32_t v[n];
  __device__ __forceinline__ static uint32_t rounded(float x) { return pack_bf16x2(0.0f, x); }
  __device__ __forceinline__ static float high(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
  __device__ __forceinline__ void set(float x) {
    v[0] = rounded(x);
    if constexpr (n == 3) {
      if (fabsf(x) <= FLT_MAX && !(fabsf(high(v[0])) <= FLT_MAX)) v[0] = __float_as_uint(x);
      const float r = fabsf(x) <= FLT_MAX ? x - high(v[0]) : 0.0f;
      v[1] = rounded(r);
      v[2] = __float_as_uint(r - high(v[1]));
    }
  }
};
// Plane p of two values as a pair.
template <typename T>
__device__ __forceinline__ uint32_t pair_of(const Planes<T>& a, const Planes<T>& b, int p) {
  return a.v[p] >> 16 | (b.v[p] & 0xffff0000u);
}

// Elements c .. c + 8 of a row of d elements into planes of rows of dp (dp a multiple of 64), zeros behind the row; src null:
// zeros.  vec: the row can be read 16 bytes at a time.
template <typename T>
struct Eight {
  float x[8];
  uint4 raw;
  __device__ __forceinline__ void load(const typename T::raw* src, int c, int d, bool vec) {
    raw = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = 0.0f;
    if (!src || c >= d) return;
    if (vec && c + 8 <= d) {
      if constexpr (T::bytes == 2) {
        raw = *reinterpret_cast<const uint4*>(src + c);
      } else {
        const float4 a = *reinterpret_cast<const float4*>(src + c), b = *reinterpret_cast<const float4*>(src + c + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
      }
      return;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (c + u < d) x[u] = T::load(src + c + u);
    if constexpr (T::bytes == 2)
      raw = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
  }
  __device__ __forceinline__ void store(uint16_t* dst, int64_t plane, int c) const {
    if constexpr (T::bytes == 2) {
      *reinterpret_cast<uint4*>(dst + c) = raw;
    } else {
      Planes<T> e[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) e[u].set(x[u]);
#pragma unroll
      for (int p = 0; p < 3; ++p)
        *reinterpret_cast<uint4*>(dst + p * plane + c) =
            make_uint4(pair_of(e[0], e[1], p), pair_of(e[2], e[3], p), pair_of(e[4], e[5], p), pair_of(e[6], e[7], p));
    }
  }
};

template <typename T>
__device__ __forceinline__ bool rows_of_16_bytes(const void* p, int64_t ld) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld * T::bytes % 16 == 0;
}

// rows(r, dst) tells the source of row r of n (null: zeros) and, in dst, its packed row (-1: none); all of them by the whole
// workgroup, four pieces of a thread under way at a time.
template <typename T, int Threads, typename F>
__device__ __forceinline__ void pack_rows(int n, uint16_t* out, int64_t plane, const Shape& s, bool vec, F&& rows) {
  const int per = int(s.dp / 8), all = n * per;
  for (int i0 = threadIdx.x; i0 < all; i0 += 4 * Threads) {
    Eight<T> e[4];
    int at[4], c[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * Threads, r = i / per;
      at[u] = -1;
      c[u] = (i - r * per) * 8;
      if (i < all) {
        const typename T::raw* src = rows(r, at[u]);
        if (at[u] >= 0) e[u].load(src, c[u], int(s.d), vec);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (at[u] >= 0) e[u].store(out + at[u] * s.dp, plane, c[u]);
  }
}

template <typename I>
__device__ __forceinline__ int count_valid(const I* labels, int64_t n, int64_t ignore) {
  int c = 0;
#pragma unroll 8
  for (int64_t t = threadIdx.x; t < n; t += kPackThreads) c += int64_t(labels[t]) != ignore;
  return c;
}

// Packs x (16384 x 1024 bf16: 19 us, 3.5 TB/s): a workgroup `groups` times 32 rows, behind the valid rows ahead of them, which
// it counts itself (the labels are small); eight more fill up the last tile with zeros, and where W has to be packed as well the rest
// take 32 of its rows each.  With loss: the loss of ignored rows, 0.
template <typename T, typename I>
__global__ __launch_bounds__(kPackThreads) void pack_kernel(const typename T::raw* __restrict__ x, int64_t ldx,
                                                            const I* __restrict__ labels, int64_t ignore, float* loss,
                                                            const typename T::raw* __restrict__ W, int64_t ldw, State st, Shape s,
                                                            int groups) {
  __shared__ int wsum[kPackThreads / kWave];
  __shared__ int place[kPackRows];
  __shared__ int taken;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int rows = groups * kPackRows, nb = int((s.T + rows - 1) / rows), b = blockIdx.x;
  if (b >= nb + kTailGroups) {
    const int64_t r0 = int64_t(b - nb - kTailGroups) * kPackRows;
    pack_rows<T, kPackThreads>(int(min(int64_t(kPackRows), s.V - r0)), st.wp, s.V * s.dp, s, rows_of_16_bytes<T>(W, ldw),
                               [&](int r, int& at) {
                                 at = int(r0) + r;
                                 return W + (r0 + r) * ldw;
                               });
    return;
  }
  if (st.first)
    for (int64_t v = int64_t(b) * kPackThreads + tid; v < s.V; v += int64_t(nb + kTailGroups) * kPackThreads) st.first[v] = INT_MAX;
  const bool tail = b >= nb;
  const int64_t begin = tail ? s.T : int64_t(b) * rows, end = min(s.T, begin + rows);
  int c = count_valid(labels, begin, ignore);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, kWave);
  if (lane == 0) wsum[wave] = c;
  __syncthreads();
  int base = 0;
#pragma unroll
  for (int w = 0; w < kPackThreads / kWave; ++w) base += wsum[w];
  const bool vec = rows_of_16_bytes<T>(x, ldx);
  const int64_t plane = s.Mp * s.dp;
  if (tail) {
    const int e = b - nb, pad = int(up(base, kRowTile));
    if (e == 0 && tid == 0) {
      st.hdr->n_valid = base;
      st.hdr->arrived = 0;
    }
    const int r0 = base + e * kPackRows, n = min(kPackRows, pad - r0);
    if (n <= 0) return;
    if (tid < n) {
      st.rowmap[r0 + tid] = -1;
      st.label[r0 + tid] = -1;
    }
    pack_rows<T, kPackThreads>(n, st.xp, plane, s, vec, [&](int r, int& at) -> const typename T::raw* {
      at = r0 + r;
      return nullptr;
    });
    return;
  }
  for (int64_t t0 = begin; t0 < end; t0 += kPackRows) {
    if (tid < kWave) {
      const int64_t t = t0 + lane;
      const bool in = lane < kPackRows && t < s.T;
      const int64_t y = in ? int64_t(labels[t]) : ignore;
      const bool ok = in && y != ignore;
      const uint64_t m = __ballot(ok);
      const int at = ok ? base + __popcll(m & ((1ull << lane) - 1)) : -1;
      if (lane < kPackRows) place[lane] = at;
      if (lane == 0) taken = __popcll(m);
      if (in) {
        st.inv[t] = at;
        if (!ok && loss) loss[t] = 0.0f;
      }
      if (ok) {
        st.rowmap[at] = int(t);
        st.label[at] = y >= 0 && y < s.V ? int(y) : -1;
      }
    }
    __syncthreads();
    base += taken;
    pack_rows<T, kPackThreads>(kPackRows, st.xp, plane, s, vec, [&](int r, int& at) {
      at = place[r];
      return x + (t0 + r) * ldx;
    });
    __syncthreads();
  }
}

// The two operands of a tile of logits: A = rows of W from v0, B = packed rows of x from t0.
struct Logits {
  const uint16_t* w;
  int64_t ldw, w_plane;
  State st;
  Shape s;
  int v0, v1;  // the piece of the vocabulary
};

// The tiles of a piece's logits, walked by persistent workgroups: a band of 8 token tiles x 4 word tiles for the 32
// workgroups of an XCD at a time.  tile(k): a workgroup's k-th.
template <int kTile>
struct Walk {
  int nt, nv, at;
  __device__ __forceinline__ Walk(const Logits& a) {
    nt = (a.st.hdr->n_valid + kTile - 1) / kTile;
    nv = (a.v1 - a.v0 + kTile - 1) / kTile;
    at = xcd_place(blockIdx.x, gridDim.x);
  }
  __device__ __forceinline__ bool tile(int& vt, int& tt) const {
    if (at >= int64_t(nt) * nv) return false;
    banded(at, nt, nv, 8, tt, vt);
    return true;
  }
};

template <typename E>
__device__ __forceinline__ void start_logits(typename E::template Multiply<false, false, true>& m, const Logits& a, int vt, int tt) {
  const int64_t v = a.v0 + int64_t(vt) * E::kTile, t = int64_t(tt) * E::kTile;
  m.start(Operand{a.w + v * a.ldw, a.ldw, a.w_plane, (a.s.V - v - 1) * a.ldw + a.s.dp},
          Operand{a.st.xp + t * a.s.dp, a.s.dp, a.s.Mp * a.s.dp, (a.s.Mp - t) * a.s.dp}, 0, int(a.s.dp / E::kStep));
}

// Forward: a tile's statistics, and the labels' logits.  The next tile's first steps are requested before the
// statistics are taken; those are some 4 VALU instructions and an exponential a logit, a tenth of the time at 1024 k.
template <typename E>
__global__ __launch_bounds__(kThreads) void stats_kernel(Logits a) {
  constexpr int kTile = E::kTile, kI = E::kI, kJ = E::kJ;
  __shared__ alignas(1024) unsigned char lds[E::kLdsBytes];
  __shared__ float2 red[2][kTile];
  Walk<kTile> walk(a);
  int vt, tt;
  bool more = walk.tile(vt, tt);
  if (!more) return;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, lo = lane & 15, g = lane >> 4;
  const int wm = E::wave_m(wave), wn = E::wave_n(wave);
  typename E::template Multiply<false, false, true> m((lds_byte*)lds);
  start_logits<E>(m, a, vt, tt);
  while (more) {
    typename E::Acc acc;
    E::clear(acc);
    m.template run<0>(acc);
    const int vb = a.v0 + vt * kTile + wm, t0 = tt * kTile;
    float2* part = a.st.part + int64_t(vt) * a.s.Mp + t0;
    const bool edge = a.v0 + (vt + 1) * kTile > a.s.V;
    walk.at += gridDim.x;
    more = walk.tile(vt, tt);
    if (more) start_logits<E>(m, a, vt, tt);
    if (edge) {
#pragma unroll
      for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (vb + frag_row<true>(i, 4 * g + r) >= a.s.V)
#pragma unroll
            for (int j = 0; j < kJ; ++j) acc[i][j][r] = -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      const int tl = wn + 16 * j + lo, t = t0 + tl;
      const int rel = a.st.label[t] - vb;
      if (rel >= 0 && rel < E::kWM && ((rel >> 3) & 3) == g) {
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < kI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (rel - 8 * g == frag_row<true>(i, r)) v = acc[i][j][r];
        a.st.target[t] = v;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, acc[i][j][r]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
      mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
      mx = fmaxf(mx, -FLT_MAX);  // finite where every logit is -inf: its terms are 2^-inf, not NaN
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum += exp_of(acc[i][j][r] - mx);
      sum += __shfl_xor(sum, 16, kWave);
      sum += __shfl_xor(sum, 32, kWave);
      if (g == 0) red[wm != 0][tl] = make_float2(mx, sum);
    }
    __syncthreads();
    if (threadIdx.x < kTile) {
      const float2 p = red[0][threadIdx.x], q = red[1][threadIdx.x];
      const float mm = fmaxf(p.x, q.x);
      part[threadIdx.x] = make_float2(mm, p.y * exp_of(p.x - mm) + q.y * exp_of(q.x - mm));
    }
  }
}

// Joins the tiles' statistics of 64 packed rows at a time, a quarter of the tiles to a wave; none: a row's loss to its place, else
// the sum over all rows (in a fixed order: the last workgroup adds the workgroups' sums), divided by the count for a mean.
// The log in fp64: loss = maximum + log of the sum - the label's logit is a difference of numbers that may be much larger than it.
__global__ __launch_bounds__(256) void join_kernel(State st, Shape s, int nv, int reduction, float* loss) {
  __shared__ float2 quarter[4][kWave];
  __shared__ double acc[256];
  __shared__ bool last;
  const int n_valid = st.hdr->n_valid, tid = threadIdx.x, wave = tid / kWave;
  double total_l = 0.0;
  for (int64_t r0 = int64_t(blockIdx.x) * kWave; r0 < s.Mp; r0 += int64_t(gridDim.x) * kWave) {
    const int64_t t = r0 + tid % kWave;
    float m = -FLT_MAX, sum = 0.0f;
    if (r0 < n_valid) {
      const float2* part = st.part + t;
      constexpr int U = 8;
      for (int v = wave; v < nv; v += 4 * U) {
        float2 p[U];
#pragma unroll
        for (int u = 0; u < U; ++u) p[u] = v + 4 * u < nv ? part[int64_t(v + 4 * u) * s.Mp] : make_float2(-FLT_MAX, 0.0f);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float n = fmaxf(m, p[u].x);
          sum = sum * exp_of(m - n) + p[u].y * exp_of(p[u].x - n);
          m = n;
        }
      }
    }
    quarter[wave][tid % kWave] = make_float2(m, sum);
    __syncthreads();
    if (wave == 0 && t < n_valid) {
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        const float2 p = quarter[w][tid];
        const float n = fmaxf(m, p.x);
        sum = sum * exp_of(m - n) + p.y * exp_of(p.x - n);
        m = n;
      }
      const double log_sum = log(double(sum));
      st.soft[t] = make_float2(m, st.label[t] < 0 ? NAN : float(log_sum * (1.0 / kLn2)));
      const double l = st.label[t] < 0 ? double(NAN) : double(m) + log_sum - double(st.target[t]);
      if (reduction == 0) loss[st.rowmap[t]] = float(l);
      total_l += l;
    } else if (wave == 0) {
      st.soft[t] = make_float2(0.0f, 0.0f);
    }
    __syncthreads();
  }
  if (reduction == 0) return;
  auto total = [&](double x) {
    acc[tid] = x;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
      if (tid < o) acc[tid] += acc[tid + o];
      __syncthreads();
    }
    return acc[0];
  };
  total_l = total(total_l);
  if (tid == 0) {
    __hip_atomic_store(&st.sums[blockIdx.x], total_l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = __hip_atomic_fetch_add(&st.hdr->arrived, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  double v = 0.0;
  for (int i = tid; i < int(gridDim.x); i += 256) v += __hip_atomic_load(&st.sums[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  v = total(v);
  if (tid == 0) *loss = float(reduction == 1 ? v / double(n_valid) : v);
}

// e^(l - lse) with the maximum taken out, as in the forward: l - m is exact where it counts, while lse itself in fp32 is off by half a
// step of the largest logit (a word of probability 1 at a logit of 10^6 would get 0.9).  At most 1: the logits of both directions are
// the same bits, so l <= m, and the sum has a term of 1.
__device__ __forceinline__ float probability(float l, float2 soft) {
  return __builtin_amdgcn_exp2f(fmaf(l - soft.x, kLog2e, -soft.y));
}

// What rounding to bf16 takes from the g of packed row t at its label: formed again from the forward's logit, which is the
// backward's to the bit (the same products in the same order).
__device__ __forceinline__ float left_at_label(const State& st, int64_t t, const float* up) {
  float p = probability(st.target[t], st.soft[t]) - 1.0f;
  if (up) p *= up[st.rowmap[t]];
  const float left = p - __uint_as_float(pack_bf16x2(0.0f, p) & 0xffff0000u);
  return fabsf(left) < FLT_MAX ? left : 0.0f;  // else g itself is NaN, or infinite
}

// Backward, first half: a tile of g into the piece's store (planes, Mp, ldg).  up: a factor for each row (reduction
// none), else null: g is stored without the common factor, which the products' results take, so that the -1 at a
// label's place stays exact in bf16.  In bf16 every other value of g is rounded once (2^-8 of itself): it has to
// enter the matrix cores as bf16, and the products' sums over many tokens or words average the roundings.  Not so at the label,
// whose g is most of a row of dx and of dW, and whose rounding has a direction (a p below 2^-9 is lost from every p - 1): what it
// leaves is added to the results in fp32, in finish_kernel and (rests_kernel) store_dw.  The stores
// (16 bytes a lane, 64 to a row) drain while the next tile's first steps run.
template <typename T, typename E>
__global__ __launch_bounds__(kThreads) void grad_kernel(Logits a, const float* up, uint16_t* G, int64_t ldg) {
  constexpr int kTile = E::kTile, kI = E::kI, kJ = E::kJ;
  __shared__ alignas(1024) unsigned char lds[E::kLdsBytes];
  const int n_valid = a.st.hdr->n_valid;
  Walk<kTile> walk(a);
  int vt, tt;
  bool more = walk.tile(vt, tt);
  if (!more) return;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, lo = lane & 15, g = lane >> 4;
  const int wm = E::wave_m(wave), wn = E::wave_n(wave);
  typename E::template Multiply<false, false, true> m((lds_byte*)lds);
  start_logits<E>(m, a, vt, tt);
  bool first = true;
  while (more) {
    typename E::Acc acc;
    E::clear(acc);
    // the last tile's stores, 16 of every plane, came after the requests for this one
    if (first)
      m.template run<0>(acc);
    else
      m.template run<kI / 2 * kJ * Planes<T>::n>(acc);
    first = false;
    const int vl = vt * kTile + wm + 8 * g, vb = a.v0 + vl, t0 = tt * kTile;
    const bool edge = a.v0 + (vt + 1) * kTile > a.s.V || t0 + kTile > n_valid;
    walk.at += gridDim.x;
    more = walk.tile(vt, tt);
    if (more) start_logits<E>(m, a, vt, tt);
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      const int t = t0 + wn + 16 * j + lo;
      const bool ok = t < n_valid;
      const float2 soft = a.st.soft[t];
      const float f = !up ? 1.0f : ok ? up[a.st.rowmap[t]] : 0.0f;
      const int rel = a.st.label[t] - vb;
      const bool hot = rel >= 0 && rel < E::kWM && (rel & 31) < 8;
      uint16_t* row = G + t * ldg + vl;
#pragma unroll
      for (int i = 0; i < kI; i += 2) {
        Planes<T> e[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          float p = probability(acc[i + r / 4][j][r % 4], soft);
          if (hot && rel == 16 * i + r) p -= 1.0f;
          if (up) p *= f;
          if (edge && (!ok || vb + 16 * i + r >= a.s.V)) p = 0.0f;
          e[r].set(p);
        }
#pragma unroll
        for (int p = 0; p < Planes<T>::n; ++p)
          *reinterpret_cast<uint4*>(row + p * a.s.Mp * ldg + 16 * i) =
              make_uint4(pair_of(e[0], e[1], p), pair_of(e[2], e[3], p), pair_of(e[4], e[5], p), pair_of(e[6], e[7], p));
      }
    }
  }
}

// bf16: what the rounding of g at the labels leaves of dW: sums[first row with a label] = sum over the rows t with it of
// left_at_label(t) x[t], fp32, in the rows' order; and State::first, the same in every backward.  A wave takes 512 columns.
constexpr int kRestColumns = kWave * 8;

struct Rests {
  State st;
  Shape s;
  const float* up;
  float* sums;       // (Mp, dp)
  const int* order;  // rows by label (token_sort.hpp), and where each label's are
  const int2* rows;
  int chunk;         // sorted rows to a wave

  __device__ __forceinline__ f32x4_t* at(int t, int64_t col) const { return reinterpret_cast<f32x4_t*>(sums + t * s.dp + col); }
};

// The wave's place among rows (chunks) x blocks of columns, and its lane's first column.  Loads below have no branches around them
// (the compiler would wait for each): a lane behind the last column reads the last ones, a row that does not count another.
__device__ __forceinline__ int64_t rest_place(const Rests& a, int64_t& col) {
  const int64_t w = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int64_t per = (a.s.dp + kRestColumns - 1) / kRestColumns, at = w / per;
  col = (w - at * per) * kRestColumns + int(threadIdx.x % kWave) * 8;
  return at;
}

// The sum over rows of one label, eight columns of it.
struct RestSum {
  float v[8];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
  }
  __device__ __forceinline__ void add(float left, const uint4& x) {
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fmaf(left, i & 1 ? bf16_hi(u[i / 2]) : bf16_lo(u[i / 2]), v[i]);
  }
  __device__ __forceinline__ void store(f32x4_t* p) const {
    p[0] = f32x4_t{v[0], v[1], v[2], v[3]};
    p[1] = f32x4_t{v[4], v[5], v[6], v[7]};
  }
};

// Few rows: a wave per row, which sums if it is its label's first; it looks through all labels, and lists the rows with its own in LDS.
// Loss and both gradients so and by the three launches below, us: 200 x 128 tokens, 97 words 46 and 53, 512 x 768, 5000 93 and 100, but
// 1024 x 128, 97 69 and 57, and where a wave has nearly all rows, 512 x 64 and one word, 93 and 52: so with eight rows to a word at most.
constexpr int kFewRows = 512, kFewToWord = 8;
__global__ __launch_bounds__(256) void few_rests_kernel(Rests a) {
  __shared__ int rows[4][kFewRows];
  __shared__ float lefts[4][kFewRows];
  const int n_valid = a.st.hdr->n_valid, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int64_t col;
  const int64_t at = rest_place(a, col);
  if (at >= n_valid) return;
  const int t = int(at), y = a.st.label[t];
  if (y < 0) return;
  int labels[kFewRows / kWave];
#pragma unroll
  for (int i = 0; i < kFewRows / kWave; ++i) {
    const int r = i * kWave + lane;
    labels[i] = r < n_valid ? a.st.label[r] : -1;
  }
  int n = 0;
#pragma unroll
  for (int i = 0; i < kFewRows / kWave; ++i) {
    const int r = i * kWave + lane;
    const uint64_t same = __ballot(labels[i] == y);
    if (n == 0 && same && i * kWave + __builtin_ctzll(same) < t) return;  // another row is the first
    if (labels[i] == y) {
      const int k = n + __popcll(same & ((uint64_t(1) << lane) - 1));
      rows[wave][k] = r;
      lefts[wave][k] = left_at_label(a.st, r, a.up);
    }
    n += __popcll(same);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (col < kRestColumns && lane == 0) a.st.first[y] = t;
  if (col >= a.s.dp) return;
  RestSum sum;
  sum.clear();
  constexpr int U = 16;
  for (int k = 0; k < n; k += U) {
    uint4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const uint4*>(a.st.xp + rows[wave][min(k + u, n - 1)] * a.s.dp + col);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u < n) sum.add(lefts[wave][k + u], x[u]);
  }
  sum.store(a.at(t, col));
}

// More rows: they are sorted by label, then a wave sums a chunk of them and leaves a sum for each label there, at the label's first row
// in the chunk; a third launch adds those of the labels that go on into later chunks.  At most kRestChunks chunks or so, that one
// label's do not become a long chain.  At 16384 x 1024, 32000 words: 11, 16 and 13 us, chains of look-ups.  (One level of
// sorting is enough: its reads, rows x words / 256, are few beside the products of rows x words.)
constexpr int kRestRows = 32, kRestChunks = 1024;

__global__ __launch_bounds__(token_sort::kSortThreads) void sort_labels_kernel(State st, int* order, int2* rows, int64_t V, int shift) {
  token_sort::sort<int>(st.label, order, rows, st.hdr->n_valid, V, -1, shift);
}

// The label of place p < n_valid of the order, its row and its places; -1 where the order has come to its end (rows whose label is out
// of range are not in it, and what it holds there is anything).
__device__ __forceinline__ int label_at(const Rests& a, int p, int n_valid, int& t, int2& r) {
  t = a.order[p];
  bool ok = t >= 0 && t < n_valid;
  t = ok ? t : 0;
  const int y = a.st.label[t];
  r = a.rows[max(y, 0)];
  ok = ok && y >= 0 && p >= r.x && p < r.x + r.y;
  return ok ? y : -1;
}

__global__ __launch_bounds__(256) void rests_kernel(Rests a) {
  const int n_valid = a.st.hdr->n_valid, lane = threadIdx.x % kWave;
  int64_t col;
  const int64_t p0 = rest_place(a, col) * a.chunk, end = min(p0 + a.chunk, int64_t(n_valid));
  const bool in = col < a.s.dp, marks = col < kRestColumns;
  RestSum sum;
  int word = -1, to = 0;
  for (int64_t p = p0; p < end; p += kRestRows) {
    int t;
    int2 r;
    int y = label_at(a, int(min(p + lane, end - 1)), n_valid, t, r);
    const float left = left_at_label(a.st, t, a.up);
    if (lane >= kRestRows || p + lane >= end) y = -1;
    if (marks && y >= 0 && p + lane == r.x) a.st.first[y] = t;
    uint4 x[kRestRows];
#pragma unroll
    for (int u = 0; u < kRestRows; ++u)
      x[u] = *reinterpret_cast<const uint4*>(a.st.xp + __builtin_amdgcn_readlane(t, u) * a.s.dp + min(col, a.s.dp - 8));
#pragma unroll
    for (int u = 0; u < kRestRows; ++u) {
      const int yu = __builtin_amdgcn_readlane(y, u);
      if (yu != word) {
        if (word >= 0 && in) sum.store(a.at(to, col));
        sum.clear();
        word = yu;
        to = __builtin_amdgcn_readlane(t, u);
      }
      if (yu >= 0) sum.add(__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(left), u)), x[u]);
    }
  }
  if (word >= 0 && in) sum.store(a.at(to, col));
}

// The wave of the chunk that a label begins in adds what later chunks have of it.
__global__ __launch_bounds__(256) void join_rests_kernel(Rests a) {
  const int n_valid = a.st.hdr->n_valid;
  int64_t col;
  const int64_t p0 = rest_place(a, col) * a.chunk, p1 = p0 + a.chunk;
  if (p1 >= n_valid) return;
  int t;
  int2 r;
  if (label_at(a, int(p1) - 1, n_valid, t, r) < 0 || r.x < p0 || r.x + r.y <= p1 || col >= a.s.dp) return;
  f32x4_t* to = a.at(a.order[r.x], col);
  f32x4_t x = to[0], y = to[1];
  constexpr int U = 8;
  const int64_t end = r.x + r.y, step = a.chunk;
  for (int64_t p = p1; p < end; p += U * step) {
    int row[U];
    f32x4_t v[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) row[u] = a.order[min(p + u * step, end - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const f32x4_t* q = a.at(row[u], col);
      v[u][0] = q[0];
      v[u][1] = q[1];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (p + u * step < end)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] += v[u][0][i];
          y[i] += v[u][1][i];
        }
  }
  to[0] = x;
  to[1] = y;
}

struct Products {
  const uint16_t* w;  // rows of W from the piece's first
  int64_t ldw, w_plane;
  const uint16_t* G;
  int64_t ldg, nv;    // columns of G in memory, and rows of W in the piece
  State st;
  Shape s;
  float* dx;          // (Mp, dp) fp32 sums, or null
  void* dw;           // dW from the piece's first row, or null
  int64_t ldo;
  const float* gloss; // the upstream gradient of a mean or sum, or null
  int reduction;
  bool add;           // dx already holds the sums of earlier pieces
  f32x4_t* slots;     // (kGroups, 2) tiles of partial sums
  const int* first;   // bf16: each word's first row, from the piece's first word; and at it what is left of dW (rests_kernel)
  const float* rests;
};

// The common factor of a mean or sum; no valid row: 0 (there is nothing to take the gradient of).
__device__ __forceinline__ float common_factor(const float* gloss, int reduction, int n_valid) {
  if (!gloss) return 1.0f;
  return reduction == 1 ? (n_valid > 0 ? *gloss / float(n_valid) : 0.0f) : *gloss;
}

template <typename T>
__device__ __forceinline__ void store4(typename T::raw* p, const f32x4_t& v, float f, int n, bool vec) {
  if (vec && n >= 4) {
    if constexpr (T::bytes == 2)
      *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0] * f, v[1] * f), pack_bf16x2(v[2] * f, v[3] * f));
    else
      *reinterpret_cast<float4*>(p) = make_float4(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
    return;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (r < n) T::store(p + r, v[r] * f);
}

// v += f x, four bf16 of a packed row (8-byte aligned).
__device__ __forceinline__ void add_scaled(f32x4_t& v, float f, const uint16_t* x) {
  const uint2 u = *reinterpret_cast<const uint2*>(x);
  v[0] = fmaf(f, bf16_lo(u.x), v[0]);
  v[1] = fmaf(f, bf16_hi(u.x), v[1]);
  v[2] = fmaf(f, bf16_lo(u.y), v[2]);
  v[3] = fmaf(f, bf16_hi(u.y), v[3]);
}

// Backward, second half: dW of the piece (over all rows) and the piece's part of dx, cut into equal shares: the steps of all
// tiles of dW, then those of dx, stand in one row, and workgroup g of n takes the stretch from g total / n to (g + 1) total / n.
// A tile that a share ends in goes to several workgroups; each leaves its sums in a slot (its first tile's in slot 0,
// its last one's, that it began, in slot 1), and join_tiles_kernel adds them in order.  So every CU has the same work whatever the
// shape, and the number of valid rows, which only the device knows, counts.  Against whole tiles and equal parts of tiles,
// 9995 x 768 x 50257 (258 tiles of 141 and 200 steps a piece) took 411 us a piece instead of 737; the slots and their sum cost 51 of
// them there, 13 where the shares end with the tiles.
// Where tiles have few steps (few tokens, or few words), a tile's first loads and its stores are longer than its products and count as
// steps of their own, `around`, before its first: else the workgroups with tiles of one step each have most of the work.  Both gradients
// without and with them, us: 19 x 200 tokens, 49872 words 112 and 76, 512 x 768, 50257 245 and 217, 25 x 768, 15915 in fp32 152 and 108; at
// 16384 x 1024, 32000, where shares without them end with the tiles, 2892 and 3122.
template <typename E>
struct Cut {
  static constexpr int kTile = E::kTile, kStep = E::kStep, kAround = kTile == 256 ? 4 : 8;
  int64_t steps_w, steps_x, units_w, units_x, all_w, all, groups;
  int nd, vt, nk_w, nk_x, tiles_w, tiles_x, around;
  __device__ __forceinline__ Cut(const Products& a, int n_valid, int groups_) {
    nd = int((a.s.dp + kTile - 1) / kTile);
    vt = int(a.ldg / kTile);
    nk_w = (n_valid + kStep - 1) / kStep;
    nk_x = int((a.nv + kStep - 1) / kStep);
    tiles_w = a.dw ? vt * nd : 0;
    tiles_x = a.dx ? (n_valid + kTile - 1) / kTile * nd : 0;
    steps_w = nk_w;
    steps_x = nk_x;
    const int least = min(a.dw ? nk_w : INT_MAX, a.dx ? nk_x : INT_MAX);
    around = least < 4 * kAround ? kAround : 0;
    units_w = steps_w + around;
    units_x = steps_x + around;
    all_w = tiles_w * units_w;
    all = all_w + tiles_x * units_x;
    groups = max(int64_t(1), min(int64_t(groups_), all / (kMinShare + around)));
  }
  __device__ __forceinline__ int64_t from(int64_t g) const { return g * all / groups; }
  __device__ __forceinline__ int owner(int64_t unit) const { return int(((unit + 1) * groups + all - 1) / all - 1); }
};

// The first rows of a lane's words in a tile of dW.
template <typename T, typename E>
struct FirstRows {
  int row[E::kJ];
  __device__ __forceinline__ FirstRows(const Products& a, int vt) {
#pragma unroll
    for (int j = 0; j < E::kJ; ++j) {
      const int64_t v = int64_t(vt) * E::kTile + E::wave_n(threadIdx.x / kWave) + 16 * j + int(threadIdx.x % 16);
      row[j] = Planes<T>::n == 1 && v < a.nv ? a.first[v] : INT_MAX;
    }
  }
};

// Fragments i0 .. i0 + N of a tile's results to where they belong.
template <typename T, typename E, int N>
__device__ __forceinline__ void store_dw(const Products& a, const Cut<E>& c, int tile, int n_valid, int i0,
                                         const f32x4_t (&acc)[N][E::kJ], const FirstRows<T, E>& rows) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, lo = lane & 15, g = lane >> 4;
  const int dt = tile % c.nd, vt = tile / c.nd;
  const float f = common_factor(a.gloss, a.reduction, n_valid);
  const bool vec = a.ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(a.dw) & (4 * T::bytes - 1)) == 0;
#pragma unroll
  for (int j = 0; j < E::kJ; ++j) {
    const int64_t v = vt * E::kTile + E::wave_n(wave) + 16 * j + lo;
    if (v >= a.nv) continue;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t d = dt * E::kTile + E::wave_m(wave) + 16 * (i0 + i) + 4 * g;
      if (d >= a.s.d) continue;
      f32x4_t sum = acc[i][j];
      if (rows.row[j] < n_valid) {
        const f32x4_t rest = *reinterpret_cast<const f32x4_t*>(a.rests + rows.row[j] * a.s.dp + d);
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[r] += rest[r];
      }
      store4<T>(static_cast<typename T::raw*>(a.dw) + v * a.ldo + d, sum, f, int(a.s.d - d), vec);
    }
  }
}

template <typename E, int N>
__device__ __forceinline__ void store_dx(const Products& a, const Cut<E>& c, int tile, int n_valid, int i0,
                                         const f32x4_t (&acc)[N][E::kJ]) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, lo = lane & 15, g = lane >> 4;
  const int dt = tile % c.nd, tt = tile / c.nd;
#pragma unroll
  for (int j = 0; j < E::kJ; ++j) {
    const int64_t t = int64_t(tt) * E::kTile + E::wave_n(wave) + 16 * j + lo;
    if (t >= n_valid) continue;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t d = dt * E::kTile + E::wave_m(wave) + 16 * (i0 + i) + 4 * g;
      if (d >= a.s.dp) continue;
      f32x4_t* p = reinterpret_cast<f32x4_t*>(a.dx + t * a.s.dp + d);
      f32x4_t v = acc[i][j];
      if (a.add) {
        const f32x4_t o = *p;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += o[r];
      }
      *p = v;
    }
  }
}

// How many of the wave's fragment columns of tile `other` (along the words for dW, the tokens for dx) have anything that is
// kept: with a few tokens most of a tile has not.
template <typename E>
__device__ __forceinline__ int columns_kept(const Products& a, bool w, int other, int n_valid) {
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int64_t left = (w ? a.nv : int64_t(n_valid)) - int64_t(other) * E::kTile - E::wave_n(wave);
  return int(max(int64_t(0), min(int64_t(E::kJ), (left + 15) / 16)));
}

template <typename E>
__device__ __forceinline__ f32x4_t* slot_of(const Products& a, int g, int which) {
  return a.slots + (int64_t(g) * 2 + which) * (E::kI * E::kJ * kThreads);
}

template <typename T, typename E>
__global__ __launch_bounds__(kThreads) void products_kernel(Products a) {
  constexpr int kTile = E::kTile, kI = E::kI, kJ = E::kJ;
  __shared__ alignas(1024) unsigned char lds[E::kLdsBytes];
  const int n_valid = a.st.hdr->n_valid;
  const Cut<E> c(a, n_valid, gridDim.x);
  typename E::Acc acc;
  if (c.nk_w == 0) {  // no row: dW is zero
    E::clear(acc);
    for (int tile = blockIdx.x; tile < c.tiles_w; tile += gridDim.x) store_dw<T, E, kI>(a, c, tile, n_valid, 0, acc, FirstRows<T, E>(a, tile / c.nd));
    return;
  }
  const int me = xcd_place(blockIdx.x, gridDim.x);
  if (me >= c.groups) return;
  int64_t at = c.from(me);
  const int64_t end = c.from(me + 1);
  while (at < end) {
    const bool w = at < c.all_w;
    const int64_t rel = w ? at : at - c.all_w, steps = w ? c.steps_w : c.steps_x, units = w ? c.units_w : c.units_x;
    const int tile = int(rel / units), u0 = int(rel - tile * units), u1 = int(min(units, u0 + (end - at)));
    const int q0 = max(0, u0 - c.around), q1 = max(0, u1 - c.around);
    at += u1 - u0;
    if (q0 == q1) continue;
    const int d0 = tile % c.nd * kTile, other = tile / c.nd;
    E::clear(acc);
    if (w) {
      typename E::template Multiply<true, true> m((lds_byte*)lds);
      m.start(Operand{a.st.xp + d0, a.s.dp, a.s.Mp * a.s.dp, a.s.Mp * a.s.dp - d0},
              Operand{a.G + other * kTile, a.ldg, a.s.Mp * a.ldg, a.s.Mp * a.ldg - other * kTile}, q0, q1);
      m.template run<0>(acc);
    } else {
      typename E::template Multiply<true, false> m((lds_byte*)lds);
      const int64_t t = int64_t(other) * kTile;
      m.start(Operand{a.w + d0, a.ldw, a.w_plane, (a.nv - 1) * a.ldw + a.s.dp - d0},
              Operand{a.G + t * a.ldg, a.ldg, a.s.Mp * a.ldg, (a.s.Mp - t) * a.ldg}, q0, q1);
      m.template run<0>(acc);
    }
    if (q1 - q0 < steps) {
      f32x4_t* s = slot_of<E>(a, me, q0 == 0);
      const int kept = columns_kept<E>(a, w, other, n_valid);
#pragma unroll
      for (int j = 0; j < kJ; ++j)
        if (j < kept)
#pragma unroll
          for (int i = 0; i < kI; ++i) s[(i * kJ + j) * kThreads + threadIdx.x] = acc[i][j];
    } else if (w) {
      store_dw<T, E, kI>(a, c, tile, n_valid, 0, acc, FirstRows<T, E>(a, other));
    } else {
      store_dx<E, kI>(a, c, tile, n_valid, 0, acc);
    }
  }
}

// Tile blockIdx.x, fragments blockIdx.y: the sum of its slots, if it has any.
template <typename T, typename E>
__global__ __launch_bounds__(kThreads) void join_tiles_kernel(Products a, int groups) {
  constexpr int kJ = E::kJ;
  const int n_valid = a.st.hdr->n_valid, i = blockIdx.y;
  const Cut<E> c(a, n_valid, groups);
  const bool w = int(blockIdx.x) < c.tiles_w;
  const int tile = w ? blockIdx.x : blockIdx.x - c.tiles_w;
  if (c.nk_w == 0 || (!w && tile >= c.tiles_x)) return;
  const int64_t units = w ? c.units_w : c.units_x, first = (w ? 0 : c.all_w) + tile * units;
  const int g0 = c.owner(first + c.around), g1 = c.owner(first + units - 1);
  if (g0 == g1) return;
  const int kept = columns_kept<E>(a, w, tile / c.nd, n_valid);
  const FirstRows<T, E> rows(a, w ? tile / c.nd : 1 << 24);  // dx: behind the last word
  f32x4_t acc[1][kJ];
#pragma unroll
  for (int j = 0; j < kJ; ++j)
    if (j < kept) acc[0][j] = slot_of<E>(a, g0, 1)[(i * kJ + j) * kThreads + threadIdx.x];
  constexpr int U = 16 / kJ;  // slots under way: where there are few tokens a tile may have two hundred
  for (int g = g0 + 1; g <= g1; g += U) {
    f32x4_t o[U][kJ];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (g + u <= g1)
#pragma unroll
        for (int j = 0; j < kJ; ++j)
          if (j < kept) o[u][j] = slot_of<E>(a, g + u, 0)[(i * kJ + j) * kThreads + threadIdx.x];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (g + u <= g1)
#pragma unroll
        for (int j = 0; j < kJ; ++j)
          if (j < kept)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[0][j][r] += o[u][j][r];
  }
  if (w)
    store_dw<T, E, 1>(a, c, tile, n_valid, i, acc, rows);
  else
    store_dx<E, 1>(a, c, tile, n_valid, i, acc);
}

// dx (T, d) = factor * (its packed fp32 sums, and in bf16 what the rounding at the label left); rows that were left out: 0.
template <typename T>
__global__ __launch_bounds__(256) void finish_kernel(const float* __restrict__ sums, typename T::raw* out, int64_t ldo, State st,
                                                     Shape s, const float* gloss, int reduction, const uint16_t* w,
                                                     int64_t ldw, const float* up) {
  const float f = common_factor(gloss, reduction, st.hdr->n_valid);
  const bool vec = ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * T::bytes - 1)) == 0;
  const int64_t r = int64_t(blockIdx.x) * 4 + threadIdx.x / kWave;
  if (r >= s.T) return;
  const int64_t at = st.inv[r];
  const int label = Planes<T>::n == 1 && at >= 0 ? st.label[at] : -1;
  const float left = label >= 0 ? left_at_label(st, at, up) : 0.0f;
  for (int64_t c = 4 * (threadIdx.x % kWave); c < s.d; c += 4 * kWave) {
    f32x4_t v{0.0f, 0.0f, 0.0f, 0.0f};
    if (at >= 0) v = *reinterpret_cast<const f32x4_t*>(sums + at * s.dp + c);
    if (label >= 0) add_scaled(v, left, w + label * ldw + c);
    store4<T>(out + r * ldo + c, v, at >= 0 ? f : 0.0f, int(s.d - c), vec);
  }
}

// The backward's workspace, and the words per piece (a multiple of the tile).
struct Plan {
  int64_t piece, g_bytes, dx_bytes, slot_bytes, order_bytes, rows_bytes, rest_bytes;
  int64_t bytes() const { return g_bytes + dx_bytes + slot_bytes + order_bytes + rows_bytes + rest_bytes; }
};

static Plan make_plan(const Shape& s) {
  Plan p{};
  const int64_t tile = s.tile, vpad = up(s.V, tile);
  const int64_t most = std::max<int64_t>(tile, kPieceBytes / (2 * s.planes * s.Mp) / tile * tile);
  const int64_t pieces = (vpad + most - 1) / most;
  p.piece = up((vpad + pieces - 1) / pieces, tile);
  p.g_bytes = up(2 * s.planes * s.Mp * p.piece, 256);
  p.dx_bytes = up(4 * s.Mp * s.dp, 256);
  p.slot_bytes = int64_t(kGroups) * 2 * tile * tile * 4;
  if (s.planes == 1) {
    p.order_bytes = up(4 * s.Mp, 256);
    p.rows_bytes = up(8 * s.V, 256);
    p.rest_bytes = p.dx_bytes;
  }
  return p;
}

static bool bad(const char* op, int dtype, int label_bytes, const void* x, int64_t ldx, const void* W, int64_t ldw,
                const void* labels, int reduction, int64_t T, int64_t V, int64_t d) {
  if (dtype != 0 && dtype != 1) {
    cdssm_host::set_error("%s: dtype must be 0 (fp32) or 1 (bf16), got %d", op, dtype);
    return true;
  }
  if (label_bytes != 4 && label_bytes != 8) {
    cdssm_host::set_error("%s: labels must have 4 or 8 bytes each, got %d", op, label_bytes);
    return true;
  }
  if (reduction < 0 || reduction > 2) {
    cdssm_host::set_error("%s: reduction must be 0 (none), 1 (mean) or 2 (sum), got %d", op, reduction);
    return true;
  }
  if (T < 1 || V < 1 || d < 1 || T > (int64_t(1) << 24) || V > (int64_t(1) << 24) || d > (1 << 16) ||
      up(V, 128) / 128 * (up(T, 128) / 128) > (int64_t(1) << 30)) {
    cdssm_host::set_error("%s: needs 1 <= T, V <= 2^24 with T V <= 2^43, and 1 <= d <= 65536 (T %lld, V %lld, d %lld)", op, (long long)T,
                          (long long)V, (long long)d);
    return true;
  }
  if (ldx < d || ldw < d || ldw > (1 << 22)) {
    cdssm_host::set_error("%s: the row strides must cover the rows (ldx %lld, ldw %lld, d %lld; ldw at most 2^22)", op,
                          (long long)ldx, (long long)ldw, (long long)d);
    return true;
  }
  if (!x || !W || !labels) {
    cdssm_host::set_error("%s: null pointer argument", op);
    return true;
  }
  return false;
}

}  // namespace lce
}  // namespace cdssm

using namespace cdssm;
using namespace cdssm::lce;

// f(type, engine) of a call.
template <typename F>
static void with_engine(int dtype, const Shape& s, F&& f) {
  if (dtype == 0)
    f(F32{}, Engine<3, 128>{});
  else if (s.tile == 128)
    f(BF16{}, Engine<1, 128>{});
  else
    f(BF16{}, Engine<1, 256>{});
}

static Logits make_logits(const Shape& s, const State& st, const void* W, int64_t ldw) {
  Logits a{};
  a.w = s.pack_w ? st.wp : static_cast<const uint16_t*>(W);
  a.ldw = s.pack_w ? s.dp : ldw;
  a.w_plane = s.V * s.dp;
  a.st = st;
  a.s = s;
  a.v0 = 0;
  a.v1 = int(s.V);
  return a;
}

extern "C" int64_t cdssm_linear_cross_entropy_workspace_bytes(int dtype, const void* W, int64_t ldw, int64_t T, int64_t V,
                                                              int64_t d) {
  if (bad("cdssm_linear_cross_entropy_workspace_bytes", dtype, 8, W, d, W, ldw, W, 0, T, V, d)) return -1;
  return carve(make_shape(dtype, W, ldw, T, V, d), nullptr).bytes;
}

extern "C" int64_t cdssm_linear_cross_entropy_bwd_workspace_bytes(int dtype, const void* W, int64_t ldw, int64_t T, int64_t V,
                                                                  int64_t d) {
  if (bad("cdssm_linear_cross_entropy_bwd_workspace_bytes", dtype, 8, W, d, W, ldw, W, 0, T, V, d)) return -1;
  return make_plan(make_shape(dtype, W, ldw, T, V, d)).bytes();
}

extern "C" int cdssm_linear_cross_entropy_fwd(int dtype, int label_bytes, const void* x, int64_t ldx, const void* W, int64_t ldw,
                                              const void* labels, int64_t ignore_index, int reduction, float* loss,
                                              void* workspace, int64_t T, int64_t V, int64_t d, hipStream_t stream) {
  const char* op = "cdssm_linear_cross_entropy_fwd";
  if (bad(op, dtype, label_bytes, x, ldx, W, ldw, labels, reduction, T, V, d)) return CDSSM_EINVAL;
  if (!loss || !workspace) {
    cdssm_host::set_error("%s: null pointer argument", op);
    return CDSSM_EINVAL;
  }
  const Shape s = make_shape(dtype, W, ldw, T, V, d);
  const State st = carve(s, workspace);
  const int groups = int(up(T, kPackRows * kPackGroups) / (kPackRows * kPackGroups));
  const dim3 pgrid(unsigned((T + groups * kPackRows - 1) / (groups * kPackRows) + kTailGroups +
                            (s.pack_w ? (V + kPackRows - 1) / kPackRows : 0)));
  float* none = reduction == 0 ? loss : nullptr;
  auto pack = [&](auto tag, auto itag) {
    using E = decltype(tag);
    using I = decltype(itag);
    using raw = typename E::raw;
    hipLaunchKernelGGL((pack_kernel<E, I>), pgrid, dim3(kPackThreads), 0, stream, static_cast<const raw*>(x), ldx,
                       static_cast<const I*>(labels), ignore_index, none, static_cast<const raw*>(W), ldw, st, s,
                       groups);
  };
  if (dtype == 1)
    label_bytes == 8 ? pack(BF16{}, int64_t{}) : pack(BF16{}, int32_t{});
  else
    label_bytes == 8 ? pack(F32{}, int64_t{}) : pack(F32{}, int32_t{});
  const Logits a = make_logits(s, st, W, ldw);
  const int tile = int(s.tile), nv = int(up(V, tile) / tile);
  const dim3 grid(unsigned(std::min<int64_t>(kGroups, nv * (up(T, tile) / tile))));
  with_engine(dtype, s, [&](auto, auto engine) {
    hipLaunchKernelGGL(stats_kernel<decltype(engine)>, grid, dim3(kThreads), 0, stream, a);
  });
  hipLaunchKernelGGL(join_kernel, dim3(unsigned(std::min<int64_t>(s.Mp / kWave, kJoinGroups))), dim3(256), 0, stream, st, s, nv, reduction, loss);
  return cdssm_host::check_launch(op);
}

extern "C" int cdssm_linear_cross_entropy_bwd(int dtype, const void* W, int64_t ldw, int reduction, const float* gloss,
                                              const void* fwd_workspace, void* dx, int64_t lddx, void* dW, int64_t lddw,
                                              void* workspace, int64_t T, int64_t V, int64_t d, hipStream_t stream) {
  const char* op = "cdssm_linear_cross_entropy_bwd";
  if (bad(op, dtype, 8, gloss, d, W, ldw, fwd_workspace, reduction, T, V, d)) return CDSSM_EINVAL;
  if ((!dx && !dW) || !workspace || (dx && lddx < d) || (dW && lddw < d)) {
    cdssm_host::set_error("%s: needs a workspace and dx or dW, with row strides that cover the rows", op);
    return CDSSM_EINVAL;
  }
  const Shape s = make_shape(dtype, W, ldw, T, V, d);
  const State st = carve(s, const_cast<void*>(fwd_workspace));
  const Plan plan = make_plan(s);
  char* ws = static_cast<char*>(workspace);
  auto* G = reinterpret_cast<uint16_t*>(ws);
  auto* dxs = reinterpret_cast<float*>(ws + plan.g_bytes);
  auto* slots = reinterpret_cast<f32x4_t*>(ws + plan.g_bytes + plan.dx_bytes);
  auto* order = reinterpret_cast<int*>(ws + plan.g_bytes + plan.dx_bytes + plan.slot_bytes);
  auto* rows = reinterpret_cast<int2*>(ws + plan.g_bytes + plan.dx_bytes + plan.slot_bytes + plan.order_bytes);
  auto* rests = reinterpret_cast<float*>(ws + plan.bytes() - plan.rest_bytes);
  const int64_t tile = s.tile, nd = (s.dp + tile - 1) / tile, nt = (T + tile - 1) / tile;
  const float *common = reduction == 0 ? nullptr : gloss, *up = reduction == 0 ? gloss : nullptr;
  if (dtype == 1 && dW) {
    const bool few = T <= std::min<int64_t>(kFewRows, V * kFewToWord);
    const int chunk = few ? 1 : int(std::max<int64_t>(kRestRows, cdssm::lce::up((T + kRestChunks - 1) / kRestChunks, kRestRows)));
    const Rests r{st, s, up, rests, order, rows, chunk};
    const int64_t waves = (T + chunk - 1) / chunk * ((s.dp + kRestColumns - 1) / kRestColumns);
    const dim3 grid(unsigned((waves + 3) / 4));
    if (few) {
      hipLaunchKernelGGL(few_rests_kernel, grid, dim3(256), 0, stream, r);
    } else {
      const int shift = token_sort::id_shift(V);
      hipLaunchKernelGGL(sort_labels_kernel, dim3(1u << shift), dim3(token_sort::kSortThreads), 0, stream, st, order, rows, V, shift);
      hipLaunchKernelGGL(rests_kernel, grid, dim3(256), 0, stream, r);
      hipLaunchKernelGGL(join_rests_kernel, grid, dim3(256), 0, stream, r);
    }
  }
  Logits a = make_logits(s, st, W, ldw);
  with_engine(dtype, s, [&](auto tag, auto engine) {
    using E = decltype(tag);
    using M = decltype(engine);
    using raw = typename E::raw;
    for (int64_t v0 = 0; v0 < V; v0 += plan.piece) {
      const int64_t v1 = std::min(V, v0 + plan.piece), vt = (v1 - v0 + tile - 1) / tile;
      a.v0 = int(v0);
      a.v1 = int(v1);
      hipLaunchKernelGGL((grad_kernel<E, M>), dim3(unsigned(std::min<int64_t>(kGroups, vt * nt))), dim3(kThreads), 0, stream, a,
                         up, G, vt * tile);
      Products p{};
      p.w = a.w + v0 * a.ldw;
      p.ldw = a.ldw;
      p.w_plane = a.w_plane;
      p.G = G;
      p.ldg = vt * tile;
      p.nv = v1 - v0;
      p.st = st;
      p.s = s;
      p.dx = dx ? dxs : nullptr;
      p.dw = dW ? static_cast<raw*>(dW) + v0 * lddw : nullptr;
      p.ldo = lddw;
      p.gloss = common;
      p.reduction = reduction;
      p.add = v0 > 0;
      p.slots = slots;
      p.first = st.first + v0;
      p.rests = rests;
      const int64_t tiles = ((dW ? vt : 0) + (dx ? nt : 0)) * nd;
      hipLaunchKernelGGL((products_kernel<E, M>), dim3(kGroups), dim3(kThreads), 0, stream, p);
      hipLaunchKernelGGL((join_tiles_kernel<E, M>), dim3(unsigned(tiles), unsigned(M::kI)), dim3(kThreads), 0, stream, p, kGroups);
    }
    if (dx)
      hipLaunchKernelGGL((finish_kernel<E>), dim3(unsigned((T + 3) / 4)), dim3(256), 0, stream, dxs, static_cast<raw*>(dx), lddx,
                         st, s, common, reduction, a.w, a.ldw, up);
  });
  return cdssm_host::check_launch(op);
}
