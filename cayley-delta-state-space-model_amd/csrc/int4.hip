// Decode products with weights of 4 bits: Y (M x N) = X' (M x K) W^T (+ bias) (+ R), M <= 64, with
//   W[n][k] = s[n][k / g] c[n][k],   c a whole number of -8 .. 7, s bf16, g 32, 64 or 128
// and X' = X, or with a norm weight X' = rs X w_norm, rs[m] = rsqrt(mean_k X[m][k]^2 + eps).  bf16 X and Y, fp32 sums.
//
// A call reads N K / 2 bytes of codes and little else, so it is bound by memory, or for the small layers by the latency of one
// load and one sum.  No weight is rounded: the codes go into the matrix cores as the whole numbers that they are, and the sum
// over a group is multiplied by its scale in fp32.  A code travels in 4 bits, 2 c where it is not negative and 2 (-c - 1) + 1 where it
// is; those bits, and 2^7 + 1 more where the lowest is set, are the fp8 number (e4m3: sign, and up to 2^-5 a whole number of 2^-9) of 2 c
// 2^-9, which the conversion to bf16 multiplies by 2^8.  8 codes take 11 instructions.  (7 would give the bf16 numbers 136 + c; but a
// sum of those loses 2^-24 of 136 |x| even where the weight is 0, and one large x costs every column its lower digits.)
//
// Layout: per 16 columns n and 128 k one KB, in the order in which a wave's lanes load it: lane l holds column
// l % 16, and of each of the four steps of 32 k eight codes from 8 (l / 16) on, in one word.  Scales: per 16 columns and 128 k,
// a lane's 128 / g next to each other.
//
// A workgroup owns 16 NT columns and 16 MT rows; its waves take blocks of 128 k in turn, and their sums are added in a
// fixed order through LDS.  Where there are no more blocks than waves, each wave keeps its block of x and the workgroup goes
// through several such columns, reading x once.
//
// MI355X, us: 1 x 3104 x 1024 3.6 (1.7 MB: launch, one load, one sum), 64 x 3104 x 1024 4.4, 64 x 32000 x 1024 10 (21 MB, 2.1 TB/s:
// launch and x 6, then units of 32 columns, each products, sum and store), 16 x 8192 x 28672 25 with the codes in the last-level
// cache, 31 without (122 MB, 4.0 TB/s; x comes from L2 256 times, twice the codes' bytes).
//
// Fragment layouts of v_mfma_f32_16x16x32_bf16: as in skinny_gemm.hip.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.hpp"
#include "lm_common.hpp"
#include "cdssm_hip.h"

namespace cdssm {
namespace w4 {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

constexpr int kCols = 16, kBlock = 128, kSteps = kBlock / 32, kMaxRows = 64;
constexpr int kStreamWaves = 8, kMaxSplits = 16;
constexpr int64_t kMaxSize = int64_t(1) << 24;  // of N and K

__device__ __forceinline__ f32x4_t mfma(uint4 a, uint4 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// Eight codes in bf16: elements 0 .. 3 in the low halves of a word's bytes, 4 .. 7 in the high ones.
__device__ __forceinline__ uint4 codes_of(uint32_t w) {
  const auto fp8 = [](uint32_t v) {
    const u16x2_t low = __builtin_bit_cast(u16x2_t, v & 0x01010101u), all = __builtin_bit_cast(u16x2_t, v & 0x0f0f0f0fu);
    return __builtin_bit_cast(uint32_t, u16x2_t(low * uint16_t(0x81) + all));
  };
  const uint32_t a = fp8(w), b = fp8(w >> 4);
  constexpr float kScale = 256.0f;
  return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, kScale, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, kScale, true)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, kScale, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, kScale, true)));
}
// A code's 4 bits and back.
__device__ __forceinline__ uint32_t bits_of(int c) {
  c = int(uint32_t(c + 8) & 15u) - 8;
  return uint32_t(c < 0 ? 2 * (-c - 1) + 1 : 2 * c);
}
__device__ __forceinline__ int code_of(uint32_t bits) { return bits & 1 ? -int(bits / 2) - 1 : int(bits / 2); }

// A causal conv step on C of the result's columns, from col0 on (cdssm_conv1d_silu_step on the rounded result): window (M, taps - 1,
// C) is read and shifted, y (M, C) written.  y null: none.
struct Conv {
  uint16_t *window, *y;
  const uint16_t *w, *bias;  // (C, taps), (C)
  int col0, C, taps;
};
constexpr int kMaxTaps = 8;

struct Args {
  const uint16_t* x;
  int64_t ldx;
  const uint4* codes;
  const uint16_t *scales, *bias, *residual, *wnorm;
  int64_t ldr;
  uint16_t* y;
  int64_t ldy;
  int M, N, K;
  float eps;
  Conv conv;
};

__device__ __forceinline__ float sum_squares(uint4 a, float s) {
  const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s = fmaf(bf16_lo(u[i]), bf16_lo(u[i]), s);
    s = fmaf(bf16_hi(u[i]), bf16_hi(u[i]), s);
  }
  return s;
}

// x w as two bf16 numbers that add up to it to 2^-17: hi, and what is left of it.
__device__ __forceinline__ void scaled(uint4 x, uint4 w, uint4& hi, uint4& lo) {
  const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ws[4] = {w.x, w.y, w.z, w.w};
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = bf16_lo(xs[i]) * bf16_lo(ws[i]), b = bf16_hi(xs[i]) * bf16_hi(ws[i]);
    h[i] = pack_bf16x2(a, b);
    l[i] = pack_bf16x2(a - bf16_lo(h[i]), b - bf16_hi(h[i]));
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}

// The scales of a lane's column in a block of 128 k, as they lie in memory.
template <int Groups>
struct Scales {
  uint32_t u[(Groups + 1) / 2];
  __device__ __forceinline__ void load(const uint16_t* p) {
    if constexpr (Groups == 4) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      u[0] = v.x;
      u[1] = v.y;
    } else if constexpr (Groups == 2) {
      u[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      u[0] = *p;
    }
  }
  __device__ __forceinline__ float get(int g) const { return g & 1 ? bf16_hi(u[g / 2]) : bf16_lo(u[g / 2]); }
};

// Codes and scales of a block of 128 k in NT tiles of columns from t0 on (the last one where there are fewer).
template <int G, int NT>
struct Codes {
  uint4 w[NT];
  Scales<kBlock / G> s[NT];
  __device__ __forceinline__ void load(const Args& a, int t0, int n_tiles, int b, int n_blocks, int lane) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int64_t at = int64_t(min(t0 + j, n_tiles - 1)) * n_blocks + b;
      w[j] = a.codes[at * kWave + lane];
      s[j].load(a.scales + (at * kCols + lane % 16) * (kBlock / G));
    }
  }
};

// A block of 16 MT rows of x from m0 on.  It is read with the 16 lanes of a row next to each other in memory (the products' order
// would touch 16 rows at once, a quarter as fast), and turned into the products' order through 4 KB of LDS per 16 rows,
// which are the wave's own: chunk c of 8 k of row r at 16 r + (c ^ r), so that neither side meets bank conflicts.
// x as the products take it has P planes: itself, or with a norm the two parts of x w_norm that add up to it.
template <bool Norm, int MT>
struct Rows {
  uint4 x[MT][4], wn[Norm ? kSteps : 1];
  __device__ __forceinline__ void load(const Args& a, int m0, int b, int lane) {
    const int col = lane % 16, kq = lane / 16, last = (a.K - 1) & ~7;  // the row's last whole chunk, which the caller filled up
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        x[i][k] = *reinterpret_cast<const uint4*>(a.x + int64_t(min(m0 + 16 * i + 4 * k + kq, a.M - 1)) * a.ldx +
                                                  min(b * kBlock + 8 * col, last));
    if constexpr (Norm)
#pragma unroll
      for (int k = 0; k < kSteps; ++k) wn[k] = *reinterpret_cast<const uint4*>(a.wnorm + min(b * kBlock + 32 * k + 8 * kq, last));
  }
  __device__ __forceinline__ void put(const Args& a, int b, int lane, uint4* lds) const {
    const int col = lane % 16, kq = lane / 16;
    const bool past = b * kBlock + 8 * col >= a.K;
    meet();
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int row = 4 * k + kq;
        lds[i * 4 * kWave + row * 16 + (col ^ row)] = past ? make_uint4(0, 0, 0, 0) : x[i][k];
      }
    meet();
  }
  template <int P>
  __device__ __forceinline__ void take(const uint4* lds, int lane, uint4 (&f)[kSteps][MT][P], float (&sq)[MT]) const {
    const int col = lane % 16, kq = lane / 16;
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint4 v = lds[i * 4 * kWave + col * 16 + ((4 * k + kq) ^ col)];
        if constexpr (Norm) {
          sq[i] = sum_squares(v, sq[i]);
          scaled(v, wn[k], f[k][i][0], f[k][i][1]);
        } else {
          f[k][i][0] = v;
        }
      }
  }
  // Other lanes' parts are read only behind their writes, and the other way round (LDS itself keeps a wave's order).
  __device__ __forceinline__ static void meet() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
};

// acc += a block's products.
template <int G, int MT, int NT, int P>
__device__ __forceinline__ void multiply(const uint4 (&x)[kSteps][MT][P], const Codes<G, NT>& c, f32x4_t (&acc)[MT][NT]) {
  constexpr int kGroups = kBlock / G, kPerGroup = G / 32;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      f32x4_t t[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) t[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < kPerGroup; ++k) {
        const int st = g * kPerGroup + k;
        const uint4 v = codes_of(st == 0 ? c.w[j].x : st == 1 ? c.w[j].y : st == 2 ? c.w[j].z : c.w[j].w);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int p = 0; p < P; ++p) t[i] = mfma(x[st][i][p], v, t[i]);
      }
      const float s = c.s[j].get(g);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(s, t[i][e], acc[i][j][e]);
    }
  }
}

template <int MT, int NT>
__device__ __forceinline__ void clear(f32x4_t (&acc)[MT][NT]) {
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
}

// A lane's part of a row's sum of squares, summed over the lanes of the row, for row 16 i + lane % 16.
template <int MT>
__device__ __forceinline__ void put_squares(const float (&sq)[MT], float* ssq, int lane) {
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    float s = sq[i];
    s += __shfl_xor(s, 16, kWave);
    s += __shfl_xor(s, 32, kWave);
    if (lane < 16) ssq[16 * i + lane] = s;
  }
}

// The sum of the waves' parts of a tile.
template <int W, int Tiles>
__device__ __forceinline__ f32x4_t join(const f32x4_t (*part)[Tiles][kWave], int tile, int lane) {
  f32x4_t c = part[0][tile][lane];
#pragma unroll
  for (int v = 1; v < W; ++v) {
    const f32x4_t p = part[v][tile][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] += p[e];
  }
  return c;
}

// Rows m .. m + 3 of column n of the result from their sums; squares(e): the sum of squares of row m + e of x.
// (Offsets stay within 2^32: row strides are at most 2^24.)
template <bool Norm, bool WithConv = false, typename Squares>
__device__ __forceinline__ void finish(const Args& a, f32x4_t c, int m, int n, Squares&& squares) {
  if (n >= a.N) return;
  const float bias = a.bias ? bf16_to_f32(a.bias[n]) : 0.0f;
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] = c[e];
    if constexpr (Norm) {
      const float q = squares(e);
      y[e] *= rsqrtf(q / float(a.K) + (a.eps + (q - q)));  // q - q: NaN for squares that fp32 does not hold, which would make the row 0
    }
    y[e] += bias;
  }
  if (a.residual) {
    uint32_t at = uint32_t(m) * uint32_t(a.ldr) + uint32_t(n);
#pragma unroll
    for (int e = 0; e < 4; ++e, at += uint32_t(a.ldr))
      if (m + e < a.M) y[e] += bf16_to_f32(a.residual[at]);
  }
  const uint32_t lo = pack_bf16x2(y[0], y[1]), hi = pack_bf16x2(y[2], y[3]);
  uint32_t at = uint32_t(m) * uint32_t(a.ldy) + uint32_t(n);
#pragma unroll
  for (int e = 0; e < 4; ++e, at += uint32_t(a.ldy))
    if (m + e < a.M) a.y[at] = uint16_t((e & 2 ? hi : lo) >> 16 * (e & 1));
  if constexpr (WithConv) {
    const Conv& cv = a.conv;
    const int ch = n - cv.col0;
    if (ch < 0 || ch >= cv.C) return;
    uint16_t win[4][kMaxTaps], w[kMaxTaps];
#pragma unroll
    for (int j = 0; j < kMaxTaps; ++j)
      if (j < cv.taps) w[j] = cv.w[int64_t(ch) * cv.taps + j];
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int j = 0; j + 1 < kMaxTaps; ++j)
        if (j + 1 < cv.taps) win[e][j] = cv.window[(int64_t(min(m + e, a.M - 1)) * (cv.taps - 1) + j) * cv.C + ch];
    const float b = bf16_to_f32(cv.bias[ch]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (m + e >= a.M) continue;
      uint16_t* to = cv.window + int64_t(m + e) * (cv.taps - 1) * cv.C + ch;
      float u = b;
#pragma unroll
      for (int j = 0; j < kMaxTaps; ++j)
        if (j < cv.taps) {
          const uint16_t in = j + 1 == cv.taps ? uint16_t((e & 2 ? hi : lo) >> 16 * (e & 1)) : win[e][j];
          u = fmaf(bf16_to_f32(w[j]), bf16_to_f32(in), u);
          if (j > 0) to[int64_t(j - 1) * cv.C] = in;
        }
      cv.y[int64_t(m + e) * cv.C + ch] = f32_to_bf16(lm::silu_fast(u));
    }
  }
}

// Where a workgroup works: groups of rows that share columns lie 8 workgroups apart, on one XCD, so that the codes come from
// HBM once and from that XCD's L2 for the others.
struct Seat {
  int m0, first, apart;  // first row; first unit of columns, and how far the next one lies
  __device__ __forceinline__ Seat(int M, int rows) {
    const int mgs = (M + rows - 1) / rows, id = int(blockIdx.x);
    m0 = id / 8 % mgs * rows;
    first = id / (8 * mgs) * 8 + id % 8;
    apart = int(gridDim.x) / mgs;
  }
};

// K of up to W blocks: a wave brings its block of x once, in registers, and its workgroup goes through units of 16 NT columns.
template <int G, bool Norm, int MT, int NT, int W, bool WithConv>
__global__ __launch_bounds__(kWave* W) void resident_kernel(Args a) {
  constexpr int P = Norm ? 2 : 1, kStage = MT * 4 * kWave, kParts = MT * NT * kWave;
  __shared__ uint4 lds[W * (kStage > kParts ? kStage : kParts)];
  __shared__ float ssq[W][16 * MT];
  auto part = reinterpret_cast<f32x4_t(*)[MT * NT][kWave]>(lds);
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave), lane = int(threadIdx.x) % kWave;
  const int n_tiles = (a.N + kCols - 1) / kCols, n_blocks = (a.K + kBlock - 1) / kBlock, units = (n_tiles + NT - 1) / NT;
  const Seat seat(a.M, 16 * MT);
  const int b = min(wave, n_blocks - 1);
  Codes<G, NT> c;
  c.load(a, seat.first * NT, n_tiles, b, n_blocks, lane);
  uint4 x[kSteps][MT][P];
  float sq[MT] = {};
  {
    Rows<Norm, MT> r;
    r.load(a, seat.m0, b, lane);
    r.put(a, wave, lane, lds + wave * kStage);  // (zeros where the wave has no block)
    r.template take<P>(lds + wave * kStage, lane, x, sq);
  }
  if constexpr (Norm) put_squares(sq, ssq[wave], lane);
  for (int unit = seat.first; unit < units; unit += seat.apart) {
    f32x4_t acc[MT][NT];
    clear(acc);
    multiply<G>(x, c, acc);
    if (unit + seat.apart < units) c.load(a, (unit + seat.apart) * NT, n_tiles, b, n_blocks, lane);
    __syncthreads();  // the rows' pieces, or the last unit's parts, have been read
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();
    for (int tile = wave; tile < MT * NT; tile += W) {
      const int m = 16 * (tile / NT) + 4 * (lane / 16);
      finish<Norm, WithConv>(a, join<W>(part, tile, lane), seat.m0 + m, (unit * NT + tile % NT) * kCols + lane % 16, [&](int e) {
        float q = 0.0f;
#pragma unroll
        for (int v = 0; v < W; ++v) q += ssq[v][m + e];
        return q;
      });
    }
  }
}

// x w_norm of rows that many workgroups will read, once: its two planes in the order in which the products take them ([16 rows][block]
// [step][plane][lane]), and the rows' squares, summed over kShare blocks ([share][64]).  A wave per block of 16 rows.
constexpr int kShare = 16;
__global__ __launch_bounds__(kWave* kShare) void norm_kernel(Args a, uint4* __restrict__ planes, float* __restrict__ squares) {
  __shared__ uint4 lds[kShare][4 * kWave];
  __shared__ float ssq[kShare][16];
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave), lane = int(threadIdx.x) % kWave;
  const int n_blocks = (a.K + kBlock - 1) / kBlock, b = int(blockIdx.x) * kShare + wave, m0 = 16 * int(blockIdx.y);
  float sq[1] = {};
  if (b < n_blocks) {
    Rows<true, 1> r;
    r.load(a, m0, b, lane);
    r.put(a, b, lane, lds[wave]);
    uint4 x[kSteps][1][2];
    r.take<2>(lds[wave], lane, x, sq);
    uint4* to = planes + (int64_t(blockIdx.y) * n_blocks + b) * kSteps * 2 * kWave + lane;
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
      for (int p = 0; p < 2; ++p) to[(2 * k + p) * kWave] = x[k][0][p];
  }
  put_squares(sq, ssq[wave], lane);
  __syncthreads();
  if (threadIdx.x < 16) {
    float q = 0.0f;
#pragma unroll
    for (int v = 0; v < kShare; ++v) q += ssq[v][threadIdx.x];
    squares[blockIdx.x * kMaxRows + m0 + threadIdx.x] = q;
  }
}

// How a wave of the next kernel comes by the rows of x of a block: as they lie; with a norm, which every workgroup applies for itself;
// or a norm's planes in order.
enum Source { kPlain, kNormed, kPlanes };
template <Source S, int MT>
struct Feed : Rows<S == kNormed, MT> {
  static constexpr int P = S == kNormed ? 2 : 1, kStage = MT * 4 * kWave;
  __device__ __forceinline__ void load(const Args& a, const uint4*, int m0, int b, int, int lane) {
    Rows<S == kNormed, MT>::load(a, m0, b, lane);
  }
};
template <int MT>
struct Feed<kPlanes, MT> {
  static constexpr int P = 2, kStage = 0;
  uint4 x[kSteps][MT][2];
  __device__ __forceinline__ void load(const Args& a, const uint4* planes, int m0, int b, int n_blocks, int lane) {
    const int last = (a.M - 1) / 16;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const uint4* from = planes + (int64_t(min(m0 / 16 + i, last)) * n_blocks + b) * kSteps * 2 * kWave + lane;
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
#pragma unroll
        for (int p = 0; p < 2; ++p) x[k][i][p] = from[(2 * k + p) * kWave];
    }
  }
  __device__ __forceinline__ void put(const Args&, int, int, uint4*) const {}
  template <int>
  __device__ __forceinline__ void take(const uint4*, int, uint4 (&f)[kSteps][MT][2], float (&)[MT]) const {
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int p = 0; p < 2; ++p) f[k][i][p] = x[k][i][p];
  }
};

// The sum of squares of a row from those of its shares.
__device__ __forceinline__ float row_squares(const float* squares, int K, int m) {
  const int shares = ((K + kBlock - 1) / kBlock + kShare - 1) / kShare;
  float q = 0.0f;
  for (int s = 0; s < shares; ++s) q += squares[s * kMaxRows + m];
  return q;
}

// Any K: a wave takes every W-th block, the next one's loads under way while one is computed.
// blockIdx.y: its share of the blocks where K is split over workgroups, whose sums go to `sums` ([split][column tile][row
// tile][64] of 4 rows each).
template <int G, Source S, int MT, int NT, bool Split>
__global__ __launch_bounds__(kWave* kStreamWaves) void stream_kernel(Args a, const uint4* __restrict__ planes,
                                                                     const float* __restrict__ squares, f32x4_t* __restrict__ sums) {
  using X = Feed<S, MT>;
  static_assert(!Split || S != kNormed, "the squares of a share are not the row's");
  constexpr int W = kStreamWaves, kParts = MT * NT * kWave;
  __shared__ uint4 lds[W * (X::kStage > kParts ? X::kStage : kParts)];
  __shared__ float ssq[S == kNormed ? W : 1][16 * MT];
  auto part = reinterpret_cast<f32x4_t(*)[MT * NT][kWave]>(lds);
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave), lane = int(threadIdx.x) % kWave;
  const int n_tiles = (a.N + kCols - 1) / kCols, n_blocks = (a.K + kBlock - 1) / kBlock;
  const Seat seat(a.M, 16 * MT);
  const int t0 = seat.first * NT;
  if (t0 >= n_tiles) return;
  const int share = Split ? (n_blocks + int(gridDim.y) - 1) / int(gridDim.y) : n_blocks;
  const int from = Split ? int(blockIdx.y) * share : 0, to = min(n_blocks, from + share);
  uint4* mine = lds + wave * X::kStage;
  f32x4_t acc[MT][NT];
  clear(acc);
  float sq[MT] = {};
  Codes<G, NT> next;
  X rows;
  int b = from + wave;
  if (b < to) {
    next.load(a, t0, n_tiles, b, n_blocks, lane);
    rows.load(a, planes, seat.m0, b, n_blocks, lane);
  }
  for (; b < to; b += W) {
    const Codes<G, NT> c = next;
    const X r = rows;
    r.put(a, b, lane, mine);
    if (b + W < to) {
      next.load(a, t0, n_tiles, b + W, n_blocks, lane);
      rows.load(a, planes, seat.m0, b + W, n_blocks, lane);
    }
    uint4 x[kSteps][MT][X::P];
    r.template take<X::P>(mine, lane, x, sq);
    multiply<G>(x, c, acc);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = acc[i][j];
  if constexpr (S == kNormed) put_squares(sq, ssq[wave], lane);
  __syncthreads();
  for (int tile = wave; tile < MT * NT; tile += W) {
    const int t = t0 + tile % NT, m = seat.m0 + 16 * (tile / NT) + 4 * (lane / 16);
    const f32x4_t c = join<W>(part, tile, lane);
    if constexpr (Split) {
      const int row_tiles = (a.M + 15) / 16, row_tile = seat.m0 / 16 + tile / NT;
      if (t < n_tiles && row_tile < row_tiles)
        sums[((int64_t(blockIdx.y) * n_tiles + t) * row_tiles + row_tile) * kWave + lane] = c;
    } else {
      finish<S != kPlain>(a, c, m, t * kCols + lane % 16, [&](int e) {
        if constexpr (S == kPlanes) return row_squares(squares, a.K, min(m + e, a.M - 1));
        float q = 0.0f;
#pragma unroll
        for (int v = 0; v < W; ++v) q += ssq[S == kNormed ? v : 0][m + e - seat.m0];
        return q;
      });
    }
  }
}

// The sums of all shares: a wave for 16 rows of 16 columns.
template <bool Norm>
__global__ __launch_bounds__(kWave) void join_kernel(Args a, const float* __restrict__ squares, const f32x4_t* __restrict__ sums,
                                                     int splits) {
  const int lane = int(threadIdx.x), n_tiles = (a.N + kCols - 1) / kCols, row_tiles = (a.M + 15) / 16;
  const int t = int(blockIdx.x) / row_tiles, row_tile = int(blockIdx.x) % row_tiles;
  f32x4_t c = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (int s = 0; s < splits; ++s) {
    const f32x4_t p = sums[((int64_t(s) * n_tiles + t) * row_tiles + row_tile) * kWave + lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] += p[e];
  }
  const int m = 16 * row_tile + 4 * (lane / 16);
  finish<Norm>(a, c, m, t * kCols + lane % 16, [&](int e) { return row_squares(squares, a.K, min(m + e, a.M - 1)); });
}

// A word of the layout above: 8 codes of column n from k on, those behind the weight's ends 0.
struct Place {
  int64_t n, k;
};
__device__ __forceinline__ Place place_of(int64_t word, int64_t blocks) {
  const int64_t block = word / (kWave * kSteps), in = word % (kWave * kSteps);
  const int64_t lane = in / kSteps, step = in % kSteps;
  return {block / blocks * kCols + lane % 16, block % blocks * kBlock + 32 * step + 8 * (lane / 16)};
}

__device__ __forceinline__ int place_in_word(int i) { return 8 * (i % 4) + 4 * (i / 4); }
__device__ __forceinline__ uint32_t word_of(const int (&c)[8]) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) w |= bits_of(c[i]) << place_in_word(i);
  return w;
}

// codes (N, K) of one byte each, scales (N, groups) to the layout: a thread per word, and per scale.
__global__ void pack_kernel(const int8_t* __restrict__ codes, const uint16_t* __restrict__ scales, uint32_t* __restrict__ words,
                            uint16_t* __restrict__ out, int64_t n_words, int64_t n_scales, int64_t N, int64_t K, int64_t blocks,
                            int64_t g) {
  const int64_t t = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (t < n_words) {
    const Place p = place_of(t, blocks);
    const int8_t* from = codes + p.n * K + p.k;
    int c[8] = {};
    if (p.n < N && p.k + 8 <= K && (reinterpret_cast<uintptr_t>(from) & 7u) == 0) {
      const uint2 u = *reinterpret_cast<const uint2*>(from);
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = int8_t((i < 4 ? u.x : u.y) >> 8 * (i % 4));
    } else if (p.n < N) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (p.k + i < K) c[i] = from[i];
    }
    words[t] = word_of(c);
  }
  if (t < n_scales) {
    const int64_t per = kBlock / g, groups = (K + g - 1) / g;
    const int64_t block = t / (kCols * per), in = t % (kCols * per);
    const int64_t n = block / blocks * kCols + in / per, j = block % blocks * per + in % per;
    out[t] = n < N && j < groups ? scales[n * groups + j] : 0;
  }
}

// The layout back to codes and scales.
__global__ void unpack_kernel(const uint32_t* __restrict__ words, const uint16_t* __restrict__ in_scales, int8_t* __restrict__ codes,
                              uint16_t* __restrict__ scales, int64_t n_words, int64_t n_scales, int64_t N, int64_t K, int64_t blocks,
                              int64_t g) {
  const int64_t t = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (t < n_words) {
    const Place p = place_of(t, blocks);
    if (p.n < N)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (p.k + i < K) codes[p.n * K + p.k + i] = int8_t(code_of(words[t] >> place_in_word(i) & 15u));
  }
  if (t < n_scales) {
    const int64_t per = kBlock / g, groups = (K + g - 1) / g;
    const int64_t block = t / (kCols * per), in = t % (kCols * per);
    const int64_t n = block / blocks * kCols + in / per, j = block % blocks * per + in % per;
    if (n < N && j < groups) scales[n * groups + j] = in_scales[t];
  }
}

// A group's scale is its largest magnitude over 7, rounded to bf16, and a code the nearest whole number to w / scale: a thread per
// group.  A group below 2^-120 throughout becomes 0; one that holds an infinity or NaN gets the scale NaN.  Once per weight, and slow: a
// lane's neighbours read 2 g bytes away.  MI355X, 8192 x 28672 bf16 11 ms (0.06 TB/s), packing 0.11, 32000 x 1024 1.3 ms and 17 us.
template <typename T>
__global__ void quantize_kernel(const typename T::raw* __restrict__ W, int64_t ldw, int8_t* __restrict__ codes,
                                uint16_t* __restrict__ scales, int64_t N, int64_t K, int64_t g) {
  const int64_t groups = (K + g - 1) / g, t = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (t >= N * groups) return;
  const int64_t n = t / groups, k0 = t % groups * g, k1 = min(K, k0 + g);
  const auto* row = W + n * ldw;
  float top = 0.0f;
  bool finite = true;
  for (int64_t k = k0; k < k1; ++k) {
    const float w = fabsf(T::load(row + k));
    finite &= w < INFINITY;
    top = fmaxf(top, w);
  }
  const bool none = !(top >= 0x1p-120f) || !finite;
  const uint16_t s = finite ? (none ? 0 : f32_to_bf16(top / 7.0f)) : 0x7fc0;
  scales[t] = s;
  const float by = none ? 1.0f : bf16_to_f32(s);
  for (int64_t k = k0; k < k1; ++k) {
    const float c = none ? 0.0f : rintf(T::load(row + k) / by);
    codes[n * K + k] = int8_t(fminf(fmaxf(c, -8.0f), 7.0f));
  }
}

// A number of what a weight holds: every 16 bytes of a row (elements behind its end 0) and their place mixed into 64 bits, which are
// added up, in any order.  Each step of the mixing is one to one, so that a change within 16 bytes always shows; others would have to add
// up to 0.  A wave takes a row at a time, a workgroup some 64 KB of one weight; weights share launches, for a model's are many and
// small.  MI355X, 97 weights of 324 MB together 80 us (4.1 TB/s), one of 470 MB 99 (4.8 TB/s).  1024 workgroups to every weight took 510 for
// the 324 MB: their additions to a weight's sum come one behind the other.
struct Weight {
  const char* at;
  int64_t ld, rows;        // ld in bytes
  int width, bytes;        // of a row and of an element
  int first, share;        // first workgroup, rows of each
  bool vectors;
};
constexpr int64_t kFingerprintShare = 65536;
constexpr int kWeights = 64;  // a launch
struct Weights {
  Weight of[kWeights];
  int count;
};
__global__ __launch_bounds__(256) void fingerprint_kernel(Weights list, unsigned long long* __restrict__ sums) {
  __shared__ uint64_t parts[4];
  int i = 0;
  while (i + 1 < list.count && list.of[i + 1].first <= int(blockIdx.x)) ++i;
  const Weight& w = list.of[i];
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave), lane = int(threadIdx.x) % kWave;
  const int per = (w.width + 15) / 16;
  uint64_t sum = 0;
  const int64_t from = int64_t(int(blockIdx.x) - w.first) * w.share, to = min(w.rows, from + w.share);
  for (int64_t n = from + wave; n < to; n += 4) {
    const char* row = w.at + n * w.ld;
    for (int c = lane; c < per; c += kWave) {
      const int left = w.width - 16 * c;  // bytes from here on
      uint32_t v[4] = {0, 0, 0, 0};
      if (w.vectors && left >= 16) {
        const uint4 u = *reinterpret_cast<const uint4*>(row + 16 * c);
        v[0] = u.x;
        v[1] = u.y;
        v[2] = u.z;
        v[3] = u.w;
      } else if (w.bytes == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (4 * e < left) v[e] = reinterpret_cast<const uint32_t*>(row)[4 * c + e];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (2 * e < left) v[e / 2] |= uint32_t(reinterpret_cast<const uint16_t*>(row)[8 * c + e]) << 16 * (e % 2);
      }
      uint64_t h = uint64_t(n * per + c + 1) * 0x9e3779b97f4a7c15ull;  // 2^64 over the golden ratio
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        h = (h ^ v[e]) * 0x6a09e667f3bcc909ull;  // 2^64 (sqrt 2 - 1), odd as it has to be
        h ^= h >> 32;
      }
      sum += h;
    }
  }
#pragma unroll
  for (int j = kWave / 2; j > 0; j /= 2) sum += __shfl_xor((unsigned long long)sum, j, kWave);
  if (lane == 0) parts[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) atomicAdd(sums + i, parts[0] + parts[1] + parts[2] + parts[3]);
}

}  // namespace w4
}  // namespace cdssm

using namespace cdssm;

namespace {
struct Size {
  int64_t tiles, blocks, words, scales;
};
}  // namespace

static int int4_size(const char* op, int64_t N, int64_t K, int64_t g, Size* s) {
  if (N < 1 || K < 1 || N > w4::kMaxSize || K > w4::kMaxSize || N * K > (int64_t(1) << 34) || (g != 32 && g != 64 && g != 128)) {
    cdssm_host::set_error("%s: needs 1 <= N, K <= 2^24 with N K <= 2^34 and groups of 32, 64 or 128, got N %lld, K %lld, %lld", op,
                          (long long)N, (long long)K, (long long)g);
    return CDSSM_EINVAL;
  }
  s->tiles = (N + w4::kCols - 1) / w4::kCols;
  s->blocks = (K + w4::kBlock - 1) / w4::kBlock;
  s->words = s->tiles * s->blocks * kWave * w4::kSteps;
  s->scales = s->tiles * s->blocks * w4::kCols * (w4::kBlock / g);
  return CDSSM_OK;
}

extern "C" int64_t cdssm_int4_code_bytes(int64_t N, int64_t K) {
  Size s;
  return int4_size("cdssm_int4_code_bytes", N, K, 128, &s) ? CDSSM_EINVAL : 4 * s.words;
}
extern "C" int64_t cdssm_int4_scale_bytes(int64_t N, int64_t K, int64_t group) {
  Size s;
  return int4_size("cdssm_int4_scale_bytes", N, K, group, &s) ? CDSSM_EINVAL : 2 * s.scales;
}

static int int4_lay_out(const char* op, bool pack, const void* codes, const void* scales, void* words, void* word_scales, int64_t N,
                        int64_t K, int64_t g, hipStream_t stream) {
  Size s;
  if (const int st = int4_size(op, N, K, g, &s)) return st;
  if (!codes || !scales || !words || !word_scales) {
    cdssm_host::set_error("%s: null pointer argument", op);
    return CDSSM_EINVAL;
  }
  if (reinterpret_cast<uintptr_t>(words) % 16 || reinterpret_cast<uintptr_t>(word_scales) % 16 || reinterpret_cast<uintptr_t>(scales) % 2) {
    cdssm_host::set_error("%s: the layout's tensors must be 16-byte aligned, the scales to their elements", op);
    return CDSSM_EINVAL;
  }
  // words are never fewer than scales: 256 of the one, 64 of the other at most for 16 columns and 128 k
  const dim3 grid(unsigned((s.words + 255) / 256));
  if (pack)
    hipLaunchKernelGGL(w4::pack_kernel, grid, dim3(256), 0, stream, static_cast<const int8_t*>(codes),
                       static_cast<const uint16_t*>(scales), static_cast<uint32_t*>(words), static_cast<uint16_t*>(word_scales),
                       s.words, s.scales, N, K, s.blocks, g);
  else
    hipLaunchKernelGGL(w4::unpack_kernel, grid, dim3(256), 0, stream, static_cast<const uint32_t*>(words),
                       static_cast<const uint16_t*>(word_scales), static_cast<int8_t*>(const_cast<void*>(codes)),
                       static_cast<uint16_t*>(const_cast<void*>(scales)), s.words, s.scales, N, K, s.blocks, g);
  return cdssm_host::check_launch(op);
}

extern "C" int cdssm_int4_pack(const void* codes, const void* scales, void* words, void* word_scales, int64_t N, int64_t K,
                               int64_t group, hipStream_t stream) {
  return int4_lay_out("cdssm_int4_pack", true, codes, scales, words, word_scales, N, K, group, stream);
}
extern "C" int cdssm_int4_unpack(const void* words, const void* word_scales, void* codes, void* scales, int64_t N, int64_t K,
                                 int64_t group, hipStream_t stream) {
  return int4_lay_out("cdssm_int4_unpack", false, codes, scales, const_cast<void*>(words), const_cast<void*>(word_scales), N, K, group,
                      stream);
}

extern "C" int cdssm_int4_quantize(int dtype, const void* W, int64_t ldw, void* codes, void* scales, int64_t N, int64_t K,
                                   int64_t group, hipStream_t stream) {
  const char* op = "cdssm_int4_quantize";
  Size s;
  if (const int st = int4_size(op, N, K, group, &s)) return st;
  if (dtype != 0 && dtype != 1) {
    cdssm_host::set_error("%s: dtype must be 0 (fp32) or 1 (bf16), got %d", op, dtype);
    return CDSSM_EINVAL;
  }
  if (!W || !codes || !scales) {
    cdssm_host::set_error("%s: null pointer argument", op);
    return CDSSM_EINVAL;
  }
  if (ldw < K || ldw > (int64_t(1) << 32) || reinterpret_cast<uintptr_t>(W) % (dtype ? 2 : 4) || reinterpret_cast<uintptr_t>(scales) % 2) {
    cdssm_host::set_error("%s: the row stride must be within K .. 2^32 and the tensors aligned to their elements", op);
    return CDSSM_EINVAL;
  }
  const dim3 grid(unsigned((N * ((K + group - 1) / group) + 255) / 256)), block(256);
  auto* c = static_cast<int8_t*>(codes);
  auto* sc = static_cast<uint16_t*>(scales);
  if (dtype)
    hipLaunchKernelGGL(w4::quantize_kernel<BF16>, grid, block, 0, stream, static_cast<const uint16_t*>(W), ldw, c, sc, N, K, group);
  else
    hipLaunchKernelGGL(w4::quantize_kernel<F32>, grid, block, 0, stream, static_cast<const float*>(W), ldw, c, sc, N, K, group);
  return cdssm_host::check_launch(op);
}

extern "C" int cdssm_int4_fingerprints(int64_t count, const int* dtype, const void* const* W, const int64_t* ldw, const int64_t* N,
                                       const int64_t* K, uint64_t* sums, hipStream_t stream) {
  const char* op = "cdssm_int4_fingerprints";
  if (count < 1 || !dtype || !W || !ldw || !N || !K || !sums || reinterpret_cast<uintptr_t>(sums) % 8) {
    cdssm_host::set_error("%s: needs at least one weight, arrays that are not null, and sums aligned to 8 bytes", op);
    return CDSSM_EINVAL;
  }
  for (int64_t i = 0; i < count; ++i) {  // all are checked before anything is launched
    Size s;
    if (const int st = int4_size(op, N[i], K[i], 128, &s)) return st;
    if (dtype[i] != 0 && dtype[i] != 1) {
      cdssm_host::set_error("%s: dtypes must be 0 (fp32) or 1 (bf16), got %d", op, dtype[i]);
      return CDSSM_EINVAL;
    }
    if (!W[i] || ldw[i] < K[i] || ldw[i] > (int64_t(1) << 32) || reinterpret_cast<uintptr_t>(W[i]) % (dtype[i] ? 2 : 4)) {
      cdssm_host::set_error("%s: weights must not be null, aligned to their elements, with row strides within K .. 2^32", op);
      return CDSSM_EINVAL;
    }
  }
  for (int64_t from = 0; from < count; from += w4::kWeights) {
    w4::Weights list{};
    list.count = int(std::min<int64_t>(w4::kWeights, count - from));
    int groups = 0;  // at most 2^22 of a weight
    for (int i = 0; i < list.count; ++i) {
      const int64_t k = from + i, bytes = dtype[k] ? 2 : 4, width = K[k] * bytes;
      const int64_t share = std::max<int64_t>(4, w4::kFingerprintShare / width);
      list.of[i] = {static_cast<const char*>(W[k]), ldw[k] * bytes, N[k], int(width), int(bytes), groups, int(share),
                    reinterpret_cast<uintptr_t>(W[k]) % 16 == 0 && ldw[k] * bytes % 16 == 0};
      groups += int((N[k] + share - 1) / share);
    }
    hipLaunchKernelGGL(w4::fingerprint_kernel, dim3(unsigned(groups)), dim3(256), 0, stream, list,
                       reinterpret_cast<unsigned long long*>(sums) + from);
    if (const int st = cdssm_host::check_launch(op)) return st;
  }
  return CDSSM_OK;
}

namespace {
// How a product is spread over the device.
struct Plan {
  int mt, nt, waves;  // rows and columns of a workgroup in sixteens; waves of the kernel that keeps x, 0: the other one
  int64_t groups;
  int splits;
  bool planes;  // a norm is applied once, by a launch of its own
};
}  // namespace

// Columns and rows of a workgroup, by what was measured.
// Short rows (the kernel that keeps x): as few as leave one workgroup per CU at most, so that every CU has work; beyond that as many as
// possible.  us, M x N x K, for 16 rows x 16 columns / 16 x 32 / 32 x 16 / 32 x 32: 64 x 1136 x 1024 4.0 / 3.5 / 3.6 / 3.9,
// 64 x 3104 x 1024 4.7 / 4.5 / 4.6 / 4.0, 5 x 4992 x 768 (norm) 5.5 / 4.6.  4096 waves keep every CU busy where a workgroup goes
// through several units: 64 x 32000 x 1024 11.6 / 10.6 / 12.4 with 2048 / 4096 / 8192.
// Others: a workgroup's turn of 8 blocks takes some 0.85 / 1.0 / 1.45 us with 16 / 32 / 64 columns (32 rows: 1.5 / 1.65 / 2.0; about a tenth
// less, all of them, with the present codes), and a second one on the same CU adds half of that; the least of what follows is taken.
// 16 x 8192 x 28672 31 / 25 / 37 us with 16 / 32 / 64 columns, 1 x 20238 x 5080 13.3 / 13.5 / 16, 11 x 8359 x 1648 (norm) 9.5 / 10.4 / 7.9,
// 64 x 8192 x 28672 105 / 81 / 72, of 32 rows 90 / 67 / 51, 40 x 2241 x 20992 20 / 17 / 27 and 30 / 23 / 34.
// Long rows of few columns are split over workgroups, at the price of a second launch: 1 x 1024 x 28672 14.9 whole, 7.4 in 8
// shares, 4 x 1166 x 26528 14.2 and 9.2; 64 x 1024 x 4096 4.6 and 7.6 in 4.  A norm is applied by every workgroup,
// or once by a launch of its own: 11 x 8359 x 1648 8.0 and 10.2, 64 x 12416 x 2048 22 and 21, 54 x 45068 x 4776 121 and 89.
// Shares and the norm's way depend on N and K alone: so does the order of a row's sum.
static Plan plan_of(const Size& s, int64_t M) {
  constexpr int64_t kWavesUnderWay = 4096, kManyBlocks = 64, kManyTurns = 12288;
  const int64_t cus = std::max(1, cdssm_host::device_cus());  // (0 where there is no device to ask)
  const auto units = [&](int nt) { return (s.tiles + nt - 1) / nt; };
  const auto row_groups = [&](int mt) { return (M + 16 * mt - 1) / (16 * mt); };
  const auto count = [&](int mt, int nt) { return units(nt) * row_groups(mt); };
  const auto eight = [](int64_t n) { return (n + 7) / 8 * 8; };
  Plan p{M > 16 ? 2 : 1, 2, 0, 0, 1, false};
  if (s.blocks <= 8) {
    p.waves = s.blocks <= 2 ? 2 : s.blocks <= 4 ? 4 : 8;
    if (count(1, 2) <= cus) p.mt = 1;
    if (count(1, 1) <= cus) p.nt = 1;
    const int64_t most = std::max<int64_t>(8, kWavesUnderWay / p.waves / row_groups(p.mt) / 8 * 8);
    p.groups = std::min(eight(units(p.nt)), most) * row_groups(p.mt);
    return p;
  }
  if (s.tiles <= cus / 2 && s.blocks >= kManyBlocks)
    p.splits = int(std::min({int64_t(w4::kMaxSplits), (cus + units(2) - 1) / units(2), s.blocks / w4::kStreamWaves}));
  p.planes = p.splits > 1 || s.tiles * s.blocks >= kManyTurns;
  double least = 0.0;
  for (int mt = 1; mt <= (M > 16 ? 2 : 1); ++mt)
    for (int i = 0; i < 3; ++i) {
      constexpr double kTurn[2][3] = {{0.85, 1.0, 1.45}, {1.5, 1.65, 2.0}};
      const int64_t on_a_cu = (count(mt, 1 << i) * p.splits + cus - 1) / cus;
      const double cost = kTurn[mt - 1][i] * (1.0 + 0.5 * double(on_a_cu - 1));
      if (least == 0.0 || cost < least) {
        least = cost;
        p.mt = mt;
        p.nt = 1 << i;
      }
    }
  p.groups = eight(units(p.nt)) * row_groups(p.mt);
  return p;
}

namespace {
// The workspace of a product with long rows: a norm's planes and squares, the shares' sums.
struct Areas {
  uint4* planes;
  float* squares;
  w4::f32x4_t* sums;
  int64_t bytes;
};
}  // namespace

static Areas areas_of(const Size& s, const Plan& p, int64_t M, bool norm, void* workspace) {
  const int64_t row_tiles = (M + 15) / 16;
  char* at = static_cast<char*>(workspace);
  Areas w{};
  const auto take = [&](int64_t n) {
    char* r = at + w.bytes;
    w.bytes += n;
    return r;
  };
  if (norm && p.planes) {
    w.planes = reinterpret_cast<uint4*>(take(16 * kWave * row_tiles * s.blocks * w4::kSteps * 2));
    w.squares = reinterpret_cast<float*>(take(4 * w4::kMaxRows * ((s.blocks + w4::kShare - 1) / w4::kShare)));
  }
  if (p.splits > 1) w.sums = reinterpret_cast<w4::f32x4_t*>(take(16 * kWave * s.tiles * row_tiles * p.splits));
  return w;
}

extern "C" int64_t cdssm_int4_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int norm) {
  const char* op = "cdssm_int4_linear_workspace_bytes";
  Size s;
  if (int4_size(op, N, K, 128, &s)) return CDSSM_EINVAL;
  if (M < 1 || M > w4::kMaxRows) {
    cdssm_host::set_error("%s: needs 1 <= M <= %d, got %lld", op, w4::kMaxRows, (long long)M);
    return CDSSM_EINVAL;
  }
  return areas_of(s, plan_of(s, M), M, norm != 0, nullptr).bytes;
}

static int int4_linear(const char* op, int dtype, const void* X, int64_t ldx, const void* words, const void* word_scales, int64_t group,
                       const void* bias, const void* R, int64_t ldr, const void* wnorm, float eps, void* Y, int64_t ldy, void* workspace,
                       int64_t M, int64_t N, int64_t K, const w4::Conv& conv, hipStream_t stream) {
  Size s;
  if (const int st = int4_size(op, N, K, group, &s)) return st;
  if (dtype != 1) {
    cdssm_host::set_error("%s: bf16 only (dtype 1), got %d", op, dtype);
    return CDSSM_EINVAL;
  }
  if (!X || !words || !word_scales || !Y) {
    cdssm_host::set_error("%s: null pointer argument", op);
    return CDSSM_EINVAL;
  }
  if (M < 1 || M > w4::kMaxRows) {
    cdssm_host::set_error("%s: needs 1 <= M <= %d, got %lld", op, w4::kMaxRows, (long long)M);
    return CDSSM_EINVAL;
  }
  const auto at = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  const int64_t whole = (K + 7) / 8 * 8, most = int64_t(1) << 24;
  if (ldx < whole || ldx % 8 || ldx > (int64_t(1) << 32) || (at(X) | at(wnorm) | at(words) | at(word_scales) | at(workspace)) % 16) {
    cdssm_host::set_error("%s: rows of X must be 16-byte aligned and cover K rounded up to 8, and wnorm, the weight's tensors and the "
                          "workspace be 16-byte aligned", op);
    return CDSSM_EINVAL;
  }
  if (ldy < N || ldy > most || (R && (ldr < N || ldr > most)) || (at(Y) | at(R) | at(bias)) % 2) {
    cdssm_host::set_error("%s: row strides of Y and R must be within N .. 2^24, and the tensors aligned to their elements", op);
    return CDSSM_EINVAL;
  }
  const w4::Args a{static_cast<const uint16_t*>(X), ldx, static_cast<const uint4*>(words), static_cast<const uint16_t*>(word_scales),
                   static_cast<const uint16_t*>(bias), static_cast<const uint16_t*>(R), static_cast<const uint16_t*>(wnorm), ldr,
                   static_cast<uint16_t*>(Y), ldy, int(M), int(N), int(K), eps, conv};
  const Plan p = plan_of(s, M);
  if (!workspace && areas_of(s, p, M, wnorm, nullptr).bytes > 0) {
    cdssm_host::set_error("%s: these sizes need a workspace", op);
    return CDSSM_EINVAL;
  }
  const auto go = [&](auto gc, auto norm, auto mt, auto nt) {
    constexpr int G = decltype(gc)::value, MT = decltype(mt)::value, NT = decltype(nt)::value;
    constexpr bool kNorm = decltype(norm)::value;
    const dim3 grid(unsigned(p.groups), unsigned(p.splits));
    if constexpr (NT <= 2) {
      const auto keep = [&](auto w) {
        constexpr int W = decltype(w)::value;
        if constexpr (kNorm)
          if (conv.y) {
            hipLaunchKernelGGL((w4::resident_kernel<G, kNorm, MT, NT, W, true>), grid, dim3(kWave * W), 0, stream, a);
            return;
          }
        hipLaunchKernelGGL((w4::resident_kernel<G, kNorm, MT, NT, W, false>), grid, dim3(kWave * W), 0, stream, a);
      };
      if (p.waves == 2) return keep(std::integral_constant<int, 2>{});
      if (p.waves == 4) return keep(std::integral_constant<int, 4>{});
      if (p.waves == 8) return keep(std::integral_constant<int, 8>{});
    }
    const dim3 block(kWave * w4::kStreamWaves);
    const Areas w = areas_of(s, p, M, kNorm, workspace);
    if constexpr (kNorm)
      if (!p.planes) {
        hipLaunchKernelGGL((w4::stream_kernel<G, w4::kNormed, MT, NT, false>), grid, block, 0, stream, a, nullptr, nullptr, nullptr);
        return;
      }
    constexpr w4::Source kSource = kNorm ? w4::kPlanes : w4::kPlain;
    if constexpr (kNorm)
      hipLaunchKernelGGL(w4::norm_kernel, dim3(unsigned((s.blocks + w4::kShare - 1) / w4::kShare), unsigned((M + 15) / 16)),
                         dim3(kWave * w4::kShare), 0, stream, a, w.planes, w.squares);
    if (p.splits == 1) {
      hipLaunchKernelGGL((w4::stream_kernel<G, kSource, MT, NT, false>), grid, block, 0, stream, a, w.planes, w.squares, nullptr);
      return;
    }
    hipLaunchKernelGGL((w4::stream_kernel<G, kSource, MT, NT, true>), grid, block, 0, stream, a, w.planes, w.squares, w.sums);
    hipLaunchKernelGGL(w4::join_kernel<kNorm>, dim3(unsigned(s.tiles * ((M + 15) / 16))), dim3(kWave), 0, stream, a, w.squares, w.sums,
                       p.splits);
  };
  using std::integral_constant;
  const auto tiles = [&](auto gc, auto norm, auto mt) {
    p.nt == 1   ? go(gc, norm, mt, integral_constant<int, 1>{})
    : p.nt == 2 ? go(gc, norm, mt, integral_constant<int, 2>{})
                : go(gc, norm, mt, integral_constant<int, 4>{});
  };
  const auto rows = [&](auto gc, auto norm) {
    p.mt == 1 ? tiles(gc, norm, integral_constant<int, 1>{}) : tiles(gc, norm, integral_constant<int, 2>{});
  };
  const auto groups = [&](auto gc) { wnorm ? rows(gc, std::true_type{}) : rows(gc, std::false_type{}); };
  group == 32   ? groups(integral_constant<int, 32>{})
  : group == 64 ? groups(integral_constant<int, 64>{})
                : groups(integral_constant<int, 128>{});
  return cdssm_host::check_launch(op);
}

extern "C" int cdssm_int4_linear(int dtype, const void* X, int64_t ldx, const void* words, const void* word_scales, int64_t group,
                                 const void* bias, const void* R, int64_t ldr, const void* wnorm, float eps, void* Y, int64_t ldy,
                                 void* workspace, int64_t M, int64_t N, int64_t K, hipStream_t stream) {
  return int4_linear("cdssm_int4_linear", dtype, X, ldx, words, word_scales, group, bias, R, ldr, wnorm, eps, Y, ldy, workspace, M, N,
                     K, w4::Conv{}, stream);
}

extern "C" int cdssm_int4_linear_conv_step(int dtype, const void* X, int64_t ldx, const void* words, const void* word_scales,
                                           int64_t group, const void* bias, const void* wnorm, float eps, void* Y, int64_t ldy,
                                           void* workspace, int64_t M, int64_t N, int64_t K, int64_t conv_col, void* window,
                                           const void* conv_weight, const void* conv_bias, void* conv_y, int64_t C, int64_t taps,
                                           hipStream_t stream) {
  const char* op = "cdssm_int4_linear_conv_step";
  if (!conv_weight || !conv_bias || !conv_y || (taps > 1 && !window)) {
    cdssm_host::set_error("%s: null pointer argument", op);
    return CDSSM_EINVAL;
  }
  if (taps < 1 || taps > w4::kMaxTaps || C < 1 || conv_col < 0 || C > N || conv_col > N - C) {
    cdssm_host::set_error("%s: needs 1 <= kernel_size <= 8 and the conv's columns inside the product's (column %lld, C %lld, N %lld, "
                          "kernel_size %lld)", op, (long long)conv_col, (long long)C, (long long)N, (long long)taps);
    return CDSSM_EINVAL;
  }
  const auto at = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  if ((at(window) | at(conv_weight) | at(conv_bias) | at(conv_y)) % 2) {
    cdssm_host::set_error("%s: the conv's tensors must be aligned to their elements", op);
    return CDSSM_EINVAL;
  }
  const w4::Conv cv{static_cast<uint16_t*>(window), static_cast<uint16_t*>(conv_y), static_cast<const uint16_t*>(conv_weight),
                    static_cast<const uint16_t*>(conv_bias), int(conv_col), int(C), int(taps)};
  // short rows with a norm in one launch, others in two: the conv's registers would cost the longer kernels half of their waves
  const bool one = wnorm && K <= 8 * w4::kBlock;
  if (const int st = int4_linear(op, dtype, X, ldx, words, word_scales, group, bias, nullptr, 0, wnorm, eps, Y, ldy, workspace, M, N, K,
                                 one ? cv : w4::Conv{}, stream))
    return st;
  return one ? CDSSM_OK : cdssm_conv1d_silu_step(dtype, static_cast<const uint16_t*>(Y) + conv_col, ldy, window, conv_weight, conv_bias,
                                                 conv_y, M, C, taps, stream);
}
