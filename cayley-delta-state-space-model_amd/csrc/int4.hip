// Decode products with weights of 4 bits: Y (M x N) = X' (M x K) W^T (+ bias) (+ R), M <= 64, with
//   W[n][k] = s[n][k / g] c[n][k],   c a whole number of -8 .. 7, s bf16, g 32, 64 or 128
// and X' = X, or with a norm weight X' = rs X w_norm, rs[m] = rsqrt(mean_k X[m][k]^2 + eps).  bf16 X and Y, fp32 sums.
//
// A call reads N K / 2 bytes of codes and little else, so it is bound by memory, or for the small layers by the latency of one
// load and one sum.  No weight is rounded: the codes go into the matrix cores as the whole numbers that they are, and the sum
// over a group is multiplied by its scale in fp32.  A code travels as c + 8 in 4 bits; with 0x4300 above it those bits are the
// bf16 number 128 + 8 + c, so 8 codes take 7 instructions, and the 136 too many are taken out by starting a group's sum from
// -136 times the sum of X over the group: the product of X with a constant, once for all columns.  (Those sums are up to 136 / 8
// times what the result's are: fp32 leaves them 2^-24 of that, far below the rounding to bf16.)
//
// Layout (int4_words): per 16 columns n and 128 k one KB, in the order in which a wave's lanes load it: lane l holds column
// l % 16, and of each of the four steps of 32 k eight codes from 8 (l / 16) on, in one word.  Scales: per 16 columns and 128 k,
// a lane's 128 / g next to each other.
//
// A workgroup owns 16 NT columns and 16 MT rows; its waves take blocks of 128 k in turn, and their sums are added in a
// fixed order through LDS.
//
// Fragment layouts of v_mfma_f32_16x16x32_bf16: as in skinny_gemm.hip.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.hpp"

namespace cdssm {
namespace w4 {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kCols = 16, kBlock = 128, kSteps = kBlock / 32, kMaxRows = 64;
constexpr int64_t kMaxSize = int64_t(1) << 24;  // of N and K

__device__ __forceinline__ f32x4_t mfma(uint4 a, uint4 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// Eight codes as 136 + c in bf16: element 2 i in nibble i, 2 i + 1 in nibble i + 4.
__device__ __forceinline__ uint4 codes_of(uint32_t w) {
  constexpr uint32_t kMask = 0x000f000fu, kBase = 0x43004300u;
  return make_uint4((w & kMask) | kBase, ((w >> 4) & kMask) | kBase, ((w >> 8) & kMask) | kBase, ((w >> 12) & kMask) | kBase);
}

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
};

// Elements k .. k + 8 of a row of K, zeros behind its end.
template <bool Aligned>
__device__ __forceinline__ uint4 load8(const uint16_t* row, int k, int K) {
  if constexpr (Aligned) {
    return k < K ? *reinterpret_cast<const uint4*>(row + k) : make_uint4(0, 0, 0, 0);
  } else {
    uint32_t e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = k + i < K ? row[k + i] : 0;
    return make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
  }
}

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

template <int G, bool Norm, bool Aligned, int MT, int NT, int W>
__global__ __launch_bounds__(kWave* W) void linear_kernel(Args a) {
  constexpr int kGroups = kBlock / G, kPerGroup = G / 32, P = Norm ? 2 : 1;
  __shared__ f32x4_t part[W][MT * NT][kWave];
  __shared__ float ssq[W][16 * MT];
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave), lane = int(threadIdx.x) % kWave;
  const int col = lane % 16, kq = lane / 16;
  const int n_tiles = (a.N + kCols - 1) / kCols, n_blocks = (a.K + kBlock - 1) / kBlock;
  const int mgs = (a.M + 16 * MT - 1) / (16 * MT);
  const int mg = int(blockIdx.x) % mgs, t0 = int(blockIdx.x) / mgs * NT, m0 = mg * 16 * MT;
  const uint16_t* xrow[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xrow[i] = a.x + int64_t(min(m0 + 16 * i + col, a.M - 1)) * a.ldx;
  f32x4_t acc[MT][NT];
  float sq[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    sq[i] = 0.0f;
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const uint4 minus = make_uint4(0xc308c308u, 0xc308c308u, 0xc308c308u, 0xc308c308u);  // -136
  for (int b = wave; b < n_blocks; b += W) {
    uint4 w[NT];
    uint16_t sc[NT][kGroups];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int64_t at = int64_t(min(t0 + j, n_tiles - 1)) * n_blocks + b;
      w[j] = a.codes[at * kWave + lane];
      const uint16_t* s = a.scales + (at * kCols + col) * kGroups;
      if constexpr (kGroups == 4) {
        const uint2 u = *reinterpret_cast<const uint2*>(s);
        sc[j][0] = uint16_t(u.x); sc[j][1] = uint16_t(u.x >> 16); sc[j][2] = uint16_t(u.y); sc[j][3] = uint16_t(u.y >> 16);
      } else if constexpr (kGroups == 2) {
        const uint32_t u = *reinterpret_cast<const uint32_t*>(s);
        sc[j][0] = uint16_t(u); sc[j][1] = uint16_t(u >> 16);
      } else {
        sc[j][0] = *s;
      }
    }
    uint4 x[kSteps][MT], wn[kSteps];
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int at = b * kBlock + 32 * k + 8 * kq;
#pragma unroll
      for (int i = 0; i < MT; ++i) x[k][i] = load8<Aligned>(xrow[i], at, a.K);
      if constexpr (Norm) wn[k] = load8<Aligned>(a.wnorm, at, a.K);
    }
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      uint4 xs[kPerGroup][MT][P];
      f32x4_t base[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) base[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < kPerGroup; ++k)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const uint4 v = x[g * kPerGroup + k][i];
          if constexpr (Norm) {
            sq[i] = sum_squares(v, sq[i]);
            scaled(v, wn[g * kPerGroup + k], xs[k][i][0], xs[k][i][1]);
          } else {
            xs[k][i][0] = v;
          }
#pragma unroll
          for (int p = 0; p < P; ++p) base[i] = mfma(xs[k][i][p], minus, base[i]);
        }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        f32x4_t t[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) t[i] = base[i];
#pragma unroll
        for (int k = 0; k < kPerGroup; ++k) {
          const int st = g * kPerGroup + k;
          const uint4 c = codes_of(st == 0 ? w[j].x : st == 1 ? w[j].y : st == 2 ? w[j].z : w[j].w);
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int p = 0; p < P; ++p) t[i] = mfma(xs[k][i][p], c, t[i]);
        }
        const float s = bf16_to_f32(sc[j][g]);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(s, t[i][e], acc[i][j][e]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = acc[i][j];
  if constexpr (Norm) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      float s = sq[i];
      s += __shfl_xor(s, 16, kWave);
      s += __shfl_xor(s, 32, kWave);
      if (kq == 0) ssq[wave][16 * i + col] = s;
    }
  }
  __syncthreads();
  for (int tile = wave; tile < MT * NT; tile += W) {
    const int i = tile / NT, n = (t0 + tile % NT) * kCols + col;
    f32x4_t c = part[0][tile][lane];
#pragma unroll
    for (int v = 1; v < W; ++v) {
      const f32x4_t p = part[v][tile][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) c[e] += p[e];
    }
    const float bias = a.bias && n < a.N ? bf16_to_f32(a.bias[n]) : 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int ml = 16 * i + 4 * kq + e, m = m0 + ml;
      if (m >= a.M || n >= a.N) continue;
      float y = c[e];
      if constexpr (Norm) {
        float s = 0.0f;
#pragma unroll
        for (int v = 0; v < W; ++v) s += ssq[v][ml];
        y *= rsqrtf(s / float(a.K) + a.eps);
      }
      y += bias;
      if (a.residual) y += bf16_to_f32(a.residual[int64_t(m) * a.ldr + n]);
      a.y[int64_t(m) * a.ldy + n] = f32_to_bf16(y);
    }
  }
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

__device__ __forceinline__ uint32_t word_of(const int (&c)[8]) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) w |= (uint32_t(c[i] + 8) & 15u) << 4 * (i / 2 + 4 * (i % 2));
  return w;
}

// codes (N, K) of one byte each, scales (N, groups) to the layout: a thread per word, and per scale.
__global__ void pack_kernel(const int8_t* __restrict__ codes, const uint16_t* __restrict__ scales, uint32_t* __restrict__ words,
                            uint16_t* __restrict__ out, int64_t n_words, int64_t n_scales, int64_t N, int64_t K, int64_t blocks,
                            int64_t g) {
  const int64_t t = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (t < n_words) {
    const Place p = place_of(t, blocks);
    int c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = p.n < N && p.k + i < K ? codes[p.n * K + p.k + i] : 0;
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
        if (p.k + i < K) codes[p.n * K + p.k + i] = int8_t(int(words[t] >> 4 * (i / 2 + 4 * (i % 2)) & 15) - 8);
  }
  if (t < n_scales) {
    const int64_t per = kBlock / g, groups = (K + g - 1) / g;
    const int64_t block = t / (kCols * per), in = t % (kCols * per);
    const int64_t n = block / blocks * kCols + in / per, j = block % blocks * per + in % per;
    if (n < N && j < groups) scales[n * groups + j] = in_scales[t];
  }
}

// A group's scale is its largest magnitude over 7, rounded to bf16, and a code the nearest whole number to w / scale: a thread per
// group.  A group below 2^-120 throughout becomes 0; one that holds an infinity or NaN gets the scale NaN.
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

extern "C" int cdssm_int4_linear(int dtype, const void* X, int64_t ldx, const void* words, const void* word_scales, int64_t group,
                                 const void* bias, const void* R, int64_t ldr, const void* wnorm, float eps, void* Y, int64_t ldy,
                                 int64_t M, int64_t N, int64_t K, hipStream_t stream) {
  const char* op = "cdssm_int4_linear";
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
  if (ldx < K || ldy < N || (R && ldr < N) || std::max(ldx, std::max(ldy, R ? ldr : 0)) > (int64_t(1) << 32) || at(words) % 16 ||
      at(word_scales) % 16 || (at(X) | at(Y) | at(R) | at(bias) | at(wnorm)) % 2) {
    cdssm_host::set_error("%s: row strides must cover the rows, the layout's tensors be 16-byte aligned, the others to their elements", op);
    return CDSSM_EINVAL;
  }
  const w4::Args a{static_cast<const uint16_t*>(X), ldx, static_cast<const uint4*>(words), static_cast<const uint16_t*>(word_scales),
                     static_cast<const uint16_t*>(bias), static_cast<const uint16_t*>(R), static_cast<const uint16_t*>(wnorm), ldr,
                     static_cast<uint16_t*>(Y), ldy, int(M), int(N), int(K), eps};
  const bool aligned = ldx % 8 == 0 && K % 8 == 0 && (at(X) | at(wnorm)) % 16 == 0;
  using std::integral_constant;
  const auto go = [&](auto gc, auto norm, auto al, auto mt, auto nt) {
    constexpr int G = decltype(gc)::value, MT = decltype(mt)::value, NT = decltype(nt)::value, W = 8;
    const int64_t groups = (s.tiles + NT - 1) / NT * ((M + 16 * MT - 1) / (16 * MT));
    hipLaunchKernelGGL((w4::linear_kernel<G, decltype(norm)::value, decltype(al)::value, MT, NT, W>), dim3(unsigned(groups)),
                       dim3(kWave * W), 0, stream, a);
  };
  const auto rows = [&](auto gc, auto norm, auto al) {
    if (M <= 16)
      go(gc, norm, al, integral_constant<int, 1>{}, integral_constant<int, 1>{});
    else if (M <= 32)
      go(gc, norm, al, integral_constant<int, 2>{}, integral_constant<int, 1>{});
    else
      go(gc, norm, al, integral_constant<int, 4>{}, integral_constant<int, 1>{});
  };
  const auto al = [&](auto gc, auto norm) { aligned ? rows(gc, norm, std::true_type{}) : rows(gc, norm, std::false_type{}); };
  const auto nm = [&](auto gc) { wnorm ? al(gc, std::true_type{}) : al(gc, std::false_type{}); };
  group == 32 ? nm(integral_constant<int, 32>{}) : group == 64 ? nm(integral_constant<int, 64>{}) : nm(integral_constant<int, 128>{});
  return cdssm_host::check_launch(op);
}
