// Matrix products on 256 x 256 tiles for gfx950: C[m][n] = sum_k A(m, k) B(n, k), bf16 operands, fp32 sums.
//
// A workgroup of 8 waves owns a tile, a wave 128 (m) x 64 (n) of it as 8 x 4 products v_mfma_f32_16x16x32_bf16
// (lane l: A row l % 16, B row l % 16, both k = 8 (l / 16) .. + 8; C column n = l % 16, rows m = 4 (l / 16) .. + 4,
// so a lane's four values lie next to each other along m).  The operands come in steps of 64 k, straight from global
// memory into LDS (16 bytes a lane), double buffered: 2 x (32 + 32) KB.  An operand lies in memory either with k
// contiguous (KMajor: LDS rows of 64 k, 128 bytes, read 16 bytes a lane) or with m (n) contiguous (MMajor: LDS rows
// of 256 m, 512 bytes, read through the transposing ds_read_b64_tr_b16, whose group of 16 lanes turns 4 rows of k x 16
// m into 16 rows of m x 4 k).  LDS is written in lane order, so its swizzles (below) are made by the order in which
// the lanes read global memory.
#pragma once

#include "common.hpp"

namespace cdssm {
namespace mma {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kTile = 256, kStep = 64, kWaves = 8, kThreads = kWaves * kWave;
constexpr int kStageBytes = kTile * kStep * 2;  // one operand's step in LDS
constexpr int kWM = 128, kWN = 64;              // a wave's part of the tile
constexpr int kI = kWM / 16, kJ = kWN / 16;

typedef f32x4_t Acc[kI][kJ];
typedef __attribute__((address_space(3))) unsigned char lds_byte;

// An operand from its tile's first row (column): element (r, k) at base[r * ld + k] (KMajor) or base[k * ld + r].
// `limit`: the rows (KMajor) or columns (MMajor, a multiple of 8) from base that exist; beyond it the last ones are read again.
// Planes (fp32 operands split into three bf16 matrices) lie `plane` elements apart.
struct Operand {
  const uint16_t* base;
  int64_t ld, plane;
  int limit;
};

// Row of the tile that row r of fragment a (of 16 rows) stands for.  Paired: two fragments interleave in fours, so that a
// lane's 2 x 4 results lie next to each other (16 bytes of bf16).
template <bool Paired>
__device__ __forceinline__ int frag_row(int a, int r) {
  return Paired ? 32 * (a >> 1) + 8 * (r >> 2) + 4 * (a & 1) + (r & 3) : 16 * a + r;
}

// The 16-byte chunk of LDS row r that logical chunk c lies in is c ^ this: the 16 rows that a read touches at once (rows
// 0 .. 15, or in pairs of fragments 0 .. 3, 8 .. 11, 16 .. 19, 24 .. 27) lie in other banks.
template <bool Paired>
__device__ __forceinline__ int swz_k(int r) {  // of 8 chunks
  return Paired ? ((r >> 1) & 1) | ((r >> 2) & 6) : (r >> 1) & 7;
}
__device__ __forceinline__ int swz_m(int k) { return ((k & 3) | ((k >> 3) & 1) << 2) * 2; }  // of 32 chunks

template <bool MMajor, bool Paired>
struct Stager {
  uint32_t voff[4];
  __device__ __forceinline__ void init(const Operand& o, int wave, int lane, int kmax = kStep) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int idx = (i * kWaves + wave) * kWave + lane;
      if constexpr (MMajor) {
        const int k = idx >> 5, c = (idx & 31) ^ swz_m(k);
        voff[i] = uint32_t(min(k, kmax - 1)) * uint32_t(o.ld * 2) + uint32_t(min(c * 8, o.limit - 8)) * 2u;
      } else {
        const int r = idx >> 3, c = (idx & 7) ^ swz_k<Paired>(r);
        voff[i] = uint32_t(min(r, o.limit - 1)) * uint32_t(o.ld * 2) + uint32_t(c) * 16u;
      }
    }
  }
  __device__ __forceinline__ void stage(const uint16_t* p, lds_byte* lds, int wave) const {
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p), short(0), -1, 0x00020000);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (__attribute__((address_space(3))) void*)(lds + (i * kWaves + wave) * kWave * 16), 16, int(voff[i]), 0, 0, 0);
  }
};

// Reads the wave's fragments of a staged step; r0: its first row in the tile.
template <bool MMajor, bool Paired, int N>
struct Reader {
  static constexpr int kAt = MMajor ? N : Paired ? 4 : 2;
  int at[kAt];
  __device__ __forceinline__ void init(int r0, int lane) {
    const int lo = lane & 15, g = lane >> 4;
    if constexpr (MMajor) {
      static_assert(!Paired, "only k-contiguous operands come in pairs of fragments");
      // lane s of a group of 16 reads 4 m at row k = 8 g + 4 h + s / 4; h and the half of the step are added below
      const int k = 8 * g + lo / 4, x = swz_m(k) * 16;
#pragma unroll
      for (int a = 0; a < N; ++a) at[a] = k * (kTile * 2) + (((r0 + 16 * a) * 2) ^ x) + 8 * (lo & 3);
    } else {
#pragma unroll
      for (int q = 0; q < kAt; ++q) {  // half of the step, and with pairs which of the two
        const int r = r0 + frag_row<Paired>(q >> 1, lo);
        at[q] = r * (kStep * 2) + (((4 * (q & 1) + g) ^ swz_k<Paired>(r)) * 16);
      }
    }
  }
  template <int S>
  __device__ __forceinline__ bf16x8_t read(const lds_byte* lds, int a) const {
    if constexpr (MMajor) {
      typedef __attribute__((address_space(3))) s16x4_t lds_s4;
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(lds + at[a] + S * 32 * kTile * 2));
      const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(lds + at[a] + (S * 32 + 4) * kTile * 2));
      return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      typedef __attribute__((address_space(3))) s16x8_t lds_s8;
      if constexpr (Paired)
        return __builtin_bit_cast(bf16x8_t, *(const lds_s8*)(lds + at[2 * (a & 1) + S] + (a >> 1) * 32 * kStep * 2));
      else
        return __builtin_bit_cast(bf16x8_t, *(const lds_s8*)(lds + at[S] + a * 16 * kStep * 2));
    }
  }
};

// The products of a pair of operands: one for bf16 planes; for fp32 operands split into three bf16 planes, the six
// products of at least 2^-16 of the largest, the small ones first.
struct Pairs {
  int n;
  __device__ __forceinline__ int a(int p) const { return n == 1 ? 0 : (0x046 >> (2 * p)) & 3; }  // 2 1 0 1 0 0
  __device__ __forceinline__ int b(int p) const { return n == 1 ? 0 : (0x124 >> (2 * p)) & 3; }  // 0 1 2 0 1 0
};

// acc += the products of steps q0 .. q1 of both operands, counted through the pairs of planes (nk steps of k each).
// start() requests the first step and may be called before the results of the last tile are done with; run() waits
// for it.  While the products of one half of a step run, the fragments of the next half are read, and the loads of the step
// after the next are under way.
template <bool AM, bool BM, bool Paired = false>
struct Multiply {
  Stager<AM, Paired> sa;
  Stager<BM, false> sb;
  Reader<AM, Paired, kI> ra;
  Reader<BM, false, kJ> rb;
  Operand A, B;
  const uint16_t *pa, *pb;
  int nk, kk, p, n, klimit;  // kk, p: k step and pair of the next step to stage; n: steps to go
  Pairs pairs;
  lds_byte* lds;
  int wave;

  __device__ __forceinline__ Multiply(Pairs pairs_, lds_byte* lds_) : pairs(pairs_), lds(lds_) {
    wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
    const int lane = int(threadIdx.x) % kWave;
    ra.init((wave >> 2) * kWM, lane);
    rb.init((wave & 3) * kWN, lane);
  }
  __device__ __forceinline__ void point() {
    pa = A.base + pairs.a(p) * A.plane + kk * (AM ? kStep * A.ld : int64_t(kStep));
    pb = B.base + pairs.b(p) * B.plane + kk * (BM ? kStep * B.ld : int64_t(kStep));
  }
  __device__ __forceinline__ void stage(int buf) {
    lds_byte* l = lds + buf * 2 * kStageBytes;
    if (AM && (kk + 1) * kStep > klimit) {
      Stager<AM, Paired> s;
      s.init(A, wave, int(threadIdx.x) % kWave, max(1, klimit - kk * kStep));
      s.stage(pa, l, wave);
    } else {
      sa.stage(pa, l, wave);
    }
    sb.stage(pb, l + kStageBytes, wave);
    pa += AM ? kStep * A.ld : int64_t(kStep);
    pb += BM ? kStep * B.ld : int64_t(kStep);
    if (++kk == nk) {
      kk = 0;
      ++p;
      point();
    }
  }
  // klimit_: the k rows of an MMajor A that exist from its base (beyond it the last one is read again; B is zero there)
  __device__ __forceinline__ void start(const Operand& A_, const Operand& B_, int nk_, int q0, int q1, int klimit_ = 1 << 30) {
    A = A_;
    B = B_;
    nk = nk_;
    klimit = klimit_;
    n = q1 - q0;
    p = q0 / nk;
    kk = q0 - p * nk;
    point();
    const int lane = int(threadIdx.x) % kWave;
    sa.init(A, wave, lane);
    sb.init(B, wave, lane);
    stage(0);
  }
  __device__ __forceinline__ void run(Acc& acc) {
    bf16x8_t fa[2][kI], fb[2][kJ];
    auto read = [&](int buf, auto sc) {
      constexpr int S = decltype(sc)::value;
      const lds_byte* la = lds + buf * 2 * kStageBytes;
#pragma unroll
      for (int j = 0; j < kJ; ++j) fb[S][j] = rb.template read<S>(la + kStageBytes, j);
#pragma unroll
      for (int i = 0; i < kI; ++i) fa[S][i] = ra.template read<S>(la, i);
    };
    auto products = [&](auto sc) {
      constexpr int S = decltype(sc)::value;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int j = 0; j < kJ; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[S][i], fb[S][j], acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    };
    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;
    __syncthreads();
    if (n > 1) stage(1);
    read(0, S0{});
    for (int s = 0; s < n; ++s) {
      read(s & 1, S1{});
      products(S0{});
      __syncthreads();  // step s + 1 is in LDS, and everyone has read step s
      if (s + 1 < n) {
        read((s + 1) & 1, S0{});
        if (s + 2 < n) stage(s & 1);
      }
      products(S1{});
    }
  }
};

__device__ __forceinline__ void clear(Acc& acc) {
#pragma unroll
  for (int i = 0; i < kI; ++i)
#pragma unroll
    for (int j = 0; j < kJ; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
}

// Workgroup b's place among n, so that the workgroups of one XCD (every eighth) have neighbouring places.
__device__ __forceinline__ int xcd_place(int b, int n) {
  const int per = n / 8, rest = n % 8, x = b % 8, i = b / 8;
  return x * per + min(x, rest) + i;
}

// Place p of a grid of rows x cols tiles, walked in bands of `band` rows.
__device__ __forceinline__ void banded(int p, int rows, int cols, int band, int& r, int& c) {
  const int g = p / (band * cols), r0 = g * band, h = min(band, rows - r0), q = p - g * band * cols;
  r = r0 + q % h;
  c = q / h;
}

}  // namespace mma
}  // namespace cdssm
