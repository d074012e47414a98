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

// An operand from its tile's first row (column): element (r, k) at base[r * ld + k] (KMajor) or base[k * ld + r]; it has
// `end` elements from there (rows of 64 k at least).  What lies behind them comes as 0: the loads go through a buffer resource, whose
// range check covers the bytes up to the end.  Rows (columns) of the tile that do not exist may bring zeros or elements of
// their neighbours; only the results' rows of theirs, which nobody keeps, see those.
// Planes (fp32 operands split into three bf16 matrices) lie `plane` elements apart.
struct Operand {
  const uint16_t* base;
  int64_t ld, plane, end;
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

// 16 bytes a lane from a buffer resource (offset voff + soff; 0 beyond its end) to LDS, lane l's to lds + 16 l.  Written
// as an instruction: for the builtin the compiler waits for every load under way before each read of LDS, which takes away
// the time that the loads have.  It has no result register; wait_and_meet() is what waits for it.
typedef int i32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void load_to_lds(const void* p, uint32_t bytes, uint32_t lds, int voff, int soff) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  const i32x4_t rs = {int(uint32_t(a)), int(uint32_t(a >> 32) & 0xffffu), int(bytes), 0x00020000};
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is the compiler's to set, which is said here
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(voff), "s"(rs), "s"(soff)
               : "memory", "m0");
#pragma clang diagnostic pop
}
// Waits until all but N of this wave's accesses to global memory, and all its reads of LDS, have come back, then for the
// other waves to get here.
template <int N>
__device__ __forceinline__ void wait_and_meet() {
  static_assert(N < 64, "vmcnt has 6 bits");
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// Brings a step of an operand into LDS, a quarter at a time: one load of 16 bytes a lane, a quarter's rows `apart` bytes
// from the last one's.
template <bool MMajor, bool Paired>
struct Stager {
  int voff, apart;
  __device__ __forceinline__ void init(const Operand& o, int wave, int lane) {
    const int idx = wave * kWave + lane;
    if constexpr (MMajor) {
      const int k = idx >> 5, c = (idx & 31) ^ swz_m(k);
      voff = k * int(o.ld * 2) + c * 16;
      apart = 16 * int(o.ld * 2);
    } else {
      const int r = idx >> 3, c = (idx & 7) ^ swz_k<Paired>(r);
      voff = r * int(o.ld * 2) + c * 16;
      apart = 64 * int(o.ld * 2);
    }
  }
  __device__ __forceinline__ void stage(const uint16_t* p, uint32_t bytes, lds_byte* lds, int wave, int i) const {
    load_to_lds(p, bytes, uint32_t(reinterpret_cast<uintptr_t>(lds)) + (i * kWaves + wave) * kWave * 16, voff, i * apart);
  }
};

// Reads the wave's fragments of a staged step; r0: its first row in the tile.
template <bool MMajor, bool Paired, int N>
struct Reader {
  static constexpr int kAt = MMajor ? 1 : Paired ? 4 : 2;
  int at[kAt];
  __device__ __forceinline__ void init(int r0, int lane) {
    const int lo = lane & 15, g = lane >> 4;
    if constexpr (MMajor) {
      static_assert(!Paired, "only k-contiguous operands come in pairs of fragments");
      // lane s of a group of 16 reads 4 m at row k = 8 g + 4 h + s / 4; h and the half of the step are added below
      const int k = 8 * g + lo / 4, x = swz_m(k) * 16;
      at[0] = k * (kTile * 2) + ((r0 * 2) ^ x) + 8 * (lo & 3);
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
      // fragment a's columns: 32 a bytes on, under the swizzle an exclusive or; formed here, as N addresses held over
      // the loop cost registers that the fragments need
      int b = at[0];
      asm("" : "+v"(b));
      b ^= 32 * a;
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(lds + b + S * 32 * kTile * 2));
      const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(lds + b + (S * 32 + 4) * kTile * 2));
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
// start() requests the first two steps and may be called before the results of the last tile are stored; run() waits
// for them, not for the stores.  While the products of one half of a step run, the fragments of the next half are read, and the loads of the step
// after the next are under way.
template <bool AM, bool BM, bool Paired = false>
struct Multiply {
  Stager<AM, Paired> sa;
  Stager<BM, false> sb;
  Reader<AM, Paired, kI> ra;
  Reader<BM, false, kJ> rb;
  Operand A, B;
  const uint16_t *pa, *pb;
  int nk, kk, p, n;  // kk, p: k step and pair of the next step to stage; n: steps to go
  uint32_t bytes_a, bytes_b;  // of the operands from pa, pb
  Pairs pairs;
  lds_byte* lds;
  int wave;

  __device__ __forceinline__ Multiply(Pairs pairs_, lds_byte* lds_) : pairs(pairs_), lds(lds_) {
    wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
    const int lane = int(threadIdx.x) % kWave;
    ra.init((wave >> 2) * kWM, lane);
    rb.init((wave & 3) * kWN, lane);
  }
  __device__ __forceinline__ static uint32_t range(int64_t elements) {
    return uint32_t(max(int64_t(0), min(elements * 2, int64_t(0xffffffff))));
  }
  __device__ __forceinline__ void point() {
    const int64_t ka = kk * (AM ? kStep * A.ld : int64_t(kStep)), kb = kk * (BM ? kStep * B.ld : int64_t(kStep));
    pa = A.base + pairs.a(p) * A.plane + ka;
    pb = B.base + pairs.b(p) * B.plane + kb;
    bytes_a = range(A.end - ka);
    bytes_b = range(B.end - kb);
  }
  // Load q of the eight of a step; the last one moves on to the next step.
  __device__ __forceinline__ void stage(int buf, int q) {
    lds_byte* l = lds + buf * 2 * kStageBytes;
    if (q < 4) {
      sa.stage(pa, bytes_a, l, wave, q);
      return;
    }
    sb.stage(pb, bytes_b, l + kStageBytes, wave, q - 4);
    if (q < 7) return;
    if (++kk == nk) {
      kk = 0;
      ++p;
    }
    point();
  }
  __device__ __forceinline__ void stage(int buf) {
#pragma unroll
    for (int q = 0; q < 8; ++q) stage(buf, q);
  }
  __device__ __forceinline__ void start(const Operand& A_, const Operand& B_, int nk_, int q0, int q1) {
    A = A_;
    B = B_;
    nk = nk_;
    n = q1 - q0;
    p = q0 / nk;
    kk = q0 - p * nk;
    point();
    const int lane = int(threadIdx.x) % kWave;
    sa.init(A, wave, lane);
    sb.init(B, wave, lane);
    stage(0);
    if (n > 1) stage(1);
  }
  // Younger: accesses to global memory that every wave has at least made since start().
  template <int Younger>
  __device__ __forceinline__ void run(Acc& acc) {
    bf16x8_t fa[2][kI], fb[2][kJ];
    // two fragments of a half: B's, then A's
    auto read = [&](int buf, auto sc, int h) {
      constexpr int S = decltype(sc)::value;
      const lds_byte* l = lds + buf * 2 * kStageBytes;
#pragma unroll
      for (int f = 2 * h; f < 2 * h + 2; ++f) {
        if (f < kJ)
          fb[S][f] = rb.template read<S>(l + kStageBytes, f);
        else if (f < kI + kJ)
          fa[S][f - kJ] = ra.template read<S>(l, f - kJ);
      }
    };
    // the products of half S, and between them between(0 .. 7): loads and reads go out among the matrix
    // instructions instead of holding them up
    auto products = [&](auto sc, auto&& between) {
      constexpr int S = decltype(sc)::value;
#pragma unroll
      for (int i = 0; i < kI; ++i) {
        between(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < kJ; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[S][i], fb[S][j], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;
    if (n > 1)
      wait_and_meet<8 + Younger>();
    else
      wait_and_meet<0>();
#pragma unroll
    for (int h = 0; h < kI; ++h) read(0, S0{}, h);
    for (int s = 0; s < n; ++s) {
      products(S0{}, [&](int h) { read(s & 1, S1{}, h); });
      // step s + 1 is in LDS, and everyone has read step s
      if (Younger && s == 0)
        wait_and_meet<Younger>();
      else
        wait_and_meet<0>();
      const bool load = s + 2 < n;
      products(S1{}, [&](int h) {
        read((s + 1) & 1, S0{}, h);  // after the last step: what is left there, for nothing
        if (load) stage(s & 1, h);
      });
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
