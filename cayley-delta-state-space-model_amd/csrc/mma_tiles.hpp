// Matrix products on square tiles for gfx950: C[m][n] = sum_k A(m, k) B(n, k), bf16 operands, fp32 sums.
//
// A workgroup of 8 waves owns a tile, a wave half (m) x a quarter (n) of it in products v_mfma_f32_16x16x32_bf16
// (lane l: A row l % 16, B row l % 16, both k = 8 (l / 16) .. + 8; C column n = l % 16, rows m = 4 (l / 16) .. + 4,
// so a lane's four values lie next to each other along m).  The operands come in steps of k, straight from global
// memory into LDS (16 bytes a lane).  An operand lies in memory either with k contiguous (KMajor: LDS rows of a step's k,
// read 16 bytes a lane) or with m (n) contiguous (MMajor: LDS rows of the tile's m, read through the transposing
// ds_read_b64_tr_b16, whose group of 16 lanes turns 4 rows of k x 16 m into 16 rows of m x 4 k).  LDS is written in lane
// order, so its swizzles (below) are made by the order in which the lanes read global memory.
//
// Three engines.  Engine<1, 256>, bf16: tiles of 256, steps of 64 k in two halves, double buffered (128 KB).  Engine<1, 128>, bf16
// where there are few tiles, and a workgroup's time is that of its loads: tiles of 128, steps of 32 k, eight buffers (128 KB), so that
// seven steps are under way.  Engine<3, 128>, fp32, an operand as three bf16 planes that add up to it: tiles of 128, steps of 32 k, all planes of both operands at once and the six products
// of planes that count on each step, three buffers (144 KB).  The same bytes for each matrix instruction, and where there are few tiles
// four times as many with half the work between barriers: loss and gradients of 100 x 1024 with 300 words take 128 us, with
// Engine<1, 256> going through the pairs of planes one after the other 336; 512 x 768 x 5000 177 and 327; 2048 x 768 x 32000
// 2294 and 2269.
#pragma once

#include "common.hpp"

namespace cdssm {
namespace mma {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) unsigned char lds_byte;

constexpr int kWaves = 8, kThreads = kWaves * kWave;

// An operand from its tile's first row (column): element (r, k) at base[r * ld + k] (KMajor) or base[k * ld + r]; it has
// `end` elements from there (rows of a step's k at least).  What lies behind them comes as 0: the loads go through a buffer
// resource, whose range check covers the bytes up to the end.  Rows (columns) of the tile that do not exist may bring zeros or
// elements of their neighbours; only the results' rows of theirs, which nobody keeps, see those.
// Planes lie `plane` elements apart.
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
template <bool Paired, int Chunks>
__device__ __forceinline__ int swz_k(int r) {
  if constexpr (Chunks == 8)
    return Paired ? ((r >> 1) & 1) | ((r >> 2) & 6) : (r >> 1) & 7;
  else
    return Paired ? (r >> 3) & 3 : (r >> 2) & 3;
}
__device__ __forceinline__ int swz_m(int k) { return ((k & 3) | ((k >> 3) & 1) << 2) * 2; }

// 16 bytes a lane from a buffer resource (offset voff + soff; 0 beyond its end) to LDS, lane l's to lds + 16 l.  Written
// as an instruction: for the builtin the compiler waits for every load under way before each read of LDS, which takes away
// the time that the loads have.  It has no result register; wait_and_meet() is what waits for it.
typedef int i32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void load_to_lds(const void* p, uint32_t bytes, uint32_t lds, int voff, int soff) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  const i32x4_t rs = {__builtin_amdgcn_readfirstlane(int(uint32_t(a))), __builtin_amdgcn_readfirstlane(int(uint32_t(a >> 32) & 0xffffu)),
                      __builtin_amdgcn_readfirstlane(int(bytes)), 0x00020000};
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

// The products of planes that count, those of at least 2^-16 of the largest, the small ones first: planes of A and B.
template <int P>
__device__ __forceinline__ constexpr int pair_a(int p) { return P == 1 ? 0 : (0x046 >> (2 * p)) & 3; }  // 2 1 0 1 0 0
template <int P>
__device__ __forceinline__ constexpr int pair_b(int p) { return P == 1 ? 0 : (0x124 >> (2 * p)) & 3; }  // 0 1 2 0 1 0

template <int P, int Tile>
struct Engine {
  static_assert((P == 1 && Tile == 256) || ((P == 1 || P == 3) && Tile == 128), "a plane at a time, or three");
  static constexpr int kTile = Tile, kPairs = P == 1 ? 1 : 6;
  static constexpr int kStep = Tile == 256 ? 64 : 32, kBuffers = Tile == 256 ? 2 : P == 1 ? 8 : 3;
  static constexpr int kWM = kTile / 2, kWN = kTile / 4, kI = kWM / 16, kJ = kWN / 16;
  static constexpr int kPlaneBytes = kTile * kStep * 2;  // an operand's plane of a step in LDS
  static constexpr int kLoads = kPlaneBytes / (kThreads * 16), kStepLoads = 2 * P * kLoads;  // loads of a lane: a plane's, a step's
  static constexpr int kBufferBytes = 2 * P * kPlaneBytes, kLdsBytes = kBuffers * kBufferBytes;
  typedef f32x4_t Acc[kI][kJ];

  __device__ __forceinline__ static int wave_m(int wave) { return (wave >> 2) * kWM; }
  __device__ __forceinline__ static int wave_n(int wave) { return (wave & 3) * kWN; }
  __device__ __forceinline__ static void clear(Acc& acc) {
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
      for (int j = 0; j < kJ; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // Brings a plane of a step into LDS: kLoads loads of 16 bytes a lane, `apart` bytes from each other.
  template <bool MMajor, bool Paired>
  struct Stager {
    int voff, apart;
    __device__ __forceinline__ void init(const Operand& o, int wave, int lane) {
      constexpr int C = MMajor ? kTile / 8 : kStep / 8;  // chunks to an LDS row
      const int idx = wave * kWave + lane, r = idx / C, c = (idx % C) ^ (MMajor ? swz_m(r) : swz_k<Paired, C>(r));
      voff = r * int(o.ld * 2) + c * 16;
      apart = kThreads / C * int(o.ld * 2);
    }
    __device__ __forceinline__ void stage(const uint16_t* p, uint32_t bytes, lds_byte* lds, int wave, int i) const {
      load_to_lds(p, bytes, uint32_t(reinterpret_cast<uintptr_t>(lds)) + (i * kWaves + wave) * kWave * 16, voff, i * apart);
    }
  };

  // Reads the wave's fragments of a staged plane; r0: its first row in the tile; h: the half (32 k) of the step.
  template <bool MMajor, bool Paired>
  struct Reader {
    static constexpr int kHalves = kStep / 32, kAt = MMajor ? 1 : Paired ? 2 * kHalves : kHalves;
    int at[kAt];
    __device__ __forceinline__ void init(int r0, int lane) {
      const int lo = lane & 15, g = lane >> 4;
      if constexpr (MMajor) {
        static_assert(!Paired, "only k-contiguous operands come in pairs of fragments");
        // lane s of a group of 16 reads 4 m at row k = 8 g + 4 q + s / 4; q and the half are added below
        const int k = 8 * g + lo / 4;
        at[0] = k * (kTile * 2) + ((r0 * 2) ^ (swz_m(k) * 16)) + 8 * (lo & 3);
      } else {
#pragma unroll
        for (int q = 0; q < kAt; ++q) {  // half of the step, and with pairs which of the two
          const int r = r0 + frag_row<Paired>(q / kHalves, lo);
          at[q] = r * (kStep * 2) + (((4 * (q % kHalves) + g) ^ swz_k<Paired, kStep / 8>(r)) * 16);
        }
      }
    }
    __device__ __forceinline__ bf16x8_t read(const lds_byte* lds, int h, int a) const {
      if constexpr (MMajor) {
        typedef __attribute__((address_space(3))) s16x4_t lds_s4;
        // fragment a's columns: 32 a bytes on, under the swizzle an exclusive or; formed here, as an address for each
        // held over the loop costs registers that the fragments need
        int b = at[0];
        asm("" : "+v"(b));
        b ^= 32 * a;
        const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(lds + b + h * 32 * kTile * 2));
        const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(lds + b + (h * 32 + 4) * kTile * 2));
        return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      } else {
        typedef __attribute__((address_space(3))) s16x8_t lds_s8;
        const int q = Paired ? (a & 1) * kHalves + h : h, rows = Paired ? (a >> 1) * 32 : a * 16;
        return __builtin_bit_cast(bf16x8_t, *(const lds_s8*)(lds + at[q] + rows * kStep * 2));
      }
    }
  };

  // acc += the products of steps q0 .. q1 of both operands.  start() requests the first kBuffers steps and may be called before
  // the results of the last tile are stored; run() waits for them, not for the stores.  While the products of a half (a
  // step of planes) run, the fragments of the next are read and a later step is requested, a load or two reads between every few
  // products, so that none holds the others up.
  // What bounds it on MI355X is power: the loop of a long bf16 sum keeps the matrix cores busy 64% of the time at 1.7 .. 1.9
  // GHz, and steps of 32 in a ring of four, loads in other places, or 4 waves of 128 x 128 gave more busy time at a lower
  // clock, or less (1.0 .. 1.2 PFLOP/s; without the loads into LDS it would be 1.5).
  template <bool AM, bool BM, bool Paired = false>
  struct Multiply {
    Stager<AM, Paired> sa;
    Stager<BM, false> sb;
    Reader<AM, Paired> ra;
    Reader<BM, false> rb;
    Operand A, B;
    const uint16_t *pa, *pb;  // the next step to request, kk
    uint32_t bytes_a, bytes_b;
    int64_t step_a, step_b;
    int n, kk;
    lds_byte* lds;
    int wave;

    __device__ __forceinline__ explicit Multiply(lds_byte* lds_) : lds(lds_) {
      wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
      const int lane = int(threadIdx.x) % kWave;
      ra.init(wave_m(wave), lane);
      rb.init(wave_n(wave), lane);
    }
    __device__ __forceinline__ static uint32_t range(int64_t elements) {
      return uint32_t(max(int64_t(0), min(elements * 2, int64_t(0xffffffff))));
    }
    __device__ __forceinline__ lds_byte* buffer(int b) const { return lds + b * kBufferBytes; }
    __device__ __forceinline__ void point() {
      const int64_t ka = kk * step_a, kb = kk * step_b;
      pa = A.base + ka;
      pb = B.base + kb;
      bytes_a = range(A.end - ka);
      bytes_b = range(B.end - kb);
    }
    // Load q of a step's; the last one moves on to the next step.
    __device__ __forceinline__ void stage(int buf, int q) {
      const int plane = q / kLoads % P, i = q % kLoads;
      lds_byte* l = buffer(buf) + q / kLoads * kPlaneBytes;
      if (q < P * kLoads)
        sa.stage(pa + plane * A.plane, bytes_a, l, wave, i);
      else
        sb.stage(pb + plane * B.plane, bytes_b, l, wave, i);
      if (q < kStepLoads - 1) return;
      ++kk;
      point();
    }
    __device__ __forceinline__ void start(const Operand& A_, const Operand& B_, int q0, int q1) {
      A = A_;
      B = B_;
      n = q1 - q0;
      kk = q0;
      step_a = AM ? kStep * A.ld : int64_t(kStep);
      step_b = BM ? kStep * B.ld : int64_t(kStep);
      point();
      const int lane = int(threadIdx.x) % kWave;
      sa.init(A, wave, lane);
      sb.init(B, wave, lane);
#pragma unroll
      for (int s = 0; s < kBuffers; ++s)
        if (s < n)
#pragma unroll
          for (int q = 0; q < kStepLoads; ++q) stage(s, q);
    }
    __device__ __forceinline__ static void product(f32x4_t& c, const bf16x8_t& a, const bf16x8_t& b) {
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }

    // Younger: accesses to global memory that every wave has at least made since start().
    template <int Younger>
    __device__ __forceinline__ void run(Acc& acc) {
      using S0 = std::integral_constant<int, 0>;
      using S1 = std::integral_constant<int, 1>;
      if (n >= kBuffers)
        wait_and_meet<(kBuffers - 1) * kStepLoads + Younger>();
      else
        wait_and_meet<0>();
      if constexpr (Tile == 256) {
        bf16x8_t fa[2][kI], fb[2][kJ];
        // two fragments of a half: B's, then A's
        auto read = [&](int buf, auto sc, int g) {
          constexpr int S = decltype(sc)::value;
          const lds_byte* l = buffer(buf);
#pragma unroll
          for (int f = 2 * g; f < 2 * g + 2; ++f) {
            if (f < kJ)
              fb[S][f] = rb.read(l + kPlaneBytes, S, f);
            else if (f < kI + kJ)
              fa[S][f - kJ] = ra.read(l, S, f - kJ);
          }
        };
        auto products = [&](auto sc, auto&& between) {
          constexpr int S = decltype(sc)::value;
#pragma unroll
          for (int i = 0; i < kI; ++i) {
            between(i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < kJ; ++j) product(acc[i][j], fa[S][i], fb[S][j]);
            __builtin_amdgcn_sched_barrier(0);
          }
        };
        static_assert(kI + kJ <= 2 * kI && kStepLoads == kI, "two reads and a load between each row of products");
#pragma unroll
        for (int g = 0; g < kI; ++g) read(0, S0{}, g);
        for (int s = 0; s < n; ++s) {
          products(S0{}, [&](int g) { read(s & 1, S1{}, g); });
          // step s + 1 is in LDS, and everyone has read step s
          if (Younger && s == 0)
            wait_and_meet<Younger>();
          else
            wait_and_meet<0>();
          const bool load = s + 2 < n;
          products(S1{}, [&](int g) {
            read((s + 1) & 1, S0{}, g);  // after the last step: what is left there, for nothing
            if (load) stage(s & 1, g);
          });
        }
      } else {
        bf16x8_t fa[2][P][kI], fb[2][P][kJ];
        constexpr int kFrags = P * (kI + kJ), kRows = kPairs * kI;
        constexpr int kReads = (kFrags + kRows - 1) / kRows, kEvery = kRows / kStepLoads;  // of each row, rows to a load
        auto read = [&](int buf, auto sc, int f) {
          constexpr int S = decltype(sc)::value;
          const lds_byte* l = buffer(buf);
          if (f < P * kJ)
            fb[S][f / kJ][f % kJ] = rb.read(l + (P + f / kJ) * kPlaneBytes, 0, f % kJ);
          else if (f < kFrags)
            fa[S][(f - P * kJ) / kI][(f - P * kJ) % kI] = ra.read(l + (f - P * kJ) / kI * kPlaneBytes, 0, (f - P * kJ) % kI);
        };
        auto step = [&](int s, int buf, auto sc) {
          constexpr int S = decltype(sc)::value;
          // step s + 1 is in LDS when all but the loads of the steps behind it (and what came after start()) are back; and
          // everyone has read step s
          constexpr int behind = (kBuffers - 2) * kStepLoads;
          if (s + kBuffers > n)
            wait_and_meet<0>();
          else if (Younger && s < kBuffers - 1)
            wait_and_meet<behind + Younger>();
          else
            wait_and_meet<behind>();
          const bool load = s + kBuffers < n;
          const int next = buf == kBuffers - 1 ? 0 : buf + 1;
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
#pragma unroll
            for (int f = 0; f < kReads; ++f) read(next, std::integral_constant<int, S ^ 1>{}, kReads * r + f);
            if (load && r % kEvery == kEvery - 1) stage(buf, r / kEvery);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < kJ; ++j) product(acc[r % kI][j], fa[S][pair_a<P>(r / kI)][r % kI], fb[S][pair_b<P>(r / kI)][j]);
            __builtin_amdgcn_sched_barrier(0);
          }
          return next;
        };
        static_assert(kRows % kStepLoads == 0, "the loads spread evenly among the products");
#pragma unroll
        for (int f = 0; f < kFrags; ++f) read(0, S0{}, f);
        int buf = 0;
        for (int s = 0; s < n; s += 2) {
          buf = step(s, buf, S0{});
          if (s + 1 < n) buf = step(s + 1, buf, S1{});
        }
      }
    }
  };
};

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
