// A stable sort of tokens by id, for sums over each id's tokens in a fixed order.
//
// Workgroup b of 2^shift owns the ids with id % 2^shift = b (so the frequent ids, which lie next to each other in a vocabulary sorted by
// frequency, fall to different workgroups) and reads all ids itself: they are small (128 KB at 16384 tokens) and come from L2.  It
// counts its ids per wave and those of the workgroups before it, which gives its place in the order without a word to the others,
// then places its tokens; a wave walks its part of the tokens in order, so the sort is stable.  MI355X: 10 us for 16384 tokens of
// 32000 ids, a chain of waits (ids from L2, LDS counts, places).
//
// A workgroup owns at most 256 ids, so with many ids and many tokens the reading is what takes the time, tokens x ids / 256.  From
// kMostReads on it is done in two levels: 256 workgroups sort the tokens into buckets, the residues that single workgroups would own
// above, at most 2^16, and in a second launch a workgroup for each 256 ids of a bucket sorts that bucket's tokens alone.
#pragma once

#include <algorithm>

#include "common.hpp"

namespace cdssm {
namespace token_sort {

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave, kMaxLocal = 256;

__device__ __forceinline__ int valid_id(int64_t id, int64_t V, int64_t padding) {
  return id >= 0 && id < V && id != padding ? int(id) : -1;  // V <= 2^28
}

// A workgroup's part of a sort of n items: load(i) the key of item i, or -1 where it is left out; place(key, lower) which of the
// workgroup's kMaxLocal it is or -1, and whether it belongs to a workgroup before; token(i) what the order says of it.  The order's
// places start at `begin`; put(l, first, count) is told of each of the workgroup's keys.
template <typename Load, typename Place, typename Token, typename Put>
__device__ __forceinline__ void sort_part(int n, int begin, int* __restrict__ order, Load&& load, Place&& place, Token&& token,
                                          Put&& put) {
  __shared__ int cnt[kSortWaves][kMaxLocal];
  __shared__ int tot[kMaxLocal / kWave];
  __shared__ int lower[kSortWaves];
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  const int per = ((n + kSortWaves - 1) / kSortWaves + kWave - 1) / kWave * kWave, t0 = wave * per;
  const int t1 = min(n, t0 + per);
  for (int i = tid; i < kSortWaves * kMaxLocal; i += kSortThreads) (&cnt[0][0])[i] = 0;
  __syncthreads();
  int low = 0;
  constexpr int U = 16;  // 16 x 64 items under way; up to 16384 items they are all that a wave has, and stay for the second pass
  int own[U];            // which of the workgroup's keys an item has, or -1
  auto fetch = [&](int s) {
#pragma unroll
    for (int u = 0; u < U; ++u) own[u] = load(min(s + u * kWave + lane, n - 1));  // no branch, so that all are under way at once
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = s + u * kWave + lane < t1 ? own[u] : -1;
      bool before = false;
      const int l = place(key, before);
      own[u] = key >= 0 ? l : -1;
      low += key >= 0 && before;
    }
  };
  for (int s = t0; s < t1; s += U * kWave) {
    fetch(s);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (own[u] >= 0) atomicAdd(&cnt[wave][own[u]], 1);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) low += __shfl_xor(low, o, kWave);
  if (lane == 0) lower[wave] = low;
  __syncthreads();
  // exclusive sums over (key, wave): thread l has key l
  int count = 0, before = 0;
  if (tid < kMaxLocal) {
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) count += cnt[w][tid];
    int sum = count;
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) {
      const int v = __shfl_up(sum, o, kWave);
      if (lane >= o) sum += v;
    }
    if (lane == kWave - 1) tot[wave] = sum;
    before = sum - count;
  }
  __syncthreads();
  if (tid < kMaxLocal) {
    before += begin;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) before += lower[w];
#pragma unroll
    for (int w = 0; w < kMaxLocal / kWave; ++w) before += w < wave ? tot[w] : 0;
    put(tid, before, count);
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = cnt[w][tid];
      cnt[w][tid] = before;
      before += c;
    }
  }
  __syncthreads();
  for (int s = t0; s < t1; s += U * kWave) {
    if (t1 - t0 > U * kWave) fetch(s);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int l = own[u];
      const bool mine = l >= 0;
      uint64_t left = __ballot(mine);
      while (left) {  // one key of the 64 items at a time
        const int lead = __builtin_ctzll(left), ll = __builtin_amdgcn_readlane(l, lead);
        const uint64_t same = __ballot(l == ll);
        int at = 0;
        if (lane == lead) at = atomicAdd(&cnt[wave][ll], __popcll(same));  // the wave's own counter
        at = __builtin_amdgcn_readlane(at, lead);
        if (l == ll) order[at + __popcll(same & ((uint64_t(1) << lane) - 1))] = token(s + u * kWave + lane);
        left &= ~same;
      }
    }
  }
}

// order (T): the tokens by id % 2^shift, id, place; rows (V): where an id's tokens start in it, and how many they are.
template <typename I>
__device__ __forceinline__ void sort(const I* __restrict__ ids, int* __restrict__ order, int2* __restrict__ rows, int T, int64_t V,
                                     int64_t padding, int shift) {
  const int mask = (1 << shift) - 1, b = blockIdx.x;
  sort_part(
      T, 0, order, [&](int t) { return valid_id(int64_t(ids[unsigned(t)]), V, padding); },
      [&](int id, bool& before) {
        before = (id & mask) < b;
        return (id & mask) == b ? id >> shift : -1;
      },
      [](int t) { return t; },
      [&](int l, int first, int count) {
        const int64_t v = (int64_t(l) << shift) + b;
        if (v < V) rows[v] = make_int2(first, count);
      });
}

// The first of two levels, workgroup b of 256: by id % 2^bits, 8 <= bits <= 16, with the buckets' starts and counts.
template <typename I>
__device__ __forceinline__ void sort_buckets(const I* __restrict__ ids, int* __restrict__ order, int2* __restrict__ buckets, int T,
                                             int64_t V, int64_t padding, int bits) {
  const int mask = (1 << bits) - 1, b = blockIdx.x;
  sort_part(
      T, 0, order, [&](int t) { return valid_id(int64_t(ids[unsigned(t)]), V, padding); },
      [&](int id, bool& before) {
        before = (id & 255) < b;
        return (id & 255) == b ? (id & mask) >> 8 : -1;
      },
      [](int t) { return t; },
      [&](int l, int first, int count) {
        if (l < 1 << (bits - 8)) buckets[(l << 8) + b] = make_int2(first, count);
      });
}

// The second, workgroup bucket + sub 2^bits: the bucket's ids from number 256 sub on, among the bucket's tokens as the first level left them.
template <typename I>
__device__ __forceinline__ void sort_bucket(const I* __restrict__ ids, const int* __restrict__ tokens,
                                            const int2* __restrict__ buckets, int* __restrict__ order, int2* __restrict__ rows,
                                            int64_t V, int bits) {
  const int bucket = int(blockIdx.x & ((1u << bits) - 1)), sub = int(blockIdx.x >> bits);
  const int2 at = buckets[bucket];
  tokens += at.x;
  sort_part(
      at.y, at.x, order, [&](int i) { return int(ids[unsigned(tokens[unsigned(i)])]) >> bits; },
      [&](int l, bool& before) {
        before = l / kMaxLocal < sub;
        return l / kMaxLocal == sub ? l % kMaxLocal : -1;
      },
      [&](int i) { return tokens[unsigned(i)]; },
      [&](int l, int first, int count) {
        const int64_t v = ((int64_t(sub) * kMaxLocal + l) << bits) + bucket;
        if (v < V) rows[v] = make_int2(first, count);
      });
}

inline int id_shift(int64_t V) {  // log2 of the sort's workgroups: at most kMaxLocal ids each
  int s = 0;
  while (s < 8 && (int64_t(1) << s) < V) ++s;
  while ((V + (int64_t(1) << s) - 1) >> s > kMaxLocal) ++s;
  return s;
}

// Reads of ids by a single level from which on two levels are taken (and there have to be more than 256 workgroups).  The table's
// gradient with a sort in one and in two, us, rows of 8: 16384 tokens of 100000 ids (2^23 reads) 34 and 47, 131072 of 100000 (2^26)
// 116 and 114, 16384 of 2^20 (2^26) 180 and 200, 131072 of 2^18 (2^27) 192 and 138, 131072 of 2^20 (2^29) 671 and 270, 2^20 of 2^20 (2^32)
// 4820 and 790.
constexpr int64_t kMostReads = int64_t(1) << 26;
inline bool two_levels(int64_t T, int64_t V) { return id_shift(V) > 8 && (T << id_shift(V)) > kMostReads; }
inline int bucket_bits(int64_t V) { return std::min(16, id_shift(V)); }
inline int64_t bucket_groups(int64_t V) {
  const int bits = bucket_bits(V);
  const int64_t ids = (V + (int64_t(1) << bits) - 1) >> bits;
  return ((ids + kMaxLocal - 1) / kMaxLocal) << bits;
}

}  // namespace token_sort
}  // namespace cdssm
