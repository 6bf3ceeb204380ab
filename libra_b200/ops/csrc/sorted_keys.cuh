// Stable counting sort of small integer keys, one pass at a time, by one cluster of CTAs.
//
// The items are dealt to the cluster's warps in consecutive runs.  A pass counts each warp's keys, sums the counts
// (warps before this one in the CTA, CTAs before this one in the cluster, bins before this one), and walks the same
// items again: an item's place is its bin's start, plus the items of its key in earlier runs, plus those before it in
// its own.  Places depend on the keys alone, never on the order in which warps run, so whatever sums follow the sorted
// order are the same every time.  One cluster and its barrier take the place of three launches (count, scan, place).
#pragma once
#include "vocab_rows.cuh"

namespace libra {
namespace sorted {

constexpr int kMaxBins = 1024, kMaxCtas = 16;

// Bins up to which a warp's lanes find their equals through words in shared memory: each sets its bit in its bin's word.
// (131072 pairs by 128 experts: 11.4 us; with __match_any_sync, which takes a step for every distinct key, 15.9.)
constexpr int kWordBins = 512;

inline size_t pass_smem(int warps, int bins) {
  return ((size_t)warps * bins * (bins <= kWordBins ? 2 : 1) + bins + 64) * 4;
}

__device__ __forceinline__ uint32_t ld_cluster_u32(const uint32_t* p, uint32_t rank) {
  return (uint32_t)vocab::ld_cluster(reinterpret_cast<const int*>(p), rank);
}

// Exclusive sum over the block's threads.
template <int kWarps>
__device__ __forceinline__ uint32_t block_before(uint32_t v, uint32_t* tmp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t s = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, s, off);
    if (lane >= off) s += o;
  }
  if (lane == 31) tmp[warp] = s;
  __syncthreads();
  uint32_t t = lane < kWarps ? tmp[lane] : 0;
#pragma unroll
  for (int off = 1; off < kWarps; off <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, t, off);
    if (lane >= off) t += o;
  }
  t = __shfl_sync(0xffffffffu, t, warp ? warp - 1 : 0);
  return s - v + (warp ? t : 0);
}

// Up to this many items a lane stay in registers between the two walks.
constexpr int kBatch = 8;

// One pass.  Items has
//   Item load(int i)            item i
//   int bin(const Item&)        its bin, or -1 for an item that gets no place
//   void put(int i, Item, uint32_t place)   (place 0xffffffff for none)
//   void group(int bin, uint32_t start, uint32_t count)   once for each bin; starts are multiples of `align`
// Every CTA of the cluster (of `ctas`, at most 16) calls it with all its kWarps warps; sm: pass_smem(kWarps, bins) bytes.
// What put writes to global memory is visible to the whole cluster afterwards.
template <int kWarps, class Items>
__device__ __forceinline__ void counting_pass(int n, int bins, uint32_t align, uint32_t* sm, int ctas, Items& items) {
  constexpr int kThreads = kWarps * 32, kMine = kMaxBins / kThreads;  // bins a thread
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = ctas > 1 ? (int)cluster_ctarank() : 0;
  uint32_t* total = sm + kWarps * bins;
  uint32_t* tmp = total + bins;
  uint32_t* mine = sm + warp * bins;
  const bool by_word = bins <= kWordBins;
  uint32_t* word = tmp + 64 + warp * bins;
  const int64_t per = (((int64_t)n + ctas * kWarps - 1) / (ctas * kWarps) + 31) / 32 * 32;
  const int64_t lo = (rank * kWarps + warp) * per;
  const int64_t hi = lo + per < n ? lo + per : n;
  typename Items::Item it[kBatch];
  auto fetch = [&](int64_t i0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int64_t i = i0 + 32 * u + lane;
      if (i < hi) it[u] = items.load((int)i);
    }
  };

  fetch(lo);
  for (int i = lane; i < bins; i += 32) {
    mine[i] = 0;
    if (by_word) word[i] = 0;
  }
  __syncwarp();
  for (int64_t i0 = lo; i0 < hi; i0 += 32 * kBatch) {
    if (i0 > lo) fetch(i0);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int key = i0 + 32 * u + lane < hi ? items.bin(it[u]) : -1;
      if (key >= 0) atomicAdd(mine + key, 1u);
    }
  }
  __syncthreads();

  // this thread's bins: m neighbours from b0
  const int m = (bins + kThreads - 1) / kThreads, b0 = threadIdx.x * m;
  uint32_t all[kMine], below[kMine], room = 0;
#pragma unroll
  for (int q = 0; q < kMine; ++q) {
    all[q] = below[q] = 0;
    if (q >= m || b0 + q >= bins) continue;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) all[q] += sm[w * bins + b0 + q];
    total[b0 + q] = all[q];
  }
  if (ctas > 1) {
    vocab::cluster_meet();
#pragma unroll
    for (int q = 0; q < kMine; ++q) {
      if (q >= m || b0 + q >= bins) continue;
      uint32_t v[kMaxCtas];
#pragma unroll
      for (int c = 0; c < kMaxCtas; ++c) v[c] = c < ctas ? ld_cluster_u32(total + b0 + q, c) : 0u;
      all[q] = 0;
#pragma unroll
      for (int c = 0; c < kMaxCtas; ++c) {
        all[q] += v[c];
        below[q] += c < rank ? v[c] : 0u;
      }
    }
  } else {
    __syncthreads();
  }
#pragma unroll
  for (int q = 0; q < kMine; ++q) room += (all[q] + align - 1) / align * align;
  uint32_t start = block_before<kWarps>(room, tmp);
#pragma unroll
  for (int q = 0; q < kMine; ++q) {
    if (q >= m || b0 + q >= bins) continue;
    if (rank == 0) items.group(b0 + q, start, all[q]);
    uint32_t at = start + below[q];
    start += (all[q] + align - 1) / align * align;
#pragma unroll 8
    for (int w = 0; w < kWarps; ++w) {
      const uint32_t c = sm[w * bins + b0 + q];
      sm[w * bins + b0 + q] = at;
      at += c;
    }
  }
  __syncthreads();

  const bool kept = per <= 32 * kBatch;
  for (int64_t i0 = lo; i0 < hi; i0 += 32 * kBatch) {
    if (!kept) fetch(i0);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (i0 + 32 * u >= hi) break;
      const int64_t i = i0 + 32 * u + lane;
      const int key = i < hi ? items.bin(it[u]) : -1;
      uint32_t peers = 0, at = 0xffffffffu;
      if (by_word) {
        if (key >= 0) atomicOr(word + key, 1u << lane);
        __syncwarp();
        if (key >= 0) peers = word[key];
      } else {
        peers = __match_any_sync(0xffffffffu, key);
      }
      const int before = __popc(peers & ((1u << lane) - 1));
      if (key >= 0) at = mine[key] + before;
      __syncwarp();
      if (key >= 0 && before == 0) {
        mine[key] += __popc(peers);
        if (by_word) word[key] = 0;
      }
      __syncwarp();
      if (i < hi) items.put((int)i, it[u], at);
    }
  }
  // the totals outlive their readers, and the next pass reads what this one wrote
  if (ctas > 1)
    vocab::cluster_meet();
  else
    __syncthreads();
}

}  // namespace sorted
}  // namespace libra
