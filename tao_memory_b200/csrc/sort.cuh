// A stable sort of a few thousand to some millions of small whole numbers by counting: tokens by expert in one
// pass, tokens by word in two or three passes of up to nine bits.
//
// A pass counts, for each block's run of elements, how many fall into each bin (count_kernel), and then places
// each element (place_kernel): a bin begins behind all smaller bins, a block's elements behind those of the
// blocks before, a warp's behind those of the warps before, and of 32 elements at a time each finds those before
// it in its bin by a match across the warp.  Only whole numbers are added atomically: the order is fixed.
// Up to kSmallSort elements one block does it in one launch.  What bounds it is latency: launches, and each
// warp's chain of rounds.  131072 pairs by 64 experts take 13 us, 32768 words of 17 bits in two passes 28 us, 512
// pairs 4 us; with 2048 elements a block the passes took 31 us, with 512 (and as many more counts to add) 34.
#pragma once
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace tao {
namespace sorting {

constexpr int kMostBins = 513;  // 512 and one for what belongs to none
constexpr int kSmallSort = 4096;  // one block and launch 8.4 us, two launches 7.6 and the host's second; 8192: 13.5, 7.6
constexpr int kMostBlocks = 128;

// A pass over n elements.  The key of element i is ids[value], value = values[i] or (values null) i: the whole id
// for `shift` < 0, else `bits` bits of it from `shift` on.  Ids outside of 0 .. limit - 1 count as `limit`.
struct Pass {
  const void* ids;
  const int* values;
  long long limit;
  int n, shift, bins, per;  // per: elements of a warp
  bool wide;                // ids have 64 bits
  const int* counts;        // [blocks][bins], of all blocks; null: this block is the only one
  int blocks;
  int* sorted;              // values in order
  int* places;              // where element i went, or null
  int* keys;                // whole ids in order, or null
  int* offsets;             // the first place of each bin, or null
  uint8_t* zero;            // what the blocks behind the sort's own fill with zeros meanwhile: on 2 bytes
  long long zero_bytes;
};

// Zeros of a range by blocks behind the sort's, by 16 bytes and what is left at its ends by two.
TAO_DEVI void clear(const Pass& p) {
  const int block = blockIdx.x - p.blocks, blocks = gridDim.x - p.blocks;
  uint8_t* const end = p.zero + p.zero_bytes;
  uint4* const from = reinterpret_cast<uint4*>((reinterpret_cast<uintptr_t>(p.zero) + 15) / 16 * 16);
  uint4* const to = reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(end) / 16 * 16);
  for (uint4* at = from + (long long)block * blockDim.x + threadIdx.x; at < to; at += (long long)blocks * blockDim.x)
    *at = make_uint4(0, 0, 0, 0);
  if (block > 0 || threadIdx.x >= 8) return;
  uint8_t* const head = p.zero + 2 * threadIdx.x;
  if (head < end && head < reinterpret_cast<uint8_t*>(from)) *reinterpret_cast<uint16_t*>(head) = 0;
  uint8_t* const tail = reinterpret_cast<uint8_t*>(to) + 2 * threadIdx.x;
  if (tail >= p.zero && tail < end) *reinterpret_cast<uint16_t*>(tail) = 0;
}

TAO_DEVI int id_of(const Pass& p, int value) {
  const long long id = p.wide ? static_cast<const long long*>(p.ids)[value] : static_cast<const int*>(p.ids)[value];
  return (int)(id < 0 || id >= p.limit ? p.limit : id);
}
TAO_DEVI int bin_of(const Pass& p, int id) { return p.shift < 0 ? id : id >> p.shift & (p.bins - 1); }

constexpr int kAhead = 4;  // rounds whose ids are on their way
// The value of element i, -1 behind the last.
TAO_DEVI int value_at(const Pass& p, long long i, int end) { return i >= end ? -1 : p.values ? p.values[i] : (int)i; }

// counts[warp][bin] of this block's warps, in shared memory.
TAO_DEVI void count_warps(const Pass& p, int* counts, int warps) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < warps * p.bins; i += blockDim.x) counts[i] = 0;
  __syncthreads();
  const long long begin = ((long long)blockIdx.x * warps + warp) * p.per;
  const int end = (int)min(begin + p.per, (long long)p.n);
  int* const mine = counts + warp * p.bins;
  for (long long i0 = begin + lane; i0 < end; i0 += 32 * kAhead) {
    int value[kAhead], id[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) value[j] = value_at(p, i0 + 32 * j, end);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) id[j] = value[j] < 0 ? 0 : id_of(p, value[j]);
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (value[j] >= 0) atomicAdd(mine + bin_of(p, id[j]), 1);
  }
  __syncthreads();
}

template <int WARPS>
__global__ void __launch_bounds__(32 * WARPS) count_kernel(const Pass p, int* out) {
  extern __shared__ int counts[];
  if (blockIdx.x >= p.blocks) return clear(p);
  count_warps(p, counts, WARPS);
  for (int b = threadIdx.x; b < p.bins; b += 32 * WARPS) {
    int s = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) s += counts[w * p.bins + b];
    out[(long long)blockIdx.x * p.bins + b] = s;
  }
}

template <int WARPS>
__global__ void __launch_bounds__(32 * WARPS) place_kernel(const Pass p) {
  extern __shared__ int counts[];
  __shared__ int first[kMostBins], before[kMostBins];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (blockIdx.x >= p.blocks) return clear(p);
  count_warps(p, counts, WARPS);
  for (int b = threadIdx.x; b < p.bins; b += 32 * WARPS) {
    int all = 0;
    if (!p.counts) {
#pragma unroll
      for (int w = 0; w < WARPS; ++w) all += counts[w * p.bins + b];
    }
    first[b] = all;
    before[b] = 0;
  }
  __syncthreads();
  if (p.counts) {  // threads that are not needed for the bins share out the blocks
    const int across = min((p.bins + 31) / 32 * 32, 32 * WARPS), parts = 32 * WARPS / across, part = threadIdx.x / across;
    if (part < parts) {
      for (int b = threadIdx.x - part * across; b < p.bins; b += across) {
        int all = 0, earlier = 0;
#pragma unroll 8
        for (int k = part; k < p.blocks; k += parts) {
          const int c = p.counts[(long long)k * p.bins + b];
          all += c;
          earlier += k < (int)blockIdx.x ? c : 0;
        }
        atomicAdd(first + b, all);
        atomicAdd(before + b, earlier);
      }
    }
  }
  __syncthreads();
  if (warp == 0) {  // the bins' sizes to their first places
    int sum = 0;
    for (int base = 0; base < p.bins; base += 32) {
      const int b = base + lane, mine = b < p.bins ? first[b] : 0;
      int s = mine;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
      }
      if (b < p.bins) first[b] = sum + s - mine;
      sum += __shfl_sync(0xffffffffu, s, 31);
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < p.bins; b += 32 * WARPS) {
    if (p.offsets && blockIdx.x == 0) p.offsets[b] = first[b];
    int at = first[b] + before[b];
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const int c = counts[w * p.bins + b];
      counts[w * p.bins + b] = at;
      at += c;
    }
  }
  __syncthreads();
  const long long begin = ((long long)blockIdx.x * WARPS + warp) * p.per;
  const int end = (int)min(begin + p.per, (long long)p.n);
  int* const mine = counts + warp * p.bins;
  for (long long base = begin; base < end; base += 32 * kAhead) {
    int value[kAhead], id[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) value[j] = value_at(p, base + 32 * j + lane, end);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) id[j] = value[j] < 0 ? 0 : id_of(p, value[j]);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const bool in = value[j] >= 0;
      const int bin = in ? bin_of(p, id[j]) : -1;
      const uint32_t same = __match_any_sync(0xffffffffu, bin);
      const int rank = __popc(same & ((1u << lane) - 1));
      const int at = in ? mine[bin] + rank : 0;
      __syncwarp();
      if (in && rank == 0) mine[bin] += __popc(same);
      __syncwarp();
      if (in) {
        p.sorted[at] = value[j];
        if (p.places) p.places[base + 32 * j + lane] = at;
        if (p.keys) p.keys[at] = id[j];
      }
    }
  }
}

inline int blocks_of(long long n) { return n <= kSmallSort ? 1 : (int)std::min<long long>((n + 1023) / 1024, kMostBlocks); }
inline size_t counts_bytes(long long n, int bins) { return n <= kSmallSort ? 0 : (size_t)blocks_of(n) * bins * sizeof(int); }

inline int launches_of(long long n) { return blocks_of(n) == 1 ? 1 : 2; }

// Bytes that become zeros while a sort runs, a share of them in each of its launches.
struct Clearing {
  uint8_t* at;
  long long bytes;
  int launches;  // of the sort, that are left
  // The next launch's share, and the blocks of `threads` for it.
  int next(Pass& p, int threads) {
    if (!launches) return 0;
    const long long share = launches == 1 ? bytes : bytes / launches / 16 * 16;
    p.zero = at, p.zero_bytes = share;
    at += share, bytes -= share, --launches;
    return (int)std::min<long long>((share + threads * 16 - 1) / (threads * 16), 148ll * 1024 / threads);
  }
};

// `counts`: counts_bytes of scratch.
inline cudaError_t run(Pass p, int* counts, cudaStream_t s, Clearing* zeros = nullptr) {
  Clearing none = {};
  if (!zeros) zeros = &none;
  p.blocks = blocks_of(p.n);
  if (p.blocks == 1) {
    p.counts = nullptr;
    p.per = (p.n + 1023) / 1024 * 32;
    static_assert(32 * kMostBins * sizeof(int) <= 96 * 1024, "");
    static std::atomic<uint64_t> ready{0};  // of the first 64 devices
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    const uint64_t mark = device < 64 ? 1ull << device : 0;
    if (e == cudaSuccess && !(ready.load(std::memory_order_relaxed) & mark)) {
      e = cudaFuncSetAttribute(place_kernel<32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               32 * kMostBins * (int)sizeof(int));
      if (e == cudaSuccess) ready |= mark;
    }
    if (e != cudaSuccess) return e;
    const int more = zeros->next(p, 1024);
    place_kernel<32><<<1 + more, 1024, 32 * p.bins * sizeof(int), s>>>(p);
    return cudaGetLastError();
  }
  const int warps = p.blocks * 8;
  p.per = (int)(((long long)p.n + warps - 1) / warps + 31) / 32 * 32;
  p.counts = counts;
  const int counting = zeros->next(p, 256);
  count_kernel<8><<<p.blocks + counting, 256, 8 * p.bins * sizeof(int), s>>>(p, counts);
  const int placing = zeros->next(p, 256);
  place_kernel<8><<<p.blocks + placing, 256, 8 * p.bins * sizeof(int), s>>>(p);
  return cudaGetLastError();
}

}  // namespace sorting
}  // namespace tao
