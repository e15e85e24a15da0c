// y = x W^T + b for a few rows of x and a 4-bit W with group scales.
//
//   W[n][k] = (code[n][k] - zero[n][k / group]) scale[n][k / group],  codes 0..15
//
// x in bf16 or fp16, or in e4m3 with one fp32 scale a row; y in the type of the weight's scales.
// How the product is formed: few_rows.cuh for up to 16 rows, which this file is about; linear4_tc.cuh for
// more.  Sums are in fp32, y is rounded once.
//
// Bound by the codes' bytes, half a byte a weight.  One block an SM.  x, or a cluster's block's part of its
// k, is laid out in shared memory once, in the order of the mma's operands.  The warps are WT x WK: WT row
// tiles at a time, each one's 128-k blocks dealt to WK warps in runs, each warp's through a ring of its own
// (registers would do, but a warp's few scoreboards make a load wait for later ones).  A warp leaves its sums
// of a tile in shared memory; these are added at the end, a cluster's blocks' through distributed shared
// memory, in a fixed order.
// With k = n = 8192 and groups of 128 one row takes 10.4 us (3.3 TB/s of its bytes), 8 rows 14.2, 16 rows 16.3: half of
// the issue slots, the rest waits at the few meetings.  A single row of k = 2048, n = 6144 takes 4.4 us, of which
// the bytes are 1: launch, x and the first weights follow one another.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "../../include/tao_b200.h"
#include "linear4_tc.cuh"

void tao_set_last_error(const char* msg);

namespace tao {
namespace {

constexpr int kSmem = 226 * 1024;
constexpr int kMaxK = 65536;  // two rows' pieces of a cluster of 8's part fit beside the rings

// The two forms of the product: signed bytes (4 columns a row), or the 16-bit type M (one).
struct Bytes {};

// COLS: columns of the mma for a row; WARPS: of a block; DEPTH: blocks of a warp's ring.  Shared memory of a
// block's 128 k of x: bytes have a row's four pieces as [half][4 row + piece][t] 16 bytes, a lane's
// operands in the order of the lanes, then [row] s / 2^7, then [group][row] the sums (P, Q); 16 bits have
// [32-k part][row][t] 16 bytes.
template <class M, int GROUP, int NT>
struct Form {
  static constexpr bool BYTES = std::is_same<M, Bytes>::value;
  static constexpr int COLS = BYTES ? 4 : 1, ROWS = 8 * NT / COLS, GROUPS = 128 / GROUP;
  static constexpr int WARPS = 16, DEPTH = 6;
  static constexpr int UNITS = ROWS * 512, SUMS = UNITS + ROWS * 4 + ROWS * 4 % 8;
  static constexpr int XBLOCK = BYTES ? (SUMS + GROUPS * ROWS * 8 + 15) / 16 * 16 : ROWS * 256;
};

// Outputs n..n + 3 (n a multiple of 4) of row m term by term, for rows of x that signed bytes cannot hold.  Rare
// (an infinity, a NaN, 128 channels that are all below 2^-100 and not all zero) and slow: a row of k = n = 8192
// takes 0.65 ms.
template <bool BF16, int GROUP>
TAO_DEVI float4 by_terms(const Linear4Args& a, long long m, int n) {
  constexpr int GROUPS = 128 / GROUP;
  float s[4] = {};
#pragma unroll 1
  for (int c = 0; c < a.kblocks * 16; ++c) {  // chunks of 8 k
    const long long block = (long long)(n / 16) * a.kblocks + c / 16;
    const int l = c % 16, group = l / (GROUP / 8);
    uint4 v = chunk_of(a, m, c * 8);
    if (a.x_type == TAO_TYPE_E4M3) v = widen_e4m3(v);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int g = n % 8 + e, high = n / 8 % 2;  // rows g and g + 8 of the tile share their bytes
      const uint2 codes = __ldg(reinterpret_cast<const uint2*>(a.w.codes + block * 1024 + (l / 8) * 512 +
                                                               (4 * g + l % 4) * 16 + l / 4 % 2 * 8));
      const long long at = (block * 8 + g) * (GROUPS * 2) + group * 2 + high;
      const uint16_t bits = __ldg(reinterpret_cast<const uint16_t*>(a.w.scales) + at);
      const float scale = BF16 ? __uint_as_float((uint32_t)bits << 16) : __half2float(__ushort_as_half(bits));
      const int zero = a.w.zeros ? __ldg(a.w.zeros + at) : 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 h = a.x_type == TAO_TYPE_BF16 ? make_float2(lo_f(w[i / 2]), hi_f(w[i / 2]))
                                                   : __half22float2(*reinterpret_cast<const __half2*>(&w[i / 2]));
        // byte b of word f is k 4f + (0, 2, 1, 3)[b]
        const uint32_t byte = (i < 4 ? codes.x : codes.y) >> (8 * (i % 4 * 2 % 3 + i % 4 / 3 * 3));
        s[e] += (float)((int)(byte >> (4 * high) & 15u) - zero) * scale * (i % 2 ? h.y : h.x);
      }
    }
  }
  return make_float4(s[0], s[1], s[2], s[3]);
}

// M: the form.  BF16: the type of scales, bias and y.  NT: column tiles of 8 columns of the mma.
template <class M, bool BF16, int GROUP, int NT>
__global__ void __launch_bounds__(32 * Form<M, GROUP, NT>::WARPS, 1) linear4_kernel(const Linear4Args a) {
  using F = Form<M, GROUP, NT>;
  using B4 = Block4<GROUP>;
  constexpr bool BYTES = F::BYTES;
  constexpr int ROWS = F::ROWS;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), warps = blockDim.x / 32;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int m0 = blockIdx.y * ROWS, rows = min(a.rows - m0, ROWS);
  const int rank = a.shift ? (int)cluster_rank() : 0;
  const int id = blockIdx.x >> a.shift, clusters = gridDim.x >> a.shift;
  const int k0 = a.kblocks * rank >> a.shift, nb = (a.kblocks * (rank + 1) >> a.shift) - k0;
  // a warp's row tiles are first, first + stride, ...; of each the `per` blocks from k0 + kw on
  const int wks = a.wk_shift, groups = warps >> wks, stride = clusters * groups;
  const int wt = warp >> wks, wk = warp & ((1 << wks) - 1), first = id * groups + wt;
  const int kw = nb * wk >> wks, per = (nb * (wk + 1) >> wks) - kw;

  // x before the weights, whose many copies in flight the others' come behind
  const int l = lane & 15;
  const bool copied = !BYTES && a.wide && a.x_type != TAO_TYPE_E4M3;
  if (copied) {
    const uint16_t* x = static_cast<const uint16_t*>(a.x) + m0 * a.x_stride;
    for (int m = warp; m < rows; m += warps)
      for (int c = lane; c < nb * 16; c += 32) {
        const int k = k0 * 128 + c * 8;
        const uint32_t to = smem_u32(smem) + (c >> 4) * F::XBLOCK + (((c >> 2 & 3) * ROWS + m) * 4 + (c & 3)) * 16;
        cp_async16(to, k < a.k ? x + m * a.x_stride + k : x, k < a.k);
      }
  }

  const int mine = first < a.tiles ? min(a.steps, (a.tiles - first + stride - 1) / stride) : 0, total = mine * per;
  const uint8_t* const ring = smem + a.ring + warp * (F::DEPTH * B4::BYTES);
  const uint32_t ring_at = smem_u32(ring);
  uint32_t next = first * a.kblocks + k0 + kw;  // block to copy
  int left = total, lk = per, to_slot = 0;
  auto issue = [&]() {
    if (left > 0) {
      --left;
      B4::issue(ring_at + to_slot, a.w, next++, lane);
      if (--lk == 0) {
        lk = per;
        next += stride * a.kblocks - per;
      }
      to_slot = to_slot == (F::DEPTH - 1) * B4::BYTES ? 0 : to_slot + B4::BYTES;
    }
    cp_commit();
  };
  const int items = copied ? 0 : rows * nb, each = warps * 2;  // 16 lanes: a row's 128 k
  auto chunk = [&](int i) {
    const int kb = rows == 1 ? i : i / rows;
    return i < items ? chunk_of(a, m0 + i - kb * rows, (k0 + kb) * 128 + l * 8) : make_uint4(0, 0, 0, 0);
  };
  const int item0 = warp * 2 + (lane >> 4);
  uint4 ahead = chunk(item0);
  cp_commit();  // x's copies
#pragma unroll 1
  for (int d = 0; d < F::DEPTH - 1; ++d) issue();
  if (copied) {
    cp_wait<F::DEPTH - 1>();
  } else {
    for (int i = item0; i - (lane >> 4) < items; i += each) {
      const int kb = rows == 1 ? i : i / rows, m = i - kb * rows;
      const bool in = i < items;
      uint4 v = ahead;
      ahead = chunk(i + each);
      uint8_t* to = smem + kb * F::XBLOCK;
      if (a.x_type == TAO_TYPE_E4M3) v = widen_e4m3(v);
      if constexpr (BYTES) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        float f[8], most = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
          f[2 * e] = a.x_type == TAO_TYPE_BF16 ? lo_f(w[e]) : h.x;
          f[2 * e + 1] = a.x_type == TAO_TYPE_BF16 ? hi_f(w[e]) : h.y;
          most = max_nan(most, max_nan(fabsf(f[2 * e]), fabsf(f[2 * e + 1])));
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
        float up, unit;
        units_of(most, up, unit);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= up;
        uint2 p[4];
        int2 sum;
        split8(f, p, sum.x, sum.y);
#pragma unroll
        for (int o = 1; o < GROUP / 8; o <<= 1) {
          sum.x += __shfl_xor_sync(0xffffffffu, sum.x, o);
          sum.y += __shfl_xor_sync(0xffffffffu, sum.y, o);
        }
        if (in) {
          if (l == 0) reinterpret_cast<float*>(to + F::UNITS)[m] = unit;
          if (l % (GROUP / 8) == 0) reinterpret_cast<int2*>(to + F::SUMS)[l / (GROUP / 8) * ROWS + m] = sum;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint2*>(to + ((l / 8 * ROWS * 4 + m * 4 + c) * 4 + l % 4) * 16 + l / 4 % 2 * 8) = p[c];
        }
      } else if (in) {
        *reinterpret_cast<uint4*>(to + ((l / 4 * ROWS + m) * 4 + l % 4) * 16) = v;
      }
    }
  }
  __syncthreads();

  // What this lane reads of a block of x.  Columns without a row hold anything; nothing uses what they give.
  constexpr int OUTS = BYTES ? 2 : 4;
  constexpr int NEXT = 8 * 64;  // bytes to the next column tile
  const uint8_t* const xfirst = smem + kw * F::XBLOCK;
  const uint8_t* xblock = xfirst;
  const int xlane = (g * 4 + t) * 16;
  const int ulane = F::UNITS + t / 2 * 4, slane = F::SUMS + t / 2 * 8 + (t & 1) * 4;
  const float part = t & 1 ? 1.f / 16384.f : 1.f;
  const int slot = rows * 16;  // floats of a warp's sums of a tile
  float* const sums = reinterpret_cast<float*>(smem + a.sums);  // [step][warp][row][16]
  float* to = sums + warp * slot;
  float acc[NT][OUTS] = {};
  int kb = per;
  auto product = [&](const B4& b) {
    if constexpr (BYTES) {
      b.template product8<BF16, NT>(
          acc,
          [&](int h, int n) { return *reinterpret_cast<const uint4*>(xblock + xlane + n * NEXT + h * ROWS * 256); },
          [&](int j, int n) { return *reinterpret_cast<const int*>(xblock + slane + (j * ROWS + n * 2) * 8); },
          [&](int n) { return *reinterpret_cast<const float*>(xblock + ulane + n * 8) * part; });
    } else {
      b.template product16<M, BF16, NT>(acc, rows, [&](int u, int n) {
        return *reinterpret_cast<const uint4*>(xblock + xlane + n * NEXT + u * ROWS * 64);
      });
    }
    xblock += F::XBLOCK;
    if (--kb == 0) {
      kb = per;
      xblock = xfirst;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if constexpr (BYTES) {
          const int m = n * 2 + t / 2;
          acc[n][0] += __shfl_xor_sync(0xffffffffu, acc[n][0], 1);
          acc[n][1] += __shfl_xor_sync(0xffffffffu, acc[n][1], 1);
          if (m < rows) to[m * 16 + g + 8 * (t & 1)] = t & 1 ? acc[n][1] : acc[n][0];
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int m = n * 8 + 2 * t + (c & 1);
            if (m < rows) to[m * 16 + g + 8 * (c >> 1)] = acc[n][c];
          }
        }
#pragma unroll
        for (int c = 0; c < OUTS; ++c) acc[n][c] = 0.f;
      }
      to += warps * slot;
    }
  };

  const bool has_zeros = a.w.zeros != nullptr;
  int slot_at = 0;
#pragma unroll 1
  for (int i = 0; i < total; ++i) {
    cp_wait<F::DEPTH - 2>();
    __syncwarp();  // the block is there for every lane, and every lane is done with the one before
    issue();
    B4 b;
    b.load(ring + slot_at, has_zeros, lane);
    slot_at = slot_at == (F::DEPTH - 1) * B4::BYTES ? 0 : slot_at + B4::BYTES;
    product(b);
  }

  // The sums added, four rows of W a thread.
  if (a.shift)
    cluster_sync();
  else
    __syncthreads();
  const int quads = a.steps * groups * rows * 4;
  for (int i = (((warp << a.shift) + rank) << 5) + lane; i < quads; i += (warps << a.shift) << 5) {
    const int mg = i / 4, gs = rows == 1 ? mg : mg / rows, m = mg - gs * rows;
    const int step = gs / groups, grp = gs - step * groups;
    const int n = (id * groups + grp + step * stride) * 16 + i % 4 * 4;
    if (n >= a.n) continue;
    const float* at = sums + (step * warps + (grp << wks)) * slot + m * 16 + i % 4 * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!a.shift) {
#pragma unroll 4
      for (int w = 0; w < 1 << wks; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(at + w * slot);
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
      }
    } else {
#pragma unroll 8
      for (int w = 0; w < 1 << (wks + a.shift); ++w) {
        const float4 v = ld_cluster(smem_u32(at + (w >> a.shift) * slot), w & ((1 << a.shift) - 1));
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
      }
    }
    if constexpr (BYTES) {
      const bool x = s.x != s.x, y = s.y != s.y, z = s.z != s.z, w = s.w != s.w;
      if (x || y || z || w) {
        const float4 v = by_terms<BF16, GROUP>(a, m0 + m, n);
        if (x) s.x = v.x;
        if (y) s.y = v.y;
        if (z) s.z = v.z;
        if (w) s.w = v.w;
      }
    }
    const float xs = a.x_scale ? a.x_scale[m0 + m] : 1.f;
    const float out[4] = {s.x * xs, s.y * xs, s.z * xs, s.w * xs};
    using T = std::conditional_t<BF16, bf16, __half>;
    const T* bias = static_cast<const T*>(a.bias);
    T* y = static_cast<T*>(a.y) + (long long)(m0 + m) * a.n;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (n + e >= a.n) break;
      if constexpr (BF16)
        y[n + e] = tobf(out[e] + (bias ? bf(bias[n + e]) : 0.f));
      else
        y[n + e] = __float2half_rn(out[e] + (bias ? __half2float(bias[n + e]) : 0.f));
    }
  }
  if (a.shift) cluster_sync();  // the others' reads of these sums are over
}

int lfail(int code, const char* msg) {
  tao_set_last_error(msg);
  return code;
}

struct Plan {
  int shift, wk_shift, warps, blocks, steps, ring, sums, smem;
};

// The split with the least time by a rough measure, in us: what the longest warp's blocks of 128 k
// take one after the other, or all of an SM's; x on its way; the additions (a cluster of 8 pays them twice:
// 4 rows of k = 14336, n = 4096 take 16.4 us in clusters of 8, 12.5 in clusters of 4).  `xblock`, `wring`: bytes
// of a block of x, and of a warp's ring.
Plan plan_of(int tiles, int kblocks, int rows, int xblock, int wring, int max_warps) {
  Plan best = {};
  double least = 1e30;
  for (int shift = 0; shift <= 3; ++shift) {
    const int cluster = 1 << shift, kb = (kblocks + cluster - 1) / cluster, x = (kb * xblock + 127) / 128 * 128;
    if (cluster > kblocks) continue;
    // clusters that the device holds at once, with one block an SM
    const int clusters = shift == 0 ? 148 : shift == 1 ? 74 : shift == 2 ? 33 : 15;
    for (int warps = 4; warps <= max_warps; warps *= 2) {
      const int slot = warps * rows * 16 * 4;  // bytes of the warps' sums of a tile each
      const int ring = warps * wring, most = std::max(0, kSmem - x - ring) / slot;
      // every warp of a block has some of its k
      for (int wks = 0; 1 << wks <= std::min(warps, kblocks / cluster); ++wks) {
        const int groups = warps >> wks, sets = (tiles + groups - 1) / groups;
        const int all = (sets + clusters - 1) / clusters, waves = (all + most - 1) / std::max(most, 1);
        if (most < 1) continue;
        const int steps = (all + waves - 1) / waves, used = (sets + steps - 1) / steps;
        const int per = (kb + (1 << wks) - 1) >> wks;
        const double cost = waves * (std::max(steps * per * 0.20, (double)steps * groups * kb * 0.024) + x * 4e-5 +
                                     (shift == 3 ? 1.4 : shift ? 0.7 : 0.) + steps * 0.05 + warps * 0.01);
        if (cost >= least) continue;
        least = cost;
        best = {shift, wks, warps, used * cluster, steps, x, x + ring, x + ring + steps * slot};
      }
    }
  }
  return best;
}

// Launches KERNEL in clusters of 2^a.shift blocks; what it may use of shared memory is set once for each of
// the first 64 devices.
template <void (*KERNEL)(Linear4Args)>
int start(const Linear4Args& a, dim3 grid, int threads, int smem, int most_smem, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  const uint64_t mark = device < 64 ? 1ull << device : 0;
  if (e == cudaSuccess && !(ready.load(std::memory_order_relaxed) & mark)) {
    e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, most_smem);
    if (e == cudaSuccess) ready |= mark;
  }
  if (e == cudaSuccess) {
    cudaLaunchConfig_t c = {};
    c.gridDim = grid;
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = smem;
    c.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1 << a.shift;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    c.attrs = attr;
    c.numAttrs = a.shift ? 1 : 0;
    e = cudaLaunchKernelEx(&c, KERNEL, a);
  }
  return e == cudaSuccess ? TAO_OK : lfail(TAO_ERR_CUDA, cudaGetErrorString(e));
}

template <class M, bool BF16, int GROUP, int NT>
int launch(Linear4Args a, cudaStream_t s) {
  using F = Form<M, GROUP, NT>;
  const Plan p = plan_of(a.tiles, a.kblocks, std::min(a.rows, F::ROWS), F::XBLOCK, F::DEPTH * Block4<GROUP>::BYTES, F::WARPS);
  if (p.steps < 1) return lfail(TAO_ERR_CAPACITY, "no split of this product fits the device");
  a.shift = p.shift;
  a.wk_shift = p.wk_shift;
  a.steps = p.steps;
  a.ring = p.ring;
  a.sums = p.sums;
  return start<linear4_kernel<M, BF16, GROUP, NT>>(a, dim3(p.blocks, (a.rows + F::ROWS - 1) / F::ROWS), p.warps * 32,
                                                   p.smem, kSmem, s);
}

// Blocks of 128 rows of W, a cluster of them for as many parts of k as the device has room for.
template <class M, bool BF16, int GROUP>
int launch_tc(Linear4Args a, cudaStream_t s) {
  using C = Linear4Tc<GROUP>;
  const int sets = (a.tiles + 7) / 8, passes = (a.rows + C::COLS - 1) / C::COLS;
  double least = 1e30;
  for (int shift = 0; shift <= 3 && 1 << shift <= a.kblocks; ++shift) {
    const int clusters = shift == 0 ? 148 : shift == 1 ? 74 : shift == 2 ? 33 : 15;
    const int waves = (sets * passes + clusters - 1) / clusters, kb = (a.kblocks + (1 << shift) - 1) >> shift;
    const double cost = waves * (kb * 0.8 + 2. + (shift ? 1. : 0.));  // us, measured
    if (cost < least) {
      least = cost;
      a.shift = shift;
    }
  }
  return start<linear4_tc_kernel<M, BF16, GROUP>>(a, dim3(sets << a.shift, passes), C::THREADS, C::SMEM, C::SMEM, s);
}

// The bytes' form costs four columns a row and little else, the 16-bit one eight more instructions for
// eight weights: of k = n = 8192 one row takes 10.4 us (13.3 in 16 bits), two 11.2 (13.8), four 13.7 (14.2 as
// bytes in two column tiles, a form that is not kept).  tcgen05 needs the weights in shared memory: 16 rows
// 26.7 us (16.2 here), 17 26.9 (28.8), 64 29.5 (60.6); of k = 2048, n = 6144 17 rows 9.9 (8.7), 32 10.3 (10.7),
// 64 11.1 (18.9).  A form whose x does not fit a cluster of 8 blocks'
// shared memory leaves the product to the next smaller one, which reads the weights again (from L2) for each
// of its row tiles.
template <class M, bool BF16, int GROUP>
int by_rows(const Linear4Args& a, cudaStream_t s) {
  if (a.rows > 16) return launch_tc<M, BF16, GROUP>(a, s);
  int rc = TAO_ERR_CAPACITY;
  if (a.rows > 8) rc = launch<M, BF16, GROUP, 2>(a, s);
  if (a.rows > 2 && rc == TAO_ERR_CAPACITY) rc = launch<M, BF16, GROUP, 1>(a, s);
  if (rc == TAO_ERR_CAPACITY) rc = launch<Bytes, BF16, GROUP, 1>(a, s);
  return rc;
}

template <class M, bool BF16>
int by_group(const Linear4Args& a, int group, cudaStream_t s) {
  if (group == 32) return by_rows<M, BF16, 32>(a, s);
  if (group == 64) return by_rows<M, BF16, 64>(a, s);
  return by_rows<M, BF16, 128>(a, s);
}

}  // namespace
}  // namespace tao

extern "C" {

int tao_linear4(const void* x, long long x_stride, int x_type, const float* x_scale, const void* codes,
                const void* scales, const void* zeros, int group, int type, const void* bias, long long rows, int n,
                int k, void* y, void* stream) {
  using namespace tao;
  if (type != TAO_TYPE_BF16 && type != TAO_TYPE_FP16) return lfail(TAO_ERR_ARG, "4-bit scales are bf16 or fp16");
  if (x_type != type && x_type != TAO_TYPE_E4M3)
    return lfail(TAO_ERR_ARG, "activations are of the scales' type, or e4m3");
  if (group != 32 && group != 64 && group != 128) return lfail(TAO_ERR_ARG, "a group is 32, 64 or 128 weights");
  if (rows < 0 || n <= 0 || k <= 0) return lfail(TAO_ERR_ARG, "rows must not be negative, n and k must be positive");
  if (n > (1 << 24) || k > kMaxK) return lfail(TAO_ERR_ARG, "n is limited to 2^24 and k to 65536");
  if (rows == 0) return TAO_OK;
  if (!x || !codes || !scales || !y) return lfail(TAO_ERR_ARG, "null pointer");
  for (const void* p : {codes, scales, zeros})
    if (reinterpret_cast<uintptr_t>(p) % 16) return lfail(TAO_ERR_ARG, "a laid-out weight starts on 16 bytes");
  const int size = x_type == TAO_TYPE_E4M3 ? 1 : 2;
  if (!on_elements({{x, (size_t)size}, {x_scale, sizeof(float)}, {bias, 2}, {y, 2}}))
    return lfail(TAO_ERR_ARG, "operands start on a whole element");
  // a block writes its part of y while others still read theirs of x
  if (rows_overlap(x, rows, x_stride * size, (long long)k * size, y, rows * n * 2) ||
      (x_scale && rows_overlap(x_scale, 1, 0, rows * 4, y, rows * n * 2)) ||
      (bias && rows_overlap(bias, 1, 0, n * 2LL, y, rows * n * 2)))
    return lfail(TAO_ERR_ARG, "a product's output must not overlap its operands");
  constexpr long long kMost = 1 << 16;  // rows of a launch: the grid's second axis has at most 65535 blocks
  for (long long at = 0; at < rows; at += kMost) {
    Linear4Args a = {};
    a.w = {static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales),
           static_cast<const uint8_t*>(zeros)};
    a.x = static_cast<const uint8_t*>(x) + at * x_stride * size;
    a.x_stride = x_stride;
    a.x_scale = x_scale ? x_scale + at : nullptr;
    a.bias = bias;
    a.y = static_cast<uint8_t*>(y) + at * n * 2;
    a.rows = (int)std::min(rows - at, kMost);
    a.n = n;
    a.k = k;
    a.tiles = (n + 15) / 16;
    a.kblocks = (k + 127) / 128;
    a.wide = k % 8 == 0 && reinterpret_cast<uintptr_t>(a.x) % (8 * size) == 0 && x_stride % 8 == 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    a.x_type = x_type;
    const int rc = x_type == TAO_TYPE_BF16 ? by_group<MmaBf16, true>(a, group, s)
                   : type == TAO_TYPE_BF16 ? by_group<MmaF16, true>(a, group, s)
                                           : by_group<MmaF16, false>(a, group, s);
    if (rc) return rc;
  }
  return TAO_OK;
}

int tao_linear4_check(int* flags, void* stream) {
  using namespace tao;
  int host = 0;
  const int none = 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemcpyFromSymbolAsync(&host, g_linear4_error, sizeof(int), 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e == cudaSuccess && host) {
    e = cudaMemcpyToSymbolAsync(g_linear4_error, &none, sizeof(int), 0, cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  }
  if (e != cudaSuccess) return lfail(TAO_ERR_CUDA, cudaGetErrorString(e));
  if (flags) *flags = host;
  return host ? lfail(TAO_ERR_DEVICE, "a 4-bit product waited too long for the tensor cores") : TAO_OK;
}

}  // extern "C"
