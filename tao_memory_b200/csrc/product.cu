// Host side of the 16-bit products: checks, tensor maps, the choice of a tile and a split, launches; and the
// kernels of the gradient that are no products (product.cuh).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "product.cuh"
#include "product_few.cuh"

void tao_set_last_error(const char* msg);

namespace tao {
namespace product {
namespace {

int pfail(int code, const char* msg) {
  tao_set_last_error(msg);
  return code;
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q{};
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// A 16-bit matrix as it lies in memory: `inner` neighbours, rows `stride` elements apart, matrices `matrix` apart.
struct Operand2 {
  const void* at;
  long long inner, rows, stride, count, matrix;
};

// Boxes of 64 neighbours (128 bytes, swizzled) of `box` rows; zeros beyond every end.
bool make_map(CUtensorMap* map, const Operand2& o, int type, int box) {
  auto fn = encode_fn();
  if (!fn) return false;
  const long long row = o.rows > 1 ? o.stride * 2 : (o.inner * 2 + 15) / 16 * 16;
  cuuint64_t dims[3] = {(cuuint64_t)o.inner, (cuuint64_t)o.rows, (cuuint64_t)o.count};
  cuuint64_t strides[2] = {(cuuint64_t)row, (cuuint64_t)(o.count > 1 ? o.matrix * 2 : row * o.rows)};
  cuuint32_t boxes[3] = {kTerms, (cuuint32_t)box, 1};
  cuuint32_t steps[3] = {1, 1, 1};
  auto encode = [&] {
    return fn(map, type == TAO_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
              const_cast<void*>(o.at), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT || r == CUDA_ERROR_NOT_INITIALIZED) {  // a thread's first call, as a gradient's
    int device = 0;
    if (cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess) r = encode();
  }
  return r == CUDA_SUCCESS;
}

int sms() {
  int device = 0, n = 148;
  if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
  return n;
}

// What a launch multiplies: operands in the order of the kernel's maps (an absent one's address is null).
struct Operands {
  Operand2 a, b, a2, b2;
};

// Clusters of `blocks` blocks that the device runs at once (how many of them find room in one GPC).
template <int FORM, int BN, bool PAIR>
int clusters_of(int blocks) {
  static std::atomic<int> known[16][9];  // of the first 16 devices
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return 1;
  if (device < 16)
    if (const int n = known[device][blocks].load(std::memory_order_relaxed)) return n;
  using C = Cfg<FORM, BN, false, true, PAIR>;
  auto kernel = product_kernel<FORM, BN, false, true, PAIR, true>;
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(blocks);
  c.blockDim = dim3(kThreads);
  c.dynamicSmemBytes = C::SMEM;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  c.attrs = attr;
  c.numAttrs = 1;
  int n = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kernel, &c) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = 1;
  }
  if (device < 16) known[device][blocks].store(n, std::memory_order_relaxed);
  return n;
}

template <int FORM, int BN, bool GATED, bool SPLIT, bool PAIR, bool BF16>
int start_typed(const Operands& o, Args a, int split, cudaStream_t stream) {
  using C = Cfg<FORM, BN, GATED, SPLIT, PAIR>;
  auto kernel = product_kernel<FORM, BN, GATED, SPLIT, PAIR, BF16>;
  CUtensorMap maps[4];
  constexpr int A_BOX = C::A_MN ? kTerms : 128, B_BOX = C::B_MN ? kTerms : PAIR ? 128 : FORM == FORWARD ? C::CT : BN;
  const Operand2* ops[4] = {&o.a, &o.b, &o.a2, &o.b2};
  for (int i = 0; i < 4; ++i) {
    if (!ops[i]->at)
      maps[i] = maps[i & 1];
    else if (!make_map(&maps[i], *ops[i], a.type, i & 1 ? B_BOX : A_BOX))
      return pfail(TAO_ERR_CUDA, "cuTensorMapEncodeTiled failed");
  }
  static std::atomic<uint64_t> ready{0};  // of the first 64 devices
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  const uint64_t mark = device < 64 ? 1ull << device : 0;
  if (e == cudaSuccess && !(ready.load(std::memory_order_relaxed) & mark)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e == cudaSuccess) ready |= mark;
  }
  if (e != cudaSuccess) return pfail(TAO_ERR_CUDA, cudaGetErrorString(e));
  const long long col_tiles = (a.cols + C::CT - 1) / C::CT;
  long long tiles;
  if (FORM == WEIGHT)
    tiles = (long long)(a.depth + C::DOWN - 1) / C::DOWN * col_tiles * a.groups * a.pairs;
  else  // of experts: no more than this
    tiles = ((a.rows + C::TT - 1) / C::TT + (a.offsets ? a.groups : 0)) * col_tiles;
  if (tiles > (1 << 29)) return pfail(TAO_ERR_CAPACITY, "the product has too many tiles");
  a.split = split;
  cudaLaunchConfig_t c = {};
  const int together = (SPLIT ? split : 1) * (PAIR ? 2 : 1);  // blocks of a cluster
  c.gridDim = dim3((unsigned)(together * (SPLIT ? tiles : std::min<long long>(tiles, sms() / together))));
  c.blockDim = dim3(kThreads);
  c.dynamicSmemBytes = C::SMEM;
  c.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = together;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  c.attrs = attr;
  c.numAttrs = SPLIT || PAIR ? 1 : 0;
  e = cudaLaunchKernelEx(&c, kernel, maps[0], maps[1], maps[2], maps[3], a);
  return e == cudaSuccess ? TAO_OK : pfail(TAO_ERR_CUDA, cudaGetErrorString(e));
}

template <int FORM, int BN, bool GATED, bool SPLIT, bool PAIR = false>
int start(const Operands& o, const Args& a, int split, cudaStream_t stream) {
  return a.type == TAO_TYPE_BF16 ? start_typed<FORM, BN, GATED, SPLIT, PAIR, true>(o, a, split, stream)
                                 : start_typed<FORM, BN, GATED, SPLIT, PAIR, false>(o, a, split, stream);
}

// Blocks that share a tile's terms, and what it takes in steps of the ring: rounds of all clusters, each of its
// steps and of `join` more for what the blocks give each other (none: of a few for the first and last tile).
struct Split {
  int blocks;
  double cost;
};
template <int FORM, int BN, bool PAIR = false>
Split split_of(long long tiles, int steps, double join) {
  constexpr int TOGETHER = PAIR ? 2 : 1;
  const int at_once = sms() / TOGETHER;
  Split best = {1, (double)((tiles + at_once - 1) / at_once) * (steps + 6)};
  for (int s = 2; s * TOGETHER <= 8 && s <= steps; ++s) {
    const int fit = clusters_of<FORM, BN, PAIR>(s * TOGETHER);
    const double cost = (double)((tiles + fit - 1) / fit) * ((steps + s - 1) / s + join);
    if (cost < best.cost) best = {s, cost};
  }
  return best;
}

// FORWARD and INPUT of many rows, by what the rounds of all SMs cost in steps of a 128 tile (about 0.2 us): a step of a
// tile of 256 columns 1.6 of them, of a pair's 256 x 256 1.48 (INPUT: 1.4) and 6 for its start, and for a split of 64
// columns some 32.  Half of an expert's last tile is taken as empty.  A pair's two blocks share one round of outputs, so
// with sums of fewer than 16 steps and an activation to compute it may lose.  Alone / pair, us, gated 1536 channels of 16384
// rows of 16 experts: 8 steps 48.7 / 58.3, 12 65.4 / 68.5, 14 75.5 / 74.4, 16 84.0 / 82.4; silu to 2304 channels with z kept,
// 4096 rows: 12 steps 24.9 / 26.7, 15 28.1 / 28.9; 32768 rows: 8 steps 116.6 / 118.8, 12 129.1 / 128.5, 15 143.7 / 137.6.
// (Many rows of one matrix would gain up to 5 % from 12 steps on.)
// Measured (us), 256 columns / 128 / 64 and split: 2048x768x2304 9.2 / 9.9 / 46; 512x2048x2048 14.4 / 10.1 / 17.3;
// 128x8192x2048 48.5 / 29.6 / 16.7.  256 columns / pair: 16384x2048x8192 379.8 / 353.3; 2048x2048x2048 22.0 / 23.3;
// INPUT of 16384x8192x2048 523.6 / 364.0; gated 4096 tokens by 8 of 64 experts 240.5 / 249.2, 16384 by 2 of 16 208.6 / 195.2.
template <int FORM, bool GATED = false>
int start_rows(const Operands& o, const Args& a, int steps, cudaStream_t s) {
  const int n = sms(), columns = GATED ? 128 : 256;
  const auto rounds = [&](int down, int across, int at_once) {
    const long long tiles = ((a.rows + down - 1) / down + (a.offsets ? a.groups / 2 : 0)) *
                            (long long)((a.cols + across - 1) / across);
    return (tiles + at_once - 1) / at_once;
  };
  const double wide = rounds(128, columns, n) * (1.6 * steps);
  const double pair = a.act != TAO_ACT_NONE && steps < 16
                          ? 2 * wide
                          : rounds(256, columns, n / 2) * ((FORM == INPUT ? 1.4 : 1.48) * steps) + 6;
  if constexpr (!GATED) {
    const double narrow = (double)rounds(128, 128, n) * steps;
    if (!a.offsets) {
      const Split split = split_of<FORM, 64>(((a.rows + 127) / 128) * (long long)((a.cols + 63) / 64), steps, 32);
      if (split.blocks > 1 && split.cost < std::min({wide, narrow, pair}))
        return start<FORM, 64, false, true>(o, a, split.blocks, s);
    }
    if (narrow < std::min(wide, pair) || a.cols <= 128) return start<FORM, 128, false, false>(o, a, 1, s);
  }
  if (pair < wide) return start<FORM, 256, GATED, false, true>(o, a, 1, s);
  return start<FORM, 256, GATED, false>(o, a, 1, s);
}

template <int EIGHTS, int WARPS, int AHEAD>
int start_few(const FewArgs& a, int type, cudaStream_t s) {
  const unsigned grid = (a.n + 15) / 16;
  if (type == TAO_TYPE_BF16)
    few_kernel<EIGHTS, WARPS, AHEAD, true><<<grid, 32 * WARPS, 0, s>>>(a);
  else
    few_kernel<EIGHTS, WARPS, AHEAD, false><<<grid, 32 * WARPS, 0, s>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TAO_OK : pfail(TAO_ERR_CUDA, cudaGetErrorString(e));
}

// Up to 32 rows; `false`: the tcgen05 form is the faster one.  More warps where there are few blocks and long sums, fewer
// where a warp would have no round.  Measured (us, warps x rounds ahead), one row: 6144 outputs of 2048 terms 8x4 7.0, 8x8 7.6,
// 4x8 7.1; 2048 of 8192 16x4 9.9, 8x8 10.8; 8192 of 8192 8x8 25.3, 8x4 29.6; 640 of 2048 16x4 3.3, 8x4 4.0; 16384 of 512 4x4
// 4.9, 8x4 9.2.  Sixteen rows: 6144 of 2048 8x2 8.4, 16x4 10.4; 2048 of 8192 16x4 11.7, 8x2 19.0.  32 rows: 2048 of 8192 16x2
// 15.4, 8x1 28.7 (tcgen05 14.7); 6144 of 2048 8x1 11.4, 16x2 14.0 (13.5); 8192 of 8192 8x1 38.4 (28.7).
bool few_rows(const FewArgs& a, int type, cudaStream_t s, int* rc) {
  const int outputs = (a.n + 15) / 16, rounds = (a.k + 31) / 32;
  const bool narrow = outputs <= 148 && rounds >= 48;
  if (a.rows <= 8)
    *rc = rounds <= 16 ? start_few<1, 4, 4>(a, type, s)
          : narrow || (rounds > 64 && outputs <= 296) ? start_few<1, 16, 4>(a, type, s)
          : rounds <= 64 ? start_few<1, 8, 4>(a, type, s)
                         : start_few<1, 8, 8>(a, type, s);
  else if (a.rows <= 16)
    *rc = narrow ? start_few<2, 16, 4>(a, type, s) : start_few<2, 8, 2>(a, type, s);
  else if (outputs >= 448)
    return false;
  else
    *rc = outputs <= 148 ? start_few<4, 16, 2>(a, type, s) : start_few<4, 8, 1>(a, type, s);
  return true;
}

// Neighbours (8, 2 or 1) that can move at once in rows of `cols` whose addresses and strides in bytes have these bits.
int unit_of(int cols, unsigned long long bits) {
  return cols % 8 == 0 && bits % 16 == 0 ? 8 : cols % 2 == 0 && bits % 4 == 0 ? 2 : 1;
}
unsigned long long bits_of(const void* p, long long stride) {
  return reinterpret_cast<uintptr_t>(p) | (unsigned long long)stride * 2;
}



// -- the gradient's elementwise part ------------------------------------------
struct SlopeArgs {
  const void *dy, *z, *u;
  const uint8_t* low;  // gated: the lower bits of z and, rows * z_stride on, of u
  long long dy_stride, z_stride, d_stride;
  void *dz, *du;
  float* sums;  // [blocks][n] of dz, or null
  long long rows;
  int n, type, act, per;  // rows of a block
};

// dz = dy act'(z), or dy u act'(z) and du = dy act(z); sums over a block's rows of dz as it is before rounding.
// A thread has VEC columns of a slab of 32 VEC and every eighth row, some rows' loads on their way at once: it is
// bound by its bytes.
template <int VEC, int ACT, bool SLOPED, bool GATED, bool BF16>
__global__ void __launch_bounds__(256) slope_kernel(const SlopeArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = (blockIdx.x * 32 + lane) * VEC;
  const long long begin = (long long)blockIdx.y * a.per, end = min(begin + a.per, a.rows);
  using Word = typename Unit<VEC>::Type;
  using Low = std::conditional_t<VEC == 8, uint2, std::conditional_t<VEC == 2, uint16_t, uint8_t>>;
  const auto widen24 = [](const Word& upper, const Low& lower, float (&v)[VEC]) {
    uint32_t up[VEC / 2 + 1], low[2] = {};
    if constexpr (VEC == 8) {
      up[0] = upper.x, up[1] = upper.y, up[2] = upper.z, up[3] = upper.w, low[0] = lower.x, low[1] = lower.y;
    } else {
      up[0] = upper, low[0] = lower;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = of24(up[i / 2] >> (16 * (i & 1)) & 0xffffu, low[i / 4] >> (8 * (i & 3)) & 0xffu);
  };
  auto widen = [](const Word& w, float (&v)[VEC]) {
    if constexpr (VEC == 8) {
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack(words[i], BF16);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      }
    } else if constexpr (VEC == 2) {
      const float2 f = unpack(w, BF16);
      v[0] = f.x, v[1] = f.y;
    } else {
      v[0] = unpack1(w, BF16);
    }
  };
  auto store = [&](void* p, long long r, const float (&v)[VEC]) {
    uint16_t* at = static_cast<uint16_t*>(p) + r * a.d_stride + col;
    if constexpr (VEC == 8)
      *reinterpret_cast<uint4*>(at) =
          make_uint4(pack(v[0], v[1], BF16), pack(v[2], v[3], BF16), pack(v[4], v[5], BF16), pack(v[6], v[7], BF16));
    else if constexpr (VEC == 2)
      *reinterpret_cast<uint32_t*>(at) = pack(v[0], v[1], BF16);
    else
      *at = pack1(v[0], BF16);
  };
  auto load = [&](const void* p, long long r, long long stride) {
    return *reinterpret_cast<const Word*>(static_cast<const uint16_t*>(p) + r * stride + col);
  };
  float sum[VEC] = {};
  constexpr int AHEAD = GATED ? 2 : 4;
  if (col < a.n) {
    for (long long r0 = begin + warp; r0 < end; r0 += 8 * AHEAD) {
      Word wy[AHEAD], wz[AHEAD], wu[AHEAD];
      Low lz[AHEAD], lu[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const long long r = r0 + 8 * j;
        if (r >= end) break;
        wy[j] = load(a.dy, r, a.dy_stride);
        if constexpr (SLOPED) wz[j] = load(a.z, r, a.z_stride);
        if constexpr (GATED) {
          wu[j] = load(a.u, r, a.z_stride);
          lz[j] = *reinterpret_cast<const Low*>(a.low + r * a.z_stride + col);
          lu[j] = *reinterpret_cast<const Low*>(a.low + (a.rows + r) * a.z_stride + col);
        }
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const long long r = r0 + 8 * j;
        if (r >= end) break;
        float dy[VEC], z[VEC], u[VEC];
        widen(wy[j], dy);
        if constexpr (SLOPED) {
          if constexpr (GATED) {
            widen24(wz[j], lz[j], z);
            widen24(wu[j], lu[j], u);
          } else {
            widen(wz[j], z);
          }
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float2 f = activate_slope(z[i], ACT);
            if constexpr (GATED) {
              z[i] = dy[i] * f.x;  // du
              dy[i] *= u[i] * f.y;
            } else {
              dy[i] *= f.y;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] += dy[i];
        if (a.dz) {  // and du
          store(a.dz, r, dy);
          if constexpr (GATED) store(a.du, r, z);
        }
      }
    }
  }
  if (!a.sums) return;
  __shared__ float part[8][32 * VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) part[warp][i * 32 + lane] = sum[i];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * VEC; i += 256) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += part[w][i];
    const int c = (blockIdx.x * 32 + (i & 31)) * VEC + i / 32;
    if (c < a.n) a.sums[(long long)blockIdx.y * a.n + c] = s;
  }
}

template <int VEC, int ACT, bool SLOPED, bool GATED>
void start_slope(const SlopeArgs& a, dim3 grid, cudaStream_t s) {
  if (a.type == TAO_TYPE_BF16)
    slope_kernel<VEC, ACT, SLOPED, GATED, true><<<grid, 256, 0, s>>>(a);
  else
    slope_kernel<VEC, ACT, SLOPED, GATED, false><<<grid, 256, 0, s>>>(a);
}
template <int VEC, int ACT>
void start_slope(const SlopeArgs& a, dim3 grid, cudaStream_t s) {
  if (a.u)
    start_slope<VEC, ACT, true, true>(a, grid, s);
  else if (ACT != TAO_ACT_NONE)  // without one dz is dy
    start_slope<VEC, ACT, true, false>(a, grid, s);
  else
    start_slope<VEC, ACT, false, false>(a, grid, s);
}
template <int VEC>
void start_slope(const SlopeArgs& a, dim3 grid, cudaStream_t s) {
  switch (a.act) {
    case TAO_ACT_RELU: return start_slope<VEC, TAO_ACT_RELU>(a, grid, s);
    case TAO_ACT_SILU: return start_slope<VEC, TAO_ACT_SILU>(a, grid, s);
    case TAO_ACT_GELU: return start_slope<VEC, TAO_ACT_GELU>(a, grid, s);
    case TAO_ACT_GELU_TANH: return start_slope<VEC, TAO_ACT_GELU_TANH>(a, grid, s);
  }
  start_slope<VEC, TAO_ACT_NONE>(a, grid, s);
}

// Adds the blocks' sums in their order: eight runs of them side by side, then those.
__global__ void __launch_bounds__(256) column_sum_kernel(const float* sums, int blocks, int n, int type, void* out) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (col < n) {
#pragma unroll 4
    for (int b = blocks * warp / 8; b < blocks * (warp + 1) / 8; ++b) s += sums[(long long)b * n + col];
  }
  __shared__ float part[8][32];
  part[warp][lane] = s;
  __syncthreads();
  if (warp || col >= n) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += part[w][lane];
  static_cast<uint16_t*>(out)[col] = pack1(s, type == TAO_TYPE_BF16);
}

// Rows of a block of the slope kernel: at least 32, and few enough blocks for four on an SM.
int slope_rows(long long rows, int n) {
  const long long slabs = (n + 255) / 256, room = std::max<long long>(1, 148 * 4 / slabs);
  return (int)std::max<long long>(32, (rows + room - 1) / room);
}
int slope_blocks(long long rows, int n) {
  const int per = slope_rows(rows, n);
  return (int)((rows + per - 1) / per);
}

}  // namespace
}  // namespace product
}  // namespace tao

namespace tao {
namespace product {
namespace {

// A matrix or matrices as a caller has them.
struct Given {
  const void* at;
  long long rows, cols, count, row, col, matrix;  // strides in elements
};

// Whether TMA can fetch it as it lies: neighbours next to each other, everything else on 16 bytes, no overlaps.
bool fetchable(const Given& g) {
  return reinterpret_cast<uintptr_t>(g.at) % 16 == 0 && (g.cols == 1 || g.col == 1) &&
         (g.rows == 1 || (g.row % 8 == 0 && g.row >= g.cols && g.row < (1ll << 38))) &&
         (g.count == 1 || (g.matrix % 8 == 0 && g.matrix >= (g.rows - 1) * g.row + g.cols && g.matrix < (1ll << 38)));
}

// Up to three of them to rows of whole 16 bytes, from whatever strides they have.
struct Laying {
  Given from[3];
  uint16_t* to[3];
  long long stride[3];
  int count;
};
// A warp a row.  Neighbours go two at a time: words of the row as they lie, and, where it starts between two words, each
// made of two.
__global__ void __launch_bounds__(256) lay_kernel(const Laying l) {
  const Given& g = l.from[blockIdx.y];
  const long long rows = g.rows * g.count;
  const int lane = threadIdx.x & 31, cols = (int)g.cols;
  constexpr int AHEAD = 8;
  for (long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); row < rows; row += (long long)gridDim.x * 8) {
    const long long matrix = row / g.rows;
    const uint16_t* const in = static_cast<const uint16_t*>(g.at) + matrix * g.matrix + (row - matrix * g.rows) * g.row;
    uint16_t* const out = l.to[blockIdx.y] + row * l.stride[blockIdx.y];
    if (g.col != 1) {
#pragma unroll 8
      for (int c = lane; c < cols; c += 32) out[c] = in[c * g.col];
      continue;
    }
    const int odd = reinterpret_cast<uintptr_t>(in) >> 1 & 1;  // elements before the first whole word
    const uint32_t* const words = reinterpret_cast<const uint32_t*>(in + odd);
    const int whole = (cols - odd) / 2;  // words of the row
    uint32_t* const to = reinterpret_cast<uint32_t*>(out);
    if (!odd) {
#pragma unroll 8
      for (int c = lane; c < whole; c += 32) to[c] = words[c];
      if (lane == 0 && cols & 1) out[cols - 1] = in[cols - 1];
      continue;
    }
    // word c of the output: the upper half of word c - 1 and the lower one of word c
    for (int c0 = 0; c0 <= whole; c0 += 32 * AHEAD) {
      uint32_t before[AHEAD], v[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int c = c0 + j * 32 + lane;
        v[j] = c < whole ? words[c] : c == whole && 2 * c < cols - 1 ? (uint32_t)in[2 * c + 1] : 0u;
        before[j] = c > whole ? 0u : c == 0 ? (uint32_t)in[0] << 16 : words[c - 1];
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int c = c0 + j * 32 + lane;
        const uint32_t w = before[j] >> 16 | v[j] << 16;
        if (2 * c + 1 < cols)
          to[c] = w;
        else if (2 * c < cols)
          out[2 * c] = (uint16_t)w;
      }
    }
  }
}

// Rooms of a workspace, one behind the other; without a base only their size is counted.
struct Rooms {
  uint8_t* base;
  size_t used;
  void* take(size_t bytes) {
    void* p = base ? base + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return p;
  }
};
long long padded(long long cols) { return (cols + 7) / 8 * 8; }

// An operand that TMA can fetch: as given, or in the workspace, to be laid there.
Operand2 operand(const Given& g, Rooms& rooms, Laying& l) {
  if (!g.at) return {};
  if (fetchable(g)) return {g.at, g.cols, g.rows, g.row, g.count, g.matrix};
  const long long stride = padded(g.cols);
  void* to = rooms.take((size_t)(g.rows * g.count * stride * 2));
  l.from[l.count] = g, l.to[l.count] = static_cast<uint16_t*>(to), l.stride[l.count++] = stride;
  return {to, g.cols, g.rows, stride, g.count, g.rows * stride};
}
void lay(const Laying& l, cudaStream_t s) {
  long long rows = 0;
  for (int i = 0; i < l.count; ++i) rows = std::max(rows, l.from[i].rows * l.from[i].count);
  if (l.count) lay_kernel<<<dim3((unsigned)std::min<long long>((rows + 7) / 8, 148 * 8), l.count), 256, 0, s>>>(l);
}

Given given_x(const TaoLinear& p) { return {p.x, p.rows, p.k, 1, p.x_row, p.x_col, 0}; }
Given given_w(const TaoLinear& p) { return {p.w, p.n, p.k, p.experts, p.w_row, p.w_col, p.w_expert}; }
Given given_up(const TaoLinear& p) { return {p.up, p.n, p.k, p.experts, p.up_row, p.up_col, p.up_expert}; }

int check(const TaoLinear* p) {
  if (!p) return pfail(TAO_ERR_ARG, "null pointer");
  if (p->type != TAO_TYPE_BF16 && p->type != TAO_TYPE_FP16) return pfail(TAO_ERR_ARG, "16-bit products take bf16 or fp16");
  if (p->activation < TAO_ACT_NONE || p->activation > TAO_ACT_GELU_TANH) return pfail(TAO_ERR_ARG, "unknown activation");
  if (p->rows < 0 || p->n <= 0 || p->k <= 0)
    return pfail(TAO_ERR_ARG, "rows must not be negative, n and k must be positive");
  if (p->rows > (1ll << 30) || p->n > (1 << 24) || p->k > (1 << 24))
    return pfail(TAO_ERR_ARG, "rows are limited to 2^30, n and k to 2^24");
  if (p->offsets ? p->experts < 1 || p->experts > kMostGroups : p->experts != 1)
    return pfail(TAO_ERR_ARG, "offsets are those of 1 to 512 experts; without them there is one matrix");
  if (p->offsets ? p->bias || p->residual : p->up != nullptr)
    return pfail(TAO_ERR_ARG, "experts have no bias or residual, and a gate needs experts");
  if (!on_elements({{p->x, 2}, {p->w, 2}, {p->up, 2}, {p->bias, 2}, {p->residual, 2}, {p->y, 2}, {p->z, 2}, {p->u, 2},
                    {p->offsets, 4}, {p->dy, 2}, {p->dx, 2}, {p->dw, 2}, {p->dup, 2}, {p->db, 2}}))
    return pfail(TAO_ERR_ARG, "operands start on a whole element");
  return TAO_OK;
}

Extent reach(const Given& g) {
  if (!g.at) return {0, 0};
  const long long across = (g.cols - 1) * g.col * 2;  // strides are not negative where they come from tensors
  return extent(g.at, g.rows, g.row * 2, across + 2, g.count, g.matrix * 2);
}
bool any_overlap(const TaoLinear& p, bool gradient) {
  const long long rows = p.rows, n = p.n, k = p.k, y = rows * n * 2, w = (long long)p.experts * n * k * 2;
  const long long kept = p.up ? rows * p.z_row * 2 : ((rows - 1) * p.z_row + n) * 2;  // gated: whole rows
  const Extent x = reach(given_x(p)), weight = reach(given_w(p)), up = reach(given_up(p)), z = extent(p.z, 1, 0, kept),
               u = extent(p.u, 1, 0, kept), low = extent(p.up ? p.low : nullptr, 1, 0, kept), offsets = extent(p.offsets, 1, 0, (p.experts + 1) * 4ll);
  if (!gradient) {
    const Extent bias = extent(p.bias, 1, 0, n * 2), residual = extent(p.residual, rows, p.r_row * 2, n * 2);
    const bool in_place = p.residual == p.y && (p.r_row == n || rows == 1);
    return overlaps(p.y, y, {x, weight, up, bias, in_place ? Extent{0, 0} : residual, z, p.z ? u : Extent{0, 0}, p.z ? low : Extent{0, 0}, offsets}) ||
           overlaps(p.z, kept, {x, weight, up, bias, residual, u, low, offsets}) ||
           (p.z && overlaps(p.u, kept, {x, weight, up, low, offsets})) ||
           (p.z && p.up && overlaps(p.low, kept, {x, weight, up, offsets}));
  }
  const Extent dy = extent(p.dy, rows, p.dy_row * 2, n * 2), dx = extent(p.dx, 1, 0, rows * k * 2), dw = extent(p.dw, 1, 0, w),
               dup = extent(p.dup, 1, 0, w);
  return overlaps(p.dx, rows * k * 2, {x, weight, up, z, u, low, offsets, dy, dw, dup}) ||
         overlaps(p.dw, w, {x, weight, up, z, u, low, offsets, dy, dup}) ||
         overlaps(p.dup, w, {x, weight, up, z, u, low, offsets, dy}) ||
         overlaps(p.db, n * 2, {x, weight, up, z, u, low, offsets, dy, dx, dw, dup});
}

// What is kept for the gradient: rows that do not reach into each other; gated, on 16 bytes.
int check_kept(const TaoLinear& p, bool gradient) {
  const bool used = p.z && (!gradient || p.activation != TAO_ACT_NONE || p.up);
  if (used && p.rows > 1 && p.z_row < p.n) return pfail(TAO_ERR_ARG, "a row of z has room for n values");
  if (p.up && p.z && (p.z_row % 16 || p.z_row < p.n ||
                      (reinterpret_cast<uintptr_t>(p.z) | reinterpret_cast<uintptr_t>(p.u) |
                       reinterpret_cast<uintptr_t>(p.low)) % 16))
    return pfail(TAO_ERR_ARG, "a gate's kept factors start on 16 bytes, in rows of a multiple of 16");
  return TAO_OK;
}

int check_room(const TaoLinear& p, size_t need) {
  if (need && (!p.workspace || reinterpret_cast<uintptr_t>(p.workspace) % 256 || p.workspace_bytes < need))
    return pfail(TAO_ERR_ARG, "the products' workspace is too small, or off 256 bytes");
  return TAO_OK;
}

int forward(const TaoLinear& p, Rooms& rooms, cudaStream_t s) {
  Laying laying = {};
  const Operand2 ox = operand(given_x(p), rooms, laying), ow = operand(given_w(p), rooms, laying),
                 ou = operand(given_up(p), rooms, laying), none = {};
  if (!rooms.base) return TAO_OK;
  lay(laying, s);
  const int n = p.n, k = p.k;
  const long long rows = p.rows;
  Args a = {};
  a.offsets = p.offsets, a.groups = p.experts, a.rows = (int)rows, a.cols = n, a.depth = k, a.pairs = 1;
  a.type = p.type, a.act = p.activation, a.bias = p.bias, a.residual = p.residual, a.r_stride = p.r_row;
  a.y = p.y, a.z = p.z, a.u = p.z ? p.u : nullptr, a.low = static_cast<uint8_t*>(p.low), a.z_stride = p.z_row;
  a.wide = unit_of(n, bits_of(p.y, n) | (p.z && !p.up ? bits_of(p.z, p.z_row) : 0) |
                          (p.residual ? bits_of(p.residual, p.r_row) : 0)) == 8;
  const int steps = (k + kTerms - 1) / kTerms;
  if (p.offsets) {
    // By the experts' mean rows, columns of 32 or 64 rows or tiles of 128.  64 experts gated 2048 to 1024 (us): mean 4
    // 63.3 / 63.5 / 66.9, 24 82.4 / 81.3 / 88.0, 32 78.2 / 70.0 / 78.1, 64 97.8 / 91.9 / 91.1, 96 120.4 / 107.2 / 100.8; 128
    // experts 1024 to 512: mean 8 36.3 / 38.2 / 40.4, 48 53.1 / 50.2 / 50.1.
    const long long mean = rows / p.experts;
    const Operands few = {ow, ox, ou, none}, many = {ox, ow, none, ou};
    if (p.up) {
      if (mean <= 24) return start<FEW, 32, true, false>(few, a, 1, s);
      if (mean <= 64) return start<FEW, 64, true, false>(few, a, 1, s);
      return start_rows<FORWARD, true>(many, a, steps, s);
    }
    if (mean <= 24) return start<FEW, 32, false, false>(few, a, 1, s);
    if (mean <= 64) return start<FEW, 64, false, false>(few, a, 1, s);
    return start_rows<FORWARD>(many, a, steps, s);
  }
  if (rows <= 32) {
    const FewArgs f = {ox.at, ow.at, p.bias, p.residual, rows > 1 ? ox.stride : 0, n > 1 ? ow.stride : 0, p.r_row,
                       (int)rows, n, k, p.activation, p.y, p.z, p.z_row};
    int rc;
    if (few_rows(f, p.type, s, &rc)) return rc;
  }
  if (rows <= 64) {
    const Operands o = {ow, ox, none, none};
    const int split = split_of<FEW, 64>((n + 127) / 128, steps, 9).blocks;
    if (split == 1)
      return rows <= 32 ? start<FEW, 32, false, false>(o, a, 1, s) : start<FEW, 64, false, false>(o, a, 1, s);
    return rows <= 32 ? start<FEW, 32, false, true>(o, a, split, s) : start<FEW, 64, false, true>(o, a, split, s);
  }
  const Operands o = {ox, ow, none, none};
  return start_rows<FORWARD>(o, a, steps, s);
}

int input_gradient(const TaoLinear& p, const Operands& o, int pairs, cudaStream_t s) {
  const int n = p.n, k = p.k;
  Args a = {};
  a.offsets = p.offsets, a.groups = p.experts, a.rows = (int)p.rows, a.cols = k, a.depth = n, a.pairs = pairs;
  a.type = p.type, a.y = p.dx;
  a.wide = unit_of(k, bits_of(p.dx, k)) == 8;
  const int steps = (n + kTerms - 1) / kTerms * pairs;
  return start_rows<INPUT>(o, a, steps, s);
}

int weight_gradient(const TaoLinear& p, const Operands& o, int pairs, cudaStream_t s) {
  const int n = p.n, k = p.k;
  Args a = {};
  a.offsets = p.offsets, a.groups = p.experts, a.rows = (int)p.rows, a.cols = k, a.depth = n, a.pairs = pairs;
  a.type = p.type, a.y = p.dw, a.u = p.dup;
  a.wide = unit_of(k, bits_of(p.dw, k) | bits_of(p.dup, 0)) == 8;
  if (p.offsets) {
    if (k > 128) return start<WEIGHT, 256, false, false>(o, a, 1, s);
    return start<WEIGHT, 128, false, false>(o, a, 1, s);
  }
  // In steps of a 128 tile, as start_rows: of 256 columns a step 1.6 and a split 26 steps of its own more, by pairs 1.42 and
  // 33.  Measured (us), 256 columns / pairs / 128: 2304x768 of 32768 rows 110.2 (split over 2) / 93.6 (over 2) / 172; 768x768
  // of them 48.9 (over 6) / 50.0 (over 4) / 67 (over 3); 4096x4096 of 4096 125.4 / 109.3; 1024x1024 of 2048 17.6 / 17.1 / 13.1.
  const long long down = (n + 127) / 128;
  const int steps = (int)((p.rows + kTerms - 1) / kTerms), all = sms();
  const double narrow = (double)((down * ((k + 127) / 128) + all - 1) / all) * steps;
  const Split wide = split_of<WEIGHT, 256>(down * ((k + 255) / 256), steps, 26);
  const Split pair = split_of<WEIGHT, 256, true>((n + 255) / 256 * (long long)((k + 255) / 256), steps, 33);
  if (k <= 128 || narrow < std::min(1.6 * wide.cost, 1.42 * pair.cost)) {
    const Split half = split_of<WEIGHT, 128>(down * ((k + 127) / 128), steps, 32);
    if (half.blocks > 1 && half.cost < narrow) return start<WEIGHT, 128, false, true>(o, a, half.blocks, s);
    return start<WEIGHT, 128, false, false>(o, a, 1, s);
  }
  if (1.42 * pair.cost < 1.6 * wide.cost) {
    if (pair.blocks > 1) return start<WEIGHT, 256, false, true, true>(o, a, pair.blocks, s);
    return start<WEIGHT, 256, false, false, true>(o, a, 1, s);
  }
  if (wide.blocks > 1) return start<WEIGHT, 256, false, true>(o, a, wide.blocks, s);
  return start<WEIGHT, 256, false, false>(o, a, 1, s);
}

int backward(const TaoLinear& p, Rooms& rooms, cudaStream_t s) {
  const bool sloped = p.activation != TAO_ACT_NONE || p.up, products = p.dx || p.dw;
  const int pairs = p.up ? 2 : 1;
  // dz and du, or dy itself
  Given gz = {p.dy, p.rows, p.n, 1, p.dy_row, 1, 0}, gd = {};
  if (sloped || p.db) {
    SlopeArgs a = {p.dy, sloped ? p.z : nullptr, p.up ? p.u : nullptr, static_cast<const uint8_t*>(p.low), p.dy_row, p.z_row, padded(p.n), nullptr, nullptr,
                   nullptr, p.rows, p.n, p.type, p.activation, slope_rows(p.rows, p.n)};
    if (sloped && products) {
      const size_t size = (size_t)(p.rows * a.d_stride * 2);
      a.dz = rooms.take(size);
      gz = {a.dz, p.rows, p.n, 1, a.d_stride, 1, 0};
      if (p.up) {
        a.du = rooms.take(size);
        gd = {a.du, p.rows, p.n, 1, a.d_stride, 1, 0};
      }
    }
    const int blocks = slope_blocks(p.rows, p.n);
    if (p.db) a.sums = static_cast<float*>(rooms.take((size_t)blocks * p.n * sizeof(float)));
    if (rooms.base) {
      const int unit = unit_of(p.n, bits_of(p.dy, p.dy_row) | (sloped ? bits_of(p.z, p.z_row) | bits_of(p.u, 0) : 0));
      const int across = 32 * unit;
      const dim3 grid((p.n + across - 1) / across, blocks);
      if (unit == 8)
        start_slope<8>(a, grid, s);
      else if (unit == 2)
        start_slope<2>(a, grid, s);
      else
        start_slope<1>(a, grid, s);
      if (p.db) column_sum_kernel<<<(p.n + 31) / 32, 256, 0, s>>>(a.sums, blocks, p.n, p.type, p.db);
    }
  }
  if (products) {
    if (sloped && !rooms.base) gz.at = gd.at = nullptr;  // their rooms are counted, and they are laid as they are made
    Laying laying = {};
    const Operand2 oz = sloped ? Operand2{gz.at, gz.cols, gz.rows, gz.row, 1, 0} : operand(gz, rooms, laying),
                   od = p.up ? Operand2{gd.at, gd.cols, gd.rows, gd.row, 1, 0} : Operand2{};
    Operand2 ow = {}, ou = {}, ox = {};
    if (p.dx) ow = operand(given_w(p), rooms, laying), ou = operand(given_up(p), rooms, laying);
    if (p.dw) ox = operand(given_x(p), rooms, laying);  // with dy, W and U three at most: dz is made where there is U
    if (rooms.base) {
      lay(laying, s);
      if (p.dx)
        if (int rc = input_gradient(p, {oz, ow, od, ou}, pairs, s)) return rc;
      if (p.dw)
        if (int rc = weight_gradient(p, {oz, ox, od, {}}, pairs, s)) return rc;
    }
  }
  if (!rooms.base) return TAO_OK;
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TAO_OK : pfail(TAO_ERR_CUDA, cudaGetErrorString(e));
}

int missing(const TaoLinear& p, bool gradient) {
  if (!gradient) return !p.x || !p.w || !p.y || (p.up && p.z && (!p.u || !p.low));
  const bool sloped = p.activation != TAO_ACT_NONE || p.up;
  return !p.dy || (p.up ? !p.dw != !p.dup : p.dup != nullptr) || (p.dx && (!p.w)) || (p.dw && !p.x) ||
         (sloped && (!p.z || (p.up && (!p.u || !p.low))));
}

}  // namespace
}  // namespace product
}  // namespace tao

extern "C" {

size_t tao_linear_sizeof(void) { return sizeof(TaoLinear); }

size_t tao_linear_workspace_bytes(const TaoLinear* p, int gradient) {
  using namespace tao::product;
  if (check(p) || p->rows == 0) return 0;
  Rooms rooms = {nullptr, 0};
  if (gradient)
    backward(*p, rooms, nullptr);
  else
    forward(*p, rooms, nullptr);
  return rooms.used;
}

int tao_linear(const TaoLinear* p, void* stream) {
  using namespace tao::product;
  if (int rc = check(p)) return rc;
  if (p->rows == 0) return TAO_OK;
  if (missing(*p, false)) return pfail(TAO_ERR_ARG, "null pointer");
  if (int rc = check_kept(*p, false)) return rc;
  if (any_overlap(*p, false)) return pfail(TAO_ERR_ARG, "a product's output must not overlap its operands");
  if (int rc = check_room(*p, tao_linear_workspace_bytes(p, 0))) return rc;
  static uint8_t none[1];  // where no room is needed
  Rooms rooms = {p->workspace ? static_cast<uint8_t*>(p->workspace) : none, 0};
  return forward(*p, rooms, static_cast<cudaStream_t>(stream));
}

int tao_linear_gradient(const TaoLinear* p, void* stream) {
  using namespace tao::product;
  if (int rc = check(p)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p->rows == 0) {
    const size_t size = (size_t)p->experts * p->n * p->k * 2;
    cudaError_t e = cudaSuccess;
    if (p->dw) e = cudaMemsetAsync(p->dw, 0, size, s);
    if (e == cudaSuccess && p->dup) e = cudaMemsetAsync(p->dup, 0, size, s);
    if (e == cudaSuccess && p->db) e = cudaMemsetAsync(p->db, 0, (size_t)p->n * 2, s);
    return e == cudaSuccess ? TAO_OK : pfail(TAO_ERR_CUDA, cudaGetErrorString(e));
  }
  if (missing(*p, true)) return pfail(TAO_ERR_ARG, "null pointer");
  if (int rc = check_kept(*p, true)) return rc;
  if (!p->dx && !p->dw && !p->db) return TAO_OK;  // dup comes with dw
  if (any_overlap(*p, true)) return pfail(TAO_ERR_ARG, "a product's output must not overlap its operands");
  if (int rc = check_room(*p, tao_linear_workspace_bytes(p, 1))) return rc;
  static uint8_t none[1];
  Rooms rooms = {p->workspace ? static_cast<uint8_t*>(p->workspace) : none, 0};
  return backward(*p, rooms, s);
}

int tao_product_check(int* flags, void* stream) {
  using namespace tao::product;
  int host = 0;
  const int none = 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemcpyFromSymbolAsync(&host, g_error, sizeof(int), 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e == cudaSuccess && host) {
    e = cudaMemcpyToSymbolAsync(g_error, &none, sizeof(int), 0, cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  }
  if (e != cudaSuccess) return pfail(TAO_ERR_CUDA, cudaGetErrorString(e));
  if (flags) *flags = host;
  return host ? pfail(TAO_ERR_DEVICE, "a 16-bit product waited too long for its operands or the tensor cores") : TAO_OK;
}

}  // extern "C"
