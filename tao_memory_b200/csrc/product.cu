// Host side of the 16-bit products: checks, tensor maps, the choice of a tile and a split, launches; and the
// kernels of the gradient that are no products (product.cuh).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "product.cuh"

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

template <int FORM, int BN, bool GATED, bool SPLIT>
int start(const Operands& o, Args a, int split, cudaStream_t stream) {
  using C = Cfg<FORM, BN, GATED, SPLIT>;
  auto kernel = product_kernel<FORM, BN, GATED, SPLIT>;
  CUtensorMap maps[4];
  constexpr int A_BOX = C::A_MN ? kTerms : 128, B_BOX = C::B_MN ? kTerms : FORM == FORWARD ? C::CT : BN;
  const Operand2* ops[4] = {&o.a, &o.b, &o.a2, &o.b2};
  for (int i = 0; i < 4; ++i) {
    const Operand2& x = ops[i]->at ? *ops[i] : *ops[i & 1];
    if (!make_map(&maps[i], x, a.type, i & 1 ? B_BOX : A_BOX)) return pfail(TAO_ERR_CUDA, "cuTensorMapEncodeTiled failed");
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
    tiles = (long long)(a.depth + 127) / 128 * col_tiles * a.groups * a.pairs;
  else  // of experts: no more than this
    tiles = ((a.rows + C::TT - 1) / C::TT + (a.offsets ? a.groups : 0)) * col_tiles;
  if (tiles > (1 << 29)) return pfail(TAO_ERR_CAPACITY, "the product has too many tiles");
  a.split = split;
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3((unsigned)(SPLIT ? tiles * split : std::min<long long>(tiles, sms())));
  c.blockDim = dim3(kThreads);
  c.dynamicSmemBytes = C::SMEM;
  c.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  c.attrs = attr;
  c.numAttrs = SPLIT ? 1 : 0;
  e = cudaLaunchKernelEx(&c, kernel, maps[0], maps[1], maps[2], maps[3], a);
  return e == cudaSuccess ? TAO_OK : pfail(TAO_ERR_CUDA, cudaGetErrorString(e));
}

// Blocks that share a tile's terms: as many as the SMs hold beside the other tiles', of four steps each at least.
int split_of(long long tiles, int blocks) {
  const long long fit = tiles > 0 ? sms() / tiles : 1;
  return (int)std::max<long long>(1, std::min<long long>({fit, 8, blocks / 4}));
}

bool on16(const void* p, long long stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0; }

int check_sizes(long long rows, int n, int k, int type, int act, const int* offsets, int experts) {
  if (type != TAO_TYPE_BF16 && type != TAO_TYPE_FP16) return pfail(TAO_ERR_ARG, "16-bit products take bf16 or fp16");
  if (act < TAO_ACT_NONE || act > TAO_ACT_GELU_TANH) return pfail(TAO_ERR_ARG, "unknown activation");
  if (rows < 0 || n <= 0 || k <= 0) return pfail(TAO_ERR_ARG, "rows must not be negative, n and k must be positive");
  if (rows > (1ll << 30) || n > (1 << 24) || k > (1 << 24))
    return pfail(TAO_ERR_ARG, "rows are limited to 2^30, n and k to 2^24");
  if (offsets ? experts < 1 || experts > kMostGroups : experts != 1)
    return pfail(TAO_ERR_ARG, "offsets are those of 1 to 512 experts; without them there is one matrix");
  if (reinterpret_cast<uintptr_t>(offsets) % 4) return pfail(TAO_ERR_ARG, "operands start on a whole element");
  return TAO_OK;
}

// Operands of the tensor maps: on 16 bytes, rows (and matrices) too, and rows that do not overlap.
bool laid(const Operand2& o) {
  return !o.at || (on16(o.at, 0) && (o.rows <= 1 || (o.stride % 8 == 0 && o.stride >= o.inner && o.stride < (1ll << 38))) &&
                   (o.count <= 1 || (o.matrix % 8 == 0 && o.matrix > 0 && o.matrix < (1ll << 38))));
}

// -- the gradient's elementwise part ------------------------------------------
struct SlopeArgs {
  const void *dy, *z, *u;
  long long dy_stride, z_stride, d_stride;
  void *dz, *du;
  float* sums;  // [blocks][n] of dz, or null
  long long rows;
  int n, type, act, per;  // rows of a block
};

// dz = dy act'(z), or dy u act'(z) and du = dy act(z); sums over a block's rows of dz as it is before rounding.
// A thread has VEC columns of a slab of 32 VEC and every eighth row.
template <int VEC>
__global__ void __launch_bounds__(256) slope_kernel(const SlopeArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool is_bf16 = a.type == TAO_TYPE_BF16;
  const int col = (blockIdx.x * 32 + lane) * VEC;
  const long long begin = (long long)blockIdx.y * a.per, end = min(begin + a.per, a.rows);
  float sum[VEC] = {};
  if (col < a.n) {
#pragma unroll 2
    for (long long r = begin + warp; r < end; r += 8) {
      float dy[VEC], z[VEC], u[VEC];
      auto load = [&](const void* p, long long stride, float (&v)[VEC]) {
        const uint16_t* at = static_cast<const uint16_t*>(p) + r * stride + col;
        if constexpr (VEC == 8) {
          const uint4 w = *reinterpret_cast<const uint4*>(at);
          const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = unpack(words[i], is_bf16);
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
          }
        } else {
          v[0] = unpack1(*at, is_bf16);
        }
      };
      auto store = [&](void* p, const float (&v)[VEC]) {
        uint16_t* at = static_cast<uint16_t*>(p) + r * a.d_stride + col;
        if constexpr (VEC == 8)
          *reinterpret_cast<uint4*>(at) = make_uint4(pack(v[0], v[1], is_bf16), pack(v[2], v[3], is_bf16),
                                                     pack(v[4], v[5], is_bf16), pack(v[6], v[7], is_bf16));
        else
          *at = pack1(v[0], is_bf16);
      };
      load(a.dy, a.dy_stride, dy);
      if (a.z) load(a.z, a.z_stride, z);
      if (a.u) load(a.u, a.z_stride, u);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if (a.z) {
          const float2 f = activate_slope(z[i], a.act);
          if (a.u) {
            z[i] = dy[i] * f.x;  // du
            dy[i] *= u[i] * f.y;
          } else {
            dy[i] *= f.y;
          }
        }
        sum[i] += dy[i];
      }
      if (a.dz) store(a.dz, dy);
      if (a.u) store(a.du, z);
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

extern "C" {

int tao_linear(const void* x, long long x_stride, const void* w, long long w_stride, long long w_expert, const void* up,
               long long up_stride, long long up_expert, const void* bias, const void* residual, long long r_stride,
               const int* offsets, int experts, long long rows, int n, int k, int type, int activation, void* y, void* z,
               void* u, long long z_stride, void* stream) {
  using namespace tao;
  using namespace tao::product;
  if (int rc = check_sizes(rows, n, k, type, activation, offsets, experts)) return rc;
  if (rows == 0) return TAO_OK;
  if (!x || !w || !y || (up && z && !u)) return pfail(TAO_ERR_ARG, "null pointer");
  if (offsets ? bias || residual : up != nullptr)
    return pfail(TAO_ERR_ARG, "experts have no bias or residual, and a gate needs experts");
  if (!on_elements({{bias, 2}, {residual, 2}, {y, 2}, {z, 2}, {u, 2}}))
    return pfail(TAO_ERR_ARG, "operands start on a whole element");
  const Operand2 ox = {x, k, rows, x_stride, 1, 0}, ow = {w, k, n, w_stride, experts, w_expert},
                 ou = {up, k, n, up_stride, experts, up_expert}, none = {};
  if (!laid(ox) || !laid(ow) || !laid(ou))
    return pfail(TAO_ERR_ARG, "operands of a 16-bit product and their rows start on 16 bytes");
  Args a = {};
  a.offsets = offsets, a.groups = experts, a.rows = (int)rows, a.cols = n, a.depth = k, a.pairs = 1;
  a.type = type, a.act = activation, a.bias = bias, a.residual = residual, a.r_stride = r_stride;
  a.y = y, a.z = z, a.u = z ? u : nullptr, a.z_stride = z_stride;
  a.wide = n % 8 == 0 && on16(y, 0) && on16(z, z_stride) && on16(u, 0) && on16(residual, r_stride);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int blocks = (k + kTerms - 1) / kTerms;
  if (offsets) {
    const long long mean = rows / experts;
    const Operands few = {ow, ox, ou, none}, many = {ox, ow, none, ou};
    if (up) {
      if (mean <= 32) return start<FEW, 32, true, false>(few, a, 1, s);
      return start<FORWARD, 256, true, false>(many, a, 1, s);
    }
    if (mean <= 32) return start<FEW, 32, false, false>(few, a, 1, s);
    return start<FORWARD, 256, false, false>(many, a, 1, s);
  }
  if (rows <= 64) {
    const Operands o = {ow, ox, none, none};
    const int split = split_of((n + 127) / 128, blocks);
    if (rows <= 16) return start<FEW, 16, false, true>(o, a, split, s);
    if (rows <= 32) return start<FEW, 32, false, true>(o, a, split, s);
    return start<FEW, 64, false, true>(o, a, split, s);
  }
  const Operands o = {ox, ow, none, none};
  const long long row_tiles = (rows + 127) / 128;
  if (row_tiles * ((n + 255) / 256) >= 120) return start<FORWARD, 256, false, false>(o, a, 1, s);
  if (row_tiles * ((n + 127) / 128) >= 100) return start<FORWARD, 128, false, false>(o, a, 1, s);
  return start<FORWARD, 64, false, true>(o, a, split_of(row_tiles * ((n + 63) / 64), blocks), s);
}

int tao_linear_input_gradient(const void* dz, const void* du, long long d_stride, const void* w, long long w_stride,
                              long long w_expert, const void* up, long long up_stride, long long up_expert,
                              const int* offsets, int experts, long long rows, int n, int k, int type, void* dx,
                              void* stream) {
  using namespace tao;
  using namespace tao::product;
  if (int rc = check_sizes(rows, n, k, type, TAO_ACT_NONE, offsets, experts)) return rc;
  if (rows == 0) return TAO_OK;
  if (!dz || !w || !dx || !du != !up) return pfail(TAO_ERR_ARG, "null pointer");
  if (!on_elements({{dx, 2}})) return pfail(TAO_ERR_ARG, "operands start on a whole element");
  const Operand2 oz = {dz, n, rows, d_stride, 1, 0}, od = {du, n, rows, d_stride, 1, 0},
                 ow = {w, k, n, w_stride, experts, w_expert}, ou = {up, k, n, up_stride, experts, up_expert};
  if (!laid(oz) || !laid(od) || !laid(ow) || !laid(ou))
    return pfail(TAO_ERR_ARG, "operands of a 16-bit product and their rows start on 16 bytes");
  Args a = {};
  a.offsets = offsets, a.groups = experts, a.rows = (int)rows, a.cols = k, a.depth = n, a.pairs = du ? 2 : 1;
  a.type = type, a.y = dx;
  a.wide = k % 8 == 0 && on16(dx, 0);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Operands o = {oz, ow, od, ou};
  const int blocks = (n + kTerms - 1) / kTerms * a.pairs;
  const long long row_tiles = (rows + 127) / 128 + (offsets ? experts / 2 : 0);
  if (row_tiles * ((k + 255) / 256) >= 120) return start<INPUT, 256, false, false>(o, a, 1, s);
  if (offsets || row_tiles * ((k + 127) / 128) >= 100) return start<INPUT, 128, false, false>(o, a, 1, s);
  return start<INPUT, 64, false, true>(o, a, split_of(row_tiles * ((k + 63) / 64), blocks), s);
}

int tao_linear_weight_gradient(const void* dz, const void* du, long long d_stride, const void* x, long long x_stride,
                               const int* offsets, int experts, long long rows, int n, int k, int type, void* dw,
                               void* dup, void* stream) {
  using namespace tao;
  using namespace tao::product;
  if (int rc = check_sizes(rows, n, k, type, TAO_ACT_NONE, offsets, experts)) return rc;
  if (!dw || !du != !dup) return pfail(TAO_ERR_ARG, "null pointer");
  if (!on_elements({{dw, 2}, {dup, 2}})) return pfail(TAO_ERR_ARG, "operands start on a whole element");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    const size_t size = (size_t)experts * n * k * 2;
    cudaError_t e = cudaMemsetAsync(dw, 0, size, s);
    if (e == cudaSuccess && dup) e = cudaMemsetAsync(dup, 0, size, s);
    return e == cudaSuccess ? TAO_OK : pfail(TAO_ERR_CUDA, cudaGetErrorString(e));
  }
  if (!dz || !x) return pfail(TAO_ERR_ARG, "null pointer");
  const Operand2 oz = {dz, n, rows, d_stride, 1, 0}, od = {du, n, rows, d_stride, 1, 0},
                 ox = {x, k, rows, x_stride, 1, 0}, none = {};
  if (!laid(oz) || !laid(od) || !laid(ox))
    return pfail(TAO_ERR_ARG, "operands of a 16-bit product and their rows start on 16 bytes");
  Args a = {};
  a.offsets = offsets, a.groups = experts, a.rows = (int)rows, a.cols = k, a.depth = n, a.pairs = du ? 2 : 1;
  a.type = type, a.y = dw, a.u = dup;
  a.wide = k % 8 == 0 && on16(dw, 0) && on16(dup, 0);
  const Operands o = {oz, ox, od, none};
  const long long down = (long long)(n + 127) / 128 * experts * a.pairs;
  if (down * ((k + 255) / 256) >= 120) return start<WEIGHT, 256, false, false>(o, a, 1, s);
  const int blocks = (int)std::min<long long>((rows + kTerms - 1) / kTerms, 1 << 20);
  if (offsets) return start<WEIGHT, 128, false, false>(o, a, 1, s);
  const long long tiles = down * ((k + 127) / 128);
  if (tiles >= 100) return start<WEIGHT, 128, false, false>(o, a, 1, s);
  return start<WEIGHT, 128, false, true>(o, a, split_of(tiles, blocks), s);
}

size_t tao_linear_slope_workspace_bytes(long long rows, int n) {
  if (rows <= 0 || n <= 0) return 0;
  return (size_t)tao::product::slope_blocks(rows, n) * n * sizeof(float);
}

int tao_linear_slope(const void* dy, long long dy_stride, const void* z, const void* u, long long z_stride,
                     long long rows, int n, int type, int activation, void* dz, void* du, long long d_stride, void* db,
                     void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tao;
  using namespace tao::product;
  if (int rc = check_sizes(rows, n, 1, type, activation, nullptr, 1)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (db && cudaMemsetAsync(db, 0, (size_t)n * 2, s) != cudaSuccess)
      return pfail(TAO_ERR_CUDA, cudaGetErrorString(cudaGetLastError()));
    return TAO_OK;
  }
  if (!dy || (u && (!z || !du)) || (z && !dz) || (!dz && !db)) return pfail(TAO_ERR_ARG, "null pointer");
  if (!on_elements({{dy, 2}, {z, 2}, {u, 2}, {dz, 2}, {du, 2}, {db, 2}, {workspace, 4}}))
    return pfail(TAO_ERR_ARG, "operands start on a whole element");
  if (db && (!workspace || workspace_bytes < tao_linear_slope_workspace_bytes(rows, n)))
    return pfail(TAO_ERR_ARG, "workspace too small for the bias's gradient");
  SlopeArgs a = {dy, z, u, dy_stride, z_stride, d_stride, dz, du, db ? static_cast<float*>(workspace) : nullptr,
                 rows, n, type, activation, slope_rows(rows, n)};
  const bool wide = n % 8 == 0 && on16(dy, dy_stride) && on16(z, z_stride) && on16(u, 0) && on16(dz, d_stride) && on16(du, 0);
  const int blocks = slope_blocks(rows, n), slab = wide ? 256 : 32;
  const dim3 grid((n + slab - 1) / slab, blocks);
  if (wide)
    slope_kernel<8><<<grid, 256, 0, s>>>(a);
  else
    slope_kernel<1><<<grid, 256, 0, s>>>(a);
  if (db) column_sum_kernel<<<(n + 31) / 32, 256, 0, s>>>(a.sums, blocks, n, type, db);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TAO_OK : pfail(TAO_ERR_CUDA, cudaGetErrorString(e));
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
