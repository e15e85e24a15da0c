// y = x W^T + b for a few rows of x and a 4-bit W with group scales.
//
//   W[n][k] = (code[n][k] - zero[n][k / group]) scale[n][k / group],  codes 0..15
//
// x in bf16 or fp16, or in e4m3 with one fp32 scale a row (read as fp16, exactly); y in
// the type of the weight's scales.  Products of codes are summed in fp32 over a group,
// scaled, and summed in fp32 over the groups; y is rounded once.
//
// Bound by the codes' bytes: half a byte a weight.  A block owns 16 output rows; its
// warps take the 128-k blocks in turn, each through a ring of its own, and add their sums
// in order through shared memory.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/tao_b200.h"
#include "few_rows.cuh"

void tao_set_last_error(const char* msg);

namespace tao {
namespace {

enum Act { kBf16 = 0, kF16 = 1, kE4m3 = 3 };

struct Linear4Args {
  Four w;
  const void* x;
  long long x_stride;
  const float* x_scale;  // one a row, or null
  const void* bias;
  void* y;
  int rows, n, k;
  int kblocks, stages;
  bool wide;      // rows of x start on 16 (e4m3: 8) bytes and k is whole chunks of 8
  bool bf16_out;  // the type of scales, bias and y
};

TAO_DEVI float scale_f(uint32_t bits, bool is_bf16) {
  if (is_bf16) return __uint_as_float(bits << 16);
  return __half2float(__ushort_as_half((unsigned short)bits));
}

constexpr int kWarps = 8;

// Bytes of one stage of a warp's ring: codes, scales, zeros, activations of `rows` rows.
__host__ __device__ constexpr int meta_bytes(int group, bool zeros) { return 128 / group * 16 * (zeros ? 3 : 2); }
__host__ __device__ constexpr int stage_bytes(int group, bool zeros, int rows, int act) {
  return 1024 + meta_bytes(group, zeros) + rows * 128 * (act == kE4m3 ? 1 : 2);
}

template <int ACT, int GROUP, int NT>
__global__ void __launch_bounds__(kWarps * 32) linear4_kernel(const Linear4Args a) {
  using M = std::conditional_t<ACT == kBf16, MmaBf16, MmaF16>;
  constexpr int XB = ACT == kE4m3 ? 1 : 2;  // bytes of an activation
  constexpr int CHUNK = 8 * XB;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tile = blockIdx.x, m0 = blockIdx.y * (8 * NT), rows = min(a.rows - m0, 8 * NT);
  const bool has_zeros = a.w.zeros != nullptr;
  constexpr int SCALES = 128 / GROUP * 32;
  const int zoff = 1024 + SCALES, xoff = 1024 + meta_bytes(GROUP, has_zeros);
  const int xrows = min(a.rows, 8 * NT);  // the ring's room, equal for all blocks
  const int stage = stage_bytes(GROUP, has_zeros, xrows, ACT);
  const uint32_t ring = smem_u32(smem) + warp * a.stages * stage;
  const int mine = a.kblocks > warp ? (a.kblocks - warp + kWarps - 1) / kWarps : 0;
  const uint8_t* x = static_cast<const uint8_t*>(a.x) + (long long)m0 * a.x_stride * XB;

  auto issue = [&](int i) {
    if (i < mine) {
      const int kb = warp + i * kWarps;
      const long long block = (long long)tile * a.kblocks + kb;
      const uint32_t to = ring + (i % a.stages) * stage;
      const uint8_t* src = a.w.codes + block * 1024 + lane * 16;
      cp_async16(to + lane * 16, src, true);
      cp_async16(to + 512 + lane * 16, src + 512, true);
      if (lane < SCALES / 16)
        cp_async16(to + 1024 + lane * 16, reinterpret_cast<const uint8_t*>(a.w.scales) + block * SCALES + lane * 16,
                   true);
      else if (has_zeros && lane >= 16 && lane < 16 + SCALES / 32)
        cp_async16(to + zoff + (lane - 16) * 16, a.w.zeros + block * (SCALES / 2) + (lane - 16) * 16, true);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int m = n * 8 + g;
        if (m < rows) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int k = kb * 128 + u * 32 + t * 8;
            const uint32_t dst = to + xoff + ((u * xrows + m) * 4 + t) * CHUNK;
            const uint8_t* from = x + ((long long)m * a.x_stride + k) * XB;
            if (a.wide) {
              if constexpr (XB == 2)
                cp_async16_l1(dst, k < a.k ? from : x, k < a.k);
              else
                cp_async8_l1(dst, k < a.k ? from : x, k < a.k);
            } else {
              uint32_t v[CHUNK / 4] = {};
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                if (k + e < a.k) {
                  if constexpr (XB == 2)
                    v[e / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(from)[e] << (16 * (e & 1));
                  else
                    v[e / 4] |= (uint32_t)from[e] << (8 * (e & 3));
                }
              }
#pragma unroll
              for (int e = 0; e < CHUNK / 4; ++e)
                asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst + 4 * e), "r"(v[e]) : "memory");
            }
          }
        }
      }
    }
    cp_commit();
  };

  float acc[NT][4] = {};
  for (int i = 0; i < a.stages - 1; ++i) issue(i);
  for (int i = 0; i < mine; ++i) {
    // stages - 2 younger groups may be open; the ring's depth is 2, 4 or 8
    if (a.stages == 2)
      cp_wait<0>();
    else if (a.stages == 4)
      cp_wait<2>();
    else
      cp_wait<6>();
    __syncwarp();  // block i is there for every lane, and every lane is done with block i - 1
    issue(i + a.stages - 1);
    const uint32_t at = ring + (i % a.stages) * stage;
    auto b = [&](int u, int n) {
      const int m = min(n * 8 + g, xrows - 1);  // columns without a row repeat one; nothing reads them
      const uint32_t from = at + xoff + ((u * xrows + m) * 4 + t) * CHUNK;
      if constexpr (XB == 2) {
        return lds16(from);
      } else {
        const uint2 v = lds8(from);
        uint4 r;
        e4m3_to_f16(v.x, r.x, r.y);
        e4m3_to_f16(v.y, r.z, r.w);
        return r;
      }
    };
    auto scale = [&](int j, int row) { return scale_f(lds_u16(at + 1024 + (j * 16 + row) * 2), a.bf16_out); };
    four_block<M, GROUP, 128, NT>(acc, at, at + zoff, has_zeros, lane, rows, b, scale);
  }
  cp_wait<0>();
  __syncthreads();  // the rings become the warps' sums [warp][column][16 rows]
  float* red = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      red[(warp * 8 * NT + n * 8 + 2 * t + (c & 1)) * 16 + g + 8 * (c >> 1)] = acc[n][c];
  __syncthreads();
  for (int i = threadIdx.x; i < rows * 16; i += kWarps * 32) {
    const int m = i / 16, n = tile * 16 + i % 16;
    if (n >= a.n) continue;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += red[(w * 8 * NT + m) * 16 + i % 16];
    if (a.x_scale) s *= a.x_scale[m0 + m];
    const long long at = (long long)(m0 + m) * a.n + n;
    if (a.bf16_out) {
      if (a.bias) s += bf(static_cast<const bf16*>(a.bias)[n]);
      static_cast<bf16*>(a.y)[at] = tobf(s);
    } else {
      if (a.bias) s += __half2float(static_cast<const __half*>(a.bias)[n]);
      static_cast<__half*>(a.y)[at] = __float2half_rn(s);
    }
  }
}

int lfail(int code, const char* msg) {
  tao_set_last_error(msg);
  return code;
}

template <int ACT, int GROUP, int NT>
int launch(const Linear4Args& a, cudaStream_t s) {
  const int xrows = std::min(a.rows, 8 * NT);
  const int smem = std::max(kWarps * a.stages * stage_bytes(GROUP, a.w.zeros != nullptr, xrows, ACT),
                            kWarps * 8 * NT * 16 * 4);
  auto kernel = linear4_kernel<ACT, GROUP, NT>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) {
    const dim3 grid((a.n + 15) / 16, (a.rows + 8 * NT - 1) / (8 * NT));
    kernel<<<grid, kWarps * 32, smem, s>>>(a);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? TAO_OK : lfail(TAO_ERR_CUDA, cudaGetErrorString(e));
}

template <int ACT, int GROUP>
int by_rows(Linear4Args a, cudaStream_t s) {
  if (a.rows <= 8) {
    a.stages = 4;
    return launch<ACT, GROUP, 1>(a, s);
  }
  a.stages = 2;
  return launch<ACT, GROUP, 2>(a, s);
}

template <int ACT>
int by_group(const Linear4Args& a, int group, cudaStream_t s) {
  if (group == 32) return by_rows<ACT, 32>(a, s);
  if (group == 64) return by_rows<ACT, 64>(a, s);
  return by_rows<ACT, 128>(a, s);
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
  if (n > (1 << 24) || k > (1 << 24)) return lfail(TAO_ERR_ARG, "n and k are limited to 2^24");
  if (rows == 0) return TAO_OK;
  if (!x || !codes || !scales || !y) return lfail(TAO_ERR_ARG, "null pointer");
  for (const void* p : {codes, scales, zeros})
    if (reinterpret_cast<uintptr_t>(p) % 16) return lfail(TAO_ERR_ARG, "a laid-out weight starts on 16 bytes");
  const int size = x_type == TAO_TYPE_E4M3 ? 1 : 2;
  constexpr long long kMost = 1 << 19;  // rows of a launch: 65536 blocks of 8 in the grid's second axis, less one
  for (long long at = 0; at < rows; at += kMost - 16) {
    Linear4Args a = {};
    a.w = {static_cast<const uint8_t*>(codes), static_cast<const uint16_t*>(scales),
           static_cast<const uint8_t*>(zeros)};
    a.x = static_cast<const uint8_t*>(x) + at * x_stride * size;
    a.x_stride = x_stride;
    a.x_scale = x_scale ? x_scale + at : nullptr;
    a.bias = bias;
    a.y = static_cast<uint8_t*>(y) + at * n * 2;
    a.rows = (int)std::min(rows - at, kMost - 16);
    a.n = n;
    a.k = k;
    a.kblocks = (k + 127) / 128;
    a.bf16_out = type == TAO_TYPE_BF16;
    a.wide = k % 8 == 0 && reinterpret_cast<uintptr_t>(a.x) % (8 * size) == 0 && x_stride % 8 == 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int rc = x_type == TAO_TYPE_E4M3 ? by_group<kE4m3>(a, group, s)
                   : x_type == TAO_TYPE_BF16 ? by_group<kBf16>(a, group, s)
                                             : by_group<kF16>(a, group, s);
    if (rc) return rc;
  }
  return TAO_OK;
}

}  // extern "C"
