// Root-mean-square norm with the residual's addition, the form between two halves of a
// decoder block, with a 16/32-bit or an e4m3 output, and its gradient.
//
//   s = round(x + residual)          the stream the next block adds to (rounded to its type)
//   n = s r,  r = rsqrt(mean(s^2) + eps)
//   y = n w                          or q = e4m3(y * 448 / m), scale = m / 448,
//                                    m = max(max|y|, 1e-30) over a row or 128 channels
//   dx = ds + r (w dy - n mean(w dy n)),   dw = sum over rows of dy n
//
// The norm is taken of the rounded s, so that the forward and the gradient see the same
// stream and the gradient needs no copy of x and residual.  All sums are in fp32.
//
// HBM-bound: each element is read and written once.  A row's threads keep it between the sum and the
// scaling in its own type (half the registers of floats, so twice the rows in flight): V vectors of 16
// bytes a thread, or V elements where rows do not start on 16 bytes.
// Of bf16 with a residual: 16384x2048 takes 43.7 us (6.1 TB/s, a copy's rate is 6.5), 32768x768 37.5 (5.3); to e4m3
// 16384x2048 52 us (4.5 TB/s), where the largest value's reduction and the conversions stand between the loads and
// the stores; forward and gradient of 32768x768 78 us (5.2 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/tao_b200.h"
#include "common.cuh"

void tao_set_last_error(const char* msg);

namespace tao {
namespace {

constexpr float kE4m3Max = 448.f, kTiny = 1e-30f;

template <class T> TAO_DEVI float to_f(T x);
template <> TAO_DEVI float to_f<bf16>(bf16 x) { return __bfloat162float(x); }
template <> TAO_DEVI float to_f<__half>(__half x) { return __half2float(x); }
template <> TAO_DEVI float to_f<float>(float x) { return x; }
template <class T> TAO_DEVI T from_f(float x);
template <> TAO_DEVI bf16 from_f<bf16>(float x) { return __float2bfloat16_rn(x); }
template <> TAO_DEVI __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> TAO_DEVI float from_f<float>(float x) { return x; }

// N neighbouring elements of a row in their own type: 16 bytes, or one element.
template <class T, int N>
struct alignas(N * sizeof(T)) Vec {
  T e[N];
  TAO_DEVI void load(const T* p) { *this = *reinterpret_cast<const Vec*>(p); }
  // Of what no one reads again soon.
  TAO_DEVI void load_once(const T* p) {
    if constexpr (N * sizeof(T) == 16) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
      *this = *reinterpret_cast<const Vec*>(&v);
    } else {
      load(p);
    }
  }
  TAO_DEVI void store(T* p) const { *reinterpret_cast<Vec*>(p) = *this; }
  TAO_DEVI void zero() {
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = from_f<T>(0.f);
  }
  TAO_DEVI float at(int i) const { return to_f<T>(e[i]); }
  // Forgets the floats that were made of it, so that they take no registers until they are made again.
  TAO_DEVI void forget() {
    if constexpr (sizeof(T) == 2 && N > 1) {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) asm volatile("" : "+r"(reinterpret_cast<uint32_t*>(e)[i]));
    }
  }
  // Two at a time where the type has a conversion of pairs.
  TAO_DEVI void set(const float (&f)[N]) {
    if constexpr (N % 2 == 0 && sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        if constexpr (std::is_same<T, bf16>::value)
          *reinterpret_cast<__nv_bfloat162*>(e + i) = __floats2bfloat162_rn(f[i], f[i + 1]);
        else
          *reinterpret_cast<__half2*>(e + i) = __floats2half2_rn(f[i], f[i + 1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = from_f<T>(f[i]);
    }
  }
  static TAO_DEVI void store_e4m3(uint8_t* p, const float (&f)[N]) {
    if constexpr (N == 1) {
      *p = __nv_cvt_float_to_fp8(f[0], __NV_SATFINITE, __NV_E4M3);
    } else {
      uint32_t w[N / 4];
#pragma unroll
      for (int i = 0; i < N / 4; ++i)
        w[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i], f[4 * i + 1]), __NV_SATFINITE, __NV_E4M3) |
               (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f[4 * i + 2], f[4 * i + 3]), __NV_SATFINITE, __NV_E4M3)
                   << 16;
      if constexpr (N == 8)
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
      else
        *reinterpret_cast<uint32_t*>(p) = w[0];
    }
  }
};

// Sum (or maximum) over the threads of a row: blockDim.x of them; more than one warp only
// where the block holds one row.  `red` has 32 floats for each value of the call's.
template <int COUNT, bool MAX = false>
TAO_DEVI void row_reduce(float (&v)[COUNT], float* red) {
#pragma unroll
  for (int c = 0; c < COUNT; ++c) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, v[c], o);
      v[c] = MAX ? max_nan(v[c], other) : v[c] + other;
    }
  }
  if (blockDim.x == 32) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  __syncthreads();  // the last call's reads of `red` are over
  if (lane == 0) {
#pragma unroll
    for (int c = 0; c < COUNT; ++c) red[c * 32 + warp] = v[c];
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < COUNT; ++c) {
    float t = lane < warps ? red[c * 32 + lane] : 0.f;  // maxima are of magnitudes
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, t, o);
      t = MAX ? max_nan(t, other) : t + other;
    }
    v[c] = t;
  }
}

struct NormArgs {
  const void *x, *residual, *weight;
  long long x_stride, r_stride, rows;
  int width, group;  // group: 0 = one scale a row, 128 = one for 128 channels
  float eps, per_width;  // per_width: 1 / width
  void *s, *y;
  float* scale;
};

// MAXT: most threads of a block; registers for four blocks of 256 an SM (three with the second scaling).
template <class T, int N, int V, bool FP8, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT > 256 ? 1 : FP8 ? 3 : 4) norm_kernel(const NormArgs a) {
  using Ve = Vec<T, N>;
  __shared__ float red[32];
  const int width = a.width, step = blockDim.x * N;
  const T* weight = static_cast<const T*>(a.weight);
  for (long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y; row < a.rows;
       row += (long long)gridDim.x * blockDim.y) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const int at0 = threadIdx.x * N;
    Ve v[V];
    float sum[1] = {0.f};
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[i].zero();
      if (at0 + i * step < width) v[i].load_once(x + at0 + i * step);
    }
    if (a.residual) {
      const T* res = static_cast<const T*>(a.residual) + row * a.r_stride;
      T* s = static_cast<T*>(a.s) + row * width;
      Ve r[V];
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (at0 + i * step < width) r[i].load_once(res + at0 + i * step);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (at0 + i * step < width) {
          float f[N];
#pragma unroll
          for (int j = 0; j < N; ++j) f[j] = v[i].at(j) + r[i].at(j);
          v[i].set(f);
          v[i].store(s + at0 + i * step);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) sum[0] += v[i].at(j) * v[i].at(j);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i].forget();
    row_reduce(sum, red);
    const float r = rsqrtf(sum[0] * a.per_width + a.eps);
    // y of vector i, zeros beyond the row
    auto scaled = [&](int i, float(&f)[N]) {
      Ve w;
      w.zero();
      if (weight && at0 + i * step < width) w.load(weight + at0 + i * step);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = v[i].at(j) * r * (weight ? w.at(j) : 1.f);
    };
    if constexpr (!FP8) {
      T* y = static_cast<T*>(a.y) + row * width;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float f[N];
        scaled(i, f);
        v[i].set(f);
        if (at0 + i * step < width) v[i].store(y + at0 + i * step);
      }
    } else {
      uint8_t* q = static_cast<uint8_t*>(a.y) + row * width;
      float f[V][N], up[V];  // up: the largest magnitude, then 448 / it
#pragma unroll
      for (int i = 0; i < V; ++i) {
        scaled(i, f[i]);
        up[i] = 0.f;
#pragma unroll
        for (int j = 0; j < N; ++j) up[i] = max_nan(up[i], fabsf(f[i][j]));
      }
      if (a.group == 0) {
        float m[1] = {up[0]};
#pragma unroll
        for (int i = 1; i < V; ++i) m[0] = max_nan(m[0], up[i]);
        row_reduce<1, true>(m, red);
        m[0] = max_nan(m[0], kTiny);
        if (threadIdx.x == 0) a.scale[row] = m[0] / kE4m3Max;
        m[0] = kE4m3Max / m[0];
#pragma unroll
        for (int i = 0; i < V; ++i) up[i] = m[0];
      } else {
        // 128 channels are 128 / N neighbouring threads of the same vector index, or (N 1) four warps
        const int groups = (width + 127) / 128;
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
          for (int o = N == 1 ? 16 : 64 / N; o > 0; o >>= 1)
            up[i] = max_nan(up[i], __shfl_xor_sync(0xffffffffu, up[i], o));
          if constexpr (N == 1) {
            __syncthreads();
            if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = up[i];
            __syncthreads();
            const int first = threadIdx.x / 128 * 4;
#pragma unroll
            for (int w = 0; w < 4; ++w) up[i] = max_nan(up[i], red[first + w]);
          }
          up[i] = max_nan(up[i], kTiny);
          const int at = at0 + i * step;
          if (at < width && at % 128 == 0) a.scale[row * groups + at / 128] = up[i] / kE4m3Max;
          up[i] = kE4m3Max / up[i];
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int j = 0; j < N; ++j) f[i][j] *= up[i];
        if (at0 + i * step < width) Ve::store_e4m3(q + at0 + i * step, f[i]);
      }
    }
  }
}

struct NormGradArgs {
  const void *dy, *ds, *s, *weight;
  long long dy_stride, ds_stride, s_stride, rows;
  int width;
  float eps, per_width;
  void* dx;
  float* partial;  // [gridDim.x][width] sums of dy n over a block's rows, or null
};

// A block walks over rows with its columns' part of dw in registers; a row's dy and s come while the one
// before is computed.
template <class T, int N, int V, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT > 256 ? 1 : 2) norm_grad_kernel(const NormGradArgs a) {
  using Ve = Vec<T, N>;
  extern __shared__ float sh[];  // 64 floats, then (one-warp rows) [blockDim.y][width padded]
  const int width = a.width, step = blockDim.x * N, at0 = threadIdx.x * N;
  const long long stride = (long long)gridDim.x * blockDim.y;
  float dw[V][N];
  Ve w[V], g[V], v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float one[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      dw[i][j] = 0.f;
      one[j] = 1.f;
    }
    w[i].set(one);
    if (a.weight && at0 + i * step < width) w[i].load(static_cast<const T*>(a.weight) + at0 + i * step);
  }
  auto load = [&](long long row) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      g[i].zero();
      v[i].zero();
      if (row < a.rows && at0 + i * step < width) {
        v[i].load_once(static_cast<const T*>(a.s) + row * a.s_stride + at0 + i * step);
        g[i].load_once(static_cast<const T*>(a.dy) + row * a.dy_stride + at0 + i * step);
      }
    }
  };
  long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  load(row);
  for (; row < a.rows; row += stride) {
    Ve d[V];
    if (a.ds) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (at0 + i * step < width)
          d[i].load_once(static_cast<const T*>(a.ds) + row * a.ds_stride + at0 + i * step);
    }
    float sum[2] = {0.f, 0.f};  // of s^2 and of w dy s
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        sum[0] += v[i].at(j) * v[i].at(j);
        sum[1] += w[i].at(j) * g[i].at(j) * v[i].at(j);
      }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[i].forget();
      g[i].forget();
      w[i].forget();
    }
    row_reduce(sum, sh);
    const float r = rsqrtf(sum[0] * a.per_width + a.eps);
    const float c = r * r * sum[1] * a.per_width;  // dx = ds + r (w dy - s c)
    T* dx = static_cast<T*>(a.dx) + row * width;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (at0 + i * step < width) {
        float f[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float gj = g[i].at(j), vj = v[i].at(j);
          dw[i][j] += gj * (vj * r);
          f[j] = (a.ds ? d[i].at(j) : 0.f) + r * (w[i].at(j) * gj - vj * c);
        }
        d[i].set(f);
      }
    }
    load(row + stride);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (at0 + i * step < width) d[i].store(dx + at0 + i * step);
  }
  if (!a.partial) return;
  float* out = a.partial + (long long)blockIdx.x * width;
  if (blockDim.y == 1) {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (at0 + i * step + j < width) out[at0 + i * step + j] = dw[i][j];
    return;
  }
  // one warp a row: the warps' parts are added in order through shared memory
  float* mine = sh + 64 + threadIdx.y * (V * 32 * N);
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) mine[at0 + i * step + j] = dw[i][j];
  __syncthreads();
  for (int c = threadIdx.y * 32 + threadIdx.x; c < width; c += 32 * blockDim.y) {
    float t = 0.f;
    for (int y = 0; y < blockDim.y; ++y) t += sh[64 + y * (V * 32 * N) + c];
    out[c] = t;
  }
}

// dw = sum of the blocks' parts: a column per lane, 32 warps share the parts.
template <class T>
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float* partial, int parts, int width, T* dw) {
  __shared__ float sh[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float t = 0.f;
  if (c < width)
    for (int p = threadIdx.y; p < parts; p += 32) t += partial[(long long)p * width + c];
  sh[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  t = warp_sum(sh[threadIdx.x][threadIdx.y]);  // warp y adds column y's 32 sums
  if (threadIdx.x == 0 && blockIdx.x * 32 + threadIdx.y < width) dw[blockIdx.x * 32 + threadIdx.y] = from_f<T>(t);
}

// Threads a row, rows a block and vectors (of `elements`) a thread.
struct Shape {
  int threads, rows, vectors;
};

// Measured in bf16 with a residual (us):
//  - rows whose vectors all fit the device at once, half full: a thread a vector, for latency.  64x768 2.3 (a warp
//    a row 3.5), 592x2048 3.2 (two vectors 3.4); above that 1184x8192 21.2 (14.1).
//  - 65 to 128 vectors: a thread a vector.  32768x768 37.5 (a warp a row 41.5); below, 32768x384 21.8 (18.4).
//    The e4m3 form needs the rows' largest values too, which a warp finds alone: 32768x768 49.3 (40.7).
//  - more: two vectors a thread.  16384x2048 43.7 (one 50.5), 16384x8192 177.7 (one 283, four 229).
//  - the gradient of 513 to 1024 vectors, whose two vectors a thread leave one block of 512 threads an SM:
//    forward and backward of 4096x8192 118 (167); of 4096 elements 136 (109).
Shape shape_of(long long rows, int width, int elements, bool fp8, bool grad) {
  const int vectors = (width + elements - 1) / elements;
  const bool fit = vectors <= 1024 && rows * vectors <= 148 * 1024;
  if (grad ? vectors > 512 && vectors <= 1024 : fit || (!fp8 && vectors > 64 && vectors <= 128))
    return {(vectors + 31) / 32 * 32, 1, 1};
  if (vectors <= 128) return {32, 8, (vectors + 31) / 32};
  int threads = 128;
  while (threads < 1024 && vectors > 2 * threads) threads *= 2;
  const int v = (vectors + threads - 1) / threads;
  return {threads, 1, v <= 4 ? v : v <= 8 ? 8 : v <= 32 ? 32 : 64};
}

int nfail(int code, const char* msg) {
  tao_set_last_error(msg);
  return code;
}

int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TAO_OK : nfail(TAO_ERR_CUDA, cudaGetErrorString(e));
}

size_t size_of(int type) { return type == TAO_TYPE_FP32 ? 4 : 2; }

// Whether rows of this base and stride start on 16 bytes (an absent operand does).
bool wide_ok(const void* p, long long stride, size_t size) {
  return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * (long long)size % 16 == 0);
}

int check(long long rows, int width, int type) {
  if (type != TAO_TYPE_BF16 && type != TAO_TYPE_FP16 && type != TAO_TYPE_FP32)
    return nfail(TAO_ERR_ARG, "the norm takes bf16, fp16 or fp32");
  if (rows < 0 || width <= 0) return nfail(TAO_ERR_ARG, "rows must not be negative and the width must be positive");
  if (width > (type == TAO_TYPE_FP32 ? 32768 : 65536))
    return nfail(TAO_ERR_ARG, "the norm's width is limited to 65536 (32768 in fp32)");
  return TAO_OK;
}

template <int N>
using Int = std::integral_constant<int, N>;

// f(vectors, most threads) as compile-time constants; WIDE: vectors of 16 bytes (their most is 8 a thread).
template <bool WIDE, class F>
int by_shape(const Shape& sh, F f) {
  if (sh.threads * sh.rows <= 256) {
    switch (sh.vectors) {
      case 1: return f(Int<1>(), Int<256>());
      case 2: return f(Int<2>(), Int<256>());
      case 3: return f(Int<3>(), Int<256>());
      case 4: return f(Int<4>(), Int<256>());
    }
    return nfail(TAO_ERR_ARG, "width");
  }
  switch (sh.vectors) {
    case 1: return f(Int<1>(), Int<1024>());
    case 2: return f(Int<2>(), Int<1024>());
    case 3:
    case 4: return f(Int<4>(), Int<1024>());
    case 8: return f(Int<8>(), Int<1024>());
  }
  if constexpr (!WIDE) {
    if (sh.vectors == 32) return f(Int<32>(), Int<1024>());
    return f(Int<64>(), Int<1024>());
  }
  return nfail(TAO_ERR_ARG, "width");
}

template <class F>
int by_type(int type, F f) {
  if (type == TAO_TYPE_BF16) return f(bf16());
  if (type == TAO_TYPE_FP16) return f(__half());
  return f(float());
}

constexpr int kMaxBlocks = 1 << 30;

// f(element type, elements of a vector) as compile-time constants.
template <class F>
int by_vector(int type, bool wide, F f) {
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    return wide ? f(t, Int<16 / sizeof(T)>()) : f(t, Int<1>());
  });
}

int forward(const NormArgs& a, int type, bool fp8, void* stream) {
  const size_t size = size_of(type);
  const bool wide = a.width % (16 / size) == 0 && wide_ok(a.x, a.x_stride, size) &&
                    wide_ok(a.residual, a.r_stride, size) && wide_ok(a.weight, 0, size) && wide_ok(a.s, 0, size) &&
                    wide_ok(a.y, 0, size);
  Shape sh = shape_of(a.rows, a.width, wide ? (int)(16 / size) : 1, fp8, false);
  // single elements: 128 channels are four whole warps of a block
  if (fp8 && a.group && !wide && sh.threads % 128) sh = {128, 1, (a.width + 127) / 128};
  if (!wide && sh.vectors > 4 && sh.threads < 256) sh = {256, 1, 4};
  const unsigned grid = (unsigned)std::min<long long>((a.rows + sh.rows - 1) / sh.rows, kMaxBlocks);
  const dim3 block(sh.threads, sh.rows);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_vector(type, wide, [&](auto t, auto n) {
    using T = decltype(t);
    constexpr int N = decltype(n)::value;
    return by_shape<(N > 1)>(sh, [&](auto v, auto most) {
      if (fp8)
        norm_kernel<T, N, decltype(v)::value, true, decltype(most)::value><<<grid, block, 0, st>>>(a);
      else
        norm_kernel<T, N, decltype(v)::value, false, decltype(most)::value><<<grid, block, 0, st>>>(a);
      return launched();
    });
  });
}

// Blocks of the gradient kernel: two of 256 threads an SM, as its registers allow.
int grad_blocks(long long rows, const Shape& sh) {
  const long long need = (rows + sh.rows - 1) / sh.rows;
  const int resident = 148 * std::max(1, 512 / (sh.threads * sh.rows));
  return (int)std::min<long long>(need, resident);
}

}  // namespace
}  // namespace tao

extern "C" {

int tao_add_rms_norm(const void* x, long long x_stride, const void* residual, long long r_stride, const void* weight,
                     long long rows, int width, int type, float eps, void* s, void* y, void* stream) {
  using namespace tao;
  if (int rc = check(rows, width, type)) return rc;
  if (rows == 0) return TAO_OK;
  if (!x || !y || (residual && !s)) return nfail(TAO_ERR_ARG, "null pointer");
  const size_t size = size_of(type);
  if (!on_elements({{x, size}, {residual, size}, {weight, size}, {s, size}, {y, size}}))
    return nfail(TAO_ERR_ARG, "operands start on a whole element");
  return forward({x, residual, weight, x_stride, r_stride, rows, width, 0, eps, 1.f / width, s, y, nullptr}, type, false,
                 stream);
}

int tao_add_rms_norm_fp8(const void* x, long long x_stride, const void* residual, long long r_stride,
                         const void* weight, long long rows, int width, int type, float eps, int group, void* s,
                         void* q, float* scale, void* stream) {
  using namespace tao;
  if (int rc = check(rows, width, type)) return rc;
  if (group != 0 && group != 128) return nfail(TAO_ERR_ARG, "8-bit scales are by row (0) or by 128 channels");
  if (rows == 0) return TAO_OK;
  if (!x || !q || !scale || (residual && !s)) return nfail(TAO_ERR_ARG, "null pointer");
  const size_t size = size_of(type);
  if (!on_elements({{x, size}, {residual, size}, {weight, size}, {s, size}, {scale, sizeof(float)}}))
    return nfail(TAO_ERR_ARG, "operands start on a whole element");
  return forward({x, residual, weight, x_stride, r_stride, rows, width, group, eps, 1.f / width, s, q, scale}, type, true,
                 stream);
}

size_t tao_add_rms_norm_workspace_bytes(long long rows, int width, int type) {
  using namespace tao;
  if (check(rows, width, type) != TAO_OK || rows == 0) return 0;
  // of the shape with the more blocks
  const int blocks = std::max(grad_blocks(rows, shape_of(rows, width, (int)(16 / size_of(type)), false, true)),
                              grad_blocks(rows, shape_of(rows, width, 1, false, true)));
  return (size_t)blocks * width * sizeof(float);
}

int tao_add_rms_norm_backward(const void* dy, long long dy_stride, const void* ds, long long ds_stride, const void* s,
                              long long s_stride, const void* weight, long long rows, int width, int type, float eps,
                              void* dx, void* dw, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tao;
  if (int rc = check(rows, width, type)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t size = size_of(type);
  if (rows == 0) {
    if (dw && cudaMemsetAsync(dw, 0, width * size, st) != cudaSuccess) return launched();
    return TAO_OK;
  }
  if (!dy || !s || !dx) return nfail(TAO_ERR_ARG, "null pointer");
  if (!on_elements({{dy, size}, {ds, size}, {s, size}, {weight, size}, {dx, size}, {dw, size}, {workspace, sizeof(float)}}))
    return nfail(TAO_ERR_ARG, "operands start on a whole element");
  if (dw && (!workspace || workspace_bytes < tao_add_rms_norm_workspace_bytes(rows, width, type)))
    return nfail(TAO_ERR_ARG, "workspace too small for the norm's weight gradient");
  const NormGradArgs a = {dy,    ds,  s,  weight, dy_stride, ds_stride, s_stride, rows, width, eps, 1.f / width, dx,
                          dw ? static_cast<float*>(workspace) : nullptr};
  const bool wide = width % (16 / size) == 0 && wide_ok(dy, dy_stride, size) && wide_ok(ds, ds_stride, size) &&
                    wide_ok(s, s_stride, size) && wide_ok(weight, 0, size) && wide_ok(dx, 0, size);
  const Shape sh = shape_of(rows, width, wide ? (int)(16 / size) : 1, false, true);
  const int grid = grad_blocks(rows, sh);
  const dim3 block(sh.threads, sh.rows);
  return by_vector(type, wide, [&](auto t, auto n) {
    using T = decltype(t);
    constexpr int N = decltype(n)::value;
    return by_shape<(N > 1)>(sh, [&](auto v, auto most) {
      constexpr int V = decltype(v)::value;
      const size_t smem = (64 + (sh.rows > 1 ? (size_t)sh.rows * V * 32 * N : 0)) * sizeof(float);
      norm_grad_kernel<T, N, V, decltype(most)::value><<<grid, block, smem, st>>>(a);
      if (int rc = launched()) return rc;
      if (dw) norm_dw_kernel<T><<<(width + 31) / 32, dim3(32, 32), 0, st>>>(a.partial, grid, width, static_cast<T*>(dw));
      return launched();
    });
  });
}

}  // extern "C"
