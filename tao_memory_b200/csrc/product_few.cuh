// y = act(x W^T + bias) + residual for a few rows of x (up to 32): the time is the time to read W.
//
// A block computes 16 outputs of every row; its warps share out the terms, 32 at a time in turn, and add their
// sums through shared memory in the warps' order.  A lane reads 16 bytes of a row of W and of the row 8 below, 16
// bytes of a row of x for each eight rows, all of its loads of a round at once, and gives them to mma.m16n8k16 as they
// are: the order of the terms inside a product is free, as long as both operands use the same (lane (g, t) has terms
// 8t .. 8t + 7 of 32).  So there is no shared memory, no barrier and no copy engine between memory and the tensor
// cores, and all of W is on its way at once.  1x2048x6144 takes 5.9 us (its bytes 3.9), 1x8192x8192 24.9 (20.5),
// 16x8192x2048 11.8 (5.1), 24x8192x2048 14.9; with 128-row tcgen05 tiles, a ring and clusters that add their parts the first
// took 14.4 us.  Of long rows each warp's rounds of loads bound it, and from 17 rows on x, read from L2 by every block.
#pragma once
#include "product.cuh"

namespace tao {
namespace product {

struct FewArgs {
  const void *x, *w, *bias, *residual;
  long long x_stride, w_stride, r_stride;
  int rows, n, k, act;
  void *y, *z;
  long long z_stride;
};

// Terms k .. k + 7 of a row of `depth`; zeros beyond (what lies there is not read).
TAO_DEVI uint4 terms(const uint16_t* row, int k, int depth) {
  if (k + 8 <= depth) {
    uint4 v;
    asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(row + k));
    return v;
  }
  if (k >= depth) return make_uint4(0, 0, 0, 0);
  uint32_t w[4] = {};
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (k + i < depth) w[i / 2] |= (uint32_t)row[k + i] << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// The same of a weight, which is read once: not kept in L1.
TAO_DEVI uint4 weight_terms(const uint16_t* row, int k, int depth) {
  if (k + 8 <= depth) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(row + k));
    return v;
  }
  return terms(row, k, depth);
}

// EIGHTS: eights of rows of x.  AHEAD: rounds whose loads are on their way at once.
template <int EIGHTS, int WARPS, int AHEAD, bool BF16>
__global__ void __launch_bounds__(32 * WARPS) few_kernel(const FewArgs a) {
  using M = std::conditional_t<BF16, MmaBf16, MmaF16>;
  __shared__ float sums[WARPS][EIGHTS * 8][17];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16;
  const uint16_t* const w0 = static_cast<const uint16_t*>(a.w) + min(n0 + g, a.n - 1) * a.w_stride;
  const uint16_t* const w1 = static_cast<const uint16_t*>(a.w) + min(n0 + g + 8, a.n - 1) * a.w_stride;
  const uint16_t* xs[EIGHTS];
#pragma unroll
  for (int e = 0; e < EIGHTS; ++e) xs[e] = static_cast<const uint16_t*>(a.x) + min(e * 8 + g, a.rows - 1) * a.x_stride;
  float acc[EIGHTS][4] = {};
  const int rounds = (a.k + 31) / 32;
  for (int r0 = warp; r0 < rounds; r0 += WARPS * AHEAD) {
    uint4 u[AHEAD], v[AHEAD], x[AHEAD][EIGHTS];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int k = (r0 + j * WARPS) * 32 + 8 * t;
      u[j] = weight_terms(w0, k, a.k);
      v[j] = weight_terms(w1, k, a.k);
#pragma unroll
      for (int e = 0; e < EIGHTS; ++e) x[j][e] = terms(xs[e], k, a.k);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const uint32_t first[4] = {u[j].x, v[j].x, u[j].y, v[j].y}, second[4] = {u[j].z, v[j].z, u[j].w, v[j].w};
#pragma unroll
      for (int e = 0; e < EIGHTS; ++e) {
        M::mma(acc[e], first, x[j][e].x, x[j][e].y);
        M::mma(acc[e], second, x[j][e].z, x[j][e].w);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < EIGHTS; ++e) {
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[warp][e * 8 + 2 * t + (i & 1)][g + (i >> 1) * 8] = acc[e][i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < EIGHTS * 8 * 16; i += 32 * WARPS) {
    const int row = i >> 4, c = i & 15, col = n0 + c;
    if (row >= a.rows || col >= a.n) continue;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) s += sums[w][row][c];
    if (a.bias) s += load1(a.bias, col, BF16);
    if (a.z) static_cast<uint16_t*>(a.z)[row * a.z_stride + col] = pack1(s, BF16);
    s = activate(s, a.act);
    if (a.residual) s += load1(a.residual, row * a.r_stride + col, BF16);
    static_cast<uint16_t*>(a.y)[(long long)row * a.n + col] = pack1(s, BF16);
  }
}

}  // namespace product
}  // namespace tao
