// What the kernels of the 4-bit product (linear4.cu, linear4_tc.cuh) share: arguments, clusters, x on its way.
#pragma once
#include <type_traits>

#include "../../include/tao_b200.h"
#include "few_rows.cuh"

namespace tao {

struct Linear4Args {
  Four w;
  const void* x;
  long long x_stride;
  const float* x_scale;  // one a row, or null
  const void* bias;
  void* y;
  int rows, n, k;
  int tiles, kblocks;
  int shift, wk_shift;  // log2 of a cluster's blocks, of a tile's warps
  int ring, sums;   // where the rings and the sums start in shared memory
  int steps;        // row tiles of a warp
  int x_type;
  bool wide;        // rows of x start on 16 (e4m3: 8) bytes and k is whole chunks of 8
};

TAO_DEVI uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
TAO_DEVI void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
TAO_DEVI float4 ld_cluster(uint32_t at, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n .reg .u32 p;\n mapa.shared::cluster.u32 p, %4, %5;\n ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [p];\n}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(at), "r"(rank)
      : "memory");
  return v;
}

// Eight activations of a row from k on (e4m3: in the first two words); zeros beyond its end.
TAO_DEVI uint4 chunk_of(const Linear4Args& a, long long m, int k) {
  const long long at = m * a.x_stride + k;
  uint32_t w[4] = {};
  if (a.x_type == TAO_TYPE_E4M3) {
    const uint8_t* p = static_cast<const uint8_t*>(a.x) + at;
    if (a.wide) {
      if (k < a.k) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
        w[0] = v.x, w[1] = v.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < a.k) w[i / 4] |= (uint32_t)__ldg(p + i) << (8 * (i & 3));
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(a.x) + at;
    if (a.wide) {
      if (k < a.k) return __ldg(reinterpret_cast<const uint4*>(p));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < a.k) w[i / 2] |= (uint32_t)__ldg(p + i) << (16 * (i & 1));
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// ... as pairs of fp16 (from e4m3).
TAO_DEVI uint4 widen_e4m3(uint4 v) {
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t q = (i < 2 ? v.x : v.y) >> (16 * (i & 1)) & 0xffff;
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)q, __NV_E4M3);
    h[i] = r.x | (uint32_t)r.y << 16;
  }
  return make_uint4(h[0], h[1], h[2], h[3]);
}

}  // namespace tao
