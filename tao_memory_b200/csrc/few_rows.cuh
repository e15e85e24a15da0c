// Products of a few activation rows with a large weight matrix: the device parts that
// the 4-bit product and the expert layer share.
//
//   D[n][m] += sum over k of W[n][k] x[m][k]
//
// The weights are the 16-row operand of mma.m16n8k16 and eight activation rows its
// columns, so a weight is used once per eight rows with no conversion to fp32; with one
// row the other seven columns compute values that nothing reads.  The work is bound by
// the weights' bytes, far from where tcgen05 tiles (128 rows, operands through shared
// memory, where 4-bit weights would first have to be written as 16 bits) would pay.
//
// The order of k inside a product is free, as long as both operands use the same:  of
// every 32 k lane (g, t) = (lane / 4, lane % 4) takes 8t..8t+7, the first four in one
// mma and the last four in the next.  So a lane reads 16 contiguous bytes of an
// activation row (and of a 16-bit weight row).  A 4-bit block of 16 rows x 128 k is
// laid out so that a lane's 64 codes are two 16-byte words:  word j of half h is the mma
// step 4h + j, and its nibble i + 4p holds element p (low, high) of operand register i.
//
// Each warp streams its blocks through a ring in shared memory filled by cp.async.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "common.cuh"

namespace tao {

TAO_DEVI void cp_async16(uint32_t dst, const void* src, bool in) {
  const int n = in ? 16 : 0;  // the rest is filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
// Through L1: activations that other warps of the SM read too.
TAO_DEVI void cp_async16_l1(uint32_t dst, const void* src, bool in) {
  const int n = in ? 16 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
TAO_DEVI void cp_async8_l1(uint32_t dst, const void* src, bool in) {
  const int n = in ? 8 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
TAO_DEVI void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
TAO_DEVI void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
TAO_DEVI uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
TAO_DEVI uint2 lds8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}
TAO_DEVI uint32_t lds_u16(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
  return v;
}
TAO_DEVI uint32_t lds_u8(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}

// The 16-bit type of the mma: what an operand register pair means, and 4-bit codes in it.
struct MmaBf16 {
  // 0x4300 | q is 128 + q exactly (7 mantissa bits); one subtraction leaves q - zero exactly.
  static constexpr uint32_t kMagic = 0x43004300u;
  static TAO_DEVI uint32_t sub(uint32_t a, uint32_t b) {
    __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
  }
  static TAO_DEVI void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                           uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
struct MmaF16 {
  static constexpr uint32_t kMagic = 0x64006400u;  // 1024 + q
  static TAO_DEVI uint32_t sub(uint32_t a, uint32_t b) {
    __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
  }
  static TAO_DEVI void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                           uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

// Two codes (nibbles i and i + 4 of w) as a pair of magic + q.
template <class M>
TAO_DEVI uint32_t codes_at(uint32_t w, int i) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xEA;" : "=r"(r) : "r"(w >> (4 * i)), "r"(M::kMagic));
  return r;
}

// Four e4m3 in 32 bits as two pairs of fp16 (exact).
TAO_DEVI void e4m3_to_f16(uint32_t v, uint32_t& lo, uint32_t& hi) {
  const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v & 0xffff), __NV_E4M3);
  const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v >> 16), __NV_E4M3);
  lo = a.x | (uint32_t)a.y << 16;
  hi = b.x | (uint32_t)b.y << 16;
}

// A 4-bit matrix laid out in blocks of 16 rows x 128 k, row tiles outermost.
struct Four {
  const uint8_t* codes;    // [tiles][blocks][1024]
  const uint16_t* scales;  // [tiles][blocks][128 / group][16]
  const uint8_t* zeros;    // the same, or null: 8
};

// KB (64 or 128) k of a 4-bit block against eight activation rows for each of NT column
// tiles, those that hold some of the `cols` rows.  `b(u, n)` gives the lane's 8 activations
// of 32-k part u as four operand registers; `scale(j, row)` the scale of group j.  The
// codes' products are summed in fp32 over a group (or the KB k of it) and scaled then, so
// no weight is ever rounded.
template <class M, int GROUP, int KB, int NT, class B, class S>
TAO_DEVI void four_block(float (&acc)[NT][4], uint32_t codes, uint32_t zeros, bool has_zeros, int lane, int cols, B b,
                         S scale) {
  constexpr int SPAN = GROUP < KB ? GROUP : KB, PARTS = SPAN / 32;  // k, and 32-k parts, under one scale
  const int g = lane >> 2;
  uint4 w = lds16(codes + lane * 16);
#pragma unroll
  for (int j = 0; j < KB / SPAN; ++j) {
    uint32_t z0 = 8, z1 = 8;
    if (has_zeros) {
      z0 = lds_u8(zeros + j * 16 + g);
      z1 = lds_u8(zeros + j * 16 + g + 8);
    }
    z0 = M::kMagic | z0 | z0 << 16;
    z1 = M::kMagic | z1 | z1 << 16;
    float t[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) t[n][0] = t[n][1] = t[n][2] = t[n][3] = 0.f;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      const int u = j * PARTS + p;
      if (u == 2) w = lds16(codes + 512 + lane * 16);
      const uint32_t w0 = u & 1 ? w.z : w.x, w1 = u & 1 ? w.w : w.y;
      uint32_t a[2][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[0][i] = M::sub(codes_at<M>(w0, i), i & 1 ? z1 : z0);
        a[1][i] = M::sub(codes_at<M>(w1, i), i & 1 ? z1 : z0);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (n && n * 8 >= cols) break;
        const uint4 x = b(u, n);
        M::mma(t[n], a[0][0], a[0][1], a[0][2], a[0][3], x.x, x.y);
        M::mma(t[n], a[1][0], a[1][1], a[1][2], a[1][3], x.z, x.w);
      }
    }
    const float s0 = scale(j, g), s1 = scale(j, g + 8);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      acc[n][0] += s0 * t[n][0];
      acc[n][1] += s0 * t[n][1];
      acc[n][2] += s1 * t[n][2];
      acc[n][3] += s1 * t[n][3];
    }
  }
}

}  // namespace tao
