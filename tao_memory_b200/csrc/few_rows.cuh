// Products of a few activation rows with a large weight matrix: the device parts that
// the 4-bit product and the expert layer share.
//
//   D[n][m] += sum over k of W[n][k] x[m][k]
//
// The weights are the 16-row operand of a warp's mma and eight activation columns the other, so a
// weight is used once per eight columns.  Up to 16 rows the work is bound by the weights' bytes and the
// instructions per weight; a tcgen05 tile has operands in shared memory, where 4-bit weights would first have
// to be written unpacked, which pays from 17 rows on (linear4_tc.cuh).
//
// A few rows (product8): the codes 0..15 go as bytes into the integer mma.m16n8k32, three
// instructions for eight of them.  The activations become sums of signed bytes under a power of
// two s for each row and 128 k,  x = s (p0 + p1 / 2^7 + p2 / 2^14 + p3 / 2^21),  a column of the mma for
// each piece.  The 128's largest magnitude is 32 s to 64 s, so x is held to 2^-27 of it, finer than the 2^-24 of
// that magnitude to which fp32 sums of its products would go: no caller's channel is lost beside one 10^5 times larger.
// Over a group
//   sum of (q - zero) x = s 2^-7 (sum of q P - zero sum of P) + s 2^-21 (the same of Q),
//   P = 2^7 p0 + p1,  Q = 2^7 p2 + p3,
// whole numbers below 2^24, so a group's product is exact in fp32; fp32 sums over the groups.
// More rows (product16): codes become 16-bit floats with their zero point subtracted, exactly, for
// mma.m16n8k16: eleven instructions for eight, but one column a row.
//
// The order of k inside a product is free, as long as both operands use the same: of every 32 k lane
// (g, t) = (lane / 4, lane % 4) takes 8t..8t+7.  A 4-bit block of 16 rows x 128 k is laid out so that a
// lane's 64 codes are two 16-byte words: byte 8i + 4f + e of half h is k = 64h + 32i + 8t + 4f + (0, 2, 1, 3)[e],
// of row g in the low nibble and of row g + 8 in the high one; nibbles 16 bits apart are neighbouring k.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "common.cuh"

namespace tao {

// Asynchronous copy of 16 bytes to shared memory; zeros where `in` is false.
TAO_DEVI void cp_async16(uint32_t to, const void* from, bool in = true) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(in ? 16 : 0) : "memory");
}
TAO_DEVI void cp_async8(uint32_t to, const void* from, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(in ? 8 : 0) : "memory");
}
TAO_DEVI void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int OPEN>
TAO_DEVI void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(OPEN) : "memory");
}

TAO_DEVI void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
TAO_DEVI void mma_u8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The 16-bit type of product16's mma: 4-bit codes in it.
struct MmaBf16 {
  // 0x4300 | q is 128 + q exactly (7 mantissa bits); adding -(128 + zero) leaves q - zero exactly.
  static constexpr uint32_t kMagic = 0x43004300u;
  static TAO_DEVI uint32_t add(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(0x3f803f80u), "r"(b));
    return r;
  }
  static TAO_DEVI void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_bf16(d, a[0], a[1], a[2], a[3], b0, b1);
  }
};
struct MmaF16 {
  static constexpr uint32_t kMagic = 0x64006400u;  // 1024 + q
  static TAO_DEVI uint32_t add(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static TAO_DEVI void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// 2^21 / s and s / 2^7 of a 128's largest magnitude: x / s is below 64.  What has no such form, a magnitude
// that is no finite number or whose 2^21 / s would not be one, makes both no numbers, and with them the row's sums.
TAO_DEVI void units_of(float most, float& up, float& unit) {
  const uint32_t e = __float_as_uint(most) >> 23;  // of a magnitude: no sign
  const uint32_t f = e > 26 ? e - 5 : 21u;         // the exponent of s; 2^21 / s is a normal number
  const bool none = e == 255 || (e < 27 && most > 0.f);
  up = __uint_as_float(none ? 0x7fc00000u : (254 + 21 - f) << 23);
  unit = __uint_as_float(none ? 0x7fc00000u : (f - 7) << 23);
}

// Eight 2^21 x / s (below 2^27 in magnitude), rounded to whole numbers, as four pieces of 8 signed
// bytes each in the order of the codes (digits of -64..63, the first up to 64), and the sums of P and of Q.
TAO_DEVI void split8(const float (&x)[8], uint2 (&p)[4], int& sum, int& sum2) {
  uint32_t w[4][2] = {};
  sum = sum2 = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int v = __float2int_rn(x[i]);
    const int v2 = (v + 64) >> 7, v1 = (v2 + 64) >> 7, v0 = (v1 + 64) >> 7;
    const int q[4] = {v0, v1 - (v0 << 7), v2 - (v1 << 7), v - (v2 << 7)};
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j][i / 4] |= (uint32_t)(q[j] & 0xff) << (8 * (i % 4 * 2 % 3 + i % 4 / 3 * 3));
    sum += v1;
    sum2 += v - (v1 << 14);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) p[j] = make_uint2(w[j][0], w[j][1]);
}

// A 4-bit matrix laid out in blocks of 16 rows x 128 k, row tiles outermost.
struct Four {
  const uint8_t* codes;   // [tiles][blocks][1024]
  const uint8_t* scales;  // [tiles][blocks][8][128 / group][2] 16-bit: rows g and g + 8 of the tile
  const uint8_t* zeros;   // the same in bytes, or null: 8
};

// A block in registers: this lane's codes, and the scales and zero points of its rows g, g + 8.
template <int GROUP>
struct Block4 {
  static constexpr int GROUPS = 128 / GROUP, PARTS = GROUP / 32;  // groups of a block, 32-k parts of a group
  uint4 c[2];
  uint32_t s[GROUPS], z[(GROUPS + 1) / 2];

  // A block in a ring in shared memory: codes, scales, zero points.
  static constexpr int SCALES = 32 * GROUPS, ZEROS = 16 * GROUPS, BYTES = 1024 + SCALES + ZEROS;

  // Starts the copy of block `block` of the matrix by the warp.
  static TAO_DEVI void issue(uint32_t to, const Four& w, uint32_t block, int lane) {
    const uint8_t* codes = w.codes + lane * 16 + (uint64_t)block * 1024u;
    cp_async16(to + lane * 16, codes);
    cp_async16(to + 512 + lane * 16, codes + 512);
    if (lane < SCALES / 16)
      cp_async16(to + 1024 + lane * 16, w.scales + lane * 16 + (uint64_t)block * (uint32_t)SCALES);
    else if (w.zeros && lane >= 16 && lane < 16 + ZEROS / 16)
      cp_async16(to + 1024 + SCALES + (lane - 16) * 16, w.zeros + (lane - 16) * 16 + (uint64_t)block * (uint32_t)ZEROS);
  }
  // From the ring, when the copy is over and the warp has met since.
  TAO_DEVI void load(const uint8_t* from, bool has_zeros, int lane) {
    c[0] = *reinterpret_cast<const uint4*>(from + lane * 16);
    c[1] = *reinterpret_cast<const uint4*>(from + 512 + lane * 16);
    const uint32_t* sp = reinterpret_cast<const uint32_t*>(from + 1024) + (lane >> 2) * GROUPS;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) s[i] = sp[i];
    const uint16_t* zp = reinterpret_cast<const uint16_t*>(from + 1024 + SCALES) + (lane >> 2) * GROUPS;
#pragma unroll
    for (int i = 0; i < (GROUPS + 1) / 2; ++i)
      z[i] = !has_zeros ? 0x08080808u : GROUPS == 1 ? zp[0] : reinterpret_cast<const uint32_t*>(zp)[i];
  }
  // Exchanges 32-k parts 0 and 1, 2 and 3, the zero points with them.
  TAO_DEVI void swap_parts() {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      c[i] = make_uint4(c[i].z, c[i].w, c[i].x, c[i].y);
      if constexpr (GROUP == 32) z[i] = z[i] >> 16 | z[i] << 16;
    }
  }
  TAO_DEVI uint32_t zeros(int j) const { return z[j / 2] >> (16 * (j & 1)); }  // of rows g, g + 8, a byte each
  template <bool BF16_SCALES>
  TAO_DEVI float2 scales(int j) const {
    if constexpr (BF16_SCALES) return make_float2(lo_f(s[j]), hi_f(s[j]));
    return __half22float2(*reinterpret_cast<const __half2*>(&s[j]));
  }
  TAO_DEVI uint32_t word(int u, int i) const {
    const uint4& w = c[u / 2];
    return u & 1 ? (i ? w.w : w.z) : (i ? w.y : w.x);
  }

  // Adds to acc[n][0..1] rows g and g + 8 of the block's product with the row of x whose pieces 0 and 1
  // (t even) or 2 and 3 (t odd) are columns 2t, 2t + 1 of column tile n; the row's whole product is the sum over
  // the two lanes.  `b(h, n)`: the lane's 16 bytes of half h; `xsum(j, n)`: the sum over group j of P (t odd:
  // of Q); `unit(n)`: s / 2^7 (t odd: s / 2^21).
  template <bool BF16_SCALES, int NT, class B, class X, class U>
  TAO_DEVI void product8(float (&acc)[NT][2], B b, X xsum, U unit) const {
    constexpr uint32_t MASK = 0x0f0f0f0fu;
    uint32_t a[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        a[u][2 * i] = word(u, i) & MASK;
        a[u][2 * i + 1] = word(u, i) >> 4 & MASK;
      }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint4 x0 = b(0, n), x1 = b(1, n);
      const uint32_t bs[4][2] = {{x0.x, x0.y}, {x0.z, x0.w}, {x1.x, x1.y}, {x1.z, x1.w}};
      const float un = unit(n);
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        int d[4] = {0, 0, 0, 0}, d2[4] = {0, 0, 0, 0};  // two chains of dependent products
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
          const int u = j * PARTS + p;
          mma_u8s8(p & 1 ? d2 : d, a[u][0], a[u][1], a[u][2], a[u][3], bs[u][0], bs[u][1]);
        }
        if constexpr (PARTS > 1) {
#pragma unroll
          for (int i = 0; i < 4; ++i) d[i] += d2[i];
        }
        const int z0 = zeros(j) & 0xff, z1 = zeros(j) >> 8 & 0xff;
        const int xs = xsum(j, n);
        const float2 sc = scales<BF16_SCALES>(j);
        acc[n][0] += sc.x * un * (float)(d[0] * 128 + d[1] - z0 * xs);
        acc[n][1] += sc.y * un * (float)(d[2] * 128 + d[3] - z1 * xs);
      }
    }
  }

  // Operand registers of 32-k part u as 16-bit floats, code - zero: of the first four k of a lane's eight
  // and of the last four; register r is row half r & 1, elements (0, 1) or (2, 3).
  template <class M>
  TAO_DEVI void operands16(int u, uint32_t (&a)[2][4]) const {
    // -(magic + zero) in both halves: the zero's byte below the magic's with its sign
    const uint32_t zz = zeros(u / PARTS);
    const uint32_t z0 = __byte_perm(zz, M::kMagic >> 24 | 0x80, 0x4040);
    const uint32_t z1 = __byte_perm(zz, M::kMagic >> 24 | 0x80, 0x4141);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        uint32_t v;
        asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xEA;" : "=r"(v) : "r"(word(u, i) >> (4 * r)), "r"(M::kMagic));
        a[i][r] = M::add(v, r & 1 ? z1 : z0);
      }
  }

  // Adds D of the block's product with eight rows of x for each of NT column tiles, those that hold some
  // of the `cols` rows.  `b(u, n)`: the lane's 8 activations of 32-k part u.
  template <class M, bool BF16_SCALES, int NT, class B>
  TAO_DEVI void product16(float (&acc)[NT][4], int cols, B b) const {
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) {
      // two chains of dependent products, or as many as there are column tiles
      constexpr int CHAINS = NT == 1 ? 2 : 1;
      float d[NT * CHAINS][4];
#pragma unroll
      for (int n = 0; n < NT * CHAINS; ++n) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.f;
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        const int u = j * PARTS + p;
        uint32_t a[2][4];
        operands16<M>(u, a);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (n && n * 8 >= cols) break;
          const uint4 x = b(u, n);
          M::mma(d[n], a[0], x.x, x.y);
          M::mma(d[n + CHAINS - 1], a[1], x.z, x.w);
        }
      }
      if constexpr (CHAINS == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) d[0][i] += d[1][i];
      }
      const float2 sc = scales<BF16_SCALES>(j);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        acc[n][0] += sc.x * d[n][0];
        acc[n][1] += sc.x * d[n][1];
        acc[n][2] += sc.y * d[n][2];
        acc[n][3] += sc.y * d[n][3];
      }
    }
  }
};

}  // namespace tao
