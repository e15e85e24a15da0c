// Products of 16-bit matrices on tcgen05 with everything around them in one kernel: the forward product
// with bias, activation, gate and residual, the two products of its gradient, and each of them for the rows
// of many experts at once.  fp32 accumulators in TMEM, one rounding when a value is stored.
//
//   FORWARD  y[t][c] = act(sum_k x[t][k] W[c][k] + bias[c]) + residual[t][c], or act(x W^T) * (x U^T)
//   FEW      the same for few rows: W is the operand of 128 rows, x the one of 32 or 64 columns, so that
//            a tile does not multiply rows that are not there
//   INPUT    dx[t][k] = sum_c dz[t][c] W[c][k] (+ du U)
//   WEIGHT   dW[c][k] = sum_t dz[t][c] x[t][k]
//
// Operands arrive as they lie in memory: one whose terms are next to each other (K-major) and one whose
// rows are (MN-major) differ in the box that TMA fetches and in the descriptor only, so nothing is transposed.
// A block keeps one CTA an SM busy over many tiles: a warp fetches 64 terms at a time into a ring, a
// warp issues the products into one of two accumulators, and eight warps turn the other one into outputs.
// Tiles go in bands of 16 row tiles, so that the blocks at work share operands in L2.
//
// What bounds it: operands.  A step of a 128 x 256 tile fetches 48 KB for 512 cycles of products, more than an SM gets from
// L2 in that time while all ask (about 700 cycles); the tensor pipe is busy 63 to 75 % of the time.  PAIR: two blocks with
// 128 rows each multiply one 256 x 256 tile from both blocks' shared memory (cta_group::2), each fetching half of B:
// 32 KB a step.  16384x2048x8192 takes 353 us in pairs (1.56 PFLOP/s; 380 alone), with bias and gelu 368;
// 32768x768x2304 93 us, its gradients 90 and 94; 32768 rows of 64 experts, gated 2048 to 1024, 232 us.
//
// SPLIT: a product with fewer tiles than SMs deals the terms of a tile to the blocks (WEIGHT: or the pairs) of a cluster,
// which add their parts through each other's shared memory in the order of their ranks.
//
// Experts: rows of x are sorted by expert, offsets[e] .. offsets[e + 1] are those of expert e.  Every block
// makes the list of tiles itself from the offsets, so the host never reads them.  A row tile never spans
// two experts; rows of a tile behind its expert's last are computed and not stored, and as terms of WEIGHT
// they are set to zero in shared memory in both operands (another expert's may be infinite).
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>

#include "../../include/tao_b200.h"
#include "common.cuh"
#include "linear4.cuh"
#include "tcgen05.cuh"

namespace tao {
namespace product {

static __device__ int g_error;  // an expired wait, until tao_product_check

enum Form { FORWARD, FEW, INPUT, WEIGHT };

constexpr int kTerms = 64;         // of a step of the ring: 128 bytes, the swizzle's width
constexpr int kMostGroups = 512;   // experts
constexpr int kWorkers = 8;        // warps that read accumulators
constexpr int kThreads = 32 * (kWorkers + 2);
constexpr int kBand = 16;          // row tiles of a band

struct Args {
  const int* offsets;  // of the experts, or null: one group of all rows
  int groups, rows;
  int cols;            // of an output row
  int depth;           // terms of a sum (FORWARD, FEW: k, INPUT: n); WEIGHT: rows of an output matrix
  int pairs;           // INPUT: pairs of operands whose products are added; WEIGHT: matrices of an expert
  int type, act;
  const void *bias, *residual;
  long long r_stride;
  void *y, *z, *u;     // z, u: act's argument and the gate's factor (FORWARD, FEW); u: the second matrix (WEIGHT)
  uint8_t* low;        // gated: the lower bits of both
  long long z_stride;
  bool wide;           // rows of y, z and the residual start on 16 bytes, and cols is a multiple of 8
  int split;           // blocks of a cluster
};

template <int FORM, int BN, bool GATED, bool SPLIT, bool PAIR = false>
struct Cfg {
  static constexpr bool A_MN = FORM == WEIGHT, B_MN = FORM == INPUT || FORM == WEIGHT;
  static constexpr int TT = FORM == FEW ? BN : PAIR ? 256 : 128;                 // token rows of a tile
  static constexpr int DOWN = PAIR ? 256 : 128;                                  // rows of a tile of WEIGHT
  static constexpr int CT = FORM == FEW ? 128 : GATED ? BN / 2 : BN;             // output columns of a tile
  static constexpr int A = (FORM == FEW && GATED ? 2 : 1) * 128 * 128, B = (PAIR ? BN / 2 : BN) * 128, STAGE = A + B;
  static constexpr int STAGING = FORM == FEW || SPLIT ? 0 : kWorkers * 2048;
  static constexpr int LISTS = SPLIT ? 0 : (2 * kMostGroups + 4) * 4;
  // parts of a split tile: of few rows in a place of their own, else over the ring
  static constexpr int PARTS = !SPLIT ? 0 : FORM == FEW ? (BN + 7) * 128 * 4 : 128 * (BN + 4) * 4;
  static constexpr int REST = STAGING + LISTS + 512 + (FORM == FEW ? PARTS : 0);
  static constexpr int FIT = (227 * 1024 - REST) / STAGE, STAGES = FIT < 12 ? FIT : 12;
  static constexpr int SMEM = STAGES * STAGE + REST;
  static constexpr int ACC = FORM == FEW && GATED ? 2 * BN : BN;
  static constexpr int SETS = SPLIT ? 1 : 2, USED = SETS * ACC;
  static constexpr int TMEM = USED <= 32 ? 32 : USED <= 64 ? 64 : USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
  static_assert(USED <= 512 && STAGES >= 3 && (FORM == FEW || PARTS <= STAGES * STAGE) && SMEM <= 227 * 1024, "");
};

// Whether a phase is over, without waiting (try_wait may suspend the thread for a while).
TAO_DEVI bool arrived(uint64_t* bar, uint32_t phase) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(ok)
               : "r"(smem_u32(bar)), "r"(phase)
               : "memory");
  return ok != 0;
}

// Waits at most about four seconds, and for the sums of a tile of WEIGHT two microseconds more for each of its steps (one
// takes 0.3, and an expert of 2^30 rows has 2^24; other forms' sums have up to 2^24 terms, 0.2 s); a wait that runs out, or another's of this block, ends all of them.
TAO_DEVI bool wait_for(uint64_t* bar, uint32_t phase, volatile int* abort, int steps = 0) {
  unsigned long long began = 0;
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, phase)) return true;
    if (i & 63u) continue;
    if (*abort) return false;
    unsigned long long now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (!began) began = now;
    if (now - began > 4000000000ull + steps * 2000ull) break;
  }
  *abort = 1;
  atomicOr(&g_error, kErrWaitTimeout);
  return false;
}
TAO_DEVI bool warp_wait_for(uint64_t* bar, uint32_t phase, volatile int* abort, int steps = 0) {
  return __all_sync(0xffffffffu, wait_for(bar, phase, abort, steps));
}

TAO_DEVI void tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// The cluster's barrier in two steps, by whole warps.
TAO_DEVI void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
TAO_DEVI void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Where a block of the cluster has what is at `at` in this one.
TAO_DEVI uint32_t peer(uint32_t at, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
  return r;
}
TAO_DEVI void put_peer(uint32_t at, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}

// PAIR: the same by the two blocks of a pair: the copy arrives at a barrier of either, the product takes 128 rows of A
// and half of B's from each one's shared memory, and the end of products arrives at the same barrier of both.
TAO_DEVI void tma_3d_pair(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
TAO_DEVI void multiply_pair(uint32_t acc, uint64_t a, uint64_t b, uint32_t idesc, uint32_t more) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(acc),
      "l"(a), "l"(b), "r"(idesc), "r"(more));
}
TAO_DEVI void commit_pair(uint64_t* bar, int first) {  // `first`: the rank of the pair's first block
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
      "h"((uint16_t)(3 << first))
      : "memory");
}
TAO_DEVI void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// One lane of a warp that has met, the same for all that ask.
TAO_DEVI bool elected() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}
// 128 rows of A times B^T, 16 terms, onto (or, more = 0, into) the accumulator.
TAO_DEVI void multiply(uint32_t acc, uint64_t a, uint64_t b, uint32_t idesc, uint32_t more) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(acc),
      "l"(a), "l"(b), "r"(idesc), "r"(more));
}

// N consecutive fp32 columns of this thread's TMEM lane.
template <int N>
TAO_DEVI void load_columns(uint32_t at, float (&v)[N]) {
  static_assert(N == 16 || N == 32, "");
  if constexpr (N == 32) {
    tc::tmem_ld32(at, v);
  } else {
    uint32_t r[N];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float(r[i]);
  }
}

// -- 16-bit values of either type -----------------------------------------
TAO_DEVI uint32_t pack(float lo, float hi, bool is_bf16) {
  if (is_bf16) return bf16x2(lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
TAO_DEVI uint16_t pack1(float v, bool is_bf16) { return (uint16_t)pack(v, 0.f, is_bf16); }
TAO_DEVI float2 unpack(uint32_t w, bool is_bf16) {
  if (is_bf16) return make_float2(lo_f(w), hi_f(w));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
TAO_DEVI float unpack1(uint16_t w, bool is_bf16) { return unpack(w, is_bf16).x; }
TAO_DEVI float load1(const void* p, long long i, bool is_bf16) {
  return unpack1(static_cast<const uint16_t*>(p)[i], is_bf16);
}

// fp32 cut to 24 bits (to 2^-15), of which the upper 16 and the lower 8 are kept apart: what a gate's two factors are
// kept in for the gradient.  Rounded to bf16 they made its error 1.8 times that of one rounding (1.4 so).
TAO_DEVI uint32_t bits24(float v) { return __float_as_uint(v); }
TAO_DEVI float of24(uint32_t upper, uint32_t lower) { return __uint_as_float(upper << 16 | lower << 8); }

// -- activations ------------------------------------------------------------
// By the special-function unit's 2^x and reciprocal (subnormal numbers are zero).  An exponent is rounded before 2^x, so
// the relative error grows with it: sigmoid(q) 2^-22 up to |q| = 5, 2^-21 at 10, 2^-18 at 80, e^(-z^2 / 2) 2^-20.5 at
// |z| = 4, 2^-17.5 at 10: far below a 16-bit step.
TAO_DEVI float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2E = 1.4426950408889634f;
TAO_DEVI float sigmoid(float q) { return reciprocal(1.f + tc::ex2(-kLog2E * q)); }
constexpr float kGeluRoot = 0.7978845608028654f, kGeluCube = 0.044715f;  // sqrt(2 / pi)

// Two fp32 values at an instruction.
struct Two {
  uint64_t v;
};
TAO_DEVI Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
TAO_DEVI Two two(float a) { return two(a, a); }
TAO_DEVI float2 apart(Two x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x.v));
  return r;
}
TAO_DEVI Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
TAO_DEVI Two mul2(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// The normal distribution's integral from the tail of z's side: with t = 1 / (1 + 0.35 x), x = |z| / sqrt(2),
// erfc(x) e^(x^2) / t is smooth on (0, 1], and half of it a polynomial in t (fitted here at Chebyshev nodes to 2^-20.2,
// 2^-19.6 in fp32).  So small values keep a relative precision, of the tail 2^-19.4 up to |z| = 4 and e^(-z^2 / 2)'s beyond,
// at two special-function instructions.  `density` is e^(-z^2 / 2).
TAO_DEVI float2 normal_integral(float2 z, float2& density) {
  const float slope = 0.35f * 0.7071067811865476f;
  const Two t = two(reciprocal(fmaf(slope, fabsf(z.x), 1.f)), reciprocal(fmaf(slope, fabsf(z.y), 1.f)));
  const Two both = two(z.x, z.y);
  const float2 e = apart(mul2(mul2(both, both), two(-0.5f * kLog2E)));
  density = make_float2(tc::ex2(e.x), tc::ex2(e.y));
  Two q = fma2(two(-0.042552598f), t, two(0.100604653f));
  q = fma2(q, t, two(-0.0072748783f));
  q = fma2(q, t, two(0.0814718946f));
  q = fma2(q, t, two(0.0773361512f));
  q = fma2(q, t, two(0.0929546698f));
  q = fma2(q, t, two(0.098726552f));
  q = fma2(q, t, two(0.0987331438f));
  const float2 tail = apart(mul2(mul2(two(density.x, density.y), t), q));
  return make_float2(z.x < 0.f ? tail.x : 1.f - tail.x, z.y < 0.f ? tail.y : 1.f - tail.y);
}
TAO_DEVI float normal_integral(float z, float& density) {
  float2 d;
  const float2 p = normal_integral(make_float2(z, z), d);
  density = d.x;
  return p.x;
}

TAO_DEVI float activate(float z, int act) {
  switch (act) {
    case TAO_ACT_RELU: return z > 0.f || z != z ? z : 0.f;
    case TAO_ACT_SILU: return z * sigmoid(z);
    case TAO_ACT_GELU: {
      float density;
      return z * normal_integral(z, density);
    }
    case TAO_ACT_GELU_TANH: return z * sigmoid(2.f * kGeluRoot * (z + kGeluCube * z * z * z));
  }
  return z;
}
// act(z) and act'(z).  `near`: far out act' is 0 or 1, but as it is written 0 times z, which may be infinite (an argument
// kept in fp16 is from 65520 on; NaN stays NaN by the other factors).
TAO_DEVI float2 activate_slope(float z, int act) {
  const float near = fminf(fmaxf(z, -128.f), 128.f);
  switch (act) {
    case TAO_ACT_RELU: return make_float2(z > 0.f || z != z ? z : 0.f, z > 0.f ? 1.f : 0.f);
    case TAO_ACT_SILU: {
      const float s = sigmoid(z);
      return make_float2(z * s, s * (1.f + near * (1.f - s)));
    }
    case TAO_ACT_GELU: {
      float density;
      const float p = normal_integral(z, density);
      return make_float2(z * p, p + near * 0.3989422804014327f * density);
    }
    case TAO_ACT_GELU_TANH: {
      const float s = sigmoid(2.f * kGeluRoot * (z + kGeluCube * z * z * z));
      return make_float2(z * s, s + near * s * (1.f - s) * 2.f * kGeluRoot * (1.f + 3.f * kGeluCube * near * near));
    }
  }
  return make_float2(z, 1.f);
}
template <int N>
TAO_DEVI void activate_all(float (&v)[N], int act) {
  switch (act) {  // the choice outside of the loop
    case TAO_ACT_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activate(v[i], TAO_ACT_RELU);
      break;
    case TAO_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activate(v[i], TAO_ACT_SILU);
      break;
    case TAO_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        float2 density;
        const float2 p = normal_integral(make_float2(v[i], v[i + 1]), density);
        v[i] *= p.x;
        v[i + 1] *= p.y;
      }
      break;
    case TAO_ACT_GELU_TANH:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activate(v[i], TAO_ACT_GELU_TANH);
      break;
  }
}

// -- tiles ----------------------------------------------------------------------
struct Tile {
  int row0, rows;  // token rows: the first, and how many of the tile's there are; WEIGHT: rows of the matrix
  int col0;
  int group, second;  // expert; WEIGHT: which of its matrices
  int from, upto;     // WEIGHT: its token rows
  int blocks;         // steps of the ring; 0: zeros
};

// The experts' last rows (not before the one before, not behind the last row) and the tiles before each;
// rows of no expert are one more group.  By one warp.
template <class C>
TAO_DEVI void make_lists(const Args& a, int* first, int* ends, int lane) {
  const int col_tiles = (a.cols + C::CT - 1) / C::CT;
  int end = 0, tiles = 0;
  for (int base = 0; base <= a.groups; base += 32) {
    const int e = base + lane;
    int v = e < a.groups ? min(max(a.offsets[e + 1], 0), a.rows) : a.rows;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int w = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v = max(v, w);
    }
    v = max(v, end);
    int before = __shfl_up_sync(0xffffffffu, v, 1);
    if (lane == 0) before = end;
    int n = e <= a.groups ? (v - before + C::TT - 1) / C::TT * col_tiles : 0;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int w = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += w;
    }
    if (e <= a.groups) {
      ends[e] = v;
      first[e + 1] = tiles + n;
    }
    end = __shfl_sync(0xffffffffu, v, 31);
    tiles += __shfl_sync(0xffffffffu, n, 31);
  }
  if (lane == 0) first[0] = 0;
}

// Tile t of all; `group` is the one of the caller's tile before (0 at first).
template <int FORM, class C>
TAO_DEVI Tile tile_of(const Args& a, const int* first, const int* ends, int t, int& group) {
  Tile tile;
  const int col_tiles = (a.cols + C::CT - 1) / C::CT;
  tile.second = tile.from = tile.upto = 0;
  if constexpr (FORM == WEIGHT) {
    const int row_tiles = (a.depth + C::DOWN - 1) / C::DOWN, per = row_tiles * col_tiles;
    const int matrix = t / per, at = t - matrix * per;
    group = matrix / a.pairs;
    tile.second = matrix - group * a.pairs;
    tile.row0 = at % row_tiles * C::DOWN;
    tile.col0 = at / row_tiles * C::CT;
    tile.rows = min(C::DOWN, a.depth - tile.row0);
    if (a.offsets) {
      tile.from = group ? ends[group - 1] : 0;
      tile.upto = ends[group];
    } else {
      tile.upto = a.rows;
    }
    tile.blocks = (tile.upto - tile.from + kTerms - 1) / kTerms;
  } else {
    int begin = 0, end = a.rows;
    if (a.offsets) {
      while (t >= first[group + 1]) ++group;
      t -= first[group];
      begin = group ? ends[group - 1] : 0;
      end = ends[group];
    }
    const int row_tiles = (end - begin + C::TT - 1) / C::TT;
    const int band = t / (kBand * col_tiles), in = t - band * (kBand * col_tiles);
    const int high = min(kBand, row_tiles - band * kBand), column = in / high;
    tile.row0 = begin + (band * kBand + in - column * high) * C::TT;
    tile.col0 = column * C::CT;
    tile.rows = min(C::TT, end - tile.row0);
    tile.blocks = a.offsets && group == a.groups ? 0 : (a.depth + kTerms - 1) / kTerms * (FORM == INPUT ? a.pairs : 1);
  }
  tile.group = group;
  return tile;
}

// -- 32 x 32 values between a warp's threads, a row each, and memory ----------------
// Through 2 KB of shared memory, 16-byte chunks of a row turned so that eight rows' meet all banks.
TAO_DEVI int staged(int row, int chunk) { return row * 64 + ((chunk ^ (row >> 1 & 3)) << 4); }

// `U` neighbours at a time (8, or 1 where the rows' addresses do not allow it), all rows on their way.
template <int U>
struct Unit;
template <>
struct Unit<8> { using Type = uint4; };
template <>
struct Unit<2> { using Type = uint32_t; };
template <>
struct Unit<1> { using Type = uint16_t; };

template <int U>
TAO_DEVI void move_rows(uint8_t* staging, uint16_t* memory, long long stride, int rows, int cols, bool in, int lane) {
  using W = typename Unit<U>::Type;
  constexpr int ACROSS = 32 / U;
  const int c = lane % ACROSS * U, first = lane / ACROSS;
  memory += first * stride + c;
  auto at = [&](int r) { return reinterpret_cast<W*>(staging + staged(r, c >> 3) + (c & 7) * 2); };
  if (in) {
    W v[ACROSS];
#pragma unroll
    for (int i = 0; i < ACROSS; ++i)
      if (i * U + first < rows && c < cols) v[i] = *reinterpret_cast<const W*>(memory + i * U * stride);
#pragma unroll
    for (int i = 0; i < ACROSS; ++i)
      if (i * U + first < rows && c < cols) *at(i * U + first) = v[i];
  } else {
#pragma unroll 4
    for (int i = 0; i < ACROSS; ++i)
      if (i * U + first < rows && c < cols) *reinterpret_cast<W*>(memory + i * U * stride) = *at(i * U + first);
  }
}
TAO_DEVI void move_rows(uint8_t* staging, void* memory, long long stride, int rows, int cols, bool wide, bool in, int lane) {
  uint16_t* const m = static_cast<uint16_t*>(memory);
  if (wide)
    move_rows<8>(staging, m, stride, rows, cols, in, lane);
  else
    move_rows<1>(staging, m, stride, rows, cols, in, lane);
}
// This thread's row of v, rounded, to memory.  All lanes of the warp.
TAO_DEVI void put_rows(uint8_t* staging, const float (&v)[32], bool is_bf16, void* to, long long stride, int rows,
                       int cols, bool wide, int lane) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    *reinterpret_cast<uint4*>(staging + staged(lane, c)) =
        make_uint4(pack(v[c * 8], v[c * 8 + 1], is_bf16), pack(v[c * 8 + 2], v[c * 8 + 3], is_bf16),
                   pack(v[c * 8 + 4], v[c * 8 + 5], is_bf16), pack(v[c * 8 + 6], v[c * 8 + 7], is_bf16));
  __syncwarp();
  move_rows(staging, to, stride, rows, cols, wide, false, lane);
  __syncwarp();
}

// This thread's row of v in 24 bits: the upper and the lower part to memory, on 16 bytes.  All lanes of the warp.
TAO_DEVI void put_rows24(uint8_t* staging, const float (&v)[32], uint16_t* upper, uint8_t* lower, long long stride, int rows,
                         int cols, int lane) {
  uint32_t low[8];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = bits24(v[c * 8 + i]);
    *reinterpret_cast<uint4*>(staging + staged(lane, c)) =
        make_uint4(__byte_perm(b[0], b[1], 0x7632), __byte_perm(b[2], b[3], 0x7632), __byte_perm(b[4], b[5], 0x7632),
                   __byte_perm(b[6], b[7], 0x7632));
#pragma unroll
    for (int i = 0; i < 2; ++i)
      low[c * 2 + i] = __byte_perm(__byte_perm(b[i * 4], b[i * 4 + 1], 0x0051), __byte_perm(b[i * 4 + 2], b[i * 4 + 3], 0x0051), 0x5410);
  }
  __syncwarp();
  move_rows<8>(staging, upper, stride, rows, cols, false, lane);
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 2; ++c)
    *reinterpret_cast<uint4*>(staging + lane * 32 + ((c ^ (lane >> 2 & 1)) << 4)) =
        make_uint4(low[c * 4], low[c * 4 + 1], low[c * 4 + 2], low[c * 4 + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = i * 16 + (lane >> 1), c = lane & 1;
    if (r < rows && c * 16 < cols)
      *reinterpret_cast<uint4*>(lower + r * stride + c * 16) =
          *reinterpret_cast<const uint4*>(staging + r * 32 + ((c ^ (r >> 2 & 1)) << 4));
  }
  __syncwarp();
}

// One output of a FORWARD, FEW or WEIGHT product that was split, from its whole sum.
template <int FORM>
TAO_DEVI float finish(const Args& a, float v, long long row, int col, bool is_bf16) {
  if constexpr (FORM == FORWARD || FORM == FEW) {
    if (a.bias) v += load1(a.bias, col, is_bf16);
    if (a.z) static_cast<uint16_t*>(a.z)[row * a.z_stride + col] = pack1(v, is_bf16);
    v = activate(v, a.act);
    if (a.residual) v += load1(a.residual, row * a.r_stride + col, is_bf16);
  }
  return v;
}

// Maps: FORWARD: x, W, -, U.  FEW: W, x, U, -.  INPUT: dz, W, du, U.  WEIGHT: dz, x, du, -.
template <int FORM, int BN, bool GATED, bool SPLIT, bool PAIR, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ CUtensorMap map_a2, const __grid_constant__ CUtensorMap map_b2,
                   const Args a) {
  using namespace tc;
  using C = Cfg<FORM, BN, GATED, SPLIT, PAIR>;
  static_assert(!PAIR || (BN == 256 && FORM != FEW && (!SPLIT || FORM == WEIGHT)), "");
  extern __shared__ __align__(1024) uint8_t sm[];
  uint8_t* const staging_all = sm + C::STAGES * C::STAGE;
  uint64_t* const full = reinterpret_cast<uint64_t*>(staging_all + C::STAGING);
  uint64_t* const empty = full + C::STAGES;
  uint64_t* const acc_full = empty + C::STAGES;  // [2]
  uint64_t* const acc_empty = acc_full + 2;      // [2]
  uint64_t* const over = acc_empty + 2;
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(over + 1);
  volatile int* const abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* const first = reinterpret_cast<int*>(staging_all + C::STAGING + 512);  // [groups + 2]
  int* const ends = first + kMostGroups + 2;                                  // [groups + 1]

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (smem_u32(sm) & 1023u) {  // 128-byte swizzled tiles start on 1024 bytes
    if (tid == 0) atomicOr(&g_error, kErrState);
    return;
  }
  constexpr bool is_bf16 = BF16;
  const int rank = SPLIT || PAIR ? (int)cluster_rank() : 0;
  constexpr int TOGETHER = PAIR ? 2 : 1;  // blocks of a tile, or of a part of its terms
  const int half_of_pair = PAIR ? rank & 1 : 0, first_of_pair = rank - half_of_pair, part_of_split = rank / TOGETHER;
  const int start = SPLIT ? (int)blockIdx.x / (a.split * TOGETHER) : (int)blockIdx.x / TOGETHER;
  const int step = SPLIT ? 1 << 30 : (int)gridDim.x / TOGETHER;
  // this block's part of a tile's steps
  auto part = [&](const Tile& t, int& k0) {
    if constexpr (!SPLIT) return k0 = 0, t.blocks;
    k0 = (int)((long long)t.blocks * part_of_split / a.split);
    return (int)((long long)t.blocks * (part_of_split + 1) / a.split) - k0;
  };
  // 64 terms of a tile into slot s, by one thread
  auto fetch = [&](const Tile& tile, int kb, int s) {
    uint8_t* const sa = sm + s * C::STAGE;
    uint8_t* const sb = sa + C::A;
    if constexpr (PAIR) {  // this block's 128 rows of A and its half of B; both blocks' copies arrive at the first one's
      if (half_of_pair == 0) mbar_expect_tx(&full[s], 2 * C::STAGE);
      const uint32_t bar = peer(smem_u32(&full[s]), first_of_pair);
      const int row0 = tile.row0 + half_of_pair * 128, col0 = tile.col0 + half_of_pair * 128;
      if constexpr (FORM == WEIGHT) {
        const int k = tile.from + kb * kTerms;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          tma_3d_pair(sa + j * 8192, tile.second ? &map_a2 : &map_a, row0 + j * 64, k, 0, bar);
          tma_3d_pair(sb + j * 8192, &map_b, col0 + j * 64, k, 0, bar);
        }
        return;
      }
      const int each = FORM == INPUT ? tile.blocks / a.pairs : tile.blocks;
      const bool other = kb >= each;
      const int k = (kb - (other ? each : 0)) * kTerms;
      tma_3d_pair(sa, other ? &map_a2 : &map_a, k, row0, 0, bar);
      if constexpr (FORM == FORWARD) {
        if constexpr (GATED)
          tma_3d_pair(sb, half_of_pair ? &map_b2 : &map_b, k, tile.col0, tile.group, bar);
        else
          tma_3d_pair(sb, &map_b, k, col0, tile.group, bar);
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) tma_3d_pair(sb + j * 8192, other ? &map_b2 : &map_b, col0 + j * 64, k, tile.group, bar);
      }
      return;
    }
    mbar_expect_tx(&full[s], C::STAGE);
    if constexpr (FORM == FORWARD) {
      const int k = kb * kTerms;
      tma_3d(sa, &map_a, k, tile.row0, 0, &full[s]);
      tma_3d(sb, &map_b, k, tile.col0, tile.group, &full[s]);
      if constexpr (GATED) tma_3d(sb + C::B / 2, &map_b2, k, tile.col0, tile.group, &full[s]);
    } else if constexpr (FORM == FEW) {
      const int k = kb * kTerms;
      tma_3d(sa, &map_a, k, tile.col0, tile.group, &full[s]);
      if constexpr (GATED) tma_3d(sa + C::A / 2, &map_a2, k, tile.col0, tile.group, &full[s]);
      tma_3d(sb, &map_b, k, tile.row0, 0, &full[s]);
    } else if constexpr (FORM == INPUT) {
      const int each = tile.blocks / a.pairs;
      const bool other = kb >= each;
      const int k = (kb - (other ? each : 0)) * kTerms;
      tma_3d(sa, other ? &map_a2 : &map_a, k, tile.row0, 0, &full[s]);
#pragma unroll
      for (int j = 0; j < BN / 64; ++j)
        tma_3d(sb + j * 8192, other ? &map_b2 : &map_b, tile.col0 + j * 64, k, tile.group, &full[s]);
    } else {
      const int k = tile.from + kb * kTerms;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        tma_3d(sa + j * 8192, tile.second ? &map_a2 : &map_a, tile.row0 + j * 64, k, 0, &full[s]);
#pragma unroll
      for (int j = 0; j < BN / 64; ++j) tma_3d(sb + j * 8192, &map_b, tile.col0 + j * 64, k, 0, &full[s]);
    }
  };
  int early = 0, group = 0;  // steps of the first tile that are fetched while the rest of the block sets itself up
  if (warp == kWorkers) {
    if (lane == 0) {
      for (int i = 0; i < C::STAGES; ++i) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&acc_full[i], 1);
        mbar_init(&acc_empty[i], PAIR ? 2 * kWorkers : kWorkers);
      }
      mbar_init(over, 1);
      *abort = 0;
      fence_mbar_init();
    }
    __syncwarp();
    if (!a.offsets && !PAIR) {
      const Tile tile = tile_of<FORM, C>(a, first, ends, start, group);  // there is one: no block is launched without
      int k0;
      early = min(part(tile, k0), C::STAGES);
      if (lane == 0)
        for (int i = 0; i < early; ++i) fetch(tile, k0 + i, i);
    }
  }
  if (warp == 0) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(C::TMEM));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(C::TMEM));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
  }
  if constexpr (!SPLIT)
    if (warp == 2 && a.offsets) make_lists<C>(a, first, ends, lane);
  fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // both blocks' barriers and accumulators are there
  fence_after();
  const uint32_t tbase = *tmem_slot;
  if constexpr (SPLIT && !PAIR) cluster_arrive();  // this block has begun: its shared memory can be written to

  int total;
  if (FORM == WEIGHT)
    total = (a.depth + C::DOWN - 1) / C::DOWN * ((a.cols + C::CT - 1) / C::CT) * a.groups * a.pairs;
  else
    total = a.offsets ? first[a.groups + 1] : (a.rows + C::TT - 1) / C::TT * ((a.cols + C::CT - 1) / C::CT);

  if (warp == kWorkers) {
    // ---- fetches operands
    int fetched = 0, s = 0, phase = 0;
    bool ok = true;
    for (int t = start; ok && t < total; t += step) {
      const Tile tile = tile_of<FORM, C>(a, first, ends, t, group);
      int k0;
      const int blocks = part(tile, k0);
      for (int kb = k0; kb < k0 + blocks; ++kb) {
        if (fetched >= early) {
          if (!(ok = warp_wait_for(&empty[s], phase ^ 1, abort))) break;
          if (lane == 0) fetch(tile, kb, s);
          __syncwarp();
        }
        ++fetched;
        if (++s == C::STAGES) s = 0, phase ^= 1;
      }
    }
    // the ends of the products that read the last slots arrive here too (PAIR: from the first block) before the block ends
#pragma unroll 1
    for (int i = 0; ok && i < C::STAGES; ++i) {
      ok = warp_wait_for(&empty[s], phase ^ 1, abort);
      if (++s == C::STAGES) s = 0, phase ^= 1;
    }
    if (!ok && !half_of_pair) {  // copies in flight (PAIR: both blocks') have their time before the block ends
      fetched = max(fetched, early);
      for (int i = max(fetched - C::STAGES, 0); i < fetched; ++i) mbar_wait(&full[i % C::STAGES], i / C::STAGES & 1, nullptr);
    }
    if (half_of_pair) mbar_wait(over, 0, nullptr);  // it arrives at both blocks: the first one's next warp waits for its own
  } else if (warp == kWorkers + 1) {
    // ---- issues the products
    const uint32_t type_bits = is_bf16 ? 1u << 7 | 1u << 10 : 0u;
    const uint32_t idesc = (idesc_bf16(PAIR ? 256 : 128, BN, C::A_MN, C::B_MN) & ~(1u << 7 | 1u << 10)) | type_bits;
    constexpr int STEP_A = (C::A_MN ? 2048 : 32) >> 4, STEP_B = (C::B_MN ? 2048 : 32) >> 4;  // 16 terms on
    const uint64_t desc_a = sdesc(smem_u32(sm), C::A_MN ? 8192 : 16, 1024);
    const uint64_t desc_b = sdesc(smem_u32(sm) + C::A, C::B_MN ? 8192 : 16, 1024);
    int s = 0, phase = 0, set = 0, set_phase = 0;
    bool ok = true;
    for (int t = half_of_pair ? total : start; ok && t < total; t += step) {  // PAIR: the first block's for both
      const Tile tile = tile_of<FORM, C>(a, first, ends, t, group);
      int k0;
      const int blocks = part(tile, k0);
      if (blocks == 0) continue;
      if (!(ok = warp_wait_for(&acc_empty[set], set_phase ^ 1, abort))) break;
      fence_after();
      const uint32_t acc = tbase + set * C::ACC;
      bool ready = arrived(&full[s], phase);
#pragma unroll 1
      for (int kb = 0; kb < blocks; ++kb) {
        if (!__all_sync(0xffffffffu, ready) && !(ok = warp_wait_for(&full[s], phase, abort))) break;
        fence_after();
        const int next = s + 1 == C::STAGES ? 0 : s + 1, next_phase = s + 1 == C::STAGES ? phase ^ 1 : phase;
        ready = arrived(&full[next], next_phase);  // its answer is on its way while these products are issued
        int steps = kTerms / 16;
        if constexpr (FORM == WEIGHT) {  // the last rows may be fewer than 64
          const int left = tile.upto - tile.from - (k0 + kb) * kTerms;
          if (left < kTerms) {
            steps = (left + 15) / 16;
            const int rows = steps * 16 - left;  // terms of the last product that are other rows'
            if (a.offsets && rows > 0) {
              for (int i = lane; i < rows * 8 * (2 + BN / 64); i += 32)
                *reinterpret_cast<uint4*>(sm + s * C::STAGE + (i / (rows * 8)) * 8192 + (left + i / 8 % rows) * 128 +
                                          (i & 7) * 16) = make_uint4(0, 0, 0, 0);
              fence_proxy_async();
              __syncwarp();
            }
          }
        }
        // descriptors count 16 bytes and are added up
        const uint64_t da = desc_a + s * (C::STAGE >> 4), db = desc_b + s * (C::STAGE >> 4);
        if (elected()) {
#pragma unroll
          for (int k = 0; k < kTerms / 16; ++k) {
            if (FORM == WEIGHT && k >= steps) break;
            if constexpr (PAIR)
              multiply_pair(acc, da + k * STEP_A, db + k * STEP_B, idesc, k > 0 ? 1 : kb);
            else
              multiply(acc, da + k * STEP_A, db + k * STEP_B, idesc, k > 0 ? 1 : kb);
            if constexpr (FORM == FEW && GATED)
              multiply(acc + BN, da + (C::A / 2 >> 4) + k * STEP_A, db + k * STEP_B, idesc, k > 0 ? 1 : kb);
          }
          if constexpr (PAIR)
            commit_pair(&empty[s], first_of_pair);
          else
            commit(&empty[s]);
        }
        __syncwarp();
        s = next, phase = next_phase;
      }
      if (!ok) break;
      if (elected()) {
        if constexpr (PAIR)
          commit_pair(&acc_full[set], first_of_pair);
        else
          commit(&acc_full[set]);
      }
      __syncwarp();
      if (++set == C::SETS) set = 0, set_phase ^= 1;
    }
    if (elected()) {  // nothing is in flight when the block ends
      if constexpr (!PAIR)
        commit(over);
      else if (half_of_pair == 0)
        commit_pair(over, first_of_pair);
      if (half_of_pair == 0) mbar_wait(over, 0, nullptr);
    }
    __syncwarp();
  } else {
    // ---- turns sums into outputs: a warp has the rows of its quarter of TMEM, and half of the columns
    const int quarter = warp & 3, half = warp >> 2;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    uint8_t* const staging = staging_all + warp * 2048;
    int set = 0, set_phase = 0;
    bool ok = true;
    for (int t = start; ok && t < total; t += step) {
      const Tile tile = tile_of<FORM, C>(a, first, ends, t, group);
      int k0;
      const int blocks = part(tile, k0);
      const uint32_t acc = tbase + set * C::ACC + lanes;
      if (blocks && (SPLIT || FORM == FEW)) {
        if (!(ok = warp_wait_for(&acc_full[set], set_phase, abort, FORM == WEIGHT ? blocks : 0))) break;
        fence_after();
      }
      if constexpr (SPLIT) {
        break;  // the block's one tile: below
      } else if constexpr (FORM == FEW) {
        constexpr int W = BN / 2;
        const int col = tile.col0 + quarter * 32 + lane, rows = tile.rows - half * W;
        if (rows > 0) {  // the same for the warp
          float v[W], u[W];
          if (blocks) {
            load_columns(acc + half * W, v);
            if constexpr (GATED) load_columns(acc + BN + half * W, u);
          } else {
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = 0.f, u[i] = 0.f;
          }
          if (col < a.cols) {
            const long long row0 = tile.row0 + half * W;
            if (a.bias) {
              const float bias = load1(a.bias, col, is_bf16);
#pragma unroll
              for (int i = 0; i < W; ++i) v[i] += bias;
            }
            // a column of W values, a row apart
            auto put = [&](void* to, long long stride, const float (&w)[W]) {
              uint16_t* out = static_cast<uint16_t*>(to) + row0 * stride + col;
#pragma unroll
              for (int i = 0; i < W; ++i, out += stride)
                if (i < rows) *out = pack1(w[i], is_bf16);
            };
            if (a.z) {
              if constexpr (GATED) {
                const auto put24 = [&](void* upper, uint8_t* lower, const float (&w)[W]) {
                  const long long at = row0 * a.z_stride + col;
#pragma unroll
                  for (int i = 0; i < W; ++i) {
                    const uint32_t b = bits24(w[i]);
                    if (i < rows) {
                      static_cast<uint16_t*>(upper)[at + i * a.z_stride] = (uint16_t)(b >> 16);
                      lower[at + i * a.z_stride] = (uint8_t)(b >> 8);
                    }
                  }
                };
                put24(a.z, a.low, v);
                put24(a.u, a.low + a.rows * a.z_stride, u);
              } else {
                put(a.z, a.z_stride, v);
              }
            }
            activate_all(v, a.act);
            if constexpr (GATED) {
#pragma unroll
              for (int i = 0; i < W; ++i) v[i] *= u[i];
            }
            if (a.residual) {
              const uint16_t* in = static_cast<const uint16_t*>(a.residual) + row0 * a.r_stride + col;
#pragma unroll
              for (int i = 0; i < W; ++i, in += a.r_stride)
                if (i < rows) v[i] += unpack1(*in, is_bf16);
            }
            put(a.y, a.cols, v);
          }
        }
        if (blocks) {
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[set]);
        }
      } else {
        constexpr int HALF = C::CT / 2;
        const int down = half_of_pair * 128 + quarter * 32;
        const long long row0 = tile.row0 + down;
        const int rows = tile.rows - down;
        uint16_t* y = static_cast<uint16_t*>(FORM == WEIGHT && tile.second ? a.u : a.y);
        if constexpr (FORM == WEIGHT) y += (long long)tile.group * a.depth * a.cols;
        const auto bias_of = [&](int c0) {  // of column `lane` of a chunk
          const int col = tile.col0 + c0 + lane;
          return FORM == FORWARD && a.bias && c0 < (half + 1) * HALF && col < a.cols ? load1(a.bias, col, is_bf16) : 0.f;
        };
        float bias = bias_of(half * HALF);
        if (blocks) {  // all that is not the sums is on its way before them
          if (!(ok = warp_wait_for(&acc_full[set], set_phase, abort, FORM == WEIGHT ? blocks : 0))) break;
          fence_after();
        }
#pragma unroll 1
        for (int c0 = half * HALF; c0 < (half + 1) * HALF; c0 += 32) {
          const int col = tile.col0 + c0, cols = a.cols - col;
          float v[32], u[GATED ? 32 : 1];
          if (blocks) {
            load_columns(acc + c0, v);
            if constexpr (GATED) load_columns(acc + BN / 2 + c0, u);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0.f, u[GATED ? i : 0] = 0.f;
          }
          if (rows <= 0 || cols <= 0) continue;  // the same for the warp
          if constexpr (FORM == FORWARD) {
            if (a.bias) {
              reinterpret_cast<float*>(staging)[lane] = bias;
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const float4 b = *reinterpret_cast<const float4*>(staging + i * 4);
                v[i] += b.x, v[i + 1] += b.y, v[i + 2] += b.z, v[i + 3] += b.w;
              }
              __syncwarp();
              bias = bias_of(c0 + 32);
            }
            if (a.z) {
              const long long at = row0 * a.z_stride + col;
              if constexpr (GATED) {  // up to the end of its padded row
                const int room = (int)a.z_stride - col;
                put_rows24(staging, v, static_cast<uint16_t*>(a.z) + at, a.low + at, a.z_stride, rows, room, lane);
                put_rows24(staging, u, static_cast<uint16_t*>(a.u) + at, a.low + a.rows * a.z_stride + at, a.z_stride, rows,
                           room, lane);
              } else {
                put_rows(staging, v, is_bf16, static_cast<uint16_t*>(a.z) + at, a.z_stride, rows, cols, a.wide, lane);
              }
            }
            activate_all(v, a.act);
            if constexpr (GATED) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] *= u[i];
            }
            if (a.residual) {
              move_rows(staging, const_cast<uint16_t*>(static_cast<const uint16_t*>(a.residual)) + row0 * a.r_stride + col,
                        a.r_stride, rows, cols, a.wide, true, lane);
              __syncwarp();
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const uint4 w = *reinterpret_cast<const uint4*>(staging + staged(lane, c));
                const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float2 f = unpack(words[i], is_bf16);
                  v[c * 8 + i * 2] += f.x;
                  v[c * 8 + i * 2 + 1] += f.y;
                }
              }
              __syncwarp();
            }
          }
          put_rows(staging, v, is_bf16, y + row0 * a.cols + col, a.cols, rows, cols, a.wide, lane);
        }
        if (blocks) {
          fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (PAIR)
              arrive_at(peer(smem_u32(&acc_empty[set]), first_of_pair));
            else
              mbar_arrive(&acc_empty[set]);
          }
        }
      }
      if (blocks && ++set == C::SETS) set = 0, set_phase ^= 1;
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();

  if constexpr (SPLIT) {
    // Every block adds a share of the tile's outputs, the blocks' parts in order of their ranks.  FEW: the parts of a
    // row of x (128 outputs, neighbours in a warp) are written to the block that adds them, one barrier.  Else a
    // thread has a row of the tile, whose remote writes would not meet: each block keeps its part, the others read it.
    fence_after();
    const Tile tile = tile_of<FORM, C>(a, first, ends, start, group);
    int k0;
    const int blocks = part(tile, k0);
    const int share = FORM == FEW ? (min(BN, tile.rows) + a.split - 1) / a.split : 0;  // rows of x of a block
    constexpr int ROW = FORM == FEW ? 128 : BN + 4;                                   // floats of a row of a part
    float* const sums = reinterpret_cast<float*>(FORM == FEW ? staging_all + 512 : sm);
    if constexpr (!PAIR) cluster_wait();
    if (warp < kWorkers) {
      constexpr int W = BN / 2 < 32 ? BN / 2 : 32;
      const int r = (warp & 3) * 32 + lane, begin = (warp >> 2) * (BN / 2);
      const uint32_t acc = tbase + ((uint32_t)((warp & 3) * 32) << 16);
      int to = FORM == FEW ? begin / share : 0, in = begin - to * share;
#pragma unroll 1
      for (int c0 = begin; c0 < begin + BN / 2; c0 += W) {
        if (FORM == FEW && c0 >= tile.rows) break;
        float v[W];
        if (blocks) {
          load_columns(acc + c0, v);
        } else {
#pragma unroll
          for (int i = 0; i < W; ++i) v[i] = 0.f;
        }
        if constexpr (FORM == FEW) {
#pragma unroll
          for (int i = 0; i < W; ++i) {
            if (c0 + i < tile.rows) put_peer(peer(smem_u32(sums + (rank * share + in) * ROW + r), to), v[i]);
            if (++in == share) in = 0, ++to;
          }
        } else {
#pragma unroll
          for (int i = 0; i < W; i += 4)
            *reinterpret_cast<float4*>(sums + r * ROW + c0 + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
      }
    }
    cluster_sync();
    uint16_t* y = static_cast<uint16_t*>(FORM == WEIGHT && tile.second ? a.u : a.y);
    constexpr int ACROSS = FORM == FEW ? 32 : BN / 4;
    const int first_row = FORM == FEW ? rank * share : half_of_pair * 128;
    const int rows = min(FORM == FEW ? share : 128, tile.rows - first_row);
    const int begin = FORM == FEW ? tid : part_of_split * kThreads + tid, stride = FORM == FEW ? kThreads : kThreads * a.split;
    constexpr int AT_ONCE = 4;  // sums whose parts are on their way
    for (int i0 = begin; i0 < ACROSS * rows; i0 += stride * AT_ONCE) {
      float4 v[AT_ONCE];
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) v[e] = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int q = 0; q < a.split; ++q) {
        float4 w[AT_ONCE];
#pragma unroll
        for (int e = 0; e < AT_ONCE; ++e) {
          const int i = min(i0 + e * stride, ACROSS * rows - 1), r = i / ACROSS, c = i % ACROSS * 4;
          w[e] = FORM == FEW ? *reinterpret_cast<const float4*>(sums + (q * share + r) * ROW + c)
                             : ld_cluster(smem_u32(sums + r * ROW + c), q * TOGETHER + half_of_pair);
        }
#pragma unroll
        for (int e = 0; e < AT_ONCE; ++e) v[e].x += w[e].x, v[e].y += w[e].y, v[e].z += w[e].z, v[e].w += w[e].w;
      }
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) {
        const int i = i0 + e * stride, r = i / ACROSS, col = tile.col0 + i % ACROSS * 4;
        if (i >= ACROSS * rows || col >= a.cols) continue;
        const long long row = tile.row0 + first_row + r;
        float o[4] = {v[e].x, v[e].y, v[e].z, v[e].w};
        if (FORM == FORWARD || FORM == FEW) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (col + j < a.cols) o[j] = finish<FORM>(a, o[j], row, col + j, is_bf16);
        }
        uint16_t* const out = y + row * a.cols + col;
        if (a.wide) {
          *reinterpret_cast<uint2*>(out) = make_uint2(pack(o[0], o[1], is_bf16), pack(o[2], o[3], is_bf16));
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (col + j < a.cols) out[j] = pack1(o[j], is_bf16);
        }
      }
    }
    __syncwarp();
    if constexpr (FORM != FEW) cluster_sync();  // the others' reads of this block's part are over
  }
  if constexpr (PAIR) {
    cluster_sync();  // neither's products, copies or arrivals need the other any more: each block has waited for those at its own
    if (warp == 0)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(C::TMEM));
  } else if (warp == 0) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(C::TMEM));
  }
}

}  // namespace product
}  // namespace tao
