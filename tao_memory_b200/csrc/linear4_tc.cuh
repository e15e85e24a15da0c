// The 4-bit product of more than a few rows (up to 64 at a time) on tcgen05: with 17 rows and more the
// legacy mma and its operand loads take several times as long as the weights' bytes.
//
// A block computes 128 rows of W (8 row tiles) against 64 rows of x over its k, a cluster's blocks a part of
// k each.  Per 128 k:  eight warps make 16-bit floats (code - zero, exact) of a tile's codes each and write
// them to the A operand (K-major, 128-byte swizzle, two buffers); a ninth issues the 8 products of 16 k into
// TMEM, an accumulator of its own for each scale group (two sets); and while those run, the eight read the
// block before's accumulators, scale them and add them in fp32 registers, row and column half a thread.  So no
// weight is rounded and every sum's order is fixed.  Eight more warps bring x to five slots of the B operand;
// codes and scales come to eight of a ring.  All copies have a memory's latency and more.
//
// 64x8192x8192 takes 28.9 us, 1.27 TB/s of its bytes and 0.30 PFLOP/s.  What bounds it is the eight warps'
// chain of a block: unpacking and the operand's writes to shared memory, fence, barrier, and the sums (about
// 1600 cycles where the products take 260 and the bytes 350).  It was 35.3 us while the eight brought x too,
// 40.5 us while one of them issued the products, and sixteen warps with half a tile each took 32.5 us: the
// same shared memory writes, and twice the warps at the barrier.
#pragma once
#include "linear4.cuh"
#include "tcgen05.cuh"

namespace tao {

static __device__ int g_linear4_error;  // an expired wait, until tao_linear4_check

// One lane of a warp that has met, the same for all that ask.
TAO_DEVI bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}

// 16 consecutive fp32 columns of this thread's TMEM lane.
TAO_DEVI void tmem_ld16(uint32_t at, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

template <int GROUP>
struct Linear4Tc {
  static constexpr int WORKERS = 8, LOADERS = 8, THREADS = 32 * (WORKERS + 1 + LOADERS), COLS = 64, GROUPS = 128 / GROUP;
  static constexpr int A = 128 * 256, X = COLS * 256, XSLOTS = 5, CODES = 8 * Block4<GROUP>::BYTES, CSLOTS = 8;
  static constexpr int RAW = 4;  // slots of x as e4m3
  static constexpr int TMEM = 2 * GROUPS * COLS;
  static constexpr int SMEM = 1024 + 2 * A + XSLOTS * X + CSLOTS * CODES + 64;
  static_assert(SMEM <= 227 * 1024, "");
};

// M: the operands' type.  BF16: the type of scales, bias and y.
template <class M, bool BF16, int GROUP>
__global__ void __launch_bounds__(Linear4Tc<GROUP>::THREADS, 1) linear4_tc_kernel(const Linear4Args a) {
  using namespace tc;
  using C = Linear4Tc<GROUP>;
  using B4 = Block4<GROUP>;
  extern __shared__ uint8_t raw[];
  uint8_t* const sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  uint8_t *const sA = sm, *const sX = sm + 2 * C::A, *const sC = sX + C::XSLOTS * C::X;
  uint64_t* const bar = reinterpret_cast<uint64_t*>(sC + C::CSLOTS * C::CODES);  // of each set of accumulators
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bar + 2);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int m0 = blockIdx.y * C::COLS, rows = min(a.rows - m0, C::COLS);
  const int rank = a.shift ? (int)cluster_rank() : 0, tile0 = (blockIdx.x >> a.shift) * 8;
  const int k0 = a.kblocks * rank >> a.shift, nb = (a.kblocks * (rank + 1) >> a.shift) - k0;
  const bool has_zeros = a.w.zeros != nullptr;

  // this warp's row tile (one beyond the matrix repeats the last), and the row whose sums this thread adds
  const uint32_t first = (uint32_t)min(tile0 + warp, a.tiles - 1) * a.kblocks + k0;
  uint8_t* const my_codes = sC + warp * B4::BYTES;
  const int r = (warp & 3) * 32 + lane, half = warp >> 2;
  const uint8_t* const scales = sC + r / 16 * B4::BYTES + 1024 + (r & 7) * (4 * C::GROUPS) + (r >> 3 & 1) * 2;

  constexpr int LOADING = 32 * C::LOADERS, STEP = LOADING / 16, EACH = C::COLS / STEP;
  // A loader brings chunk c of 8 k of rows m, m + 16, m + 32, m + 48 of x to `place` and 16 rows on in a slot
  // of the B operand.  e4m3 is widened on its way, from a ring of raw chunks in the last two slots' room.
  const int loader = tid - 32 * (C::WORKERS + 1), m = loader >> 4, c = loader & 15;
  const uint32_t place = (c >> 3) * (C::COLS * 128) + m * 128 + (((c & 7) ^ (m & 7)) << 4);
  const bool copied = a.wide && a.x_type != TAO_TYPE_E4M3, staged = a.wide && a.x_type == TAO_TYPE_E4M3;
  const long long x_at = (long long)(m0 + m) * a.x_stride + k0 * 128 + c * 8;
  const uint8_t* const x = static_cast<const uint8_t*>(a.x) + (staged ? x_at : x_at * 2);
  const long long x_step = (staged ? STEP : 2 * STEP) * a.x_stride;  // of STEP rows, in bytes
  uint8_t* const sRaw = sX + 3 * C::X + loader * 8;
  auto x_slot = [&](int kb) { return sX + kb % (copied ? C::XSLOTS : 3) * C::X; };
  auto copy_codes = [&](int kb) {
    if (kb < nb) B4::issue(smem_u32(my_codes + (kb & (C::CSLOTS - 1)) * C::CODES), a.w, first + kb, lane);
    cp_commit();
  };
  auto copy_x = [&](int kb) {
    const bool in = (k0 + kb) * 128 + c * 8 < a.k;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      if (kb >= nb || m + STEP * j >= rows) break;
      if (copied)
        cp_async16(smem_u32(x_slot(kb) + place + j * STEP * 128), in ? x + kb * 256 + j * x_step : x, in);
      else if (staged)
        cp_async8(smem_u32(sRaw + (kb & (C::RAW - 1)) * (C::X / 2) + j * (LOADING * 8)), in ? x + kb * 128 + j * x_step : x, in);
    }
    cp_commit();
  };
  uint4 ahead[EACH];  // x off its alignment, a block ahead
  auto fetch = [&](int kb) {
#pragma unroll
    for (int j = 0; j < EACH; ++j)
      if (kb < nb && m + STEP * j < rows) ahead[j] = chunk_of(a, m0 + m + STEP * j, (k0 + kb) * 128 + c * 8);
  };
  if (warp < C::WORKERS) {
    for (int kb = 0; kb < 6; ++kb) copy_codes(kb);
  } else if (warp > C::WORKERS) {
    for (int kb = 0; kb < 3; ++kb) copy_x(kb);
    if (!a.wide) fetch(0);
  }

  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(C::TMEM));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (tid == 0) {
    mbar_init(&bar[0], 1);
    mbar_init(&bar[1], 1);
    fence_mbar_init();
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tbase = *tmem_slot;

  float acc[32] = {};
  bool ok = true;  // after a wait that ran out nothing more is waited for
  // adds block kb's accumulators
  auto add = [&](int kb) {
    if (ok) ok = mbar_wait(&bar[kb & 1], kb >> 1 & 1, &g_linear4_error);
    __syncwarp();
    fence_after();
#pragma unroll
    for (int j = 0; j < C::GROUPS; ++j) {
      const uint16_t bits = *reinterpret_cast<const uint16_t*>(scales + (kb & (C::CSLOTS - 1)) * C::CODES + j * 4);
      const float s = BF16 ? __uint_as_float((uint32_t)bits << 16) : __half2float(__ushort_as_half(bits));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[16];
        tmem_ld16(tbase + ((uint32_t)((warp & 3) * 32) << 16) + ((kb & 1) * C::GROUPS + j) * C::COLS + half * 32 + h * 16, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[h * 16 + i] += s * v[i];
      }
    }
    fence_before();
  };

  // one barrier a block: its operands are written, and what it overwrites has been read
  if (warp == C::WORKERS) {
    constexpr uint32_t TYPE = std::is_same<M, MmaBf16>::value ? 1u << 7 | 1u << 10 : 0u;  // bf16, or fp16
    constexpr uint32_t I = (idesc_bf16(128, C::COLS, 0, 0) & ~(1u << 7 | 1u << 10)) | TYPE;
#pragma unroll 1
    for (int kb = 0; kb < nb; ++kb) {
      const uint64_t pa = sdesc(smem_u32(sA + (kb & 1) * C::A), 16, 1024);
      const uint64_t px = sdesc(smem_u32(x_slot(kb)), 16, 1024);  // addresses count 16 bytes
      __syncthreads();
      fence_after();
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          tc::mma(tbase + ((kb & 1) * C::GROUPS + k * 16 / GROUP) * C::COLS,
                  pa + (((k >> 2) * (C::A / 2) + (k & 3) * 32) >> 4), px + (((k >> 2) * (C::X / 2) + (k & 3) * 32) >> 4),
                  I, k * 16 % GROUP ? 1u : 0u);
        commit(&bar[kb & 1]);
      }
      __syncwarp();
    }
  } else if (warp < C::WORKERS) {
#pragma unroll 1
    for (int kb = 0; kb < nb; ++kb) {
      cp_wait<5>();  // this block's codes; younger ones may be on their way
      __syncwarp();
      // A: two chunks of 16 bytes (rows g, g + 8) for each 32 k; odd rows' lanes take the parts of 64 k in the
      // other order, so that 8 lanes write to all banks
      B4 b;
      b.load(my_codes + (kb & (C::CSLOTS - 1)) * C::CODES, has_zeros, lane);
      const int odd = g & 1;
      if (odd) b.swap_parts();
      uint8_t* const to = sA + (kb & 1) * C::A + (warp * 16 + g) * 128;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        uint32_t v[2][4];
        b.template operands16<M>(u, v);
        uint8_t* const at = to + (u >> 1) * (C::A / 2) + (((((u & 1) ^ odd) * 4 + t) ^ g) << 4);
        *reinterpret_cast<uint4*>(at) = make_uint4(v[0][0], v[0][2], v[1][0], v[1][2]);
        *reinterpret_cast<uint4*>(at + 8 * 128) = make_uint4(v[0][1], v[0][3], v[1][1], v[1][3]);
      }
      fence_proxy_async();
      fence_before();
      __syncthreads();
      if (kb > 0) add(kb - 1);
      copy_codes(kb + 6);  // into the slot of block kb - 2, whose scales all have used
    }
    add(nb - 1);
    if (!ok) mbar_wait(&bar[(nb - 1) & 1], (nb - 1) >> 1 & 1, nullptr);  // what is in flight has its time before it ends
  } else {
#pragma unroll 1
    for (int kb = 0; kb < nb; ++kb) {
      cp_wait<2>();
      if (!copied) {
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
          if (m + STEP * j >= rows) break;
          uint4 v = ahead[j];
          if (staged) {
            const uint2 raw = *reinterpret_cast<const uint2*>(sRaw + (kb & (C::RAW - 1)) * (C::X / 2) + j * (LOADING * 8));
            v.x = raw.x, v.y = raw.y;
          }
          if (a.x_type == TAO_TYPE_E4M3) v = widen_e4m3(v);
          *reinterpret_cast<uint4*>(x_slot(kb) + place + j * STEP * 128) = v;
        }
      }
      fence_proxy_async();
      __syncthreads();
      if (!a.wide) fetch(kb + 1);
      copy_x(kb + 3);  // into the slot of block kb - 2: its sums were added before this barrier
    }
  }
  cp_wait<0>();
  fence_before();
  __syncthreads();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(C::TMEM));

  using T = std::conditional_t<BF16, bf16, __half>;
  const T* bias = static_cast<const T*>(a.bias);
  auto put = [&](int m, int n, float o) {
    if (a.x_scale) o *= a.x_scale[m0 + m];
    T* y = static_cast<T*>(a.y) + (long long)(m0 + m) * a.n + n;
    if constexpr (BF16)
      *y = tobf(o + (bias ? bf(bias[n]) : 0.f));
    else
      *y = __float2half_rn(o + (bias ? __half2float(bias[n]) : 0.f));
  };
  const int n0 = tile0 * 16;
  if (!a.shift) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (warp < C::WORKERS && half * 32 + i < rows && n0 + r < a.n) put(half * 32 + i, n0 + r, acc[i]);
    return;
  }
  float* sums = reinterpret_cast<float*>(sm);  // [column][128 rows], over the operands
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (warp < C::WORKERS) sums[(half * 32 + i) * 128 + r] = acc[i];
  cluster_sync();
  for (int i = (((warp << a.shift) + rank) << 5) + lane; i < rows * 32; i += C::THREADS << a.shift) {
    const int m = i >> 5, n = n0 + (i & 31) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int q = 0; q < 1 << a.shift; ++q) {
      const float4 v = ld_cluster(smem_u32(sums + m * 128 + (i & 31) * 4), q);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    const float o[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.n) put(m, n + e, o[e]);
  }
  cluster_sync();  // the others' reads of these sums are over
}

}  // namespace tao
