// A mixture-of-experts layer for a few tokens, in one kernel.
//
//   p = softmax(x R^T), the top_k largest of a row (ties to the lowest expert), their weights
//   p or p / sum of the chosen;  out = sum over them of weight * down_e(silu(gate_e x) * (up_e x))
//
// Bound by the bytes of the chosen experts.  One cooperative launch, its blocks all resident, in
// three parts with a grid barrier between them:
//   1. logits [token][expert], 16 experts x 8 tokens to a block;
//   2. every block picks the top_k itself (the same arithmetic in all of them) and sorts the
//      (token, expert) pairs by expert; then 16 inner channels of one expert's gate and up at a
//      time, h = silu(gate) up;
//   3. 32 outputs of one expert's down at a time, a row of sums for each pair; the block that
//      completes 32 outputs adds the tokens' pairs in the order of their choice.
// Parts 1 to 3 are the same product of a few rows (few_rows.cuh): the eight warps split k, each
// streams its blocks through a ring that runs on from one unit of work to the next.
// h is kept as the sum of two bf16 (16 mantissa bits), which are two columns of one mma: with bf16
// alone its rounding would add as much to the error as the output's own.  Every sum's order is fixed.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/tao_b200.h"
#include "few_rows.cuh"

void tao_set_last_error(const char* msg);

namespace tao {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kTokens = 64;    // of a launch: a bit each of an expert's mask
constexpr int kExperts = 512;  // most experts, and
constexpr int kTop = 16;       // most of them for a token
constexpr int kCols = 8;       // tokens of an entry: (expert, up to 8 of its tokens)
constexpr int kHeader = 256;   // workspace: error word, barrier word; then the outputs' counters

struct Matrix16 {  // bf16 [experts][rows][k], the last axis contiguous
  const bf16* at;
  long long expert, row;
};

struct ExpertArgs {
  const bf16* x;
  long long x_stride;
  Matrix16 router, gate16, up16, down16;
  Four gate4, up4, down4;
  int tokens, width, inner, experts, top_k, group;
  bool renormalize;
  bf16* out;
  int* ids;          // [tokens][top_k] and their weights, or null
  float* id_weights;
  int* error;
  unsigned* barrier;
  int* counters;     // [ceil(width / 32)], zero between launches
  float* logits;     // [tokens][experts]
  bf16* h;           // [2][pairs][inner]: rounded, and what the rounding left
  float* pair_out;   // [pairs][width]
};

// 16-bit weights: blocks of 16 rows x 32 k.
struct W16 {
  static constexpr int KB = 32, BYTES = 1024;
  struct Ref {
    const bf16 *r0, *r1;
  };
  static TAO_DEVI Ref ref(const Matrix16& m, int rows, int e, int tile, int lane) {
    const int r = tile * 16 + (lane >> 2);  // rows beyond the matrix repeat its last one
    const bf16* at = m.at + e * m.expert + (lane & 3) * 8;
    return {at + min(r, rows - 1) * m.row, at + min(r + 8, rows - 1) * m.row};
  }
  static TAO_DEVI void issue(uint32_t to, const Ref& w, int kb, int k, int lane) {
    const bool in = kb * 32 + (lane & 3) * 8 < k;
    const int at = in ? kb * 32 : 0;
    cp_async16(to + lane * 16, in ? w.r0 + at : w.r0 - (lane & 3) * 8, in);
    cp_async16(to + 512 + lane * 16, in ? w.r1 + at : w.r1 - (lane & 3) * 8, in);
  }
  template <int NT, class B>
  static TAO_DEVI void compute(float (&acc)[NT][4], uint32_t at, bool, int lane, int cols, B b) {
    const uint4 w0 = lds16(at + lane * 16), w1 = lds16(at + 512 + lane * 16);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (n && n * 8 >= cols) break;
      const uint4 x = b(0, n);
      MmaBf16::mma(acc[n], w0.x, w1.x, w0.y, w1.y, x.x, x.y);
      MmaBf16::mma(acc[n], w0.z, w1.z, w0.w, w1.w, x.z, x.w);
    }
  }
};

// 4-bit weights: blocks of 16 rows x 128 k, or halves of them where the rows' part of a
// ring's stage would leave no room for two.
template <int GROUP, int KBLOCK>
struct W4 {
  static constexpr int KB = KBLOCK, CODES = KB * 8, SCALES = (KB > GROUP ? KB / GROUP : 1) * 32;
  static constexpr int BYTES = CODES + SCALES + SCALES / 2;
  static constexpr int SHARED = KB < GROUP ? GROUP / KB : 1;  // blocks under one scale
  struct Ref {
    const uint8_t *codes, *scales, *zeros;
  };
  static TAO_DEVI Ref ref(const Four& m, int rows, int k, int e, int tile, int lane) {
    const int tiles = (rows + 15) / 16, blocks = (k + 127) / 128;
    const long long at = ((long long)e * tiles + min(tile, tiles - 1)) * blocks;
    constexpr int ALL = 128 / GROUP * 32;
    return {m.codes + at * 1024 + lane * 16, reinterpret_cast<const uint8_t*>(m.scales) + at * ALL + lane * 16,
            m.zeros ? m.zeros + at * (ALL / 2) + (lane - 16) * 16 : nullptr};
  }
  static TAO_DEVI void issue(uint32_t to, const Ref& w, int kb, int, int lane) {
#pragma unroll
    for (int i = 0; i < CODES / 512; ++i)
      cp_async16(to + i * 512 + lane * 16, w.codes + kb * (long long)CODES + i * 512, true);
    if (lane < SCALES / 16)
      cp_async16(to + CODES + lane * 16, w.scales + kb / SHARED * (long long)SCALES, true);
    else if (w.zeros && lane >= 16 && lane < 16 + SCALES / 32)
      cp_async16(to + CODES + SCALES + (lane - 16) * 16, w.zeros + kb / SHARED * (long long)(SCALES / 2), true);
  }
  template <int NT, class B>
  static TAO_DEVI void compute(float (&acc)[NT][4], uint32_t at, bool zeros, int lane, int cols, B b) {
    auto scale = [&](int j, int row) { return __uint_as_float(lds_u16(at + CODES + (j * 16 + row) * 2) << 16); };
    four_block<MmaBf16, GROUP, KB, NT>(acc, at, at + CODES + SCALES, zeros, lane, cols, b, scale);
  }
};

// One unit of a part: R weight tiles against `cols` rows.
template <class W, int R, int NT>
struct Unit {
  typename W::Ref w[R];
  const bf16* x[NT];  // this lane's column of each column tile, or null
  int cols;
};

struct Shared {
  unsigned long long mask[kExperts];
  int base[kExperts];
  uint32_t entry[kExperts + kTokens * kTop / kCols];  // expert << 16 | first row << 4 | tokens
  uint16_t id[kTokens * kTop], row[kTokens * kTop];   // of a token's choices: expert, row of its pair
  float weight[kTokens * kTop];
  uint8_t token[kTokens * kTop];                      // of a pair's row
  int entries, last;
  bool ok;
};

template <int N>
TAO_DEVI void wait_open() { cp_wait<N>(); }
TAO_DEVI void wait_open(int n) {
  switch (n) {
    case 0: cp_wait<0>(); break;
    case 1: cp_wait<1>(); break;
    case 2: cp_wait<2>(); break;
    case 3: cp_wait<3>(); break;
    case 4: cp_wait<4>(); break;
    case 5: cp_wait<5>(); break;
    default: cp_wait<6>(); break;
  }
}

// The units blockIdx.x, blockIdx.x + gridDim.x, ... of a part.  `unit(u)` gives a unit; `sink(u,
// sum)` takes its sums, sum(r, column, row), where the columns of a PAIR are added in twos.
// `red` holds 8 * R * (PAIR ? 4 : 8) * NT * 16 floats.
template <class W, int R, int NT, bool PAIR, class UnitOf, class Sink>
TAO_DEVI void run_part(int units, int k, int cols_max, bool zeros, uint32_t ring, int ring_bytes, float* red,
                       UnitOf unit_of, Sink sink) {
  constexpr int COLS = PAIR ? 4 * NT : 8 * NT;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kblocks = (k + W::KB - 1) / W::KB, per = (kblocks + kWarps - 1) / kWarps;
  const int stage = R * W::BYTES + cols_max * W::KB * 2, depth = min(8, ring_bytes / stage);
  const int mine = units > (int)blockIdx.x ? (units - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
  const int total = mine * per;

  int iu = blockIdx.x, ib = 0, islot = 0, iat = 0;  // what is issued next
  Unit<W, R, NT> next;
  auto issue = [&]() {
    if (iat < total) {
      if (ib == 0) next = unit_of(iu);
      const int kb = ib * kWarps + warp;
      if (kb < kblocks) {
        const uint32_t to = ring + islot * stage;
#pragma unroll
        for (int r = 0; r < R; ++r) W::issue(to + r * W::BYTES, next.w[r], kb, k, lane);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (next.x[n]) {
#pragma unroll
            for (int u = 0; u < W::KB / 32; ++u) {
              const int at = kb * W::KB + u * 32 + t * 8;
              cp_async16(to + R * W::BYTES + ((u * cols_max + n * 8 + g) * 4 + t) * 16,
                         at < k ? next.x[n] + at : next.x[n], at < k);
            }
          }
        }
      }
      ++iat;
      if (++ib == per) {
        ib = 0;
        iu += gridDim.x;
      }
      if (++islot == depth) islot = 0;
    }
    cp_commit();
  };

  float acc[R][NT][4];
  int slot = 0;
  for (int i = 0; i < depth - 1; ++i) issue();
  for (int ui = 0, u = blockIdx.x; ui < mine; ++ui, u += gridDim.x) {
    const int cols = unit_of(u).cols;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[r][n][0] = acc[r][n][1] = acc[r][n][2] = acc[r][n][3] = 0.f;
    for (int i = 0; i < per; ++i) {
      wait_open(depth - 2);
      __syncwarp();  // the block is there for every lane, and every lane is done with the one before
      issue();
      const uint32_t at = ring + slot * stage;
      if (++slot == depth) slot = 0;
      if (i * kWarps + warp >= kblocks) continue;
      auto b = [&](int uu, int n) {
        const int m = min(n * 8 + g, cols - 1);  // columns without a row repeat one; nothing reads them
        return lds16(at + R * W::BYTES + ((uu * cols_max + m) * 4 + t) * 16);
      };
#pragma unroll
      for (int r = 0; r < R; ++r) W::template compute<NT>(acc[r], at + r * W::BYTES, zeros, lane, cols, b);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if constexpr (PAIR) {
          float* to = red + ((warp * R + r) * COLS + n * 4 + t) * 16 + g;
          to[0] = acc[r][n][0] + acc[r][n][1];
          to[8] = acc[r][n][2] + acc[r][n][3];
        } else {
          float* to = red + ((warp * R + r) * COLS + n * 8 + 2 * t) * 16 + g;
          to[0] = acc[r][n][0];
          to[16] = acc[r][n][1];
          to[8] = acc[r][n][2];
          to[24] = acc[r][n][3];
        }
      }
    __syncthreads();
    sink(u, [&](int r, int col, int row) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) s += red[((w * R + r) * COLS + col) * 16 + row];
      return s;
    });
    __syncthreads();
  }
  cp_wait<0>();
}

// All blocks of the launch meet.  The word's top bit flips when the last one arrives (block 0
// adds what the others leave to 2^31), so it needs no reset and any grid may use it next.
TAO_DEVI bool grid_meet(const ExpertArgs& a, Shared& s) {
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned add = blockIdx.x == 0 ? 0x80000000u - (gridDim.x - 1) : 1u;
    const unsigned old = (unsigned)atomic_add_release(reinterpret_cast<int*>(a.barrier), (int)add);
    bool ok = false;
    for (int i = 0; i < (1 << 22) && !ok; ++i) {  // seconds; every block is resident, so none is expected to be late
      unsigned now;
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(now) : "l"(a.barrier) : "memory");
      ok = ((now ^ old) & 0x80000000u) != 0;
    }
    fence_acquire();
    if (!ok) atomicOr(a.error, kErrWaitTimeout);
    s.ok = ok;
  }
  __syncthreads();
  return s.ok;
}

// A float's order as an unsigned's; 0 and 1 are below every number (taken, and not a number).
TAO_DEVI uint32_t order_of(float v) {
  if (v != v) return 1u;
  const uint32_t u = __float_as_uint(v + 0.f);  // -0 is 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The top_k of one token by one warp: ids and weights to shared memory.
TAO_DEVI void choose(const ExpertArgs& a, Shared& s, int token, int lane) {
  constexpr int N = kExperts / 32;
  float v[N];
  uint32_t key[N];
  bool nan = false;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = i * 32 + lane;
    key[i] = 0;
    if (i * 32 < a.experts && e < a.experts) {
      v[i] = __ldcg(a.logits + token * a.experts + e);
      key[i] = order_of(v[i]);
      nan |= v[i] != v[i];
    } else {
      v[i] = -INFINITY;
    }
  }
  nan = __any_sync(0xffffffffu, nan);
  float top = 0.f, sum = 0.f, mine = 0.f;
  int my_id = 0;
  for (int j = 0; j < a.top_k; ++j) {
    uint32_t best = 0;
    float bv = 0.f;
    int bi = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i * 32 < a.experts && key[i] > best) {
        best = key[i];
        bi = i;
        bv = v[i];
      }
    }
    const uint32_t most = __reduce_max_sync(0xffffffffu, best);
    const int e = (int)__reduce_min_sync(0xffffffffu, best == most ? (uint32_t)(bi * 32 + lane) : 0xffffffffu);
    const float chosen = __shfl_sync(0xffffffffu, bv, e & 31);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i * 32 + lane == e) key[i] = 0;
    if (j == 0) {
      top = chosen;
      if (!a.renormalize) {
#pragma unroll
        for (int i = 0; i < N; ++i) sum += i * 32 + lane < a.experts ? expf(v[i] - top) : 0.f;
        sum = warp_sum(sum);
      }
    }
    const float p = expf(chosen - top);
    if (a.renormalize) sum += p;
    if (lane == j) {
      mine = p;
      my_id = e;
    }
  }
  if (lane < a.top_k) {
    const float w = nan ? NAN : mine / sum;
    s.id[token * a.top_k + lane] = (uint16_t)my_id;
    s.weight[token * a.top_k + lane] = w;
    if (blockIdx.x == 0 && a.ids) {
      a.ids[token * a.top_k + lane] = my_id;
      a.id_weights[token * a.top_k + lane] = w;
    }
  }
}

// Pairs sorted by expert, then token; entries of up to kCols tokens.
TAO_DEVI void sort_pairs(const ExpertArgs& a, Shared& s) {
  const int pairs = a.tokens * a.top_k;
  for (int e = threadIdx.x; e < a.experts; e += kThreads) s.mask[e] = 0;
  __syncthreads();
  for (int p = threadIdx.x; p < pairs; p += kThreads) atomicOr(&s.mask[s.id[p]], 1ull << (p / a.top_k));
  __syncthreads();
  if (threadIdx.x < 32) {
    int rows = 0, entries = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int e = e0 + threadIdx.x;
      const int count = e < a.experts ? __popcll(s.mask[e]) : 0, parts = (count + kCols - 1) / kCols;
      int r = count, n = parts;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int r2 = __shfl_up_sync(0xffffffffu, r, o), n2 = __shfl_up_sync(0xffffffffu, n, o);
        if ((int)threadIdx.x >= o) {
          r += r2;
          n += n2;
        }
      }
      const int first = rows + r - count;
      if (e < a.experts) s.base[e] = first;
      for (int i = 0; i < parts; ++i)
        s.entry[entries + n - parts + i] =
            (uint32_t)e << 16 | (uint32_t)(first + i * kCols) << 4 | min(kCols, count - i * kCols);
      rows += __shfl_sync(0xffffffffu, r, 31);
      entries += __shfl_sync(0xffffffffu, n, 31);
    }
    if (threadIdx.x == 0) s.entries = entries;
  }
  __syncthreads();
  for (int p = threadIdx.x; p < pairs; p += kThreads) {
    const int t = p / a.top_k, e = s.id[p];
    const int row = s.base[e] + __popcll(s.mask[e] & ((1ull << t) - 1));
    s.row[p] = (uint16_t)row;
    s.token[row] = (uint8_t)t;
  }
  __syncthreads();
}

// The experts' matrices in the layer's format; In and Down: the forms of parts 2 and 3.
struct Layer16 {
  using In = W16;
  using Down = W16;
  static TAO_DEVI W16::Ref gate(const ExpertArgs& a, int e, int tile, int lane) {
    return W16::ref(a.gate16, a.inner, e, tile, lane);
  }
  static TAO_DEVI W16::Ref up(const ExpertArgs& a, int e, int tile, int lane) {
    return W16::ref(a.up16, a.inner, e, tile, lane);
  }
  static TAO_DEVI W16::Ref down(const ExpertArgs& a, int e, int tile, int lane) {
    return W16::ref(a.down16, a.width, e, tile, lane);
  }
  static TAO_DEVI bool zeros(const ExpertArgs&) { return false; }
};
template <int GROUP>
struct Layer4 {
  using In = W4<GROUP, 128>;
  using Down = W4<GROUP, 64>;
  static TAO_DEVI typename In::Ref gate(const ExpertArgs& a, int e, int tile, int lane) {
    return In::ref(a.gate4, a.inner, a.width, e, tile, lane);
  }
  static TAO_DEVI typename In::Ref up(const ExpertArgs& a, int e, int tile, int lane) {
    return In::ref(a.up4, a.inner, a.width, e, tile, lane);
  }
  static TAO_DEVI typename Down::Ref down(const ExpertArgs& a, int e, int tile, int lane) {
    return Down::ref(a.down4, a.width, a.inner, e, tile, lane);
  }
  static TAO_DEVI bool zeros(const ExpertArgs& a) { return a.gate4.zeros != nullptr; }
};

constexpr int kRed = kWarps * 2 * 8 * 16;  // floats of the warps' sums, in every part
// Two blocks an SM: half of its shared memory, less what the driver keeps of it for each.
constexpr int kFixed = kRed * 4 + (int)sizeof(Shared);
constexpr int kRing = (113 * 1024 - kFixed) / kWarps / 16 * 16;
// Every part's ring holds two stages at least, with all of an entry's columns.
static_assert(kRing >= 2 * (2 * W4<32, 128>::BYTES + 8 * 256), "");
static_assert(kRing >= 2 * (2 * W4<32, 64>::BYTES + 16 * 128), "");
static_assert(kRing >= 2 * (2 * W16::BYTES + 16 * 64), "");

template <class L>
__global__ void __launch_bounds__(kThreads, 2) experts_kernel(const ExpertArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  float* red = reinterpret_cast<float*>(smem);
  const uint32_t ring = smem_u32(smem + kRed * 4) + (threadIdx.x >> 5) * kRing;
  Shared& s = *reinterpret_cast<Shared*>(smem + kRed * 4 + kWarps * kRing);
  const int lane = threadIdx.x & 31, g = lane >> 2, warp = threadIdx.x >> 5;
  const bool zeros = L::zeros(a);

  {  // 1. logits
    const int tiles = (a.experts + 15) / 16, cols_max = min(a.tokens, 8);
    run_part<W16, 1, 1, false>(
        tiles * ((a.tokens + 7) / 8), a.width, cols_max, false, ring, kRing, red,
        [&](int u) {
          Unit<W16, 1, 1> r;
          const int m = u / tiles * 8 + g;
          r.w[0] = W16::ref(a.router, a.experts, 0, u % tiles, lane);
          r.x[0] = m < a.tokens ? a.x + m * a.x_stride : nullptr;
          r.cols = min(8, a.tokens - u / tiles * 8);
          return r;
        },
        [&](int u, auto sum) {
          const int cols = min(8, a.tokens - u / tiles * 8);
          for (int i = threadIdx.x; i < cols * 16; i += kThreads) {
            const int e = u % tiles * 16 + i % 16;
            if (e < a.experts) a.logits[(u / tiles * 8 + i / 16) * a.experts + e] = sum(0, i / 16, i % 16);
          }
        });
  }
  if (!grid_meet(a, s)) return;
  for (int t = warp; t < a.tokens; t += kWarps) choose(a, s, t, lane);
  __syncthreads();
  sort_pairs(a, s);

  const int pairs = a.tokens * a.top_k;
  {  // 2. h
    const int tiles = (a.inner + 15) / 16;
    using W = typename L::In;
    run_part<W, 2, 1, false>(
        s.entries * tiles, a.width, min(a.tokens, 8), zeros, ring, kRing, red,
        [&](int u) {
          Unit<W, 2, 1> r;
          const uint32_t en = s.entry[u / tiles];
          const int e = en >> 16, first = en >> 4 & 0xfff;
          r.w[0] = L::gate(a, e, u % tiles, lane);
          r.w[1] = L::up(a, e, u % tiles, lane);
          r.cols = en & 15;
          r.x[0] = g < r.cols ? a.x + s.token[first + g] * a.x_stride : nullptr;
          return r;
        },
        [&](int u, auto sum) {
          const uint32_t en = s.entry[u / tiles];
          const int cols = en & 15, first = en >> 4 & 0xfff;
          for (int i = threadIdx.x; i < cols * 16; i += kThreads) {
            const int c = u % tiles * 16 + i % 16;
            if (c >= a.inner) continue;
            const float gate = sum(0, i / 16, i % 16), up = sum(1, i / 16, i % 16);
            const float h = gate / (1.f + expf(-gate)) * up;
            const long long at = (long long)(first + i / 16) * a.inner + c;
            const bf16 high = tobf(h);
            a.h[at] = high;
            // an infinite h leaves nothing: infinity minus itself would be no number
            a.h[at + (long long)pairs * a.inner] = isinf(bf(high)) ? tobf(0.f) : tobf(h - bf(high));
          }
        });
  }
  if (!grid_meet(a, s)) return;
  {  // 3. the pairs' outputs, and the tokens'
    const int tiles = (a.width + 31) / 32;
    using W = typename L::Down;
    run_part<W, 2, 2, true>(
        s.entries * tiles, a.inner, min(2 * a.tokens, 16), zeros, ring, kRing, red,
        [&](int u) {
          Unit<W, 2, 2> r;
          const uint32_t en = s.entry[u / tiles];
          const int e = en >> 16, first = en >> 4 & 0xfff;
          r.w[0] = L::down(a, e, u % tiles * 2, lane);
          r.w[1] = L::down(a, e, u % tiles * 2 + 1, lane);
          r.cols = 2 * (en & 15);
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int c = n * 8 + g;  // column: token c / 2, its high or its low part
            r.x[n] = c < r.cols ? a.h + ((long long)(c & 1) * pairs + first + c / 2) * a.inner : nullptr;
          }
          return r;
        },
        [&](int u, auto sum) {
          const uint32_t en = s.entry[u / tiles];
          const int cols = en & 15, first = en >> 4 & 0xfff, tile = u % tiles;
          for (int i = threadIdx.x; i < cols * 32; i += kThreads) {
            const int n = tile * 32 + i % 32;
            if (n < a.width) a.pair_out[(long long)(first + i / 32) * a.width + n] = sum(i % 32 / 16, i / 32, i % 16);
          }
          __syncthreads();
          if (threadIdx.x == 0) {
            const int done = atomic_add_release(a.counters + tile, 1) + 1;
            s.last = done == s.entries;
            if (s.last) {
              fence_acquire();
              a.counters[tile] = 0;
            }
          }
          __syncthreads();
          if (!s.last) return;
          for (int i = threadIdx.x; i < a.tokens * 32; i += kThreads) {
            const int t = i / 32, n = tile * 32 + i % 32;
            if (n >= a.width) continue;
            float o = 0.f;
            for (int j = 0; j < a.top_k; ++j) {
              const int p = t * a.top_k + j;
              o += s.weight[p] * __ldcg(a.pair_out + (long long)s.row[p] * a.width + n);
            }
            a.out[(long long)t * a.width + n] = tobf(o);
          }
        });
  }
}

int efail(int code, const char* msg) {
  tao_set_last_error(msg);
  return code;
}

size_t round_up(size_t n) { return (n + 255) / 256 * 256; }

struct Room {
  size_t counters, logits, h, pair_out, total;
};

Room room_of(int tokens, int width, int inner, int experts, int top_k) {
  const size_t t = std::min(tokens, kTokens), pairs = t * top_k;
  Room r;
  r.counters = kHeader;
  r.logits = r.counters + round_up((size_t)(width + 31) / 32 * 4);
  r.h = r.logits + round_up(t * experts * 4);
  r.pair_out = r.h + round_up(2 * pairs * inner * 2);
  r.total = r.pair_out + round_up(pairs * width * 4);
  return r;
}

int check(const TaoExperts* p, int tokens) {
  if (!p) return efail(TAO_ERR_ARG, "null layer");
  if (tokens < 0 || p->width <= 0 || p->inner <= 0) return efail(TAO_ERR_ARG, "tokens, width and inner must be positive");
  if (p->width % 8 || p->inner % 8) return efail(TAO_ERR_ARG, "the expert layer's width and inner are multiples of 8");
  if (p->width > (1 << 20) || p->inner > (1 << 20)) return efail(TAO_ERR_ARG, "width and inner are limited to 2^20");
  if (p->experts <= 0 || p->experts > kExperts) return efail(TAO_ERR_ARG, "an expert layer has 1 to 512 experts");
  if (p->top_k <= 0 || p->top_k > kTop || p->top_k > p->experts)
    return efail(TAO_ERR_ARG, "top_k is 1 to 16 and at most the number of experts");
  if (p->group != 0 && p->group != 32 && p->group != 64 && p->group != 128)
    return efail(TAO_ERR_ARG, "a group is 32, 64 or 128 weights (0: bf16 weights)");
  return TAO_OK;
}

template <class L>
int launch(ExpertArgs a, cudaStream_t s) {
  const int smem = kFixed + kWarps * kRing;
  auto kernel = experts_kernel<L>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  int device = 0, sms = 0, per = 0;
  if (e == cudaSuccess) e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, kThreads, smem);
  if (e == cudaSuccess) {
    void* args[] = {&a};
    e = cudaLaunchCooperativeKernel((const void*)kernel, dim3(sms * per), dim3(kThreads), args, smem, s);
  }
  return e == cudaSuccess ? TAO_OK : efail(TAO_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace
}  // namespace tao

extern "C" {

size_t tao_expert_workspace_bytes(const TaoExperts* layer, int tokens) {
  using namespace tao;
  if (check(layer, tokens) != TAO_OK) return 0;
  return room_of(tokens, layer->width, layer->inner, layer->experts, layer->top_k).total;
}

int tao_expert_layer(const TaoExperts* p, const void* x, long long x_stride, int tokens, void* out, int* ids,
                     float* id_weights, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tao;
  if (int rc = check(p, tokens)) return rc;
  if (tokens == 0) return TAO_OK;
  if (!x || !out || !workspace || !p->router || !p->gate || !p->up || !p->down || (ids && !id_weights))
    return efail(TAO_ERR_ARG, "null pointer");
  if (p->group && (!p->gate_scales || !p->up_scales || !p->down_scales ||
                   !p->gate_zeros != !p->up_zeros || !p->gate_zeros != !p->down_zeros))
    return efail(TAO_ERR_ARG, "4-bit experts have scales, and zero points all or none");
  const void* aligned[] = {x, workspace, p->router, p->gate, p->up, p->down, p->gate_scales, p->up_scales,
                           p->down_scales, p->gate_zeros, p->up_zeros, p->down_zeros};
  for (const void* q : aligned)
    if (reinterpret_cast<uintptr_t>(q) % 16) return efail(TAO_ERR_ARG, "the expert layer's operands start on 16 bytes");
  const long long strides[] = {x_stride, p->gate_expert, p->gate_row, p->up_expert, p->up_row, p->down_expert,
                               p->down_row};
  for (int i = 0; i < (p->group ? 1 : 7); ++i)
    if (strides[i] % 8) return efail(TAO_ERR_ARG, "the expert layer's rows start on 16 bytes");
  if (workspace_bytes < tao_expert_workspace_bytes(p, tokens)) return efail(TAO_ERR_ARG, "workspace too small");
  auto M = [](const void* at, long long e, long long r) { return Matrix16{static_cast<const bf16*>(at), e, r}; };
  auto F = [](const void* c, const void* s, const void* z) {
    return Four{static_cast<const uint8_t*>(c), static_cast<const uint16_t*>(s), static_cast<const uint8_t*>(z)};
  };
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const Room room = room_of(tokens, p->width, p->inner, p->experts, p->top_k);
  for (int at = 0; at < tokens; at += kTokens) {
    ExpertArgs a = {};
    a.x = static_cast<const bf16*>(x) + at * x_stride;
    a.x_stride = x_stride;
    a.router = M(p->router, 0, p->width);
    if (p->group) {
      a.gate4 = F(p->gate, p->gate_scales, p->gate_zeros);
      a.up4 = F(p->up, p->up_scales, p->up_zeros);
      a.down4 = F(p->down, p->down_scales, p->down_zeros);
    } else {
      a.gate16 = M(p->gate, p->gate_expert, p->gate_row);
      a.up16 = M(p->up, p->up_expert, p->up_row);
      a.down16 = M(p->down, p->down_expert, p->down_row);
    }
    a.tokens = std::min(tokens - at, kTokens);
    a.width = p->width;
    a.inner = p->inner;
    a.experts = p->experts;
    a.top_k = p->top_k;
    a.group = p->group;
    a.renormalize = p->renormalize != 0;
    a.out = static_cast<bf16*>(out) + (long long)at * p->width;
    a.ids = ids ? ids + (long long)at * p->top_k : nullptr;
    a.id_weights = ids ? id_weights + (long long)at * p->top_k : nullptr;
    a.error = reinterpret_cast<int*>(ws);
    a.barrier = reinterpret_cast<unsigned*>(ws + 128);
    a.counters = reinterpret_cast<int*>(ws + room.counters);
    a.logits = reinterpret_cast<float*>(ws + room.logits);
    a.h = reinterpret_cast<bf16*>(ws + room.h);
    a.pair_out = reinterpret_cast<float*>(ws + room.pair_out);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int rc = p->group == 0     ? launch<Layer16>(a, s)
                   : p->group == 32  ? launch<Layer4<32>>(a, s)
                   : p->group == 64  ? launch<Layer4<64>>(a, s)
                                     : launch<Layer4<128>>(a, s);
    if (rc) return rc;
  }
  return TAO_OK;
}

int tao_expert_check(void* workspace, size_t workspace_bytes, int* flags, void* stream) {
  using namespace tao;
  if (!workspace) return efail(TAO_ERR_ARG, "null workspace");
  int host = 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemcpyAsync(&host, workspace, sizeof(int), cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  // a wait that ran out leaves the barrier and the counters anywhere: all of it starts again
  if (e == cudaSuccess && host) e = cudaMemsetAsync(workspace, 0, workspace_bytes, s);
  if (e != cudaSuccess) return efail(TAO_ERR_CUDA, cudaGetErrorString(e));
  if (flags) *flags = host;
  return host ? efail(TAO_ERR_DEVICE, "an expert layer's blocks did not meet in time") : TAO_OK;
}

}  // extern "C"
