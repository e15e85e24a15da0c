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
//   3. 32 outputs of one expert's down at a time, a row of sums for each pair; and after a last
//      barrier a token's pairs are added in the order of their choice.
// Parts 1 to 3 are the same product of a few rows (few_rows.cuh).  One block an SM takes a run of
// neighbouring units of work, so that its rows' activations stay in L1; its 16 warps are WT x WK, WT
// units at a time, each one's k dealt to WK warps in runs, each warp's weights through a ring of its own
// that runs on from unit to unit (part 3's starts before the barrier).
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

constexpr int kWarps = 16, kThreads = kWarps * 32;
constexpr int kTokens = 64;    // of a launch: a bit each of an expert's mask
constexpr int kExperts = 512;  // most experts, and
constexpr int kTop = 16;       // most of them for a token
constexpr int kCols = 8;       // tokens of an entry: (expert, up to 8 of its tokens)
constexpr int kHeader = 256;   // workspace: error word and barrier word

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
  float* logits;     // [tokens][experts]
  bf16* h;           // [2][pairs][inner]: rounded, and what the rounding left
  float* pair_out;   // [pairs][width]
};

// A run of blocks of a row tile of 16-bit weights, 16 rows x 32 k each, straight from the matrix' rows.
struct W16 {
  static constexpr int KB = 32, BYTES = 1024, DEPTH = 4;
  using Matrix = Matrix16;
  const bf16 *r0, *r1, *any;
  int left;  // of k from this lane's next chunk on

  // From block `kb` on; rows beyond the matrix repeat its last one.
  TAO_DEVI void start(const Matrix& m, int rows, int k, int e, int tile, int kb, int lane) {
    const int r = tile * 16 + (lane >> 2), at = kb * KB + (lane & 3) * 8;
    any = m.at + e * m.expert;
    r0 = any + min(r, rows - 1) * m.row + at;
    r1 = any + min(r + 8, rows - 1) * m.row + at;
    left = k - at;
  }
  TAO_DEVI void issue(uint32_t to, int lane) {
    cp_async16(to + lane * 16, left > 0 ? r0 : any, left > 0);
    cp_async16(to + 512 + lane * 16, left > 0 ? r1 : any, left > 0);
    r0 += KB;
    r1 += KB;
    left -= KB;
  }
  template <int NT, class B>
  static TAO_DEVI void product(float (&acc)[NT][4], const uint8_t* from, bool, int lane, int cols, B b) {
    const uint4 w0 = *reinterpret_cast<const uint4*>(from + lane * 16);
    const uint4 w1 = *reinterpret_cast<const uint4*>(from + 512 + lane * 16);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (n && n * 8 >= cols) break;
      const uint4 x = b(0, n);
      mma_bf16(acc[n], w0.x, w1.x, w0.y, w1.y, x.x, x.y);
      mma_bf16(acc[n], w0.z, w1.z, w0.w, w1.w, x.z, x.w);
    }
  }
};

// The same of 4-bit weights, 16 rows x 128 k each.
template <int GROUP>
struct W4 {
  static constexpr int KB = 128, BYTES = Block4<GROUP>::BYTES, DEPTH = 4;
  using Matrix = Four;
  const Four* m;
  uint32_t block;

  TAO_DEVI void start(const Matrix& matrix, int rows, int k, int e, int tile, int kb, int) {
    const uint32_t tiles = (rows + 15) / 16, blocks = (k + 127) / 128;
    m = &matrix;
    block = (e * tiles + min((uint32_t)tile, tiles - 1)) * blocks + kb;
  }
  TAO_DEVI void issue(uint32_t to, int lane) { Block4<GROUP>::issue(to, *m, block++, lane); }
  template <int NT, class B>
  static TAO_DEVI void product(float (&acc)[NT][4], const uint8_t* from, bool zeros, int lane, int cols, B b) {
    Block4<GROUP> block;
    block.load(from, zeros, lane);
    block.template product16<MmaBf16, true, NT>(acc, cols, b);
  }
};

struct Shared {
  unsigned long long mask[kExperts];
  int base[kExperts];
  uint32_t entry[kExperts + kTokens * kTop / kCols];  // expert << 16 | first row << 4 | tokens
  uint16_t id[kTokens * kTop], row[kTokens * kTop];   // of a token's choices: expert, row of its pair
  float weight[kTokens * kTop];
  uint8_t token[kTokens * kTop];                      // of a pair's row
  int entries;
  bool ok;
};

constexpr int kSlot = 2 * 8 * 16;             // floats of a warp's sums of a unit
constexpr int kSums = 2 * kWarps * kSlot;     // of the unit at hand and the one before

// Warps of a unit: the fewest blocks on the longest warp's way, then the fewest warps.
TAO_DEVI int pick_wk(int units, int kblocks) {
  const int n = (units + gridDim.x - 1) / gridDim.x;
  int best = 0, least = 1 << 30;
#pragma unroll
  for (int shift = 0; 1 << shift <= kWarps; ++shift) {
    const int groups = kWarps >> shift, cost = (n + groups - 1) / groups * ((kblocks + (1 << shift) - 1) >> shift);
    if (cost < least && 1 << shift <= kblocks) {
      least = cost;
      best = shift;
    }
  }
  return best;
}

// A part's units, a run of neighbours for each block: unit u is row tiles R (u % tiles) ... of entry
// u / tiles.  `weights(w, r, entry, tile, kb)` starts run w at block kb of unit (entry, tile)'s matrix r;
// `rows(entry, c)` gives the row of column c or null; `cols(entry)` their number; `meet()` is called when
// the first weights are on their way and before the first row is read; `sink(entry, tile, column, row,
// sum)` takes sum(r) of each column and row, where the columns of a PAIR are added in twos.
template <class W, int R, int NT, bool PAIR, class Weights, class Rows, class Cols, class Meet, class Sink>
TAO_DEVI bool run_part(int entries, int tiles, int k, bool zeros, uint8_t* rings, float* sums, Weights weights,
                       Rows rows, Cols cols, Meet meet, Sink sink) {
  constexpr int STAGE = R * W::BYTES;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kblocks = (k + W::KB - 1) / W::KB, units = entries * tiles;
  const int wks = pick_wk(units, kblocks), groups = kWarps >> wks;
  const int wt = warp >> wks, wk = warp & ((1 << wks) - 1);
  const int kw = kblocks * wk >> wks, per = (kblocks * (wk + 1) >> wks) - kw;
  const int lo = (int)((long long)units * blockIdx.x / gridDim.x);
  const int hi = (int)((long long)units * (blockIdx.x + 1) / gridDim.x);
  const int mine = lo + wt < hi ? (hi - lo - wt + groups - 1) / groups : 0;
  uint8_t* const ring = rings + warp * (W::DEPTH * STAGE);
  const uint32_t ring_at = smem_u32(ring);

  int entry = (lo + wt) / tiles, tile = lo + wt - entry * tiles;
  int le = entry, lt = tile, lk = 0, left = mine * per, to_slot = 0;  // what is copied next
  W w[R];
  auto issue = [&]() {
    if (left > 0) {
      --left;
      if (lk == 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) weights(w[r], r, le, lt, kw);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) w[r].issue(ring_at + to_slot + r * W::BYTES, lane);
      to_slot = to_slot == (W::DEPTH - 1) * STAGE ? 0 : to_slot + STAGE;
      if (++lk == per) {
        lk = 0;
        for (lt += groups; lt >= tiles; lt -= tiles) ++le;
      }
    }
    cp_commit();
  };
#pragma unroll 1
  for (int d = 0; d < W::DEPTH - 1; ++d) issue();
  if (!meet()) {
    cp_wait<0>();
    return false;
  }

  int slot = 0, parity = 0;
#pragma unroll 1
  for (int u = 0; u < mine; ++u) {
    const int n_cols = cols(entry);
    const bf16* x[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) x[n] = n * 8 + g < n_cols ? rows(entry, n * 8 + g) + t * 8 : nullptr;
    float acc[R][NT][4] = {};
#pragma unroll 1
    for (int i = 0; i < per; ++i) {
      const int k0 = (kw + i) * W::KB;
      uint4 v[W::KB / 32][NT];
#pragma unroll
      for (int p = 0; p < W::KB / 32; ++p)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          v[p][n] = make_uint4(0, 0, 0, 0);
          if (x[n] && k0 + p * 32 + t * 8 < k) v[p][n] = *reinterpret_cast<const uint4*>(x[n] + k0 + p * 32);
        }
      cp_wait<W::DEPTH - 2>();
      __syncwarp();  // the stage is there for every lane, and every lane is done with the one before
      issue();
#pragma unroll
      for (int r = 0; r < R; ++r)
        W::template product<NT>(acc[r], ring + slot + r * W::BYTES, zeros, lane, n_cols,
                                [&](int p, int n) { return v[p][n]; });
      slot = slot == (W::DEPTH - 1) * STAGE ? 0 : slot + STAGE;
    }
    float* to = sums + (parity * kWarps + warp) * kSlot;  // [R][column][16 rows]
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if constexpr (PAIR) {
          float* c = to + (r * 8 + n * 4 + t) * 16 + g;
          c[0] = acc[r][n][0] + acc[r][n][1];
          c[8] = acc[r][n][2] + acc[r][n][3];
        } else {
          float* c = to + (r * 8 + n * 8 + 2 * t) * 16 + g;
          c[0] = acc[r][n][0];
          c[16] = acc[r][n][1];
          c[8] = acc[r][n][2];
          c[24] = acc[r][n][3];
        }
      }
    // the unit's warps meet; the sums before the last ones are free again
    if (wks == 0)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(1 + wt), "r"(32 << wks) : "memory");
    const float* from = sums + (parity * kWarps + (wt << wks)) * kSlot;
    const int outs = (PAIR ? n_cols / 2 : n_cols) * 16;
    for (int i = wk * 32 + lane; i < outs; i += 32 << wks)
      sink(entry, tile, i / 16, i % 16, [&](int r) {
        float s = 0.f;
        for (int q = 0; q < 1 << wks; ++q) s += from[q * kSlot + r * 128 + i];
        return s;
      });
    parity ^= 1;
    for (tile += groups; tile >= tiles; tile -= tiles) ++entry;
  }
  cp_wait<0>();
  __syncthreads();
  return true;
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

// The experts' matrices in the layer's format.
struct Layer16 {
  using W = W16;
  static TAO_DEVI const Matrix16& gate(const ExpertArgs& a) { return a.gate16; }
  static TAO_DEVI const Matrix16& up(const ExpertArgs& a) { return a.up16; }
  static TAO_DEVI const Matrix16& down(const ExpertArgs& a) { return a.down16; }
};
template <int GROUP>
struct Layer4 {
  using W = W4<GROUP>;
  static TAO_DEVI const Four& gate(const ExpertArgs& a) { return a.gate4; }
  static TAO_DEVI const Four& up(const ExpertArgs& a) { return a.up4; }
  static TAO_DEVI const Four& down(const ExpertArgs& a) { return a.down4; }
};

template <class W>
constexpr int kRings = kWarps * (W::DEPTH * 2 * W::BYTES > W16::DEPTH * W16::BYTES ? W::DEPTH * 2 * W::BYTES
                                                                                  : W16::DEPTH * W16::BYTES);
template <class W>
constexpr int kSmem = kRings<W> + kSums * 4 + (int)sizeof(Shared);
static_assert(kSmem<W16> <= 227 * 1024 && kSmem<W4<32>> <= 227 * 1024, "");

template <class L>
__global__ void __launch_bounds__(kThreads, 1) experts_kernel(const __grid_constant__ ExpertArgs a) {
  using W = typename L::W;
  extern __shared__ __align__(16) uint8_t smem[];
  float* sums = reinterpret_cast<float*>(smem + kRings<W>);
  Shared& s = *reinterpret_cast<Shared*>(smem + kRings<W> + kSums * 4);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const auto now = [] { return true; };

  // 1. logits: an entry is 8 tokens
  run_part<W16, 1, 1, false>(
      (a.tokens + 7) / 8, (a.experts + 15) / 16, a.width, false, smem, sums,
      [&](W16& w, int, int, int tile, int kb) { w.start(a.router, a.experts, a.width, 0, tile, kb, lane); },
      [&](int entry, int c) { return a.x + (entry * 8 + c) * a.x_stride; },
      [&](int entry) { return min(8, a.tokens - entry * 8); }, now,
      [&](int entry, int tile, int col, int row, auto sum) {
        const int e = tile * 16 + row;
        if (e < a.experts) a.logits[(entry * 8 + col) * a.experts + e] = sum(0);
      });
  if (!grid_meet(a, s)) return;
  for (int t = warp; t < a.tokens; t += kWarps) choose(a, s, t, lane);
  __syncthreads();
  sort_pairs(a, s);

  const int pairs = a.tokens * a.top_k;
  const bool zeros = a.gate4.zeros != nullptr;
  const auto expert = [&](int entry) { return (int)(s.entry[entry] >> 16); };
  const auto first = [&](int entry) { return (int)(s.entry[entry] >> 4 & 0xfff); };
  const auto count = [&](int entry) { return (int)(s.entry[entry] & 15); };
  // 2. h
  run_part<W, 2, 1, false>(
      s.entries, (a.inner + 15) / 16, a.width, zeros, smem, sums,
      [&](W& w, int r, int entry, int tile, int kb) {
        w.start(r ? L::up(a) : L::gate(a), a.inner, a.width, expert(entry), tile, kb, lane);
      },
      [&](int entry, int c) { return a.x + s.token[first(entry) + c] * a.x_stride; }, count, now,
      [&](int entry, int tile, int col, int row, auto sum) {
        const int c = tile * 16 + row;
        if (c >= a.inner) return;
        const float gate = sum(0), up = sum(1);
        const float h = gate / (1.f + expf(-gate)) * up;
        const long long at = (long long)(first(entry) + col) * a.inner + c;
        const bf16 high = tobf(h);
        a.h[at] = high;
        // an infinite h leaves nothing: infinity minus itself would be no number
        a.h[at + (long long)pairs * a.inner] = isinf(bf(high)) ? tobf(0.f) : tobf(h - bf(high));
      });
  // 3. the pairs' outputs: two columns a token, its h's high and low parts; and the tokens'
  const bool met = run_part<W, 2, 2, true>(
      s.entries, (a.width + 31) / 32, a.inner, zeros, smem, sums,
      [&](W& w, int r, int entry, int tile, int kb) {
        w.start(L::down(a), a.width, a.inner, expert(entry), tile * 2 + r, kb, lane);
      },
      [&](int entry, int c) { return a.h + ((long long)(c & 1) * pairs + first(entry) + c / 2) * a.inner; },
      [&](int entry) { return 2 * count(entry); }, [&] { return grid_meet(a, s); },
      [&](int entry, int tile, int col, int row, auto sum) {
        float* to = a.pair_out + (long long)(first(entry) + col) * a.width;
        const int n = tile * 32 + row;
        if (n < a.width) to[n] = sum(0);
        if (n + 16 < a.width) to[n + 16] = sum(1);
      });
  if (!met || !grid_meet(a, s)) return;
  const int quads = a.width / 4;
  for (int i = blockIdx.x * kThreads + threadIdx.x; i < a.tokens * quads; i += gridDim.x * kThreads) {
    const int t = i / quads, n = i % quads * 4;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = 0; j < a.top_k; ++j) {
      const int p = t * a.top_k + j;
      const float w = s.weight[p];
      const float4 v = __ldcg(reinterpret_cast<const float4*>(a.pair_out + (long long)s.row[p] * a.width + n));
      o.x += w * v.x, o.y += w * v.y, o.z += w * v.z, o.w += w * v.w;
    }
    *reinterpret_cast<uint2*>(a.out + (long long)t * a.width + n) = make_uint2(bf16x2(o.x, o.y), bf16x2(o.z, o.w));
  }
}

int efail(int code, const char* msg) {
  tao_set_last_error(msg);
  return code;
}

size_t round_up(size_t n) { return (n + 255) / 256 * 256; }

struct Room {
  size_t logits, h, pair_out, total;
};

Room room_of(int tokens, int width, int inner, int experts, int top_k) {
  const size_t t = std::min(tokens, kTokens), pairs = t * top_k;
  Room r;
  r.logits = kHeader;
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
  const int smem = kSmem<typename L::W>;
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
    return Four{static_cast<const uint8_t*>(c), static_cast<const uint8_t*>(s), static_cast<const uint8_t*>(z)};
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
  // a wait that ran out leaves the barrier anywhere: all of it starts again
  if (e == cudaSuccess && host) e = cudaMemsetAsync(workspace, 0, workspace_bytes, s);
  if (e != cudaSuccess) return efail(TAO_ERR_CUDA, cudaGetErrorString(e));
  if (flags) *flags = host;
  return host ? efail(TAO_ERR_DEVICE, "an expert layer's blocks did not meet in time") : TAO_OK;
}

}  // extern "C"
