// A mixture-of-experts layer for a few tokens, in one kernel.
//
//   p = softmax(x R^T), the top_k largest of a row (ties to the lowest expert), their weights
//   p or p / sum of the chosen;  out = sum over them of weight * down_e(silu(gate_e x) * (up_e x))
//
// Bound by the bytes of the chosen experts; with a token or two by what lies between the reads, so the
// code is short (it comes from memory too) and the blocks meet seldom.  One cooperative launch, a block
// an SM, in three parts with a grid barrier between them:
//   1. logits, one expert's to a block;
//   2. every block picks the top_k itself (the same arithmetic in all of them) and sorts the
//      (token, expert) pairs by expert; then 16 inner channels of one expert's gate and up at a
//      time, h = silu(gate) up;
//   3. 32 outputs of one expert's down at a time, a row of sums for each pair; and after a last
//      barrier a token's pairs are added in the order of their choice.
// Parts 2 and 3 are the same product of a few rows (few_rows.cuh).  A block takes a run of neighbouring
// units of work, so that its rows' activations stay in L1; its 16 warps are WT x WK, WT units at a time,
// each one's k dealt to WK warps in runs, each warp's weights through a ring of its own that runs on from
// unit to unit (part 3's starts before the barrier).
// h is kept as the sum of two bf16 (16 mantissa bits), which are two columns of one mma: with bf16
// alone its rounding would add as much to the error as the output's own.  Every sum's order is fixed.
// Of 64 experts (2048, 1024) with 8 for a token: one token 30.3 us (3.3 TB/s), 8 tokens 101 us (5.2), in 4 bits 63.1
// (2.2: the unpacking's instructions); 64 tokens of 128 experts (2048, 768) 230 us (5.2).
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "../../include/tao_b200.h"
#include "few_rows.cuh"

void tao_set_last_error(const char* msg);

namespace tao {
namespace {

constexpr int kWarps = 16, kThreads = kWarps * 32;
constexpr int kBlocks = 148;   // one an SM
constexpr int kTokens = 64;    // of a launch: a bit each of an expert's mask, four a warp
constexpr int kExperts = 512;  // most experts, and
constexpr int kTop = 16;       // most of them for a token
constexpr int kCols = 4;       // tokens of an entry (an expert and some of its tokens) for each column tile
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
  int tokens, width, inner, experts, top_k;
  bool renormalize;
  bf16* out;
  int* ids;          // [tokens][top_k] and their weights, or null
  float* id_weights;
  int *error, *device_error;  // the second may be null
  unsigned* barrier;
  float* logits;     // [tokens][experts]
  bf16* h;           // [2][pairs][inner]: rounded, and what the rounding left
  float* pair_out;   // [pairs][width]
};

// A run of blocks of a row tile of 16-bit weights, 16 rows x 32 k each, straight from the matrix' rows.
struct W16 {
  static constexpr int KB = 32, BYTES = 1024;
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
  static constexpr int KB = 128, BYTES = Block4<GROUP>::BYTES;
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
  uint32_t entry[kExperts + kTokens * kTop / kCols];  // expert << 16 | first row << 5 | tokens
  uint16_t id[kTokens * kTop], row[kTokens * kTop];   // of a token's choices: expert, row of its pair
  float weight[kTokens * kTop];
  uint8_t token[kTokens * kTop];                      // of a pair's row
  uint32_t parts[kWarps];                             // of the sort: a warp's pairs and entries
  int entries;
  bool ok;
};

// All blocks of the launch meet.  The word's top bit flips when the last one arrives (block 0
// adds what the others leave to 2^31), so it needs no reset and any grid may use it next.  `bit` is
// thread 0's, the bit before.
TAO_DEVI bool grid_meet(const ExpertArgs& a, Shared& s, uint32_t& bit) {
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t add = blockIdx.x == 0 ? 0x80000000u - (gridDim.x - 1) : 1u;
    asm volatile("red.release.gpu.global.add.u32 [%0], %1;" ::"l"(a.barrier), "r"(add) : "memory");
    bool ok = false;
    for (int i = 0; i < (1 << 21) && !ok; ++i) {  // a second or two; every block is resident, so none is expected to be late
      uint32_t now;
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(now) : "l"(a.barrier) : "memory");
      ok = ((now ^ bit) & 0x80000000u) != 0;
    }
    bit ^= 0x80000000u;
    if (!ok) {
      atomicOr(a.error, kErrWaitTimeout);
      if (a.device_error) atomicOr(a.device_error, kErrWaitTimeout);
    }
    s.ok = ok;
  }
  __syncthreads();
  return s.ok;
}

// Part 1: a block takes an expert, its warps 128 channels at a time, 16 lanes the even tokens and 16 the
// odd ones, eight of them at once.  `sums`: [token][warp].
TAO_DEVI void logits(const ExpertArgs& a, float* sums) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, k0 = warp * 128 + (lane & 15) * 8;
  for (int e = blockIdx.x; e < a.experts; e += gridDim.x) {
    const bf16* r = a.router.at + e * a.router.row;
#pragma unroll 1
    for (int first = 0; first < a.tokens; first += 8) {  // all lanes' trips: they meet in the sums
      const int t0 = first + (lane >> 4);
      float sum[4] = {};
#pragma unroll 1
      for (int k = k0; k < a.width; k += kWarps * 128) {
        const uint4 r8 = __ldg(reinterpret_cast<const uint4*>(r + k));
        uint4 x8[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)  // a token beyond the last repeats it
          x8[j] = __ldg(reinterpret_cast<const uint4*>(a.x + min(t0 + 2 * j, a.tokens - 1) * a.x_stride + k));
        float w[8], v[8];
        unpack8(r8, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          unpack8(x8[j], v);
#pragma unroll
          for (int i = 0; i < 8; ++i) sum[j] += w[i] * v[i];
        }
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], o);
      if ((lane & 15) == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (t0 + 2 * j < a.tokens) sums[(t0 + 2 * j) * kWarps + warp] = sum[j];
      }
    }
    __syncthreads();
    if (threadIdx.x < a.tokens) {
      float l = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) l += sums[threadIdx.x * kWarps + i];
      a.logits[threadIdx.x * a.experts + e] = l;
    }
    __syncthreads();
  }
}

// A float's order as an unsigned's; 0 and 1 are below every number (taken, and not a number).
TAO_DEVI uint32_t order_of(float v) {
  if (v != v) return 1u;
  const uint32_t u = __float_as_uint(v + 0.f);  // -0 is 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The top_k of TOK tokens (token, token + kWarps, ...) by one warp: ids and weights to shared memory.
// Lane l has the experts l EACH .. l EACH + EACH - 1; the best of all is the lowest lane's with the most.
// A token's choices come one after the other, several tokens' side by side.
template <int EACH, int TOK>
TAO_DEVI void choose(const ExpertArgs& a, Shared& s, int token, int lane) {
  float v[TOK][EACH];
  uint32_t key[TOK][EACH];
  float mine[TOK], top[TOK];
  int my_id[TOK];
#pragma unroll
  for (int q = 0; q < TOK; ++q) {
    const int t = min(token + q * kWarps, a.tokens - 1);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int e = lane * EACH + i;
      v[q][i] = e < a.experts ? __ldcg(a.logits + t * a.experts + e) : -INFINITY;
    }
  }
#pragma unroll
  for (int q = 0; q < TOK; ++q)
#pragma unroll
    for (int i = 0; i < EACH; ++i) key[q][i] = lane * EACH + i < a.experts ? order_of(v[q][i]) : 0u;
#pragma unroll 1
  for (int j = 0; j < a.top_k; ++j) {
#pragma unroll
    for (int q = 0; q < TOK; ++q) {
      uint32_t best = key[q][0];
      int at = 0;
      float bv = v[q][0];
#pragma unroll
      for (int i = 1; i < EACH; ++i) {
        if (key[q][i] > best) {
          best = key[q][i];
          at = i;
          bv = v[q][i];
        }
      }
      const uint32_t most = __reduce_max_sync(0xffffffffu, best);
      const int who = __ffs(__ballot_sync(0xffffffffu, best == most)) - 1;
      const float chosen = __shfl_sync(0xffffffffu, bv, who);
      const int id = __shfl_sync(0xffffffffu, lane * EACH + at, who);
#pragma unroll
      for (int i = 0; i < EACH; ++i)
        if (lane == who && i == at) key[q][i] = 0;
      if (j == 0) top[q] = chosen;
      if (lane == j) {
        mine[q] = chosen;
        my_id[q] = id;
      }
    }
  }
#pragma unroll
  for (int q = 0; q < TOK; ++q) {
    const int t = token + q * kWarps;
    bool nan = false;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      nan |= v[q][i] != v[q][i];
      if (!a.renormalize) sum += lane * EACH + i < a.experts ? expf(v[q][i] - top[q]) : 0.f;
    }
    if (a.renormalize) sum = lane < a.top_k ? expf(mine[q] - top[q]) : 0.f;
    sum = warp_sum(sum);
    nan = __any_sync(0xffffffffu, nan);
    if (lane < a.top_k && t < a.tokens) {
      const float w = nan ? NAN : expf(mine[q] - top[q]) / sum;
      s.id[t * a.top_k + lane] = (uint16_t)my_id[q];
      s.weight[t * a.top_k + lane] = w;
      if (blockIdx.x == 0 && a.ids) {
        a.ids[t * a.top_k + lane] = my_id[q];
        a.id_weights[t * a.top_k + lane] = w;
      }
    }
  }
}

// Up to 32 pairs, by one warp: entries of up to `cols` tokens in the order of the experts' first pairs.
TAO_DEVI void group_few_pairs(const ExpertArgs& a, Shared& s, int cols, int lane) {
  const int pairs = a.tokens * a.top_k;
  const bool in = lane < pairs;
  const int id = in ? s.id[lane] : -1;
  const uint32_t same = __match_any_sync(0xffffffffu, id), below = (1u << lane) - 1;
  const int count = __popc(same), parts = (count + cols - 1) / cols;
  const bool leads = in && (same & below) == 0;
  const uint32_t own = leads ? (uint32_t)count << 16 | parts : 0u;
  uint32_t run = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t before = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += before;
  }
  const int first = (int)((run - own) >> 16), at = (int)((run - own) & 0xffff);
  if (leads)
    for (int i = 0; i < parts; ++i)
      s.entry[at + i] = (uint32_t)id << 16 | (uint32_t)(first + i * cols) << 5 | min(cols, count - i * cols);
  const int row = __shfl_sync(0xffffffffu, first, __ffs(same) - 1) + __popc(same & below);
  if (in) {
    s.row[lane] = (uint16_t)row;
    s.token[row] = (uint8_t)(lane / a.top_k);
  }
  if (lane == 31) s.entries = (int)(run & 0xffff);
}

// Pairs sorted by expert, then token; entries of up to `cols` tokens.  Thread e has expert e.
TAO_DEVI void sort_pairs(const ExpertArgs& a, Shared& s, int cols) {
  static_assert(kThreads >= kExperts, "");
  const int pairs = a.tokens * a.top_k, e = threadIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  s.mask[e] = 0;
  __syncthreads();
  for (int p = threadIdx.x; p < pairs; p += kThreads) atomicOr(&s.mask[s.id[p]], 1ull << (p / a.top_k));
  __syncthreads();
  const int count = __popcll(s.mask[e]), parts = (count + cols - 1) / cols;
  uint32_t run = (uint32_t)count << 16 | parts;  // sums over the experts up to this one
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t before = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += before;
  }
  if (lane == 31) s.parts[warp] = run;
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) run += s.parts[w];
  }
  const int first = (int)(run >> 16) - count, at = (int)(run & 0xffff) - parts;
  s.base[e] = first;
  for (int i = 0; i < parts; ++i)
    s.entry[at + i] = (uint32_t)e << 16 | (uint32_t)(first + i * cols) << 5 | min(cols, count - i * cols);
  if (e == kThreads - 1) s.entries = (int)(run & 0xffff);
  __syncthreads();
  for (int p = threadIdx.x; p < pairs; p += kThreads) {
    const int t = p / a.top_k, x = s.id[p], row = s.base[x] + __popcll(s.mask[x] & ((1ull << t) - 1));
    s.row[p] = (uint16_t)row;
    s.token[row] = (uint8_t)t;
  }
  __syncthreads();
}

// The experts' matrices in the layer's format.
struct Layer16 {
  using W = W16;
  static TAO_DEVI const Matrix16& of(const ExpertArgs& a, int part, int r) {
    return part ? a.down16 : r ? a.up16 : a.gate16;
  }
};
template <int GROUP>
struct Layer4 {
  using W = W4<GROUP>;
  static TAO_DEVI const Four& of(const ExpertArgs& a, int part, int r) { return part ? a.down4 : r ? a.up4 : a.gate4; }
};

template <int NT>
constexpr int kDepth = NT == 4 ? 3 : 4;  // stages of a warp's ring, as shared memory allows
template <int NT>
constexpr int kSlot = 2 * kCols * NT * 16;  // floats of a warp's sums of a unit: [matrix][token][16 rows]

// log2 of a unit's warps: the fewest blocks on the longest warp's way, then the fewest warps.
TAO_DEVI int pick_wk(int units_of_block, int kblocks) {
  int best = 0, least = 1 << 30;
#pragma unroll
  for (int shift = 0; 1 << shift <= kWarps; ++shift) {
    const int groups = kWarps >> shift;
    const int cost = (units_of_block + groups - 1) / groups * ((kblocks + (1 << shift) - 1) >> shift);
    if (cost < least && 1 << shift <= kblocks) {
      least = cost;
      best = shift;
    }
  }
  return best;
}

// Parts 2 (`part` 0) and 3 (1).  A unit is an entry's 16 inner channels or 32 outputs, two row tiles in
// both; a column of the mma a token's x or (in turn) the two parts of its h.
template <class L, int NT>
TAO_DEVI bool run_part(const ExpertArgs& a, Shared& s, uint8_t* rings, float* sums, int part, uint32_t& bit) {
  using W = typename L::W;
  constexpr int STAGE = 2 * W::BYTES, SLOT = kSlot<NT>, DEPTH = kDepth<NT>;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int k = part ? a.inner : a.width, rows = part ? a.width : a.inner, pairs = a.tokens * a.top_k;
  const int tiles = part ? (a.width + 31) / 32 : (a.inner + 15) / 16;
  const int kblocks = (k + W::KB - 1) / W::KB, units = s.entries * tiles;
  // a run of neighbouring units for each block
  const int each = units / gridDim.x, more = units - each * gridDim.x, b = blockIdx.x;
  const int lo = each * b + min(b, more), hi = lo + each + (b < more);
  const int wks = pick_wk(each + (more > 0), kblocks), groups = kWarps >> wks;
  const int wt = warp >> wks, wk = warp & ((1 << wks) - 1);
  const int kw = kblocks * wk >> wks, per = (kblocks * (wk + 1) >> wks) - kw;
  const int mine = lo + wt < hi ? (hi - lo - wt + groups - 1) >> (4 - wks) : 0;
  uint8_t* const ring = rings + warp * (DEPTH * STAGE);
  const uint32_t ring_at = smem_u32(ring);
  const bool zeros = a.gate4.zeros != nullptr;

  int entry = (lo + wt) / tiles, tile = lo + wt - entry * tiles;
  int le = entry, lt = tile, lk = 0, left = mine * per, to_slot = 0;  // what is copied next
  W w[2];
  auto issue = [&]() {
    if (left > 0) {
      --left;
      if (lk == 0) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
          w[r].start(L::of(a, part, r), rows, k, s.entry[le] >> 16, part ? lt * 2 + r : lt, kw, lane);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) w[r].issue(ring_at + to_slot + r * W::BYTES, lane);
      to_slot = to_slot == (DEPTH - 1) * STAGE ? 0 : to_slot + STAGE;
      if (++lk == per) {
        lk = 0;
        for (lt += groups; lt >= tiles; lt -= tiles) ++le;
      }
    }
    cp_commit();
  };
#pragma unroll 1
  for (int d = 0; d < DEPTH - 1; ++d) issue();
  if (part && !grid_meet(a, s, bit)) {
    cp_wait<0>();
    return false;
  }

  int slot = 0, parity = 0;
#pragma unroll 1
  for (int u = 0; u < mine; ++u) {
    const uint32_t en = s.entry[entry];
    const int first = en >> 5 & 0x7ff, tokens = en & 31, cols = tokens << part;
    const bf16* x[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int c = n * 8 + g;
      x[n] = c >= cols ? nullptr
             : part    ? a.h + ((long long)(c & 1) * pairs + first + c / 2) * a.inner + t * 8
                       : a.x + s.token[first + c] * a.x_stride + t * 8;
    }
    float acc[2][NT][4] = {};
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
      cp_wait<DEPTH - 2>();
      __syncwarp();  // the stage is there for every lane, and every lane is done with the one before
      issue();
#pragma unroll
      for (int r = 0; r < 2; ++r)
        W::template product<NT>(acc[r], ring + slot + r * W::BYTES, zeros, lane, cols,
                                [&](int p, int n) { return v[p][n]; });
      slot = slot == (DEPTH - 1) * STAGE ? 0 : slot + STAGE;
    }
    float* to = sums + (parity * kWarps + warp) * SLOT + g;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float* c = to + r * (SLOT / 2) + n * 8 * 16;
        if (part) {  // a token's two columns
          c = to + r * (SLOT / 2) + (n * 4 + t) * 16;
          c[0] = acc[r][n][0] + acc[r][n][1];
          c[8] = acc[r][n][2] + acc[r][n][3];
        } else if (n * 8 + 2 * t < kCols * NT) {  // two tokens
          c += 2 * t * 16;
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
    const float* from = sums + (parity * kWarps + (wt << wks)) * SLOT;
    for (int i = wk * 32 + lane; i < tokens * 16; i += 32 << wks) {
      float s0 = 0.f, s1 = 0.f;
#pragma unroll 4
      for (int q = 0; q < 1 << wks; ++q) {
        s0 += from[q * SLOT + i];
        s1 += from[q * SLOT + SLOT / 2 + i];
      }
      const long long pair = first + i / 16;
      if (part) {
        const int n = tile * 32 + i % 16;
        float* out = a.pair_out + pair * a.width + n;
        if (n < a.width) out[0] = s0;
        if (n + 16 < a.width) out[16] = s1;
      } else {
        const int c = tile * 16 + i % 16;
        if (c < a.inner) {
          const float h = s0 / (1.f + expf(-s0)) * s1;
          const bf16 high = tobf(h);
          a.h[pair * a.inner + c] = high;
          // an infinite h leaves nothing: infinity minus itself would be no number
          a.h[(pair + pairs) * a.inner + c] = isinf(bf(high)) ? tobf(0.f) : tobf(h - bf(high));
        }
      }
    }
    parity ^= 1;
    for (tile += groups; tile >= tiles; tile -= tiles) ++entry;
  }
  cp_wait<0>();
  __syncthreads();
  return true;
}

template <class W, int NT>
constexpr int kRings = kWarps * kDepth<NT> * 2 * W::BYTES;
template <class W, int NT>  // the sums of the unit at hand and of the one before
constexpr int kSmem = kRings<W, NT> + 2 * kWarps * kSlot<NT> * 4 + (int)sizeof(Shared);
static_assert(kSmem<W16, 4> <= 227 * 1024 && kSmem<W4<32>, 4> <= 227 * 1024, "");
static_assert(kSlot<1> * 2 * kWarps >= kTokens * kWarps, "part 1's sums fit too");

// NT: column tiles of an entry in part 3.
template <class L, int NT>
__global__ void __launch_bounds__(kThreads, 1) experts_kernel(const __grid_constant__ ExpertArgs a) {
  using W = typename L::W;
  extern __shared__ __align__(16) uint8_t smem[];
  float* sums = reinterpret_cast<float*>(smem + kRings<W, NT>);
  Shared& s = *reinterpret_cast<Shared*>(smem + kRings<W, NT> + 2 * kWarps * kSlot<NT> * 4);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t bit = threadIdx.x == 0 ? *reinterpret_cast<volatile unsigned*>(a.barrier) : 0;

  logits(a, sums);
  if (!grid_meet(a, s, bit)) return;
  if (a.experts <= 128) {
    if (a.tokens <= kWarps) {
      if (warp < a.tokens) choose<4, 1>(a, s, warp, lane);
    } else {
      choose<4, 4>(a, s, warp, lane);
    }
  } else {
    for (int t = warp; t < a.tokens; t += kWarps) choose<16, 1>(a, s, t, lane);
  }
  __syncthreads();
  if (a.tokens * a.top_k <= 32) {
    if (warp == 0) group_few_pairs(a, s, kCols * NT, lane);
    __syncthreads();
  } else {
    sort_pairs(a, s, kCols * NT);
  }
#pragma unroll 1
  for (int part = 0; part < 2; ++part)
    if (!run_part<L, NT>(a, s, smem, sums, part, bit)) return;
  if (!grid_meet(a, s, bit)) return;
  const int quads = a.width / 4;
  for (int i = blockIdx.x * kThreads + threadIdx.x; i < a.tokens * quads; i += gridDim.x * kThreads) {
    const int t = i / quads, n = (i - t * quads) * 4;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
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

template <class L, int NT>
int launch_as(ExpertArgs a, cudaStream_t s) {
  const int smem = kSmem<typename L::W, NT>;
  auto kernel = experts_kernel<L, NT>;
  static std::atomic<uint64_t> ready{0};  // devices (the first 64) on which the kernel may use its shared memory
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  const uint64_t mark = device < 64 ? 1ull << device : 0;
  if (e == cudaSuccess && !(ready.load(std::memory_order_relaxed) & mark)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) ready |= mark;
  }
  if (e == cudaSuccess) {
    void* args[] = {&a};
    e = cudaLaunchCooperativeKernel((const void*)kernel, dim3(kBlocks), dim3(kThreads), args, smem, s);
  }
  return e == cudaSuccess ? TAO_OK : efail(TAO_ERR_CUDA, cudaGetErrorString(e));
}

// An entry's weights come once for its 4, 8 or 16 tokens, and from L2 for each further entry of the
// expert; columns that few entries fill cost instructions.  So by the mean tokens of an expert; us, of 64 experts
// (2048, 1024) with 8 for a token and of 8 (4096, 2048) with 2:
//   mean 2 (16 of 64):          bf16 137.9, 138.4, 140.7    4 bits 83.5, 87.4, 149.2
//   mean 4 (32 of 64):          bf16 189.5, 172.3, 173.9    4 bits 125.8, 113.3, 171.1
//   mean 8 (64 of 64, 32 of 8): bf16 197.1, 217.0, 190.7 and 121.5, 111.0, 107.9    4 bits 175.3, 154.0, 191.8
//   mean 16 (64 of 8):          bf16 218.9, 175.1, 141.6    4 bits 162.7, 146.3, 158.5
// Four tiles leave 4-bit weights, which need registers to be unpacked, too few.
template <class L>
int launch(const ExpertArgs& a, cudaStream_t s) {
  const int pairs = a.tokens * a.top_k;
  if (pairs <= 2 * a.experts) return launch_as<L, 1>(a, s);
  if constexpr (std::is_same<L, Layer16>::value) {
    if (pairs > 4 * a.experts) return launch_as<L, 4>(a, s);
  }
  return launch_as<L, 2>(a, s);
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
  // (8 bytes are stored at a time; a row is whole 16 bytes)
  if (reinterpret_cast<uintptr_t>(out) % 8) return efail(TAO_ERR_ARG, "the expert layer's output starts on 8 bytes");
  if (!on_elements({{ids, sizeof(int)}, {id_weights, sizeof(float)}, {p->error, sizeof(int)}}))
    return efail(TAO_ERR_ARG, "operands start on a whole element");
  const long long strides[] = {x_stride, p->gate_expert, p->gate_row, p->up_expert, p->up_row, p->down_expert,
                               p->down_row};
  for (int i = 0; i < (p->group ? 1 : 7); ++i)
    if (strides[i] % 8) return efail(TAO_ERR_ARG, "the expert layer's rows start on 16 bytes");
  // a launch writes after its last read of x; a later one's rows it may not write, unless it has read them itself
  const long long row = p->width * 2LL;
  if (tokens > kTokens && !(out == x && x_stride == p->width) &&
      rows_overlap(x, tokens, x_stride * 2, row, out, tokens * row))
    return efail(TAO_ERR_ARG, "the expert layer's output must not overlap a later launch's tokens");
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
    a.renormalize = p->renormalize != 0;
    a.out = static_cast<bf16*>(out) + (long long)at * p->width;
    a.ids = ids ? ids + (long long)at * p->top_k : nullptr;
    a.id_weights = ids ? id_weights + (long long)at * p->top_k : nullptr;
    a.error = reinterpret_cast<int*>(ws);
    a.device_error = p->error;
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
  // a wait that ran out leaves the barrier anywhere: all of it starts again, before a launch on any stream
  if (e == cudaSuccess && host) {
    e = cudaMemsetAsync(workspace, 0, workspace_bytes, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  }
  if (e != cudaSuccess) return efail(TAO_ERR_CUDA, cudaGetErrorString(e));
  if (flags) *flags = host;
  return host ? efail(TAO_ERR_DEVICE, "an expert layer's blocks did not meet in time") : TAO_OK;
}

}  // extern "C"
