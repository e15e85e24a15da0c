// Rows of a table by tokens' ids, scaled, and the table's gradient.
//
// Forward: bound by its bytes (and for a few tokens by the launch); a thread has 16 bytes of a row.
// Gradient: the tokens are sorted by id (sort.cuh, stably), and a block adds the rows of a run of kRun sorted
// tokens, in fp32 and in their order, a sum for each id.  An id whose tokens lie within the run is written at
// once; the sums of one that goes on in the next run are joined by a second kernel, in a fixed order of the runs, so a
// word that comes 10000 times is added by 625 blocks and the result does not depend on when they ran.  Rows of no
// token are zeros, written by blocks beside the sort's (bound by latency), before the sums.  32768 tokens, 65536 x 768 in
// bf16: sort and zeros 37 us (one after the other 28 and 18), the runs 19 (with runs of 32 and of 64, eight rows on
// their way, 35 and 47), the joins 5; the forward pass 18 after a flush, 13 in turn (5.2 TB/s).
#include <cuda_runtime.h>

#include "rows.cuh"
#include "sort.cuh"

void tao_set_last_error(const char* msg);

namespace tao {
namespace {

using namespace rows;

constexpr int kRun = 16;

int efail(int code, const char* msg) {
  tao_set_last_error(msg);
  return code;
}
int launched(cudaError_t e) { return e == cudaSuccess ? TAO_OK : efail(TAO_ERR_CUDA, cudaGetErrorString(e)); }

struct EmbedArgs {
  const void* ids;
  long long n, vocab, stride;
  int width;
  bool wide_ids;
  float scale;
  const void* in;
  void* out;
};

// EACH: tokens of a thread, whose rows are on their way at once.
template <class T, int N, bool WIDE, int EACH>
__global__ void __launch_bounds__(256) embed_kernel(const EmbedArgs a) {
  const int c = first_of<N, WIDE>(blockIdx.y, blockDim.x, threadIdx.x), step = blockDim.x;
  if (c >= a.width) return;
  const long long t0 = (long long)blockIdx.x * (blockDim.y * EACH) + threadIdx.y;
  long long id[EACH];
  Part<T, N, WIDE> v[EACH];
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const long long t = min(t0 + j * (int)blockDim.y, a.n - 1);
    id[j] = a.wide_ids ? static_cast<const long long*>(a.ids)[t] : static_cast<const int*>(a.ids)[t];
  }
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    if (id[j] < 0 || id[j] >= a.vocab) id[j] = -1;
    v[j].load(static_cast<const T*>(a.in) + max(id[j], 0ll) * a.stride, c, step, a.width);
  }
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const long long t = t0 + j * (int)blockDim.y;
    float f[N];
    v[j].widen(f);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = id[j] < 0 ? 0.f : f[i] * a.scale;
    if (t < a.n) Part<T, N, WIDE>::of(f).store(static_cast<T*>(a.out) + t * a.width, c, step, a.width);
  }
}

struct SumArgs {
  const int *tokens, *ids;  // sorted by id
  int n, vocab, width;
  float scale;
  const void* dy;
  long long dy_stride;
  void* out;
  float* parts;  // [runs][2][width]: of an id that began before the run, and of one that goes on behind it
};

// A thread's sums in fp32, in the workspace.
template <int N, bool WIDE>
TAO_DEVI void put_sums(float* row, int first, int step, int width, const float (&v)[N]) {
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    if constexpr (WIDE) {
      *reinterpret_cast<float4*>(row + first + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    } else {
#pragma unroll
      for (int i = e; i < e + 4; ++i)
        if (first + i * step < width) row[first + i * step] = v[i];
    }
  }
}
template <int N, bool WIDE>
TAO_DEVI void add_sums(const float* row, int first, int step, int width, float (&v)[N]) {
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    if constexpr (WIDE) {
      const float4 w = *reinterpret_cast<const float4*>(row + first + e);
      v[e] += w.x, v[e + 1] += w.y, v[e + 2] += w.z, v[e + 3] += w.w;
    } else {
#pragma unroll
      for (int i = e; i < e + 4; ++i)
        if (first + i * step < width) v[i] += row[first + i * step];
    }
  }
}

// Sums of run blockIdx.x, for the columns that a thread has.
template <class T, int N, bool WIDE>
__global__ void __launch_bounds__(256) run_kernel(const SumArgs a) {
  __shared__ int ids[kRun + 2], tokens[kRun];  // ids[0] and ids[count + 1]: the neighbours'
  const int begin = blockIdx.x * kRun, count = min(kRun, a.n - begin);
  for (int i = threadIdx.x; i < count + 2; i += blockDim.x) {
    const int at = begin + i - 1;
    ids[i] = at >= 0 && at < a.n ? a.ids[at] : -1;
    if (i < count) tokens[i] = a.tokens[begin + i];
  }
  __syncthreads();
  const int c = first_of<N, WIDE>(blockIdx.y, blockDim.x, threadIdx.x), step = blockDim.x;
  if (c >= a.width) return;
  float sum[N] = {};
  Part<T, N, WIDE> v[kRun];  // all rows on their way
#pragma unroll
  for (int i = 0; i < kRun; ++i)
    v[i].load(static_cast<const T*>(a.dy) + tokens[min(i, count - 1)] * a.dy_stride, c, step, a.width);
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    if (i >= count) break;
    const int id = ids[i + 1], next = ids[i + 2];
    float f[N];
    v[i].widen(f);
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] += f[e];
    if (id == next && i < count - 1) continue;
    if (id < a.vocab) {
      const bool older = id == ids[0];  // sorted: all from the run's first on
      if (older || id == next) {
        put_sums<N, WIDE>(a.parts + ((long long)blockIdx.x * 2 + (older ? 0 : 1)) * a.width, c, step, a.width, sum);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] *= a.scale;
        Part<T, N, WIDE>::of(sum).store(static_cast<T*>(a.out) + (long long)id * a.width, c, step, a.width);
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] = 0.f;
  }
}

// Ids that begin in one of the block's eight runs and go on behind it.  A warp looks at a run and joins up to eight that
// follow it by itself.  An id that goes on further has the blocks whose runs have no other to help the one where it
// begins: they share out its columns in fours (of the 32 threads' that gridDim.y parts have), and a block's threads the
// runs, whose sums are added in order.  200000 tokens of 50257 words 24 us (each joined by all warps of a block: 68),
// with a quarter of them one word's 60 (by its first block alone: 188).
template <class T, int N, bool WIDE>
__global__ void __launch_bounds__(256) join_kernel(const SumArgs a) {
  constexpr int SHARES = 32, LANES = 8;
  __shared__ float sums[SHARES][N][LANES + 1];
  __shared__ int head;  // the run where an id of more than nine runs begins: one in eight at most
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, runs = (a.n + kRun - 1) / kRun, run8 = blockIdx.x * 8;
  const auto begins = [&](int run, int id) { return run < runs && a.ids[min(run, runs - 1) * kRun] == id; };
  if (threadIdx.x == 0) head = -1;
  __syncthreads();
  {
    const int run = run8 + warp, begin = run * kRun, end = begin + kRun;
    int id = -1;
    if (end < a.n) {  // the last run goes on nowhere
      const int last = a.ids[end - 1], before = a.ids[max(begin - 1, 0)], first = a.ids[begin], next = a.ids[end];
      if (next == last && last < a.vocab && !(begin > 0 && first == last && before == last)) id = last;
    }
    const bool more = id >= 0 && lane < 8 && begins(run + 2 + lane, id);
    const int count = 1 + __popc(__ballot_sync(0xffffffffu, more));
    if (id >= 0 && count > 8) {
      if (lane == 0) head = run;
    } else if (id >= 0) {
      const int c = first_of<N, WIDE>(blockIdx.y, 32, lane);
      if (c < a.width) {
        float sum[N] = {};
        add_sums<N, WIDE>(a.parts + ((long long)run * 2 + 1) * a.width, c, 32, a.width, sum);
#pragma unroll 4
        for (int r = 0; r < count; ++r)
          add_sums<N, WIDE>(a.parts + ((long long)run + 1 + r) * 2 * a.width, c, 32, a.width, sum);
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] *= a.scale;
        Part<T, N, WIDE>::of(sum).store(static_cast<T*>(a.out) + (long long)id * a.width, c, 32, a.width);
      }
    }
  }
  __syncthreads();
  // sorted: the runs that begin with an id follow each other
  int run0 = head, id;
  if (run0 >= 0) {
    id = a.ids[min(run0 * kRun + kRun, a.n) - 1];
  } else {
    if (run8 == 0 || run8 + 8 >= runs) return;
    id = a.ids[run8 * kRun];
    if (id >= a.vocab || a.ids[run8 * kRun - 1] != id || a.ids[(run8 + 8) * kRun] != id) return;
    run0 = run8;  // the first that begins with it
    for (int more = 256; more == 256;) {
      const int run = run0 - 1 - (int)threadIdx.x;
      more = __syncthreads_count(run >= 0 && begins(run, id));
      run0 -= more;
    }
    if (run0 > 0 && a.ids[run0 * kRun - 1] == id) --run0;
  }
  int last = head >= 0 ? run0 + 1 : run8 + 8;  // the last that does
  for (int more = 256; more == 256;) {
    more = __syncthreads_count(begins(last + 1 + threadIdx.x, id));
    last += more;
  }
  const int count = last - run0, rank = blockIdx.x - run0 / 8, helpers = max(1, last / 8 - run0 / 8);
  const int share = threadIdx.x / LANES, at = threadIdx.x % LANES;
  for (int slice = rank; slice < 32 / LANES; slice += helpers) {
    const int c = first_of<N, WIDE>(blockIdx.y, 32, slice * LANES + at);
    float sum[N] = {};
    if (c < a.width) {
      if (share == 0) add_sums<N, WIDE>(a.parts + ((long long)run0 * 2 + 1) * a.width, c, 32, a.width, sum);
      const int to = (int)((long long)count * (share + 1) / SHARES);
#pragma unroll 8
      for (int r = (int)((long long)count * share / SHARES); r < to; ++r)
        add_sums<N, WIDE>(a.parts + ((long long)run0 + 1 + r) * 2 * a.width, c, 32, a.width, sum);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) sums[share][e][at] = sum[e];
    __syncthreads();
    if (share < N) {
      float s = sums[0][share][at];
#pragma unroll 8
      for (int w = 1; w < SHARES; ++w) s += sums[w][share][at];
      sums[0][share][at] = s * a.scale;  // this thread's own
    }
    __syncthreads();
    if (share == 0 && c < a.width) {
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] = sums[0][e][at];
      Part<T, N, WIDE>::of(sum).store(static_cast<T*>(a.out) + (long long)id * a.width, c, 32, a.width);
    }
    __syncthreads();
  }
}

// Passes of the sort and bits of each, for ids 0 .. vocab (vocab: none).
int bits_of(long long vocab, int* passes) {
  int bits = 1;
  while (vocab >> bits) ++bits;
  *passes = (bits + 8) / 9;
  return (bits + *passes - 1) / *passes;
}

// Parts of the gradient's workspace.
struct Room {
  size_t values[2], ids, counts, parts, bytes;
};
Room room_of(long long n, long long vocab, int width) {
  int passes;
  const int bits = bits_of(vocab, &passes);
  Room r;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  r.values[0] = take(n * 4);
  r.values[1] = take(n * 4);
  r.ids = take(n * 4);
  r.counts = take(sorting::counts_bytes(n, 1 << bits));
  r.parts = take((size_t)((n + kRun - 1) / kRun) * 2 * width * 4);
  r.bytes = at;
  return r;
}

int check(int id_bytes, long long n, long long vocab, int width, int type) {
  if (id_bytes != 4 && id_bytes != 8) return efail(TAO_ERR_ARG, "ids have 32 or 64 bits");
  if (!known(type)) return efail(TAO_ERR_ARG, "a table is bf16, fp16 or fp32");
  if (n < 0 || n > (1ll << 30) || vocab < 1 || vocab > (1ll << 26) || width < 1 || width > (1 << 20))
    return efail(TAO_ERR_ARG, "there are up to 2^30 ids and 1 to 2^26 rows of 1 to 2^20 channels");
  return TAO_OK;
}

}  // namespace
}  // namespace tao

extern "C" {

int tao_embed(const void* ids, int id_bytes, long long n, const void* table, long long stride, long long vocab, int width,
              int type, float scale, void* y, void* stream) {
  using namespace tao;
  if (int rc = check(id_bytes, n, vocab, width, type)) return rc;
  if (n == 0) return TAO_OK;
  const size_t size = size_of(type);
  if (!ids || !table || !y) return efail(TAO_ERR_ARG, "null pointer");
  if (!on_elements({{ids, (size_t)id_bytes}, {table, size}, {y, size}}))
    return efail(TAO_ERR_ARG, "operands start on a whole element");
  if (overlaps(y, n * width * size, {extent(table, vocab, stride * size, width * size), extent(ids, 1, 0, n * id_bytes)}))
    return efail(TAO_ERR_ARG, "embedded rows must not overlap the table or the ids");
  const EmbedArgs a = {ids, n, vocab, stride, width, id_bytes == 8, scale, table, y};
  const bool wide = width * size % 16 == 0 && on16(table, stride, size) && on16(y, 0, size);
  return by_part(type, wide, [&](auto t, auto v, auto w) {
    const Mapping m = mapping(n, (width + decltype(v)::value - 1) / decltype(v)::value);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if ((long long)m.grid.x * m.grid.y < 148 * 8) {  // all at once, a token a thread (32768x768: 22 us, four a thread 13)
      embed_kernel<decltype(t), decltype(v)::value, decltype(w)::value, 1><<<m.grid, m.block, 0, s>>>(a);
    } else {
      const dim3 grid((m.grid.x + 3) / 4, m.grid.y);
      embed_kernel<decltype(t), decltype(v)::value, decltype(w)::value, 4><<<grid, m.block, 0, s>>>(a);
    }
    return launched(cudaGetLastError());
  });
}

size_t tao_embed_gradient_workspace_bytes(long long n, long long vocab, int width) {
  return n <= 0 || vocab < 1 || width < 1 ? 0 : tao::room_of(n, vocab, width).bytes;
}

int tao_embed_gradient(const void* ids, int id_bytes, long long n, const void* dy, long long dy_stride, long long vocab,
                       int width, int type, float scale, void* dtable, void* workspace, size_t workspace_bytes,
                       void* stream) {
  using namespace tao;
  if (int rc = check(id_bytes, n, vocab, width, type)) return rc;
  const size_t size = size_of(type);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!dtable) return efail(TAO_ERR_ARG, "null pointer");
  if (!on_elements({{ids, (size_t)id_bytes}, {dy, size}, {dtable, size}}))
    return efail(TAO_ERR_ARG, "operands start on a whole element");
  if (n > 0) {
    if (!ids || !dy) return efail(TAO_ERR_ARG, "null pointer");
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 ||
        workspace_bytes < tao_embed_gradient_workspace_bytes(n, vocab, width))
      return efail(TAO_ERR_ARG, "workspace too small for the embedding's gradient, or off 16 bytes");
  }
  if (overlaps(dtable, vocab * width * size, {extent(dy, n, dy_stride * size, width * size), extent(ids, 1, 0, n * id_bytes)}))
    return efail(TAO_ERR_ARG, "the table's gradient must not overlap the rows' or the ids");
  if (n == 0) return launched(cudaMemsetAsync(dtable, 0, (size_t)vocab * width * size, s));
  cudaError_t e = cudaSuccess;
  const Room r = room_of(n, vocab, width);
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  int passes;
  const int bits = bits_of(vocab, &passes);
  sorting::Pass p = {};
  sorting::Clearing zeros = {static_cast<uint8_t*>(dtable), vocab * width * (long long)size, passes * sorting::launches_of(n)};
  p.ids = ids, p.limit = vocab, p.n = (int)n, p.bins = 1 << bits, p.wide = id_bytes == 8;
  for (int i = 0; i < passes; ++i) {
    p.shift = i * bits;
    p.sorted = reinterpret_cast<int*>(ws + r.values[i & 1]);
    p.keys = i + 1 == passes ? reinterpret_cast<int*>(ws + r.ids) : nullptr;
    e = sorting::run(p, reinterpret_cast<int*>(ws + r.counts), s, &zeros);
    if (e != cudaSuccess) return launched(e);
    p.values = p.sorted;
  }
  const SumArgs a = {p.values, reinterpret_cast<const int*>(ws + r.ids), (int)n, (int)vocab, width, scale, dy, dy_stride,
                     dtable, reinterpret_cast<float*>(ws + r.parts)};
  const bool wide = width * size % 16 == 0 && on16(dy, dy_stride, size) && on16(dtable, 0, size);
  return by_part(type, wide, [&](auto t, auto v, auto w) {
    constexpr int N = decltype(v)::value;
    const int vectors = (width + N - 1) / N, threads = std::min(256, (vectors + 31) / 32 * 32);
    const dim3 grid((unsigned)((n + kRun - 1) / kRun), (vectors + threads - 1) / threads);
    run_kernel<decltype(t), N, decltype(w)::value><<<grid, threads, 0, s>>>(a);
    if (grid.x > 1)
      join_kernel<decltype(t), N, decltype(w)::value><<<dim3((grid.x + 6) / 8, (vectors + 31) / 32), 256, 0, s>>>(a);
    return launched(cudaGetLastError());
  });
}

}  // extern "C"
