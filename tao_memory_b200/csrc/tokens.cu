// Tokens sorted by expert and back: the order (sort.cuh), rows copied to their pairs' places, and the experts'
// rows added into their tokens by weight, with the gradients.  All bound by their bytes: a thread has 16 bytes of
// a token's row and goes over the token's pairs, so that x is read and y written once; a token's pairs are added
// in the order of its choices.  32768 tokens of 768 bf16 channels to 4 of 64 experts: gather 38 us (6.6 TB/s), return 50
// (5.0; 80 while a branch stood between a pair's place and its row), rows' gradient 45, weights' gradient 56.
#include <cuda_runtime.h>

#include "rows.cuh"
#include "sort.cuh"

void tao_set_last_error(const char* msg);

namespace tao {
namespace {

using namespace rows;

int tfail(int code, const char* msg) {
  tao_set_last_error(msg);
  return code;
}
int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TAO_OK : tfail(TAO_ERR_CUDA, cudaGetErrorString(e));
}

struct TokenArgs {
  const int* places;  // [tokens][k]
  const int* kept;    // pairs that have an expert (their places come first), or null: all
  long long tokens, pairs;
  int k, width;
  const void *in, *other, *weights;  // rows; weights null: ones
  long long in_stride, other_stride;
  int weight_type;
  void *out, *dw;
};

// At most all pairs, whatever the number says.
TAO_DEVI int kept_of(const TokenArgs& a) {
  return a.kept ? (int)min((long long)max(*a.kept, 0), a.pairs) : (int)a.pairs;
}

// out[places[t][j]] = in[t], or, WEIGHTED, weights[t][j] in[t] (zeros for a pair that is not kept).
template <class T, int N, bool WIDE, bool WEIGHTED>
__global__ void __launch_bounds__(256) gather_kernel(const TokenArgs a) {
  const long long t = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  const int c = first_of<N, WIDE>(blockIdx.y, blockDim.x, threadIdx.x), step = blockDim.x;
  if (t >= a.tokens || c >= a.width) return;
  const int kept = WEIGHTED ? kept_of(a) : 0;
  Part<T, N, WIDE> v;
  v.load(static_cast<const T*>(a.in) + t * a.in_stride, c, step, a.width);
#pragma unroll 4
  for (int j = 0; j < a.k; ++j) {
    const int place = a.places[t * a.k + j];
    if ((unsigned)place >= (unsigned)a.pairs) continue;
    T* const to = static_cast<T*>(a.out) + (long long)place * a.width;
    if constexpr (WEIGHTED) {
      const float w = a.weights ? value_of(a.weights, t * a.k + j, a.weight_type) : 1.f;
      float f[N];
      v.widen(f);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = place < kept ? f[i] * w : 0.f;
      Part<T, N, WIDE>::of(f).store(to, c, step, a.width);
    } else {
      v.store(to, c, step, a.width);
    }
  }
}

// out[t] = sum over j of weights[t][j] in[places[t][j]]
// AT_ONCE: rows on their way; no branch stands between their places and their loads.
template <class T, int N, bool WIDE, int AT_ONCE>
__global__ void __launch_bounds__(256) return_kernel(const TokenArgs a) {
  const long long t = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  const int c = first_of<N, WIDE>(blockIdx.y, blockDim.x, threadIdx.x), step = blockDim.x;
  if (t >= a.tokens || c >= a.width) return;
  const int kept = kept_of(a);
  float sum[N] = {};
  for (int j0 = 0; j0 < a.k; j0 += AT_ONCE) {
    int place[AT_ONCE];
    float w[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) place[j] = a.places[t * a.k + min(j0 + j, a.k - 1)];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) w[j] = a.weights ? value_of(a.weights, t * a.k + min(j0 + j, a.k - 1), a.weight_type) : 1.f;
    Part<T, N, WIDE> v[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const bool in = j0 + j < a.k && (unsigned)place[j] < (unsigned)kept;
      v[j].load(static_cast<const T*>(a.in) + (in ? place[j] : 0) * a.in_stride, c, step, a.width);
      place[j] = in;
    }
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      float f[N];
      v[j].widen(f);
#pragma unroll
      for (int i = 0; i < N; ++i) sum[i] = place[j] ? sum[i] + w[j] * f[i] : sum[i];
    }
  }
  Part<T, N, WIDE>::of(sum).store(static_cast<T*>(a.out) + t * a.width, c, step, a.width);
}

// dw[t][j] = in[t] . other[places[t][j]], zero for a pair that is not kept.  WARPS a token (one, or where that leaves the
// device empty eight, whose sums are added in their order: 100 tokens of 3584 fp32 channels to 6 experts 6.3 us, by one
// warp each 21.5), AT_ONCE experts' rows on their way at once.  (In one
// kernel with the rows' gradient, which writes as much as this reads, the two took 115 to 156 us for 32768 tokens of 768
// channels and 4 experts.)
template <class T, int N, bool WIDE, int AT_ONCE, int WARPS>
__global__ void __launch_bounds__(256) weight_gradient_kernel(const TokenArgs a) {
  __shared__ float parts[AT_ONCE][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long t = WARPS == 1 ? (long long)blockIdx.x * 8 + warp : (long long)blockIdx.x;
  if (t >= a.tokens) return;
  const int kept = kept_of(a);
  const T* const dy = static_cast<const T*>(a.in) + t * a.in_stride;
  for (int j0 = 0; j0 < a.k; j0 += AT_ONCE) {
    const T* rows[AT_ONCE];
    float dot[AT_ONCE] = {};
    bool in[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int place = a.places[t * a.k + min(j0 + j, a.k - 1)];
      in[j] = (unsigned)place < (unsigned)kept;
      rows[j] = static_cast<const T*>(a.other) + (in[j] ? place : 0) * a.other_stride;
    }
#pragma unroll 2
    for (int c = first_of<N, WIDE>(WARPS == 1 ? 0 : warp, 32, lane); c < a.width; c += WARPS * 32 * N) {
      Part<T, N, WIDE> v[AT_ONCE], y;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) v[j].load(rows[j], c, 32, a.width);
      float d[N], f[N];
      y.load(dy, c, 32, a.width);
      y.widen(d);
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        v[j].widen(f);
#pragma unroll
        for (int i = 0; i < N; ++i) dot[j] += d[i] * f[i];
      }
    }
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      float s = warp_sum(dot[j]);
      if constexpr (WARPS > 1) {
        if (lane == 0) parts[j][warp] = s;
        __syncthreads();
        s = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) s += parts[j][w];
      }
      if (lane == 0 && (WARPS == 1 || warp == 0) && j0 + j < a.k)
        set_value(a.dw, t * a.k + j0 + j, in[j] ? s : 0.f, a.weight_type);
    }
    if constexpr (WARPS > 1) __syncthreads();
  }
}
template <class T, int N, bool WIDE, int AT_ONCE>
void start_weight_gradient(const TokenArgs& a, cudaStream_t s) {
  if (a.tokens <= 148 * 8)
    weight_gradient_kernel<T, N, WIDE, AT_ONCE, 8><<<(unsigned)a.tokens, 256, 0, s>>>(a);
  else
    weight_gradient_kernel<T, N, WIDE, AT_ONCE, 1><<<(unsigned)((a.tokens + 7) / 8), 256, 0, s>>>(a);
}

int check(const TokenArgs& a, int type) {
  if (!known(type)) return tfail(TAO_ERR_ARG, "tokens are bf16, fp16 or fp32");
  if (a.weights && a.weight_type != TAO_TYPE_FP32 && a.weight_type != type)
    return tfail(TAO_ERR_ARG, "weights are fp32 or of the rows' type");
  if (a.tokens < 0 || a.k < 1 || a.width < 1 || a.k > (1 << 20) || a.width > (1 << 20) || a.tokens > (1ll << 30) / a.k)
    return tfail(TAO_ERR_ARG, "a token has at least one choice and 1 to 2^20 channels, and there are up to 2^30 pairs");
  return TAO_OK;
}

}  // namespace
}  // namespace tao

extern "C" {

size_t tao_sort_tokens_workspace_bytes(long long pairs, int experts) {
  return pairs <= 0 || experts < 1 ? 0 : tao::sorting::counts_bytes(pairs, experts + 1);
}

int tao_sort_tokens(const void* ids, int id_bytes, long long pairs, int experts, int* sorted, int* places, int* offsets,
                    void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tao;
  if (id_bytes != 4 && id_bytes != 8) return tfail(TAO_ERR_ARG, "ids have 32 or 64 bits");
  if (experts < 1 || experts >= sorting::kMostBins) return tfail(TAO_ERR_ARG, "there are 1 to 512 experts");
  if (pairs < 0 || pairs > (1ll << 30)) return tfail(TAO_ERR_ARG, "there are up to 2^30 pairs");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!offsets) return tfail(TAO_ERR_ARG, "null pointer");
  if (!on_elements({{ids, (size_t)id_bytes}, {sorted, 4}, {places, 4}, {offsets, 4}, {workspace, 4}}))
    return tfail(TAO_ERR_ARG, "operands start on a whole element");
  if (pairs == 0) {
    const cudaError_t e = cudaMemsetAsync(offsets, 0, (experts + 1) * sizeof(int), s);
    return e == cudaSuccess ? TAO_OK : tfail(TAO_ERR_CUDA, cudaGetErrorString(e));
  }
  if (!ids || !sorted || !places) return tfail(TAO_ERR_ARG, "null pointer");
  const Extent id = extent(ids, 1, 0, pairs * id_bytes), by = extent(sorted, 1, 0, pairs * 4), at = extent(places, 1, 0, pairs * 4);
  if (overlaps(sorted, pairs * 4, {id, at}) || overlaps(places, pairs * 4, {id}) ||
      overlaps(offsets, (experts + 1) * 4ll, {id, by, at}))
    return tfail(TAO_ERR_ARG, "an order's parts must not overlap each other or the ids");
  const size_t need = tao_sort_tokens_workspace_bytes(pairs, experts);
  if (need && (!workspace || workspace_bytes < need)) return tfail(TAO_ERR_ARG, "workspace too small for the sort");
  sorting::Pass p = {};
  p.ids = ids, p.limit = experts, p.n = (int)pairs, p.shift = -1, p.bins = experts + 1, p.wide = id_bytes == 8;
  p.sorted = sorted, p.places = places, p.offsets = offsets;
  const cudaError_t e = sorting::run(p, static_cast<int*>(workspace), s);
  return e == cudaSuccess ? TAO_OK : tfail(TAO_ERR_CUDA, cudaGetErrorString(e));
}

int tao_gather_tokens(const void* x, long long x_stride, const int* places, long long tokens, int top_k, int width,
                      int type, void* xs, void* stream) {
  using namespace tao;
  TokenArgs a = {};
  a.places = places, a.tokens = tokens, a.k = top_k, a.width = width, a.in = x, a.in_stride = x_stride, a.out = xs;
  if (int rc = check(a, type)) return rc;
  if (tokens == 0) return TAO_OK;
  a.pairs = tokens * top_k;
  const size_t size = size_of(type);
  if (!x || !places || !xs) return tfail(TAO_ERR_ARG, "null pointer");
  if (!on_elements({{x, size}, {xs, size}, {places, 4}})) return tfail(TAO_ERR_ARG, "operands start on a whole element");
  if (overlaps(xs, a.pairs * width * size, {extent(x, tokens, x_stride * size, width * size), extent(places, 1, 0, a.pairs * 4)}))
    return tfail(TAO_ERR_ARG, "gathered rows must not overlap what they are gathered from");
  const bool wide = width * size % 16 == 0 && on16(x, x_stride, size) && on16(xs, 0, size);
  return by_part(type, wide, [&](auto t, auto n, auto w) {
    const Mapping m = mapping(tokens, (width + decltype(n)::value - 1) / decltype(n)::value);
    gather_kernel<decltype(t), decltype(n)::value, decltype(w)::value, false><<<m.grid, m.block, 0, static_cast<cudaStream_t>(stream)>>>(a);
    return launched();
  });
}

int tao_return_tokens(const void* ys, long long ys_stride, const int* places, const int* kept, const void* weights,
                      int weight_type, long long tokens, int top_k, int width, int type, void* y, void* stream) {
  using namespace tao;
  TokenArgs a = {};
  a.places = places, a.kept = kept, a.tokens = tokens, a.k = top_k, a.width = width, a.in = ys, a.in_stride = ys_stride;
  a.weights = weights, a.weight_type = weight_type, a.out = y;
  if (int rc = check(a, type)) return rc;
  if (tokens == 0) return TAO_OK;
  a.pairs = tokens * top_k;
  const size_t size = size_of(type);
  if (!ys || !places || !y) return tfail(TAO_ERR_ARG, "null pointer");
  if (!on_elements({{ys, size}, {y, size}, {places, 4}, {kept, 4}, {weights, weights ? size_of(weight_type) : 1}}))
    return tfail(TAO_ERR_ARG, "operands start on a whole element");
  if (overlaps(y, tokens * width * size, {extent(ys, a.pairs, ys_stride * size, width * size), extent(places, 1, 0, a.pairs * 4),
                                          extent(kept, 1, 0, 4), extent(weights, 1, 0, a.pairs * size_of(weight_type))}))
    return tfail(TAO_ERR_ARG, "returned rows must not overlap what they are made of");
  const bool wide = width * size % 16 == 0 && on16(ys, ys_stride, size) && on16(y, 0, size);
  return by_part(type, wide, [&](auto t, auto n, auto w) {
    const Mapping m = mapping(tokens, (width + decltype(n)::value - 1) / decltype(n)::value);
    using T = decltype(t);
    constexpr int N = decltype(n)::value;
    constexpr bool WIDE = decltype(w)::value;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (top_k == 1)
      return_kernel<T, N, WIDE, 1><<<m.grid, m.block, 0, s>>>(a);
    else if (top_k == 2)
      return_kernel<T, N, WIDE, 2><<<m.grid, m.block, 0, s>>>(a);
    else
      return_kernel<T, N, WIDE, 4><<<m.grid, m.block, 0, s>>>(a);
    return launched();
  });
}

int tao_return_tokens_gradient(const void* dy, long long dy_stride, const void* ys, long long ys_stride, const int* places,
                               const int* kept, const void* weights, int weight_type, long long tokens, int top_k,
                               int width, int type, void* dys, void* dw, void* stream) {
  using namespace tao;
  TokenArgs a = {};
  a.places = places, a.kept = kept, a.tokens = tokens, a.k = top_k, a.width = width, a.in = dy, a.in_stride = dy_stride;
  a.other = ys, a.other_stride = ys_stride, a.weights = weights, a.weight_type = weight_type, a.out = dys, a.dw = dw;
  if (int rc = check(a, type)) return rc;
  if (tokens == 0) return TAO_OK;
  a.pairs = tokens * top_k;
  const size_t size = size_of(type);
  if (!dy || !places || (!dys && !dw) || (dw && (!ys || !weights))) return tfail(TAO_ERR_ARG, "null pointer");
  const size_t weight_size = weights ? size_of(weight_type) : 1;
  if (!on_elements({{dy, size}, {ys, size}, {dys, size}, {places, 4}, {kept, 4}, {weights, weight_size}, {dw, weight_size}}))
    return tfail(TAO_ERR_ARG, "operands start on a whole element");
  const long long out = a.pairs * width * size;
  const Extent from = extent(dy, tokens, dy_stride * size, width * size), rows_of = extent(ys, a.pairs, ys_stride * size, width * size),
               at = extent(places, 1, 0, a.pairs * 4), number = extent(kept, 1, 0, 4),
               by = extent(weights, 1, 0, a.pairs * (long long)weight_size);
  if (overlaps(dys, out, {from, rows_of, at, number, by}) ||
      overlaps(dw, a.pairs * (long long)weight_size, {from, rows_of, at, number, by, extent(dys, 1, 0, out)}))
    return tfail(TAO_ERR_ARG, "gradients must not overlap what they are made of");
  const bool wide = width * size % 16 == 0 && on16(dy, dy_stride, size) && on16(ys, ys_stride, size) && on16(dys, 0, size);
  return by_part(type, wide, [&](auto t, auto n, auto w) {
    using T = decltype(t);
    constexpr int N = decltype(n)::value;
    constexpr bool WIDE = decltype(w)::value;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const Mapping m = mapping(tokens, (width + N - 1) / N);
    if (dys) gather_kernel<T, N, WIDE, true><<<m.grid, m.block, 0, s>>>(a);
    if (dw && top_k == 1)
      start_weight_gradient<T, N, WIDE, 1>(a, s);
    else if (dw && top_k == 2)
      start_weight_gradient<T, N, WIDE, 2>(a, s);
    else if (dw)
      start_weight_gradient<T, N, WIDE, 4>(a, s);
    return launched();
  });
}

}  // extern "C"
