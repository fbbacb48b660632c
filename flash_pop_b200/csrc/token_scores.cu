// Log probabilities of given tokens under rows of logits, with the rows' entropies and most likely alternatives, and the
// gradient of all three.  With m = max z, s = sum exp(z - m):
//   log p_j = (z_j - m) - log s,   H = log s - sum exp(z - m) (z - m) / s
//   dz_j = -p_j (G + g_H (log p_j + H)) + [j = token] g + sum over alternatives a of [j = a] g_a,   G = g + sum of g_a
// The order of the alternatives is that of the logits, equal ones by index, NaN (which makes every number of the row NaN) first.
// A row of -inf only has no distribution: log p = -inf, H = 0, no gradient.
// Bound by HBM: one read forward, one read and one write backward.
#include "fpb_common.cuh"
#include "vec_io.cuh"

namespace fpb {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;

struct ScoreParams {
  const void* logits; int64_t row_stride;
  const int64_t* tokens;
  float *logprob, *entropy, *stats;                 // stats: (rows, 2) of m and log s
  float* top_logprob; int64_t* top_tokens;          // (rows, top)
  int64_t rows;
  int32_t V, top;
};

// order of the values in 32 bits, equal ones by index in the lower 32: unique, never 0
__device__ __forceinline__ uint64_t rank_key(float z, int index) {
  z += 0.0f;                                        // (-0 is 0)
  const uint32_t b = __float_as_uint(z);
  const uint32_t order = z != z ? 0xffffffffu : (b & 0x80000000u ? ~b : b | 0x80000000u);
  return (uint64_t)order << 32 | (uint32_t)~index;
}

constexpr float LEAST = -1e4f;

// max(a, LEAST), or NaN where a is
__device__ __forceinline__ float at_least(float a) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(LEAST));
  return r;
}

// running (max, sum of exp(z - max), sum of exp(z - max) (z - max)); nothing yet, or only -inf: max = -inf, sums 0
struct Stats {
  float m, s, t;
};
__device__ __forceinline__ void merge(Stats& a, const Stats& b) {
  if (b.m != b.m || a.m != a.m) { a.m = NAN; a.s = a.t = NAN; return; }
  if (b.m == -INFINITY) return;
  if (a.m == -INFINITY) { a = b; return; }
  // (differences below LEAST count as that: their exponential is 0 as well, and no product of theirs overflows)
  const float m = fmaxf(a.m, b.m), da = fmaxf(a.m - m, LEAST), db = fmaxf(b.m - m, LEAST);
  const float ea = expf(da), eb = expf(db);
  a.t = ea * (a.t + a.s * da) + eb * (b.t + b.s * db);
  a.s = ea * a.s + eb * b.s;
  a.m = m;
}
__device__ __forceinline__ void add(Stats& a, float z) { merge(a, Stats{z, 1.0f, 0.0f}); }

__device__ __forceinline__ uint64_t warp_max(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o);
    v = v > w ? v : w;
  }
  return v;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) scores_kernel(const __grid_constant__ ScoreParams p) {
  const int64_t row = blockIdx.x;
  const T* z = (const T*)p.logits + row * p.row_stride;
  Stats a{-INFINITY, 0.0f, 0.0f};
  for (int c = threadIdx.x; c < p.V; c += THREADS) add(a, to_float(z[c]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    merge(a, Stats{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.t, o)});
  __shared__ Stats parts[WARPS];
  __shared__ uint64_t keys[2][WARPS];
  if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = a;
  __syncthreads();
  a = parts[0];
  for (int w = 1; w < WARPS; ++w) merge(a, parts[w]);
  const bool empty = a.m == -INFINITY;
  const float ls = empty ? 0.0f : a.m == INFINITY ? NAN : logf(a.s);
  if (threadIdx.x == 0) {
    const int64_t t = p.tokens[row];
    p.logprob[row] = t >= 0 && t < p.V ? (empty ? -INFINITY : (to_float(z[t]) - a.m) - ls) : 0.0f;
    p.entropy[row] = empty ? 0.0f : ls - a.t / a.s;
    p.stats[2 * row] = a.m;
    p.stats[2 * row + 1] = ls;
  }
  // one alternative after another: the largest key below the last one
  uint64_t last = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    uint64_t best = 0;
    for (int c = threadIdx.x; c < p.V; c += THREADS) {
      const uint64_t key = rank_key(to_float(z[c]), c);
      if (key < last && key > best) best = key;
    }
    best = warp_max(best);
    if ((threadIdx.x & 31) == 0) keys[k & 1][threadIdx.x >> 5] = best;
    __syncthreads();
    for (int w = 0; w < WARPS; ++w) best = best > keys[k & 1][w] ? best : keys[k & 1][w];
    last = best;
    if (threadIdx.x == 0) {
      const int c = (int)~(uint32_t)best;
      p.top_tokens[row * p.top + k] = c;
      p.top_logprob[row * p.top + k] = empty ? -INFINITY : (to_float(z[c]) - a.m) - ls;
    }
  }
}

struct ScoreGradParams {
  const void* logits; int64_t row_stride;
  const int64_t* tokens;
  const float *entropy, *stats;
  const int64_t* top_tokens;
  const float *g_logprob, *g_entropy, *g_top;       // each may be null
  void* d_logits; int64_t d_stride;
  int64_t rows;
  int32_t V, top;
};

template <typename T>
__global__ void __launch_bounds__(THREADS) scores_grad_kernel(const __grid_constant__ ScoreGradParams p) {
  const int64_t row = blockIdx.x;
  const T* z = (const T*)p.logits + row * p.row_stride;
  T* d = (T*)p.d_logits + row * p.d_stride;
  const float m = p.stats[2 * row], ls = p.stats[2 * row + 1], H = p.entropy[row];
  const int64_t t = p.tokens[row];
  const float g = p.g_logprob && t >= 0 && t < p.V ? p.g_logprob[row] : 0.0f, gh = p.g_entropy ? p.g_entropy[row] : 0.0f;
  float total = g;
  if (p.g_top)
    for (int k = 0; k < p.top; ++k) total += p.g_top[row * p.top + k];
  for (int c = threadIdx.x; c < p.V; c += THREADS) {
    float v = 0.0f;
    if (m != -INFINITY) {
      const float lp = at_least((to_float(z[c]) - m) - ls);
      v = -expf(lp) * (total + gh * (lp + H));
      if (c == t) v += g;
      if (p.g_top)
        for (int k = 0; k < p.top; ++k)
          if (p.top_tokens[row * p.top + k] == c) v += p.g_top[row * p.top + k];
    }
    d[c] = from_float<T>(v);
  }
}

}  // namespace

int launch_token_scores(int dtype, int64_t rows, int V, int top, const void* logits, int64_t row_stride, const int64_t* tokens, float* logprob,
                        float* entropy, float* stats, float* top_logprob, int64_t* top_tokens, cudaStream_t stream) {
  const ScoreParams p{logits, row_stride, tokens, logprob, entropy, stats, top_logprob, top_tokens, rows, V, top};
  const cudaError_t e = dtype == FPB_BF16 ? launch_kernel(scores_kernel<__nv_bfloat16>, dim3((unsigned)rows), THREADS, 0, false, p, stream)
                                          : launch_kernel(scores_kernel<float>, dim3((unsigned)rows), THREADS, 0, false, p, stream);
  return e == cudaSuccess ? FPB_OK : FPB_ERR_LAUNCH;
}

int launch_token_scores_grad(int dtype, int64_t rows, int V, int top, const void* logits, int64_t row_stride, const int64_t* tokens,
                             const float* entropy, const float* stats, const int64_t* top_tokens, const float* g_logprob,
                             const float* g_entropy, const float* g_top, void* d_logits, int64_t d_stride, cudaStream_t stream) {
  const ScoreGradParams p{logits, row_stride, tokens, entropy, stats, top_tokens, g_logprob, g_entropy, g_top, d_logits, d_stride, rows, V, top};
  const cudaError_t e = dtype == FPB_BF16 ? launch_kernel(scores_grad_kernel<__nv_bfloat16>, dim3((unsigned)rows), THREADS, 0, false, p, stream)
                                          : launch_kernel(scores_grad_kernel<float>, dim3((unsigned)rows), THREADS, 0, false, p, stream);
  return e == cudaSuccess ? FPB_OK : FPB_ERR_LAUNCH;
}

}  // namespace fpb
