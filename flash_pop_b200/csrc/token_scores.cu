// Log probabilities of given tokens under rows of logits, with the rows' entropies and most likely alternatives, and the
// gradient of all three.  With m = max z, s = sum exp(z - m):
//   log p_j = (z_j - m) - log s,   H = log s - sum exp(z - m) (z - m) / s
//   dz_j = -p_j (G + g_H (log p_j + H)) + [j = token] g + sum over alternatives a of [j = a] g_a,   G = g + sum of g_a
// The order of the alternatives is that of the logits, equal ones by index, NaN (which makes every number of the row NaN) first.
// A row of -inf only has no distribution: log p = -inf, H = 0, no gradient.
// Bound by HBM: one read forward, one read and one write backward.
#include <type_traits>

#include "fpb_common.cuh"
#include "vec_io.cuh"

namespace fpb {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr float LEAST = -1e4f;
constexpr unsigned ALL = 0xffffffffu;

// max(a, LEAST), or NaN where a is
__device__ __forceinline__ float at_least(float a) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(LEAST));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// e^x by the hardware's 2^x; results below the smallest normal number are 0
__device__ __forceinline__ float exponential(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.44269504088896f));
  return r;
}

// ---- a row as vectors -----------------------------------------------------------------------------------------------
// A row starts at any element; it is read as the 16-byte vectors that it lies in, the first and the last element by element.
template <typename T> struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* z;
  int V, skew, vectors;             // element i is number (i + skew) % E of vector (i + skew) / E

  __device__ Row(const void* logits, int64_t row, int64_t stride, int n) : z((const T*)logits + row * stride), V(n) {
    skew = (int)(((uintptr_t)z % 16) / sizeof(T));
    vectors = (skew + V + E - 1) / E;
  }
  __device__ __forceinline__ int index(int vector, int e) const { return vector * E + e - skew; }
  __device__ __forceinline__ bool whole(int vector) const { return index(vector, 0) >= 0 && index(vector, E) <= V; }
  __device__ __forceinline__ bool real(int i) const { return (unsigned)i < (unsigned)V; }
  // what is not of the row counts as -inf
  __device__ __forceinline__ uint4 read(int vector) const {
    if (whole(vector)) return *reinterpret_cast<const uint4*>(z + index(vector, 0));
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = index(vector, e);
      if constexpr (sizeof(T) == 2) {
        const uint32_t h = real(i) ? (uint32_t)reinterpret_cast<const uint16_t*>(z)[i] : 0xff80u;
        w[e / 2] = e & 1 ? w[e / 2] | h << 16 : h;
      } else {
        w[e] = real(i) ? reinterpret_cast<const uint32_t*>(z)[i] : 0xff800000u;
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
__device__ __forceinline__ uint32_t word(const uint4& r, int i) { return i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w; }
template <typename T> __device__ __forceinline__ float element(const uint4& r, int e) {
  if constexpr (sizeof(T) == 2) return __uint_as_float(e & 1 ? word(r, e / 2) & 0xffff0000u : word(r, e / 2) << 16);
  else return __uint_as_float(word(r, e));
}
// the largest of a vector, NaN where one is
template <typename T> __device__ __forceinline__ float largest(const uint4& r) {
  if constexpr (sizeof(T) == 2) {
    auto h = [&](int i) { const uint32_t w = word(r, i); return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h(0), h(1)), __hmax2_nan(h(2), h(3)));
    return max_nan(__low2float(m), __high2float(m));
  } else {
    return max_nan(max_nan(element<T>(r, 0), element<T>(r, 1)), max_nan(element<T>(r, 2), element<T>(r, 3)));
  }
}

// ---- sums -----------------------------------------------------------------------------------------------------------
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

// ---- alternatives ---------------------------------------------------------------------------------------------------
// The order of the values in 32 bits (NaN highest; a zero's sign does not count); with the index below it, unique and never 0.
__device__ __forceinline__ uint32_t order_of(float z) {
  z += 0.0f;
  const uint32_t b = __float_as_uint(z);
  return z != z ? 0xffffffffu : (b & 0x80000000u ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ uint64_t rank_key(float z, int index) { return (uint64_t)order_of(z) << 32 | (uint32_t)~index; }
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return o == 0xffffffffu ? NAN : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// Keys of a warp, one a lane, largest first: the compare-and-exchange steps of a bitonic sort.
__device__ __forceinline__ uint64_t exchange(uint64_t k, int distance, bool larger) {
  const uint64_t other = __shfl_xor_sync(ALL, k, distance);
  return (k > other) == larger ? k : other;
}
__device__ __forceinline__ uint64_t sort_warp(uint64_t k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int d = size / 2; d > 0; d /= 2) k = exchange(k, d, ((lane & d) == 0) == ((lane & size) == 0 || size == 32));
  return k;
}
// the 32 largest of two sorted lists, sorted
__device__ __forceinline__ uint64_t merge_sorted(uint64_t a, uint64_t b) {
  const int lane = threadIdx.x & 31;
  const uint64_t r = __shfl_sync(ALL, b, 31 - lane);
  uint64_t k = a > r ? a : r;
#pragma unroll
  for (int d = 16; d > 0; d /= 2) k = exchange(k, d, (lane & d) == 0);
  return k;
}

struct ScoreParams {
  const void* logits; int64_t row_stride;
  const int64_t* tokens;
  float *logprob, *entropy, *stats;                 // stats: (rows, 2) of m and log s
  float* top_logprob; int64_t* top_tokens;          // (rows, top)
  int64_t rows;
  int32_t V, top;
};

constexpr int U = 8;                  // vectors of a thread: a tile of the row, 32 KB, stays in the CTA's registers
constexpr int CANDIDATES = 512;

struct Tile {
  uint4 r[U];
};

struct Shared {
  uint64_t candidate[CANDIDATES];
  uint32_t count[WARPS];
  int found;
  uint32_t least;                     // upper half of the order of the last key that counts so far
  Stats parts[WARPS];
};

// Candidates of a tile where more than CANDIDATES elements are as large as the bound (masked or constant rows): the tile's k-th
// largest value exactly, by bisection over its elements; all above it, and of its equals the first ones.
template <typename T> __device__ __noinline__ void exact_candidates(const Row<T> row, const Tile tile, int first, int end, int top, Shared& sh) {
  constexpr int SHIFT = sizeof(T) == 2 ? 16 : 0;
  const uint4 (&r)[U] = tile.r;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto total = [&](int n) {
    n = (int)__reduce_add_sync(ALL, (unsigned)n);
    __syncthreads();
    if (lane == 0) sh.count[warp] = (uint32_t)n;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < WARPS; ++w) all += (int)sh.count[w];
    return all;
  };
  auto at_or_above = [&](uint32_t bound) {
    int n = 0;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int v = first + j * THREADS + threadIdx.x;
#pragma unroll
      for (int e = 0; e < Row<T>::E; ++e) n += v < end && row.real(row.index(v, e)) && (order_of(element<T>(r[j], e)) >> SHIFT) >= bound;
    }
    return total(n);
  };
  uint32_t lo = 0, hi = 0xffffffffu >> SHIFT;
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2 + 1;
    if (at_or_above(mid) >= top) lo = mid; else hi = mid - 1;
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.found = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < U; ++j) {
    const int v = first + j * THREADS + threadIdx.x;
#pragma unroll
    for (int e = 0; e < Row<T>::E; ++e) {
      const int i = row.index(v, e);
      const float z = element<T>(r[j], e);
      if (v < end && row.real(i) && (order_of(z) >> SHIFT) > lo) sh.candidate[atomicAdd(&sh.found, 1)] = rank_key(z, i);      // (fewer than top)
    }
  }
  __syncthreads();
  int taken = sh.found;
#pragma unroll
  for (int j = 0; j < U; ++j) {        // the vectors' order is that of the indices: round by round, thread by thread
    if (taken >= top) break;
    const int v = first + j * THREADS + threadIdx.x;
    unsigned equal = 0;
#pragma unroll
    for (int e = 0; e < Row<T>::E; ++e)
      equal |= (v < end && row.real(row.index(v, e)) && (order_of(element<T>(r[j], e)) >> SHIFT) == lo ? 1u : 0u) << e;
    int before = __popc(equal);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(ALL, before, o);
      if (lane >= o) before += n;
    }
    const int all = total(lane == 31 ? before : 0);
    before -= __popc(equal);
    for (int w = 0; w < warp; ++w) before += (int)sh.count[w];
#pragma unroll
    for (int e = 0; e < Row<T>::E; ++e) {
      if (equal >> e & 1) {
        if (taken + before < top) sh.candidate[taken + before] = rank_key(element<T>(r[j], e), row.index(v, e));
        ++before;
      }
    }
    taken += all;
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.found = min(taken, top);
  __syncthreads();
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(THREADS, 3) scores_kernel(const __grid_constant__ ScoreParams p) {
  __shared__ Shared sh;
  constexpr int E = Row<T>::E;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t n = blockIdx.x;
  const Row<T> row(p.logits, n, p.row_stride, p.V);
  Stats a{-INFINITY, 0.0f, 0.0f};
  uint64_t list = 0;                                 // warp 0: the most likely so far, one a lane, sorted
  if (TOP && threadIdx.x == 0) sh.least = 0;

  for (int first = 0; first < row.vectors; first += U * THREADS) {
    const int end = row.vectors;
    Tile tile;
    uint4 (&r)[U] = tile.r;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int v = first + j * THREADS + threadIdx.x;
      r[j] = v < end ? row.read(v) : sizeof(T) == 2 ? make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u)
                                                    : make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
    }
    float most = largest<T>(r[0]);
#pragma unroll
    for (int j = 1; j < U; ++j) most = max_nan(most, largest<T>(r[j]));

    // sums against the largest so far
    const float m = max_nan(a.m, most);
    if (m != a.m && a.m != -INFINITY) {
      const float d = fmaxf(a.m - m, LEAST), c = exponential(d);
      a.t = c * (a.t + a.s * d);
      a.s *= c;
    }
    a.m = m;
    const float origin = m == -INFINITY ? 0.0f : m;
    float s[2] = {0.0f, 0.0f}, t[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (first + j * THREADS + (int)threadIdx.x >= end) break;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = element<T>(r[j], e) - origin, x = exponential(d);
        s[e & 1] += x;
        t[e & 1] = fmaf(x, d, t[e & 1]);
      }
    }
    if (t[0] + t[1] != t[0] + t[1]) {                // 0 * -inf of a masked element (or NaN for good): again, with a floor under d
      t[0] = t[1] = 0.0f;
#pragma unroll
      for (int j = 0; j < U; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float d = at_least(element<T>(r[j], e) - origin);
          t[e & 1] = fmaf(exponential(d), d, t[e & 1]);
        }
    }
    a.s += s[0] + s[1];
    a.t += t[0] + t[1];

    if constexpr (TOP) {
      // A bound that at least `top` elements reach: the largest that the maxima of `top` threads do, or the last key so far.
      const uint32_t mine = order_of(most) >> 16;
      if (threadIdx.x == 0) sh.found = 0;
      __syncthreads();
      uint32_t lo = sh.least, hi = 0xffffu;
      while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (__syncthreads_count(mine >= mid) >= p.top) lo = mid; else hi = mid - 1;
      }
      if (mine >= lo) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const int v = first + j * THREADS + threadIdx.x;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float z = element<T>(r[j], e);
            if (order_of(z) >> 16 >= lo && v < end && row.real(row.index(v, e))) {
              const int at = atomicAdd(&sh.found, 1);
              if (at < CANDIDATES) sh.candidate[at] = rank_key(z, row.index(v, e));
            }
          }
        }
      }
      __syncthreads();
      if (sh.found > CANDIDATES) exact_candidates<T>(row, tile, first, end, p.top, sh);
      if (warp == 0) {
        const int found = sh.found;
        for (int c = 0; c < found; c += 32) list = merge_sorted(list, sort_warp(c + lane < found ? sh.candidate[c + lane] : 0));
        if (lane == p.top - 1) sh.least = (uint32_t)(list >> 48);
      }
      __syncthreads();
    }
  }

#pragma unroll
  for (int o = 16; o > 0; o >>= 1) merge(a, Stats{__shfl_xor_sync(ALL, a.m, o), __shfl_xor_sync(ALL, a.s, o), __shfl_xor_sync(ALL, a.t, o)});
  if (lane == 0) sh.parts[warp] = a;
  __syncthreads();
  if (warp > 0) return;
  a = sh.parts[lane % WARPS];
#pragma unroll
  for (int o = WARPS / 2; o > 0; o >>= 1) merge(a, Stats{__shfl_xor_sync(ALL, a.m, o), __shfl_xor_sync(ALL, a.s, o), __shfl_xor_sync(ALL, a.t, o)});
  const bool empty = a.m == -INFINITY;
  const float ls = empty ? 0.0f : a.m == INFINITY ? NAN : logf(a.s);
  if (lane == 0) {
    const int64_t t = p.tokens[n];
    p.logprob[n] = t >= 0 && t < p.V ? (empty ? -INFINITY : (to_float(row.z[t]) - a.m) - ls) : 0.0f;
    p.entropy[n] = empty ? 0.0f : ls - a.t / a.s;
    p.stats[2 * n] = a.m;
    p.stats[2 * n + 1] = ls;
  }
  if (TOP && lane < p.top) {
    p.top_tokens[n * p.top + lane] = (int)~(uint32_t)list;
    p.top_logprob[n * p.top + lane] = empty ? -INFINITY : (value_of(list) - a.m) - ls;
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

// One read and one write of the row; then the elements that are somebody's token again, with their own gradient.
template <typename T>
__global__ void __launch_bounds__(THREADS) scores_grad_kernel(const __grid_constant__ ScoreGradParams p) {
  constexpr int E = Row<T>::E, AHEAD = 4;
  const int64_t n = blockIdx.x;
  const Row<T> row(p.logits, n, p.row_stride, p.V);
  T* d = (T*)p.d_logits + n * p.d_stride;
  const float m = p.stats[2 * n], ls = p.stats[2 * n + 1], H = p.entropy[n];
  const int64_t t = p.tokens[n];
  const float g = p.g_logprob && t >= 0 && t < p.V ? p.g_logprob[n] : 0.0f, gh = p.g_entropy ? p.g_entropy[n] : 0.0f;
  float total = g;
  if (p.g_top)
    for (int k = 0; k < p.top; ++k) total += p.g_top[n * p.top + k];
  const bool empty = m == -INFINITY;
  auto gradient = [&](float z) {
    const float lp = at_least((z - m) - ls);
    const float e = sizeof(T) == 2 ? exponential(lp) : expf(lp);
    return empty ? 0.0f : -e * fmaf(gh, lp + H, total);
  };
  const bool together = (uintptr_t)d % 16 == (uintptr_t)row.z % 16;       // vectors of z are vectors of d
  for (int v0 = threadIdx.x; v0 < row.vectors; v0 += THREADS * AHEAD) {
    uint4 r[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (v0 + j * THREADS < row.vectors) r[j] = row.read(v0 + j * THREADS);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int v = v0 + j * THREADS;
      if (v >= row.vectors) break;
      float f[E];
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = gradient(element<T>(r[j], e));
      if (together && row.whole(v)) {
        T out[E];
#pragma unroll
        for (int e = 0; e < E; ++e) out[e] = from_float<T>(f[e]);
        *reinterpret_cast<uint4*>(d + row.index(v, 0)) = *reinterpret_cast<const uint4*>(out);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (row.real(row.index(v, e))) d[row.index(v, e)] = from_float<T>(f[e]);
      }
    }
  }
  const int named = 1 + (p.g_top ? p.top : 0);                            // the token itself, and the alternatives
  __syncthreads();
  if ((int)threadIdx.x >= named || empty) return;
  auto token = [&](int k) { return k == 0 ? t : p.top_tokens[n * p.top + k - 1]; };
  const int64_t mine = token(threadIdx.x);
  if (mine < 0 || mine >= p.V) return;
  float own = 0.0f;
  for (int k = 0; k < named; ++k) {
    if (token(k) != mine) continue;
    if (k < (int)threadIdx.x) return;                                     // (an earlier thread writes it)
    own += k == 0 ? g : p.g_top[n * p.top + k - 1];
  }
  d[mine] = from_float<T>(gradient(to_float(row.z[mine])) + own);
}

}  // namespace

int launch_token_scores(int dtype, int64_t rows, int V, int top, const void* logits, int64_t row_stride, const int64_t* tokens, float* logprob,
                        float* entropy, float* stats, float* top_logprob, int64_t* top_tokens, cudaStream_t stream) {
  const ScoreParams p{logits, row_stride, tokens, logprob, entropy, stats, top_logprob, top_tokens, rows, V, top};
  const dim3 grid((unsigned)rows);
  const cudaError_t e = dtype == FPB_BF16 ? (top ? launch_kernel(scores_kernel<__nv_bfloat16, true>, grid, THREADS, 0, false, p, stream)
                                                 : launch_kernel(scores_kernel<__nv_bfloat16, false>, grid, THREADS, 0, false, p, stream))
                                          : (top ? launch_kernel(scores_kernel<float, true>, grid, THREADS, 0, false, p, stream)
                                                 : launch_kernel(scores_kernel<float, false>, grid, THREADS, 0, false, p, stream));
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
