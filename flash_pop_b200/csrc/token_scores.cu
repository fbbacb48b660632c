// Log probabilities of given tokens under rows of logits, with the rows' entropies and most likely alternatives, and the
// gradient of all three.  With m = max z, s = sum exp(z - m):
//   log p_j = (z_j - m) - log s,   H = log s - sum exp(z - m) (z - m) / s
//   dz_j = -p_j (G + g_H (log p_j + H)) + [j = token] g + sum over alternatives a of [j = a] g_a,   G = g + sum of g_a
// The order of the alternatives is that of the logits, equal ones by index, NaN (which makes every number of the row NaN) first.
// A row of -inf only has no distribution: log p = -inf, H = 0, no gradient.
// Bound by HBM: one read forward, one read and one write backward.
#include <cooperative_groups.h>

#include "fpb_common.cuh"
#include "vec_io.cuh"

namespace fpb {
namespace {

constexpr float LEAST = -1e4f;
constexpr unsigned ALL = 0xffffffffu;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// differences below LEAST count as that: their exponential is 0 as well, and no product of theirs overflows (NaN stays)
__device__ __forceinline__ float at_least(float a) { return max_nan(a, LEAST); }
// 2^x; results below the smallest normal number are 0
__device__ __forceinline__ float exp2_of(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float LOG2E = 1.44269504088896f, LN2 = 0.693147180559945f;

// Two floats to an instruction: the row's arithmetic is issue-bound beside the memory it reads.
struct Pair {
  uint64_t v;
};
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 both(Pair a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// ---- a row as vectors -----------------------------------------------------------------------------------------------
// A row starts at any element; it is read as the 16-byte vectors that it lies in, the first and the last element by element.
template <int N> struct Vectors {
  uint4 r[N];
};
template <typename T> struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* z;
  int V, skew, vectors;             // element i is number (i + skew) % E of vector (i + skew) / E
  int inner, inner_end;             // vectors that lie in the row as a whole

  __device__ Row(const void* logits, int64_t row, int64_t stride, int n) : z((const T*)logits + row * stride), V(n) {
    skew = (int)(((uintptr_t)z % 16) / sizeof(T));
    vectors = (skew + V + E - 1) / E;
    inner = skew ? 1 : 0;
    inner_end = (skew + V) / E;
  }
  __device__ __forceinline__ int index(int vector, int e) const { return vector * E + e - skew; }
  __device__ __forceinline__ bool whole(int vector) const { return vector >= inner && vector < inner_end; }
  __device__ __forceinline__ bool real(int i) const { return (unsigned)i < (unsigned)V; }
  __device__ __forceinline__ const uint4* base() const { return reinterpret_cast<const uint4*>(z - skew); }
  // what of a vector is not of the row counts as -inf
  __device__ __forceinline__ uint4 read(int vector) const { return whole(vector) ? base()[vector] : read_part(z, V, index(vector, 0)); }
  static __device__ __noinline__ uint4 read_part(const T* z, int V, int first) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = first + e;
      const bool real = (unsigned)i < (unsigned)V;
      if constexpr (sizeof(T) == 2) w[e / 2] |= (real ? (uint32_t)reinterpret_cast<const uint16_t*>(z)[i] : 0xff80u) << (e & 1 ? 16 : 0);
      else w[e] = real ? reinterpret_cast<const uint32_t*>(z)[i] : 0xff800000u;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // a thread's vectors first, first + NT, ...; those from `end` on are filled with a value that no sum feels
  template <int NT, int N> __device__ __forceinline__ void read(Vectors<N>& to, int tile, int end) const {
    const int first = tile + threadIdx.x;
    if (tile >= inner && tile + N * NT <= min(end, inner_end)) {
#pragma unroll
      for (int j = 0; j < N; ++j) to.r[j] = base()[first + j * NT];
    } else {
      const uint32_t w = sizeof(T) == 2 ? 0xf149f149u : 0xf149f2cau;          // -1e30
#pragma unroll
      for (int j = 0; j < N; ++j) to.r[j] = first + j * NT < end ? read(first + j * NT) : make_uint4(w, w, w, w);
    }
  }
};
__device__ __forceinline__ uint32_t word(const uint4& r, int i) { return i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w; }
template <typename T> __device__ __forceinline__ float element(const uint4& r, int e) {
  if constexpr (sizeof(T) == 2) return __uint_as_float(e & 1 ? word(r, e / 2) & 0xffff0000u : word(r, e / 2) << 16);
  else return __uint_as_float(word(r, e));
}
template <typename T> __device__ __forceinline__ Pair elements(const uint4& r, int i) { return pair(element<T>(r, 2 * i), element<T>(r, 2 * i + 1)); }
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
// In powers of two: with L = log2 e and c = m L rounded, x = 2^(z L - c) is one rounding of the exponent (a fused product) and one
// exponential; that c is not m L exactly shifts all exponents alike and is put right once, in the logarithm of the sum.  Where
// c could overflow, and where a mask has filled what is left with huge negative numbers, x = 2^((z - m) L).
constexpr float LARGEST = 2e38f, SMALLEST = -1e29f;
__device__ __forceinline__ bool ordinary(float m) { return m > SMALLEST && m < LARGEST; }
__device__ __forceinline__ float origin(float m) { return __fmul_rn(m, LOG2E); }        // c (never fused into what follows)
__device__ __forceinline__ float exponent(float z, float m) { return ordinary(m) ? fmaf(z, LOG2E, -origin(m)) : (z - m) * LOG2E; }

// running (max, sum of x, sum of x times its exponent); nothing yet, or only -inf: max = -inf, sums 0
struct Stats {
  float m, s, t;
};
// the same sums against another maximum, at least as large
__device__ __forceinline__ void move_to(Stats& a, float m) {
  const float d = ordinary(m) && ordinary(a.m) ? __fsub_rn(origin(a.m), origin(m)) : (a.m - (m == -INFINITY ? 0.0f : m)) * LOG2E;
  const float y = at_least(d), c = exp2_of(y);
  a.t = c * fmaf(a.s, y, a.t);
  a.s *= c;
  a.m = m;
}
// over groups of `lanes` lanes
template <int LANES> __device__ __forceinline__ void join(Stats& a) {
  float m = a.m;
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(ALL, m, o));
  move_to(a, m);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(ALL, a.s, o);
    a.t += __shfl_xor_sync(ALL, a.t, o);
  }
}
__device__ __forceinline__ float log_sum(const Stats& a) {       // log of the sum of exp(z - m)
  if (a.m == -INFINITY) return 0.0f;
  if (a.m == INFINITY) return NAN;
  return logf(a.s) - (ordinary(a.m) ? LN2 * fmaf(a.m, LOG2E, -origin(a.m)) : 0.0f);
}
__device__ __forceinline__ float entropy_of(const Stats& a) {
  return a.m == -INFINITY ? 0.0f : a.m == INFINITY ? NAN : logf(a.s) - LN2 * (a.t / a.s);
}

// The sums of `count` vectors where the ordinary way meets 0 * -inf (masked elements) or does not apply.
template <typename T, int N> __device__ __noinline__ float2 careful_sums(const Vectors<N> from, int count, float m) {
  float s = 0.0f, t = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (j >= count) break;
#pragma unroll
    for (int e = 0; e < Row<T>::E; ++e) {
      const float y = at_least(exponent(element<T>(from.r[j], e), m)), x = exp2_of(y);
      s += x;
      t = fmaf(x, y, t);
    }
  }
  return make_float2(s, t);
}

// N vectors of a thread, of which the first `count` are of the row and the first `slots` are of some thread's; most: their largest
template <typename T, int N> __device__ __forceinline__ void add(Stats& a, const Vectors<N>& from, int count, int slots, float most) {
  const float m = max_nan(a.m, most);
  if (m == -INFINITY) return;
  if (m != a.m) move_to(a, m);
  const float c = -origin(m);
  const Pair minus = pair(c, c), log2e = pair(LOG2E, LOG2E);
  Pair s = pair(0.0f, 0.0f), t = s;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (j >= slots) break;
#pragma unroll
    for (int i = 0; i < Row<T>::E / 2; ++i) {
      const Pair y = fma(elements<T>(from.r[j], i), log2e, minus);
      const float2 f = both(y);
      const Pair x = pair(exp2_of(f.x), exp2_of(f.y));
      s = s + x;
      t = fma(x, y, t);
    }
  }
  const float2 ss = both(s), tt = both(t);
  float2 sums = make_float2(ss.x + ss.y, tt.x + tt.y);
  if (!ordinary(m) || sums.y != sums.y) sums = careful_sums<T, N>(from, count, m);
  a.s += sums.x;
  a.t += sums.y;
}

// ---- alternatives ---------------------------------------------------------------------------------------------------
// The order of the values in 32 bits (NaN highest; a zero's sign does not count); with the index below it, unique and never 0.
__device__ __forceinline__ uint32_t order_of(float z) {
  z += 0.0f;
  const uint32_t b = __float_as_uint(z);
  return z != z ? 0xffffffffu : (b & 0x80000000u ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) { return o == 0xffffffffu ? NAN : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ uint64_t rank_key(float z, int index) { return (uint64_t)order_of(z) << 32 | (uint32_t)~index; }

// Values of a warp, one a lane, largest first: the compare-and-exchange steps of a bitonic sort.
__device__ __forceinline__ uint32_t exchange(uint32_t k, int distance, bool larger) {
  const uint32_t other = __shfl_xor_sync(ALL, k, distance);
  return larger ? max(k, other) : min(k, other);
}
__device__ __forceinline__ uint32_t sort_warp(uint32_t k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int d = size / 2; d > 0; d /= 2) k = exchange(k, d, ((lane & d) == 0) == ((lane & size) == 0 || size == 32));
  return k;
}
// the 32 largest of two sorted warps of values, sorted
__device__ __forceinline__ uint32_t merge_sorted(uint32_t a, uint32_t b) {
  const int lane = threadIdx.x & 31;
  uint32_t k = max(a, __shfl_sync(ALL, b, 31 - lane));
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
  int32_t V, top, split;                            // CTAs (of a cluster) that share a row
};

constexpr int U = 8;                  // vectors of a thread: a tile of the row stays in the CTA's registers
constexpr int CANDIDATES = 512, MAX_SPLIT = 8, FEW = 20;

typedef Vectors<U> Tile;
template <int WARPS> struct Shared {
  alignas(16) uint64_t candidate[CANDIDATES];       // (both are read two at a time)
  alignas(16) uint64_t best[MAX_SPLIT * 32];        // the alternatives of a row's CTAs, in the first one
  uint32_t group[2][64];              // the largest of each part of a tile, tiles in turn
  int found;
  uint32_t count[WARPS];
  Stats parts[WARPS];
  Stats shares[MAX_SPLIT];            // sums of a row's CTAs, in the first one
};

// For each of n keys (unique but for 0, which stands for none) that is among the `top` largest: to(key, how many are larger).
template <int NT, typename F> __device__ __forceinline__ void rank_keys(const uint64_t* keys, int n, int top, F to) {
  for (int i = threadIdx.x; i < n; i += NT) {
    const uint64_t key = keys[i];
    int larger = n & 1 && keys[n - 1] > key;
#pragma unroll 4
    for (int k = 0; k + 1 < n; k += 2) {
      const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(keys + k);
      larger += (two.x > key) + (two.y > key);
    }
    if (larger < top && key) to(key, larger);
  }
}

// Candidates of a tile where more elements than there is room for reach the bound (masked or constant rows): the tile's k-th
// largest value exactly, by bisection over its elements; all above it, and of its equals the first ones.  They go behind the
// `kept` candidates of earlier tiles.
template <typename T, int NT> __device__ __noinline__ void exact_candidates(const Row<T> row, const Tile tile, int first, int end, int top, int kept,
                                                                            Shared<NT / 32>& sh) {
  constexpr int SHIFT = sizeof(T) == 2 ? 16 : 0, WARPS = NT / 32;
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
  auto order = [&](int j, int e) { return order_of(element<T>(r[j], e)) >> SHIFT; };
  auto here = [&](int j, int e) {
    const int v = first + j * NT + threadIdx.x;
    return v < end && row.real(row.index(v, e));
  };
  auto at_or_above = [&](uint32_t bound) {
    int n = 0;
#pragma unroll
    for (int j = 0; j < U; ++j)
#pragma unroll
      for (int e = 0; e < Row<T>::E; ++e) n += here(j, e) && order(j, e) >= bound;
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
  uint64_t* to = sh.candidate + kept;
#pragma unroll
  for (int j = 0; j < U; ++j)
#pragma unroll
    for (int e = 0; e < Row<T>::E; ++e)
      if (here(j, e) && order(j, e) > lo) to[atomicAdd(&sh.found, 1)] = rank_key(element<T>(r[j], e), row.index(first + j * NT + threadIdx.x, e));      // (fewer than top)
  __syncthreads();
  int taken = sh.found;
#pragma unroll
  for (int j = 0; j < U; ++j) {        // the vectors' order is that of the indices: round by round, thread by thread
    if (taken >= top) break;
    unsigned equal = 0;
#pragma unroll
    for (int e = 0; e < Row<T>::E; ++e) equal |= (here(j, e) && order(j, e) == lo ? 1u : 0u) << e;
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
        if (taken + before < top) to[taken + before] = rank_key(element<T>(r[j], e), row.index(first + j * NT + threadIdx.x, e));
        ++before;
      }
    }
    taken += all;
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.found = kept + min(taken, top);
  __syncthreads();
}

template <typename T, int NT, bool TOP>
__global__ void __launch_bounds__(NT, 1024 / NT) scores_kernel(const __grid_constant__ ScoreParams p) {
  constexpr int E = Row<T>::E, WARPS = NT / 32;
  __shared__ Shared<WARPS> sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int share = blockIdx.x % p.split;
  const int64_t n = blockIdx.x / p.split;
  const Row<T> row(p.logits, n, p.row_stride, p.V);
  const int each = (row.vectors + p.split - 1) / p.split, begin = share * each, end = min(begin + each, row.vectors);
  Stats a{-INFINITY, 0.0f, 0.0f};
  int kept = 0;                                      // candidates of the tiles so far
  if (p.split > 1) cooperative_groups::this_cluster().barrier_arrive();

  if constexpr (!TOP) {
    // the next vectors are on their way while these are added
    constexpr int N = U / 2;
    Vectors<N> now, next;
    row.template read<NT>(now, begin, end);
    for (int first = begin; first < end; first += N * NT) {
      row.template read<NT>(next, first + N * NT, end);
      const int count = (end - first - (int)threadIdx.x + NT - 1) / NT;
      float most = -INFINITY;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < count) most = max_nan(most, largest<T>(now.r[j]));
      add<T, N>(a, now, count, (end - first + NT - 1) / NT, most);
      now = next;
    }
  } else {
    if (threadIdx.x == 0) sh.found = 0;
    uint32_t least = 0;                              // order that at least `top` elements of the row so far reach
    int parity = 0;
    for (int first = begin; first < end; first += U * NT, parity ^= 1) {
      Tile tile;
      uint4 (&r)[U] = tile.r;
      row.template read<NT>(tile, first, end);
      const int count = (end - first - (int)threadIdx.x + NT - 1) / NT;
      float half[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < U; ++j)
        if (j < count) half[j * 2 / U] = max_nan(half[j * 2 / U], largest<T>(r[j]));
      const float most = max_nan(half[0], half[1]);

      // `top` of the 32 parts of the tile reach their top-th largest maximum: so many elements do, and of any order of the
      // elements not many more are to be expected, 32 ln(32 / (32 - top)).  For more than FEW alternatives 64 parts.
      const bool few = p.top <= FEW;
      uint32_t g[2] = {order_of(few ? most : half[0]), order_of(half[1])};
#pragma unroll
      for (int o = 1; o < WARPS; o *= 2) g[0] = max(g[0], __shfl_xor_sync(ALL, g[0], o));
      if (!few) {
#pragma unroll
        for (int o = 1; o < WARPS; o *= 2) g[1] = max(g[1], __shfl_xor_sync(ALL, g[1], o));
      }
      if (lane % WARPS == 0) {
        sh.group[parity][threadIdx.x / WARPS] = g[0];
        if (!few) sh.group[parity][32 + threadIdx.x / WARPS] = g[1];
      }
      add<T, U>(a, tile, count, (end - first + NT - 1) / NT, most);
      __syncthreads();
      uint32_t sorted = sort_warp(sh.group[parity][lane]);
      if (!few) sorted = merge_sorted(sorted, sort_warp(sh.group[parity][32 + lane]));
      least = max(least, __shfl_sync(ALL, sorted, p.top - 1));
      const float bound = value_of(least);
      if (!(most < bound)) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
          if (largest<T>(r[j]) < bound) continue;
          const int v = first + j * NT + threadIdx.x;
          unsigned reach = 0;
#pragma unroll
          for (int e = 0; e < E; ++e) reach |= !(element<T>(r[j], e) < bound) && v < end && row.real(row.index(v, e)) ? 1u << e : 0u;
          for (; reach; reach &= reach - 1) {
            const int e = __ffs(reach) - 1, at = atomicAdd(&sh.found, 1);
            const uint32_t w = word(r[j], sizeof(T) == 2 ? e / 2 : e);
            const float z = __uint_as_float(sizeof(T) == 2 ? (e & 1 ? w & 0xffff0000u : w << 16) : w);
            if (at < CANDIDATES) sh.candidate[at] = rank_key(z, row.index(v, e));
          }
        }
      }
      __syncthreads();
      if (sh.found > CANDIDATES) {
        // no room: the `top` best that earlier tiles left, and this tile's
        __syncthreads();
        rank_keys<NT>(sh.candidate, kept, p.top, [&](uint64_t key, int larger) { sh.best[larger] = key; });
        __syncthreads();
        kept = min(kept, p.top);
        if ((int)threadIdx.x < kept) sh.candidate[threadIdx.x] = sh.best[threadIdx.x];
        exact_candidates<T, NT>(row, tile, first, end, p.top, kept, sh);
      }
      kept = sh.found;
    }
    __syncthreads();
  }

  join<32>(a);
  if constexpr (WARPS > 1) {
    if (lane == 0) sh.parts[warp] = a;
    __syncthreads();
    a = sh.parts[lane % WARPS];
    join<WARPS>(a);
  }
  if (p.split > 1) {
    // the shares of a row meet in the first CTA of the cluster
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    cluster.barrier_wait();                          // (the first CTA has started)
    Shared<WARPS>* to = cluster.map_shared_rank(&sh, 0);
    if (threadIdx.x == 0) to->shares[share] = a;
    if constexpr (TOP) {
      if ((int)threadIdx.x >= kept && (int)threadIdx.x < p.top) to->best[share * p.top + threadIdx.x] = 0;      // (fewer found)
      rank_keys<NT>(sh.candidate, kept, p.top, [&](uint64_t key, int larger) { to->best[share * p.top + larger] = key; });
    }
    cluster.sync();
    if (share > 0) return;
    a = lane < p.split ? sh.shares[lane] : Stats{-INFINITY, 0.0f, 0.0f};
    join<32>(a);
  }
  const bool empty = a.m == -INFINITY;
  const float ls = log_sum(a);
  if (threadIdx.x == 0) {
    const int64_t t = p.tokens[n];
    p.logprob[n] = t >= 0 && t < p.V ? (empty ? -INFINITY : (to_float(row.z[t]) - a.m) - ls) : 0.0f;
    p.entropy[n] = entropy_of(a);
    p.stats[2 * n] = a.m;
    p.stats[2 * n + 1] = ls;
  }
  if constexpr (TOP) {
    const bool shared = p.split > 1;
    rank_keys<NT>(shared ? sh.best : sh.candidate, shared ? p.split * p.top : kept, p.top, [&](uint64_t key, int place) {
      p.top_tokens[n * p.top + place] = (int)~(uint32_t)key;
      p.top_logprob[n * p.top + place] = empty ? -INFINITY : (value_of((uint32_t)(key >> 32)) - a.m) - ls;
    });
  }
}

template <typename T, int NT> cudaError_t scores(const ScoreParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.rows * p.split)); cfg.blockDim = dim3(NT); cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)p.split; attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr; cfg.numAttrs = p.split > 1 ? 1 : 0;
  return p.top ? cudaLaunchKernelEx(&cfg, scores_kernel<T, NT, true>, p) : cudaLaunchKernelEx(&cfg, scores_kernel<T, NT, false>, p);
}

template <typename T> cudaError_t scores(ScoreParams p, cudaStream_t stream) {
  // Threads for a row: as few as hold it in one tile, so that short rows leave no thread without work; 256 at most.
  const int64_t vectors = ((int64_t)p.V + 16 / sizeof(T) - 1) / (16 / sizeof(T)) + 1;
  p.split = 1;
  if (vectors <= 32 * U) return scores<T, 32>(p, stream);
  if (vectors <= 64 * U) return scores<T, 64>(p, stream);
  if (vectors <= 128 * U) return scores<T, 128>(p, stream);
  // Few rows: a row over a cluster of CTAs, a vector a thread at least, up to four CTAs an SM.
  while (p.split < MAX_SPLIT && p.rows * p.split * 2 <= 592 && vectors >= 256 * 2 * p.split) p.split *= 2;
  return scores<T, 256>(p, stream);
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
template <typename T, int NT>
__global__ void __launch_bounds__(NT) scores_grad_kernel(const __grid_constant__ ScoreGradParams p) {
  constexpr int E = Row<T>::E, AHEAD = 4;
  const int64_t n = blockIdx.x;
  const Row<T> row(p.logits, n, p.row_stride, p.V);
  const int each = (row.vectors + gridDim.y - 1) / gridDim.y, begin = blockIdx.y * each, end = min(begin + each, row.vectors);
  T* d = (T*)p.d_logits + n * p.d_stride;
  const float m = p.stats[2 * n], ls = p.stats[2 * n + 1], H = p.entropy[n];
  const int64_t t = p.tokens[n];
  const float g = p.g_logprob && t >= 0 && t < p.V ? p.g_logprob[n] : 0.0f, gh = p.g_entropy ? p.g_entropy[n] : 0.0f;
  const int lane = threadIdx.x & 31;
  float total = p.g_top && lane < p.top ? p.g_top[n * p.top + lane] : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(ALL, total, o);
  total += g;
  const bool empty = m == -INFINITY;
  const Pair minus_m = pair(-m, -m), minus_ls = pair(-ls, -ls), log2e = pair(LOG2E, LOG2E), gh2 = pair(-gh, -gh);
  const float offset = fmaf(gh, H, total);
  const Pair offset2 = pair(-offset, -offset);
  // -p (total + gh (log p + H)) of two elements
  auto gradient = [&](Pair z) {
    const float2 raw = both((z + minus_m) + minus_ls);
    const Pair lp = pair(at_least(raw.x), at_least(raw.y));
    const float2 y = both(lp * log2e);
    const Pair e = sizeof(T) == 2 ? pair(exp2_of(y.x), exp2_of(y.y)) : pair(expf(at_least(raw.x)), expf(at_least(raw.y)));
    return both(e * fma(gh2, lp, offset2));
  };
  const bool together = (uintptr_t)d % 16 == (uintptr_t)row.z % 16;       // vectors of z are vectors of d
  for (int v0 = begin + threadIdx.x; v0 < end; v0 += NT * AHEAD) {
    uint4 r[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (v0 + j * NT < end) r[j] = row.read(v0 + j * NT);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int v = v0 + j * NT;
      if (v >= end) break;
      float f[E];
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        const float2 x = gradient(elements<T>(r[j], i));
        f[2 * i] = empty ? 0.0f : x.x;
        f[2 * i + 1] = empty ? 0.0f : x.y;
      }
      if (together && row.whole(v)) {
        if constexpr (E == 8) store8(d + row.index(v, 0), f);
        else *reinterpret_cast<float4*>(d + row.index(v, 0)) = make_float4(f[0], f[1], f[2], f[3]);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (row.real(row.index(v, e))) d[row.index(v, e)] = from_float<T>(f[e]);
      }
    }
  }
  const int named = 1 + (p.g_top ? p.top : 0);                            // the token itself, and the alternatives
  __syncthreads();
  if (empty) return;
  auto token = [&](int k) { return k == 0 ? t : p.top_tokens[n * p.top + k - 1]; };
  for (int w = threadIdx.x; w < named; w += NT) {
    const int64_t mine = token(w);
    if (mine < 0 || mine >= p.V) continue;
    const int v = (int)(mine + row.skew) / E;
    if (v < begin || v >= end) continue;
    float own = 0.0f;
    bool first = true;
    for (int k = 0; k < named; ++k) {
      if (token(k) != mine) continue;
      if (k < w) { first = false; break; }                                // (written with that one)
      own += k == 0 ? g : p.g_top[n * p.top + k - 1];
    }
    const float z = to_float(row.z[mine]);
    if (first) d[mine] = from_float<T>(gradient(pair(z, z)).x + own);
  }
}

template <typename T, int NT> cudaError_t scores_grad(const ScoreGradParams& p, int split, cudaStream_t stream) {
  return launch_kernel(scores_grad_kernel<T, NT>, dim3((unsigned)p.rows, split), NT, 0, false, p, stream);
}
template <typename T> cudaError_t scores_grad(const ScoreGradParams& p, cudaStream_t stream) {
  const int64_t vectors = ((int64_t)p.V + 16 / sizeof(T) - 1) / (16 / sizeof(T)) + 1;
  if (vectors <= 32 * 8) return scores_grad<T, 32>(p, 1, stream);
  if (vectors <= 64 * 8) return scores_grad<T, 64>(p, 1, stream);
  if (vectors <= 128 * 8) return scores_grad<T, 128>(p, 1, stream);
  int split = 1;                                                          // few rows: shares of a row
  while (split < 64 && p.rows * split * 2 <= 1184 && vectors >= 256 * 2 * split) split *= 2;
  return scores_grad<T, 256>(p, split, stream);
}

}  // namespace

int launch_token_scores(int dtype, int64_t rows, int V, int top, const void* logits, int64_t row_stride, const int64_t* tokens, float* logprob,
                        float* entropy, float* stats, float* top_logprob, int64_t* top_tokens, cudaStream_t stream) {
  const ScoreParams p{logits, row_stride, tokens, logprob, entropy, stats, top_logprob, top_tokens, rows, V, top, 1};
  const cudaError_t e = dtype == FPB_BF16 ? scores<__nv_bfloat16>(p, stream) : scores<float>(p, stream);
  return e == cudaSuccess ? FPB_OK : FPB_ERR_LAUNCH;
}

int launch_token_scores_grad(int dtype, int64_t rows, int V, int top, const void* logits, int64_t row_stride, const int64_t* tokens,
                             const float* entropy, const float* stats, const int64_t* top_tokens, const float* g_logprob,
                             const float* g_entropy, const float* g_top, void* d_logits, int64_t d_stride, cudaStream_t stream) {
  const ScoreGradParams p{logits, row_stride, tokens, entropy, stats, top_tokens, g_logprob, g_entropy, g_top, d_logits, d_stride, rows, V, top};
  const cudaError_t e = dtype == FPB_BF16 ? scores_grad<__nv_bfloat16>(p, stream) : scores_grad<float>(p, stream);
  return e == cudaSuccess ? FPB_OK : FPB_ERR_LAUNCH;
}

}  // namespace fpb
