// Log probabilities of given tokens under rows of logits, with the rows' entropies and most likely alternatives, and the
// gradient of all three.  With m = max z, s = sum exp(z - m):
//   log p_j = (z_j - m) - log s,   H = log s - sum exp(z - m) (z - m) / s
//   dz_j = -p_j (G + g_H (log p_j + H)) + [j = token] g + sum over alternatives a of [j = a] g_a,   G = g + sum of g_a
// The order of the alternatives is that of the logits, equal ones by index, NaN (which makes every number of the row NaN) first.
// A row of -inf only has no distribution: log p = -inf, H = 0, no gradient.
// Bound by HBM: one read forward, one read and one write backward.
#include <cooperative_groups.h>

#include <type_traits>

#include "fpb_common.cuh"
#include "vec_io.cuh"

namespace fpb {
namespace {

// (the row's arithmetic is issue-bound beside the memory it reads: pairs of floats, vec_io.cuh)
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

// ---- a row as vectors -----------------------------------------------------------------------------------------------
// A row starts at any element: it is so many single elements up to a 16-byte boundary, whole vectors, and a rest.
template <int N> struct Vectors {
  uint4 r[N];
};
template <typename T> struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* z;
  int V, head, vectors;

  __device__ Row(const void* logits, int64_t row, int64_t stride, int n) : z((const T*)logits + row * stride), V(n) {
    const int skew = (int)(((uintptr_t)z % 16) / sizeof(T));
    head = min(skew ? E - skew : 0, V);
    vectors = (V - head) / E;
  }
  __device__ __forceinline__ int index(int vector, int e) const { return head + vector * E + e; }
  __device__ __forceinline__ const uint4* base() const { return reinterpret_cast<const uint4*>(z + head); }
  // the elements outside the vectors, fewer than 2 E
  __device__ __forceinline__ int edges() const { return V - vectors * E; }
  __device__ __forceinline__ int edge(int i) const { return i < head ? i : i + vectors * E; }
  // a thread's vectors tile + its number, and every NT-th after it; those from `end` on are filled with a value that no sum feels
  template <int NT, int N> __device__ __forceinline__ void read(Vectors<N>& to, int tile, int end) const {
    const uint4* from = base() + tile + threadIdx.x;
    if (NT == 32 && tile >= end) return;             // (never looked at; for longer rows the check costs more than it saves)
    if (tile + N * NT <= end) {
#pragma unroll
      for (int j = 0; j < N; ++j) to.r[j] = from[j * NT];
    } else {
      const uint32_t w = sizeof(T) == 2 ? 0xf149f149u : 0xf149f2cau;          // FILL and a little
#pragma unroll
      for (int j = 0; j < N; ++j) to.r[j] = tile + (int)threadIdx.x + j * NT < end ? from[j * NT] : make_uint4(w, w, w, w);
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
// exponential; that c is not m L exactly shifts all exponents alike and is put right once, in the logarithm of the sum.  The shift is half a
// unit in c's last place at most: 2^-4 below |m| = 2^20, but 2^7 and more from |m| = 2^31 on, where 2^shift is 0 or infinite.  So larger
// maxima (masks of finite numbers among them), and m = -inf, take x = 2^((z - m) L), a rounding more, without a shift.
constexpr float ORDINARY = 1048576.0f;
__device__ __forceinline__ bool ordinary(float m) { return fabsf(m) < ORDINARY; }
__device__ __forceinline__ float origin(float m) { return __fmul_rn(m, LOG2E); }        // c (never fused into what follows)
__device__ __forceinline__ float exponent(float z, float m) { return ordinary(m) ? fmaf(z, LOG2E, -origin(m)) : (z - m) * LOG2E; }
// Alternatives' bounds below SMALLEST are those of a masked row; FILL stands for the elements behind a row, which no sum feels.
constexpr float SMALLEST = -1e29f, FILL = -9e29f;

// running (max, sum of x, sum of x times its exponent); nothing yet, or only -inf: max = -inf, sums 0
struct Stats {
  float m, s, t;
};
// the same sums against another maximum, at least as large; either may have a shift, which goes with its exponents
__device__ __forceinline__ void move_to(Stats& a, float m) {
  const float base = m == -INFINITY ? 0.0f : m;
  const float d = ordinary(a.m) ? (ordinary(m) ? __fsub_rn(origin(a.m), origin(m)) : -fmaf(m, LOG2E, -origin(a.m)))
                                : (ordinary(m) ? fmaf(a.m, LOG2E, -origin(m)) : (a.m - base) * LOG2E);
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
// log of the sum of exp(z - m), and the entropy
__device__ __forceinline__ float2 results(const Stats& a) {
  if (a.m == -INFINITY) return make_float2(0.0f, 0.0f);
  if (a.m == INFINITY) return make_float2(NAN, NAN);
  const float log_s = logf(a.s);
  return make_float2(log_s - (ordinary(a.m) ? LN2 * fmaf(a.m, LOG2E, -origin(a.m)) : 0.0f), log_s - LN2 * __fdividef(a.t, a.s));
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

// The largest of a thread's vectors, of which the first `count` are of the row.
template <typename T, bool FULL, int N> __device__ __forceinline__ float largest_of(const Vectors<N>& from, int count) {
  float most;
  if constexpr (sizeof(T) == 2) {
    auto h = [&](int j, int i) { const uint32_t w = word(from.r[j], i); return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    __nv_bfloat162 m = h(0, 0);
#pragma unroll
    for (int i = 1; i < 4 * N; ++i) m = __hmax2_nan(m, h(i / 4, i % 4));
    most = max_nan(__low2float(m), __high2float(m));
  } else {
    most = largest<T>(from.r[0]);
#pragma unroll
    for (int j = 1; j < N; ++j) most = max_nan(most, largest<T>(from.r[j]));
  }
  if (!FULL && count < N && !(most > FILL)) {        // (what stands for those behind the row is more than a mask's value)
    most = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < count) most = max_nan(most, largest<T>(from.r[j]));
  }
  return most;
}

// N vectors of a thread, of which the first `count` are of the row and the first `slots` are of some thread's; most: their largest
template <typename T, bool FULL, int N> __device__ __forceinline__ void add(Stats& a, const Vectors<N>& from, int count, int slots, float most) {
  const float m = max_nan(a.m, most);
  if (m == -INFINITY) return;
  if (m != a.m) move_to(a, m);
  const float c = -origin(m);
  const Pair minus = pair(c, c), log2e = pair(LOG2E, LOG2E);
  Pair s = pair(0.0f, 0.0f), t = s;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (!FULL && j >= slots) break;
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

constexpr int N = 4;                  // vectors of a thread in flight at a time, a tile
constexpr int RECORDS = 512, CANDIDATES = 256, MAX_EDGES = 14, MAX_SPLIT = 8;
// Up to FEW alternatives the bound comes from 32 parts of the row, for more from 64: the top-th largest of n parts' maxima lets about n ln(n / (n - top))
// elements of a tile through, 22 and 34 at 16 and 21 alternatives of 32 parts, 18 and 25 of 64, whose order costs a second sort.  With 32 and 64 parts:
// 16384 rows of 32000 bf16 logits, 17, 20, 24 and 28 alternatives 254 and 251, 272 and 262, 295 and 278, 348 and 290 us.
constexpr int FEW = 16;

template <int WARPS> struct Sums {
  Stats parts[WARPS];
  Stats shares[MAX_SPLIT];            // of a row's CTAs, in the first one
};
template <int WARPS> struct Shared {
  static constexpr int LISTS = WARPS == 8 ? MAX_SPLIT : 1;      // (shorter rows are not shared)
  alignas(16) uint64_t candidate[CANDIDATES + MAX_EDGES];       // (both are read two at a time)
  alignas(16) uint64_t best[LISTS * 32];                        // the alternatives of a row's CTAs, in the first one
  uint2 record[RECORDS];              // order of the largest of a thread's N vectors, the first of them
  uint32_t group[2][64];              // the largest of each part of a tile, tiles in turn
  int records, found;
  uint32_t count[WARPS];
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

// The maxima of the parts that the tiles seen are cut into, 32 or, where more than FEW alternatives are wanted and there are more threads, 64;
// one or two a lane of every warp.  A part is the same threads' share of every tile.
struct Parts {
  uint32_t a = 0, b = 0;
};
// `most`: a thread's maximum of this tile.  One barrier, but with a single warp.
template <int NT> __device__ __forceinline__ void add_maxima(Parts& parts, float most, bool few, uint32_t (&group)[64]) {
  const int lane = threadIdx.x & 31;
  uint32_t g = order_of(most);
  if (NT == 32) { parts.a = max(parts.a, g); return; }
#pragma unroll
  for (int o = 1; o < NT / 64; o *= 2) g = max(g, __shfl_xor_sync(ALL, g, o));
  if (few) {
    g = max(g, __shfl_xor_sync(ALL, g, NT / 64));
    if (lane % (NT / 32) == 0) group[threadIdx.x / (NT / 32)] = g;
  } else if (lane % (NT / 64 ? NT / 64 : 1) == 0) {
    group[threadIdx.x / (NT / 64 ? NT / 64 : 1)] = g;
  }
  __syncthreads();
  parts.a = max(parts.a, group[lane]);
  if (!few) parts.b = max(parts.b, group[32 + lane]);
}
// the top-th largest of them
template <int NT> __device__ __forceinline__ uint32_t kth(const Parts& parts, int top) {
  if (top == 1) return __reduce_max_sync(ALL, parts.a);
  uint32_t sorted = sort_warp(parts.a);
  if (NT > 32 && top > FEW) sorted = merge_sorted(sorted, sort_warp(parts.b));
  return __shfl_sync(ALL, sorted, top - 1);
}

// The elements of a thread's vectors that reach the bound join the candidates, as far as there is room.
template <typename T, int NT, int N> __device__ __forceinline__ void push(const Row<T>& row, const Vectors<N>& from, int first, int end, float bound,
                                                                         Shared<NT / 32>& sh) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int v = first + j * NT + threadIdx.x;
    unsigned reach = 0;
#pragma unroll
    for (int e = 0; e < Row<T>::E; ++e) reach |= element<T>(from.r[j], e) < bound ? 0u : 1u << e;
    if (v >= end) reach = 0;
    for (; reach; reach &= reach - 1) {
      const int e = __ffs(reach) - 1, at = atomicAdd(&sh.found, 1);
      const uint32_t w = word(from.r[j], sizeof(T) == 2 ? e / 2 : e);
      const float z = __uint_as_float(sizeof(T) == 2 ? (e & 1 ? w & 0xffff0000u : w << 16) : w);
      if (at < CANDIDATES) sh.candidate[at] = rank_key(z, row.index(v, e));
    }
  }
}

// The candidates of a row where the bound let too many through (constant, rising or oddly masked rows): the top-th largest of its
// vectors' elements exactly, a digit of its order at a time from counts of the digits; all above it, and of its equals the first ones.
// In the kernel and with few registers: as a function of its own with tiles in registers it cost the rows that never come here 7 %
// (16384 rows of 32000 bf16 logits, 8 alternatives) and 16 rows 2 of 12 us.
template <typename T, int NT> __device__ __forceinline__ void exact_candidates(const Row<T>& row, int begin, int end, int top, Shared<NT / 32>& sh) {
  constexpr int SHIFT = sizeof(T) == 2 ? 16 : 0, E = Row<T>::E, WARPS = NT / 32, DIGITS = 256;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int* count = reinterpret_cast<int*>(sh.record);                          // of the digits; then the digit, and how many are above it
  const uint4* from = row.base();
  uint32_t key = 0;
  int need = top;                                                          // of those whose upper digits are the key's
  for (int s = 32 - SHIFT - 8; s >= 0; s -= 8) {
    __syncthreads();
    for (int d = threadIdx.x; d < DIGITS; d += NT) count[d] = 0;
    __syncthreads();
#pragma unroll 2
    for (int v = begin + threadIdx.x; v < end; v += NT) {
      const uint4 r = from[v];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t o = order_of(element<T>(r, e)) >> SHIFT >> s;
        if (o >> 8 == key) atomicAdd(&count[o & 255], 1);
      }
    }
    __syncthreads();
    if (warp == 0) {                                                       // a lane's eight digits, the largest ones in lane 0
      int all = 0;
#pragma unroll
      for (int d = 0; d < 8; ++d) all += count[DIGITS - 1 - 8 * lane - d];
      int upto = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(ALL, upto, o);
        if (lane >= o) upto += n;
      }
      if (upto - all < need && need <= upto) {
        int above = upto - all, d = DIGITS - 1 - 8 * lane;
        while (above + count[d] < need) above += count[d--];
        count[DIGITS] = d;
        count[DIGITS + 1] = above;
      }
    }
    __syncthreads();
    key = key << 8 | (uint32_t)count[DIGITS];
    need -= count[DIGITS + 1];
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.found = 0;
  __syncthreads();
#pragma unroll 2
  for (int v = begin + threadIdx.x; v < end; v += NT) {
    const uint4 r = from[v];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float z = element<T>(r, e);
      if (order_of(z) >> SHIFT > key) sh.candidate[atomicAdd(&sh.found, 1)] = rank_key(z, row.index(v, e));      // (fewer than top)
    }
  }
  for (int first = begin, taken = 0; first < end && taken < need; first += NT) {                                  // the equals, in order
    const int v = first + threadIdx.x;
    const uint4 r = from[min(v, end - 1)];
    unsigned equal = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) equal |= (v < end && order_of(element<T>(r, e)) >> SHIFT == key ? 1u : 0u) << e;
    int before = __popc(equal);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(ALL, before, o);
      if (lane >= o) before += n;
    }
    __syncthreads();
    if (lane == 31) sh.count[warp] = (uint32_t)before;
    __syncthreads();
    before += taken - __popc(equal);
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) before += (int)sh.count[w];
      taken += (int)sh.count[w];
    }
    for (; equal && before < need; equal &= equal - 1, ++before) {
      const int e = __ffs(equal) - 1;
      sh.candidate[top - need + before] = rank_key(element<T>(r, e), row.index(v, e));
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.found = top;
  __syncthreads();
}

// now, wherever the value is used
__device__ __forceinline__ float load_now(const float* p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ float load_now(const __nv_bfloat16* p) {
  uint16_t v;
  asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return __uint_as_float((uint32_t)v << 16);
}

// One pass over the row, the next vectors on their way while these are added.  Alternatives: a thread whose N vectors reach the
// bound so far notes where they are; when the bound is final the few that still reach it are looked at again.
template <typename T, int NT, bool TOP>
__global__ void __launch_bounds__(NT, 1024 / NT) scores_kernel(const __grid_constant__ ScoreParams p) {
  constexpr int E = Row<T>::E, WARPS = NT / 32;
  __shared__ Sums<WARPS> sums;
  __shared__ typename std::conditional<TOP, Shared<WARPS>, int>::type sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int share = blockIdx.x % p.split;
  const int64_t n = blockIdx.x / p.split;
  const Row<T> row(p.logits, n, p.row_stride, p.V);
  const int each = (row.vectors + p.split - 1) / p.split, begin = share * each, end = min(begin + each, row.vectors);
  int kept = 0;                                      // candidates
  if (p.split > 1) cooperative_groups::this_cluster().barrier_arrive();

  Stats a{-INFINITY, 0.0f, 0.0f};
  const bool has_edge = share == 0 && (int)threadIdx.x < row.edges();
  const float edge = has_edge ? to_float(row.z[row.edge(threadIdx.x)]) : -INFINITY;
  if (edge != -INFINITY) {
    const float y = at_least(exponent(edge, edge)), x = exp2_of(y);
    a = Stats{edge, x, x * y};
  }
  // `top` parts of the tiles seen reach the top-th largest of the parts' maxima: so many elements do, and of any order of the
  // elements not many more are to be expected (of one tile 32 ln(32 / (32 - top))).  The bound is taken again when as many
  // tiles have passed as before: it lets about as many through from one time to the next.  Maxima of all tiles, the bound at the tiles 0, 3,
  // 7, 15, ...: 16384 rows of 32000 bf16 logits, 128 threads and 1, 8 and 32 alternatives 209, 243 and 331 us (193, 223 and 307 since the exact
  // choice is no call); at the tile 1 as well 212, 250 and 340, and with maxima of those tiles alone 213, 262 and 405; at 0, 3 and 15 (8
  // and 32) 248 and 374, at 0, 4, 12, ... 244 and 354.
  float mine = -INFINITY;                            // a thread's maximum of all tiles so far (a NaN only lowers the bound)
  uint32_t least = order_of(-INFINITY);              // the bound's order; `bound`: the smallest value that counts
  bool masked = true;
  float bound = value_of(least + masked);
  if constexpr (TOP) {
    if (threadIdx.x == 0) sh.records = sh.found = 0;
    if (NT == 32) __syncthreads();
  }

  auto take = [&](auto full, const Vectors<N>& tile, int first, int i) {
    constexpr bool FULL = decltype(full)::value;
    const int count = FULL ? N : (end - first - (int)threadIdx.x + NT - 1) / NT;
    const float most = largest_of<T, FULL>(tile, count);
    add<T, FULL>(a, tile, count, FULL ? N : (end - first + NT - 1) / NT, most);
    if constexpr (TOP) {
      mine = fmaxf(mine, most);
      if ((i & (i + 1)) == 0 && i != 1) {
        Parts parts;
        add_maxima<NT>(parts, mine, p.top <= FEW, sh.group[(__popc(i) + (i > 0)) & 1]);
        least = kth<NT>(parts, p.top);
        // (a bound as low as a mask's value: only what is above it, the rest of the choice is made below)
        masked = value_of(least) < SMALLEST;
        bound = value_of(least + masked);
      }
      if (!(most < bound)) {
        if (NT == 32 && end - begin <= N * NT) {     // (all there is: nothing to wait for; with more threads its code costs the rest)
          push<T, NT>(row, tile, first, end, bound, sh);
        } else {
          const int at = atomicAdd(&sh.records, 1);
          if (at < RECORDS) sh.record[at] = make_uint2(order_of(most), (uint32_t)(first + threadIdx.x));
        }
      }
    }
  };
  const std::true_type whole{};
  const std::false_type part{};
  Vectors<N> now, next;
  int first = begin, i = 0;
  row.template read<NT>(now, first, end);
  float given = 0.0f;                                // the token's logit, behind the first vectors instead of at the end
  bool inside = false;
  if (threadIdx.x == 0) {
    const int64_t t = p.tokens[n];
    inside = t >= 0 && t < p.V;
    given = load_now(row.z + (inside ? t : 0));
  }
  for (; first + N * NT <= end; first += N * NT, ++i) {
    row.template read<NT>(next, first + N * NT, end);
    take(whole, now, first, i);
    now = next;
  }
  for (; first < end; first += N * NT, ++i) {
    row.template read<NT>(next, first + N * NT, end);
    take(part, now, first, i);
    now = next;
  }

  if constexpr (TOP) {
    __syncthreads();
    const int records = sh.records;
    if (records <= RECORDS) {
      for (int q = warp; q < records; q += WARPS) {
        const uint2 at = sh.record[q];
        const int v = (int)at.y + lane / E * NT;
        if (at.x < least || lane >= N * E || v >= end) continue;
        const float z = to_float(row.z[row.index(v, lane % E)]);
        if (z < bound) continue;
        const int to = atomicAdd(&sh.found, 1);
        if (to < CANDIDATES) sh.candidate[to] = rank_key(z, row.index(v, lane % E));
      }
    }
    __syncthreads();
    int found = sh.found;
    if (masked && records <= RECORDS && found < p.top) {
      // A row of masked elements but for a few: of the first elements at the bound there are enough, as a rule.
      __syncthreads();                               // (all have read `found`)
      const int there = (end - begin) * E;
      for (int i = threadIdx.x; i < 4 * p.top && i < there; i += NT) {
        const float z = to_float(row.z[row.index(begin, i)]);
        if (order_of(z) == least) sh.candidate[atomicAdd(&sh.found, 1)] = rank_key(z, row.index(begin, i));
      }
      __syncthreads();
      found = sh.found;
      if (found < p.top && there > 4 * p.top) found = CANDIDATES + 1;
    }
    if (records > RECORDS || found > CANDIDATES) exact_candidates<T, NT>(row, begin, end, p.top, sh);
    if (share == 0 && row.edges()) {
      __syncthreads();                               // (all have read `found`)
      if (has_edge && order_of(edge) >= least) sh.candidate[atomicAdd(&sh.found, 1)] = rank_key(edge, row.edge(threadIdx.x));
      __syncthreads();
    }
    kept = sh.found;
  }

  join<32>(a);
  if constexpr (WARPS > 1) {
    if (lane == 0) sums.parts[warp] = a;
    __syncthreads();
    // (the row's results are left to the threads that have a candidate to rank)
    if (p.split == 1 && warp > 0 && (!TOP || warp * 32 >= kept)) return;
    a = sums.parts[lane % WARPS];
    join<WARPS>(a);
  }
  if (p.split > 1) {
    // the shares of a row meet in the first CTA of the cluster
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    cluster.barrier_wait();                          // (the first CTA has started)
    if (threadIdx.x == 0) cluster.map_shared_rank(&sums, 0)->shares[share] = a;
    if constexpr (TOP) {
      auto* to = cluster.map_shared_rank(&sh, 0);
      if ((int)threadIdx.x >= kept && (int)threadIdx.x < p.top) to->best[share * p.top + threadIdx.x] = 0;      // (fewer found)
      rank_keys<NT>(sh.candidate, kept, p.top, [&](uint64_t key, int larger) { to->best[share * p.top + larger] = key; });
    }
    cluster.sync();
    if (share > 0) return;
    a = lane < p.split ? sums.shares[lane] : Stats{-INFINITY, 0.0f, 0.0f};
    join<32>(a);
  }
  const bool empty = a.m == -INFINITY;
  const float2 sums_of = results(a);
  const float ls = sums_of.x;
  if (threadIdx.x == 0) {
    p.logprob[n] = inside ? (empty ? -INFINITY : (given - a.m) - ls) : 0.0f;
    p.entropy[n] = sums_of.y;
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
#ifdef FPB_DIAGNOSTICS
  if (launch_refused()) cfg.blockDim = dim3(0);
#endif
  return p.top ? cudaLaunchKernelEx(&cfg, scores_kernel<T, NT, true>, p) : cudaLaunchKernelEx(&cfg, scores_kernel<T, NT, false>, p);
}

template <typename T> cudaError_t scores(ScoreParams p, cudaStream_t stream) {
  const int64_t vectors = p.V / (16 / sizeof(T));
  p.split = 1;
  // Few threads a row where rows are many: what a row costs beside its elements (joins, ranks, barriers) grows with them.  bf16 logits, 8
  // alternatives, with 64, 128 and 256 threads: 16384 rows of 32000 209, 223 and 264 us, 8192 rows 120 and 123, 1024 rows 31, 27 and 29, 300
  // rows 22, 16 and 16; 64 and 128: 16384 rows of 4000 74 and 82, 2048 rows equal, 4096 rows of 128000 211 and 193, and without
  // alternatives 16384 rows of 8192 61 and 68, 8192 rows of 32000 108 and 103.  A short row gets what holds it in one round of loads.
  // A warp has 32 parts for any number of alternatives below 32; with 32 and 64 threads 65536 rows of 1000 with 20, 24, 28 and 31 alternatives take 115
  // and 231, 133 and 250, 162 and 272, 236 and 288 us.
  if (vectors <= 32 * N && p.top < 32) return scores<T, 32>(p, stream);
  if (vectors <= 64 * N || (p.rows >= 2048 && vectors <= 64 * N * (p.top ? 16 : 4))) return scores<T, 64>(p, stream);
  if (vectors <= 128 * N || p.rows >= 592) return scores<T, 128>(p, stream);
  // Very few rows: a row over a cluster of CTAs, a vector a thread at least, two CTAs an SM at most.  One CTA a row, two, four and eight:
  // 16 rows 12.3, 12.3, 10.2 and 10.2 us (sums alone 10.2, 10.2, 8.2, 8.2), 64 rows 12.3, 12.3, 12.3 and 14.3, 148 rows 12, 14, 18 and 22.
  while (p.split < MAX_SPLIT && p.rows * p.split * 2 <= 256 && vectors >= 256 * 2 * p.split) p.split *= 2;
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
  if (blockIdx.y == 0 && (int)threadIdx.x < row.edges()) {
    const int i = row.edge(threadIdx.x);
    const float z = to_float(row.z[i]);
    d[i] = from_float<T>(empty ? 0.0f : gradient(pair(z, z)).x);
  }
  const bool together = (uintptr_t)d % 16 == (uintptr_t)row.z % 16;       // vectors of z are vectors of d
  const uint4* base = row.base();
  for (int v0 = begin + threadIdx.x; v0 < end; v0 += NT * AHEAD) {
    uint4 r[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (v0 + j * NT < end) r[j] = base[v0 + j * NT];
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
      T* to = d + row.index(v, 0);
      if (together) {
        if constexpr (E == 8) store8(to, f);
        else *reinterpret_cast<float4*>(to) = make_float4(f[0], f[1], f[2], f[3]);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) to[e] = from_float<T>(f[e]);
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
    // (who wrote it first writes it again: the CTA of its vector, or the first one)
    const int v = mine < row.head ? row.vectors : (int)(mine - row.head) / E;
    if (v < row.vectors ? v < begin || v >= end : blockIdx.y > 0) continue;
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
  int split = 1;                   // few rows: shares of a row (16 rows of 32000 bf16: 10.2 us whole, 6.1 in four shares or more, 300 rows 14.3 and 12.3)
  while (split < 16 && p.rows * split * 2 <= 1184 && vectors >= 256 * 2 * split) split *= 2;
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
