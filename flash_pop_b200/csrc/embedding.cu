// Rows of an embedding table for token ids, scaled, and the table's gradient.
//   y[n] = scale W[t_n],   dW[v] = scale sum over { n : t_n = v } of dy[n]
// An id outside the table has a zero row and no part in the gradient, and so has the padding id in the gradient.
// Bound by HBM: forward reads the rows in use and writes N rows, backward reads N rows and writes the dense table.  The
// gradient has to put the ids in order first (else rows of one id are added by atomics, in another order every time).
#include "fpb_common.cuh"
#include "vec_io.cuh"

namespace fpb {
namespace {

constexpr int THREADS = 256;

struct LookupParams {
  const int64_t* tokens;
  const void* weight; int64_t w_stride;
  void* y;
  int64_t N, V;
  int32_t D, units, log_threads;     // units of eight elements (WIDE) or one a row; threads that share a row
  float scale;
};

template <typename T, bool WIDE>
__global__ void __launch_bounds__(THREADS) lookup_kernel(const __grid_constant__ LookupParams p) {
  const int per = 1 << p.log_threads, lane = threadIdx.x & (per - 1);
  const int64_t n = (int64_t)blockIdx.x * (THREADS >> p.log_threads) + (threadIdx.x >> p.log_threads);
  if (n >= p.N) return;
  const int64_t t = p.tokens[n];
  const bool inside = t >= 0 && t < p.V;
  const T* w = (const T*)p.weight + (inside ? t : 0) * p.w_stride;
  T* y = (T*)p.y + n * p.D;
  for (int u = lane; u < p.units; u += per) {
    if constexpr (WIDE) {
      float f[8];
      load8(w + u * 8, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = inside ? f[e] * p.scale : 0.0f;
      store8(y + u * 8, f);
    } else {
      y[u] = from_float<T>(inside ? to_float(w[u]) * p.scale : 0.0f);
    }
  }
}

// ---- gradient: ids in order -----------------------------------------------------------------------------------------
// The ids are brought into order with their positions by a stable radix sort, so that the rows of one id follow one another in
// the order of their positions.  An id without a part (outside the table, or the padding) counts as V and comes last.
constexpr int RADIX_BITS = 8, RADIX = 1 << RADIX_BITS, SORT_WARPS = THREADS / 32, PER_THREAD = 16, SUB = THREADS * PER_THREAD, MAX_TILES = 256;

struct SortParams {
  const int64_t* tokens;       // first pass: the ids as the caller gave them
  const uint2* in;             // later passes: (id, position)
  uint2* out;
  uint32_t* counts;            // (tiles, RADIX)
  int64_t N, V, padding;
  int32_t tiles, subs;         // a tile is `subs` times SUB ids
  int32_t shift, bits, passes; // of the digit; passes: of the one-CTA sort
  uint4* zero; int64_t zero_units; void* zero_tail; int64_t zero_elements; int32_t element;      // the table's gradient, cleared on the side
};

__device__ __forceinline__ uint2 entry(const SortParams& p, int64_t n) {
  if (p.in) return p.in[n];
  const int64_t t = p.tokens[n];
  return make_uint2((uint32_t)(t >= 0 && t < p.V && t != p.padding ? t : p.V), (uint32_t)n);
}
__device__ __forceinline__ uint32_t digit(const SortParams& p, uint32_t key, int shift) { return (key >> shift) & ((1u << p.bits) - 1u); }

__device__ void clear_table(const SortParams& p, int cta, int ctas) {
  for (int64_t i = (int64_t)cta * THREADS + threadIdx.x; i < p.zero_units; i += (int64_t)ctas * THREADS) p.zero[i] = make_uint4(0, 0, 0, 0);
  for (int64_t i = (int64_t)cta * THREADS + threadIdx.x; i < p.zero_elements; i += (int64_t)ctas * THREADS) {
    if (p.element == 2) ((uint16_t*)p.zero_tail)[i] = 0; else ((uint32_t*)p.zero_tail)[i] = 0;
  }
}

// How often each digit stands in each tile.  The CTAs behind the tiles' clear the table meanwhile (first pass): the sort leaves
// the memory idle.
__global__ void __launch_bounds__(THREADS) digit_counts_kernel(const __grid_constant__ SortParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if ((int)blockIdx.x >= p.tiles) {
    clear_table(p, blockIdx.x - p.tiles, gridDim.x - p.tiles);
    return;
  }
  __shared__ uint32_t count[RADIX];
  count[threadIdx.x] = 0;
  __syncthreads();
  const int64_t n0 = (int64_t)blockIdx.x * p.subs * SUB, n1 = min(n0 + (int64_t)p.subs * SUB, p.N);
#pragma unroll 4
  for (int64_t n = n0 + threadIdx.x; n < n1; n += THREADS) atomicAdd(&count[digit(p, entry(p, n).x, p.shift)], 1u);
  __syncthreads();
  p.counts[blockIdx.x * RADIX + threadIdx.x] = count[threadIdx.x];
}

// sum over the threads before this one
__device__ uint32_t block_scan(uint32_t v, uint32_t (&sums)[SORT_WARPS]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  for (int w = 0; w < warp; ++w) x += sums[w];
  return x - v;
}

// Ranks of a CTA's SUB entries among those of the same digit, in their order: each warp has 32 * PER_THREAD consecutive ones.
// Leaves in `before` what stands of the digit in the warp so far.
__device__ __forceinline__ void warp_ranks(const uint32_t (&d)[PER_THREAD], uint32_t (&rank)[PER_THREAD], uint32_t* before) {
  const unsigned lower = (1u << (threadIdx.x & 31)) - 1u;
#pragma unroll
  for (int i = 0; i < PER_THREAD; ++i) {
    const unsigned same = __match_any_sync(0xffffffffu, d[i]);
    const bool real = d[i] < RADIX;
    if (real) rank[i] = before[d[i]] + __popc(same & lower);
    __syncwarp();
    if (real && (same & lower) == 0) before[d[i]] += __popc(same);
    __syncwarp();
  }
}

// Every entry to its place: behind all smaller digits, and behind the same digit in earlier tiles, warps and lanes.
__global__ void __launch_bounds__(THREADS) scatter_kernel(const __grid_constant__ SortParams p) {
  __shared__ uint32_t before[SORT_WARPS][RADIX], sums[SORT_WARPS];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  uint32_t mine = 0, all = 0;                                      // of digit threadIdx.x, in earlier tiles and in all
#pragma unroll 8
  for (int t = 0; t < p.tiles; ++t) {
    const uint32_t c = p.counts[t * RADIX + threadIdx.x];
    all += c;
    if (t < (int)blockIdx.x) mine += c;
  }
  uint32_t base = block_scan(all, sums) + mine;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int s = 0; s < p.subs; ++s) {
    const int64_t n0 = ((int64_t)blockIdx.x * p.subs + s) * SUB + warp * 32 * PER_THREAD + lane;
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) before[w][threadIdx.x] = 0;
    __syncthreads();
    uint2 e[PER_THREAD];
    uint32_t d[PER_THREAD], rank[PER_THREAD];
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
      const int64_t n = n0 + i * 32;
      d[i] = RADIX;
      if (n < p.N) { e[i] = entry(p, n); d[i] = digit(p, e[i].x, p.shift); }
    }
    warp_ranks(d, rank, before[warp]);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) {
      const uint32_t c = before[w][threadIdx.x];
      before[w][threadIdx.x] = base;
      base += c;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i)
      if (d[i] < RADIX) p.out[before[warp][d[i]] + rank[i]] = e[i];
    __syncthreads();
  }
}

// All passes of up to SUB ids in the first CTA; the others clear the table.
__global__ void __launch_bounds__(THREADS) small_sort_kernel(const __grid_constant__ SortParams p) {
  __shared__ uint32_t before[SORT_WARPS][RADIX], sums[SORT_WARPS];
  __shared__ uint2 moved[SUB];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (blockIdx.x > 0) {
    clear_table(p, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n0 = warp * 32 * PER_THREAD + lane;
  uint2 e[PER_THREAD];
  uint32_t d[PER_THREAD], rank[PER_THREAD];
#pragma unroll
  for (int i = 0; i < PER_THREAD; ++i)
    if (n0 + i * 32 < p.N) e[i] = entry(p, n0 + i * 32);
  for (int pass = 0; pass < p.passes; ++pass) {
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) before[w][threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) d[i] = n0 + i * 32 < p.N ? digit(p, e[i].x, pass * p.bits) : RADIX;
    warp_ranks(d, rank, before[warp]);
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) all += before[w][threadIdx.x];
    uint32_t base = block_scan(all, sums);
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) {
      const uint32_t c = before[w][threadIdx.x];
      before[w][threadIdx.x] = base;
      base += c;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i)
      if (d[i] < RADIX) moved[before[warp][d[i]] + rank[i]] = e[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i)
      if (n0 + i * 32 < p.N) e[i] = moved[n0 + i * 32];
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < PER_THREAD; ++i)
    if (n0 + i * 32 < p.N) p.out[n0 + i * 32] = e[i];
}

// ---- gradient: sums over the rows of an id --------------------------------------------------------------------------
// The sorted entries are cut into windows of W, whatever ids they hold, so that every group of threads has the same work.  A run
// of one id that lies inside a window is summed and written; the parts of a run that goes over windows' ends are left in
// `partial`, slot 0 of a window for a run that began before it, slot 1 for one that begins in it and goes on, and added up by
// join_kernel in the order of the windows.  Where windows end depends on N and D alone: the same bits every time.
constexpr int SUM_THREADS = 128, AHEAD = 8, MAX_WINDOW = 128;

struct SumParams {
  const uint2* sorted;
  const void* dy; int64_t dy_stride;
  void* dw;
  float* partial;              // (windows, 2, pitch)
  int64_t N, windows;
  uint32_t V;
  int32_t D, pitch, W, log_threads;       // threads that share a window
  float scale;
};

template <typename T, bool WIDE>
__global__ void __launch_bounds__(SUM_THREADS) run_sums_kernel(const __grid_constant__ SumParams p) {
  constexpr int C = WIDE ? 8 : 1;          // columns of a thread
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int per = 1 << p.log_threads;
  const int64_t window = (int64_t)blockIdx.x * (SUM_THREADS >> p.log_threads) + (threadIdx.x >> p.log_threads);
  const int64_t col = ((int64_t)blockIdx.y * per + (threadIdx.x & (per - 1))) * C;
  if (window >= p.windows || col >= p.D) return;
  const int64_t begin = window * p.W, end = min(begin + p.W, p.N);
  const uint32_t before = begin > 0 ? p.sorted[begin - 1].x : p.V, after = end < p.N ? p.sorted[end].x : p.V;
  const T* dy = (const T*)p.dy + col;
  uint2 e[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) e[j] = begin + j < end ? p.sorted[begin + j] : make_uint2(p.V, 0);
  uint32_t id = e[0].x;
  if (id == p.V) return;
  bool open = id == before;                // the run in hand began before this window
  float acc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) acc[c] = 0.0f;

  auto finish = [&](bool goes_on) {
    if (open || goes_on) {
      float* to = p.partial + (window * 2 + (open ? 0 : 1)) * p.pitch + col;
      if constexpr (WIDE) store8(to, acc); else *to = acc[0];
    } else {
      T* to = (T*)p.dw + (int64_t)id * p.D + col;
#pragma unroll
      for (int c = 0; c < C; ++c) acc[c] *= p.scale;
      if constexpr (WIDE) store8(to, acc); else *to = from_float<T>(acc[0]);
    }
  };

  for (int64_t i = begin; i < end; i += AHEAD) {
    Raw8<T> rows[WIDE ? AHEAD : 1];
    T single[WIDE ? 1 : AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const T* from = dy + (int64_t)e[j].y * p.dy_stride;         // (an entry behind the last one stands for row 0)
      if constexpr (WIDE) read8(from, rows[j]); else single[j] = *from;
    }
    uint2 ahead[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) ahead[j] = i + AHEAD + j < end ? p.sorted[i + AHEAD + j] : make_uint2(p.V, 0);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (e[j].x != id) {
        finish(false);                     // (windows are multiples of AHEAD: only the last one has entries behind its end)
        id = e[j].x;
        if (id == p.V) return;
        open = false;
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] = 0.0f;
      }
      if constexpr (WIDE) {
        float f[8];
        unpack8(rows[j], f);
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] += f[c];
      } else {
        acc[0] += to_float(single[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) e[j] = ahead[j];
  }
  finish(after == id);
}

// Four columns a thread, JOIN_SLICES threads for the same columns of a run, each every fourth window of it.
constexpr int JOIN_COLS = 128, JOIN_SLICES = 4, JOIN_THREADS = JOIN_COLS * JOIN_SLICES;

template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const __grid_constant__ SumParams p) {
  __shared__ float4 sums[JOIN_SLICES][JOIN_COLS];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int slice = threadIdx.x / JOIN_COLS, lane = threadIdx.x % JOIN_COLS;
  const int64_t col = ((int64_t)blockIdx.y * JOIN_COLS + lane) * 4;
  for (int64_t w = blockIdx.x; w + 1 < p.windows; w += gridDim.x) {
    const int64_t begin = w * p.W, last = begin + p.W - 1;
    const uint32_t id = p.sorted[last].x;
    if (id == p.V || p.sorted[last + 1].x != id) continue;                                 // no run goes on behind this window
    if (p.sorted[begin].x == id && begin > 0 && p.sorted[begin - 1].x == id) continue;     // it began before this window
    int64_t windows = 1;                                                                    // that it goes through after this one
    for (;;) {
      const int64_t first = (w + windows + 1 + threadIdx.x) * p.W;                           // of the window after each of them
      const int more = __syncthreads_count(first < p.N && p.sorted[first].x == id);         // (the first `more` threads: ids are in order)
      windows += more;
      if (more < JOIN_THREADS) break;
    }
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (col < p.pitch) {
      if (slice == 0) a = *reinterpret_cast<const float4*>(p.partial + (w * 2 + 1) * p.pitch + col);
#pragma unroll 8
      for (int64_t u = w + 1 + slice; u <= w + windows; u += JOIN_SLICES) {
        const float4 b = *reinterpret_cast<const float4*>(p.partial + u * 2 * p.pitch + col);
        a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
      }
    }
    sums[slice][lane] = a;
    __syncthreads();
    if (slice == 0) {
#pragma unroll
      for (int s = 1; s < JOIN_SLICES; ++s) {
        const float4 b = sums[s][lane];
        a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
      }
      const float f[4] = {a.x, a.y, a.z, a.w};
      T* to = (T*)p.dw + (int64_t)id * p.D + col;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (col + c < p.D) to[c] = from_float<T>(f[c] * p.scale);
    }
    __syncthreads();
  }
}

// How a gradient is cut up, and where its scratch memory lies.
struct GradPlan {
  int tiles, subs, passes, bits, window;
  int64_t windows, pitch;
  int64_t sorted[2], counts, partial, bytes;      // byte offsets
};
GradPlan plan_grad(int64_t N, int64_t V, int D) {
  GradPlan g{};
  const int64_t subs = (N + SUB - 1) / SUB;
  g.subs = (int)((subs + MAX_TILES - 1) / MAX_TILES);
  g.tiles = (int)((subs + g.subs - 1) / g.subs);
  int bits = 1;
  while (V >> bits) ++bits;                        // of the ids and of V itself
  g.passes = (bits + RADIX_BITS - 1) / RADIX_BITS;
  g.bits = (bits + g.passes - 1) / g.passes;
  // windows as long as leaves 1024 threads an SM: fewer parts to join
  const int64_t columns = (D + 7) / 8;
  g.window = MAX_WINDOW;
  while (g.window > 16 && (N + g.window - 1) / g.window * columns < 148 * 1024) g.window /= 2;
  g.windows = (N + g.window - 1) / g.window;
  g.pitch = (D + 3) / 4 * 4;
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t a = at; at += (bytes + 15) / 16 * 16; return a; };
  g.sorted[0] = take(8 * N); g.sorted[1] = take(8 * N);
  g.counts = take((int64_t)g.tiles * RADIX * 4);
  g.partial = take(g.windows * 2 * g.pitch * 4);
  g.bytes = at;
  return g;
}

template <typename T>
cudaError_t table_grad(const GradPlan& g, SortParams s, SumParams q, bool wide, char* space, cudaStream_t stream, int* n_launched) {
  constexpr int CLEARING = 592;                    // CTAs
  uint2* buffers[2] = {(uint2*)(space + g.sorted[0]), (uint2*)(space + g.sorted[1])};
  cudaError_t e;
  if (g.tiles * g.subs == 1) {
    s.out = buffers[0];
    e = launch_kernel(small_sort_kernel, dim3(1 + CLEARING), THREADS, 0, false, s, stream);
    *n_launched += 1;
    q.sorted = buffers[0];
  } else {
    e = cudaSuccess;
    for (int pass = 0; pass < g.passes && e == cudaSuccess; ++pass) {
      s.in = pass == 0 ? nullptr : buffers[(pass - 1) & 1];
      s.out = buffers[pass & 1];
      s.shift = pass * g.bits;
      e = launch_kernel(digit_counts_kernel, dim3(g.tiles + (pass == 0 ? CLEARING : 0)), THREADS, 0, pass > 0, s, stream);
      if (e == cudaSuccess) e = launch_kernel(scatter_kernel, dim3(g.tiles), THREADS, 0, true, s, stream);
      *n_launched += 2;
    }
    q.sorted = buffers[(g.passes - 1) & 1];
  }
  if (e != cudaSuccess) return e;
  const int64_t units = wide ? q.D / 8 : q.D;
  q.log_threads = 0;
  while ((1 << q.log_threads) < units && (1 << q.log_threads) < SUM_THREADS) ++q.log_threads;
  const int per = 1 << q.log_threads, groups = SUM_THREADS >> q.log_threads;
  const dim3 grid((unsigned)((q.windows + groups - 1) / groups), (unsigned)((units + per - 1) / per));
  e = wide ? launch_kernel(run_sums_kernel<T, true>, grid, SUM_THREADS, 0, true, q, stream)
           : launch_kernel(run_sums_kernel<T, false>, grid, SUM_THREADS, 0, true, q, stream);
  *n_launched += 1;
  if (e == cudaSuccess && q.windows > 1) {
    const dim3 joins((unsigned)(q.windows < 592 ? q.windows : 592), (unsigned)((q.D + 4 * JOIN_COLS - 1) / (4 * JOIN_COLS)));
    e = launch_kernel(join_kernel<T>, joins, JOIN_THREADS, 0, true, q, stream);
    *n_launched += 1;
  }
  return e;
}

template <typename T>
cudaError_t lookup(LookupParams p, bool wide, cudaStream_t stream) {
  p.units = wide ? p.D / 8 : p.D;
  p.log_threads = 0;
  while ((1 << p.log_threads) < p.units && p.log_threads < 8) ++p.log_threads;
  const int rows = THREADS >> p.log_threads;
  const dim3 grid((unsigned)((p.N + rows - 1) / rows));
  return wide ? launch_kernel(lookup_kernel<T, true>, grid, THREADS, 0, false, p, stream)
              : launch_kernel(lookup_kernel<T, false>, grid, THREADS, 0, false, p, stream);
}

}  // namespace

int launch_embedding(int dtype, int64_t N, int64_t V, int D, const int64_t* tokens, const void* weight, int64_t w_stride, float scale, void* y,
                     cudaStream_t stream) {
  const LookupParams p{tokens, weight, w_stride, y, N, V, D, 0, 0, scale};
  const int vec = dtype == FPB_BF16 ? 8 : 4;
  const bool wide = D % 8 == 0 && w_stride % vec == 0 && ((uintptr_t)weight | (uintptr_t)y) % 16 == 0;
  const cudaError_t e = dtype == FPB_BF16 ? lookup<__nv_bfloat16>(p, wide, stream) : lookup<float>(p, wide, stream);
  return e == cudaSuccess ? FPB_OK : FPB_ERR_LAUNCH;
}

int64_t embedding_workspace(int64_t N, int64_t V, int D) {
  return N > 0 && V > 0 && D > 0 && N < (1ll << 31) && V < (1ll << 31) ? plan_grad(N, V, D).bytes : 0;
}

int launch_embedding_grad(int dtype, int64_t N, int64_t V, int D, const int64_t* tokens, int64_t padding, float scale, const void* dy,
                          int64_t dy_stride, void* dw, void* workspace, cudaStream_t stream, int* n_launched) {
  const GradPlan g = plan_grad(N, V, D);
  const int size = dtype == FPB_BF16 ? 2 : 4;
  SortParams s{};
  s.tokens = tokens; s.N = N; s.V = V; s.padding = padding;
  s.tiles = g.tiles; s.subs = g.subs; s.bits = g.bits; s.passes = g.passes;
  s.counts = (uint32_t*)((char*)workspace + g.counts);
  const int64_t bytes = V * D * size;
  s.element = size;
  s.zero = (uint4*)dw;
  s.zero_units = (uintptr_t)dw % 16 == 0 ? bytes / 16 : 0;
  s.zero_tail = (char*)dw + s.zero_units * 16;
  s.zero_elements = (bytes - s.zero_units * 16) / size;
  SumParams q{};
  q.dy = dy; q.dy_stride = dy_stride; q.dw = dw; q.partial = (float*)((char*)workspace + g.partial);
  q.N = N; q.windows = g.windows; q.V = (uint32_t)V; q.D = D; q.pitch = (int32_t)g.pitch; q.W = g.window; q.scale = scale;
  const int vec = 16 / size;
  const bool wide = D % 8 == 0 && (N <= 1 || dy_stride % vec == 0) && ((uintptr_t)dy | (uintptr_t)dw) % 16 == 0;
  *n_launched = 0;
  const cudaError_t e = dtype == FPB_BF16 ? table_grad<__nv_bfloat16>(g, s, q, wide, (char*)workspace, stream, n_launched)
                                          : table_grad<float>(g, s, q, wide, (char*)workspace, stream, n_launched);
  return e == cudaSuccess ? FPB_OK : FPB_ERR_LAUNCH;
}

}  // namespace fpb
