// Rows of an embedding table for token ids, scaled, and the table's gradient.
//   y[n] = scale W[t_n],   dW[v] = scale sum over { n : t_n = v } of dy[n]
// An id outside the table has a zero row and no part in the gradient, and so has the padding id in the gradient.
// Bound by HBM: forward reads the rows in use and writes N rows, backward reads N rows and writes the dense table.  The
// gradient has to put the ids in order first (else rows of one id are added by atomics, in another order every time).
#include <algorithm>
#include <atomic>

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

// Threads share a row, units apart; each has ROWS rows in flight.
constexpr int ROWS = 4;

template <typename T, bool WIDE>
__global__ void __launch_bounds__(THREADS) lookup_kernel(const __grid_constant__ LookupParams p) {
  const int per = 1 << p.log_threads, lane = threadIdx.x & (per - 1), groups = THREADS >> p.log_threads;
  const int64_t n0 = (int64_t)blockIdx.x * groups * ROWS + (threadIdx.x >> p.log_threads);
  if (n0 >= p.N) return;
  int64_t token[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) token[i] = n0 + i * groups < p.N ? p.tokens[n0 + i * groups] : -1;
  for (int u = lane; u < p.units; u += per) {
    Raw8<T> row[WIDE ? ROWS : 1];
    T single[WIDE ? 1 : ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const bool inside = token[i] >= 0 && token[i] < p.V;
      const T* w = (const T*)p.weight + (inside ? token[i] : 0) * p.w_stride;
      if constexpr (WIDE) read8(w + u * 8, row[i]); else single[i] = w[u];
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int64_t n = n0 + i * groups;
      if (n >= p.N) break;
      const bool inside = token[i] >= 0 && token[i] < p.V;
      T* y = (T*)p.y + n * p.D;
      if constexpr (WIDE) {
        float f[8];
        unpack8(row[i], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = inside ? f[e] * p.scale : 0.0f;
        store8(y + u * 8, f);
      } else {
        y[u] = from_float<T>(inside ? to_float(single[i]) * p.scale : 0.0f);
      }
    }
  }
}

// ---- gradient: ids in order -----------------------------------------------------------------------------------------
// The ids are brought into order with their positions by a stable radix sort, so that the rows of one id follow one another in
// the order of their positions.  An id without a part (outside the table, or the padding) counts as V and comes last.
constexpr int RADIX_BITS = 8, RADIX = 1 << RADIX_BITS, PER_THREAD = 8, MAX_TILES = 256;
constexpr int TILE_THREADS = 512, SUB = TILE_THREADS * PER_THREAD, CLEARING = 592;      // CTAs that clear a table

struct SortParams {
  const int64_t* tokens;       // first pass: the ids as the caller gave them
  const uint2* in;             // later passes: (id, position)
  uint2* out;
  uint32_t* counts;            // (tiles, RADIX)
  int64_t N, V, padding;
  int32_t tiles, subs;         // a tile is `subs` times SUB ids
  int32_t shift, bits;         // of the digit
  uint4* zero; int64_t zero_units; void* zero_tail; int64_t zero_elements; int32_t element;      // the table's gradient, cleared on the side
};

__device__ __forceinline__ uint2 entry(const SortParams& p, int64_t n) {
  if (p.in) return p.in[n];
  const int64_t t = p.tokens[n];
  return make_uint2((uint32_t)(t >= 0 && t < p.V && t != p.padding ? t : p.V), (uint32_t)n);
}
__device__ __forceinline__ uint32_t digit(const SortParams& p, uint32_t key, int shift) { return (key >> shift) & ((1u << p.bits) - 1u); }

template <int T> __device__ void clear_table(const SortParams& p, int cta, int ctas) {
  for (int64_t i = (int64_t)cta * T + threadIdx.x; i < p.zero_units; i += (int64_t)ctas * T) p.zero[i] = make_uint4(0, 0, 0, 0);
  for (int64_t i = (int64_t)cta * T + threadIdx.x; i < p.zero_elements; i += (int64_t)ctas * T) {
    if (p.element == 2) ((uint16_t*)p.zero_tail)[i] = 0; else ((uint32_t*)p.zero_tail)[i] = 0;
  }
}

// How often each digit stands in each tile.
__global__ void __launch_bounds__(TILE_THREADS) digit_counts_kernel(const __grid_constant__ SortParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ uint32_t count[RADIX];
  if (threadIdx.x < RADIX) count[threadIdx.x] = 0;
  __syncthreads();
  const int64_t n0 = (int64_t)blockIdx.x * p.subs * SUB, n1 = min(n0 + (int64_t)p.subs * SUB, p.N);
  for (int64_t n = n0 + threadIdx.x; n < n1; n += SUB) {
    // (entries behind the end repeat the last one and are not counted: a load behind a branch would wait for the one before)
    uint32_t d[PER_THREAD];
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) d[i] = digit(p, entry(p, min(n + i * TILE_THREADS, n1 - 1)).x, p.shift);
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i)
      if (n + i * TILE_THREADS < n1) atomicAdd(&count[d[i]], 1u);
  }
  __syncthreads();
  if (threadIdx.x < RADIX) p.counts[blockIdx.x * RADIX + threadIdx.x] = count[threadIdx.x];
}

// The places of a CTA's T * PER_THREAD entries when they are put in order of one digit, equal digits in the order they stand in:
// each warp has 32 * PER_THREAD consecutive ones, lane after lane.
template <int T> struct Order {
  static constexpr int WARPS = T / 32;
  uint32_t before[WARPS][RADIX], sums[RADIX / 32];

  __device__ void clear() {
    for (int i = threadIdx.x; i < WARPS * RADIX; i += T) (&before[0][0])[i] = 0;
    __syncthreads();
  }
  // Ranks of a warp's entries among those of the same digit; leaves in `before` how many of each digit the warp has.  Which lanes share a digit is
  // found by a ballot for each of its bits.  One barrier.  `each`: how many entries a thread has.
  __device__ void rank(const uint32_t (&d)[PER_THREAD], uint32_t (&r)[PER_THREAD], int each = PER_THREAD) {
    const unsigned lower = (1u << (threadIdx.x & 31)) - 1u;
    uint32_t* mine = before[threadIdx.x >> 5];
    unsigned same[PER_THREAD];
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
      if (i >= each) break;
      same[i] = __ballot_sync(0xffffffffu, d[i] < RADIX);
#pragma unroll
      for (int b = 0; b < RADIX_BITS; ++b) {
        const bool one = d[i] >> b & 1u;
        const unsigned ones = __ballot_sync(0xffffffffu, one);
        same[i] &= one ? ones : ~ones;
      }
    }
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
      if (i >= each) break;
      const bool real = d[i] < RADIX;
      if (real) r[i] = mine[d[i]] + __popc(same[i] & lower);
      __syncwarp();
      if (real && (same[i] & lower) == 0) mine[d[i]] += __popc(same[i]);
      __syncwarp();
    }
    __syncthreads();
  }
  // sum over the digits before thread's (threads below RADIX); one barrier
  __device__ uint32_t scan(uint32_t v) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31 && warp < RADIX / 32) sums[warp] = x;
    __syncthreads();
    for (int w = 0; w < warp && w < RADIX / 32; ++w) x += sums[w];
    return x - v;
  }
  // counts of the warps -> where each warp's part of a digit begins; base: where the digit does, moved on.  One barrier.
  __device__ void place(uint32_t& base) {
    if (threadIdx.x < RADIX) {
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const uint32_t c = before[w][threadIdx.x];
        before[w][threadIdx.x] = base;
        base += c;
      }
    }
    __syncthreads();
  }
  __device__ uint32_t at(uint32_t d, uint32_t r) const { return before[threadIdx.x >> 5][d] + r; }
};

// Every entry to its place: behind all smaller digits, and behind the same digit in earlier tiles, warps and lanes.  The CTAs behind
// the tiles' clear the table meanwhile (first pass): 13 us of latency that leave the memory idle.  (Nothing before this call's first launch
// is still running, so they need not wait.)
__global__ void __launch_bounds__(TILE_THREADS) scatter_kernel(const __grid_constant__ SortParams p) {
  __shared__ Order<TILE_THREADS> order;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if ((int)blockIdx.x >= p.tiles) {
    clear_table<TILE_THREADS>(p, blockIdx.x - p.tiles, gridDim.x - p.tiles);
    return;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  uint32_t mine = 0, all = 0;                                      // of digit threadIdx.x, in earlier tiles and in all
  if (threadIdx.x < RADIX) {
    for (int t0 = 0; t0 < p.tiles; t0 += 16) {
      uint32_t c[16];
#pragma unroll
      for (int t = 0; t < 16; ++t) c[t] = p.counts[min(t0 + t, p.tiles - 1) * RADIX + threadIdx.x];
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        if (t0 + t < p.tiles) all += c[t];
        if (t0 + t < (int)blockIdx.x) mine += c[t];
      }
    }
  }
  uint32_t base = order.scan(all) + mine;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int s = 0; s < p.subs; ++s) {
    const int64_t n0 = ((int64_t)blockIdx.x * p.subs + s) * SUB + warp * 32 * PER_THREAD + lane;
    uint2 e[PER_THREAD];
    uint32_t d[PER_THREAD], r[PER_THREAD];
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
      const int64_t n = n0 + i * 32;
      e[i] = entry(p, min(n, p.N - 1));
      d[i] = n < p.N ? digit(p, e[i].x, p.shift) : RADIX;
    }
    order.clear();
    order.rank(d, r);
    order.place(base);
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i)
      if (d[i] < RADIX) p.out[order.at(d[i], r[i])] = e[i];
    __syncthreads();
  }
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
  for (int j = 0; j < AHEAD; ++j) {
    e[j] = p.sorted[min(begin + j, end - 1)];
    if (begin + j >= end) e[j].x = p.V;
  }
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
      const T* from = dy + (int64_t)e[j].y * p.dy_stride;
      if constexpr (WIDE) read8(from, rows[j]); else single[j] = *from;
    }
    uint2 ahead[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      ahead[j] = p.sorted[min(i + AHEAD + j, end - 1)];
      if (i + AHEAD + j >= end) ahead[j].x = p.V;
    }
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

// A CTA a window, four columns a thread: the run that begins in the window and goes on, if there is one.
constexpr int JOIN_THREADS = 128, JOIN_COLS = 4 * JOIN_THREADS;

template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const __grid_constant__ SumParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t w = blockIdx.x, begin = w * p.W, last = begin + p.W - 1;                 // (not the last window: there is a next one)
  const int64_t col = ((int64_t)blockIdx.y * JOIN_THREADS + threadIdx.x) * 4;
  const uint32_t id = p.sorted[last].x, next = p.sorted[last + 1].x, first = p.sorted[begin].x, before = begin > 0 ? p.sorted[begin - 1].x : p.V;
  if (id == p.V || next != id) return;                                                   // no run goes on behind this window
  if (first == id && before == id) return;                                               // it began before this window
  int64_t windows = 1;                                                                   // that it goes through after this one
  for (;;) {
    const int64_t at = (w + windows + 1 + threadIdx.x) * p.W;                            // of the window after each of them
    const int more = __syncthreads_count(at < p.N && p.sorted[at].x == id);             // (the first `more` threads: ids are in order)
    windows += more;
    if (more < JOIN_THREADS) break;
  }
  if (col >= p.pitch) return;
  float4 a = *reinterpret_cast<const float4*>(p.partial + (w * 2 + 1) * p.pitch + col);
  const int64_t end = w + windows;
  for (int64_t u = w + 1; u <= end; u += 16) {
    float4 b[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) b[i] = *reinterpret_cast<const float4*>(p.partial + min(u + i, end) * 2 * p.pitch + col);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (u + i <= end) { a.x += b[i].x; a.y += b[i].y; a.z += b[i].z; a.w += b[i].w; }
  }
  const float f[4] = {a.x, a.y, a.z, a.w};
  T* to = (T*)p.dw + (int64_t)id * p.D + col;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (col + c < p.D) to[c] = from_float<T>(f[c] * p.scale);
}

// ---- gradient of a few ids: one launch ------------------------------------------------------------------------------
// A CTA has every share-th row of the table, FEW_COLUMNS columns of it (or several such tiles, for very wide rows), and all that happens to
// them: it clears them (but for large tables), picks their ids from all N, puts them in order in shared memory, and sums.  Rows next to one
// another belong to different CTAs, as frequent ids often are neighbours.  The ordered ids are cut into a piece for each strand of eight
// threads, whatever ids they hold; parts of a run that goes over pieces' ends meet in shared memory, in the order of the pieces.  What
// shares and pieces are depends on N, V, D and the ids alone: the same bits every time.
// The calls it is for wait for the host (a launch is 3 to 4 us there) and for latency: between events around the call 5003 ids of 8001 rows of 333
// fp32 take 25 us where a sort, the sums and a join of windows as launches of their own took 30, 8192 ids of 32000 x 1024 bf16 31 and 34, 64 of
// them 21 and 28 (10 of which the 66 MB of zeros), 8192 equal ids 49 and 46; 9000 ids, by those launches, take 41.
constexpr int FEW_THREADS = 1024, STRAND = 8, STRANDS = FEW_THREADS / STRAND, FEW_COLUMNS = STRAND * 8, RANKED = 256;
static_assert(FEW_THREADS * PER_THREAD == FPB_EMBEDDING_FEW, "an id is held by a thread from the start");

struct FewParams {
  const int64_t* tokens;
  const void* dy; int64_t dy_stride;
  void* dw;
  int64_t V, padding;
  int32_t N, D, share, tiles, bits, passes, clears;      // clears: the rows as well (else the launch before does)
  float scale;
};
struct FewShared {
  Order<FEW_THREADS> order;
  uint2 sorted[FPB_EMBEDDING_FEW];                                 // (row / share, position)
  float part[2][STRANDS][FEW_COLUMNS];                             // of a run that began in an earlier piece; of one that goes on in a later one
  uint32_t count[FEW_THREADS / 32];
};

template <typename T, bool WIDE>
__global__ void __launch_bounds__(FEW_THREADS) few_grad_kernel(const __grid_constant__ FewParams p) {
  constexpr int FLIGHT = WIDE && sizeof(T) == 2 ? 8 : 4;          // rows in flight: 32 registers
  extern __shared__ __align__(16) unsigned char dynamic[];
  FewShared& sh = *reinterpret_cast<FewShared*>(dynamic);
  const int strand = threadIdx.x / STRAND, lane = threadIdx.x % STRAND, warp = threadIdx.x / 32, n0 = warp * 32 * PER_THREAD + threadIdx.x % 32;
  const unsigned lower = (1u << threadIdx.x % 32) - 1u;
  const uint32_t share = (uint32_t)p.share;
  // a thread's columns of a tile: eight beside one another, or (c * STRAND + lane)
  auto column = [&](int tile, int c) { return (int64_t)tile * FEW_COLUMNS + (WIDE ? lane * 8 + c : c * STRAND + lane); };
  auto write = [&](int64_t row, int tile, const float (&f)[8]) {
    T* to = (T*)p.dw + row * p.D;
    if constexpr (WIDE) {
      if (column(tile, 0) < p.D) store8(to + column(tile, 0), f);
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (column(tile, c) < p.D) to[column(tile, c)] = from_float<T>(f[c]);
    }
  };

  uint2 e[PER_THREAD];
  unsigned with[PER_THREAD];                       // lanes whose id is a row of this share
  int found = 0;                                   // (of the warp)
#pragma unroll
  for (int i = 0; i < PER_THREAD; ++i) {
    const int64_t t = p.tokens[min(n0 + i * 32, p.N - 1)];
    const bool inside = n0 + i * 32 < p.N && t >= 0 && t < p.V && t != p.padding;
    e[i] = make_uint2((uint32_t)t / share, (uint32_t)(n0 + i * 32));
    with[i] = __ballot_sync(0xffffffffu, inside && (uint32_t)t % share == blockIdx.x);
    found += __popc(with[i]);
  }
  if (threadIdx.x % 32 == 0) sh.count[warp] = (uint32_t)found;
  // The share's rows are cleared: a strand a row, or where rows are not aligned a warp.
  for (int tile = blockIdx.y; tile < p.tiles && p.clears; tile += gridDim.y) {
    constexpr int TEAM = WIDE ? STRAND : 32, UNIT = WIDE ? 16 / (int)sizeof(T) : 1;
    const int64_t last = min((int64_t)(tile + 1) * FEW_COLUMNS, (int64_t)p.D);
    for (int64_t row = blockIdx.x + (int64_t)(threadIdx.x / TEAM) * share; row < p.V; row += (int64_t)(FEW_THREADS / TEAM) * share) {
#pragma unroll
      for (int c = threadIdx.x % TEAM * UNIT; c < FEW_COLUMNS; c += TEAM * UNIT) {
        const int64_t col = (int64_t)tile * FEW_COLUMNS + c;
        if (col >= last) break;
        T* to = (T*)p.dw + row * p.D + col;
        if constexpr (WIDE) *reinterpret_cast<uint4*>(to) = make_uint4(0, 0, 0, 0); else *to = from_float<T>(0.0f);
      }
    }
  }
  __syncthreads();
  {
    const uint32_t mine = sh.count[threadIdx.x % 32];              // of 32 warps
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (threadIdx.x % 32 >= (unsigned)o) upto += x;
    }
    found = (int)__shfl_sync(0xffffffffu, upto, 31);               // (of all)
    uint32_t at = __shfl_sync(0xffffffffu, upto - mine, warp);
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
      if (with[i] >> threadIdx.x % 32 & 1u) sh.sorted[at + __popc(with[i] & lower)] = e[i];
      at += __popc(with[i]);
    }
  }
  __syncthreads();
  // They stand in the order of their positions.  Up to RANKED of them go to their places by counting, each with four threads or more, who goes
  // before it: those in front with a key that is not larger, those behind with a smaller one.  More go by digits, as many a thread as
  // it takes all threads.  By counting and by two digits: 255 of them 3.7 and 6 us, 500 7.9 and 6.4.
  if (found <= RANKED) {
    uint32_t* keys = &sh.order.before[0][0];
    if (threadIdx.x < RANKED) keys[threadIdx.x] = (int)threadIdx.x < found ? sh.sorted[threadIdx.x].x : 0xffffffffu;
    __syncthreads();
    int per = FEW_THREADS / RANKED;
    while (per < 32 && found * per * 2 <= FEW_THREADS) per *= 2;
    const int i = threadIdx.x / per;
    const uint2 own = i < found ? sh.sorted[i] : make_uint2(0, 0);
    uint32_t before = 0;
    const int group = i & ~3;                      // (four keys at a time, those of i's own group once more)
    for (int j = threadIdx.x % per * 4; j < found; j += per * 4) {
      const uint4 k = *reinterpret_cast<const uint4*>(keys + j);
      const uint32_t limit = own.x + (j < group);
      before += (k.x < limit) + (k.y < limit) + (k.z < limit) + (k.w < limit);
    }
    if (threadIdx.x % per == 0)
      for (int j = group; j < i; ++j) before += keys[j] == own.x;
    for (int o = 1; o < per; o *= 2) before += __shfl_xor_sync(0xffffffffu, before, o);
    __syncthreads();
    if (i < found && threadIdx.x % per == 0) sh.sorted[before] = own;
    __syncthreads();
  } else {
    const int each = (found + FEW_THREADS - 1) / FEW_THREADS, first = warp * 32 * each + threadIdx.x % 32;
    uint32_t d[PER_THREAD], r[PER_THREAD];
    for (int pass = 0; pass < p.passes; ++pass) {
#pragma unroll
      for (int i = 0; i < PER_THREAD; ++i) {
        const bool real = i < each && first + i * 32 < found;
        if (real) e[i] = sh.sorted[first + i * 32];
        d[i] = real ? (e[i].x >> pass * p.bits) & ((1u << p.bits) - 1u) : RADIX;
      }
      sh.order.clear();
      sh.order.rank(d, r, each);
      uint32_t all = 0;
      if (threadIdx.x < RADIX) {
#pragma unroll
        for (int w = 0; w < FEW_THREADS / 32; ++w) all += sh.order.before[w][threadIdx.x];
      }
      uint32_t base = sh.order.scan(all);
      sh.order.place(base);
#pragma unroll
      for (int i = 0; i < PER_THREAD; ++i)
        if (d[i] < RADIX) sh.sorted[sh.order.at(d[i], r[i])] = e[i];
      __syncthreads();
    }
  }

  // (the barriers above are also between the clearing and what is written to the same rows now, as is this wait for the launch before)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int piece = (found + STRANDS - 1) / STRANDS, begin = min(strand * piece, found), end = min(begin + piece, found);
  auto key = [&](int i) { return sh.sorted[i].x; };
  auto goes_on = [&](int at) { return at < found && key(at) == key(at - 1); };     // the run before `at`
  const bool starts_open = begin < end && begin > 0 && goes_on(begin);
  for (int tile = blockIdx.y; tile < p.tiles; tile += gridDim.y) {
    if (begin < end) {
      uint32_t id = key(begin);
      bool open = starts_open;
      float acc[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[c] = 0.0f;
      auto finish = [&](bool on) {
        if (open || on) {
          float* to = sh.part[open ? 0 : 1][strand];
#pragma unroll
          for (int c = 0; c < 8; ++c) to[WIDE ? lane * 8 + c : c * STRAND + lane] = acc[c];
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c) acc[c] *= p.scale;
          write(blockIdx.x + (int64_t)id * share, tile, acc);
        }
      };
      for (int i = begin; i < end; i += FLIGHT) {
        Raw8<T> rows[WIDE ? FLIGHT : 1];
        T single[WIDE ? 1 : FLIGHT][8];
#pragma unroll
        for (int j = 0; j < FLIGHT; ++j) {
          // (behind the piece its last row again, and of columns behind the end the last one: loads behind a branch would wait for one another)
          const T* from = (const T*)p.dy + (int64_t)sh.sorted[min(i + j, end - 1)].y * p.dy_stride;
          if constexpr (WIDE) {
            read8(from + min(column(tile, 0), (int64_t)p.D - 8), rows[j]);
          } else {
#pragma unroll
            for (int c = 0; c < 8; ++c) single[j][c] = from[min(column(tile, c), (int64_t)p.D - 1)];
          }
        }
#pragma unroll
        for (int j = 0; j < FLIGHT; ++j) {
          if (i + j >= end) break;
          if (key(i + j) != id) {
            finish(false);
            id = key(i + j);
            open = false;
#pragma unroll
            for (int c = 0; c < 8; ++c) acc[c] = 0.0f;
          }
          float f[8];
          if constexpr (WIDE) {
            unpack8(rows[j], f);
          } else {
#pragma unroll
            for (int c = 0; c < 8; ++c) f[c] = to_float(single[j][c]);
          }
#pragma unroll
          for (int c = 0; c < 8; ++c) acc[c] += f[c];
        }
      }
      finish(goes_on(end));
    }
    __syncthreads();
    // the strand in whose piece a run begins that goes on adds up its parts
    if (begin < end && goes_on(end) && !(starts_open && key(begin) == key(end - 1))) {
      const uint32_t id = key(end - 1);
      int last = end;                              // of the run
      for (int step = 1 << 12; step; step /= 2)
        if (last + step < found && key(last + step) == id) last += step;
      float a[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) a[c] = sh.part[1][strand][WIDE ? lane * 8 + c : c * STRAND + lane];
#pragma unroll 4
      for (int s = strand + 1; s <= last / piece; ++s) {
#pragma unroll
        for (int c = 0; c < 8; ++c) a[c] += sh.part[0][s][WIDE ? lane * 8 + c : c * STRAND + lane];
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) a[c] *= p.scale;
      write(blockIdx.x + (int64_t)id * share, tile, a);
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
  if (N <= FPB_EMBEDDING_FEW) {
    g.bytes = 16;                                  // (nothing in it)
    return g;
  }
  const int64_t subs = (N + SUB - 1) / SUB;
  g.subs = (int)((subs + MAX_TILES - 1) / MAX_TILES);
  g.tiles = (int)((subs + g.subs - 1) / g.subs);
  int bits = 1;
  while (V >> bits) ++bits;                        // of the ids and of V itself
  g.passes = (bits + RADIX_BITS - 1) / RADIX_BITS;
  g.bits = (bits + g.passes - 1) / g.passes;
  // Windows as long as leaves 1024 threads an SM, 32 rows at least: a frequent id's parts are joined one after another (32768 ids of 1024
  // columns: windows of 16 rows 58 us, of 32 55, of 64 53; 100000 ids: of 64 92, of 128 98; 262144: of 64 162, of 128 or 256 152).
  const int64_t columns = (D + 7) / 8;
  g.window = MAX_WINDOW;
  while (g.window > 32 && (N + g.window - 1) / g.window * columns < 148 * 1024) g.window /= 2;
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
  uint2* buffers[2] = {(uint2*)(space + g.sorted[0]), (uint2*)(space + g.sorted[1])};
  cudaError_t e = cudaSuccess;
  for (int pass = 0; pass < g.passes && e == cudaSuccess; ++pass) {
    s.in = pass == 0 ? nullptr : buffers[(pass - 1) & 1];
    s.out = buffers[pass & 1];
    s.shift = pass * g.bits;
    e = launch_kernel(digit_counts_kernel, dim3(g.tiles), TILE_THREADS, 0, pass > 0, s, stream);
    if (e == cudaSuccess) e = launch_kernel(scatter_kernel, dim3(g.tiles + (pass == 0 ? CLEARING : 0)), TILE_THREADS, 0, true, s, stream);
    *n_launched += 2;
  }
  q.sorted = buffers[(g.passes - 1) & 1];
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
    const dim3 joins((unsigned)(q.windows - 1), (unsigned)((q.D + JOIN_COLS - 1) / JOIN_COLS));
    e = launch_kernel(join_kernel<T>, joins, JOIN_THREADS, 0, true, q, stream);
    *n_launched += 1;
  }
  return e;
}

// The table of a few ids where their kernel would clear it in too many pieces.
__global__ void __launch_bounds__(TILE_THREADS) clear_kernel(const __grid_constant__ SortParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  clear_table<TILE_THREADS>(p, blockIdx.x, gridDim.x);
}

template <typename T, bool WIDE> cudaError_t few_grad(FewParams p, const SortParams& table, cudaStream_t stream, int* n_launched) {
  static std::atomic<bool> configured[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    if ((e = cudaFuncSetAttribute(few_grad_kernel<T, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(FewShared))) != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  p.tiles = (p.D + FEW_COLUMNS - 1) / FEW_COLUMNS;
  const int across = p.tiles < 148 ? p.tiles : 148;                // one CTA an SM
  p.share = (int32_t)std::min<int64_t>(148 / across, p.V);
  int bits = 1;
  while ((p.V - 1) / p.share >> bits) ++bits;
  p.passes = (bits + RADIX_BITS - 1) / RADIX_BITS;
  p.bits = (bits + p.passes - 1) / p.passes;
  // The kernel clears pieces of 64 columns, and saves the 3 to 4 us of a launch; many pieces are cleared faster in one stretch before it, those of
  // unaligned rows above all.  Between events around the call, cleared here and before: 20000 rows of 333 fp32 (120 thousand pieces) 24.6 and 24.6 us,
  // 50000 33 and 29, 100000 59 and 38, 10^6 rows of 7 bf16 37 and 16; whole vectors: 60000 rows of 1024 fp32 (10^6 pieces) 58 and 59, 10^6 rows
  // of 8 bf16 16 and 14, 10^7 66 and 34.
  p.clears = p.V * p.tiles <= (WIDE ? 1 << 20 : 1 << 17);
  if (!p.clears) {
    if ((e = launch_kernel(clear_kernel, dim3(CLEARING), TILE_THREADS, 0, false, table, stream)) != cudaSuccess) return e;
    *n_launched += 1;
  }
  *n_launched += 1;
  return launch_kernel(few_grad_kernel<T, WIDE>, dim3((unsigned)p.share, (unsigned)across), FEW_THREADS, sizeof(FewShared), !p.clears, p, stream);
}

template <typename T>
cudaError_t lookup(LookupParams p, bool wide, cudaStream_t stream) {
  p.units = wide ? p.D / 8 : p.D;
  p.log_threads = 0;
  while ((1 << p.log_threads) < p.units && p.log_threads < 8) ++p.log_threads;
  const int rows = (THREADS >> p.log_threads) * ROWS;
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
  const int size = dtype == FPB_BF16 ? 2 : 4, vec = 16 / size;
  const bool wide = D % 8 == 0 && (N <= 1 || dy_stride % vec == 0) && ((uintptr_t)dy | (uintptr_t)dw) % 16 == 0;
  SortParams s{};
  s.tokens = tokens; s.N = N; s.V = V; s.padding = padding;
  s.tiles = g.tiles; s.subs = g.subs; s.bits = g.bits;
  s.counts = (uint32_t*)((char*)workspace + g.counts);
  const int64_t bytes = V * D * size;
  s.element = size;
  s.zero = (uint4*)dw;
  s.zero_units = (uintptr_t)dw % 16 == 0 ? bytes / 16 : 0;
  s.zero_tail = (char*)dw + s.zero_units * 16;
  s.zero_elements = (bytes - s.zero_units * 16) / size;
  *n_launched = 0;
  if (N <= FPB_EMBEDDING_FEW) {
    const FewParams p{tokens, dy, dy_stride, dw, V, padding, (int32_t)N, D, 1, 1, 1, 1, 1, scale};
    const cudaError_t e = dtype == FPB_BF16 ? (wide ? few_grad<__nv_bfloat16, true>(p, s, stream, n_launched) : few_grad<__nv_bfloat16, false>(p, s, stream, n_launched))
                                            : (wide ? few_grad<float, true>(p, s, stream, n_launched) : few_grad<float, false>(p, s, stream, n_launched));
    return e == cudaSuccess ? FPB_OK : FPB_ERR_LAUNCH;
  }
  SumParams q{};
  q.dy = dy; q.dy_stride = dy_stride; q.dw = dw; q.partial = (float*)((char*)workspace + g.partial);
  q.N = N; q.windows = g.windows; q.V = (uint32_t)V; q.D = D; q.pitch = (int32_t)g.pitch; q.W = g.window; q.scale = scale;
  const cudaError_t e = dtype == FPB_BF16 ? table_grad<__nv_bfloat16>(g, s, q, wide, (char*)workspace, stream, n_launched)
                                          : table_grad<float>(g, s, q, wide, (char*)workspace, stream, n_launched);
  return e == cudaSuccess ? FPB_OK : FPB_ERR_LAUNCH;
}

}  // namespace fpb
