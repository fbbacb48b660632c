// Norms of queries and keys over each head, with the position rotation in the same pass, and their gradients.
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  y = R (n w)          R: rotation of the channel pairs (2i, 2i+1) by the token's phasors
//   g = R^T dy,  dw = sum over all rows of g n,  dx = r (g w - n mean(g w n))
// fp32 arithmetic on bf16 or fp32 tensors; bound by HBM: forward one read and one write, backward two reads and one write.
//
// A row (token, head) of d <= 256 channels belongs to d / 8 lanes, a power of two of them set aside, eight channels each: a lane
// keeps its channels' weights for the whole launch.  A group of lanes takes HEADS heads of a token, which share its phasors, and
// moves from token to token by adding strides; the arithmetic runs on pairs of floats.  Issue slots and loads in flight both count: with
// one head at a time, an index worked out for every row and scalar arithmetic 32768 tokens of 8 + 8 heads of 128 took 78 us forward
// and 112 backward, with two heads, strides and pairs 58 and 103 (cold and dirty caches; 64 registers: 4 CTAs an SM; left to itself
// the compiler takes 102 and 144, and 75 and 155 us).  fp32 rows need more registers and fewer of them in flight.
#include "fpb_common.cuh"
#include "vec_io.cuh"

namespace fpb {
namespace {

constexpr int THREADS = 256, ROUNDS = 8;      // tokens in a row, at most

struct QkNormParams {
  SeqView x[2], dy[2], out[2];      // queries, keys: input, upstream gradient (backward), result
  const float* w[2];                // d weights each, null: ones
  const float2* phasors;            // (rows, T, d/2), null: no rotation
  int64_t ph_sb;                    // in float2 units, 0: one table for all batch rows
  float* partial;                   // backward: (CTAs, 2, d) sums of the weights' gradients
  int32_t B, T, H[2], d, rounds;    // rounds: tokens in a row
  float eps, inv_d;
};

// sum over the row's lanes
template <int L> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Eight channels as (first of a channel pair) x 4, (second) x 4.
struct Eight {
  Pair a[2], b[2];
};
__device__ __forceinline__ Eight split(const float (&f)[8]) {
  return Eight{{pair(f[0], f[2]), pair(f[4], f[6])}, {pair(f[1], f[3]), pair(f[5], f[7])}};
}
__device__ __forceinline__ void together(const Eight& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 a = both(v.a[i]), b = both(v.b[i]);
    f[4 * i] = a.x; f[4 * i + 1] = b.x; f[4 * i + 2] = a.y; f[4 * i + 3] = b.y;
  }
}
// each element times one number; elementwise products and sums; the sum of products
__device__ __forceinline__ Eight times(const Eight& x, float f) {
  const Pair p = pair(f, f);
  return Eight{{x.a[0] * p, x.a[1] * p}, {x.b[0] * p, x.b[1] * p}};
}
__device__ __forceinline__ Eight times(const Eight& x, const Eight& y) {
  return Eight{{x.a[0] * y.a[0], x.a[1] * y.a[1]}, {x.b[0] * y.b[0], x.b[1] * y.b[1]}};
}
__device__ __forceinline__ Eight plus_times(const Eight& z, const Eight& x, const Eight& y) {
  return Eight{{fma(x.a[0], y.a[0], z.a[0]), fma(x.a[1], y.a[1], z.a[1])}, {fma(x.b[0], y.b[0], z.b[0]), fma(x.b[1], y.b[1], z.b[1])}};
}
__device__ __forceinline__ Eight plus_times(const Eight& z, const Eight& x, float f) {
  const Pair p = pair(f, f);
  return Eight{{fma(x.a[0], p, z.a[0]), fma(x.a[1], p, z.a[1])}, {fma(x.b[0], p, z.b[0]), fma(x.b[1], p, z.b[1])}};
}
__device__ __forceinline__ float dot(const Eight& x, const Eight& y) {
  const float2 s = both(fma(x.b[1], y.b[1], fma(x.b[0], y.b[0], fma(x.a[1], y.a[1], x.a[0] * y.a[0]))));
  return s.x + s.y;
}
// rotated by the angles whose (cos, sin) are c, s; `minus`: -s
__device__ __forceinline__ Eight rotate(const Eight& x, const Pair (&c)[2], const Pair (&s)[2], const Pair (&minus)[2]) {
  Eight y;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    y.a[i] = fma(x.b[i], minus[i], x.a[i] * c[i]);
    y.b[i] = fma(x.b[i], c[i], x.a[i] * s[i]);
  }
  return y;
}

// eight elements of the packed word `w` (two bf16 or one fp32)
__device__ __forceinline__ void fill8(Raw8<__nv_bfloat16>& r, uint32_t w) { r.a = make_uint4(w, w, w, w); }
__device__ __forceinline__ void fill8(Raw8<float>& r, uint32_t w) { r.a = r.b = make_uint4(w, w, w, w); }

template <typename T, int L, int HEADS, bool BWD>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 4 ? 2 : 4) qk_norm_kernel(const __grid_constant__ QkNormParams p) {
  constexpr int GROUPS = THREADS / L;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");        // (the sum over the backward's slabs)
  const int which = blockIdx.y, H = p.H[which];
  const SeqView vx = p.x[which], vg = p.dy[which], vo = p.out[which];
  const int group = threadIdx.x / L, lane = threadIdx.x % L, c0 = lane * 8;
  const bool live = c0 < p.d;
  // What stands for a row that is not there: ones, whose r is finite without eps too, under a gradient of zeros; lanes behind d add nothing.
  const uint32_t blank = live ? (sizeof(T) == 2 ? 0x3f803f80u : 0x3f800000u) : 0u;
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = live && p.w[which] ? p.w[which][c0 + e] : 1.0f;
  const Eight w = split(f);
  const Pair zero = pair(0.0f, 0.0f);
  Eight dw{{zero, zero}, {zero, zero}};

  // A CTA takes items of (batch row, stretch of tokens, block of heads).
  const int sets = (H + HEADS - 1) / HEADS, block = min(sets, GROUPS), per = block ? GROUPS / block : 1;      // groups of heads; tokens at a time
  const int blocks = block ? (sets + block - 1) / block : 0, stretch = per * p.rounds, stretches = (p.T + stretch - 1) / stretch;
  const int64_t items = (int64_t)p.B * stretches * blocks;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t rest = item / blocks;
    const int b = (int)(rest / stretches), t0 = (int)(rest % stretches) * stretch + group / block;
    const int h = ((int)(item % blocks) * block + group % block) * HEADS;
    const int heads = live && group < per * block ? min(H - h, HEADS) : 0, tokens = (p.T - t0 + per - 1) / per;      // (those left; `rounds` at most)
    const T* x_at = (const T*)vx.data + b * vx.sb + t0 * vx.st + h * vx.sh + c0;
    const T* g_at = BWD ? (const T*)vg.data + b * vg.sb + t0 * vg.st + h * vg.sh + c0 : nullptr;
    T* o_at = (T*)vo.data + b * vo.sb + t0 * vo.st + h * vo.sh + c0;
    const float4* ph_at = reinterpret_cast<const float4*>(p.phasors + b * p.ph_sb + (int64_t)t0 * (p.d / 2) + lane * 4);
    const int64_t x_step = per * vx.st, g_step = BWD ? per * vg.st : 0, o_step = per * vo.st;
    const int ph_step = per * (p.d / 4);
#pragma unroll 1
    for (int n = 0; n < p.rounds; ++n) {
      if (n * per + (int)(rest % stretches) * stretch >= p.T) break;          // (no token left for any group)
      const bool here = n < tokens;
      Raw8<T> rx[HEADS], rg[BWD ? HEADS : 1];
      float4 u = make_float4(1.0f, 0.0f, 1.0f, 0.0f), v = u;
#pragma unroll
      for (int j = 0; j < HEADS; ++j) {
        fill8(rx[j], blank);
        if constexpr (BWD) rg[j] = Raw8<T>{};
        if (here && j < heads) {
          read8(x_at + j * vx.sh, rx[j]);
          if constexpr (BWD) read8(g_at + j * vg.sh, rg[j]);
        }
      }
      if (p.phasors && here && heads > 0) { u = __ldg(ph_at); v = __ldg(ph_at + 1); }
      const Pair c[2] = {pair(u.x, u.z), pair(v.x, v.z)}, s[2] = {pair(u.y, u.w), pair(v.y, v.w)}, minus[2] = {pair(-u.y, -u.w), pair(-v.y, -v.w)};
#pragma unroll
      for (int j = 0; j < HEADS; ++j) {
        unpack8(rx[j], f);
        const Eight x = split(f);
        float sq = dot(x, x);
        Eight y;
        if constexpr (BWD) {
          unpack8(rg[j], f);
          const Eight g = rotate(split(f), c, minus, s), gw = times(g, w);     // back through the rotation, then the weights
          const float along = group_sum<L>(dot(gw, x));
          const float r = rsqrtf(group_sum<L>(sq) * p.inv_d + p.eps), m = -along * r * r * p.inv_d;       // -r mean(g w n), as n = x r
          dw = plus_times(dw, g, times(x, r));
          y = times(plus_times(gw, x, m), r);
        } else {
          const float r = rsqrtf(group_sum<L>(sq) * p.inv_d + p.eps);
          y = rotate(times(times(x, r), w), c, s, minus);
        }
        together(y, f);
        if (here && j < heads) store8(o_at + j * vo.sh, f);
      }
      x_at += x_step; o_at += o_step; ph_at += ph_step;
      if constexpr (BWD) g_at += g_step;
    }
  }
  if constexpr (BWD) {
    // the CTA's sums, group after group in a fixed order
    __shared__ float sums[GROUPS][L * 8 + 1];
    together(dw, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[group][lane + e * L] = f[e];               // (lanes next to one another: no bank twice)
    __syncthreads();
    for (int i = threadIdx.x; i < L * 8; i += THREADS) {
      float a = 0.0f;
#pragma unroll 4
      for (int q = 0; q < GROUPS; ++q) a += sums[q][i];
      const int ch = (i % L) * 8 + i / L;
      if (ch < p.d) p.partial[((int64_t)blockIdx.x * 2 + which) * p.d + ch] = a;
    }
  }
}

struct QkSumParams {
  const float* partial;
  float* dw[2];
  int32_t d, slabs;
};
// A CTA sums 32 of the 2 d columns, a warp every 32nd slab (eight warps took 11 us for 592 slabs: each load waited for the eight before).
constexpr int SUM_WARPS = 32, AT_ONCE = (FPB_QK_NORM_SLABS + SUM_WARPS - 1) / SUM_WARPS;
__global__ void __launch_bounds__(32 * SUM_WARPS) qk_weight_sums_kernel(const __grid_constant__ QkSumParams p) {
  __shared__ float part[SUM_WARPS][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane;
  float v[AT_ONCE], s = 0.0f;
#pragma unroll
  for (int i = 0; i < AT_ONCE; ++i) {
    const int n = warp + i * SUM_WARPS;
    v[i] = c < 2 * p.d && n < p.slabs ? p.partial[(int64_t)n * 2 * p.d + c] : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < AT_ONCE; ++i) s += v[i];
  part[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < 2 * p.d) {
#pragma unroll 8
    for (int n = 1; n < SUM_WARPS; ++n) s += part[n][lane];
    float* to = c < p.d ? p.dw[0] : p.dw[1];
    if (to) to[c < p.d ? c : c - p.d] = s;
  }
}

template <typename T, int HEADS, bool BWD>
cudaError_t launch(QkNormParams p, cudaStream_t stream, int* slabs) {
  int lanes = 1;
  while (lanes * 8 < p.d) lanes *= 2;
  const int groups = THREADS / lanes, H = p.H[0] > p.H[1] ? p.H[0] : p.H[1], sets = (H + HEADS - 1) / HEADS, block = sets < groups ? sets : groups;
  // as many tokens in a row as leave four CTAs an SM over both tensors
  int64_t items;
  for (p.rounds = ROUNDS;; p.rounds /= 2) {
    const int stretch = groups / block * p.rounds;
    items = (int64_t)p.B * ((p.T + stretch - 1) / stretch) * ((sets + block - 1) / block);
    if (items >= FPB_QK_NORM_SLABS / 2 || p.rounds == 1) break;
  }
  // at most eight CTAs an SM over both tensors; the backward's leave a slab of sums each
  const dim3 grid((unsigned)(items < FPB_QK_NORM_SLABS ? items : FPB_QK_NORM_SLABS), 2);
  *slabs = (int)grid.x;
  switch (lanes) {
    case 1: return launch_kernel(qk_norm_kernel<T, 1, HEADS, BWD>, grid, THREADS, 0, false, p, stream);
    case 2: return launch_kernel(qk_norm_kernel<T, 2, HEADS, BWD>, grid, THREADS, 0, false, p, stream);
    case 4: return launch_kernel(qk_norm_kernel<T, 4, HEADS, BWD>, grid, THREADS, 0, false, p, stream);
    case 8: return launch_kernel(qk_norm_kernel<T, 8, HEADS, BWD>, grid, THREADS, 0, false, p, stream);
    case 16: return launch_kernel(qk_norm_kernel<T, 16, HEADS, BWD>, grid, THREADS, 0, false, p, stream);
    default: return launch_kernel(qk_norm_kernel<T, 32, HEADS, BWD>, grid, THREADS, 0, false, p, stream);
  }
}
template <typename T, bool BWD> cudaError_t launch(const QkNormParams& p, cudaStream_t stream, int* slabs) {
  return p.H[0] > 1 || p.H[1] > 1 ? launch<T, 2, BWD>(p, stream, slabs) : launch<T, 1, BWD>(p, stream, slabs);
}

}  // namespace

int launch_qk_norm(int dtype, bool backward, int B, int T, int Hq, int Hk, int d, float eps, const float* const w[2], const float* phasors,
                   int64_t phasor_stride_b, const SeqView x[2], const SeqView dy[2], const SeqView out[2], float* const dw[2], float* partial,
                   cudaStream_t stream) {
  QkNormParams p{};
  for (int k = 0; k < 2; ++k) { p.x[k] = x[k]; p.out[k] = out[k]; p.w[k] = w[k]; if (backward) p.dy[k] = dy[k]; }
  p.phasors = (const float2*)phasors; p.ph_sb = phasor_stride_b; p.partial = partial;
  p.B = B; p.T = T; p.H[0] = Hq; p.H[1] = Hk; p.d = d; p.eps = eps; p.inv_d = 1.0f / (float)d;
  cudaError_t e;
  int slabs = 0;
  if (!backward) {
    e = dtype == FPB_BF16 ? launch<__nv_bfloat16, false>(p, stream, &slabs) : launch<float, false>(p, stream, &slabs);
  } else {
    e = dtype == FPB_BF16 ? launch<__nv_bfloat16, true>(p, stream, &slabs) : launch<float, true>(p, stream, &slabs);
    if (e == cudaSuccess && (dw[0] || dw[1])) {
      const QkSumParams s{partial, {dw[0], dw[1]}, d, slabs};
      e = launch_kernel(qk_weight_sums_kernel, dim3((2 * d + 31) / 32), 32 * SUM_WARPS, 0, true, s, stream);
    }
  }
  return e == cudaSuccess ? FPB_OK : FPB_ERR_LAUNCH;
}

}  // namespace fpb
