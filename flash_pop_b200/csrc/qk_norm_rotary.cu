// Norms of queries and keys over each head, with the position rotation in the same pass, and their gradients.
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  y = R (n w)          R: rotation of the channel pairs (2i, 2i+1) by the token's phasors
//   g = R^T dy,  dw = sum over all rows of g n,  dx = r (g w - n mean(g w n))
// fp32 arithmetic on bf16 or fp32 tensors; bound by HBM: forward one read and one write, backward two reads and one write.
//
// A row (token, head) of d <= 256 channels belongs to d / 8 lanes, a power of two of them set aside, eight channels each; such
// a group of lanes walks over heads of one token - queries, then keys - so that the token's phasors (8 floats a lane) and
// the weights are read once for all of them.
#include "fpb_common.cuh"
#include "vec_io.cuh"

namespace fpb {
namespace {

constexpr int THREADS = 256, AHEAD = 4;       // heads a group has in flight

struct QkNormParams {
  SeqView x[2], dy[2], out[2];      // queries, keys: input, upstream gradient (backward), result
  const float* w[2];                // d weights each, null: ones
  const float2* phasors;            // (rows, T, d/2), null: no rotation
  int64_t ph_sb;                    // in float2 units, 0: one table for all batch rows
  float* partial;                   // backward: (CTAs, 2, d) sums of the weights' gradients
  int64_t tokens;                   // B T
  int32_t T, H[2], d;
  int32_t pieces, heads;            // a token's heads are shared out over `pieces` groups, `heads` to each
  float eps, inv_d;
};

template <int L> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ void rotate(float (&v)[8], const float (&c)[4], const float (&s)[4], float sign) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = v[2 * i], b = v[2 * i + 1], t = sign * s[i];
    v[2 * i] = a * c[i] - b * t;
    v[2 * i + 1] = a * t + b * c[i];
  }
}

template <typename T, int L, bool BWD>
__global__ void __launch_bounds__(THREADS) qk_norm_kernel(const __grid_constant__ QkNormParams p) {
  constexpr int GROUPS = THREADS / L;
  const int group = threadIdx.x / L, lane = threadIdx.x % L, c0 = lane * 8;
  const bool live = c0 < p.d;
  float w[2][8], dw[2][8];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[k][e] = live && p.w[k] ? p.w[k][c0 + e] : 1.0f;
      dw[k][e] = 0.0f;
    }
  const int64_t items = p.tokens * p.pieces, stride = (int64_t)gridDim.x * GROUPS;
  const int64_t rounds = (items + stride - 1) / stride;           // (the same for all groups: the shuffles below need whole warps)
  const int both = p.H[0] + p.H[1];
  for (int64_t n = 0; n < rounds; ++n) {
    const int64_t item = n * stride + (int64_t)blockIdx.x * GROUPS + group;
    const bool here = item < items;
    const int64_t token = here ? item / p.pieces : 0;
    const int first = here ? (int)(item % p.pieces) * p.heads : 0, end = here ? min(first + p.heads, both) : 0;
    const int64_t b = token / p.T, t = token % p.T;
    float c[4], s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { c[i] = 1.0f; s[i] = 0.0f; }
    if (p.phasors && live && here) {
      const float4* ph = reinterpret_cast<const float4*>(p.phasors + b * p.ph_sb + t * (p.d / 2) + lane * 4);
      const float4 u = __ldg(ph), v = __ldg(ph + 1);
      c[0] = u.x; s[0] = u.y; c[1] = u.z; s[1] = u.w; c[2] = v.x; s[2] = v.y; c[3] = v.z; s[3] = v.w;
    }
    for (int h0 = 0; h0 < p.heads; h0 += AHEAD) {
      Raw8<T> rx[AHEAD], rg[BWD ? AHEAD : 1];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int h = first + h0 + j;
        if (h < end && live) {
          const int k = h >= p.H[0];
          const int64_t hh = k ? h - p.H[0] : h;
          read8((const T*)p.x[k].data + b * p.x[k].sb + t * p.x[k].st + hh * p.x[k].sh + c0, rx[j]);
          if constexpr (BWD) read8((const T*)p.dy[k].data + b * p.dy[k].sb + t * p.dy[k].st + hh * p.dy[k].sh + c0, rg[j]);
        } else {
          rx[j] = Raw8<T>{};
          if constexpr (BWD) rg[j] = Raw8<T>{};
        }
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int h = first + h0 + j, k = h >= p.H[0];
        float x[8], g[8];
        unpack8(rx[j], x);
        float sq = 0.0f, dot = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sq += x[e] * x[e];
        if constexpr (BWD) {
          unpack8(rg[j], g);
          rotate(g, c, s, -1.0f);
#pragma unroll
          for (int e = 0; e < 8; ++e) dot += g[e] * (k ? w[1][e] : w[0][e]) * x[e];
          dot = group_sum<L>(dot);
        }
        const float r = rsqrtf(group_sum<L>(sq) * p.inv_d + p.eps);
        if (!(h < end && live)) continue;
        float y[8];
        if constexpr (BWD) {
          const float m = dot * r * r * p.inv_d;                  // r mean(g w n), as n = x r
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float gn = g[e] * x[e] * r;
            if (k) dw[1][e] += gn; else dw[0][e] += gn;
            y[e] = r * (g[e] * (k ? w[1][e] : w[0][e]) - x[e] * m);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = x[e] * r * (k ? w[1][e] : w[0][e]);
          rotate(y, c, s, 1.0f);
        }
        const int64_t hh = k ? h - p.H[0] : h;
        store8((T*)p.out[k].data + b * p.out[k].sb + t * p.out[k].st + hh * p.out[k].sh + c0, y);
      }
    }
  }
  if constexpr (BWD) {
    // the CTA's sums, group after group in a fixed order
    __shared__ float sums[GROUPS][L * 8 + 1];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[group][lane + e * L] = dw[k][e];         // (lanes next to one another: no bank twice)
      __syncthreads();
      for (int i = threadIdx.x; i < L * 8; i += THREADS) {
        float a = 0.0f;
#pragma unroll 4
        for (int q = 0; q < GROUPS; ++q) a += sums[q][i];
        const int ch = (i % L) * 8 + i / L;
        if (ch < p.d) p.partial[((int64_t)blockIdx.x * 2 + k) * p.d + ch] = a;
      }
    }
  }
}

struct QkSumParams {
  const float* partial;
  float* dw[2];
  int32_t d, slabs;
};
// a CTA sums 32 of the 2 d columns, a warp every eighth slab
__global__ void __launch_bounds__(256) qk_weight_sums_kernel(const __grid_constant__ QkSumParams p) {
  __shared__ float part[8][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (c < 2 * p.d)
#pragma unroll 8
    for (int n = warp; n < p.slabs; n += 8) s += p.partial[(int64_t)n * 2 * p.d + c];
  part[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < 2 * p.d) {
#pragma unroll
    for (int n = 1; n < 8; ++n) s += part[n][lane];
    float* to = c < p.d ? p.dw[0] : p.dw[1];
    if (to) to[c < p.d ? c : c - p.d] = s;
  }
}

template <typename T, bool BWD>
cudaError_t launch(const QkNormParams& p, int ctas, cudaStream_t stream) {
  if (p.d <= 8) return launch_kernel(qk_norm_kernel<T, 1, BWD>, dim3(ctas), THREADS, 0, false, p, stream);
  if (p.d <= 16) return launch_kernel(qk_norm_kernel<T, 2, BWD>, dim3(ctas), THREADS, 0, false, p, stream);
  if (p.d <= 32) return launch_kernel(qk_norm_kernel<T, 4, BWD>, dim3(ctas), THREADS, 0, false, p, stream);
  if (p.d <= 64) return launch_kernel(qk_norm_kernel<T, 8, BWD>, dim3(ctas), THREADS, 0, false, p, stream);
  if (p.d <= 128) return launch_kernel(qk_norm_kernel<T, 16, BWD>, dim3(ctas), THREADS, 0, false, p, stream);
  return launch_kernel(qk_norm_kernel<T, 32, BWD>, dim3(ctas), THREADS, 0, false, p, stream);
}

}  // namespace

int launch_qk_norm(int dtype, bool backward, int B, int T, int Hq, int Hk, int d, float eps, const float* const w[2], const float* phasors,
                   int64_t phasor_stride_b, const SeqView x[2], const SeqView dy[2], const SeqView out[2], float* const dw[2], float* partial,
                   cudaStream_t stream) {
  QkNormParams p{};
  for (int k = 0; k < 2; ++k) { p.x[k] = x[k]; p.out[k] = out[k]; p.w[k] = w[k]; if (backward) p.dy[k] = dy[k]; }
  p.phasors = (const float2*)phasors; p.ph_sb = phasor_stride_b; p.partial = partial;
  p.tokens = (int64_t)B * T; p.T = T; p.H[0] = Hq; p.H[1] = Hk; p.d = d; p.eps = eps; p.inv_d = 1.0f / (float)d;
  int lanes = 1;
  while (lanes * 8 < d) lanes *= 2;
  const int groups = THREADS / lanes, most = FPB_QK_NORM_SLABS;
  // all heads of a token to one group where that leaves a group for every slot of the GPU, else four heads (one round of
  // loads), so that a few tokens spread over the SMs
  p.heads = p.tokens >= (int64_t)most * groups ? Hq + Hk : AHEAD;
  p.pieces = (Hq + Hk + p.heads - 1) / p.heads;
  const int64_t ctas = (p.tokens * p.pieces + groups - 1) / groups;
  const int grid = (int)(ctas < most ? ctas : most);
  cudaError_t e;
  if (!backward) {
    e = dtype == FPB_BF16 ? launch<__nv_bfloat16, false>(p, grid, stream) : launch<float, false>(p, grid, stream);
  } else {
    e = dtype == FPB_BF16 ? launch<__nv_bfloat16, true>(p, grid, stream) : launch<float, true>(p, grid, stream);
    if (e == cudaSuccess && (dw[0] || dw[1])) {
      const QkSumParams s{partial, {dw[0], dw[1]}, d, grid};
      e = launch_kernel(qk_weight_sums_kernel, dim3((2 * d + 31) / 32), 256, 0, false, s, stream);
    }
  }
  return e == cudaSuccess ? FPB_OK : FPB_ERR_LAUNCH;
}

}  // namespace fpb
