// Rows of an embedding table for token ids, scaled, and the table's gradient.
//   y[n] = scale W[t_n],   dW[v] = scale sum over { n : t_n = v } of dy[n]
// An id outside the table has a zero row and no part in the gradient, and so has the padding id in the gradient.
// Bound by HBM: forward reads the rows in use and writes N rows, backward reads N rows and writes the dense table.
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

struct GradParams {
  const int64_t* tokens;
  const void* dy; int64_t dy_stride;
  void* dw;
  int64_t N, V, padding;
  int32_t D;
  float scale;
};

// A CTA a row of the table: it looks through all ids, in order, for its own.
template <typename T>
__global__ void __launch_bounds__(THREADS) table_grad_kernel(const __grid_constant__ GradParams p) {
  __shared__ int64_t found[THREADS];
  __shared__ int count;
  const int64_t v = blockIdx.x;
  for (int c0 = 0; c0 < p.D; c0 += THREADS) {
    const int c = c0 + threadIdx.x;
    float sum = 0.0f;
    for (int64_t n0 = 0; n0 < p.N; n0 += THREADS) {
      const int64_t n = n0 + threadIdx.x;
      const bool mine = n < p.N && p.tokens[n] == v && v != p.padding;
      if (!__syncthreads_or(mine)) continue;
      // the matching positions in order
      for (int w = 0; w < THREADS / 32; ++w) {
        if (threadIdx.x == 0 && w == 0) count = 0;
        __syncthreads();
        if ((int)threadIdx.x >> 5 == w) {
          const unsigned all = __ballot_sync(0xffffffffu, mine);
          if (mine) found[count + __popc(all & ((1u << (threadIdx.x & 31)) - 1))] = n;
          __syncwarp();
          if ((threadIdx.x & 31) == 0) count += __popc(all);
        }
      }
      __syncthreads();
      if (c < p.D)
        for (int i = 0; i < count; ++i) sum += to_float(((const T*)p.dy)[found[i] * p.dy_stride + c]);
      __syncthreads();
    }
    if (c < p.D) ((T*)p.dw)[v * p.D + c] = from_float<T>(sum * p.scale);
  }
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

int64_t embedding_workspace(int64_t N, int64_t V, int D) { return N > 0 && V > 0 && D > 0 ? 16 : 0; }

int launch_embedding_grad(int dtype, int64_t N, int64_t V, int D, const int64_t* tokens, int64_t padding, float scale, const void* dy,
                          int64_t dy_stride, void* dw, void* workspace, cudaStream_t stream, int* n_launched) {
  const GradParams p{tokens, dy, dy_stride, dw, N, V, padding, D, scale};
  const cudaError_t e = dtype == FPB_BF16 ? launch_kernel(table_grad_kernel<__nv_bfloat16>, dim3((unsigned)V), THREADS, 0, false, p, stream)
                                          : launch_kernel(table_grad_kernel<float>, dim3((unsigned)V), THREADS, 0, false, p, stream);
  *n_launched = 1;
  return e == cudaSuccess ? FPB_OK : FPB_ERR_LAUNCH;
}

}  // namespace fpb
