// Dropout whose mask is never stored, alone or added to a residual: y = [r +] keep ? x / (1 - p) : 0.  The mask comes from the
// counter-based generator Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011)
// under the call's 64-bit seed as its key, so the backward pass makes the same mask again from the seed alone.
// Element i has 16 bits: half word i % 8 (low halves first) of the four words of counter i / 8, and goes where they are below
// p in units of 2^-16.  16 bits instead of 32 halve the generator's work, which at 32 would bound the kernel (10 rounds of
// two wide products for four elements); what is kept is scaled by 1 / (1 - p) of the p that the 16 bits stand for, so
// the expectation is exact, and p itself is off by at most 2^-17.
#include <cmath>

#include "fpb_common.cuh"
#include "vec_io.cuh"

namespace fpb {
namespace {

constexpr int THREADS = 256;

struct DropoutParams {
  const void *x, *residual;
  void* y;
  const int64_t* seed;
  int64_t n;
  uint32_t threshold;          // 0 .. 65536
  float factor;
};

__device__ __forceinline__ uint4 philox(uint64_t counter, uint32_t k0, uint32_t k1) {
  uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = 0, c3 = 0;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0; c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1; c3 = (uint32_t)a;
    k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// GROUPS groups of eight elements a thread, a CTA's width apart.  WIDE: 16-byte accesses (pointers 16-byte aligned).
// Four groups share the generator's keys and have their loads in flight together: 33.5M bf16 elements 31 us instead of 37 with one (134 MB,
// 21 us at the copy rate), with a residual 39 either way (201 MB, 31 us).  Without one 64 % of the issue slots and two thirds of the copy rate are in use:
// neither is full, and which wait is the rest is not known.
constexpr int GROUPS = 4;
template <typename T, bool WIDE, bool RES>
__global__ void __launch_bounds__(THREADS) dropout_kernel(const __grid_constant__ DropoutParams p) {
  const int64_t first = (int64_t)blockIdx.x * (THREADS * GROUPS) + threadIdx.x;
  const T *x = (const T*)p.x, *r = (const T*)p.residual;
  T* y = (T*)p.y;
  Raw8<T> rx[GROUPS], rr[RES ? GROUPS : 1];
  if constexpr (WIDE) {
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) {
      const int64_t i0 = (first + j * THREADS) * 8;
      if (i0 + 8 > p.n) continue;
      read8(x + i0, rx[j]);
      if constexpr (RES) read8(r + i0, rr[j]);
    }
  }
  const uint64_t seed = (uint64_t)*p.seed;
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) {
    const int64_t group = first + j * THREADS, i0 = group * 8;
    if (i0 >= p.n) return;
    const bool whole = WIDE && i0 + 8 <= p.n;
    float v[8], s[8];
    if (whole) {
      unpack8(rx[j], v);
      if constexpr (RES) unpack8(rr[j], s);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = i0 + e < p.n ? to_float(x[i0 + e]) : 0.0f;
        if constexpr (RES) s[e] = i0 + e < p.n ? to_float(r[i0 + e]) : 0.0f;
      }
    }
    const uint4 w = philox((uint64_t)group, (uint32_t)seed, (uint32_t)(seed >> 32));
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t half = e & 1 ? words[e >> 1] >> 16 : words[e >> 1] & 0xffffu;
      v[e] = half >= p.threshold ? v[e] * p.factor : 0.0f;        // (selected, not multiplied: what goes leaves no NaN behind)
      if constexpr (RES) v[e] += s[e];
    }
    if (whole) {
      store8(y + i0, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i0 + e < p.n) y[i0 + e] = from_float<T>(v[e]);
    }
  }
}

template <typename T>
cudaError_t launch(const DropoutParams& p, bool wide, cudaStream_t stream) {
  const dim3 grid((unsigned)((p.n + 8 * THREADS * GROUPS - 1) / (8 * THREADS * GROUPS)));
  if (wide)
    return p.residual ? launch_kernel(dropout_kernel<T, true, true>, grid, THREADS, 0, false, p, stream)
                      : launch_kernel(dropout_kernel<T, true, false>, grid, THREADS, 0, false, p, stream);
  return p.residual ? launch_kernel(dropout_kernel<T, false, true>, grid, THREADS, 0, false, p, stream)
                    : launch_kernel(dropout_kernel<T, false, false>, grid, THREADS, 0, false, p, stream);
}

}  // namespace

int launch_dropout(int dtype, int64_t n, double prob, const int64_t* seed, const void* x, const void* residual, void* y, cudaStream_t stream) {
  const uint32_t threshold = (uint32_t)std::nearbyint(prob * 65536.0);
  const DropoutParams p{x, residual, y, seed, n, threshold, threshold < 65536 ? 65536.0f / (float)(65536 - threshold) : 0.0f};
  const bool wide = ((uintptr_t)x | (uintptr_t)residual | (uintptr_t)y) % 16 == 0;
  const cudaError_t e = dtype == FPB_BF16 ? launch<__nv_bfloat16>(p, wide, stream) : launch<float>(p, wide, stream);
  return e == cudaSuccess ? FPB_OK : FPB_ERR_LAUNCH;
}

}  // namespace fpb
