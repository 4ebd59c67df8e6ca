// Kernel-side parameter blocks, launchers and shared device code of the
// selective state-space operators: the short causal convolution, the scan and
// the (gated) layer norm.  Internal to libttt_amd.so.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/ttt_amd.h"
#include "ttt_tile.h"

namespace ttt {

// ---------------------------------------------------------------- parameters
struct ConvParams {
  const void *x, *state;  // [B*L][ldx], [B][W-1][C] (may be null: zeros)
  const float *w, *bias;  // [C][W], [C] (may be null)
  void *y, *last;         // [B*L][C], [B][W-1][C] (may be null)
  const void *dy, *dlast; // as y and last (either may be null)
  void *dx, *dstate;      // [B*L][C], [B][W-1][C] (may be null)
  float* partial;         // [parts][W+1][C] sums of dw and dbias
  float *dw, *dbias;      // [C][W], [C]
  int B, L, C, W;
  long long ldx, ldy;     // (the step: rows of x; y's rows are C long)
  bool silu;
};
hipError_t launch_conv_fwd(const ConvParams& p, int dtype, hipStream_t stream);
hipError_t launch_conv_bwd(const ConvParams& p, int dtype, hipStream_t stream);
hipError_t launch_conv_step(const ConvParams& p, int dtype, hipStream_t stream);
int conv_bwd_parts(int B, int L, int C);

struct NormParams {
  const void *x, *gate;  // [R][ldx], [R][ldg] (gate may be null)
  const float *w, *b;    // [D] (both or neither)
  void* y;               // [R][D]
  float* stats;          // [R][2]: mean and 1/sigma
  const void* dy;        // [R][D]
  void *dx, *dgate;      // [R][D]
  float* partial;        // [parts][2][D]
  float *dw, *db;        // [D]
  long long R, ldx, ldg;
  int D;
  float eps;
};
constexpr int kNormMaxD = 16384;  // 16 values to each of a row's 1,024 lanes
hipError_t launch_norm_fwd(const NormParams& p, int dtype, hipStream_t stream);
hipError_t launch_norm_bwd(const NormParams& p, int dtype, hipStream_t stream);
int norm_bwd_parts(long long R, int D);

// ---------------------------------------------------------------- rows of any alignment
// V (4 or 8) consecutive elements of a row, one load where all are there.  Rows of odd
// length start at any multiple of the element's size: the loads and stores are declared
// so aligned, which the vector memory takes.
template <typename T, int V> struct RowVec {
  typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};
// raw elements of the row's columns [0, n) from p, zeros behind them
template <typename T, int V> struct Raw {
  typename RowVec<T, V>::type v;
  __device__ __forceinline__ void load(const T* __restrict__ p, int n) {
    if (n >= V) {
      v = *reinterpret_cast<const typename RowVec<T, V>::type*>(p);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = e < n ? p[e] : (T)0.0f;
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (T)0.0f;
  }
  __device__ __forceinline__ float f(int e) const { return (float)v[e]; }
  __device__ __forceinline__ void store(T* __restrict__ p, int n) const {
    if (n >= V) {
      *reinterpret_cast<typename RowVec<T, V>::type*>(p) = v;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < n) p[e] = v[e];
    }
  }
};
// V values, rounded to T
template <typename T, int V> __device__ __forceinline__ void store_row(T* __restrict__ p, int n, const float (&v)[V]) {
  Raw<T, V> r;
#pragma unroll
  for (int q = 0; q < V; q += 4) {
    const auto a = to_frag<T>(f4{v[q], v[q + 1], v[q + 2], v[q + 3]}).v;
#pragma unroll
    for (int e = 0; e < 4; ++e) r.v[q + e] = a[e];
  }
  r.store(p, n);
}

// 1 / (1 + e^-z): e^-z overflows to inf for z < -88, whose reciprocal is the 0 that is meant
__device__ __forceinline__ float sigmoid_f(float z) {
  return rcp_f(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z));
}

// A workgroup of 256 sums `parts` rows of n partial sums: thread t has column i, shared by
// the threads t, t + 16, .., and every 16th row; threads 0..15 return the sums, which
// do not depend on anything but their order here.
__device__ __forceinline__ float sum_parts(const float* __restrict__ part, long long n, long long i, int parts) {
  __shared__ float red[16][17];
  const int g = threadIdx.x >> 4, c = threadIdx.x & 15;
  constexpr int AT_ONCE = 8;
  float s[AT_ONCE] = {};
  if (i < n) {
    int q = g;
    for (; q + 16 * (AT_ONCE - 1) < parts; q += 16 * AT_ONCE)
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) s[k] += part[(long long)(q + 16 * k) * n + i];
#pragma unroll
    for (int k = 0; k < AT_ONCE - 1; ++k)
      if (q + 16 * k < parts) s[k] += part[(long long)(q + 16 * k) * n + i];
  }
  red[g][c] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  float v = 0.f;
  if (threadIdx.x < 16)
#pragma unroll
    for (int k = 0; k < 16; ++k) v += red[k][c];
  return v;
}

}  // namespace ttt
