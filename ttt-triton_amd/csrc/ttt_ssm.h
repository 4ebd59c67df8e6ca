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
constexpr int kNormMaxD = 16384;
hipError_t launch_norm_fwd(const NormParams& p, int dtype, hipStream_t stream);
hipError_t launch_norm_bwd(const NormParams& p, int dtype, hipStream_t stream);
int norm_bwd_parts(long long R, int D);

// ---------------------------------------------------------------- rows of any alignment
// Eight consecutive elements of a row, 16 bytes a load where all eight are
// there.  Rows of odd length start at any multiple of the element's size: the
// loads and stores are declared so aligned, which the vector memory takes.
typedef unsigned u4v __attribute__((ext_vector_type(4)));
template <typename T> struct RowVec;
template <> struct RowVec<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8), aligned(2)));
};
template <> struct RowVec<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8), aligned(2)));
};
template <> struct RowVec<float> {
  typedef float v8 __attribute__((ext_vector_type(8), aligned(4)));
};

// raw elements of the row's columns [0, n) from p, zeros behind them
template <typename T> struct Raw8 {
  T v[8];
  __device__ __forceinline__ void load(const T* __restrict__ p, int n) {
    if (n >= 8) {
      const typename RowVec<T>::v8 x = *reinterpret_cast<const typename RowVec<T>::v8*>(p);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = x[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : (T)0.0f;
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (T)0.0f;
  }
  __device__ __forceinline__ float f(int e) const { return (float)v[e]; }
};
template <typename T> __device__ __forceinline__ void store8(T* __restrict__ p, int n, const float (&v)[8]) {
  const auto a = to_frag<T>(f4{v[0], v[1], v[2], v[3]}).v, b = to_frag<T>(f4{v[4], v[5], v[6], v[7]}).v;
  if (n >= 8) {
    typename RowVec<T>::v8 x = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    *reinterpret_cast<typename RowVec<T>::v8*>(p) = x;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = e < 4 ? a[e] : b[e - 4];
  }
}
template <typename T> __device__ __forceinline__ void store8(T* __restrict__ p, int n, const Raw8<T>& r) {
  if (n >= 8) {
    typename RowVec<T>::v8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = r.v[e];
    *reinterpret_cast<typename RowVec<T>::v8*>(p) = x;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = r.v[e];
  }
}

// 1 / (1 + e^-z): e^-z overflows to inf for z < -88, whose reciprocal is the 0 that is meant
__device__ __forceinline__ float sigmoid_f(float z) {
  return rcp_f(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z));
}

}  // namespace ttt
