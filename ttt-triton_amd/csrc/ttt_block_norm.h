// The norms around a block with its gate and residual scale on gfx950: parameters and shared
// device code (ttt_block_norm_fwd.hip, ttt_block_norm_bwd.hip).
//
//   n = x i w,  i = 1/sqrt(mean x^2 + eps)      the norm after the block (or n = x)
//   r = residual + s n silu(z)                  residual, s and z where there are any
//   y = r j w2, j = 1/sqrt(mean r^2 + eps)      the norm before the next block, where wanted
// and backward, from the gradients dr and dy of r and y, with dn = D s silu(z):
//   D = dr + j (dy w2) - r j^3 mean(dy w2 r),   dresidual = D
//   dx = i (dn w) - x i^3 mean(dn w x),         dz = D s n silu'(z)
//   dw = sum dn x i,   ds = sum D n silu(z),    dw2 = sum dy r j
// The backward forms r again from x, z and the residual, the values that y was normed from,
// in place of reading the r that was stored, rounded: the bytes are the same.
//
// Both are bound by HBM (32,768 rows of 768 in bf16 with an fp32 residual and both norms: 60 us forward,
// 5.0 TB/s, and 95 back, 4.8 TB/s; with a gate, by heads of 64: 29 and 44, 5.2 and 5.7).  A row is read once and held in registers over its reductions, by
// 8 to 64 lanes of a wave or by 4 or 8 waves, so that few lanes' places are empty; a lane has
// 4, 8, 12 or 16 values of it.  Heads are rows side by side in a wider row.
#pragma once

#include "ttt_ssm.h"

namespace ttt {

struct BlockNormParams {
  const void *x, *gate, *res;  // [R/heads][ldx] and so on, `heads` rows of D in each (gate, res may be null)
  const float *w, *s, *w2;     // [D] each, or null
  void *r, *y;                 // [R][D]; y only with w2
  float* stats;                // [R][2]: i and j
  const void *dr, *dy;         // [R][D], or null for zeros
  void *dx, *dgate, *dres;     // [R][D]
  float* partial;              // [parts][3][D]: dw, ds, dw2 (may be null)
  float *dw, *ds, *dw2;        // [D], or null
  long long R, ldx, ldg, ldr;
  int D, heads;
  float eps;
};
constexpr int kBlockNormMaxD = 8192;
// res_dtype: the residual's type, or -1 without one
hipError_t launch_block_norm_fwd(const BlockNormParams& p, int dtype, int res_dtype, hipStream_t stream);
hipError_t launch_block_norm_bwd(const BlockNormParams& p, int dtype, int res_dtype, hipStream_t stream);
int block_norm_parts(long long R, int D, int waves = 3);

// lanes to a row
constexpr int block_lanes(int D) { return D <= 64 ? 8 : D <= 128 ? 16 : D <= 256 ? 32 : D <= 1024 ? 64 : D <= 4096 ? 256 : 512; }
constexpr int block_threads(int LANES) { return LANES < 256 ? 256 : LANES; }

// the sum over the lanes that share a row, in every one of them
template <int LANES> __device__ __forceinline__ float share_sum(float s, float* red) {
  if constexpr (LANES <= 64) {
#pragma unroll
    for (int m = 1; m < LANES; m *= 2) s += __shfl_xor(s, m);
    return s;
  } else {
    s = sum_wave(s);
    __syncthreads();  // the last sum's readers are done
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < LANES / 64; ++k) v += red[k];
    return v;
  }
}

struct NoResidual {};  // (in place of its type)
template <typename TR, typename T> struct ResidualOf { typedef TR type; };
template <typename T> struct ResidualOf<NoResidual, T> { typedef T type; };

// Calls f with the kernel's instantiation for rows of D values: F::run<LANES, V, NCH>
template <template <int, int, int> class F, typename... A> hipError_t by_width(int D, A&&... a) {
  const int lanes = block_lanes(D), four = (D + 4 * lanes - 1) / (4 * lanes);  // values to a lane, in fours
  switch (lanes) {
    case 8: return four == 1 ? F<8, 4, 1>::run(a...) : F<8, 8, 1>::run(a...);
    case 16: return F<16, 8, 1>::run(a...);
    case 32: return F<32, 8, 1>::run(a...);
    case 64: return four == 2 ? F<64, 8, 1>::run(a...) : four == 3 ? F<64, 4, 3>::run(a...) : F<64, 8, 2>::run(a...);
    case 256: return four == 2 ? F<256, 8, 1>::run(a...) : four == 3 ? F<256, 4, 3>::run(a...) : F<256, 8, 2>::run(a...);
    default: return four == 3 ? F<512, 4, 3>::run(a...) : F<512, 8, 2>::run(a...);
  }
}

}  // namespace ttt
