// The norms around a block, forwards (mathematics: ttt_block_norm.h).
#include <math.h>

#include <algorithm>

#include "ttt_block_norm.h"

namespace ttt {

namespace {

template <typename T, typename TR, int LANES, int V, int NCH>
__global__ __launch_bounds__(block_threads(LANES)) void block_norm_fwd_kernel(BlockNormParams p) {
  constexpr bool RES = !__is_same(TR, NoResidual);
  typedef typename ResidualOf<TR, T>::type R;
  constexpr int ROWS = block_threads(LANES) / LANES;
  const int l = threadIdx.x & (LANES - 1), D = p.D;
  __shared__ float red[8];
  const long long row = (long long)blockIdx.x * ROWS + threadIdx.x / LANES;
  if (row >= p.R) return;  // the lanes of a row together; never a part of a workgroup with one row
  const long long outer = p.heads == 1 ? row : row / p.heads, in = p.heads == 1 ? 0 : (row - outer * p.heads) * D;
  float n[NCH][V];
  Raw<R, V> res[NCH];
  Raw<T, V> z[NCH];
  {
    Raw<T, V> x[NCH];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = V * (LANES * i + l), left = D - c;
      x[i].zero();
      res[i].zero();
      z[i].zero();
      if (left > 0) {
        x[i].load(static_cast<const T*>(p.x) + outer * p.ldx + in + c, left);
        if (RES) res[i].load(static_cast<const R*>(p.res) + outer * p.ldr + in + c, left);
        if (p.gate != nullptr) z[i].load(static_cast<const T*>(p.gate) + outer * p.ldg + in + c, left);
      }
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        n[i][e] = x[i].f(e);
        s = __builtin_fmaf(n[i][e], n[i][e], s);
      }
    float inv = 1.f;
    if (p.w != nullptr) inv = 1.0f / sqrtf(share_sum<LANES>(s, red) / (float)D + p.eps);
    if (l == 0 && p.stats != nullptr) p.stats[2 * row] = inv;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = V * (LANES * i + l), left = D - c;
      if (p.w != nullptr && left > 0) {
        Raw<float, V> w;
        w.load(p.w + c, left);
#pragma unroll
        for (int e = 0; e < V; ++e) n[i][e] *= inv * w.v[e];
      }
    }
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = V * (LANES * i + l), left = D - c;
    if (left > 0) {
      if (p.gate != nullptr) {
#pragma unroll
        for (int e = 0; e < V; ++e) n[i][e] *= z[i].f(e) * sigmoid_f(z[i].f(e));
      }
      if (p.s != nullptr) {
        Raw<float, V> k;
        k.load(p.s + c, left);
#pragma unroll
        for (int e = 0; e < V; ++e) n[i][e] *= k.v[e];
      }
      if (RES) {
#pragma unroll
        for (int e = 0; e < V; ++e) n[i][e] += res[i].f(e);
      }
      store_row<R, V>(static_cast<R*>(p.r) + row * D + c, left, n[i]);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < left) s = __builtin_fmaf(n[i][e], n[i][e], s);
    }
  }
  if (!RES || p.w2 == nullptr) return;
  const float inv = 1.0f / sqrtf(share_sum<LANES>(s, red) / (float)D + p.eps);
  if (l == 0 && p.stats != nullptr) p.stats[2 * row + 1] = inv;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = V * (LANES * i + l), left = D - c;
    if (left > 0) {
      Raw<float, V> w;
      w.load(p.w2 + c, left);
#pragma unroll
      for (int e = 0; e < V; ++e) n[i][e] *= inv * w.v[e];
      store_row<T, V>(static_cast<T*>(p.y) + row * D + c, left, n[i]);
    }
  }
}

template <typename T, typename TR> struct Fwd {
  template <int LANES, int V, int NCH> struct Of {
    static hipError_t run(const BlockNormParams& p, hipStream_t stream) {
      typedef typename ResidualOf<TR, T>::type R;
      constexpr int NT = block_threads(LANES), ROWS = NT / LANES;
      const long long most = 0xffffffffLL / NT * ROWS / p.heads * p.heads;  // of a launch: 2^32 threads
      for (long long r0 = 0; r0 < p.R; r0 += most) {
        BlockNormParams q = p;
        const long long o0 = r0 / p.heads;
        q.R = std::min(most, p.R - r0);
        q.x = static_cast<const T*>(p.x) + o0 * p.ldx;
        if (p.gate != nullptr) q.gate = static_cast<const T*>(p.gate) + o0 * p.ldg;
        if (p.res != nullptr) q.res = static_cast<const R*>(p.res) + o0 * p.ldr;
        q.r = static_cast<R*>(p.r) + r0 * p.D;
        if (p.y != nullptr) q.y = static_cast<T*>(p.y) + r0 * p.D;
        if (p.stats != nullptr) q.stats = p.stats + 2 * r0;
        hipLaunchKernelGGL((block_norm_fwd_kernel<T, TR, LANES, V, NCH>), dim3((unsigned)((q.R + ROWS - 1) / ROWS)),
                           dim3(NT), 0, stream, q);
      }
      return hipGetLastError();
    }
  };
};
template <typename T, typename TR> hipError_t run_t(const BlockNormParams& p, hipStream_t s) {
  return by_width<Fwd<T, TR>::template Of>(p.D, p, s);
}
template <typename T> hipError_t residual_t(const BlockNormParams& p, int dtype, int res_dtype, hipStream_t s) {
  if (res_dtype < 0) return run_t<T, NoResidual>(p, s);
  if (res_dtype == dtype) return run_t<T, T>(p, s);
  if constexpr (sizeof(T) == 2) return run_t<T, float>(p, s);
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_block_norm_fwd(const BlockNormParams& p, int dtype, int res_dtype, hipStream_t s) {
  return dtype == TTT_DTYPE_BF16 ? residual_t<__bf16>(p, dtype, res_dtype, s)
         : dtype == TTT_DTYPE_F16 ? residual_t<_Float16>(p, dtype, res_dtype, s)
                                  : residual_t<float>(p, dtype, res_dtype, s);
}

}  // namespace ttt
