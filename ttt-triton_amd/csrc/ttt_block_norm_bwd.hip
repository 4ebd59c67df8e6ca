// The norms around a block, backwards (mathematics: ttt_block_norm.h).  The workgroups walk
// rows, the next one on its way, with the sums of the parameters' gradients in registers, and
// write one partial sum each, added up by a second launch in a fixed order.
#include <math.h>

#include <algorithm>

#include "ttt_block_norm.h"

namespace ttt {

namespace {

// Waves to a SIMD that the registers are cut to: three where a lane has up to 12 values and no
// residual (32,768 rows of 12 heads of 64 in bf16 with a gate: 44 us), else two (32,768 rows of 768 in
// bf16 with an fp32 residual: 95 us; 115 with three, which spill 18 registers); one where 16 values, a gate
// and a residual would spill a hundred, but for rows of 512 lanes, whose eight waves are two to a SIMD
// whatever is asked for: above 6,144 columns with a gate and a residual 36 to 86 registers spill (4,096 rows
// of 8,192 in bf16 with an fp32 residual, forward and backward: 333 us, 195 without the gate; of 6,144 181 and 170)
template <typename T, typename TR, bool GATE, int LANES, int V, int NCH>
constexpr int kWaves = V * NCH <= 12 && LANES < 512 && __is_same(TR, NoResidual) ? 3
                       : V * NCH == 16 && GATE && !__is_same(TR, NoResidual) && LANES < 512                   ? 1
                                                                                                             : 2;

template <typename T, typename TR, bool GATE, int LANES, int V, int NCH>
__global__ __launch_bounds__(block_threads(LANES), (kWaves<T, TR, GATE, LANES, V, NCH>)) void block_norm_bwd_kernel(BlockNormParams p) {
  constexpr bool RES = !__is_same(TR, NoResidual);
  typedef typename ResidualOf<TR, T>::type R;
  constexpr int NT = block_threads(LANES), ROWS = NT / LANES;
  const int l = threadIdx.x & (LANES - 1), D = p.D;
  __shared__ float red[8];
  float dw[NCH][V], ds[NCH][V], dw2[NCH][V];
  Raw<T, V> nx[NCH], nz[NCH], ny[NCH];  // the next row
  Raw<R, V> nres[NCH], nr[NCH];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    nx[i].zero();
    nz[i].zero();
    ny[i].zero();
    nres[i].zero();
    nr[i].zero();
#pragma unroll
    for (int e = 0; e < V; ++e) dw[i][e] = ds[i][e] = dw2[i][e] = 0.f;
  }
  float ni = 1.f, nj = 0.f;
  const bool next = RES && p.w2 != nullptr;
  const auto fetch = [&](long long row) {
    const long long outer = p.heads == 1 ? row : row / p.heads, in = p.heads == 1 ? 0 : (row - outer * p.heads) * D;
    ni = p.stats[2 * row];
    if (next) nj = p.stats[2 * row + 1];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = V * (LANES * i + l), left = D - c;
      if (left > 0) {
        nx[i].load(static_cast<const T*>(p.x) + outer * p.ldx + in + c, left);
        if (GATE) nz[i].load(static_cast<const T*>(p.gate) + outer * p.ldg + in + c, left);
        if (p.dr != nullptr) nr[i].load(static_cast<const R*>(p.dr) + row * D + c, left);
        if (next) {
          nres[i].load(static_cast<const R*>(p.res) + outer * p.ldr + in + c, left);
          if (p.dy != nullptr) ny[i].load(static_cast<const T*>(p.dy) + row * D + c, left);
        }
      }
    }
  };
  // The parameters are in LDS, 1 where there is none: read from memory behind the next row's loads, they
  // would wait for those
  constexpr int COLS = LANES * V * NCH;
  extern __shared__ __attribute__((aligned(16))) float par[];
  for (int c = threadIdx.x; c < COLS; c += NT) {
    par[c] = p.w != nullptr && c < D ? p.w[c] : 1.f;
    par[COLS + c] = p.s != nullptr && c < D ? p.s[c] : 1.f;
    par[2 * COLS + c] = next && c < D ? p.w2[c] : 1.f;
  }
  __syncthreads();
  const auto params = [&](int which, int c, float (&v)[V]) {
#pragma unroll
    for (int q = 0; q < V; q += 4) {
      const f4 a = *reinterpret_cast<const f4*>(par + which * COLS + c + q);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[q + e] = a[e];
    }
  };
  const long long step = (long long)gridDim.x * ROWS;
  // (rows of a wave's lanes: each group ends by itself; of more waves: together)
  long long row = (long long)blockIdx.x * ROWS + threadIdx.x / LANES;
  if (row < p.R) fetch(row);
  for (; row < p.R; row += step) {
    const float inv = ni, jnv = nj;
    // x i; silu(z) and n silu'(z); D; and r j, then dn w
    float u[NCH][V], si[GATE ? NCH : 1][V], dsi[GATE ? NCH : 1][V], d[NCH][V], g[NCH][V];
    float s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = V * (LANES * i + l), left = D - c;
      float w[V], sc[V], w2[V];
      params(0, c, w);
      if (next) {
        params(1, c, sc);
        params(2, c, w2);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        u[i][e] = nx[i].f(e) * inv;
        const float n = u[i][e] * w[e];
        float of = n;  // what the residual is added to
        if (GATE) {
          const float z = nz[i].f(e), sg = sigmoid_f(z);
          si[i][e] = z * sg;
          dsi[i][e] = n * sg * __builtin_fmaf(z, 1.0f - sg, 1.0f);
          of *= si[i][e];
        }
        d[i][e] = nr[i].f(e);
        g[i][e] = 0.f;
        if (next) {
          of *= sc[e];
          const float dy = ny[i].f(e), rj = (nres[i].f(e) + of) * jnv;
          if (e < left) {
            const float dyw = dy * w2[e];
            dw2[i][e] = __builtin_fmaf(dy, rj, dw2[i][e]);
            s2 = __builtin_fmaf(dyw, rj, s2);
            d[i][e] = __builtin_fmaf(dyw, jnv, d[i][e]);
          }
          g[i][e] = rj;
        }
      }
    }
    if (next) {
      const float m = share_sum<LANES>(s2, red) / (float)D * jnv;
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) d[i][e] = __builtin_fmaf(-m, g[i][e], d[i][e]);
    }
    if (row + step < p.R) fetch(row + step);
    float s1 = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = V * (LANES * i + l), left = D - c;
      if (left > 0) {
        if (RES && p.dres != nullptr) store_row<R, V>(static_cast<R*>(p.dres) + row * D + c, left, d[i]);
        float w[V], sc[V], dz[V];
        params(0, c, w);
        params(1, c, sc);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float we = w[e], gate = GATE ? si[i][e] : 1.f;
          ds[i][e] = __builtin_fmaf(d[i][e], u[i][e] * we * gate, ds[i][e]);
          const float dm = d[i][e] * sc[e], dn = dm * gate;
          if (GATE) dz[e] = dm * dsi[i][e];
          dw[i][e] = __builtin_fmaf(dn, u[i][e], dw[i][e]);
          g[i][e] = dn * we;
          if (e < left) s1 = __builtin_fmaf(g[i][e], u[i][e], s1);
        }
        if (GATE) store_row<T, V>(static_cast<T*>(p.dgate) + row * D + c, left, dz);
      }
    }
    const float m1 = p.w != nullptr ? share_sum<LANES>(s1, red) / (float)D : 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = V * (LANES * i + l), left = D - c;
      if (left > 0) {
        float dx[V];
#pragma unroll
        for (int e = 0; e < V; ++e) dx[e] = inv * __builtin_fmaf(-m1, u[i][e], g[i][e]);
        store_row<T, V>(static_cast<T*>(p.dx) + row * D + c, left, dx);
      }
    }
  }
  if (p.partial == nullptr) return;
  float* part = p.partial + (long long)blockIdx.x * 3 * D;
  const auto write = [&](float (&a)[NCH][V], int which) {
    if constexpr (LANES < 256) {  // the groups of a wave, then the four waves, in order
      __shared__ float acc[4][LANES * V * NCH];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float v = a[i][e];
#pragma unroll
          for (int m = LANES; m < 64; m *= 2) v += __shfl_xor(v, m);
          if ((threadIdx.x & 63) < LANES) acc[threadIdx.x >> 6][LANES * (V * i + e) + l] = v;
        }
      __syncthreads();
      for (int o = threadIdx.x; o < LANES * V * NCH; o += NT) {
        const int ie = o / LANES, i = ie / V, c = V * (LANES * i + o % LANES) + ie % V;
        if (c < D) part[(long long)which * D + c] = (acc[0][o] + acc[1][o]) + (acc[2][o] + acc[3][o]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int c = V * (LANES * i + l), left = D - c;
        if (left > 0) store_row<float, V>(part + (long long)which * D + c, left, a[i]);
      }
    }
  };
  if (p.dw != nullptr) write(dw, 0);
  if (p.ds != nullptr) write(ds, 1);
  if (p.dw2 != nullptr) write(dw2, 2);
}

// dw, ds, dw2: the sum over the workgroups' partial sums
__global__ __launch_bounds__(256) void block_norm_param_grads_kernel(BlockNormParams p, int parts) {
  const int blocks = (p.D + 15) / 16, which = blockIdx.x / blocks;
  float* to = which == 0 ? p.dw : which == 1 ? p.ds : p.dw2;
  if (to == nullptr) return;
  const int c = (blockIdx.x - which * blocks) * 16 + (threadIdx.x & 15);
  const float s = sum_parts(p.partial, 3LL * p.D, c < p.D ? (long long)which * p.D + c : 3LL * p.D, parts);
  if (threadIdx.x < 16 && c < p.D) to[c] = s;
}

template <typename T, typename TR> struct Bwd {
  template <int LANES, int V, int NCH> struct Of {
    template <bool GATE> static hipError_t launch(const BlockNormParams& p, int parts, hipStream_t stream) {
      constexpr int lds = 3 * LANES * V * NCH * 4;
      const auto kernel = block_norm_bwd_kernel<T, TR, GATE, LANES, V, NCH>;
      if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
      }
      hipLaunchKernelGGL(kernel, dim3(parts), dim3(block_threads(LANES)), lds, stream, p);
      return hipGetLastError();
    }
    static hipError_t run(const BlockNormParams& p, hipStream_t stream) {
      const int parts = block_norm_parts(
          p.R, p.D, p.gate != nullptr ? kWaves<T, TR, true, LANES, V, NCH> : kWaves<T, TR, false, LANES, V, NCH>);
      const hipError_t e = p.gate != nullptr ? launch<true>(p, parts, stream) : launch<false>(p, parts, stream);
      if (e != hipSuccess) return e;
      if (p.partial != nullptr)
        hipLaunchKernelGGL(block_norm_param_grads_kernel, dim3(3 * ((p.D + 15) / 16)), dim3(256), 0, stream, p, parts);
      return hipGetLastError();
    }
  };
};
template <typename T, typename TR> hipError_t run_t(const BlockNormParams& p, hipStream_t s) {
  return by_width<Bwd<T, TR>::template Of>(p.D, p, s);
}
template <typename T> hipError_t residual_t(const BlockNormParams& p, int dtype, int res_dtype, hipStream_t s) {
  if (res_dtype < 0) return run_t<T, NoResidual>(p, s);
  if (res_dtype == dtype) return run_t<T, T>(p, s);
  if constexpr (sizeof(T) == 2) return run_t<T, float>(p, s);
  return hipErrorInvalidValue;
}

}  // namespace

// Workgroups of the backward: as many as are held at once with `waves` to a SIMD (the partial sums
// are sized for three, of which there are the most)
int block_norm_parts(long long R, int D, int waves) {
  const int lanes = block_lanes(D), rows = block_threads(lanes) / lanes;
  const long long blocks = (R + rows - 1) / rows, most = lanes == 512 ? 256 : 256 * waves;
  return (int)std::max(1LL, std::min(blocks, most));
}
hipError_t launch_block_norm_bwd(const BlockNormParams& p, int dtype, int res_dtype, hipStream_t s) {
  return dtype == TTT_DTYPE_BF16 ? residual_t<__bf16>(p, dtype, res_dtype, s)
         : dtype == TTT_DTYPE_F16 ? residual_t<_Float16>(p, dtype, res_dtype, s)
                                  : residual_t<float>(p, dtype, res_dtype, s);
}

}  // namespace ttt
