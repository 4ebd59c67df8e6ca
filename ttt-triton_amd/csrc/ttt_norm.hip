// Layer norm over the last axis, of x or of x silu(gate), forward and backward
// on gfx950.
//
//   v = x, or x z sigma(z) with the gate z;   u = (v - mean v) r,  r = 1/sqrt(var v + eps)
//   y = u w + b
// and backward, with g = dy w:
//   dv = r (g - mean g - u mean(g u)),   dw = sum dy u,  db = sum dy
//   dx = dv z sigma(z),   dz = dv x sigma(z) (1 + z (1 - sigma(z)))
//
// Both are bound by HBM: a row is read once and held in registers over its two
// reductions (the variance is that of the centred values).  Rows up to 1,024
// values have a wave each, longer ones a workgroup of four.  The backward's
// workgroups walk rows with the sums of dw and db in registers and write one
// partial sum each, added up by a second launch in a fixed order.
#include <math.h>

#include <algorithm>

#include "ttt_ssm.h"

namespace ttt {

namespace {

// the sum over the lanes that share a row, in every one of them
template <int NW> __device__ __forceinline__ float row_sum(float s, float* red) {
  s = sum_wave(s);
  if constexpr (NW == 1) {
    return s;
  } else {
    __syncthreads();  // the last sum's readers are done
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    return ((red[0] + red[1]) + red[2]) + red[3];
  }
}

// NW waves to a row, NCH x 8 values to a lane
template <typename T, int NW, int NCH, bool GATE>
__global__ __launch_bounds__(256) void norm_fwd_kernel(NormParams p) {
  constexpr int LANES = 64 * NW;
  const int l = threadIdx.x & (LANES - 1);
  const long long row = NW == 1 ? (long long)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  __shared__ float red[4];
  if (row >= p.R) return;  // a whole wave of a one-wave row; never with NW = 4
  const int D = p.D;
  float v[NCH][8];
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = 8 * (LANES * i + l), n = D - c;
    Raw8<T> x, z;
    if (n > 0) {
      x.load(static_cast<const T*>(p.x) + row * p.ldx + c, n);
      if (GATE) z.load(static_cast<const T*>(p.gate) + row * p.ldg + c, n);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[i][e] = e < n ? x.f(e) : 0.f;
      if (GATE && e < n) v[i][e] *= z.f(e) * sigmoid_f(z.f(e));
      s += v[i][e];
    }
  }
  const float mean = row_sum<NW>(s, red) / (float)D;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int n = D - 8 * (LANES * i + l);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) {
        const float d = v[i][e] - mean;
        s = __builtin_fmaf(d, d, s);
      }
  }
  const float rstd = 1.0f / sqrtf(row_sum<NW>(s, red) / (float)D + p.eps);
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = 8 * (LANES * i + l), n = D - c;
    if (n > 0) {
      float o[8];
      Raw8<float> w, b;
      if (p.w != nullptr) {
        w.load(p.w + c, n);
        b.load(p.b + c, n);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        o[e] = (v[i][e] - mean) * rstd;
        if (p.w != nullptr) o[e] = __builtin_fmaf(o[e], w.v[e], b.v[e]);
      }
      store8(static_cast<T*>(p.y) + row * D + c, n, o);
    }
  }
  if (l == 0 && p.stats != nullptr) {
    p.stats[2 * row] = mean;
    p.stats[2 * row + 1] = rstd;
  }
}

template <typename T, int NW, int NCH, bool GATE>
__global__ __launch_bounds__(256) void norm_bwd_kernel(NormParams p) {
  constexpr int LANES = 64 * NW, ROWS = 4 / NW;
  const int l = threadIdx.x & (LANES - 1);
  __shared__ float red[4];
  const int D = p.D;
  float dw[NCH][8], db[NCH][8];
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i][e] = db[i][e] = 0.f;
  // (rows of one wave: each wave ends by itself; of four: together)
  for (long long row = (long long)blockIdx.x * ROWS + (NW == 1 ? threadIdx.x >> 6 : 0); row < p.R;
       row += (long long)gridDim.x * ROWS) {
    const float mean = p.stats[2 * row], rstd = p.stats[2 * row + 1];
    float u[NCH][8], g[NCH][8];
    Raw8<T> x[NCH], z[NCH];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = 8 * (LANES * i + l), n = D - c;
      Raw8<T> dy;
      Raw8<float> w;
      if (n > 0) {
        x[i].load(static_cast<const T*>(p.x) + row * p.ldx + c, n);
        dy.load(static_cast<const T*>(p.dy) + row * D + c, n);
        if (GATE) z[i].load(static_cast<const T*>(p.gate) + row * p.ldg + c, n);
        if (p.w != nullptr) w.load(p.w + c, n);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        u[i][e] = g[i][e] = 0.f;
        if (e < n) {
          float v = x[i].f(e);
          if (GATE) v *= z[i].f(e) * sigmoid_f(z[i].f(e));
          u[i][e] = (v - mean) * rstd;
          g[i][e] = p.w != nullptr ? dy.f(e) * w.v[e] : dy.f(e);
          dw[i][e] = __builtin_fmaf(dy.f(e), u[i][e], dw[i][e]);
          db[i][e] += dy.f(e);
          s1 += g[i][e];
          s2 = __builtin_fmaf(g[i][e], u[i][e], s2);
        }
      }
    }
    const float m1 = row_sum<NW>(s1, red) / (float)D, m2 = row_sum<NW>(s2, red) / (float)D;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = 8 * (LANES * i + l), n = D - c;
      if (n > 0) {
        float dx[8], dz[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float dv = (g[i][e] - m1 - u[i][e] * m2) * rstd;
          dx[e] = dv;
          if (GATE) {
            const float zz = z[i].f(e), sg = sigmoid_f(zz);
            dx[e] = dv * zz * sg;
            dz[e] = dv * x[i].f(e) * sg * __builtin_fmaf(zz, 1.0f - sg, 1.0f);
          }
        }
        store8(static_cast<T*>(p.dx) + row * D + c, n, dx);
        if (GATE) store8(static_cast<T*>(p.dgate) + row * D + c, n, dz);
      }
    }
  }
  if (p.partial == nullptr) return;
  float* part = p.partial + (long long)blockIdx.x * 2 * D;
  if constexpr (NW == 1) {  // the four waves' sums, one after the other
    __shared__ float acc[2][64 * 8 * NCH];
#pragma unroll 1
    for (int q = 0; q < 4; ++q) {
      if ((threadIdx.x >> 6) == q) {
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int j = 64 * (8 * i + e) + l;  // lane-major: no two lanes share a bank
            acc[0][j] = q == 0 ? dw[i][e] : acc[0][j] + dw[i][e];
            acc[1][j] = q == 0 ? db[i][e] : acc[1][j] + db[i][e];
          }
      }
      __syncthreads();
    }
    for (int k = threadIdx.x >> 6; k < 2 * NCH; k += 4) {
      const int which = k / NCH, i = k - which * NCH, c = 8 * (64 * i + l), n = D - c;
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = acc[which][64 * (8 * i + e) + l];
      if (n > 0) store8(part + (long long)which * D + c, n, o);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = 8 * (LANES * i + l), n = D - c;
      if (n > 0) {
        store8(part + c, n, dw[i]);
        store8(part + D + c, n, db[i]);
      }
    }
  }
}

// dw, db: the sum over the workgroups' partial sums
__global__ __launch_bounds__(256) void norm_param_grads_kernel(NormParams p, int parts) {
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63;
  const long long n = 2LL * p.D, i = (long long)blockIdx.x * 64 + l;
  __shared__ float red[4][64];
  float s = 0.f;
  if (i < n)
    for (int q = wave; q < parts; q += 4) s += p.partial[q * n + i];
  red[wave][l] = s;
  __syncthreads();
  if (wave == 0 && i < n) {
    s = ((red[0][l] + red[1][l]) + red[2][l]) + red[3][l];
    if (i < p.D)
      p.dw[i] = s;
    else
      p.db[i - p.D] = s;
  }
}

template <typename T, int NW, int NCH, bool GATE>
hipError_t run_t(const NormParams& p, bool bwd, hipStream_t stream) {
  if (!bwd) {
    const long long blocks = NW == 1 ? (p.R + 3) / 4 : p.R;
    hipLaunchKernelGGL((norm_fwd_kernel<T, NW, NCH, GATE>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
    return hipGetLastError();
  }
  const int parts = norm_bwd_parts(p.R, p.D);
  hipLaunchKernelGGL((norm_bwd_kernel<T, NW, NCH, GATE>), dim3(parts), dim3(256), 0, stream, p);
  if (p.partial != nullptr)
    hipLaunchKernelGGL(norm_param_grads_kernel, dim3((2 * p.D + 63) / 64), dim3(256), 0, stream, p, parts);
  return hipGetLastError();
}
template <typename T, int NW, int NCH> hipError_t gate_t(const NormParams& p, bool bwd, hipStream_t s) {
  return p.gate != nullptr ? run_t<T, NW, NCH, true>(p, bwd, s) : run_t<T, NW, NCH, false>(p, bwd, s);
}
template <typename T> hipError_t size_t_(const NormParams& p, bool bwd, hipStream_t s) {
  if (p.D <= 512) return gate_t<T, 1, 1>(p, bwd, s);
  if (p.D <= 1024) return gate_t<T, 1, 2>(p, bwd, s);
  if (p.D <= 2048) return gate_t<T, 4, 1>(p, bwd, s);
  if (p.D <= 4096) return gate_t<T, 4, 2>(p, bwd, s);
  if (p.D <= 8192) return gate_t<T, 4, 4>(p, bwd, s);
  return gate_t<T, 4, 8>(p, bwd, s);
}
hipError_t launch(const NormParams& p, int dtype, bool bwd, hipStream_t s) {
  if (p.D < 1 || p.D > kNormMaxD) return hipErrorInvalidValue;
  return dtype == TTT_DTYPE_BF16 ? size_t_<__bf16>(p, bwd, s)
         : dtype == TTT_DTYPE_F16 ? size_t_<_Float16>(p, bwd, s) : size_t_<float>(p, bwd, s);
}

}  // namespace

// workgroups of the backward: up to 4 a compute unit
int norm_bwd_parts(long long R, int D) {
  const long long rows = D <= 1024 ? (R + 3) / 4 : R;
  return (int)std::max(1LL, std::min(rows, 1024LL));
}
hipError_t launch_norm_fwd(const NormParams& p, int dtype, hipStream_t s) { return launch(p, dtype, false, s); }
hipError_t launch_norm_bwd(const NormParams& p, int dtype, hipStream_t s) { return launch(p, dtype, true, s); }

}  // namespace ttt
