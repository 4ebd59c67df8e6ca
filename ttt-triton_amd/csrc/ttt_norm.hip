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
// reductions (the variance is that of the centred values).  A row has 1, 4, 8 or 16
// waves and a lane 4, 8, 12 or 16 of its values, in groups of 4 or 8 that one load
// brings.  The backward's workgroups walk rows, the next one on its way (not with 16
// waves, which have 128 registers), with the sums of dw and db in registers, and write one
// partial sum each, added up by a second launch in a fixed order.
// In a trace of whole passes, 32,768 gated rows of 768 in bf16: forward 34 us (151 MB, 4.5 TB/s),
// backward 51 (252 MB, 4.9) and 4 for the partial sums; 4,099 rows of 5,001 in fp16, whose rows
// begin on odd addresses: 24, 38 and 9 (82 and 123 MB, 3.4 and 3.3 TB/s).  A device copy runs at
// 5.2 TB/s.  Above 8,192 values the backward does not fit its 128 registers, but for
// 12 values a lane without a gate: up to 32 bytes a lane go to scratch without one, 56 to 204 with
// one.  4,096 rows of 12,288 in bf16, forward and backward: 136 us without a gate (3.0 TB/s), 404
// with one (1.5), where 8,192 values take 87 and 123 (3.1 and 3.3).
#include <math.h>

#include <algorithm>

#include "ttt_ssm.h"

namespace ttt {

namespace {

constexpr int threads_of(int NW) { return NW == 1 ? 256 : 64 * NW; }

// the sum over the lanes that share a row, in every one of them
template <int NW> __device__ __forceinline__ float row_sum(float s, float* red) {
  s = sum_wave(s);
  if constexpr (NW == 1) {
    return s;
  } else {
    __syncthreads();  // the last sum's readers are done
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) v += red[k];
    return v;
  }
}

// NW waves to a row, NCH groups of V values to a lane
template <typename T, int NW, int V, int NCH, bool GATE>
__global__ __launch_bounds__(threads_of(NW)) void norm_fwd_kernel(NormParams p) {
  constexpr int LANES = 64 * NW;
  const int l = threadIdx.x & (LANES - 1);
  const long long row = NW == 1 ? (long long)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  __shared__ float red[16];
  if (row >= p.R) return;  // a whole wave of a one-wave row; never with more waves
  const int D = p.D;
  float v[NCH][V];
  float s = 0.f;
  {
    Raw<T, V> x[NCH], z[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = V * (LANES * i + l), n = D - c;
      x[i].zero();
      if (GATE) z[i].zero();
      if (n > 0) {
        x[i].load(static_cast<const T*>(p.x) + row * p.ldx + c, n);
        if (GATE) z[i].load(static_cast<const T*>(p.gate) + row * p.ldg + c, n);
      }
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[i][e] = x[i].f(e);
        if (GATE) v[i][e] *= z[i].f(e) * sigmoid_f(z[i].f(e));
        s += v[i][e];
      }
  }
  const float mean = row_sum<NW>(s, red) / (float)D;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int n = D - V * (LANES * i + l);
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < n) {
        const float d = v[i][e] - mean;
        s = __builtin_fmaf(d, d, s);
      }
  }
  const float rstd = 1.0f / sqrtf(row_sum<NW>(s, red) / (float)D + p.eps);
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = V * (LANES * i + l), n = D - c;
    if (n > 0) {
      float o[V];
      Raw<float, V> w, b;
      if (p.w != nullptr) {
        w.load(p.w + c, n);
        b.load(p.b + c, n);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        o[e] = (v[i][e] - mean) * rstd;
        if (p.w != nullptr) o[e] = __builtin_fmaf(o[e], w.v[e], b.v[e]);
      }
      store_row<T, V>(static_cast<T*>(p.y) + row * D + c, n, o);
    }
  }
  if (l == 0 && p.stats != nullptr) {
    p.stats[2 * row] = mean;
    p.stats[2 * row + 1] = rstd;
  }
}

template <typename T, int NW, int V, int NCH, bool GATE>
__global__ __launch_bounds__(threads_of(NW)) void norm_bwd_kernel(NormParams p) {
  constexpr int LANES = 64 * NW, ROWS = NW == 1 ? 4 : 1;
  constexpr bool AHEAD = NW < 16;
  const int l = threadIdx.x & (LANES - 1);
  __shared__ float red[16];
  const int D = p.D;
  float dw[NCH][V], db[NCH][V];
  Raw<T, V> nx[NCH], nz[NCH], ny[NCH];  // the next row
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    nx[i].zero();
    nz[i].zero();
    ny[i].zero();
#pragma unroll
    for (int e = 0; e < V; ++e) dw[i][e] = db[i][e] = 0.f;
  }
  float nmean = 0.f, nrstd = 0.f;
  const auto fetch = [&](long long row) {
    nmean = p.stats[2 * row];
    nrstd = p.stats[2 * row + 1];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = V * (LANES * i + l), n = D - c;
      if (n > 0) {
        nx[i].load(static_cast<const T*>(p.x) + row * p.ldx + c, n);
        if (GATE) nz[i].load(static_cast<const T*>(p.gate) + row * p.ldg + c, n);
        ny[i].load(static_cast<const T*>(p.dy) + row * D + c, n);
      }
    }
  };
  const long long step = (long long)gridDim.x * ROWS;
  // (rows of one wave: each wave ends by itself; of more: together)
  long long row = (long long)blockIdx.x * ROWS + (NW == 1 ? threadIdx.x >> 6 : 0);
  if (AHEAD && row < p.R) fetch(row);
  for (; row < p.R; row += step) {
    if (!AHEAD) fetch(row);
    const float mean = nmean, rstd = nrstd;
    float u[NCH][V], g[NCH][V], sx[NCH][V], sz[NCH][V];  // (sx, sz: what dv is multiplied with)
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = V * (LANES * i + l), n = D - c;
      Raw<float, V> w;
      if (p.w != nullptr && n > 0) w.load(p.w + c, n);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float x = nx[i].f(e), dy = ny[i].f(e);
        float v = x;
        if (GATE) {
          const float z = nz[i].f(e), sg = sigmoid_f(z);
          v *= z * sg;
          if (AHEAD) {
            sx[i][e] = z * sg;
            sz[i][e] = x * sg * __builtin_fmaf(z, 1.0f - sg, 1.0f);
          }
        }
        u[i][e] = e < n ? (v - mean) * rstd : 0.f;
        g[i][e] = p.w != nullptr && e < n ? dy * w.v[e] : dy;
        dw[i][e] = __builtin_fmaf(dy, u[i][e], dw[i][e]);
        db[i][e] += dy;
        s1 += g[i][e];
        s2 = __builtin_fmaf(g[i][e], u[i][e], s2);
      }
    }
    if (AHEAD && row + step < p.R) fetch(row + step);
    const float m1 = row_sum<NW>(s1, red) / (float)D, m2 = row_sum<NW>(s2, red) / (float)D;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = V * (LANES * i + l), n = D - c;
      float dx[V], dz[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float dv = (g[i][e] - m1 - u[i][e] * m2) * rstd;
        if (GATE && !AHEAD) {
          const float z = nz[i].f(e), sg = sigmoid_f(z);
          sx[i][e] = z * sg;
          sz[i][e] = nx[i].f(e) * sg * __builtin_fmaf(z, 1.0f - sg, 1.0f);
        }
        dx[e] = GATE ? dv * sx[i][e] : dv;
        if (GATE) dz[e] = dv * sz[i][e];
      }
      if (n > 0) {
        store_row<T, V>(static_cast<T*>(p.dx) + row * D + c, n, dx);
        if (GATE) store_row<T, V>(static_cast<T*>(p.dgate) + row * D + c, n, dz);
      }
    }
  }
  if (p.partial == nullptr) return;
  float* part = p.partial + (long long)blockIdx.x * 2 * D;
  if constexpr (NW == 1) {  // the four waves' sums, one after the other
    __shared__ float acc[2][64 * V * NCH];
#pragma unroll 1
    for (int q = 0; q < 4; ++q) {
      if ((threadIdx.x >> 6) == q) {
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const int j = 64 * (V * i + e) + l;  // lane-major: no two lanes share a bank
            acc[0][j] = q == 0 ? dw[i][e] : acc[0][j] + dw[i][e];
            acc[1][j] = q == 0 ? db[i][e] : acc[1][j] + db[i][e];
          }
      }
      __syncthreads();
    }
    for (int k = threadIdx.x >> 6; k < 2 * NCH; k += 4) {
      const int which = k / NCH, i = k - which * NCH, c = V * (64 * i + l), n = D - c;
      float o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = acc[which][64 * (V * i + e) + l];
      if (n > 0) store_row<float, V>(part + (long long)which * D + c, n, o);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = V * (LANES * i + l), n = D - c;
      if (n > 0) {
        store_row<float, V>(part + c, n, dw[i]);
        store_row<float, V>(part + D + c, n, db[i]);
      }
    }
  }
}

// dw, db: the sum over the workgroups' partial sums
__global__ __launch_bounds__(256) void norm_param_grads_kernel(NormParams p, int parts) {
  const long long n = 2LL * p.D, i = (long long)blockIdx.x * 16 + (threadIdx.x & 15);
  const float s = sum_parts(p.partial, n, i, parts);
  if (threadIdx.x < 16 && i < n) (i < p.D ? p.dw[i] : p.db[i - p.D]) = s;
}

template <typename T, int NW, int V, int NCH, bool GATE>
hipError_t run_t(const NormParams& p, bool bwd, hipStream_t stream) {
  if (!bwd) {
    constexpr long long kRows = 0xffffffffLL / (64 * NW) / 4 * 4;  // of a launch: 2^32 threads
    for (long long r0 = 0; r0 < p.R; r0 += kRows) {
      NormParams q = p;
      q.R = std::min(kRows, p.R - r0);
      q.x = static_cast<const T*>(p.x) + r0 * p.ldx;
      q.gate = static_cast<const T*>(p.gate) + (GATE ? r0 * p.ldg : 0);
      q.y = static_cast<T*>(p.y) + r0 * p.D;
      q.stats = p.stats != nullptr ? p.stats + 2 * r0 : nullptr;
      const long long blocks = NW == 1 ? (q.R + 3) / 4 : q.R;
      hipLaunchKernelGGL((norm_fwd_kernel<T, NW, V, NCH, GATE>), dim3((unsigned)blocks), dim3(threads_of(NW)), 0, stream, q);
    }
    return hipGetLastError();
  }
  const int parts = norm_bwd_parts(p.R, p.D);
  hipLaunchKernelGGL((norm_bwd_kernel<T, NW, V, NCH, GATE>), dim3(parts), dim3(threads_of(NW)), 0, stream, p);
  if (p.partial != nullptr)
    hipLaunchKernelGGL(norm_param_grads_kernel, dim3((2 * p.D + 15) / 16), dim3(256), 0, stream, p, parts);
  return hipGetLastError();
}
template <typename T, int NW, int V, int NCH> hipError_t gate_t(const NormParams& p, bool bwd, hipStream_t s) {
  return p.gate != nullptr ? run_t<T, NW, V, NCH, true>(p, bwd, s) : run_t<T, NW, V, NCH, false>(p, bwd, s);
}
// Waves to a row and values to a lane, so that few lanes' places are empty
template <typename T, int NW> hipError_t lanes_t(const NormParams& p, bool bwd, hipStream_t s) {
  const int four = (p.D + 256 * NW - 1) / (256 * NW);  // values to a lane, in fours
  if constexpr (NW <= 4) {
    if (four == 1) return gate_t<T, NW, 4, 1>(p, bwd, s);
    if (four == 2) return gate_t<T, NW, 8, 1>(p, bwd, s);
  }
  return four == 3 ? gate_t<T, NW, 4, 3>(p, bwd, s) : gate_t<T, NW, 8, 2>(p, bwd, s);
}
// (Gated bf16 rows, forward and backward: 32,768 of 768 with one wave 90 us, with four 124;
// 8,192 of 2,304 with four 73, with eight 134; of 4,096 119 and 159; 4,096 of 5,120 with eight
// 94, with sixteen 266.)
constexpr int waves_of(int D) { return D <= 1024 ? 1 : D <= 4096 ? 4 : D <= 8192 ? 8 : 16; }
template <typename T> hipError_t waves_t(const NormParams& p, bool bwd, hipStream_t s) {
  const int w = waves_of(p.D);
  return w == 1 ? lanes_t<T, 1>(p, bwd, s) : w == 4 ? lanes_t<T, 4>(p, bwd, s) : w == 8 ? lanes_t<T, 8>(p, bwd, s)
                                                                               : lanes_t<T, 16>(p, bwd, s);
}
hipError_t launch(const NormParams& p, int dtype, bool bwd, hipStream_t s) {
  if (p.D < 1 || p.D > kNormMaxD) return hipErrorInvalidValue;
  return dtype == TTT_DTYPE_BF16 ? waves_t<__bf16>(p, bwd, s)
         : dtype == TTT_DTYPE_F16 ? waves_t<_Float16>(p, bwd, s) : waves_t<float>(p, bwd, s);
}

}  // namespace

// Workgroups of the backward, in waves to a compute unit: 12 of rows of one and of four waves, 16
// of rows of eight; 8 of all three where a lane has 16 values; 16, one workgroup, of rows of sixteen
// waves.  Forward and backward in us with fewer, these and more: 32,768 gated rows of 768, 95 (8), 89
// (12), 100 (16); 4,099 of 5,001 without a gate 81 (8), 75 (12), 70 (16), 4,096 gated of 5,000 85, 100, 91;
// with 16 values 16,384 gated of 1,024, 60 (8) and 69 (12), 8,192 of 4,096, 119 and 133, 4,096 of 8,192,
// 125 (8) and 132 (16); 2,048 of 16,384, 277 (16) and 300 (two workgroups for one place).
int norm_bwd_parts(long long R, int D) {
  const int w = waves_of(D);
  const bool full = (D + 256 * w - 1) / (256 * w) > 3;  // 16 values to a lane
  const long long rows = w == 1 ? (R + 3) / 4 : R, most = w == 16 ? 256 : w == 8 ? (full ? 256 : 512) : full ? 512 : 768;
  return (int)std::max(1LL, std::min(rows, most));
}
hipError_t launch_norm_fwd(const NormParams& p, int dtype, hipStream_t s) { return launch(p, dtype, false, s); }
hipError_t launch_norm_bwd(const NormParams& p, int dtype, hipStream_t s) { return launch(p, dtype, true, s); }

}  // namespace ttt
