// The short causal convolution of the selective state-space layer on gfx950.
//
// With s = (state, x), the W-1 inputs before the first token and the L tokens,
//   z[t][c] = bias[c] + sum_{k<W} w[c][k] s[t+k][c],   y = z or z sigma(z)
// and the state left behind is s[L..L+W-2].  Backward, with dz = dy y'(z):
//   ds[u] = sum_k w[k] dz[u-k]  (+ the gradient of the state left, for u >= L)
//   dw[c][k] = sum_t dz[t] s[t+k],   dbias = sum_t dz[t]
// ds[u] is the state's gradient for u < W-1 and that of token u-W+1 behind it.
//
// Everything is bound by HBM.  A thread owns four channels (kV: 8 bytes of a 16-bit
// row) and walks a run of tokens with the window in registers, so that a row is
// read once and W-1 rows again per run; z is formed again in the backward, which
// costs W multiply-adds instead of a stored row.  Eight channels a thread need twice the
// registers for the rows on their way: 176 us for forward and backward of 32,768 tokens of
// 896 bf16 channels, 94 with four.  Of that 36 are the forward's in a graph of its own (117 MB,
// 3.3 TB/s); in a trace of whole passes it has 40 us and the backward 62 (176 MB, 2.8 TB/s),
// where a device copy runs at 5.2.  What is missing: every row's load stands behind branches of its
// own (is the row there, are all four channels), and waits with them, so that a thread has one
// row on its way; and the backward's 139 registers leave three waves to a SIMD.  One token of 64
// sequences: 4 us, a launch.
#include <math.h>

#include <algorithm>

#include "ttt_ssm.h"

namespace ttt {

namespace {

constexpr int kV = 4;
constexpr int kLanes = 32;   // backward: channel groups (of V) per workgroup
constexpr int kSubs = 256 / kLanes;  // and runs
constexpr int kRunBwd = 32;  // and tokens of a run (32,768 x 896 in bf16: 61 us with 16, 59 with 32, 57 with 64,
                             // which would halve the workgroups of short batches)

// row u of s, n of its channels from c on; zeros outside
template <typename T>
__device__ __forceinline__ Raw<T, kV> seen_row(const ConvParams& p, long long b, int u, int c, int n) {
  Raw<T, kV> r;
  const int W1 = p.W - 1;
  if (u < 0 || u >= p.L + W1) {
    r.zero();
  } else if (u < W1) {
    if (p.state != nullptr)
      r.load(static_cast<const T*>(p.state) + (b * W1 + u) * p.C + c, n);
    else
      r.zero();
  } else {
    r.load(static_cast<const T*>(p.x) + (b * p.L + (u - W1)) * p.ldx + c, n);
  }
  return r;
}

template <int W> struct Taps {
  float w[kV][W], bias[kV];
  __device__ __forceinline__ void load(const ConvParams& p, int c, int n) {
#pragma unroll
    for (int e = 0; e < kV; ++e) {
#pragma unroll
      for (int k = 0; k < W; ++k) w[e][k] = e < n ? p.w[(long long)(c + e) * W + k] : 0.f;
      bias[e] = e < n && p.bias != nullptr ? p.bias[c + e] : 0.f;
    }
  }
};

// RUN tokens to a thread: 16, or 8 where those are not enough threads for 16 waves to a
// compute unit (1,021 x 3 tokens of 999 channels in fp32: 11 and 18 us; 32,768 of 896 in
// bf16: 33 and 31)
template <typename T, int W, bool ACT, int RUN>
__global__ __launch_bounds__(256) void conv_fwd_kernel(ConvParams p, int groups, int runs, long long threads) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= threads) return;
  const int cg = (int)(id % groups);
  const long long br = id / groups;
  const int run = (int)(br % runs);
  const long long b = br / runs;
  const int c = kV * cg, n = min(kV, p.C - c);
  Taps<W> tp;
  tp.load(p, c, n);
  const int u0 = run * RUN, last = p.L + W - 1;
  Raw<T, kV> win[W];
#pragma unroll
  for (int k = 0; k < W - 1; ++k) win[k + 1] = seen_row<T>(p, b, u0 - (W - 1) + k, c, n);
#pragma unroll
  for (int i = 0; i < RUN; ++i) {
    const int u = u0 + i;
    if (u < last) {
#pragma unroll
      for (int k = 0; k < W - 1; ++k) win[k] = win[k + 1];
      win[W - 1] = seen_row<T>(p, b, u, c, n);
      if (u >= W - 1) {
        float o[kV];
#pragma unroll
        for (int e = 0; e < kV; ++e) {
          float z = tp.bias[e];
#pragma unroll
          for (int k = 0; k < W; ++k) z = __builtin_fmaf(tp.w[e][k], win[k].f(e), z);
          o[e] = ACT ? z * sigmoid_f(z) : z;
        }
        store_row<T, kV>(static_cast<T*>(p.y) + (b * p.L + (u - W + 1)) * p.C + c, n, o);
      }
      if (u >= p.L && p.last != nullptr)
        win[W - 1].store(static_cast<T*>(p.last) + (b * (W - 1) + (u - p.L)) * p.C + c, n);
    }
  }
}

// A workgroup: kLanes channel groups x kSubs runs of kRunBwd tokens, then the next
// kSubs runs of the rows `step` further.  A lane's sums of dw and dbias go over its
// runs, then over the runs of its workgroup in a fixed order.
template <typename T, int W, bool ACT>
__global__ __launch_bounds__(256) void conv_bwd_kernel(ConvParams p, int groups, int runs, long long jobs) {
  const int lane = threadIdx.x & (kLanes - 1), sub = threadIdx.x / kLanes;
  const int cg = blockIdx.y * kLanes + lane;
  const bool act = cg < groups;
  const int c = kV * cg, n = act ? min(kV, p.C - c) : 0;
  Taps<W> tp;
  tp.load(p, c, n);
  float dw[W][kV], dbias[kV];
#pragma unroll
  for (int e = 0; e < kV; ++e) {
    dbias[e] = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) dw[k][e] = 0.f;
  }
  const int last = p.L + W - 1;
  for (long long job = (long long)blockIdx.x * kSubs + sub; act && job < jobs; job += (long long)gridDim.x * kSubs) {
    const int run = (int)(job % runs);
    const long long b = job / runs;
    const int u0 = run * kRunBwd;
    // Step m handles token t = u0 - (W-1) + m, in groups of W steps whose rows are
    // asked for a group ahead (each behind its own branches).  Row s[t + W-1] has place m % W, dz[t] too, so that
    // s[t + k] is at (m + 1 + k) % W and dz[t - k] at (m - k) % W.
    Raw<T, kV> win[W], nx[W], ng[W];
    float dz[W][kV];
    const auto fetch = [&](int m, Raw<T, kV>& x, Raw<T, kV>& g) {
      const int t = u0 - (W - 1) + m;
      x = seen_row<T>(p, b, t + W - 1, c, n);
      if (t >= 0 && t < p.L && p.dy != nullptr)
        g.load(static_cast<const T*>(p.dy) + (b * p.L + t) * p.ldy + c, n);
      else
        g.zero();
    };
#pragma unroll
    for (int k = 0; k < W; ++k) {
      if (k < W - 1) win[(k + 1) % W] = seen_row<T>(p, b, u0 - (W - 1) + k, c, n);
#pragma unroll
      for (int e = 0; e < kV; ++e) dz[k][e] = 0.f;
      fetch(k, nx[k], ng[k]);
    }
    for (int m0 = 0; m0 < kRunBwd + W - 1; m0 += W) {
      Raw<T, kV> cx[W], cg[W];
#pragma unroll
      for (int k = 0; k < W; ++k) {
        cx[k] = nx[k];
        cg[k] = ng[k];
      }
      if (m0 + W < kRunBwd + W - 1) {
#pragma unroll
        for (int k = 0; k < W; ++k) fetch(m0 + W + k, nx[k], ng[k]);
      }
#pragma unroll
      for (int q = 0; q < W; ++q) {
        const int m = m0 + q, t = u0 - (W - 1) + m;
        win[q] = cx[q];
#pragma unroll
        for (int e = 0; e < kV; ++e) {
          float d = cg[q].f(e);
          if (ACT) {
            float z = tp.bias[e];
#pragma unroll
            for (int k = 0; k < W; ++k) z = __builtin_fmaf(tp.w[e][k], win[(q + 1 + k) % W].f(e), z);
            const float s = sigmoid_f(z);
            d *= s * __builtin_fmaf(z, 1.0f - s, 1.0f);
          }
          dz[q][e] = t >= 0 && t < p.L ? d : 0.f;
        }
        if (m < W - 1 || m >= kRunBwd + W - 1 || t >= last) continue;
        float o[kV];
#pragma unroll
        for (int e = 0; e < kV; ++e) {
          dbias[e] += dz[q][e];
          o[e] = 0.f;
#pragma unroll
          for (int k = 0; k < W; ++k) {
            // (rows behind the sequence are zeros there, as dz is)
            dw[k][e] = __builtin_fmaf(dz[q][e], win[(q + 1 + k) % W].f(e), dw[k][e]);
            o[e] = __builtin_fmaf(tp.w[e][k], dz[(q + W - k) % W][e], o[e]);
          }
        }
        if (t >= p.L && p.dlast != nullptr) {
          Raw<T, kV> r;
          r.load(static_cast<const T*>(p.dlast) + (b * (W - 1) + (t - p.L)) * p.C + c, n);
#pragma unroll
          for (int e = 0; e < kV; ++e) o[e] += r.f(e);
        }
        if (t >= W - 1)
          store_row<T, kV>(static_cast<T*>(p.dx) + (b * p.L + (t - W + 1)) * p.C + c, n, o);
        else if (p.dstate != nullptr)
          store_row<T, kV>(static_cast<T*>(p.dstate) + (b * (W - 1) + t) * p.C + c, n, o);
      }
    }
  }
  // lanes l and l ^ 32 hold the same channels; then the four waves
  static_assert(kLanes == 32, "half a wave");
  __shared__ float red[4][W + 1][kLanes * kV];
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int e = 0; e < kV; ++e) {
#pragma unroll
    for (int k = 0; k <= W; ++k) {
      const float v = k < W ? dw[k < W ? k : 0][e] : dbias[e], s = v + __shfl_xor(v, 32);
      if ((threadIdx.x & 63) < kLanes) red[wave][k][kV * lane + e] = s;
    }
  }
  __syncthreads();
  const int c0 = blockIdx.y * kLanes * kV;
  for (int i = threadIdx.x; i < (W + 1) * kLanes * kV; i += 256) {
    const int k = i / (kLanes * kV), j = i - k * kLanes * kV;
    if (c0 + j < p.C)
      p.partial[((long long)blockIdx.x * (W + 1) + k) * p.C + c0 + j] =
          ((red[0][k][j] + red[1][k][j]) + red[2][k][j]) + red[3][k][j];
  }
}

// dw, dbias: the sum over the workgroups' partial sums, 16 lanes to a channel and tap
__global__ __launch_bounds__(256) void conv_param_grads_kernel(ConvParams p, int parts) {
  const long long n = (long long)(p.W + 1) * p.C, i = (long long)blockIdx.x * 16 + (threadIdx.x & 15);
  const float s = sum_parts(p.partial, n, i, parts);
  if (threadIdx.x < 16 && i < n) {
    const int k = (int)(i / p.C);
    const long long c = i - (long long)k * p.C;
    if (k < p.W)
      p.dw[c * p.W + k] = s;
    else if (p.dbias != nullptr)
      p.dbias[c] = s;
  }
}

// one token: y from (state, x), and the state moved up by one, in place
template <typename T, int W, bool ACT>
__global__ __launch_bounds__(256) void conv_step_kernel(ConvParams p, int groups, long long threads) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= threads) return;
  const long long b = id / groups;
  const int c = kV * (int)(id % groups), n = min(kV, p.C - c);
  T* st = static_cast<T*>(p.last) + b * (W - 1) * p.C + c;
  Raw<T, kV> win[W];
#pragma unroll
  for (int k = 0; k < W - 1; ++k) win[k].load(st + (long long)k * p.C, n);
  win[W - 1].load(static_cast<const T*>(p.x) + b * p.ldx + c, n);
  Taps<W> tp;
  tp.load(p, c, n);
  float o[kV];
#pragma unroll
  for (int e = 0; e < kV; ++e) {
    float z = tp.bias[e];
#pragma unroll
    for (int k = 0; k < W; ++k) z = __builtin_fmaf(tp.w[e][k], win[k].f(e), z);
    o[e] = ACT ? z * sigmoid_f(z) : z;
  }
  store_row<T, kV>(static_cast<T*>(p.y) + b * p.C + c, n, o);
#pragma unroll
  for (int k = 0; k < W - 1; ++k) win[k + 1].store(st + (long long)k * p.C, n);
}

template <typename T, int W, bool ACT, int RUN> hipError_t fwd_run(const ConvParams& p, hipStream_t stream) {
  const int groups = (p.C + kV - 1) / kV, runs = (p.L + W - 1 + RUN - 1) / RUN;
  const long long threads = (long long)p.B * runs * groups;
  hipLaunchKernelGGL((conv_fwd_kernel<T, W, ACT, RUN>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, p,
                     groups, runs, threads);
  return hipGetLastError();
}
template <typename T, int W, bool ACT> hipError_t fwd_t(const ConvParams& p, hipStream_t stream) {
  const long long threads = (long long)p.B * ((p.L + 18) / 16) * ((p.C + kV - 1) / kV);
  return threads >= 256 * 16 * 64 ? fwd_run<T, W, ACT, 16>(p, stream) : fwd_run<T, W, ACT, 8>(p, stream);
}
template <typename T, int W, bool ACT> hipError_t bwd_t(const ConvParams& p, hipStream_t stream) {
  const int groups = (p.C + kV - 1) / kV, runs = (p.L + W - 1 + kRunBwd - 1) / kRunBwd;
  const int parts = conv_bwd_parts(p.B, p.L, p.C);
  hipLaunchKernelGGL((conv_bwd_kernel<T, W, ACT>), dim3(parts, (groups + kLanes - 1) / kLanes), dim3(256), 0, stream, p,
                     groups, runs, (long long)p.B * runs);
  const long long n = (long long)(W + 1) * p.C;
  hipLaunchKernelGGL(conv_param_grads_kernel, dim3((unsigned)((n + 15) / 16)), dim3(256), 0, stream, p, parts);
  return hipGetLastError();
}
template <typename T, int W, bool ACT> hipError_t step_t(const ConvParams& p, hipStream_t stream) {
  const int groups = (p.C + kV - 1) / kV;
  const long long threads = (long long)p.B * groups;
  hipLaunchKernelGGL((conv_step_kernel<T, W, ACT>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, p,
                     groups, threads);
  return hipGetLastError();
}

enum class ConvPass { Fwd, Bwd, Step };
template <typename T, int W, bool ACT> hipError_t pass_t(const ConvParams& p, ConvPass q, hipStream_t s) {
  return q == ConvPass::Fwd ? fwd_t<T, W, ACT>(p, s) : q == ConvPass::Bwd ? bwd_t<T, W, ACT>(p, s) : step_t<T, W, ACT>(p, s);
}
template <typename T, int W> hipError_t taps_t(const ConvParams& p, ConvPass q, hipStream_t s) {
  return p.silu ? pass_t<T, W, true>(p, q, s) : pass_t<T, W, false>(p, q, s);
}
template <typename T> hipError_t dtype_t(const ConvParams& p, ConvPass q, hipStream_t s) {
  return p.W == 4 ? taps_t<T, 4>(p, q, s) : p.W == 3 ? taps_t<T, 3>(p, q, s) : p.W == 2 ? taps_t<T, 2>(p, q, s)
                                                                             : hipErrorInvalidValue;
}
hipError_t launch(const ConvParams& p, int dtype, ConvPass q, hipStream_t s) {
  return dtype == TTT_DTYPE_BF16 ? dtype_t<__bf16>(p, q, s)
         : dtype == TTT_DTYPE_F16 ? dtype_t<_Float16>(p, q, s) : dtype_t<float>(p, q, s);
}

}  // namespace

// Workgroups over the tokens of the backward: enough for 8 workgroups a compute
// unit over all channels, and no more than there are runs
int conv_bwd_parts(int B, int L, int C) {
  const long long jobs = (long long)B * ((L + 3 + kRunBwd - 1) / kRunBwd);
  const int by = (C + kV * kLanes - 1) / (kV * kLanes);
  return (int)std::max(1LL, std::min((jobs + kSubs - 1) / kSubs, (2048LL + by - 1) / by));
}
hipError_t launch_conv_fwd(const ConvParams& p, int dtype, hipStream_t s) { return launch(p, dtype, ConvPass::Fwd, s); }
hipError_t launch_conv_bwd(const ConvParams& p, int dtype, hipStream_t s) { return launch(p, dtype, ConvPass::Bwd, s); }
hipError_t launch_conv_step(const ConvParams& p, int dtype, hipStream_t s) { return launch(p, dtype, ConvPass::Step, s); }

}  // namespace ttt
