// The selective scan's walks along a sequence on gfx950 (mathematics and layouts:
// ttt_scan.h).  Forwards they give the outputs y and the last state; backwards, the
// same with the roles of B and C and the order of the tokens exchanged, the gradient
// of x and of the states:
//   y_i  = sum_{j<=i} F_ij d_j (C_i . B_j) x_j + e^{c_i} H C_i + D x_i
//   dx_j = d_j (sum_{i>=j} F_ij (C_i . B_j) dy_i + e^{c_Q - c_j} Gam B_j) + D dy_j
//   Gam' = e^{c_Q} Gam + sum_i e^{c_i} dy_i (x) C_i
// with F_ij = e^{c_i - c_j}.  Below, the keys are what enters the state (B forwards, C
// backwards) and the queries what reads it.
//
// A workgroup walks one sequence and head, or one segment of it, chunk by chunk with
// the state in registers; wave w has the 16 features 16w..16w+15.  Per chunk the waves
// share out the triangle of masked products of keys and queries, pass it through LDS,
// and each forms its features' outputs and its part of the state behind the chunk.
// The next chunk's rows are on their way meanwhile.
//
// Where there are few sequences and heads, the tokens are cut into segments: their
// end states from a zero start (the same walk without outputs), the states entering
// them (scan_join_kernel), then all segments at once.
#include <math.h>

#include "ttt_scan.h"

namespace ttt {

namespace {

enum class Walk { Forward, Back };

template <typename T, int P, int NP, bool OUT> struct WalkShared {
  static constexpr int IN = ScanType<T>::IN, MID = ScanType<T>::MID, Q = chunk_of<T, NP>(), TB = Q / 16;
  Planes<IN, Q, P> x;
  Planes<IN, Q, NP> key;
  Planes<IN, OUT ? Q : 1, NP> query;
  bf4 m[MID][OUT ? TB * (TB + 1) / 2 : 1][64];  // the masked products, by tile and lane
  Decays<Q> dec[2];
};

__device__ __forceinline__ bool not_finite(__bf16 v) {
  return (__builtin_bit_cast(unsigned short, v) & 0x7f80) == 0x7f80;
}
// whether any of four values' first planes is not finite
__device__ __forceinline__ bool not_finite(bf4 v) {
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  const u2 u = __builtin_bit_cast(u2, v) & 0x7f807f80u;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 2; ++i) bad |= (u[i] & 0xffffu) == 0x7f80u || (u[i] >> 16) == 0x7f80u;
  return bad;
}

// OUT: outputs too; else the segments' end states and decays alone
template <typename T, int P, int NP, Walk WALK, bool OUT>
__global__ __launch_bounds__(4 * P) void scan_walk_kernel(ScanParams p) {
  using Sh = WalkShared<T, P, NP, OUT>;
  constexpr bool BACK = WALK == Walk::Back;
  constexpr int IN = Sh::IN, MID = Sh::MID, Q = Sh::Q, TB = Sh::TB, W = P / 16, NT = 4 * P, NC2 = NP / 32;
  constexpr int NB = StateTiles<NP>::NB;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Sh& sh = *reinterpret_cast<Sh*>(smem);
  const int w = wave_id(), l = lane_id(), g = l >> 4, r = l & 15;
  // without outputs, the last segment of the walk has nothing to add
  const int segs = OUT ? p.S : p.S - 1;
  const long long chain = blockIdx.x / segs;
  const int s = blockIdx.x % segs + (!OUT && BACK ? 1 : 0);
  const int b = (int)(chain / p.H), h = (int)(chain - (long long)b * p.H), grp = h / (p.H / p.G);
  const int NC = (p.L + Q - 1) / Q, c0 = s * p.per, n = min(NC, c0 + p.per) - c0;
  const float A = p.A[h], D = p.D != nullptr ? p.D[h] : 0.f;
  const long long row0 = (long long)b * p.L;
  const T* X = static_cast<const T*>(BACK ? p.dy : p.x) + h * P;
  const T* Key = static_cast<const T*>(BACK ? p.Cm : p.Bm) + grp * p.N;
  const T* Query = static_cast<const T*>(BACK ? p.Bm : p.Cm) + grp * p.N;
  const long long ldx = BACK ? p.ldy : p.ldx, ldk = BACK ? p.ldc : p.ldb, ldq = BACK ? p.ldb : p.ldc;
  T* Y = static_cast<T*>(BACK ? p.dx : p.y);

  StateTiles<NP> st;
  if (!OUT)
    st.load(nullptr, 0, 0, w);
  else if (p.seg != nullptr)
    st.load(p.seg + (chain * p.S + s) * P * NP, NP, NP, w);
  else
    st.load(p.h0 != nullptr ? p.h0 + chain * P * p.N : nullptr, p.N, p.N, w);

  Stage<T, Q, P, NT> sx;
  Stage<T, Q, NP, NT> sk, sq;
  float dt = 0.f, sum = 0.f;
  const auto chunk = [&](int k) { return BACK ? c0 + n - 1 - k : c0 + k; };
  const auto fetch = [&](int k) {
    const int t0 = chunk(k) * Q, left = p.L - t0;
    sx.load(X + (row0 + t0) * ldx, ldx, left, P);
    sk.load(Key + (row0 + t0) * ldk, ldk, left, p.N);
    if (OUT) sq.load(Query + (row0 + t0) * ldq, ldq, left, p.N);
    if (w == 0) dt = l < Q && l < left ? token_step<T>(p, row0 + t0 + l, h) : 0.f;
  };
  fetch(0);
  if (w == 0) sh.dec[0].fill(dt, A);
  for (int k = 0; k < n; ++k) {
    const int c = chunk(k);
    if (k > 0) __syncthreads();  // the last chunk's readers are done
    sx.store(sh.x);
    sk.store(sh.key);
    if constexpr (OUT) sq.store(sh.query);
    __syncthreads();
    if (k + 1 < n) fetch(k + 1);
    const Decays<Q>& dec = sh.dec[k & 1];

    Op<IN> xt[Q / 32];  // x^T: free feature, contraction token
    if constexpr (OUT) {
      // F (C . B), forwards times d_j, as tiles with the keys' tokens as rows: operands
      // with free query and contraction over the keys.  Tile (a, b), a >= b: token blocks
      // a of C and b of B
      for (int t = w; t < TB * (TB + 1) / 2; t += W) {
        const int hb = tri_row(t), lb = t - tri(hb, 0), kb = BACK ? hb : lb, qb = BACK ? lb : hb;
        f4 acc = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < NC2; ++q) mma<MID>(acc, sh.key.rows(16 * kb, 32 * q), sh.query.rows(16 * qb, 32 * q));
        const int tq = 16 * qb + r, tk = 16 * kb + 4 * g;
        const float qh = dec.hi[tq], ql = dec.lo[tq];
        const f4 kh = dec.four(dec.hi, tk), kl = dec.four(dec.lo, tk);
        const f4 dk = BACK ? f4{1.f, 1.f, 1.f, 1.f} : dec.four(dec.d, tk);
        bf4 o[MID];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = BACK ? (kh[e] - qh) + (kl[e] - ql) : (qh - kh[e]) + (ql - kl[e]);
          const float f = __builtin_amdgcn_exp2f(x);
          __bf16 q[MID];
          split1<MID>((BACK ? tk + e >= tq : tk + e <= tq) ? acc[e] * f * dk[e] : 0.f, q);
#pragma unroll
          for (int a = 0; a < MID; ++a) o[a][e] = q[a];
        }
#pragma unroll
        for (int a = 0; a < MID; ++a) sh.m[a][t][l] = o[a];
      }
      __syncthreads();
    }
    unsigned bad = 0;  // blocks of 16 tokens with a value that is not finite
#pragma unroll
    for (int q = 0; q < Q / 32; ++q) {
      xt[q] = sh.x.template cols<>(32 * q, 16 * w);
      if (OUT && !BACK) {
        const bf4 a = __builtin_shufflevector(xt[q].v[0], xt[q].v[0], 0, 1, 2, 3);
        const bf4 z = __builtin_shufflevector(xt[q].v[0], xt[q].v[0], 4, 5, 6, 7);
        bad |= (__ballot(not_finite(a)) != 0 ? 1u : 0u) << (2 * q) | (__ballot(not_finite(z)) != 0 ? 2u : 0u) << (2 * q);
      }
    }
    if constexpr (OUT) {
      if (p.states != nullptr) st.keep(p.states + (chain * NC + c) * (long long)(P * NP), P, w);
      // outputs, transposed: rows are features, columns tokens
      f4 y[TB];
#pragma unroll
      for (int ob = 0; ob < TB; ++ob) y[ob] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < NC2; ++q) {
        const Op<MID> hq = st.template op<MID>(q);
#pragma unroll
        for (int ob = 0; ob < TB; ++ob) mma<MID>(y[ob], hq, sh.query.rows(16 * ob, 32 * q));
      }
#pragma unroll
      for (int ob = 0; ob < TB; ++ob) {
        const int o = 16 * ob + r;
        const bf4 zero = {(__bf16)0.f, (__bf16)0.f, (__bf16)0.f, (__bf16)0.f};
        y[ob] *= BACK ? dec.tail[o] : dec.head[o];
#pragma unroll
        for (int q = 0; q < Q / 32; ++q) {
          const int b0 = 2 * q, b1 = 2 * q + 1;
          const bool in0 = BACK ? b0 >= ob : b0 <= ob, in1 = BACK ? b1 >= ob : b1 <= ob;
          if (!in0 && !in1) continue;
          Op<MID> m;
#pragma unroll
          for (int a = 0; a < MID; ++a)
            m.v[a] = cat(in0 ? sh.m[a][in0 ? (BACK ? tri(b0, ob) : tri(ob, b0)) : 0][l] : zero,
                         in1 ? sh.m[a][in1 ? (BACK ? tri(b1, ob) : tri(ob, b1)) : 0][l] : zero);
          // A token that is not finite reaches the tokens behind it alone: 0 times it is
          // no 0, so it is left out where its block meets itself, and so is the half of an
          // operand that is not wanted; its part in its own block follows below.
          Op<IN> xk = xt[q];
          if (!BACK && bad != 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int blk = e < 4 ? b0 : b1;
              if (blk > ob || (blk == ob && not_finite(xt[q].v[0][e])))
#pragma unroll
                for (int a = 0; a < IN; ++a) xk.v[a][e] = (__bf16)0.f;
            }
          }
          mma<MID>(y[ob], xk, m);
        }
        if (!BACK && (bad >> ob & 1)) {
          for (int j = 0; j < 16; ++j) {
            // lane (g', i) of the tile has rows j = 4g' + e of column i
            float m = 0.f;
#pragma unroll
            for (int a = MID - 1; a >= 0; --a) m += (float)sh.m[a][tri(ob, ob)][16 * (j >> 2) + r][j & 3];
            const f4 xj = sh.x.quad(16 * ob + j, 16 * w + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (j <= r && !(fabsf(xj[e]) < HUGE_VALF)) y[ob][e] += m * xj[e];
          }
        }
        if (BACK) y[ob] *= dec.d[o];
        if (p.D != nullptr) y[ob] += sh.x.quad(o, 16 * w + 4 * g) * D;
        const int t = c * Q + o;
        if (t < p.L) store4(Y + ((row0 + t) * p.H + h) * P + 16 * w + 4 * g, y[ob]);
      }
    }
    // the state behind the chunk
    if (!OUT) sum += dec.total;
    const float end = dec.end;
#pragma unroll
    for (int i = 0; i < NB; ++i) st.t[i] *= end;
#pragma unroll
    for (int q = 0; q < Q / 32; ++q) {
      float v[8];
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        const int t = 32 * q + 16 * o + 4 * g;
        const f4 in = BACK ? dec.four(dec.head, t) : dec.four(dec.d, t) * dec.four(dec.tail, t);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * o + e] = join(xt[q], 4 * o + e) * in[e];
      }
      const Op<kFull> xw = split8<kFull>(v);
#pragma unroll
      for (int i = 0; i < NB; ++i)
        mma<kFull>(st.t[i], sh.key.template cols<true>(32 * q, 32 * (i >> 1) + 4 * (i & 1)), xw);
    }
    if (w == 0 && k + 1 < n) sh.dec[(k + 1) & 1].fill(dt, A);
  }
  if (!OUT) {
    st.store(p.seg + (chain * p.S + s) * P * NP, NP, NP, w);
    if (threadIdx.x == 0) p.seg_decay[chain * p.S + s] = sum;
  } else if (p.h_last != nullptr && s == (BACK ? 0 : p.S - 1)) {
    st.store(p.h_last + chain * P * p.N, p.N, p.N, w);
  }
}

// Segments' results -> the states they start from, in place: a thread has four
// values of a state and goes over the sequence's segments.
template <int P, int NP, Walk WALK> __global__ __launch_bounds__(256) void scan_join_kernel(ScanParams p, long long quads) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= quads) return;
  constexpr int PER = P * NP / 4;
  const long long chain = id / PER;
  const int q = (int)(id - chain * PER), row = q / (NP / 4), n = 4 * (q - row * (NP / 4));
  f4 hs = f4{0.f, 0.f, 0.f, 0.f};
  if (p.h0 != nullptr && n < p.N) hs = *reinterpret_cast<const f4*>(p.h0 + (chain * P + row) * p.N + n);
  for (int k = 0; k < p.S; ++k) {
    const long long s = chain * p.S + (WALK == Walk::Back ? p.S - 1 - k : k);
    f4* m = reinterpret_cast<f4*>(p.seg + s * P * NP) + q;
    if (k + 1 < p.S) {
      const f4 made = *m;
      *m = hs;
      hs = hs * __builtin_amdgcn_exp2f(p.seg_decay[s]) + made;
    } else {
      *m = hs;
    }
  }
}

template <typename K> hipError_t allow_lds(K k, size_t bytes) {
  return bytes <= 65536 ? hipSuccess
                        : hipFuncSetAttribute(reinterpret_cast<const void*>(k),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

template <typename T, int P, int NP, Walk WALK> hipError_t walk_t(const ScanParams& p, hipStream_t stream) {
  const long long chains = (long long)p.B * p.H, quads = chains * P * NP / 4;
  constexpr size_t lds = sizeof(WalkShared<T, P, NP, true>), lds1 = sizeof(WalkShared<T, P, NP, false>);
  static_assert(lds <= 160 * 1024, "LDS of a compute unit");
  hipError_t e = allow_lds(scan_walk_kernel<T, P, NP, WALK, true>, lds);
  if (e != hipSuccess) return e;
  if (p.S > 1) {
    e = allow_lds(scan_walk_kernel<T, P, NP, WALK, false>, lds1);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((scan_walk_kernel<T, P, NP, WALK, false>), dim3((unsigned)(chains * (p.S - 1))), dim3(4 * P), lds1,
                       stream, p);
    hipLaunchKernelGGL((scan_join_kernel<P, NP, WALK>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, stream, p, quads);
  }
  hipLaunchKernelGGL((scan_walk_kernel<T, P, NP, WALK, true>), dim3((unsigned)(chains * p.S)), dim3(4 * P), lds, stream, p);
  return hipGetLastError();
}
template <typename T, int P, Walk WALK> hipError_t width_t(const ScanParams& p, hipStream_t s) {
  return p.N <= 32 ? walk_t<T, P, 32, WALK>(p, s) : p.N <= 64 ? walk_t<T, P, 64, WALK>(p, s) : walk_t<T, P, 128, WALK>(p, s);
}
template <typename T, Walk WALK> hipError_t head_t(const ScanParams& p, int P, hipStream_t s) {
  return P == 64 ? width_t<T, 64, WALK>(p, s) : P == 32 ? width_t<T, 32, WALK>(p, s) : hipErrorInvalidValue;
}
template <Walk WALK> hipError_t launch(const ScanParams& p, int P, int dtype, hipStream_t s) {
  return dtype == TTT_DTYPE_BF16 ? head_t<__bf16, WALK>(p, P, s)
         : dtype == TTT_DTYPE_F16 ? head_t<_Float16, WALK>(p, P, s) : head_t<float, WALK>(p, P, s);
}

}  // namespace

hipError_t launch_scan_fwd(const ScanParams& p, int P, int dtype, hipStream_t s) { return launch<Walk::Forward>(p, P, dtype, s); }
hipError_t launch_scan_walk_back(const ScanParams& p, int P, int dtype, hipStream_t s) {
  return launch<Walk::Back>(p, P, dtype, s);
}

}  // namespace ttt
