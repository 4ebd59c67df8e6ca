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
// end states from a zero start (the same walk without outputs), then all segments at
// once.  Up to 8 of them, a workgroup joins those before its own by itself; more are
// joined beforehand (scan_join_kernel).
//
// What bounds it, at 32,768 tokens of 12 heads of 64 features and 64 states in bf16 (4
// segments of 192 chains, three workgroups a compute unit): 68 us for the outputs with the
// states kept for the backward, 210 MB of which 101 are those states, 3.1 TB/s; the loads
// and stores alone take 57, the arithmetic alone 48 (exponentials, masks and planes
// of the products more than the matrix instructions), with three workgroups to cover one
// another.  27 us more for the end states of three segments: 8 chunks one after the other,
// latency.  Walking back the same (67, 59 and 45).
#include <math.h>
#include <stddef.h>

#include <type_traits>

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
  Decays<Q, true> dec[2];
};

__device__ __forceinline__ bool not_finite(__bf16 v) {
  return (__builtin_bit_cast(unsigned short, v) & 0x7f80) == 0x7f80;
}
// whether any of N operands' first planes has a value that is not finite, over the wave
template <int N, int PL> __device__ __forceinline__ bool any_not_finite(const Op<PL> (&x)[N]) {
  typedef unsigned short us8 __attribute__((ext_vector_type(8)));
  typedef unsigned short us2 __attribute__((ext_vector_type(2)));
  us2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const us8 u = __builtin_bit_cast(us8, x[i].v[0]) & (unsigned short)0x7f80;
#pragma unroll
    for (int e = 0; e < 8; e += 2) m = __builtin_elementwise_max(m, us2{u[e], u[e + 1]});
  }
  return __ballot(m[0] == 0x7f80 || m[1] == 0x7f80) != 0;
}

// Waves to a SIMD that the registers are cut to: three in bf16 (164 registers), but where
// that would spill (P = 32, N = 64, 32,768 tokens of 24 heads: 190 us so, 117 without)
template <typename T, int P, int NP>
constexpr int kWaves = NP == 128 || ScanType<T>::IN > 1 || (P == 32 && NP == 64) ? 1 : 3;

// OUT: outputs too; else the segments' end states and decays alone
template <typename T, int P, int NP, Walk WALK, bool OUT>
__global__ __launch_bounds__(4 * P, (kWaves<T, P, NP>)) void scan_walk_kernel(ScanParams p) {
  using Sh = WalkShared<T, P, NP, OUT>;
  static_assert(offsetof(Sh, dec) % 16 == 0 && sizeof(Sh::dec[0]) % 16 == 0 && offsetof(Sh, key) % 16 == 0 &&
                    offsetof(Sh, query) % 16 == 0 && offsetof(Sh, m) % 16 == 0,
                "read 16 bytes at a time");
  constexpr bool BACK = WALK == Walk::Back;
  constexpr int IN = Sh::IN, MID = Sh::MID, Q = Sh::Q, TB = Sh::TB, W = P / 16, NT = 4 * P, NC2 = NP / 32;
  constexpr int NB = StateTiles<NP>::NB;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Sh& sh = *reinterpret_cast<Sh*>(smem);
  const int w = wave_id(), l = lane_id(), g = l >> 4, r = l & 15;
  // without outputs, the last segment of the walk has nothing to add
  const int segs = OUT ? p.S : p.S - 1;
  const unsigned at = on_xcd(blockIdx.x, gridDim.x);
  const int h = (int)(at % p.H), s = (int)(at / p.H % segs) + (!OUT && BACK ? 1 : 0), b = (int)(at / p.H / segs);
  const int grp = h / (p.H / p.G);
  const long long chain = (long long)b * p.H + h;
  const int NC = (p.L + Q - 1) / Q, c0 = s * p.per, n = min(NC, c0 + p.per) - c0;
  const float A = p.A[h], D = p.D != nullptr ? p.D[h] : 0.f;
  const long long row0 = (long long)b * p.L;
  const T* X = static_cast<const T*>(BACK ? p.dy : p.x) + h * P;
  const T* Key = static_cast<const T*>(BACK ? p.Cm : p.Bm) + grp * p.N;
  const T* Query = static_cast<const T*>(BACK ? p.Bm : p.Cm) + grp * p.N;
  const long long ldx = BACK ? p.ldy : p.ldx, ldk = BACK ? p.ldc : p.ldb, ldq = BACK ? p.ldb : p.ldc;
  T* Y = static_cast<T*>(BACK ? p.dx : p.y);

  StateTiles<NP> st;
  const float* made = p.seg + chain * p.S * P * NP;
  if (!OUT)
    st.load(nullptr, 0, 0, w);
  else if (p.S > 1 && p.joined)
    st.load(made + (long long)s * P * NP, NP, NP, w);
  else
    st.load(p.h0 != nullptr ? p.h0 + chain * P * p.N : nullptr, p.N, p.N, w);
  if (OUT && p.S > 1 && !p.joined) {  // a few segments before this one
    for (int k = 0; k < (BACK ? p.S - 1 - s : s); ++k) {
      const int q = BACK ? p.S - 1 - k : k;
      const float f = __builtin_amdgcn_exp2f(p.seg_decay[chain * p.S + q]);
      StateTiles<NP> m;
      m.load(made + (long long)q * P * NP, NP, NP, w);
#pragma unroll
      for (int i = 0; i < NB; ++i) st.t[i] = st.t[i] * f + m.t[i];
    }
  }

  // rows on their way: of the next chunk, and without outputs, where there are registers
  // for it, of the one behind it
  constexpr int AHEAD = OUT ? 1 : 2;
  Stage<T, Q, P, NT> sx[AHEAD];
  Stage<T, Q, NP, NT> sk[AHEAD], sq;
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    sx[i].place(ldx, P);
    sk[i].place(ldk, p.N);
  }
  if (OUT) sq.place(ldq, p.N);
  float sum = 0.f;
  const auto chunk = [&](int k) { return BACK ? c0 + n - 1 - k : c0 + k; };
  const long long t00 = row0 + (long long)chunk(0) * Q, dir = BACK ? -Q : Q;
  const T *xp = X + t00 * ldx, *kp = Key + t00 * ldk, *qp = Query + t00 * ldq;
  char* yp = reinterpret_cast<char*>(Y + (t00 * p.H + h) * P);
  const long long xstep = dir * ldx, kstep = dir * ldk, qstep = dir * ldq, ystep = dir * p.H * P * (int)sizeof(T);
  const unsigned ylane = (unsigned)(r * p.H * P + 16 * w + 4 * g) * (unsigned)sizeof(T);  // in the rows of y
  const unsigned yblock = (unsigned)(16 * p.H * P) * (unsigned)sizeof(T);
  const auto fetch = [&](int k, Stage<T, Q, P, NT>& x, Stage<T, Q, NP, NT>& key) {
    const int left = min(Q, p.L - chunk(k) * Q);
    x.load(xp, left);
    key.load(kp, left);
    if (OUT) sq.load(qp, left);
    xp += xstep;
    kp += kstep;
    qp += qstep;
  };
  // The steps of the chunk behind the next one: the last wave, which has fewer tiles than
  // the first, forms the next chunk's decays while those are formed
  const bool steps = w == W - 1;
  const float bias = p.dt_bias != nullptr ? p.dt_bias[h] : 0.f;
  const auto step_of = [&](int k) {
    const int t0 = chunk(k) * Q;
    return steps && k < n && l < Q && t0 + l < p.L ? dt_bits<T>(p, row0 + t0 + l, h) : 0u;
  };
  const auto decays = [&](int k, unsigned bits) {
    const int t0 = chunk(k) * Q;
    const float raw = dt_value<T>(p, bits, bias);
    sh.dec[k & 1].fill(l < Q && t0 + l < p.L ? (p.softplus ? softplus_f(raw) : raw) : 0.f, A);
  };
  const unsigned dt0 = step_of(0);
  unsigned dt = step_of(1);
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (i < n) fetch(i, sx[i], sk[i]);
  if (steps) decays(0, dt0);
  const auto step = [&](int k, Stage<T, Q, P, NT>& sx, Stage<T, Q, NP, NT>& sk) {
    const int c = chunk(k);
    if (k > 0) __syncthreads();  // the last chunk's readers are done
    sx.store(sh.x);
    sk.store(sh.key);
    if constexpr (OUT) sq.store(sh.query);
    if (OUT && p.states != nullptr) st.keep(p.states + (chain * NC + c) * (long long)(P * NP), P, w);
    __syncthreads();
    // (the steps were asked for a chunk ago, and before that chunk's rows: waiting for them
    // is not waiting for rows)
    const Decays<Q, true>& dec = sh.dec[k & 1];
    if (steps && k + 1 < n) decays(k + 1, dt);
    dt = step_of(k + 2);
    if (k + AHEAD < n) fetch(k + AHEAD, sx, sk);

    Op<IN> xt[Q / 32];  // x^T: free feature, contraction token
    if constexpr (OUT) {
      // F (C . B), forwards times d_j, as tiles with the keys' tokens as rows: operands
      // with free query and contraction over the keys.  Tile (a, b), a >= b: token blocks
      // a of C and b of B
      constexpr int TILES = TB * (TB + 1) / 2;
#pragma unroll
      for (int i = 0; i < (TILES + W - 1) / W; ++i) {
        const int t = w + W * i;
        if (t >= TILES) break;
        const int hb = tri_row(t), lb = t - tri(hb, 0), kb = BACK ? hb : lb, qb = BACK ? lb : hb;
        f4 acc = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < NC2; ++q) mma<MID>(acc, sh.key.rows(16 * kb, 32 * q), sh.query.rows(16 * qb, 32 * q));
        const int tq = 16 * qb + r, tk = 16 * kb + 4 * g;
        const float qh = dec.hi[tq], ql = dec.lo[tq];
        const f4 kh = dec.four(dec.hi, tk), kl = dec.four(dec.lo, tk);
        f4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = BACK ? (kh[e] - qh) + (kl[e] - ql) : (qh - kh[e]) + (ql - kl[e]);
          v[e] = acc[e] * __builtin_amdgcn_exp2f(x);
        }
        if (!BACK) v *= dec.four(dec.d, tk);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = only_if(BACK ? tk + e >= tq : tk + e <= tq, v[e]);
        bf4 o[MID];
        split4<MID>(v, o);
#pragma unroll
        for (int a = 0; a < MID; ++a) sh.m[a][t][l] = o[a];
      }
      __syncthreads();
    }
#pragma unroll
    for (int q = 0; q < Q / 32; ++q) xt[q] = sh.x.template cols<>(32 * q, 16 * w);
    if constexpr (OUT) {
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
      const auto outputs = [&](auto flagged) {
        constexpr bool BAD = decltype(flagged)::value;
        const bf4 zero = {(__bf16)0.f, (__bf16)0.f, (__bf16)0.f, (__bf16)0.f};
#pragma unroll
        for (int ob = 0; ob < TB; ++ob) {
          const int o = 16 * ob + r;
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
            Op<IN> xk = xt[q];
            if constexpr (BAD) {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const int blk = e < 4 ? b0 : b1;
                const bool out = blk > ob || (blk == ob && not_finite(xt[q].v[0][e]));
#pragma unroll
                for (int a = 0; a < IN; ++a) xk.v[a][e] = out ? (__bf16)0.f : xk.v[a][e];
              }
            }
            mma<MID>(y[ob], xk, m);
          }
          if constexpr (BAD) {
#pragma unroll 1
            for (int j = 0; j < 16; ++j) {
              // lane (g', i) of the tile has rows j = 4g' + e of column i
              float m = 0.f;
#pragma unroll
              for (int a = MID - 1; a >= 0; --a) m += (float)sh.m[a][tri(ob, ob)][16 * (j >> 2) + r][j & 3];
              const f4 xj = sh.x.quad(16 * ob + j, 16 * w + 4 * g);
#pragma unroll
              for (int e = 0; e < 4; ++e) y[ob][e] += j <= r && !(fabsf(xj[e]) < HUGE_VALF) ? m * xj[e] : 0.f;
            }
          }
          if (BACK) y[ob] *= dec.d[o];
          y[ob] += sh.x.quad(o, 16 * w + 4 * g) * D;
        }
      };
      // A token that is not finite reaches the tokens behind it alone.  0 times it is no
      // 0: where there is one, it is left out where its block meets itself, and so is the
      // half of an operand that is not wanted; its part in its own block is added by itself.
      if (!BACK && any_not_finite(xt))
        outputs(std::true_type{});
      else
        outputs(std::false_type{});
      // the next chunk's rows are here before the stores are sent: waiting for them
      // afterwards would be waiting for the stores
      sx.settle();
      sk.settle();
      sq.settle();
      const int left = p.L - c * Q;
#pragma unroll
      for (int ob = 0; ob < TB; ++ob)
        if (16 * ob + r < left) store4(reinterpret_cast<T*>(yp + (ylane + ob * yblock)), y[ob]);
      yp += ystep;
    }
    // the state behind the chunk
    if (!OUT) sum += dec.total;
    const float end = dec.end;
#pragma unroll
    for (int i = 0; i < NB; ++i) st.t[i] *= end;
#pragma unroll
    for (int q = 0; q < Q / 32; ++q) {
      f4 v[2];
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        const int t = 32 * q + 16 * o + 4 * g;
        v[o] = join4(xt[q], o) * (BACK ? dec.four(dec.head, t) : dec.four(dec.in, t));
      }
      const Op<kFull> xw = split8<kFull>(v[0], v[1]);
#pragma unroll
      for (int i = 0; i < NB; ++i)
        mma<kFull>(st.t[i], sh.key.template cols<true>(32 * q, 32 * (i >> 1) + 4 * (i & 1)), xw);
    }
  };
  for (int k = 0; k < n; k += AHEAD) {
    step(k, sx[0], sk[0]);
    if (AHEAD > 1 && k + 1 < n) step(k + 1, sx[AHEAD - 1], sk[AHEAD - 1]);
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
  constexpr int R = 8;  // segments read at once
  for (int k0 = 0; k0 < p.S; k0 += R) {
    f4 made[R];
    float f[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const long long s = chain * p.S + (WALK == Walk::Back ? p.S - 1 - k0 - i : k0 + i);
      if (k0 + i + 1 < p.S) {  // (the last segment's own state is not formed)
        made[i] = *(reinterpret_cast<const f4*>(p.seg + s * P * NP) + q);
        f[i] = p.seg_decay[s];
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const long long s = chain * p.S + (WALK == Walk::Back ? p.S - 1 - k0 - i : k0 + i);
      if (k0 + i < p.S) *(reinterpret_cast<f4*>(p.seg + s * P * NP) + q) = hs;
      if (k0 + i + 1 < p.S) hs = hs * __builtin_amdgcn_exp2f(f[i]) + made[i];
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
    if (p.joined)
      hipLaunchKernelGGL((scan_join_kernel<P, NP, WALK>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, stream, p,
                         quads);
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

hipError_t launch_scan_fwd(const ScanParams& p, int P, int dtype, hipStream_t s) {
  return launch<Walk::Forward>(p, P, dtype, s);
}
hipError_t launch_scan_walk_back(const ScanParams& p, int P, int dtype, hipStream_t s) {
  return launch<Walk::Back>(p, P, dtype, s);
}

}  // namespace ttt
