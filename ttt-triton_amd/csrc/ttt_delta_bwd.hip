// The gated delta rule's backward on gfx950 beside its walk back (ttt_delta_walk.hip): the
// gradients of q, k, the decays and b (mathematics: ttt_delta.h).
//
// Given the states S entering the chunks and x (kept by the forward), and the gradients dS'
// of those leaving them, y and dv = b y (kept by the walk back), every chunk of a head stands
// alone.  With u = b x, h_i = e^{c_i}, w_j = e^{c_Q - c_j}, and q, k at unit length or as they are:
//   X_ij = s F_ij (do_i . u_j), j <= i;   Y_ij = -F_ij (dv_i . u_j), j < i
//   dq_i = s h_i S^T do_i + sum_j X_ij k_j
//   dk_j = w_j dS'^T u_j - h_j S^T dv_j + sum_i X_ij q_i + sum_i Y_ij k_i + sum_i Y_ji k_i
//   dbeta_i = y_i . x_i
// The gradient of a decay g_t is what passes it: from tokens before t to tokens from t on,
// from S to tokens from t on, from tokens before t to dS', and from S to dS':
//   dg_t = sum_{j<t<=i} (X_ij (q_i . k_j) + Y_ij (k_i . k_j)) + sum_{i>=t} a_i + sum_{j<t} d_j
//          + e^{c_Q} <dS', S>
//   a_i = s h_i q_i . (S^T do_i) - h_i k_i . (S^T dv_i),   d_j = w_j k_j . (dS'^T u_j)
// the first sum as that over i >= t of the rows' sums less the columns', whose equal terms
// cancel in 64 bits.  X and Y are kept with the factors that bring q and k to unit length, so
// that the products take the raw rows; what comes out is dq rq and dk rk, and
//   dq <- dq - rq^2 (q . dq) q
// is the gradient of the raw rows.
//
// A workgroup has a chunk of one head.  32 features of do, u and dv are in LDS at once, the next
// 32 on their way, with the sums over the features in registers: two workgroups to a compute unit
// (32,768 tokens of 12 heads of 64 x 64 in bf16: 215 us; 300 with all features at once, one workgroup).
// 700 MB go through it, 3.3 TB/s; its plain instructions, most of them splits of fp32 values into
// planes, take 58% of the issue slots and the matrix instructions 21%.  (Two workgroups to a compute unit
// leave 128 registers to a lane; with states of 64 in bf16 5 spill.)
#include <math.h>
#include <stddef.h>

#include "ttt_delta.h"

namespace ttt {

namespace {

constexpr int kSlice = 32;  // features that are in LDS at once

template <typename T, int NP> struct GradShared {
  static constexpr int IN = ScanType<T>::IN, MID = ScanType<T>::MID, Q = kDeltaQ<T>, TB = Q / 16;
  static constexpr int TILES = delta_tiles(Q), NB = NP / 16;
  static constexpr int WAVES = NB * TB < 8 ? NB * TB : 8;
  Planes<IN, Q, NP> q, k;
  union {
    struct {
      Planes<IN, Q, kSlice> dO;
      Planes<kFull, Q, kSlice> u, dv;
    };
    struct {  // behind the slices
      bf4 x[MID][TILES][64], y[MID][TILES][64];
      float a[NB][Q], d[NB][Q];    // by blocks of columns
      float qd[NB][Q], kd[NB][Q];  // q . dq and k . dk
    };
  };
  DeltaTok<Q> tok;
  float row[TILES][16], col[TILES][16];  // of X (q . k) + Y (k . k)
  float db[Q], gh[WAVES];
};

// 32 features of columns n = 16 nb + r of a state [NP][PB] in memory: lane (g, r) has values
// 8g + e of column r
struct Columns {
  f4 v[2];
  __device__ __forceinline__ void load(const float* __restrict__ s, int ld, int nb) {
    const int l = lane_id(), g = l >> 4, r = l & 15;
#pragma unroll
    for (int o = 0; o < 2; ++o) v[o] = *reinterpret_cast<const f4*>(s + (16 * nb + r) * ld + 8 * g + 4 * o);
  }
  __device__ __forceinline__ Op<kFull> op() const { return split8<kFull>(v[0], v[1]); }
  __device__ __forceinline__ float dot(const Columns& o) const {
    const f4 s = v[0] * o.v[0] + v[1] * o.v[1];
    return (s[0] + s[1]) + (s[2] + s[3]);
  }
};

// one of a token's gradients, in the type of what it is the gradient of
template <typename T> __device__ __forceinline__ void put(void* to, bool f32, long long o, float v) {
  if (sizeof(T) == 4 || f32)
    static_cast<float*>(to)[o] = v;
  else
    static_cast<T*>(to)[o] = (T)v;
}

template <typename T, int NP>
__global__ __launch_bounds__((64 * GradShared<T, NP>::WAVES), (NP == 128 && ScanType<T>::IN != 2 ? 2 : 4)) void delta_bwd_kernel(DeltaParams p) {
  using Sh = GradShared<T, NP>;
  static_assert(offsetof(Sh, tok) % 16 == 0 && offsetof(Sh, x) % 16 == 0 && offsetof(Sh, y) % 16 == 0 &&
                    offsetof(Sh, k) % 16 == 0 && offsetof(Sh, dO) % 16 == 0 && offsetof(Sh, u) % 16 == 0 &&
                    offsetof(Sh, dv) % 16 == 0 && offsetof(Sh, row) % 16 == 0,
                "read 16 bytes at a time");
  constexpr int IN = Sh::IN, MID = Sh::MID, Q = Sh::Q, TB = Sh::TB, QB = Q / 32, TILES = Sh::TILES, NB = Sh::NB;
  constexpr int WAVES = Sh::WAVES, NT = 64 * WAVES, NC2 = NP / 32, OWN = (TILES + WAVES - 1) / WAVES;
  // a wave has a block of 16 columns and every SHARE-th block of 16 tokens
  constexpr int SHARE = WAVES / NB, TOK = TB / SHARE;
  static_assert(SHARE * NB == WAVES && TOK * SHARE == TB, "whole shares");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Sh& sh = *reinterpret_cast<Sh*>(smem);
  const int w = wave_id(), l = lane_id(), g = l >> 4, r = l & 15, nb = w % NB, tb0 = w / NB, n0 = 16 * nb;
  const int PB = delta_part(p.P), parts = p.P / PB, NC = (p.L + Q - 1) / Q;
  const unsigned at = on_xcd(blockIdx.x, gridDim.x);
  const int h = (int)(at % p.H), c = (int)(at / p.H % NC), b = (int)(at / p.H / NC);
  const int HG = p.H / p.G, grp = h / HG;
  const int t0 = c * Q, left = min(Q, p.L - t0);
  const long long row0 = (long long)b * p.L + t0, head = (long long)b * p.H + h;

  // a slice's rows and columns on their way
  using Sf = Stage<float, Q, kSlice, NT>;
  Stage<T, Q, kSlice, NT> so;
  Sf sx, sy;
  Columns st, gs;  // S and dS'
  so.place(p.lddo, kSlice);
  sx.place(PB, kSlice);
  sy.place(PB, kSlice);
  const auto fetch = [&](int f) {
    const int part = f / PB, off = f - part * PB;
    const long long chunk = (head * parts + part) * NC + c;
    so.load(static_cast<const T*>(p.dO) + row0 * p.lddo + (long long)h * p.P + f, left);
    sx.load(p.x + chunk * (Q * PB) + off, Q);
    sy.load(p.rows + chunk * (Q * PB) + off, Q);
    st.load(p.states + chunk * (NP * PB) + off, PB, nb);
    gs.load(p.gstates + chunk * (NP * PB) + off, PB, nb);
  };
  {
    Stage<T, Q, NP, NT> sk, sq;
    sk.place(p.ldk, p.N);
    sq.place(p.ldq, p.N);
    sk.load(static_cast<const T*>(p.k) + row0 * p.ldk + (long long)grp * p.N, left);
    sq.load(static_cast<const T*>(p.q) + row0 * p.ldq + (long long)grp * p.N, left);
    fetch(0);
    const float* tok = p.tok + (head * NC + c) * delta_tok_floats(Q);
    for (int i = threadIdx.x; i < delta_tok_floats(Q) / 4; i += NT)
      reinterpret_cast<f4*>(&sh.tok)[i] = reinterpret_cast<const f4*>(tok)[i];
    sk.store(sh.k);
    sq.store(sh.q);
  }
  __syncthreads();
  const DeltaTok<Q>& tok = sh.tok;
  f4 tx[OWN], ty[OWN];  // do . u and dv . u, tiles of rows i and columns j
#pragma unroll
  for (int k = 0; k < OWN; ++k) tx[k] = ty[k] = f4{0.f, 0.f, 0.f, 0.f};
  f4 ia[TOK], iv[TOK], id[TOK];  // S^T do, S^T dv, dS'^T u, rows n and columns tokens
#pragma unroll
  for (int o = 0; o < TOK; ++o) ia[o] = iv[o] = id[o] = f4{0.f, 0.f, 0.f, 0.f};
  float db[Sf::CNT] = {}, gh = 0.f;
#pragma unroll 1
  for (int f = 0; f < p.P; f += kSlice) {
    if (f > 0) __syncthreads();  // the last slice's readers are done
#pragma unroll
    for (int i = 0; i < Sf::CNT; ++i) {
      const f4 x = __builtin_bit_cast(f4, sx.v[i]), y = __builtin_bit_cast(f4, sy.v[i]);
      const float beta = tok.beta[Sf::row(i) < Q ? Sf::row(i) : 0];
      const f4 xy = x * y;
      db[i] += (xy[0] + xy[1]) + (xy[2] + xy[3]);
      sx.v[i] = __builtin_bit_cast(u4v, x * beta);
      sy.v[i] = __builtin_bit_cast(u4v, y * beta);
    }
    so.store(sh.dO);
    sx.store(sh.u);
    sy.store(sh.dv);
    const Op<kFull> so_ = st.op(), go_ = gs.op();
    if (tb0 == 0) gh += gs.dot(st);
    __syncthreads();
    if (f + kSlice < p.P) fetch(f + kSlice);
#pragma unroll
    for (int k = 0; k < OWN; ++k) {
      const int t = w + WAVES * k;
      if (t >= TILES) break;
      const int ib = tri_row(t), jb = t - tri(ib, 0);
      const Op<kFull> u = sh.u.rows(16 * jb, 0);
      mma<kFull>(tx[k], sh.dO.rows(16 * ib, 0), u);
      mma<kFull>(ty[k], sh.dv.rows(16 * ib, 0), u);
    }
#pragma unroll
    for (int o = 0; o < TOK; ++o) {
      const int tb = SHARE * o + tb0;
      mma<kFull>(ia[o], so_, sh.dO.rows(16 * tb, 0));
      mma<kFull>(iv[o], so_, sh.dv.rows(16 * tb, 0));
      mma<kFull>(id[o], go_, sh.u.rows(16 * tb, 0));
    }
  }
#pragma unroll
  for (int i = 0; i < Sf::CNT; ++i) {
#pragma unroll
    for (int m = 1; m < Sf::PER; m *= 2) db[i] += __shfl_xor(db[i], m);
    if (Sf::has() && Sf::col(i) == 0) sh.db[Sf::row(i)] = db[i];
  }
  gh = sum_wave(gh);
  if (l == 0) sh.gh[w] = gh;
  __syncthreads();  // X and Y go where the slices were
#pragma unroll
  for (int k = 0; k < OWN; ++k) {
    const int t = w + WAVES * k;
    if (t >= TILES) break;
    const int ib = tri_row(t), jb = t - tri(ib, 0);
    f4 qk = f4{0.f, 0.f, 0.f, 0.f}, kk = qk;
#pragma unroll
    for (int q = 0; q < NC2; ++q) {
      const Op<IN> kj = sh.k.rows(16 * jb, 32 * q);
      mma<kFull>(qk, sh.q.rows(16 * ib, 32 * q), kj);
      mma<kFull>(kk, sh.k.rows(16 * ib, 32 * q), kj);
    }
    const int i0 = 16 * ib + 4 * g, j = 16 * jb + r;
    const f4 ih = tok.four(tok.hi, i0), il = tok.four(tok.lo, i0);
    const float jh = tok.hi[j], jl = tok.lo[j], rj = tok.rk[j];
    f4 fr;
#pragma unroll
    for (int e = 0; e < 4; ++e) fr[e] = __builtin_amdgcn_exp2f((ih[e] - jh) + (il[e] - jl)) * rj;
    f4 x = tx[k] * fr * tok.four(tok.rq, i0) * p.scale, y = ty[k] * fr * tok.four(tok.rk, i0) * -1.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = only_if(j <= i0 + e, x[e]);
      y[e] = only_if(j < i0 + e, y[e]);
    }
    bf4 o[MID];
    split4<MID>(x, o);
#pragma unroll
    for (int a = 0; a < MID; ++a) sh.x[a][t][l] = o[a];
    split4<MID>(y, o);
#pragma unroll
    for (int a = 0; a < MID; ++a) sh.y[a][t][l] = o[a];
    // What passes the decays between two tokens.  (A token's own pair passes none: left out, so
    // that a row's sum is of what reaches it from before)
    f4 pass = x * qk + y * kk;
#pragma unroll
    for (int e = 0; e < 4; ++e) pass[e] = j < i0 + e ? pass[e] : 0.f;
    const float cs = sum_col4((pass[0] + pass[1]) + (pass[2] + pass[3]));
    if (g == 0) sh.col[t][r] = cs;
#pragma unroll
    for (int e = 0; e < 4; ++e) pass[e] = sum_row16(pass[e]);
    if (r == 0) *reinterpret_cast<f4*>(&sh.row[t][4 * g]) = pass;
  }
  __syncthreads();

  const bf4 zero = {(__bf16)0.f, (__bf16)0.f, (__bf16)0.f, (__bf16)0.f};
  // tiles of X or Y as an operand with free column j and contracted rows i, or (the transposing
  // read of a tile, whose lane 16 a + j holds rows 4a..4a+3 of column j) the other way
  const int slot = 16 * (l & 3) + 4 * g + (r >> 2);
  const auto by_col = [&](const bf4 (&m)[MID][TILES][64], int jb, int q) {
    const bool one = 2 * q >= jb;
    Op<MID> o;
#pragma unroll
    for (int a = 0; a < MID; ++a)
      o.v[a] = cat(one ? m[a][one ? tri(2 * q, jb) : 0][l] : zero, m[a][tri(2 * q + 1, jb)][l]);
    return o;
  };
  const auto by_row = [&](const bf4 (&m)[MID][TILES][64], int ib, int q) {
    const bool two = 2 * q + 1 <= ib;
    Op<MID> o;
#pragma unroll
    for (int a = 0; a < MID; ++a) {
      const bf4 lo = read_tr(reinterpret_cast<const __bf16*>(&m[a][tri(ib, 2 * q)][slot]));
      const bf4 hi = read_tr(reinterpret_cast<const __bf16*>(&m[a][two ? tri(ib, 2 * q + 1) : 0][slot]));
      o.v[a] = cat(lo, two ? hi : zero);
    }
    return o;
  };
  Op<IN> qt[QB], kt[QB];  // columns of q and k: free n, contracted tokens
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    qt[q] = sh.q.template cols<>(32 * q, n0);
    kt[q] = sh.k.template cols<>(32 * q, n0);
  }
  f4 dq[TOK], dk[TOK];  // rows n, columns tokens
#pragma unroll
  for (int o = 0; o < TOK; ++o) {
    const int tb = SHARE * o + tb0, i = 16 * tb + r;
    f4 a = ia[o] * tok.eq[i], v = iv[o] * tok.er[i], d = id[o] * tok.wr[i];
    const f4 qi = sh.q.quad(i, n0 + 4 * g), ki = sh.k.quad(i, n0 + 4 * g);
    const f4 pa = a * qi - v * ki, pd = d * ki;
    const float sa = sum_col4((pa[0] + pa[1]) + (pa[2] + pa[3])), sd = sum_col4((pd[0] + pd[1]) + (pd[2] + pd[3]));
    d -= v;
#pragma unroll
    for (int q = 0; q < QB; ++q) {
      if (2 * q <= tb) {
        mma<MID>(a, kt[q], by_row(sh.x, tb, q));
        mma<MID>(d, kt[q], by_row(sh.y, tb, q));
      }
      if (2 * q + 1 >= tb) {
        mma<MID>(d, qt[q], by_col(sh.x, tb, q));
        mma<MID>(d, kt[q], by_col(sh.y, tb, q));
      }
    }
    dq[o] = a;
    dk[o] = d;
    const f4 qq = a * qi, kk = d * ki;
    const float sq = sum_col4((qq[0] + qq[1]) + (qq[2] + qq[3])), sk = sum_col4((kk[0] + kk[1]) + (kk[2] + kk[3]));
    if (g == 0) {
      sh.a[nb][i] = sa;
      sh.d[nb][i] = sd;
      sh.qd[nb][i] = sq;
      sh.kd[nb][i] = sk;
    }
  }
  __syncthreads();
#pragma unroll
  for (int o = 0; o < TOK; ++o) {
    const int tb = SHARE * o + tb0, i = 16 * tb + r;
    if (p.l2) {
      float sq = 0.f, sk = 0.f;
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        sq += sh.qd[k][i];
        sk += sh.kd[k][i];
      }
      dq[o] -= sh.q.quad(i, n0 + 4 * g) * (sq * tok.rq[i] * tok.rq[i]);
      dk[o] -= sh.k.quad(i, n0 + 4 * g) * (sk * tok.rk[i] * tok.rk[i]);
    }
    const int n = n0 + 4 * g;
    if (n < p.N && i < left) {
      const long long at = ((row0 + i) * p.G + grp) * p.N + n;
      if (p.dqp != nullptr) {
        const long long all = (long long)p.B * p.L * p.G * p.N;
        *reinterpret_cast<f4*>(p.dqp + (h - grp * HG) * all + at) = dq[o];
        *reinterpret_cast<f4*>(p.dkp + (h - grp * HG) * all + at) = dk[o];
      } else {
        store4(static_cast<T*>(p.dq) + at, dq[o]);
        store4(static_cast<T*>(p.dk) + at, dk[o]);
      }
    }
  }
  if (w != WAVES - 1) return;
  // the decays and b, lane t with token t
  const bool in = l < Q;
  const int t = in ? l : 0, tb = t >> 4, tr = t & 15;
  double passes = 0.0, reach = 0.0;  // sums of rows less columns and a; of d
  if (in) {
    for (int k = 0; k <= tb; ++k) passes += (double)sh.row[tri(tb, k)][tr];
    for (int k = tb; k < TB; ++k) passes -= (double)sh.col[tri(k, tb)][tr];
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      passes += (double)sh.a[k][t];
      reach += (double)sh.d[k][t];
    }
  }
  gh = 0.f;
#pragma unroll
  for (int k = 0; k < NB; ++k) gh += sh.gh[k];
  const double upto = lane_sums(passes), all = lane_value(upto, 63), before = lane_sums(reach) - reach;
  if (in && t < left) {
    const float dg = (float)((all - upto + passes) + before + (double)(tok.end * gh));
    const long long at = (row0 + t) * p.H + h;
    put<T>(p.dg, p.g_f32, at, dg);
    put<T>(p.dbeta, p.beta_f32, at, sh.db[t]);
  }
}

// q's and k's gradients of the heads that share them
template <typename T> __global__ __launch_bounds__(256) void delta_shared_kernel(DeltaParams p, long long quads, int n) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= 2 * quads) return;
  const bool second = id >= quads;
  const long long q = second ? id - quads : id;
  const float* s = (second ? p.dkp : p.dqp) + 4 * q;
  f4 v = *reinterpret_cast<const f4*>(s);
  for (int k = 1; k < n; ++k) v += *reinterpret_cast<const f4*>(s + 4 * k * quads);
  store4(static_cast<T*>(second ? p.dk : p.dq) + 4 * q, v);
}
template <typename T, int NP> hipError_t bwd_t(const DeltaParams& p, hipStream_t stream) {
  using Sh = GradShared<T, NP>;
  constexpr size_t lds = sizeof(Sh);
  static_assert(2 * lds <= 160 * 1024, "two workgroups to a compute unit");
  const hipError_t e = allow_lds(delta_bwd_kernel<T, NP>, lds);
  if (e != hipSuccess) return e;
  const long long blocks = (long long)p.B * ((p.L + Sh::Q - 1) / Sh::Q) * p.H;
  hipLaunchKernelGGL((delta_bwd_kernel<T, NP>), dim3((unsigned)blocks), dim3(64 * Sh::WAVES), lds, stream, p);
  if (p.dqp != nullptr) {
    const long long quads = (long long)p.B * p.L * p.G * p.N / 4;
    hipLaunchKernelGGL(delta_shared_kernel<T>, dim3((unsigned)((2 * quads + 255) / 256)), dim3(256), 0, stream, p, quads,
                       p.H / p.G);
  }
  return hipGetLastError();
}
template <typename T> hipError_t width_t(const DeltaParams& p, hipStream_t s) {
  return p.N <= 32 ? bwd_t<T, 32>(p, s) : p.N <= 64 ? bwd_t<T, 64>(p, s) : bwd_t<T, 128>(p, s);
}

}  // namespace

hipError_t launch_delta_bwd(const DeltaParams& p, int dtype, hipStream_t s) {
  return dtype == TTT_DTYPE_BF16 ? width_t<__bf16>(p, s)
         : dtype == TTT_DTYPE_F16 ? width_t<_Float16>(p, s) : width_t<float>(p, s);
}

}  // namespace ttt
