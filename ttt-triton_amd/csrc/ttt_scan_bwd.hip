// The selective scan's backward on gfx950 beside its walk back (ttt_scan_walk.hip):
// the gradients of B, C, the steps and the rates (mathematics and layouts: ttt_scan.h).
//
// Given the states H entering the chunks (kept by the forward) and the gradients Gam
// of those leaving them (kept by the walk back), every chunk stands alone.  With F_ij =
// e^{c_i - c_j} for j <= i, 0 elsewhere, e_i = e^{c_i}, w_j = e^{c_Q - c_j}:
//   dB_j = sum_i W_ij C_i + d_j w_j Gam^T x_j,    W_ij = F_ij d_j (x_j . dy_i)
//   dC_i = sum_j W_ij B_j + e_i H^T dy_i
// dB and dC are sums over a group's heads: a workgroup has a chunk and goes over the
// heads with both in registers, and C_i . B_j, which all heads share, too.
//
// The gradient of a decay a_t is what passes it: from tokens before t to tokens from
// t on, from H to tokens from t on, from tokens before t to Gam, and from H to Gam:
//   da_t = sum_{j<t<=i} W_ij (C_i . B_j) + sum_{i>=t} u_i + sum_{j<t} v_j + e^{c_Q} <Gam, H>
//   u_i = e_i C_i . (H^T dy_i),   v_j = d_j w_j B_j . (Gam^T x_j)
// (the first sum by its blocks of 16 x 16, so that nothing is a difference of sums: the
// block that t crosses, the rows from t on of the blocks left of it, the columns before t
// of those below it, and the blocks left and below), and the step's
//   dd_t = sum_{i>=t} F_it (x_t . dy_i) (C_i . B_t) + w_t B_t . (Gam^T x_t) + A da_t
//
// At 32,768 tokens of 12 heads of 64 x 64 in bf16: 106 us, 308 MB (two states of 16 KB to
// a chunk and head are 201 of them; 2.9 TB/s).  Loads and stores alone take 76, the arithmetic
// alone 82: per head ten 16 x 16 tiles of x . dy with their exponentials, row and column
// sums, then the products into dB and dC, with three barriers between them and eight waves a
// compute unit (237 registers).
#include <math.h>
#include <stddef.h>

#include "ttt_scan.h"

namespace ttt {

namespace {

// Waves for 16 features, one or two: two where a workgroup has two waves for its features
// and the state of each is small, and where one would hold two planes of everything (but not
// where a compute unit then has one workgroup in place of two: fp16, 32 x 64).
// us with one and with two, 32,768 tokens (fp32 16,384), 12 heads of 64 or 24 of 32:
//              N 32        64        128
//   P 32 bf16  163 124   177 157   249 308
//        fp16  192 136   210 270   320 426
//        fp32  120 102   154 135   185 278
//   P 64 bf16   84 114   101 142   193 303
//        fp16   94 128   197 164   242 327
//        fp32   74 103    91 129   172 230
template <typename T, int P, int NP>
constexpr int kRoles = P == 32 ? (NP == 32 || (NP == 64 && ScanType<T>::IN != 2) ? 2 : 1)
                               : (NP == 64 && ScanType<T>::IN == 2 ? 2 : 1);

// Whether a wave adds up its columns' shares of u and v before they go to LDS.  32,768 tokens, us
// without and with: 24 heads of 32 x 64 in fp16 417 and 209 (two workgroups a compute unit in place of
// one, by 1.4 KB of LDS), in bf16 186 and 177, of 32 x 128 273 and 249; but 12 of 64 x 128 in fp16 242
// and 304 (four registers more than two workgroups have).
template <typename T, int P, int NP> constexpr bool kByWave = !(ScanType<T>::IN == 2 && P == 64 && NP == 128);

template <typename T, int P, int NP> struct BwdShared {
  static constexpr int IN = ScanType<T>::IN, MID = ScanType<T>::MID, Q = chunk_of<T, NP>(), TB = Q / 16;
  static constexpr int W = P / 16, TILES = TB * (TB + 1) / 2, NB = NP / 16;
  Planes<IN, Q, P> x, dy;
  Planes<IN, Q, NP> b, c;
  bf4 wv[MID][TILES][64];  // W, tile rows i, columns j
  Decays<Q> dec[3];        // of the head before, this one and the next
  // What is left of a head for the gradient of its steps: of W (C . B) by tiles the sums of
  // the columns, before d_j, and of the rows (of a block that meets itself what crosses its
  // tokens), and shares of u_i and of v_j / d_j by a wave's columns or by 16 columns
  static constexpr int PARTS = kByWave<T, P, NP> && W < NB ? W : NB;
  struct alignas(16) Head {
    float row[TILES][16], col[TILES][16];
    float u[PARTS][Q], v[PARTS][Q];
    float dD[W * kRoles<T, P, NP>], gh[W];
  } head[2];
};

// Columns n = 16 nb + r of a state [NP][P] in memory, all P values of them: lane (g, r)
// has values 32k + 8g + e of column r
template <int P> struct StateColumns {
  static constexpr int K = P / 32;
  f4 v[K][2];
  __device__ __forceinline__ void load(const float* __restrict__ s, int nb) {
    const int l = lane_id(), g = l >> 4, r = l & 15;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int o = 0; o < 2; ++o) v[k][o] = *reinterpret_cast<const f4*>(s + (16 * nb + r) * P + 32 * k + 8 * g + 4 * o);
  }
  __device__ __forceinline__ Op<kFull> op(int k) const {
    return split8<kFull>(v[k][0], v[k][1]);
  }
  __device__ __forceinline__ float dot(const StateColumns& o) const {
    f4 s = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; ++k) s += v[k][0] * o.v[k][0] + v[k][1] * o.v[k][1];
    return (s[0] + s[1]) + (s[2] + s[3]);
  }
};

// sums over a row of 16 lanes from its first lane to this one, and from this one to its last
template <int CTRL> __device__ __forceinline__ float dpp0(float x) {  // 0 from outside the row
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float row_upto(float x) {
  x += dpp0<0x111>(x);  // row_shr:1, 2, 4, 8
  x += dpp0<0x112>(x);
  x += dpp0<0x114>(x);
  return x + dpp0<0x118>(x);
}
__device__ __forceinline__ float row_from(float x) {
  x += dpp0<0x101>(x);  // row_shl:1, 2, 4, 8
  x += dpp0<0x102>(x);
  x += dpp0<0x104>(x);
  return x + dpp0<0x108>(x);
}
__device__ __forceinline__ float lane_read(float x, int l) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l));
}

template <typename T> __device__ __forceinline__ void put_dt(const ScanParams& p, long long o, float v) {
  if (p.dt_f32)
    static_cast<float*>(p.ddt)[o] = v;
  else
    static_cast<T*>(p.ddt)[o] = (T)v;
}

// A head's steps, from its sums in LDS, by one wave (lane t with token t): the gradients
// of dt, and the chunk's part of those of A, D and dt_bias
template <typename T, int P, int NP>
__device__ __forceinline__ void steps_grad(const ScanParams& p, const BwdShared<T, P, NP>& sh, unsigned bits, int h,
                                           long long row0, int left, long long chunk) {
  using Sh = BwdShared<T, P, NP>;
  constexpr int Q = Sh::Q, TB = Sh::TB, NB = Sh::NB, W = Sh::W;
  const typename Sh::Head& s = sh.head[h & 1];
  const Decays<Q>& dec = sh.dec[h % 3];
  const int l = lane_id();
  const bool in = l < Q;
  const int t = in ? l : 0, tb = t >> 4, tr = t & 15;
  float u = 0.f, v = 0.f, dir = 0.f, gh = 0.f, dsum = 0.f, before = 0.f, past = 0.f, over = 0.f;
  if (in) {
    for (int k = tb + 1; k < TB; ++k) before += s.col[tri(k, tb)][tr];
#pragma unroll
    for (int k = 0; k < Sh::PARTS; ++k) {
      u += s.u[k][t];
      v += s.v[k][t];
    }
    past = s.row[tri(tb, tb)][tr];
    dir = (s.col[tri(tb, tb)][tr] + before) + v;
  }
#pragma unroll
  for (int k = 0; k < W; ++k) {
    if (k < NB) gh += s.gh[k];  // (waves that share a block of columns count it once)
  }
#pragma unroll
  for (int k = 0; k < W * kRoles<T, P, NP>; ++k) dsum += s.dD[k];
  // rows from t on of the blocks left of t's, and whole blocks left of and below it
  const float d = in ? dec.d[t] : 0.f;
#pragma unroll
  for (int jb = 0; jb + 1 < TB; ++jb) {
    float rows = in && jb < tb ? s.row[tri(tb, jb)][tr] : 0.f;
    rows = row_from(rows);  // the row's lanes from this one on
    past += rows;
#pragma unroll
    for (int ib = jb + 2; ib < TB; ++ib) {
      const float all = lane_read(rows, 16 * ib);
      if (tb > jb && tb < ib) over += all;
    }
  }
  before *= d;
  past += row_upto(dpp0<0x111>(before)) + over;
  v *= d;
  const double run = lane_sums(u), all = lane_value(run, 63);
  const float da = past + (float)(all - run + (double)u) + (float)(lane_sums(v) - (double)v) + dec.end * gh;
  float dr = 0.f;
  if (in && t < left) {
    const float raw = dt_value<T>(p, bits, p.dt_bias != nullptr ? p.dt_bias[h] : 0.f);
    dr = (dir + p.A[h] * da) * (p.softplus ? sigmoid_f(raw) : 1.0f);
    put_dt<T>(p, (row0 + t) * p.H + h, dr);
  }
  const float sa = sum_wave(in && t < left ? d * da : 0.f), sr = sum_wave(dr);
  if (l == 0) {
    const long long n = (long long)p.B * ((p.L + Q - 1) / Q), o = (long long)h * n + chunk;
    p.partial[o] = sa;
    p.partial[(long long)p.H * n + o] = dsum;
    p.partial[2LL * p.H * n + o] = sr;
  }
}

// A wave for every 16 features has dB and dC of its columns; with ROLES = 2 there are two,
// the first P/16 waves with dB and the others with dC
template <typename T, int P, int NP, int ROLES>
__global__ __launch_bounds__(4 * P * ROLES) void scan_bwd_kernel(ScanParams p) {
  using Sh = BwdShared<T, P, NP>;
  static_assert(offsetof(Sh, dec) % 16 == 0 && sizeof(Sh::dec[0]) % 16 == 0 && offsetof(Sh, head) % 16 == 0 &&
                    sizeof(Sh::head[0]) % 16 == 0 && offsetof(Sh, dy) % 16 == 0 && offsetof(Sh, b) % 16 == 0 &&
                    offsetof(Sh, c) % 16 == 0 && offsetof(Sh, wv) % 16 == 0,
                "read and written 16 bytes at a time");
  constexpr int IN = Sh::IN, MID = Sh::MID, Q = Sh::Q, TB = Sh::TB, W = Sh::W, NB = Sh::NB, NC2 = NP / 32;
  constexpr int WAVES = W * ROLES, NT = 64 * WAVES, BOTH = 3 - ROLES;
  constexpr int TILES = Sh::TILES, OWN = (TILES + WAVES - 1) / WAVES;
  // A wave's part of dB or dC: with as many blocks of 16 columns as waves for it, or more,
  // all tokens of its blocks; else one block and every SHARE-th 16 tokens
  constexpr int COLS = NB >= W ? NB / W : 1, SHARE = NB >= W ? 1 : W / NB, TOK = TB / SHARE;
  static_assert(COLS * W * TOK == NB * TB, "whole shares");
  constexpr bool BY_WAVE = kByWave<T, P, NP>;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Sh& sh = *reinterpret_cast<Sh*>(smem);
  const int w = wave_id(), l = lane_id(), g = l >> 4, r = l & 15;
  const int wr = ROLES == 2 && w >= W ? w - W : w, nb0 = SHARE == 1 ? wr : wr % NB, tb0 = SHARE == 1 ? 0 : wr / NB;
  const bool hasB = w < W, hasC = ROLES == 1 || !hasB;
  const int NC = (p.L + Q - 1) / Q, HG = p.H / p.G, per = (HG + p.splits - 1) / p.splits;
  int id = blockIdx.x;
  const int split = id % p.splits;
  id /= p.splits;
  const int grp = id % p.G;
  id /= p.G;
  const int c = id % NC, b = id / NC;
  const int t0 = c * Q, left = min(Q, p.L - t0);
  const long long row0 = (long long)b * p.L + t0, chunk = (long long)b * NC + c;
  const int h0 = grp * HG + split * per, h1 = min(grp * HG + HG, h0 + per);

  Stage<T, Q, P, NT> sx, sdy;
  StateColumns<P> st[BOTH][COLS];  // Gam and H, or the role's
  sx.place(p.ldx, P);
  sdy.place(p.ldy, P);
  const T* xp = static_cast<const T*>(p.x) + row0 * p.ldx;
  const T* dyp = static_cast<const T*>(p.dy) + row0 * p.ldy;
  const auto tokens = [&](int h) {
    sx.load(xp + h * P, left);
    sdy.load(dyp + h * P, left);
  };
  const auto state_of = [&](int h) { return (((long long)b * p.H + h) * NC + c) * (long long)(P * NP); };
  const auto states = [&](int h, int which) {
#pragma unroll
    for (int q = 0; q < COLS; ++q)
      st[BOTH == 1 ? 0 : which][q].load((which == 0 ? p.gstates : p.states) + state_of(h), nb0 + W * q);
  };
  // Steps are read two heads ahead and decays formed one ahead, while the tiles are; the
  // wave that forms them and the one that finishes the head before have the fewest tiles
  const bool fills = w == WAVES - 2, ends = w == WAVES - 1;
  const auto bits_of = [&](int h) {
    return (fills || ends) && h < h1 && l < left ? dt_bits<T>(p, row0 + l, h) : 0u;
  };
  const auto decays = [&](int h, unsigned bits) {
    const float raw = dt_value<T>(p, bits, p.dt_bias != nullptr ? p.dt_bias[h] : 0.f);
    sh.dec[h % 3].fill(l < left ? (p.softplus ? softplus_f(raw) : raw) : 0.f, p.A[h]);
  };
  unsigned bits0 = 0, bits1 = 0, bits2 = 0;  // of the head before, this one and the next
  if (h0 < h1) {
    bits1 = bits_of(h0);
    bits2 = bits_of(h0 + 1);
    Stage<T, Q, NP, NT> sb, sc;
    sb.place(p.ldb, p.N);
    sc.place(p.ldc, p.N);
    sb.load(static_cast<const T*>(p.Bm) + row0 * p.ldb + grp * p.N, left);
    sc.load(static_cast<const T*>(p.Cm) + row0 * p.ldc + grp * p.N, left);
    tokens(h0);
    if (hasB) states(h0, 0);
    if (hasC) states(h0, 1);
    sb.store(sh.b);
    sc.store(sh.c);
    if (fills) decays(h0, bits1);
  }
  __syncthreads();
  f4 cb[OWN];  // C_i . B_j, rows i
#pragma unroll
  for (int k = 0; k < OWN; ++k) {
    const int t = w + WAVES * k, ib = tri_row(t), jb = t - tri(ib, 0);
    cb[k] = f4{0.f, 0.f, 0.f, 0.f};
    if (t < TILES) {
#pragma unroll
      for (int q = 0; q < NC2; ++q) mma<kFull>(cb[k], sh.c.rows(16 * ib, 32 * q), sh.b.rows(16 * jb, 32 * q));
    }
  }
  f4 sum[BOTH][COLS][TOK];  // dB and dC, or the role's
#pragma unroll
  for (int z = 0; z < BOTH; ++z)
#pragma unroll
    for (int q = 0; q < COLS; ++q)
#pragma unroll
      for (int s = 0; s < TOK; ++s) sum[z][q][s] = f4{0.f, 0.f, 0.f, 0.f};
  const bf4 zero = {(__bf16)0.f, (__bf16)0.f, (__bf16)0.f, (__bf16)0.f};

  for (int h = h0; h < h1; ++h) {
    typename Sh::Head& hd = sh.head[h & 1];
    const Decays<Q>& dec = sh.dec[h % 3];
    sx.store(sh.x);
    sdy.store(sh.dy);
    // The sum of x dy, for dD: not from the diagonal of the tiles below.  The matrix
    // instruction's sums are cut off rather than rounded, which adds up over the tokens of
    // all sequences: 1.0e-6 off that way at 16,384 tokens, 4 heads of 32
    float xdy = sx.dot(sdy);
    __syncthreads();
    if (h + 1 < h1) {
      if (fills) decays(h + 1, bits2);
      tokens(h + 1);
    }
    if (ends && h > h0) steps_grad<T, P, NP>(p, sh, bits0, h - 1, row0, left, chunk);
    bits0 = bits1;
    bits1 = bits2;
    bits2 = bits_of(h + 2);
    if (hasC && tb0 == 0) {  // <Gam, H>
      float s = 0.f;
#pragma unroll
      for (int q = 0; q < COLS; ++q) {
        if constexpr (BOTH == 2) {
          s += st[0][q].dot(st[1][q]);
        } else {
          StateColumns<P> gam;
          gam.load(p.gstates + state_of(h), nb0 + W * q);
          s += gam.dot(st[0][q]);
        }
      }
      s = sum_wave(s);
      if (l == 0) hd.gh[wr] = s;
    }

#pragma unroll
    for (int k = 0; k < OWN; ++k) {
      const int t = w + WAVES * k, ib = tri_row(t), jb = t - tri(ib, 0);
      if (t < TILES) {
        f4 xy = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < P / 32; ++q) mma<kFull>(xy, sh.dy.rows(16 * ib, 32 * q), sh.x.rows(16 * jb, 32 * q));
        const int j = 16 * jb + r, i0 = 16 * ib + 4 * g;
        const float jh = dec.hi[j], jl = dec.lo[j], d = dec.d[j];
        const f4 ih = dec.four(dec.hi, i0), il = dec.four(dec.lo, i0);
        f4 wv;
#pragma unroll
        for (int e = 0; e < 4; ++e) wv[e] = __builtin_amdgcn_exp2f((ih[e] - jh) + (il[e] - jl)) * xy[e];
        if (ib == jb) {
#pragma unroll
          for (int e = 0; e < 4; ++e) wv[e] = only_if(4 * g + e >= r, wv[e]);
        }
        f4 pass = wv * cb[k];
        bf4 ow[MID];
        split4<MID>(wv * d, ow);
#pragma unroll
        for (int a = 0; a < MID; ++a) sh.wv[a][t][l] = ow[a];
        const float cs = sum_col4((pass[0] + pass[1]) + (pass[2] + pass[3]));
        if (g == 0) hd.col[t][r] = cs;
        pass *= d;
        if (ib == jb) {  // from row 4g + e on, by columns, then the columns before it
          pass[2] += pass[3];
          pass[1] += pass[2];
          pass[0] += pass[1];
          const float b1 = __shfl_down(pass[0], 16), b2 = __shfl_down(pass[0], 32), b3 = __shfl_down(pass[0], 48);
          pass += (g < 3 ? b1 : 0.f) + (g < 2 ? b2 : 0.f) + (g < 1 ? b3 : 0.f);
#pragma unroll
          for (int e = 0; e < 4; ++e) pass[e] = r < 4 * g + e ? pass[e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) pass[e] = sum_row16(pass[e]);
        if (r == 0) *reinterpret_cast<f4*>(&hd.row[t][4 * g]) = pass;
      }
    }
    xdy = sum_wave(xdy);
    if (l == 0) hd.dD[w] = xdy;
    __syncthreads();

    if (hasB) {  // rows are columns n of B, columns tokens j
      Op<kFull> s[COLS][P / 32];
#pragma unroll
      for (int q = 0; q < COLS; ++q)
#pragma unroll
        for (int k = 0; k < P / 32; ++k) s[q][k] = st[0][q].op(k);
      if (h + 1 < h1) states(h + 1, 0);
      float part[TOK] = {};
#pragma unroll
      for (int q = 0; q < COLS; ++q) {
        const int n0 = 16 * (nb0 + W * q);
        Op<IN> ct[Q / 32];
#pragma unroll
        for (int k = 0; k < Q / 32; ++k) ct[k] = sh.c.template cols<>(32 * k, n0);
#pragma unroll
        for (int o = 0; o < TOK; ++o) {
          const int jb = SHARE * o + tb0, j = 16 * jb + r;
          f4 acc = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < P / 32; ++k) mma<kFull>(acc, s[q][k], sh.x.rows(16 * jb, 32 * k));
          acc *= dec.tail[j];
          const f4 vv = acc * sh.b.quad(j, n0 + 4 * g);
          part[o] = (BY_WAVE ? part[o] : 0.f) + ((vv[0] + vv[1]) + (vv[2] + vv[3]));
          if (!BY_WAVE || q + 1 == COLS) {
            const float sv = sum_col4(part[o]);
            if (g == 0) hd.v[BY_WAVE ? nb0 : nb0 + W * q][j] = sv;
          }
          sum[0][q][o] += acc * dec.d[j];
#pragma unroll
          for (int k = 0; k < Q / 32; ++k) {
            if (2 * k + 1 < jb) continue;
            const bool one = 2 * k >= jb;
            Op<MID> m;
#pragma unroll
            for (int a = 0; a < MID; ++a)
              m.v[a] = cat(one ? sh.wv[a][one ? tri(2 * k, jb) : 0][l] : zero, sh.wv[a][tri(2 * k + 1, jb)][l]);
            mma<MID>(sum[0][q][o], ct[k], m);
          }
        }
      }
    }
    if (hasC) {  // rows are columns n of C, columns tokens i
      constexpr int Z = BOTH - 1;
      Op<kFull> s[COLS][P / 32];
#pragma unroll
      for (int q = 0; q < COLS; ++q)
#pragma unroll
        for (int k = 0; k < P / 32; ++k) s[q][k] = st[Z][q].op(k);
      if (h + 1 < h1) states(h + 1, 1);
      float part[TOK] = {};
#pragma unroll
      for (int q = 0; q < COLS; ++q) {
        const int n0 = 16 * (nb0 + W * q);
        Op<IN> bt[Q / 32];
#pragma unroll
        for (int k = 0; k < Q / 32; ++k) bt[k] = sh.b.template cols<>(32 * k, n0);
#pragma unroll
        for (int o = 0; o < TOK; ++o) {
          const int ib = SHARE * o + tb0, i = 16 * ib + r;
          f4 acc = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < P / 32; ++k) mma<kFull>(acc, s[q][k], sh.dy.rows(16 * ib, 32 * k));
          acc *= dec.head[i];
          const f4 uu = acc * sh.c.quad(i, n0 + 4 * g);
          part[o] = (BY_WAVE ? part[o] : 0.f) + ((uu[0] + uu[1]) + (uu[2] + uu[3]));
          if (!BY_WAVE || q + 1 == COLS) {
            const float su = sum_col4(part[o]);
            if (g == 0) hd.u[BY_WAVE ? nb0 : nb0 + W * q][i] = su;
          }
          sum[Z][q][o] += acc;
          // W as an operand with free i and contraction j: the transposing read of its tiles,
          // whose lane 16 a + j holds rows 4a..4a+3 of column j
          const int slot = 16 * (l & 3) + 4 * g + (r >> 2);
#pragma unroll
          for (int k = 0; k < Q / 32; ++k) {
            if (2 * k > ib) continue;
            const bool two = 2 * k + 1 <= ib;
            Op<MID> m;
#pragma unroll
            for (int a = 0; a < MID; ++a) {
              const bf4 lo = read_tr(reinterpret_cast<const __bf16*>(&sh.wv[a][tri(ib, 2 * k)][slot]));
              const bf4 hi = read_tr(reinterpret_cast<const __bf16*>(&sh.wv[a][two ? tri(ib, 2 * k + 1) : 0][slot]));
              m.v[a] = cat(lo, two ? hi : zero);
            }
            mma<MID>(sum[Z][q][o], bt[k], m);
          }
        }
      }
    }
    __syncthreads();
  }
  if (ends && h0 < h1) steps_grad<T, P, NP>(p, sh, bits0, h1 - 1, row0, left, chunk);

#pragma unroll
  for (int z = 0; z < BOTH; ++z)
#pragma unroll
    for (int q = 0; q < COLS; ++q)
#pragma unroll
      for (int s = 0; s < TOK; ++s) {
        const int n = 16 * (nb0 + W * q) + 4 * g, j = 16 * (SHARE * s + tb0) + r;
        const bool ofB = BOTH == 2 ? z == 0 : hasB;
        if (n < p.N && t0 + j < p.L) {
          const long long o = ((row0 + j) * p.G + grp) * p.N + n;
          float* part = ofB ? p.dBp : p.dCp;
          if (part != nullptr)
            *reinterpret_cast<f4*>(part + split * ((long long)p.B * p.L * p.G * p.N) + o) = sum[z][q][s];
          else
            store4(static_cast<T*>(ofB ? p.dB : p.dC) + o, sum[z][q][s]);
        }
      }
}

// dB and dC of a group whose heads were split over workgroups
template <typename T> __global__ __launch_bounds__(256) void scan_groups_kernel(ScanParams p, long long quads) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= 2 * quads) return;
  const bool second = id >= quads;
  const long long q = second ? id - quads : id;
  const float* s = (second ? p.dCp : p.dBp) + 4 * q;
  f4 v = *reinterpret_cast<const f4*>(s);
  for (int k = 1; k < p.splits; ++k) v += *reinterpret_cast<const f4*>(s + 4 * k * quads);
  store4(static_cast<T*>(second ? p.dC : p.dB) + 4 * q, v);
}

// dA, dD and ddt_bias: the sums over the chunks of all sequences, a workgroup each
__global__ __launch_bounds__(256) void scan_param_grads_kernel(ScanParams p, int n) {
  const int k = blockIdx.x / p.H, h = blockIdx.x - k * p.H;
  float* out = k == 0 ? p.dA : k == 1 ? p.dD : p.ddt_bias;
  if (out == nullptr) return;
  const float* s = p.partial + (long long)blockIdx.x * n;
  double v = 0.0;  // (chunks' sums cancel, those of dA and the bias above all)
  for (int i = threadIdx.x; i < n; i += 256) v += (double)s[i];
#pragma unroll
  for (int k = 32; k > 0; k /= 2) v += __shfl_xor(v, k);
  __shared__ double red[4];
  if (lane_id() == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) out[h] = (float)(((red[0] + red[1]) + red[2]) + red[3]);
}

template <typename T, int P, int NP> hipError_t bwd_t(const ScanParams& p, hipStream_t stream) {
  constexpr size_t lds = sizeof(BwdShared<T, P, NP>);
  static_assert(lds <= 160 * 1024, "LDS of a compute unit");
  constexpr int Q = chunk_of<T, NP>();
  const int NC = (p.L + Q - 1) / Q;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(scan_bwd_kernel<T, P, NP, kRoles<T, P, NP>>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  const long long blocks = (long long)p.B * NC * p.G * p.splits;
  hipLaunchKernelGGL((scan_bwd_kernel<T, P, NP, kRoles<T, P, NP>>), dim3((unsigned)blocks), dim3(4 * P * kRoles<T, P, NP>),
                     lds, stream, p);
  if (p.dBp != nullptr) {
    const long long quads = (long long)p.B * p.L * p.G * p.N / 4;
    hipLaunchKernelGGL(scan_groups_kernel<T>, dim3((unsigned)((2 * quads + 255) / 256)), dim3(256), 0, stream, p, quads);
  }
  hipLaunchKernelGGL(scan_param_grads_kernel, dim3(3 * p.H), dim3(256), 0, stream, p, p.B * NC);
  return hipGetLastError();
}
template <typename T, int P> hipError_t width_t(const ScanParams& p, hipStream_t s) {
  return p.N <= 32 ? bwd_t<T, P, 32>(p, s) : p.N <= 64 ? bwd_t<T, P, 64>(p, s) : bwd_t<T, P, 128>(p, s);
}
template <typename T> hipError_t head_t(const ScanParams& p, int P, hipStream_t s) {
  return P == 64 ? width_t<T, 64>(p, s) : P == 32 ? width_t<T, 32>(p, s) : hipErrorInvalidValue;
}

// One token of every sequence: h = e^{dA} h + d x (x) B in place, y = h C + D x.  The
// state is read and written once, which bounds it; LANES lanes have a feature's row of
// the state, four values each, and add up their share of h C.  64 sequences, 12 heads of 64 x 64:
// 10.3 us for 25 MB from HBM (2.4 TB/s; one round of loads, latency), one sequence 4 us, a launch.
template <typename T, int LANES> __global__ __launch_bounds__(256) void scan_step_kernel(ScanStepParams p, long long rows) {
  const long long row = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;  // (b, h, feature)
  if (row >= rows) return;  // (whole groups of LANES)
  const int n = 4 * (threadIdx.x & (LANES - 1)), f = (int)(row % p.P);
  const long long bh = row / p.P;
  const long long b = bh / p.H;
  const int h = (int)(bh - b * p.H), grp = h / (p.H / p.G);
  const bool in = n < p.N;
  f4 hs = f4{0.f, 0.f, 0.f, 0.f}, bv = hs, cv = hs;
  float* hp = p.h + row * p.N + n;
  if (in) {
    hs = *reinterpret_cast<const f4*>(hp);
    bv = load4(static_cast<const T*>(p.Bm) + b * p.ldb + (long long)grp * p.N + n);
    cv = load4(static_cast<const T*>(p.Cm) + b * p.ldc + (long long)grp * p.N + n);
  }
  const float x = (float)static_cast<const T*>(p.x)[b * p.ldx + (long long)h * p.P + f];
  float d = p.dt_f32 ? static_cast<const float*>(p.dt)[b * p.lddt + h] : (float)static_cast<const T*>(p.dt)[b * p.lddt + h];
  if (p.dt_bias != nullptr) d += p.dt_bias[h];
  if (p.softplus) d = softplus_f(d);
  hs = hs * __builtin_amdgcn_exp2f(d * p.A[h] * 1.4426950408889634f) + bv * (d * x);
  if (in) *reinterpret_cast<f4*>(hp) = hs;
  const f4 y = hs * cv;
  float s = (y[0] + y[1]) + (y[2] + y[3]);
#pragma unroll
  for (int k = LANES / 2; k > 0; k /= 2) s += __shfl_xor(s, k);
  if (n == 0) {
    if (p.D != nullptr) s = __builtin_fmaf(p.D[h], x, s);
    static_cast<T*>(p.y)[row] = (T)s;
  }
}
template <typename T, int LANES> hipError_t step_t(const ScanStepParams& p, hipStream_t stream) {
  const long long rows = (long long)p.B * p.H * p.P;
  constexpr int per = 256 / LANES;
  hipLaunchKernelGGL((scan_step_kernel<T, LANES>), dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, stream, p, rows);
  return hipGetLastError();
}
template <typename T> hipError_t step_lanes(const ScanStepParams& p, hipStream_t s) {
  return p.N <= 16   ? step_t<T, 4>(p, s)
         : p.N <= 32 ? step_t<T, 8>(p, s)
         : p.N <= 64 ? step_t<T, 16>(p, s)
                     : step_t<T, 32>(p, s);
}

}  // namespace

hipError_t launch_scan_bwd(const ScanParams& p, int P, int dtype, hipStream_t s) {
  return dtype == TTT_DTYPE_BF16 ? head_t<__bf16>(p, P, s)
         : dtype == TTT_DTYPE_F16 ? head_t<_Float16>(p, P, s) : head_t<float>(p, P, s);
}
hipError_t launch_scan_step(const ScanStepParams& p, int dtype, hipStream_t s) {
  return dtype == TTT_DTYPE_BF16 ? step_lanes<__bf16>(p, s)
         : dtype == TTT_DTYPE_F16 ? step_lanes<_Float16>(p, s) : step_lanes<float>(p, s);
}

}  // namespace ttt
