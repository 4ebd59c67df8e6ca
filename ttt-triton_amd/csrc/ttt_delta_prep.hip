// The gated delta rule's first launch on gfx950 (mathematics: ttt_delta.h): what a chunk's
// keys, queries, decays and steps b give without the state.  A workgroup of four waves has
// a chunk of one sequence and head:
//   A_ij = F_ij (k_i . k_j), j < i      by matrix instructions from the raw rows
//   Z = A - A b Z                       row by row in the blocks of 16 on the diagonal (one
//                                       wave, a block to its 16 lanes), then
//     Z_IJ = Y - Z_II b Y,  Y = A_IJ - sum_{J<=K<I} A_IK b Z_KJ
//                                       a wave to a column of blocks, in fp32 products
//   M_ij = s F_ij (q_i . k_j), j <= i
// Z and M are written in fp32 by blocks, as the walks' operands take them.
//
// 32,768 tokens of 12 heads of 64 x 64 in bf16: 64 us for 100 MB of q and k read and 138 MB written,
// 3.8 TB/s; bound by memory and by the solve's plain instructions (half of the time each).  A in the
// place of the rows makes that seven workgroups to a compute unit: 76 us with both side by side.
// The backward takes the forward's Z and M (walk back 20 us dearer by reads of 4 bytes, 3 with
// M's planes shared in LDS) in place of another launch of this kernel with transposed blocks (63 us).
#include <math.h>

#include "ttt_delta.h"

namespace ttt {

namespace {

template <typename T, int NP> struct PrepShared {
  static constexpr int IN = ScanType<T>::IN, Q = kDeltaQ<T>;
  union {  // A, then Z, in the place of the rows that it comes of: more workgroups to a compute unit
    struct {
      Planes<IN, Q, NP> k, q;
    };
    float a[Q][Q + 4];
  };
  DeltaTok<Q> tok;
  Decays<Q> dec;
  float nq[Q], nk[Q];
};

// the sums of the squares of a stage's rows
template <typename T, int ROWS, int COLS, int NT>
__device__ __forceinline__ void row_squares(const Stage<T, ROWS, COLS, NT>& s, float* out) {
  using St = Stage<T, ROWS, COLS, NT>;
  typedef T tv __attribute__((ext_vector_type(St::VE)));
#pragma unroll
  for (int i = 0; i < St::CNT; ++i) {
    const tv a = __builtin_bit_cast(tv, s.v[i]);
    float v = 0.f;
#pragma unroll
    for (int e = 0; e < St::VE; ++e) v = __builtin_fmaf((float)a[e], (float)a[e], v);
#pragma unroll
    for (int m = 1; m < St::PER; m *= 2) v += __shfl_xor(v, m);
    if (St::has() && St::col(i) == 0) out[St::row(i)] = v;
  }
}

template <typename T, int NP> __global__ __launch_bounds__(256) void delta_prep_kernel(DeltaParams p) {
  using Sh = PrepShared<T, NP>;
  constexpr int IN = Sh::IN, Q = Sh::Q, TB = Q / 16, NC2 = NP / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Sh& sh = *reinterpret_cast<Sh*>(smem);
  const int w = wave_id(), l = lane_id(), g = l >> 4, r = l & 15;
  const int NC = (p.L + Q - 1) / Q;
  const unsigned id = on_xcd(blockIdx.x, gridDim.x);
  const int h = (int)(id % p.H), c = (int)(id / p.H % NC), b = (int)(id / p.H / NC), grp = h / (p.H / p.G);
  const int t0 = c * Q, left = min(Q, p.L - t0);
  const long long row0 = (long long)b * p.L + t0, chunk = ((long long)b * p.H + h) * NC + c;

  {
    Stage<T, Q, NP, 256> sk, sq;
    sk.place(p.ldk, p.N);
    sq.place(p.ldq, p.N);
    sk.load(static_cast<const T*>(p.k) + row0 * p.ldk + (long long)grp * p.N, left);
    sq.load(static_cast<const T*>(p.q) + row0 * p.ldq + (long long)grp * p.N, left);
    if (w == 3) {
      float gv = 0.f, bv = 0.f;
      if (l < left) {
        gv = bounded_decay(token_value<T>(p.g, p.g_f32, (row0 + l) * p.ldg + h));
        bv = token_value<T>(p.beta, p.beta_f32, (row0 + l) * p.ldbeta + h);
      }
      sh.dec.fill(gv, 1.f);
      if (l < Q) sh.tok.beta[l] = bv;
    }
    sk.store(sh.k);
    sq.store(sh.q);
    if (p.l2) {
      row_squares(sk, sh.nk);
      row_squares(sq, sh.nq);
    }
  }
  __syncthreads();
  if (threadIdx.x < Q) {
    const int t = threadIdx.x;
    const float rk = p.l2 ? 1.0f / sqrtf(sh.nk[t] + kUnitEps) : 1.f, rq = p.l2 ? 1.0f / sqrtf(sh.nq[t] + kUnitEps) : 1.f;
    sh.tok.hi[t] = sh.dec.hi[t];
    sh.tok.lo[t] = sh.dec.lo[t];
    sh.tok.rk[t] = rk;
    sh.tok.rq[t] = rq;
    sh.tok.er[t] = sh.dec.head[t] * rk;
    sh.tok.wr[t] = sh.dec.tail[t] * rk;
    sh.tok.eq[t] = sh.dec.head[t] * rq * p.scale;
    if (t == 0) sh.tok.end = sh.dec.end;
  }
  __syncthreads();
  const DeltaTok<Q>& tok = sh.tok;
  static_assert(sizeof(DeltaTok<Q>) == delta_tok_floats(Q) * 4, "as the workspace has it");
  for (int i = threadIdx.x; i < delta_tok_floats(Q) / 4; i += 256)
    reinterpret_cast<f4*>(p.tok + chunk * delta_tok_floats(Q))[i] = reinterpret_cast<const f4*>(&tok)[i];

  // F_ij over a tile's rows (tokens tr..) and its column tc; the rows are tokens i, or j
  const auto decays = [&](int tr, int tc, bool rows_later) {
    const f4 h4 = tok.four(tok.hi, tr), l4 = tok.four(tok.lo, tr);
    const float hc = tok.hi[tc], lc = tok.lo[tc];
    f4 f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = (h4[e] - hc) + (l4[e] - lc);
      f[e] = __builtin_amdgcn_exp2f(rows_later ? x : -x);
    }
    return f;
  };
  // A, tiles of rows i and columns j
  constexpr int TILES = TB * (TB + 1) / 2, OWN = (TILES + 3) / 4;
  f4 at[OWN];
#pragma unroll
  for (int u = 0; u < OWN; ++u) {
    const int t = w + 4 * u;
    if (t >= TILES) break;
    const int ib = tri_row(t), jb = t - tri(ib, 0);
    f4 acc = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < NC2; ++q) mma<kFull>(acc, sh.k.rows(16 * ib, 32 * q), sh.k.rows(16 * jb, 32 * q));
    const int i = 16 * ib + 4 * g, j = 16 * jb + r;
    acc *= decays(i, j, true) * tok.four(tok.rk, i) * tok.rk[j];
#pragma unroll
    for (int e = 0; e < 4; ++e) at[u][e] = only_if(j < i + e, acc[e]);
  }
  // M: rows j, columns i
  float* mp = p.m + chunk * (TILES * 256);
#pragma unroll
  for (int t = w; t < TILES; t += 4) {
    const int ib = tri_row(t), jb = t - tri(ib, 0);  // blocks of q and of k
    f4 acc = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < NC2; ++q) mma<kFull>(acc, sh.k.rows(16 * jb, 32 * q), sh.q.rows(16 * ib, 32 * q));
    const int j = 16 * jb + 4 * g, i = 16 * ib + r;
    acc *= decays(j, i, false) * tok.four(tok.rk, j) * (tok.rq[i] * p.scale);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = only_if(j + e <= i, acc[e]);
    *reinterpret_cast<f4*>(mp + (t * 64 + l) * 4) = acc;
  }
  __syncthreads();  // the rows have been read
#pragma unroll
  for (int u = 0; u < OWN; ++u) {
    const int t = w + 4 * u;
    if (t >= TILES) break;
    const int ib = tri_row(t), jb = t - tri(ib, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) sh.a[16 * ib + 4 * g + e][16 * jb + r] = at[u][e];
  }
  __syncthreads();
  // the blocks of Z on the diagonal: lane (g, r) has column r of block g
  if (w == 0 && g < TB) {
    float z[16], y[16];  // y = b z
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      f4 row[4];
#pragma unroll
      for (int j = 0; j < i; j += 4) row[j / 4] = *reinterpret_cast<const f4*>(&sh.a[16 * g + i][16 * g + j]);
      float s[2] = {sh.a[16 * g + i][16 * g + r], 0.f};
#pragma unroll
      for (int j = 0; j < i; ++j) s[j & 1] = __builtin_fmaf(-row[j / 4][j & 3], y[j], s[j & 1]);
      z[i] = s[0] + s[1];
      y[i] = z[i] * tok.beta[16 * g + i];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) sh.a[16 * g + i][16 * g + r] = z[i];
  }
  __syncthreads();
  // the blocks below them: wave w has the column of blocks w
  f4 zt[TB];
  const auto left_op = [&](int ib, int kb) {  // free row, contracted columns
    return Frag<float>{*reinterpret_cast<const f4*>(&sh.a[16 * ib + r][16 * kb + 4 * g])};
  };
  if (w < TB - 1) {
#pragma unroll
    for (int I = 0; I < TB; ++I) {
      if (I < w) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) zt[I][e] = sh.a[16 * I + 4 * g + e][16 * w + r];
      if (I == w) continue;
      f4 acc = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int K = 0; K < I; ++K)
        if (K >= w) mma16(acc, left_op(I, K), Frag<float>{zt[K] * tok.four(tok.beta, 16 * K + 4 * g)});
      const f4 y = zt[I] - acc;
      f4 by[1] = {y * tok.four(tok.beta, 16 * I + 4 * g)};
      acc = f4{0.f, 0.f, 0.f, 0.f};
      // A token that is not finite reaches the rows behind it alone: 0 times it is no 0
      const int bad = first_not_finite(by);
      if (__ballot(bad < 16) != 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) by[0][e] = 4 * g + e < bad ? by[0][e] : 0.f;
      }
      mma16(acc, left_op(I, I), Frag<float>{by[0]});
      zt[I] = y - acc;
      if (__ballot(bad < 16) != 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) zt[I][e] = 4 * g + e < bad ? zt[I][e] : __builtin_nanf("");
      }
    }
  }
  __syncthreads();
  if (w < TB - 1) {
#pragma unroll
    for (int I = 0; I < TB; ++I)
      if (I > w)
#pragma unroll
        for (int e = 0; e < 4; ++e) sh.a[16 * I + 4 * g + e][16 * w + r] = zt[I][e];
  }
  __syncthreads();
  float* zp = p.z + chunk * (TILES * 256);
#pragma unroll
  for (int t = w; t < TILES; t += 4) {
    const int ib = tri_row(t), jb = t - tri(ib, 0);
    const f4 v = *reinterpret_cast<const f4*>(&sh.a[16 * ib + r][16 * jb + 4 * g]);
    *reinterpret_cast<f4*>(zp + (t * 64 + l) * 4) = v;
  }
}

template <typename T, int NP> hipError_t prep_t(const DeltaParams& p, hipStream_t stream) {
  constexpr size_t lds = sizeof(PrepShared<T, NP>);
  static_assert(lds <= 160 * 1024, "LDS of a compute unit");
  constexpr int Q = kDeltaQ<T>;
  const hipError_t e = allow_lds(delta_prep_kernel<T, NP>, lds);
  if (e != hipSuccess) return e;
  const long long blocks = (long long)p.B * p.H * ((p.L + Q - 1) / Q);
  hipLaunchKernelGGL((delta_prep_kernel<T, NP>), dim3((unsigned)blocks), dim3(256), lds, stream, p);
  return hipGetLastError();
}
template <typename T> hipError_t width_t(const DeltaParams& p, hipStream_t s) {
  return p.N <= 32 ? prep_t<T, 32>(p, s) : p.N <= 64 ? prep_t<T, 64>(p, s) : prep_t<T, 128>(p, s);
}

}  // namespace

hipError_t launch_delta_prep(const DeltaParams& p, int dtype, hipStream_t s) {
  return dtype == TTT_DTYPE_BF16 ? width_t<__bf16>(p, s)
         : dtype == TTT_DTYPE_F16 ? width_t<_Float16>(p, s) : width_t<float>(p, s);
}

}  // namespace ttt
