// The gated delta rule's walks along a sequence on gfx950 (mathematics and layouts:
// ttt_delta.h): forwards the outputs and the states, backwards dv and the gradients of the
// states.
//
// A workgroup walks 16 W features of one sequence and head, chunk by chunk.  W waves have 16 of
// them each, with their part of the state in registers, and go through what a chunk's state needs
// of the one before it alone.  The features do not meet, and each product's result is, where it
// lies, an operand of the next, without LDS or barriers in between:
//   S (rows n) -> K S (rows tokens) -> r -> Z b r -> x -> u -> S' = e^{c_Q} S + K^T u
// W more waves do the rest beside them: they bring the next chunk's rows to LDS, and forwards
// form the outputs of the chunk before (transposed, rows features, from S, Q and u, M) from the
// state's planes and x, backwards the next chunk's M^T do and Q^T do; both are handed over through
// LDS.  A barrier ends a chunk; another one, in its course, lets what was handed over be written
// again.
//
// 32,768 tokens in 16 sequences of 12 heads of 64 x 64 in bf16: 190 us forward and 177 back (190 with
// branches around its loads, which waits then count as none), 192 workgroups at once with 32
// chunks each, 5.9 us (12,600 clocks) a chunk and 2.8 TB/s.  A chunk's chain bounds it:
// 84 matrix instructions and 550 plain ones with 45 waits in a wave that has the state, 34 and 500 in
// the wave beside it on the SIMD; together they fill half of the issue slots.
//
// States of more than 64 are walked by 32 features, four waves to a workgroup.  In fp32 the rows of k on
// their way in the forward's helping waves (eight 16-byte values a lane) lie in scratch memory there, 336
// bytes a lane, though no register spills: 32,768 tokens of 12 heads of 128 x 128, forward, 2,960 us, where fp16
// takes 730 and bf16 470 (64 x 64: 281, 200 and 185 through the public call).
//
// Where there are few sequences and heads, the tokens are cut into segments.  A segment takes
// the state S that enters it to T S + E, with T = prod e^{g_t} (1 - b_t k_t (x) k_t): a first walk
// without outputs, of all segments at once, gives E from the state 0 and T from the columns of
// the identity, as features without values; one launch goes over the segments with their
// products (delta_join_kernel), and then all segments are walked at once.  Back, a segment takes
// the gradient dS' to T^T dS' + E', with the forward's T.
#include <math.h>
#include <stddef.h>

#include <type_traits>

#include "ttt_buf.h"
#include "ttt_delta.h"

namespace ttt {

namespace {

template <typename T, int W, int NP, bool BACK, bool OUT> struct WalkShared {
  static constexpr int IN = ScanType<T>::IN, MID = ScanType<T>::MID, Q = kDeltaQ<T>, PAIRS = delta_pairs(Q);
  static constexpr int TB = Q / 16, NB = NP / 16, NC2 = NP / 32;
  struct alignas(16) Side {  // a chunk's, in turn
    Planes<IN, Q, NP> k;
    bf8 z[kFull][PAIRS][64];
    DeltaTok<Q> tok;
    Planes<IN, BACK ? 1 : Q, 16 * W> v;
  } side[2];
  // backwards the chunk's that the helpers form M^T do and Q^T do of
  Planes<IN, BACK ? Q : 1, NP> q;
  Planes<IN, BACK ? Q : 1, 16 * W> dO;
  // and its M, which all waves take; of 3 blocks each wave has its own from memory
  static constexpr bool MS = BACK && Q == 64;
  bf8 m[MS ? kFull : 1][MS ? PAIRS : 1][MS ? 64 : 1];
  // what is handed over
  static constexpr bool YS = OUT && !BACK;
  bf8 s[YS ? W : 1][YS ? MID : 1][YS ? NC2 : 1][YS ? 64 : 1];
  f4 x[YS ? W : 1][YS ? TB : 1][YS ? 64 : 1];
  f4 md[BACK ? W : 1][BACK ? TB : 1][BACK ? 64 : 1], qd[BACK ? W : 1][BACK ? NB : 1][BACK ? 64 : 1];
};

// a chunk's blocks of Z on their way from memory to operands in planes
template <int Q, int W, bool BACK> struct Blocks {
  static constexpr int ALL = delta_tiles(Q), CNT = (ALL + W - 1) / W;
  f4 v[CNT];
  __device__ __forceinline__ void load(const float* p, int w) {
#pragma unroll
    for (int i = 0; i < CNT; ++i)
      if (i * W + w < ALL) v[i] = tile_at<BACK>(p, i * W + w);
  }
  __device__ __forceinline__ void store(bf8 (*to)[delta_pairs(Q)][64], int w) const {
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int t = i * W + w;
      if (t >= ALL) continue;
      const int hb = tri_row(t), lb = t - tri(hb, 0), blk = BACK ? lb : hb, in = BACK ? hb : lb;
      bf4 o[kFull];
      split4<kFull>(v[i], o);
#pragma unroll
      for (int a = 0; a < kFull; ++a)
        reinterpret_cast<bf4*>(&to[a][pair_at(BACK, Q, blk, in / 2)][lane_id()])[in & 1] = o[a];
    }
  }
};
// a chunk's blocks of M in a wave's registers, as operands
template <int Q, bool BACK> struct Masked {
  f4 v[delta_tiles(Q)];
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int t = 0; t < delta_tiles(Q); ++t) v[t] = tile_at<BACK>(p, t);
  }
  // of the free block b, contracted blocks 2q and 2q + 1
  template <int PL> __device__ __forceinline__ Op<PL> op(int b, int q) const {
    const auto tile = [&](int in) {
      const bool has = meets(BACK, b, in);
      return has ? v[has ? (BACK ? tri(in, b) : tri(b, in)) : 0] : f4{0.f, 0.f, 0.f, 0.f};
    };
    return split8<PL>(tile(2 * q), tile(2 * q + 1));
  }
};
// floats on their way to LDS as they lie in memory
template <int FLOATS, int NT> struct Copy {
  static constexpr int ALL = FLOATS / 4, CNT = (ALL + NT - 1) / NT;
  f4 v[CNT];
  __device__ __forceinline__ static int at(int i) { return i * NT + (int)threadIdx.x; }
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int o = at(i);
      if (o < ALL) v[i] = reinterpret_cast<const f4*>(p)[o];
    }
  }
  __device__ __forceinline__ void store(float* p) const {
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int o = at(i);
      if (o < ALL) reinterpret_cast<f4*>(p)[o] = v[i];
    }
  }
};

// (dropped past the buffer's range)
template <typename E> __device__ __forceinline__ void bstore_one(rsrc_t r, int voff, int soff, E v) {
  if constexpr (sizeof(E) == 2)
    __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(short, v), r, voff, soff, 0);
  else
    bstore_f32(r, voff, soff, v);
}

// what StateTiles::keep wrote
template <int NP> __device__ __forceinline__ void take_kept(StateTiles<NP>& st, const float* __restrict__ s, int ld, int w) {
  const int l = lane_id();
#pragma unroll
  for (int i = 0; i < NP / 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) st.t[i][e] = s[(StateTiles<NP>::col(i >> 1) + 4 * (i & 1) + e) * ld + 16 * w + (l & 15)];
}

// a row's eight values as an operand in planes
template <typename T> __device__ __forceinline__ Op<ScanType<T>::IN> row_op(const T* p) {
  constexpr int IN = ScanType<T>::IN;
  if constexpr (IN == 1) {
    Op<1> o;
    o.v[0] = *reinterpret_cast<const bf8*>(p);
    return o;
  } else {
    return split8<IN>(load4(p), load4(p + 4));
  }
}

// workgroups that have the columns of the identity between them
constexpr int identity_groups(int W, int NP) { return (NP + 16 * W - 1) / (16 * W); }
// segments whose products are formed: those before the last, and where a way back follows that too
__host__ __device__ __forceinline__ int product_segments(const DeltaParams& p) { return p.states != nullptr ? p.S : p.S - 1; }

// OUT: outputs too; else the segments' ends alone
template <typename T, int W, int NP, bool BACK, bool OUT>
__global__ __launch_bounds__(128 * W) void delta_walk_kernel(DeltaParams p) {
  using Sh = WalkShared<T, W, NP, BACK, OUT>;
  static_assert(offsetof(Sh, q) % 16 == 0 && offsetof(Sh, dO) % 16 == 0 && offsetof(Sh, m) % 16 == 0 && offsetof(Sh, s) % 16 == 0 &&
                    offsetof(Sh, x) % 16 == 0 && offsetof(typename Sh::Side, z) % 16 == 0 &&
                    offsetof(typename Sh::Side, tok) % 16 == 0 && offsetof(typename Sh::Side, v) % 16 == 0,
                "read 16 bytes at a time");
  constexpr int IN = Sh::IN, MID = Sh::MID, Q = Sh::Q, TB = Sh::TB, QB = Q / 32, NT = 64 * W, NC2 = Sh::NC2, NB = Sh::NB;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Sh& sh = *reinterpret_cast<Sh*>(smem);
  const bool helps = wave_id() < W;  // (a stage's threads are a workgroup's first)
  const int w = helps ? wave_id() : wave_id() - W, l = lane_id(), g = l >> 4, r = l & 15;
  const int PB = delta_part(p.P), parts = p.P / PB, cols = PB / (16 * W), NC = (p.L + Q - 1) / Q;
  const unsigned at = on_xcd(blockIdx.x, gridDim.x);
  // groups of columns to a head: of its features, and for the segments' products of the identity
  const int own = parts * cols, groups = own + (OUT || BACK ? 0 : identity_groups(W, NP));
  const int segs = OUT ? p.S : BACK ? p.S - 1 : product_segments(p);
  const int grp_c = (int)(at % groups);
  const int s = (int)(at / groups % segs) + (!OUT && BACK ? 1 : 0);
  const long long head = at / groups / segs;  // sequence and head
  const bool features = OUT || BACK || grp_c < own;
  if (!OUT && !BACK && features && s == p.S - 1) return;  // (the way back takes its product alone)
  const int b = (int)(head / p.H), h = (int)(head - (long long)b * p.H), grp = h / (p.H / p.G);
  const int part = features ? grp_c / cols : 0, f0 = features ? 16 * W * (grp_c % cols) : 16 * W * (grp_c - own);
  const int hp = h * parts + part;
  const long long chain = head * parts + part;  // f0: the first feature in the part, or column of the identity
  const long long ldo = (long long)p.H * p.P;
  const int c0 = s * p.per, n = min(NC, c0 + p.per) - c0;
  const auto chunk_of = [&](int k) { return BACK ? c0 + n - 1 - k : c0 + k; };
  const auto first_row = [&](int c) { return (long long)b * p.L + (long long)c * Q; };
  // (an operand's half beside the triangle stays 0)
  for (int i = threadIdx.x; i < 2 * (int)sizeof(Sh::Side::z) / 16; i += 2 * NT) {
    const int side = i >= (int)sizeof(Sh::Side::z) / 16, o = i - side * (int)sizeof(Sh::Side::z) / 16;
    reinterpret_cast<f4*>(&sh.side[side].z)[o] = f4{0.f, 0.f, 0.f, 0.f};
  }
  if constexpr (Sh::MS)
    for (int i = threadIdx.x; i < (int)sizeof(Sh::m) / 16; i += 2 * NT) reinterpret_cast<f4*>(&sh.m)[i] = f4{0.f, 0.f, 0.f, 0.f};
  __syncthreads();

  if (helps) {
    const T* K = static_cast<const T*>(p.k) + (long long)grp * p.N;
    const T* Qr = static_cast<const T*>(p.q) + (long long)grp * p.N;
    const long long ldv = BACK ? p.lddo : p.ldv;
    const T* V = static_cast<const T*>(BACK ? p.dO : p.v) + (features ? (long long)hp * PB + f0 : 0);
    Stage<T, Q, NP, NT> sk, sq;
    Stage<T, Q, 16 * W, NT> sv;
    Blocks<Q, W, BACK> bz, bm;
    Copy<delta_tok_floats(Q), NT> ct;
    Masked<Q, BACK> m;
    sk.place(p.ldk, p.N);
    sq.place(p.ldq, p.N);
    sv.place(ldv, 16 * W);
    // what the other waves take of a chunk
    const auto fetch = [&](int c) {
      const int left = min(Q, p.L - c * Q);
      sk.load(K + first_row(c) * p.ldk, left);
      if constexpr (!BACK) sv.load(V + first_row(c) * ldv, features ? left : 0);
      bz.load(p.z + (head * NC + c) * (delta_tiles(Q) * 256), w);
      ct.load(p.tok + (head * NC + c) * delta_tok_floats(Q));
    };
    const auto put = [&](typename Sh::Side& to) {
      sk.store(to.k);
      if constexpr (!BACK) sv.store(to.v);
      bz.store(to.z, w);
      ct.store(to.tok.hi);
    };
    if constexpr (!BACK) {
      Op<IN> qr[TB][NC2];  // rows of q
      // (rows and columns past the last ones are those again: nothing that is written comes of them)
      const auto fetch_out = [&](int c) {
        m.load(p.m + (head * NC + c) * (delta_tiles(Q) * 256));
        const int last = min(Q, p.L - c * Q) - 1;
#pragma unroll
        for (int ob = 0; ob < TB; ++ob)
#pragma unroll
          for (int q = 0; q < NC2; ++q)
            qr[ob][q] = row_op<T>(Qr + (first_row(c) + min(16 * ob + r, last)) * p.ldq + min(32 * q + 8 * g, p.N - 8));
      };
      // What is asked for past the last chunk is the last one again, and outputs past the last
      // token are dropped by the buffers' ranges: no branches, so that a wait for loads waits for
      // nothing that was sent after them
      const auto stage = [&](int k) {
        put(sh.side[(k + 1) & 1]);
        fetch(chunk_of(min(k + 2, n - 1)));
      };
      fetch(chunk_of(0));
      put(sh.side[0]);
      fetch(chunk_of(min(1, n - 1)));
      if (OUT) fetch_out(chunk_of(0));
      __syncthreads();
      __syncthreads();
      stage(0);
      __syncthreads();
#pragma unroll 1
      for (int k = 1; k <= n; ++k) {
        if constexpr (!OUT) {
          __syncthreads();
          stage(k);
          __syncthreads();
          continue;
        }
        // the outputs of the chunk before
        const DeltaTok<Q>& tok = sh.side[(k - 1) & 1].tok;
        Op<MID> so[NC2];
        f4 x[TB], u[TB];
        float eq[TB];
#pragma unroll
        for (int q = 0; q < NC2; ++q)
#pragma unroll
          for (int a = 0; a < MID; ++a) so[q].v[a] = sh.s[w][a][q][l];
#pragma unroll
        for (int ob = 0; ob < TB; ++ob) {
          x[ob] = sh.x[w][ob][l];
          u[ob] = x[ob] * tok.four(tok.beta, 16 * ob + 4 * g);
          eq[ob] = tok.eq[16 * ob + r];
        }
        __syncthreads();  // what was handed over has been read
        const int c = chunk_of(k - 1), left = min(Q, p.L - c * Q);
        // (x is no number from the first token on whose row is not finite: below)
        const int bad = any_not_finite(x) ? first_not_finite(x) : Q;
        if (__ballot(bad < Q) != 0) {
#pragma unroll
          for (int ob = 0; ob < TB; ++ob)
#pragma unroll
            for (int e = 0; e < 4; ++e) u[ob][e] = 16 * ob + 4 * g + e < bad ? u[ob][e] : 0.f;
        }
        f4 y[TB];
#pragma unroll
        for (int ob = 0; ob < TB; ++ob) {
          y[ob] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int q = 0; q < NC2; ++q) mma<MID>(y[ob], so[q], qr[ob][q]);
          y[ob] *= eq[ob];
        }
        Op<MID> uo[QB];
#pragma unroll
        for (int q = 0; q < QB; ++q) uo[q] = split8<MID>(u[2 * q], u[2 * q + 1]);
#pragma unroll
        for (int ob = 0; ob < TB; ++ob)
#pragma unroll
          for (int q = 0; q < QB; ++q)
            if (meets(false, ob, 2 * q)) mma<MID>(y[ob], uo[q], m.template op<MID>(ob, q));
        if (__ballot(bad < Q) != 0) {  // (a lane has the features 4g + e of a token here)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int first = __shfl(bad, 4 * g + e);
#pragma unroll
            for (int ob = 0; ob < TB; ++ob) y[ob][e] = 16 * ob + r < first ? y[ob][e] : __builtin_nanf("");
          }
        }
        fetch_out(chunk_of(min(k, n - 1)));
        const rsrc_t rows = make_rsrc(p.rows + ((chain * NC + c) * Q) * PB + f0 + 16 * w,
                                      p.rows != nullptr ? (unsigned)(Q * PB * 4) : 0u);
        const int at_row = (4 * g * PB + r) * 4, at_o = (r * (int)ldo + 4 * g) * (int)sizeof(T);
#pragma unroll
        for (int ob = 0; ob < TB; ++ob)
#pragma unroll
          for (int e = 0; e < 4; ++e) bstore_f32(rows, at_row + (16 * ob + e) * PB * 4, 0, x[ob][e]);
        const rsrc_t out = make_rsrc(static_cast<T*>(p.o) + first_row(c) * ldo + (long long)hp * PB + f0 + 16 * w,
                                     (unsigned)left * (unsigned)ldo * (unsigned)sizeof(T));
#pragma unroll
        for (int ob = 0; ob < TB; ++ob)
          bstore_frag<T>(out, at_o + 16 * ob * (int)ldo * (int)sizeof(T), 0, to_frag<T>(y[ob]));
        stage(k);
        __syncthreads();
      }
    } else {
      const auto fetch_do = [&](int c) {
        const int left = min(Q, p.L - c * Q);
        sq.load(Qr + first_row(c) * p.ldq, left);
        sv.load(V + first_row(c) * ldv, features ? left : 0);
        if constexpr (Sh::MS) bm.load(p.m + (head * NC + c) * (delta_tiles(Q) * 256), w);
      };
      f4 eq[QB][2];
      const auto fetch_own = [&](int c) {
        if constexpr (!Sh::MS) m.load(p.m + (head * NC + c) * (delta_tiles(Q) * 256));
        const float* of = p.tok + (head * NC + c) * delta_tok_floats(Q) + 7 * Q + 4 * g;
#pragma unroll
        for (int q = 0; q < QB; ++q)
#pragma unroll
          for (int o = 0; o < 2; ++o) eq[q][o] = *reinterpret_cast<const f4*>(of + 32 * q + 16 * o);
      };
      const auto put_do = [&] {
        sq.store(sh.q);
        sv.store(sh.dO);
        if constexpr (Sh::MS) bm.store(sh.m, w);
      };
      // M^T do and Q^T do, the latter with its factors
      f4 md[TB], qd[NB];
      const auto form = [&] {
        Op<IN> dt[QB];  // do: free feature, contracted token
#pragma unroll
        for (int q = 0; q < QB; ++q) dt[q] = sh.dO.template cols<>(32 * q, 16 * w);
#pragma unroll
        for (int ob = 0; ob < TB; ++ob) {
          md[ob] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int q = 0; q < QB; ++q)
            if (meets(true, ob, 2 * q + 1)) {
              Op<kFull> mo;
              if constexpr (Sh::MS) {
#pragma unroll
                for (int a = 0; a < kFull; ++a) mo.v[a] = sh.m[a][pair_at(true, Q, ob, q)][l];
              } else {
                mo = m.template op<kFull>(ob, q);
              }
              mma<kFull>(md[ob], mo, dt[q]);
            }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) qd[i] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < QB; ++q) {
          const Op<kFull> d = split8<kFull>(join4(dt[q], 0) * eq[q][0], join4(dt[q], 1) * eq[q][1]);
#pragma unroll
          for (int i = 0; i < NB; ++i) mma<kFull>(qd[i], sh.q.template cols<true>(32 * q, 32 * (i >> 1) + 4 * (i & 1)), d);
        }
      };
      const auto hand = [&] {
#pragma unroll
        for (int ob = 0; ob < TB; ++ob) sh.md[w][ob][l] = md[ob];
#pragma unroll
        for (int i = 0; i < NB; ++i) sh.qd[w][i][l] = qd[i];
      };
      fetch(chunk_of(0));
      fetch_do(chunk_of(0));
      fetch_own(chunk_of(0));
      put(sh.side[0]);
      put_do();
      __syncthreads();
      form();
      hand();
      // (past the last chunk it is the last one again, as forwards)
      const auto ask = [&](int k, const auto& f) { f(chunk_of(min(k, n - 1))); };
      ask(1, fetch);
      ask(1, fetch_do);
      ask(1, fetch_own);
      __syncthreads();
      put_do();
      __syncthreads();
#pragma unroll 1
      for (int k = 0; k < n; ++k) {
        ask(k + 2, fetch_do);
        form();
        ask(k + 2, fetch_own);
        __syncthreads();  // what was handed over has been read, and so have q and do
        hand();
        put(sh.side[(k + 1) & 1]);
        ask(k + 2, fetch);
        put_do();
        __syncthreads();
      }
    }
    return;
  }

  // (the segments' ends wait for these waves alone: 55 to 51 us of 16,384 tokens of 12 heads of 64 x 64;
  // with outputs the waves beside them are as long, and first place for either gains nothing)
  if (!OUT) __builtin_amdgcn_s_setprio(2);
  StateTiles<NP> st;
  if (!OUT) {
    st.load(nullptr, 0, 0, w);
    if (!BACK && !features) {
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) st.t[i][e] = StateTiles<NP>::col(i >> 1) + 4 * (i & 1) + e == f0 + 16 * w + r ? 1.f : 0.f;
    }
  } else if (p.S > 1) {
    take_kept(st, p.seg + (chain * p.S + s) * (NP * PB) + f0, PB, w);
  } else {
    st.load(p.h0 != nullptr ? p.h0 + (chain * PB + f0) * p.N : nullptr, p.N, p.N, w);
  }
  __syncthreads();
  if constexpr (BACK) {
    __syncthreads();
    __syncthreads();
  }
#pragma unroll 1
  for (int k = 0; k < n; ++k) {
    const int c = chunk_of(k);
    const typename Sh::Side& in = sh.side[k & 1];
    const DeltaTok<Q>& tok = in.tok;
    if (OUT && p.states != nullptr) st.keep(p.states + (chain * NC + c) * (long long)(NP * PB) + f0, PB, w);
    f4 t[TB];  // K S, rows tokens
#pragma unroll
    for (int ob = 0; ob < TB; ++ob) t[ob] = f4{0.f, 0.f, 0.f, 0.f};
    Op<kFull> so[NC2];
#pragma unroll
    for (int q = 0; q < NC2; ++q) {
      so[q] = st.template op<kFull>(q);
#pragma unroll
      for (int ob = 0; ob < TB; ++ob) mma<kFull>(t[ob], in.k.rows(16 * ob, 32 * q), so[q]);
    }
    f4 qd[BACK ? NB : 1];
    if constexpr (BACK) {  // du
#pragma unroll
      for (int ob = 0; ob < TB; ++ob) t[ob] = t[ob] * tok.four(tok.wr, 16 * ob + 4 * g) + sh.md[w][ob][l];
#pragma unroll
      for (int i = 0; i < NB; ++i) qd[i] = sh.qd[w][i][l];
    } else {  // r
#pragma unroll
      for (int q = 0; q < QB; ++q) {
        const Op<IN> v = in.v.template cols<>(32 * q, 16 * w);
#pragma unroll
        for (int o = 0; o < 2; ++o) t[2 * q + o] = join4(v, o) - t[2 * q + o] * tok.four(tok.er, 32 * q + 16 * o + 4 * g);
      }
    }
    if constexpr (!BACK) {
      __syncthreads();
      if constexpr (OUT) {
#pragma unroll
        for (int q = 0; q < NC2; ++q)
#pragma unroll
          for (int a = 0; a < MID; ++a) sh.s[w][a][q][l] = so[q].v[a];
      }
    }
    // x = r - Z b r, or y = du - Z^T b du
    Op<kFull> br[QB];
    int bad = Q;
    {
      f4 by[TB];
#pragma unroll
      for (int ob = 0; ob < TB; ++ob) by[ob] = t[ob] * tok.four(tok.beta, 16 * ob + 4 * g);
      if constexpr (!BACK) {
        // A token that is not finite reaches the tokens behind it alone: 0 times it is no 0
        if (any_not_finite(by)) bad = first_not_finite(by);
        if (__ballot(bad < Q) != 0) {
#pragma unroll
          for (int ob = 0; ob < TB; ++ob)
#pragma unroll
            for (int e = 0; e < 4; ++e) by[ob][e] = 16 * ob + 4 * g + e < bad ? by[ob][e] : 0.f;
        }
      }
#pragma unroll
      for (int q = 0; q < QB; ++q) br[q] = split8<kFull>(by[2 * q], by[2 * q + 1]);
    }
#pragma unroll
    for (int ob = 0; ob < TB; ++ob) {
      f4 s = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < QB; ++q)
        if (BACK ? meets(true, ob, 2 * q + 1) : meets(false, ob, 2 * q)) {
          Op<kFull> z;
#pragma unroll
          for (int a = 0; a < kFull; ++a) z.v[a] = in.z[a][pair_at(BACK, Q, ob, q)][l];
          mma<kFull>(s, z, br[q]);
        }
      t[ob] -= s;
    }
    if constexpr (!BACK) {
      if (__ballot(bad < Q) != 0) {
#pragma unroll
        for (int ob = 0; ob < TB; ++ob)
#pragma unroll
          for (int e = 0; e < 4; ++e) t[ob][e] = 16 * ob + 4 * g + e < bad ? t[ob][e] : __builtin_nanf("");
      }
      if constexpr (OUT) {
#pragma unroll
        for (int ob = 0; ob < TB; ++ob) sh.x[w][ob][l] = t[ob];
      }
    }
    f4 u[TB];  // b x, or dv
#pragma unroll
    for (int ob = 0; ob < TB; ++ob) u[ob] = t[ob] * tok.four(tok.beta, 16 * ob + 4 * g);
    if constexpr (BACK) {
      __syncthreads();
      if constexpr (OUT) {
        const int left = min(Q, p.L - c * Q), es = (int)sizeof(T);
        const rsrc_t rows = make_rsrc(p.rows + ((chain * NC + c) * Q) * PB + f0 + 16 * w, (unsigned)(Q * PB * 4));
        const rsrc_t out = make_rsrc(static_cast<T*>(p.o) + first_row(c) * ldo + (long long)hp * PB + f0 + 16 * w,
                                     (unsigned)left * (unsigned)ldo * (unsigned)es);
        const int at_row = (4 * g * PB + r) * 4, at_o = (4 * g * (int)ldo + r) * es;
#pragma unroll
        for (int ob = 0; ob < TB; ++ob) {
          const auto d = to_frag<T>(u[ob]).v;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            bstore_f32(rows, at_row + (16 * ob + e) * PB * 4, 0, t[ob][e]);
            bstore_one(out, at_o + (16 * ob + e) * (int)ldo * es, 0, d[e]);
          }
        }
      }
    }
    // the state behind the chunk, or the gradient of the one before it
    const float end = tok.end;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      st.t[i] *= end;
      if constexpr (BACK) st.t[i] += qd[i];
    }
#pragma unroll
    for (int q = 0; q < QB; ++q) {
      f4 d[2];
#pragma unroll
      for (int o = 0; o < 2; ++o)
        d[o] = BACK ? u[2 * q + o] * tok.four(tok.er, 32 * q + 16 * o + 4 * g) * -1.f
                    : u[2 * q + o] * tok.four(tok.wr, 32 * q + 16 * o + 4 * g);
      const Op<kFull> dk = split8<kFull>(d[0], d[1]);
#pragma unroll
      for (int i = 0; i < NB; ++i) mma<kFull>(st.t[i], in.k.template cols<true>(32 * q, 32 * (i >> 1) + 4 * (i & 1)), dk);
    }
    if constexpr (!BACK) {
      if (__ballot(bad < Q) != 0) {
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) st.t[i][e] = bad < Q ? __builtin_nanf("") : st.t[i][e];
      }
    }
    __syncthreads();
  }
  if constexpr (!BACK) {  // the helpers' last outputs
    __syncthreads();
    __syncthreads();
  }
  if (!OUT) {
    if (BACK || features)
      st.keep(p.seg + (chain * p.S + s) * (NP * PB) + f0, PB, w);
    else if (f0 + 16 * w < NP)  // (32 columns leave two of four waves without any)
      st.keep(p.trans + (head * p.S + s) * (NP * NP) + f0, NP, w);
  } else if (p.h_last != nullptr && s == (BACK ? 0 : p.S - 1)) {
    st.store(p.h_last + (chain * PB + f0) * p.N, p.N, p.N, w);
  }
}

// The segments' ends -> the states they start from, in place: a workgroup has 16 features of a
// part and goes over the segments, a wave to 16 rows of the state, which go from one to the next
// through LDS; the products of the next four are on their way (with one: 20 us for 20 segments of 64 x 64).
constexpr int kAhead = 4;
static_assert(kAhead % 2 == 0, "two places in turn");
template <int NP, bool BACK> __global__ __launch_bounds__(4 * NP) void delta_join_kernel(DeltaParams p) {
  constexpr int NB = NP / 16, NC2 = NP / 32;
  __shared__ Planes<kFull, 16, NP> sh[2];  // features by n
  const int w = wave_id(), l = lane_id(), g = l >> 4, r = l & 15;
  const int PB = delta_part(p.P), cols = PB / 16, parts = p.P / PB, f = 16 * (int)(blockIdx.x % cols) + r;
  const long long chain = blockIdx.x / cols, head = chain / parts;
  const int n = 16 * w + 4 * g;  // a lane's rows
  f4 st = f4{0.f, 0.f, 0.f, 0.f}, end;
  if (p.h0 != nullptr && n < p.N) st = *reinterpret_cast<const f4*>(p.h0 + (chain * PB + f) * p.N + n);
  const auto seg = [&](int k) { return BACK ? p.S - 1 - k : k; };
  const auto at = [&](int k) { return p.seg + (chain * p.S + seg(k)) * (NP * PB) + n * PB + f; };
  struct Segment {
    f4 a[NC2][2];  // row 16 w + r, columns 32q + 8g.., back of the transposed
    f4 end;
  } on[kAhead];
  // (past the last one that one again: no branches, so that a wait is for the oldest loads alone)
  const auto fetch = [&](Segment& to, int k) {
    k = min(k, p.S - 2);
    const float* t = p.trans + (head * p.S + seg(k)) * (NP * NP) + (BACK ? 8 * g * NP + 16 * w + r : (16 * w + r) * NP + 8 * g);
#pragma unroll
    for (int q = 0; q < NC2; ++q)
#pragma unroll
      for (int o = 0; o < 2; ++o)
        if constexpr (BACK) {
#pragma unroll
          for (int e = 0; e < 4; ++e) to.a[q][o][e] = t[(32 * q + 4 * o + e) * NP];
        } else {
          to.a[q][o] = *reinterpret_cast<const f4*>(t + 32 * q + 4 * o);
        }
#pragma unroll
    for (int e = 0; e < 4; ++e) to.end[e] = at(k)[e * PB];
  };
  const auto keep = [&](int k, f4 v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) at(k)[e * PB] = v[e];
  };
#pragma unroll
  for (int d = 0; d < kAhead; ++d) fetch(on[d], d);
  const auto go = [&](int k0, auto more) {
#pragma unroll
    for (int d = 0; d < kAhead; ++d) {
      const int k = k0 + d;
      if (!more && k + 1 >= p.S) break;
      Planes<kFull, 16, NP>& of = sh[d & 1];
      bf4 o[kFull];
      split4<kFull>(st, o);
#pragma unroll
      for (int q = 0; q < kFull; ++q) *reinterpret_cast<bf4*>(&of.d[q][r][n]) = o[q];
      Op<kFull> m[NC2];
#pragma unroll
      for (int q = 0; q < NC2; ++q) m[q] = split8<kFull>(on[d].a[q][0], on[d].a[q][1]);
      const f4 last = st;
      st = on[d].end;
      // (two places in turn: a wave is at most one segment ahead of another)
      __syncthreads();
      keep(k, last);
      if constexpr (more) fetch(on[d], k + kAhead);
#pragma unroll
      for (int q = 0; q < NC2; ++q) mma<kFull>(st, m[q], of.rows(0, 32 * q));
    }
  };
  int k = 0;
#pragma unroll 1
  for (; k + kAhead + 1 < p.S; k += kAhead) go(k, std::true_type{});
  go(k, std::false_type{});
  keep(p.S - 1, st);
}

template <typename T, int W, int NP, bool BACK> hipError_t walk_t(const DeltaParams& p, hipStream_t stream) {
  constexpr size_t lds = sizeof(WalkShared<T, W, NP, BACK, true>), lds1 = sizeof(WalkShared<T, W, NP, BACK, false>);
  static_assert(lds <= 160 * 1024, "LDS of a compute unit");
  hipError_t e = allow_lds(delta_walk_kernel<T, W, NP, BACK, true>, lds);
  if (e != hipSuccess) return e;
  const long long heads = (long long)p.B * p.H;
  if (p.S > 1) {
    e = allow_lds(delta_walk_kernel<T, W, NP, BACK, false>, lds1);
    if (e != hipSuccess) return e;
    const long long groups =
        BACK ? heads * (p.S - 1) * (p.P / (16 * W)) : heads * product_segments(p) * (p.P / (16 * W) + identity_groups(W, NP));
    hipLaunchKernelGGL((delta_walk_kernel<T, W, NP, BACK, false>), dim3((unsigned)groups), dim3(128 * W), lds1, stream, p);
    hipLaunchKernelGGL((delta_join_kernel<NP, BACK>), dim3((unsigned)(heads * p.P / 16)), dim3(4 * NP), 0, stream,
                       p);
  }
  hipLaunchKernelGGL((delta_walk_kernel<T, W, NP, BACK, true>), dim3((unsigned)(heads * p.S * p.P / (16 * W))), dim3(128 * W),
                     lds, stream, p);
  return hipGetLastError();
}
template <typename T, int W, bool BACK> hipError_t width_t(const DeltaParams& p, hipStream_t s) {
  return p.N <= 32 ? walk_t<T, W, 32, BACK>(p, s) : p.N <= 64 ? walk_t<T, W, 64, BACK>(p, s) : walk_t<T, 2, 128, BACK>(p, s);
}
template <typename T, bool BACK> hipError_t part_t(const DeltaParams& p, hipStream_t s) {
  return delta_part(p.P) == 64 ? width_t<T, 4, BACK>(p, s) : width_t<T, 2, BACK>(p, s);
}
template <bool BACK> hipError_t launch(const DeltaParams& p, int dtype, hipStream_t s) {
  return dtype == TTT_DTYPE_BF16 ? part_t<__bf16, BACK>(p, s)
         : dtype == TTT_DTYPE_F16 ? part_t<_Float16, BACK>(p, s) : part_t<float, BACK>(p, s);
}

// One token of every sequence, the state in place: the state is read and written once, which
// bounds it.  LANES lanes have a feature's row of it, four values each.  (64 sequences of 12 heads of
// 64 x 64: 25 MB in 10.3 us, 2.5 TB/s: one round of loads and a launch.)
template <typename T, int LANES> __global__ __launch_bounds__(256) void delta_step_kernel(DeltaStepParams p, long long rows) {
  const long long row = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;  // (b, h, feature)
  if (row >= rows) return;  // (whole groups of LANES)
  const int n = 4 * (threadIdx.x & (LANES - 1)), f = (int)(row % p.P);
  const long long bh = row / p.P, b = bh / p.H;
  const int h = (int)(bh - b * p.H), grp = h / (p.H / p.G);
  const bool in = n < p.N;
  f4 s = f4{0.f, 0.f, 0.f, 0.f}, k = s, q = s;
  float* hp = p.h + row * p.N + n;
  if (in) {
    s = *reinterpret_cast<const f4*>(hp);
    k = load4(static_cast<const T*>(p.k) + b * p.ldk + (long long)grp * p.N + n);
    q = load4(static_cast<const T*>(p.q) + b * p.ldq + (long long)grp * p.N + n);
  }
  const float v = (float)static_cast<const T*>(p.v)[b * p.ldv + (long long)h * p.P + f];
  const float a = __builtin_amdgcn_exp2f(1.4426950408889634f * token_value<T>(p.g, p.g_f32, b * p.ldg + h));
  const float beta = token_value<T>(p.beta, p.beta_f32, b * p.ldbeta + h);
  const auto dot = [](f4 x, f4 y) {
    const f4 z = x * y;
    float d = (z[0] + z[1]) + (z[2] + z[3]);
#pragma unroll
    for (int m = LANES / 2; m > 0; m /= 2) d += __shfl_xor(d, m);
    return d;
  };
  if (p.l2) {
    k *= 1.0f / sqrtf(dot(k, k) + kUnitEps);
    q *= 1.0f / sqrtf(dot(q, q) + kUnitEps);
  }
  s *= a;
  s += k * (beta * (v - dot(s, k)));
  if (in) *reinterpret_cast<f4*>(hp) = s;
  const float o = dot(s, q) * p.scale;
  if (n == 0) static_cast<T*>(p.o)[row] = (T)o;
}
template <typename T, int LANES> hipError_t step_t(const DeltaStepParams& p, hipStream_t stream) {
  const long long rows = (long long)p.B * p.H * p.P;
  constexpr int per = 256 / LANES;
  hipLaunchKernelGGL((delta_step_kernel<T, LANES>), dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, stream, p, rows);
  return hipGetLastError();
}
template <typename T> hipError_t step_lanes(const DeltaStepParams& p, hipStream_t s) {
  return p.N <= 16   ? step_t<T, 4>(p, s)
         : p.N <= 32 ? step_t<T, 8>(p, s)
         : p.N <= 64 ? step_t<T, 16>(p, s)
                     : step_t<T, 32>(p, s);
}

}  // namespace

hipError_t launch_delta_fwd(const DeltaParams& p, int dtype, hipStream_t s) { return launch<false>(p, dtype, s); }
hipError_t launch_delta_walk_back(const DeltaParams& p, int dtype, hipStream_t s) { return launch<true>(p, dtype, s); }
hipError_t launch_delta_step(const DeltaStepParams& p, int dtype, hipStream_t s) {
  return dtype == TTT_DTYPE_BF16 ? step_lanes<__bf16>(p, s)
         : dtype == TTT_DTYPE_F16 ? step_lanes<_Float16>(p, s) : step_lanes<float>(p, s);
}

}  // namespace ttt
