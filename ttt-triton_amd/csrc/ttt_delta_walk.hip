// The gated delta rule's walks along a sequence on gfx950 (mathematics and layouts:
// ttt_delta.h): forwards the outputs and the states, backwards dv and the gradients of the
// states.
//
// A workgroup walks 16 W features of one sequence and head, chunk by chunk; wave w has 16 of
// them, with their part of the state in registers.  The features do not meet: behind the one
// barrier at which a chunk's rows and operands are in LDS, a wave goes through its products
// by itself, and each product's result is, where it lies, an operand of the next:
//   S (rows n) -> K S (rows tokens) -> r -> Z b r -> x -> u -> S' = e^{c_Q} S + K^T u
// and the outputs, transposed (rows features), from S, Q and u, M.
//
// Where there are few sequences and heads, the tokens are cut into segments.  A segment takes
// the state S that enters it to T S + E, with T = prod e^{g_t} (1 - b_t k_t (x) k_t): a first walk
// without outputs, of all segments at once, gives E from the state 0 and T from the columns of
// the identity, as features without values; one launch goes over the segments with their
// products (delta_join_kernel), and then all segments are walked at once.
#include <math.h>
#include <stddef.h>

#include "ttt_delta.h"

namespace ttt {

namespace {

template <typename T, int W, int NP, bool BACK> struct WalkShared {
  static constexpr int IN = ScanType<T>::IN, Q = kDeltaQ<T>, PAIRS = delta_pairs(Q);
  static constexpr int MP = BACK || IN > 1 ? kFull : 2;
  Planes<IN, Q, NP> k, q;
  Planes<IN, Q, 16 * W> v;
  bf8 z[kFull][PAIRS][64], m[MP][PAIRS][64];
  DeltaTok<Q> tok;
};

// a chunk's blocks of Z or M on their way from memory to operands in planes
template <int Q, int W, bool BACK> struct Blocks {
  static constexpr int ALL = delta_tiles(Q), CNT = (ALL + W - 1) / W;
  f4 v[CNT];
  __device__ __forceinline__ void load(const float* p, int w) {
#pragma unroll
    for (int i = 0; i < CNT; ++i)
      if (i * W + w < ALL) v[i] = *reinterpret_cast<const f4*>(p + ((i * W + w) * 64 + lane_id()) * 4);
  }
  template <int PL> __device__ __forceinline__ void store(bf8 (*to)[delta_pairs(Q)][64], int w) const {
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int t = i * W + w;
      if (t >= ALL) continue;
      const int hb = tri_row(t), lb = t - tri(hb, 0), blk = BACK ? lb : hb, in = BACK ? hb : lb;
      bf4 o[PL];
      split4<PL>(v[i], o);
#pragma unroll
      for (int a = 0; a < PL; ++a)
        reinterpret_cast<bf4*>(&to[a][pair_at(BACK, Q, blk, in / 2)][lane_id()])[in & 1] = o[a];
    }
  }
};
// floats on their way to LDS as they lie in memory
template <int FLOATS, int NT> struct Copy {
  static constexpr int ALL = FLOATS / 4, CNT = (ALL + NT - 1) / NT;
  f4 v[CNT];
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int o = i * NT + (int)threadIdx.x;
      if (o < ALL) v[i] = reinterpret_cast<const f4*>(p)[o];
    }
  }
  __device__ __forceinline__ void store(float* p) const {
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int o = i * NT + (int)threadIdx.x;
      if (o < ALL) reinterpret_cast<f4*>(p)[o] = v[i];
    }
  }
};

// what StateTiles::keep wrote
template <int NP> __device__ __forceinline__ void take_kept(StateTiles<NP>& st, const float* __restrict__ s, int ld, int w) {
  const int l = lane_id();
#pragma unroll
  for (int i = 0; i < NP / 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) st.t[i][e] = s[(StateTiles<NP>::col(i >> 1) + 4 * (i & 1) + e) * ld + 16 * w + (l & 15)];
}

// OUT: outputs too; else the segments' ends alone
template <typename T, int W, int NP, bool BACK, bool OUT>
__global__ __launch_bounds__(64 * W) void delta_walk_kernel(DeltaParams p) {
  using Sh = WalkShared<T, W, NP, BACK>;
  static_assert(offsetof(Sh, q) % 16 == 0 && offsetof(Sh, v) % 16 == 0 && offsetof(Sh, z) % 16 == 0 &&
                    offsetof(Sh, m) % 16 == 0 && offsetof(Sh, tok) % 16 == 0,
                "read 16 bytes at a time");
  constexpr int IN = Sh::IN, MP = Sh::MP, Q = Sh::Q, TB = Q / 16, QB = Q / 32, NT = 64 * W, NC2 = NP / 32, NB = NP / 16;
  constexpr int MID = IN > 1 ? kFull : 2;
  constexpr bool READS = OUT || BACK;  // q and M
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Sh& sh = *reinterpret_cast<Sh*>(smem);
  const int w = wave_id(), l = lane_id(), g = l >> 4, r = l & 15;
  const int PB = delta_part(p.P), parts = p.P / PB, cols = PB / (16 * W), NC = (p.L + Q - 1) / Q;
  const unsigned at = on_xcd(blockIdx.x, gridDim.x);
  // groups of columns to a head: of its features, and without outputs of the identity behind them
  const int own = parts * cols, groups = own + (OUT ? 0 : NP / (16 * W)), segs = OUT ? p.S : p.S - 1;
  const int grp_c = (int)(at % groups);
  const int s = (int)(at / groups % segs) + (!OUT && BACK ? 1 : 0);
  const long long head = at / groups / segs;  // sequence and head
  const bool features = OUT || grp_c < own;
  const int b = (int)(head / p.H), h = (int)(head - (long long)b * p.H), grp = h / (p.H / p.G);
  const int part = features ? grp_c / cols : 0, f0 = features ? 16 * W * (grp_c % cols) : 16 * W * (grp_c - own);
  const int hp = h * parts + part;
  const long long chain = head * parts + part;  // f0: the first feature in the part, or column of the identity
  const T* K = static_cast<const T*>(p.k) + (long long)grp * p.N;
  const T* Qr = static_cast<const T*>(p.q) + (long long)grp * p.N;
  const long long ldv = BACK ? p.lddo : p.ldv;
  const T* V = static_cast<const T*>(BACK ? p.dO : p.v) + (features ? (long long)hp * PB + f0 : 0);
  T* O = static_cast<T*>(p.o) + (long long)hp * PB + f0;
  const long long ldo = (long long)p.H * p.P;
  const int c0 = s * p.per, n = min(NC, c0 + p.per) - c0;

  StateTiles<NP> st;
  if (!OUT) {
    st.load(nullptr, 0, 0, w);
    if (!features) {
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

  Stage<T, Q, NP, NT> sk, sq;
  Stage<T, Q, 16 * W, NT> sv;
  Blocks<Q, W, BACK> bz, bm;
  Copy<delta_tok_floats(Q), NT> ct;
  sk.place(p.ldk, p.N);
  sq.place(p.ldq, p.N);
  sv.place(ldv, 16 * W);
  const auto fetch = [&](int c) {
    const int left = min(Q, p.L - c * Q);
    const long long row = (long long)b * p.L + (long long)c * Q, chunk = head * NC + c;
    sk.load(K + row * p.ldk, left);
    sv.load(V + row * ldv, features ? left : 0);
    bz.load(p.z + chunk * (delta_tiles(Q) * 256), w);
    if constexpr (READS) {
      sq.load(Qr + row * p.ldq, left);
      bm.load(p.m + chunk * (delta_tiles(Q) * 256), w);
    }
    ct.load(p.tok + chunk * delta_tok_floats(Q));
  };
  const auto z_op = [&](int u) {
    Op<kFull> o;
#pragma unroll
    for (int a = 0; a < kFull; ++a) o.v[a] = sh.z[a][u][l];
    return o;
  };
  const auto m_op = [&](int u) {
    Op<MP> o;
#pragma unroll
    for (int a = 0; a < MP; ++a) o.v[a] = sh.m[a][u][l];
    return o;
  };
  const auto chunk_of_step = [&](int k) { return BACK ? c0 + n - 1 - k : c0 + k; };
  fetch(chunk_of_step(0));
  // (an operand's half beside the triangle stays 0)
  for (int i = threadIdx.x; i < (int)(offsetof(Sh, tok) - offsetof(Sh, z)) / 16; i += NT)
    reinterpret_cast<f4*>(&sh.z)[i] = f4{0.f, 0.f, 0.f, 0.f};
  __syncthreads();
#pragma unroll 1
  for (int k = 0; k < n; ++k) {
    const int c = chunk_of_step(k);
    if (k > 0) __syncthreads();  // the last chunk's readers are done
    sk.store(sh.k);
    sv.store(sh.v);
    bz.template store<kFull>(sh.z, w);
    if constexpr (READS) {
      sq.store(sh.q);
      bm.template store<MP>(sh.m, w);
    }
    ct.store(sh.tok.hi);
    __syncthreads();
    if (k + 1 < n) fetch(chunk_of_step(k + 1));
    if (OUT && p.states != nullptr) st.keep(p.states + (chain * NC + c) * (long long)(NP * PB) + f0, PB, w);
    const DeltaTok<Q>& tok = sh.tok;
    const int left = p.L - c * Q;
    const long long row = (long long)b * p.L + (long long)c * Q;

    f4 t[TB];  // K S, rows tokens
#pragma unroll
    for (int ob = 0; ob < TB; ++ob) t[ob] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < NC2; ++q) {
      const Op<kFull> s = st.template op<kFull>(q);
#pragma unroll
      for (int ob = 0; ob < TB; ++ob) mma<kFull>(t[ob], sh.k.rows(16 * ob, 32 * q), s);
    }
    Op<IN> vt[QB];  // v or do: free feature, contracted token
#pragma unroll
    for (int q = 0; q < QB; ++q) vt[q] = sh.v.template cols<>(32 * q, 16 * w);
    // r, or du
#pragma unroll
    for (int ob = 0; ob < TB; ++ob) {
      const int i = 16 * ob + 4 * g;
      if constexpr (BACK) {
        t[ob] *= tok.four(tok.wr, i);
#pragma unroll
        for (int q = 0; q < QB; ++q)
          if (meets(true, ob, 2 * q + 1)) mma<kFull>(t[ob], m_op(pair_at(true, Q, ob, q)), vt[q]);
      } else {
        t[ob] = join4(vt[ob / 2], ob & 1) - t[ob] * tok.four(tok.er, i);
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
        bad = first_not_finite(by);
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
    f4 u[TB];  // b x, or dv
#pragma unroll
    for (int ob = 0; ob < TB; ++ob) {
      f4 s = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < QB; ++q)
        if (BACK ? meets(true, ob, 2 * q + 1) : meets(false, ob, 2 * q)) mma<kFull>(s, z_op(pair_at(BACK, Q, ob, q)), br[q]);
      t[ob] -= s;
      u[ob] = t[ob] * tok.four(tok.beta, 16 * ob + 4 * g);
    }
    if constexpr (!BACK) {
      if (__ballot(bad < Q) != 0) {
#pragma unroll
        for (int ob = 0; ob < TB; ++ob)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool keep = 16 * ob + 4 * g + e < bad;
            u[ob][e] = keep ? u[ob][e] : 0.f;
            t[ob][e] = keep ? t[ob][e] : __builtin_nanf("");
          }
      }
    }
    if (OUT && p.rows != nullptr) {
      float* to = p.rows + ((chain * NC + c) * Q) * PB + f0 + 16 * w + r;
#pragma unroll
      for (int ob = 0; ob < TB; ++ob)
#pragma unroll
        for (int e = 0; e < 4; ++e) to[(16 * ob + 4 * g + e) * PB] = t[ob][e];
    }
    if constexpr (!OUT) {
    } else if constexpr (BACK) {
      T* to = O + row * ldo + 16 * w + r;
#pragma unroll
      for (int ob = 0; ob < TB; ++ob) {
        const auto d = to_frag<T>(u[ob]).v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 16 * ob + 4 * g + e;
          if (i < left) to[i * ldo] = d[e];
        }
      }
    } else {
      f4 y[TB];
#pragma unroll
      for (int ob = 0; ob < TB; ++ob) y[ob] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < NC2; ++q) {
        const Op<MID> s = st.template op<MID>(q);
#pragma unroll
        for (int ob = 0; ob < TB; ++ob) mma<MID>(y[ob], s, sh.q.rows(16 * ob, 32 * q));
      }
      Op<MID> uo[QB];
#pragma unroll
      for (int q = 0; q < QB; ++q) uo[q] = split8<MID>(u[2 * q], u[2 * q + 1]);
#pragma unroll
      for (int ob = 0; ob < TB; ++ob) {
        const int i = 16 * ob + r;
        y[ob] *= tok.eq[i];
#pragma unroll
        for (int q = 0; q < QB; ++q)
          if (meets(false, ob, 2 * q)) mma<MID>(y[ob], uo[q], m_op(pair_at(false, Q, ob, q)));
      }
      if (__ballot(bad < Q) != 0) {  // (a lane has the features 4g + e of a token here)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int first = __shfl(bad, 4 * g + e);
#pragma unroll
          for (int ob = 0; ob < TB; ++ob) y[ob][e] = 16 * ob + r < first ? y[ob][e] : __builtin_nanf("");
        }
      }
#pragma unroll
      for (int ob = 0; ob < TB; ++ob)
        if (16 * ob + r < left) store4(O + (row + 16 * ob + r) * ldo + 16 * w + 4 * g, y[ob]);
    }
    // the state behind the chunk, or the gradient of the one before it
    const float end = tok.end;
#pragma unroll
    for (int i = 0; i < NB; ++i) st.t[i] *= end;
#pragma unroll
    for (int q = 0; q < QB; ++q) {
      f4 a[2], d[2];
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        const int i = 32 * q + 16 * o + 4 * g;
        if constexpr (BACK) {
          a[o] = join4(vt[q], o) * tok.four(tok.eq, i);
          d[o] = u[2 * q + o] * tok.four(tok.er, i) * -1.f;
        } else {
          d[o] = u[2 * q + o] * tok.four(tok.wr, i);
        }
      }
      const Op<kFull> dk = split8<kFull>(d[0], d[1]);
#pragma unroll
      for (int i = 0; i < NB; ++i) mma<kFull>(st.t[i], sh.k.template cols<true>(32 * q, 32 * (i >> 1) + 4 * (i & 1)), dk);
      if constexpr (BACK) {
        const Op<kFull> dq = split8<kFull>(a[0], a[1]);
#pragma unroll
        for (int i = 0; i < NB; ++i) mma<kFull>(st.t[i], sh.q.template cols<true>(32 * q, 32 * (i >> 1) + 4 * (i & 1)), dq);
      }
    }
    if constexpr (!BACK) {
      if (__ballot(bad < Q) != 0) {
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) st.t[i][e] = bad < Q ? __builtin_nanf("") : st.t[i][e];
      }
    }
  }
  if (!OUT) {
    if (features)
      st.keep(p.seg + (chain * p.S + s) * (NP * PB) + f0, PB, w);
    else
      st.keep(p.trans + (head * p.S + s) * (NP * NP) + f0, NP, w);
  } else if (p.h_last != nullptr && s == (BACK ? 0 : p.S - 1)) {
    st.store(p.h_last + (chain * PB + f0) * p.N, p.N, p.N, w);
  }
}

// The segments' ends -> the states they start from, in place: a wave has 16 features of a part and
// goes over the segments, the next one's product on its way.
template <int NP, bool BACK> __global__ __launch_bounds__(64) void delta_join_kernel(DeltaParams p) {
  constexpr int NB = NP / 16, NC2 = NP / 32;
  const int l = lane_id(), g = l >> 4, r = l & 15;
  const int PB = delta_part(p.P), cols = PB / 16, parts = p.P / PB;
  const int w = (int)(blockIdx.x % cols);
  const long long chain = blockIdx.x / cols, head = chain / parts;
  StateTiles<NP> st, end;
  st.load(p.h0 != nullptr ? p.h0 + chain * PB * p.N : nullptr, p.N, p.N, w);
  const auto seg = [&](int k) { return BACK ? p.S - 1 - k : k; };
  const auto at = [&](int k) { return p.seg + (chain * p.S + seg(k)) * (NP * PB); };
  f4 a[NB][NC2][2];  // rows n as a state's tiles have them, columns 32q + 8g..
  const auto fetch = [&](int k) {
    const float* t = p.trans + (head * p.S + seg(k)) * (NP * NP);
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int q = 0; q < NC2; ++q)
#pragma unroll
        for (int o = 0; o < 2; ++o)
          a[i][q][o] = *reinterpret_cast<const f4*>(
              t + (32 * (i >> 1) + 8 * (r >> 2) + 4 * (i & 1) + (r & 3)) * NP + 32 * q + 8 * g + 4 * o);
    take_kept(end, at(k), PB, w);
  };
  fetch(0);
#pragma unroll 1
  for (int k = 0; k + 1 < p.S; ++k) {
    st.keep(at(k), PB, w);
    Op<kFull> s[NC2];
#pragma unroll
    for (int q = 0; q < NC2; ++q) s[q] = st.template op<kFull>(q);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      st.t[i] = end.t[i];
#pragma unroll
      for (int q = 0; q < NC2; ++q) mma<kFull>(st.t[i], split8<kFull>(a[i][q][0], a[i][q][1]), s[q]);
    }
    if (k + 2 < p.S) fetch(k + 1);
  }
  st.keep(at(p.S - 1), PB, w);
}

template <typename T, int W, int NP, bool BACK> hipError_t walk_t(const DeltaParams& p, hipStream_t stream) {
  constexpr size_t lds = sizeof(WalkShared<T, W, NP, BACK>);
  static_assert(lds <= 160 * 1024, "LDS of a compute unit");
  hipError_t e = allow_lds(delta_walk_kernel<T, W, NP, BACK, true>, lds);
  if (e != hipSuccess) return e;
  const long long heads = (long long)p.B * p.H;
  if (p.S > 1) {
    e = allow_lds(delta_walk_kernel<T, W, NP, BACK, false>, lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((delta_walk_kernel<T, W, NP, BACK, false>), dim3((unsigned)(heads * (p.S - 1) * (p.P + NP) / (16 * W))),
                       dim3(64 * W), lds, stream, p);
    hipLaunchKernelGGL((delta_join_kernel<NP, BACK>), dim3((unsigned)(heads * p.P / 16)), dim3(64), 0, stream, p);
  }
  hipLaunchKernelGGL((delta_walk_kernel<T, W, NP, BACK, true>), dim3((unsigned)(heads * p.S * p.P / (16 * W))), dim3(64 * W),
                     lds, stream, p);
  return hipGetLastError();
}
template <typename T, int W, bool BACK> hipError_t width_t(const DeltaParams& p, hipStream_t s) {
  return p.N <= 32 ? walk_t<T, W, 32, BACK>(p, s) : p.N <= 64 ? walk_t<T, W, 64, BACK>(p, s) : walk_t<T, W, 128, BACK>(p, s);
}
template <typename T, bool BACK> hipError_t part_t(const DeltaParams& p, hipStream_t s) {
  return delta_part(p.P) == 64 ? width_t<T, 4, BACK>(p, s) : width_t<T, 2, BACK>(p, s);
}
template <bool BACK> hipError_t launch(const DeltaParams& p, int dtype, hipStream_t s) {
  return dtype == TTT_DTYPE_BF16 ? part_t<__bf16, BACK>(p, s)
         : dtype == TTT_DTYPE_F16 ? part_t<_Float16, BACK>(p, s) : part_t<float, BACK>(p, s);
}

// One token of every sequence, the state in place: the state is read and written once, which
// bounds it.  LANES lanes have a feature's row of it, four values each.
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
