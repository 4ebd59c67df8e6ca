// The gated feed-forward projections on gfx950: y = act(x Wg^T + bg) * (x Wu^T + bu), forward
// and backward.
//
//   a = x Wg^T + bg,  b = x Wu^T + bu,  y = f(a) b
//   da = dy b f'(a),  db = dy f(a)                        (a and b formed again, not kept)
//   dx = da Wg + db Wu,   dWg = da^T x,   dWu = db^T x,   dbg = sum da,   dbu = sum db
//
// All four products are one kernel: tiles of 256 x 256 (eight waves) or 128 x 128 (four) from
// steps of 64 contracted values, which go from memory straight to LDS, two steps' places in
// turn.  An operand whose contracted values are neighbours in memory is read 16 bytes a lane;
// one whose free values are (the weights for dx, both operands of dW) by the transposing
// read, so that nothing is transposed in memory.  The 16-byte pieces of a row lie in LDS
// permuted by the row's number, so that reads meet in no bank, but for the first operand's transposing
// ones (dx's weights, dW's x), which take two turns; pieces outside a matrix read 0.
// The gate's and the other projection's columns of a tile meet in one wave, which forms y, or
// da and db, from its accumulators.
//
// fp32 operands are three bf16 planes, exact in each, and a product is the six of the planes
// a, b with a + b < 3, one after the other, smallest first: 2^-24 of the value, at a sixth of
// the rate of bf16 (the fp32 matrix instructions have a sixteenth).  da and db of 16-bit calls
// are rounded to the activations' type where dx and dW read them, as a layer that formed them
// one after the other would hand them on: their rounding adds to that at the store, each
// half a step (1.4 times the store's alone); two planes would double the two products.  In fp16 they
// may be past its largest number where dx and dW are not: such values go, 2^-30 times themselves, to
// a second plane, whose products are formed (first, and then brought to scale) only if there is one.
// Blocks with one are marked; one more launch puts zeros in the plane's other blocks, or finds no mark.
//
// 32,768 rows, 768 by 2,048, bf16: y 235 us (877 TFLOP/s), da and db 269, dx 262 in one round of large
// tiles and one of small, dW 241 and a join of 12 (294 and 257 before that and before the reads' order);
// in fp16 y 217, da and db 264, dx 254, dW 232 and 12.
// A step of a large tile is 64 KB to LDS by 1 KB loads, 192 KB of reads from it and 2,048 clocks of
// matrix instructions on each SIMD; it takes about 3,600.  Without the loads to LDS the products
// alone take 86% of the time, the loads alone 70%: they overlap in part, with a barrier a step.
// Steps of 32 with three on their way wait for less and meet twice as many barriers: 15 to 20% slower.
//
// Few rows (up to 64, a token of each sequence): a workgroup has 16 columns and up to 32 rows, the
// contraction shared out over eight waves; nothing goes through LDS but the waves' sums.  The weights
// are read once for 32 rows, twice for 33 to 64, the second time from a cache.  (768 by 2,048, 6.7 MB,
// in a graph: 4.4 us for 16 rows, 5.2 for 32, 5.3 for 64: a launch and its latency.)
#include <math.h>

#include <algorithm>

#include "ttt_ffn.h"
#include "ttt_scan.h"

namespace ttt {

namespace {

typedef __attribute__((address_space(3))) void lds_void;

template <typename T> struct Elem { typedef T type; };
template <> struct Elem<float> { typedef __bf16 type; };

template <typename E> __device__ __forceinline__ f4 product(bf8 p, bf8 q, f4 acc) {
  if constexpr (sizeof(E) == 2 && __is_same(E, _Float16))
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, p), __builtin_bit_cast(h8, q), acc, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(p, q, acc, 0, 0, 0);
}

// f(a) and f'(a)
template <bool GRAD> __device__ __forceinline__ float act_value(int act, float a, float& d) {
  if (act == TTT_ACT_SILU) {
    const float s = sigmoid_f(a);
    if (GRAD) d = s * __builtin_fmaf(a, 1.0f - s, 1.0f);
    return a * s;
  }
  const float c = 0.5f * erfcf(-0.7071067811865476f * a);  // the normal distribution's integral
  if (GRAD) d = __builtin_fmaf(a * 0.3989422804014327f, expf(-0.5f * a * a), c);
  return a * c;
}

// .. of N values, one branch for all of them: their exponentials and reciprocals overlap
template <bool GRAD, int N> __device__ __forceinline__ void act_values(int act, const float (&a)[N], float (&f)[N], float (&d)[N]) {
  if (act == TTT_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = act_value<GRAD>(TTT_ACT_SILU, a[e], d[e]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = act_value<GRAD>(TTT_ACT_GELU, a[e], d[e]);
  }
}

enum class Job { Fwd, Grad, Dx, Dw };
// how an operand lies: its contracted values side by side, or its free ones
enum class Lies { Contracted, Free };

// A step's part of an operand in LDS: FREE rows of 64 contracted values, or 64 rows of FREE
// (SIDE of an operand: the first's free values go to a lane's registers, eight neighbours of
// a pair of tiles, so that results are read and written 16 bytes a lane; the second's to lanes)
enum class Side { First, Second };
template <Lies L, Side S, int FREE> struct Panel {
  static constexpr int PIECES = (L == Lies::Contracted ? kFfnStep : FREE) / 8;  // of 16 bytes, to a row
  static constexpr int ROWS = L == Lies::Contracted ? FREE : kFfnStep;
  static constexpr int BYTES = FREE * kFfnStep * 2;
  // the rows that are read at once: 0..7 of eight, or of the first operand 0..3 and 8..11 of
  // sixteen; of free values rows 0..3 and 8..11 too, whose lanes have 32 bytes of each, or every other
  // 8 of 64: the first operand's take two turns in any order
  __device__ __forceinline__ static int place(int row, int piece) {
    if constexpr (L == Lies::Contracted)
      return piece ^ (S == Side::First ? (row & 3) | ((row >> 1) & 4) : row & 7);
    else
      return piece ^ (S == Side::First ? (row & 3) << 2 : ((row & 3) | ((row >> 1) & 4)) << 1);
  }
};

// Sends the step's rows of a matrix on their way to LDS.  `base`: the panel's first value;
// `rows` and `pieces` of it are in the matrix (whole rows `ld` bytes apart).
template <Lies L, Side S, int FREE, int NW>
__device__ __forceinline__ void send(const char* base, long long ld, int rows, int pieces, unsigned char* lds, int w) {
  using P = Panel<L, S, FREE>;
  constexpr int CNT = P::BYTES / 1024 / NW;
  static_assert(CNT * NW * 1024 == P::BYTES, "whole kilobytes to a wave");
  const int l = lane_id();
  rows = rows < P::ROWS ? rows : P::ROWS;
  const unsigned bytes = rows > 0 && pieces > 0 ? (unsigned)(rows - 1) * (unsigned)ld + (unsigned)min(pieces, P::PIECES) * 16u : 0u;
  const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), (short)0, (int)bytes, 0x00020000);
#pragma unroll
  for (int i = 0; i < CNT; ++i) {
    const int at = (i * NW + w) * 64 + l, row = at / P::PIECES, piece = P::place(row, at % P::PIECES);
    unsigned off = (unsigned)row * (unsigned)ld + (unsigned)piece * 16u;
    if (piece >= pieces) off = 0x80000000u;  // (past every panel: they stay below 2^31 bytes)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(lds + (i * NW + w) * 1024), 16, (int)off, 0, 0, 0);
  }
}
// A panel's operands of a tile's 16 free values and contracted values 32 k.. + 8g + (0..7).
// Tile t of the second operand has the free values 16 t + r; of the first, two tiles have 32, the
// even one 8 (r >> 2) + (r & 3) of them and the odd one those 4 behind.
template <Lies L, Side S, int FREE> __device__ __forceinline__ bf8 take(const unsigned char* lds, int t, int k) {
  using P = Panel<L, S, FREE>;
  const int l = lane_id(), g = l >> 4, r = l & 15;
  if constexpr (L == Lies::Contracted) {
    const int row = S == Side::First ? 32 * (t >> 1) + 8 * (r >> 2) + 4 * (t & 1) + (r & 3) : 16 * t + r;
    return *reinterpret_cast<const bf8*>(lds + row * kFfnStep * 2 + (P::place(row, 4 * k + g) << 4));
  } else {
    const int row = 32 * k + 8 * g + (r >> 2);
    const int piece = S == Side::First ? 4 * (t >> 1) + (l & 3) : 2 * t + ((l & 3) >> 1);
    const int half = S == Side::First ? t & 1 : l & 1;
    const auto at = [&](int rw) {
      return reinterpret_cast<const __bf16*>(lds + rw * FREE * 2 + (P::place(rw, piece) << 4) + half * 8);
    };
    return cat(read_tr(at(row)), read_tr(at(row + 4)));
  }
}

// The order of a step's reads of LDS and products: the first operands, then a read to every few
// products, two or more tiles ahead of them.  (By itself the compiler has each pair of reads right
// before its products, which wait for them.)
template <int N, int PER> __device__ __forceinline__ void interleave() {
  if constexpr (N > 0) {
    __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);  // matrix instructions
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);    // reads of LDS
    interleave<N - 1, PER>();
  }
}
template <int TN, int TM, Lies LN, Lies LM> __device__ __forceinline__ void reads_ahead() {
  constexpr int rn = LN == Lies::Free ? 2 : 1, rm = LM == Lies::Free ? 2 : 1, K = kFfnStep / 32;
  constexpr int head = TN * rn + 2 * rm, rest = K * (TN * rn + TM * rm) - head, products = K * TN * TM, per = (products - 2 * TN) / rest;
  static_assert(per > 0, "a product to a read at least");
  __builtin_amdgcn_sched_group_barrier(0x100, head, 0);
  interleave<rest, per>();
  __builtin_amdgcn_sched_group_barrier(0x008, products - rest * per, 0);
}

// 4 values of T behind each other from p, of n there are
template <typename T> __device__ __forceinline__ f4 load_up_to4(const T* p, int n) {
  Raw<T, 4> v;
  v.load(p, n);
  return f4{v.f(0), v.f(1), v.f(2), v.f(3)};
}
template <typename T> __device__ __forceinline__ void store_up_to4(T* p, int n, f4 v) {
  const float o[4] = {v[0], v[1], v[2], v[3]};
  store_row<T, 4>(p, n, o);
}
// eight values of da or db, in planes where T is fp32
template <typename T> __device__ __forceinline__ void store_grad(const FfnMatrix& m, long long row, int col, const float (&v)[8]) {
  char* to = static_cast<char*>(const_cast<void*>(m.p)) + row * m.ld + col * 2;
  if constexpr (sizeof(T) == 4) {
    const Op<3> o = split8<3>(f4{v[0], v[1], v[2], v[3]}, f4{v[4], v[5], v[6], v[7]});
#pragma unroll
    for (int a = 0; a < 3; ++a) *reinterpret_cast<bf8*>(to + a * m.plane) = o.v[a];
  } else {
    store_row<T, 8>(reinterpret_cast<T*>(to), 8, v);
  }
}
// fp16: where some are past its largest number, those that are finite go, scaled, to the second plane.
// (Beyond that one's range any product but with 0 is past the results' too.)
constexpr float kMostF16 = 65520.f;   // rounds to infinity
constexpr float kFar = 1073741824.f;  // 2^30: 2^16 is 2^-14 of it, a normal number, and 2^46 its largest
__device__ __forceinline__ void store_far(const FfnMatrix& m, long long row, int col, const float (&v)[8]) {
  float near[8], far[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool past = fabsf(v[e]) >= kMostF16 && fabsf(v[e]) < __builtin_inff();
    near[e] = past ? 0.f : v[e];
    far[e] = past ? fminf(fmaxf(v[e] * (1.f / kFar), -65504.f), 65504.f) : 0.f;
  }
  store_grad<_Float16>(m, row, col, near);
  store_grad<_Float16>({static_cast<const char*>(m.p) + m.plane, m.ld, 0}, row, col, far);
}

// Tiles of WN TN 16 columns (the first operand's free values, four to a lane's registers) by
// WM TM 16 rows (the second's, a lane each)
template <typename T, Job JOB, int WN, int WM, int TN, int TM>
__global__ __launch_bounds__(64 * WN * WM) void ffn_kernel(FfnParams p) {
  typedef typename Elem<T>::type E;
  constexpr bool UP = JOB == Job::Fwd || JOB == Job::Grad;  // both projections' columns in a tile
  constexpr Lies LN = UP ? Lies::Contracted : Lies::Free, LM = JOB == Job::Dw ? Lies::Free : Lies::Contracted;
  constexpr int BN = 16 * WN * TN, BM = 16 * WM * TM, NW = WN * WM, HALF = BN / 2;
  constexpr int STEP = Panel<LN, Side::First, BN>::BYTES + Panel<LM, Side::Second, BM>::BYTES;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int w = wave_id(), l = lane_id(), g = l >> 4, r = l & 15, wn = w % WN, wm = w / WN;
  // rows and columns of all tiles, and contracted values
  const int M = JOB == Job::Dw ? 2 * p.Fp : p.R, N = UP ? p.F : p.D, K = JOB == Job::Dw ? p.R : JOB == Job::Dx ? p.Fp : p.Dp;
  // (behind whole rounds of large tiles: those that are left, in four)
  constexpr bool SMALL = BM == 128;
  const int in_four = SMALL && p.whole > 0 ? 2 : 1, HM = in_four * BM, HN = in_four * (UP ? HALF : BN);
  const int tm = (M + HM - 1) / HM, tn = (N + HN - 1) / HN;
  // Neighbours on a die have eight rows of tiles by all columns, one column after the other
  unsigned id = on_xcd(blockIdx.x, gridDim.x);
  const unsigned quarter = in_four == 2 ? id & 3 : 0;
  if (in_four == 2) id = p.whole + id / 4;
  const int split = (int)(id / (unsigned)(tm * tn));
  id -= split * (tm * tn);
  const int band = (int)(id / (8u * tn)), high = min(8, tm - 8 * band);
  id -= band * 8 * tn;
  const int m0 = (8 * band + (int)(id % high)) * HM + (int)(quarter & 1) * BM;
  const int n0 = (int)(id / high) * HN + (int)(quarter >> 1) * (UP ? HALF : BN);
  if (m0 >= M || n0 >= N) return;

  const int ksteps = (K + kFfnStep - 1) / kFfnStep, pairs = p.planes == 3 ? 6 : 1, segs = JOB == Job::Dx ? 2 : 1;
  const int all = ksteps * pairs * segs, per = UP ? all : (all + p.splits - 1) / p.splits;
  const int first = split * per, own = min(all, first + per) - first;
  // (the second plane's steps are those of the first again, before them: a share has the same values)
  constexpr bool WIDE = __is_same(T, _Float16) && !UP;
  const bool far = WIDE && *p.far != 0;
  const int steps = far ? 2 * own : own;

  // the step that is sent next: its contracted values, of which weights, and the planes
  int sk = first % ksteps, ss = first / ksteps % segs, sp = first / (ksteps * segs), sent = 0;
  long long beside = far ? p.grad.plane : 0;  // to the plane of `grad`
  const auto next = [&](int buf) {
    // planes a of the first operand and b of the second: (2,0) (1,1) (0,2) (1,0) (0,1) (0,0)
    const int pa = pairs == 1 ? 0 : (0x001012 >> (4 * sp)) & 15;
    const int pb = pairs == 1 ? 0 : (0x010210 >> (4 * sp)) & 15;
    const int k = sk * kFfnStep, left = K - k;
    unsigned char* to = smem + buf * STEP;
    if constexpr (UP) {
      const int pieces = left / 8;
      const long long a = pa * p.wg.plane + (long long)n0 * p.wg.ld + k * 2;
      send<LN, Side::First, HALF, NW>(static_cast<const char*>(p.wg.p) + a, p.wg.ld, N - n0, pieces, to, w);
      send<LN, Side::First, HALF, NW>(static_cast<const char*>(p.wu.p) + a, p.wu.ld, N - n0, pieces, to + HALF * kFfnStep * 2, w);
      send<LM, Side::Second, BM, NW>(static_cast<const char*>(p.x.p) + pb * p.x.plane + (long long)m0 * p.x.ld + k * 2, p.x.ld, M - m0,
                       pieces, to + Panel<LN, Side::First, BN>::BYTES, w);
    } else if constexpr (JOB == Job::Dx) {
      const FfnMatrix& wt = ss == 0 ? p.wg : p.wu;
      send<LN, Side::First, BN, NW>(static_cast<const char*>(wt.p) + pa * wt.plane + (long long)k * wt.ld + n0 * 2, wt.ld, p.F - k,
                       (p.Dp - n0) / 8, to, w);
      send<LM, Side::Second, BM, NW>(static_cast<const char*>(p.grad.p) + (WIDE ? beside : pb * p.grad.plane) +
                           (long long)m0 * p.grad.ld + ((long long)ss * p.Fp + k) * 2,
                       p.grad.ld, M - m0, left / 8, to + Panel<LN, Side::First, BN>::BYTES, w);
    } else {
      send<LN, Side::First, BN, NW>(static_cast<const char*>(p.x.p) + pa * p.x.plane + (long long)k * p.x.ld + n0 * 2, p.x.ld, left,
                       (p.Dp - n0) / 8, to, w);
      send<LM, Side::Second, BM, NW>(static_cast<const char*>(p.grad.p) + (WIDE ? beside : pb * p.grad.plane) +
                           (long long)k * p.grad.ld + m0 * 2, p.grad.ld,
                       left, (M - m0) / 8, to + Panel<LN, Side::First, BN>::BYTES, w);
    }
    if (++sk == ksteps) {
      sk = 0;
      if (++ss == segs) {
        ss = 0;
        ++sp;
      }
    }
    if constexpr (WIDE) {  // (no branch: a step's reads and products stay in one block)
      const bool again = ++sent == own;
      sk = again ? first % ksteps : sk;
      ss = again ? first / ksteps : ss;
      beside = again ? 0 : beside;
    }
  };

  f4 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
  // a wave's tiles of columns: of both halves where a tile has both projections
  const auto tile_n = [&](int i) { return UP ? (i < TN / 2 ? wn * (TN / 2) + i : HALF / 16 + wn * (TN / 2) + i - TN / 2) : wn * TN + i; };
  if (steps > 0) next(0);
  const auto go = [&](int from, int to) {
#pragma unroll 1
    for (int s = from; s < to; ++s) {
      // the step is here, in all waves, and the one before it has been read
      __builtin_amdgcn_s_waitcnt(0x0F70);  // (vmcnt(0))
      __syncthreads();
      if (s + 1 < steps) next((s + 1) & 1);
      const unsigned char* at = smem + (s & 1) * STEP;
#pragma unroll
      for (int k = 0; k < kFfnStep / 32; ++k) {
        bf8 pn[TN], pm[TM];
#pragma unroll
        for (int i = 0; i < TN; ++i) pn[i] = take<LN, Side::First, BN>(at, tile_n(i), k);
#pragma unroll
        for (int j = 0; j < TM; ++j) pm[j] = take<LM, Side::Second, BM>(at + Panel<LN, Side::First, BN>::BYTES, wm * TM + j, k);
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
          for (int i = 0; i < TN; ++i) acc[i][j] = product<E>(pn[i], pm[j], acc[i][j]);
      }
      reads_ahead<TN, TM, LN, LM>();
    }
  };
  if constexpr (WIDE) {
    if (far) {
      go(0, own);
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] *= kFar;
    }
    go(steps - own, steps);
  } else {
    go(0, steps);
  }

  // A pair of tiles' columns are eight neighbours in a lane: 8g + 4i + e of 32
  if constexpr (UP) {
#pragma unroll
    for (int i = 0; i < TN / 2; i += 2) {
      const int f = n0 + 16 * (wn * (TN / 2) + i) + 8 * g, left = N - f;
      Raw<T, 8> bg, bu;
      bg.zero();
      bu.zero();
      if (p.bg != nullptr && left > 0) bg.load(static_cast<const T*>(p.bg) + f, left);
      if (p.bu != nullptr && left > 0) bu.load(static_cast<const T*>(p.bu) + f, left);
      float sg[8], su[8];
      Raw<T, 8> dy[JOB == Job::Grad ? TM : 1];
      if constexpr (JOB == Job::Grad) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sg[e] = su[e] = 0.f;
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          const int m = m0 + 16 * (wm * TM + j) + r;
          dy[j].zero();
          if (m < M && left > 0) dy[j].load(static_cast<const T*>(p.dy) + (long long)m * p.lddy + f, left);
        }
      }
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const int m = m0 + 16 * (wm * TM + j) + r;
        float u[8], v[8];  // y; or da and db
        float a[8], fa[8], d[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = acc[i + e / 4][j][e & 3] + bg.f(e);
        act_values<JOB == Job::Grad>(p.act, a, fa, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float b = acc[TN / 2 + i + e / 4][j][e & 3] + bu.f(e);
          if constexpr (JOB == Job::Fwd) {
            u[e] = fa[e] * b;
          } else {
            // (0 past the last row and column: nothing from there reaches the sums)
            const float y = dy[j].f(e);
            const bool in = m < M && e < left;
            v[e] = in ? y * fa[e] : 0.f;
            u[e] = in ? y * b * d[e] : 0.f;
            sg[e] += u[e];
            su[e] += v[e];
          }
        }
        if constexpr (JOB == Job::Fwd) {
          if (m < M && left > 0) store_row<T, 8>(static_cast<T*>(p.y) + (long long)m * p.F + f, left, u);
        } else {
          bool any = false;
          if constexpr (__is_same(T, _Float16)) {
            float most = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fmaxf(fabsf(u[e]), fabsf(v[e])));
            any = __ballot(most >= kMostF16) != 0;
          }
          if (m < M && f < p.Fp) {
            if (any) {
              store_far(p.grad, m, f, u);
              store_far(p.grad, m, p.Fp + f, v);
            } else {
              store_grad<T>(p.grad, m, f, u);
              store_grad<T>(p.grad, m, p.Fp + f, v);
            }
          }
          if constexpr (__is_same(T, _Float16)) {
            const int rows = m0 + 16 * (wm * TM + j), cols = n0 + 16 * (wn * (TN / 2) + i);  // the block's first
            if (l == 0 && rows < M && cols < N) p.over[(long long)(rows / kFfnFarRows) * ffn_far_cols(p.F) + cols / kFfnFarCols] = any;
          }
        }
      }
      if (JOB == Job::Grad && p.bias_part != nullptr) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sg[e] = sum_row16(sg[e]);
          su[e] = sum_row16(su[e]);
        }
        if (r == 0 && f < p.Fp) {
          float* to = p.bias_part + (long long)(m0 / BM * WM + wm) * 2 * p.Fp + f;
          store_row<float, 8>(to, 8, sg);
          store_row<float, 8>(to + p.Fp, 8, su);
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < TN; i += 2) {
      const int n = n0 + 16 * (wn * TN + i) + 8 * g, left = N - n;
      if (left <= 0) continue;
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const int m = m0 + 16 * (wm * TM + j) + r;
        if (m >= M) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = acc[i + e / 4][j][e & 3];
        if (p.splits > 1) {
          store_row<float, 8>(p.part + ((long long)split * M + m) * p.Dp + n, 8, v);
        } else if constexpr (JOB == Job::Dx) {
          store_row<T, 8>(static_cast<T*>(p.dx) + (long long)m * p.D + n, left, v);
        } else {
          const int f = m < p.Fp ? m : m - p.Fp;
          if (f < p.F) store_row<T, 8>(static_cast<T*>(m < p.Fp ? p.dwg : p.dwu) + (long long)f * p.D + n, left, v);
        }
      }
    }
  }
}

// dx, or dWg and dWu, from the sums of the shares
template <typename T, Job JOB> __global__ __launch_bounds__(256) void ffn_join_kernel(FfnParams p, long long quads) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= quads) return;
  const int per = p.Dp / 4, m = (int)(id / per), n = 4 * (int)(id - (long long)m * per);
  const int f = JOB == Job::Dx ? m : m < p.Fp ? m : m - p.Fp;
  if (JOB == Job::Dw && f >= p.F) return;
  const float* s = p.part + 4 * id;
  f4 v = *reinterpret_cast<const f4*>(s);
  for (int k = 1; k < p.splits; ++k) v += *reinterpret_cast<const f4*>(s + 4 * k * quads);
  T* to = static_cast<T*>(JOB == Job::Dx ? p.dx : m < p.Fp ? p.dwg : p.dwu);
  store_up_to4(to + (long long)f * p.D + n, p.D - n, v);
}
// fp16: whether any block has a mark, and if so zeros to the second plane's blocks without one.  (32,768
// rows by 2,048: 5 us without a mark.)
__global__ __launch_bounds__(256) void ffn_far_kernel(FfnParams p, long long blocks) {
  unsigned any = 0;
  const long long whole = blocks / 16;
#pragma unroll 8
  for (long long i = threadIdx.x; i < whole; i += 256) {
    const u4v v = reinterpret_cast<const u4v*>(p.over)[i];
    any |= v[0] | v[1] | v[2] | v[3];
  }
  if (16 * whole + threadIdx.x < blocks) any |= p.over[16 * whole + threadIdx.x];
  const bool far = __syncthreads_or(any != 0) != 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.far = far;
  if (!far) return;
  const int cols = ffn_far_cols(p.F);
  constexpr int PIECES = kFfnFarCols / 8, EACH = kFfnFarRows * PIECES;  // of 16 bytes, to a row and block
  for (long long k = (long long)blockIdx.x * (256 / EACH) + threadIdx.x / EACH; k < blocks; k += (long long)gridDim.x * (256 / EACH)) {
    if (p.over[k] != 0) continue;
    const int at = threadIdx.x % EACH;
    const long long rb = k / cols, row = kFfnFarRows * rb + at / PIECES;
    const int c = kFfnFarCols * (int)(k - rb * cols) + 8 * (at % PIECES);
    if (row >= p.R || c >= p.Fp) continue;
    char* to = static_cast<char*>(const_cast<void*>(p.grad.p)) + p.grad.plane + row * p.grad.ld;
    *reinterpret_cast<u4v*>(to + c * 2) = u4v{0, 0, 0, 0};
    *reinterpret_cast<u4v*>(to + (p.Fp + c) * 2) = u4v{0, 0, 0, 0};
  }
}
template <typename T> __global__ __launch_bounds__(256) void ffn_bias_kernel(FfnParams p) {
  const int n = 2 * p.Fp, c = blockIdx.x * 16 + (threadIdx.x & 15);
  const float s = sum_parts(p.bias_part, n, c, p.bias_parts);
  if (threadIdx.x >= 16 || c >= n) return;
  const int f = c < p.Fp ? c : c - p.Fp;
  T* to = static_cast<T*>(c < p.Fp ? p.dbg : p.dbu);
  if (f < p.F && to != nullptr) to[f] = (T)s;
}

// 8 values to a thread
template <typename T> __global__ __launch_bounds__(256) void ffn_planes_kernel(const T* from, long long ld, int width, int pieces,
                                                                              long long all, char* to, long long plane) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= all) return;
  const long long row = id / pieces;
  const int c = 8 * (int)(id - row * pieces);
  Raw<T, 8> v;
  v.load(from + row * ld + c, width - c);
  if constexpr (sizeof(T) == 4) {
    const Op<3> o = split8<3>(f4{v.f(0), v.f(1), v.f(2), v.f(3)}, f4{v.f(4), v.f(5), v.f(6), v.f(7)});
#pragma unroll
    for (int a = 0; a < 3; ++a) *reinterpret_cast<bf8*>(to + a * plane + id * 16) = o.v[a];
  } else {
    Raw<T, 8> o = v;
    *reinterpret_cast<u4v*>(to + id * 16) = __builtin_bit_cast(u4v, o.v);
  }
}

// Few rows: a workgroup has 16 columns of both projections and 16 or 32 rows, a wave every
// eighth 32 contracted values
constexpr int kFewWaves = 8;
template <typename T> struct FewOp { typedef Op<3> type; };
template <> struct FewOp<__bf16> { typedef bf8 type; };
template <> struct FewOp<_Float16> { typedef bf8 type; };
template <typename T> __device__ __forceinline__ typename FewOp<T>::type few_op(const T* p, int n) {
  Raw<T, 8> v;
  v.load(p, n);
  if constexpr (sizeof(T) == 4)
    return split8<3>(f4{v.f(0), v.f(1), v.f(2), v.f(3)}, f4{v.f(4), v.f(5), v.f(6), v.f(7)});
  else
    return __builtin_bit_cast(bf8, v.v);
}
__device__ __forceinline__ void few_mma(f4& acc, const Op<3>& a, const Op<3>& b, float) { mma<3>(acc, a, b); }
__device__ __forceinline__ void few_mma(f4& acc, bf8 a, bf8 b, __bf16) { acc = product<__bf16>(a, b, acc); }
__device__ __forceinline__ void few_mma(f4& acc, bf8 a, bf8 b, _Float16) { acc = product<_Float16>(a, b, acc); }

template <typename T, int TM> __global__ __launch_bounds__(64 * kFewWaves) void ffn_few_kernel(FfnParams p) {
  const int w = wave_id(), l = lane_id(), g = l >> 4, r = l & 15;
  const int f0 = 16 * blockIdx.x, m0 = 16 * TM * blockIdx.y, fr = min(f0 + r, p.F - 1);
  const long long ldw = p.wg.ld / (long long)sizeof(T), ldx = p.x.ld / (long long)sizeof(T);
  const T *wg = static_cast<const T*>(p.wg.p) + fr * ldw, *wu = static_cast<const T*>(p.wu.p) + fr * ldw;
  const T* x = static_cast<const T*>(p.x.p);
  f4 acc[2][TM];
#pragma unroll
  for (int j = 0; j < TM; ++j) acc[0][j] = acc[1][j] = f4{0.f, 0.f, 0.f, 0.f};
  for (int k = 32 * w; k < p.D; k += 32 * kFewWaves) {
    const int c = k + 8 * g, n = p.D - c, cc = n > 0 ? c : 0;
    // (a lane without values reads none: Raw's loads take n <= 0 as zeros)
    const auto a = few_op<T>(wg + cc, n), b = few_op<T>(wu + cc, n);
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int m = min(m0 + 16 * j + r, p.R - 1);
      const auto q = few_op<T>(x + m * ldx + cc, n);
      few_mma(acc[0][j], a, q, T());
      few_mma(acc[1][j], b, q, T());
    }
  }
  __shared__ f4 red[kFewWaves][2][TM][64];
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    red[w][0][j][l] = acc[0][j];
    red[w][1][j][l] = acc[1][j];
  }
  __syncthreads();
  if (w >= TM) return;
  f4 a = red[0][0][w][l], b = red[0][1][w][l];
#pragma unroll
  for (int k = 1; k < kFewWaves; ++k) {
    a += red[k][0][w][l];
    b += red[k][1][w][l];
  }
  const int f = f0 + 4 * g, left = p.F - f, m = m0 + 16 * w + r;
  if (left <= 0 || m >= p.R) return;
  if (p.bg != nullptr) a += load_up_to4(static_cast<const T*>(p.bg) + f, left);
  if (p.bu != nullptr) b += load_up_to4(static_cast<const T*>(p.bu) + f, left);
  f4 y;
  float d;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = act_value<false>(p.act, a[e], d) * b[e];
  store_up_to4(static_cast<T*>(p.y) + (long long)m * p.F + f, left, y);
}

template <typename K> hipError_t allow_lds(K k, size_t bytes) {
  return bytes <= 65536 ? hipSuccess
                        : hipFuncSetAttribute(reinterpret_cast<const void*>(k),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}
template <typename T, Job JOB, int WN, int WM, int TN, int TM> hipError_t tile_t(const FfnParams& p, hipStream_t s) {
  constexpr int BN = 16 * WN * TN, BM = 16 * WM * TM, lds = 2 * (BN + BM) * kFfnStep * 2;
  const auto kernel = ffn_kernel<T, JOB, WN, WM, TN, TM>;
  const hipError_t e = allow_lds(kernel, lds);
  if (e != hipSuccess) return e;
  constexpr bool up = JOB == Job::Fwd || JOB == Job::Grad;
  const long long M = JOB == Job::Dw ? 2LL * p.Fp : p.R, N = up ? 2LL * p.F : p.D;
  const long long large = ((M + 255) / 256) * ((N + 255) / 256);
  const long long blocks = p.whole == 0 ? ((M + BM - 1) / BM) * ((N + BN - 1) / BN) * p.splits
                           : BM == 256  ? p.whole
                                        : 4 * (large - p.whole);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * WN * WM), lds, s, p);
  if (p.splits > 1) {
    const long long quads = M * p.Dp / 4;
    hipLaunchKernelGGL((ffn_join_kernel<T, JOB>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s, p, quads);
  }
  return hipGetLastError();
}
template <typename T, Job JOB> hipError_t job_t(const FfnParams& p, bool large, hipStream_t s) {
  if (p.whole > 0) {
    const hipError_t e = tile_t<T, JOB, 4, 2, 4, 8>(p, s);
    if (e != hipSuccess) return e;
  }
  return large ? tile_t<T, JOB, 4, 2, 4, 8>(p, s) : tile_t<T, JOB, 2, 2, 4, 4>(p, s);
}
template <Job JOB> hipError_t type_t(FfnParams p, FfnCut cut, int dtype, hipStream_t s) {
  p.splits = cut.splits;
  p.whole = cut.whole;
  return dtype == TTT_DTYPE_BF16 ? job_t<__bf16, JOB>(p, cut.large, s)
         : dtype == TTT_DTYPE_F16 ? job_t<_Float16, JOB>(p, cut.large, s) : job_t<float, JOB>(p, cut.large, s);
}

template <typename T> hipError_t few_t(const FfnParams& p, hipStream_t s) {
  const unsigned cols = (unsigned)((p.F + 15) / 16);
  if (p.R <= 16)
    hipLaunchKernelGGL((ffn_few_kernel<T, 1>), dim3(cols), dim3(64 * kFewWaves), 0, s, p);
  else
    hipLaunchKernelGGL((ffn_few_kernel<T, 2>), dim3(cols, (unsigned)((p.R + 31) / 32)), dim3(64 * kFewWaves), 0, s, p);
  return hipGetLastError();
}
template <typename T> hipError_t bias_t(const FfnParams& p, hipStream_t s) {
  hipLaunchKernelGGL(ffn_bias_kernel<T>, dim3((unsigned)((2 * p.Fp + 15) / 16)), dim3(256), 0, s, p);
  return hipGetLastError();
}
template <typename T>
hipError_t planes_t(const void* from, long long ld, int rows, int width, void* to, hipStream_t s) {
  const int pieces = ffn_pad(width) / 8;
  const long long all = (long long)rows * pieces;
  hipLaunchKernelGGL(ffn_planes_kernel<T>, dim3((unsigned)((all + 255) / 256)), dim3(256), 0, s, static_cast<const T*>(from), ld,
                     width, pieces, all, static_cast<char*>(to), all * 16);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_ffn_few(const FfnParams& p, int dtype, hipStream_t s) {
  return dtype == TTT_DTYPE_BF16 ? few_t<__bf16>(p, s) : dtype == TTT_DTYPE_F16 ? few_t<_Float16>(p, s) : few_t<float>(p, s);
}
hipError_t launch_ffn_fwd(const FfnParams& p, int dtype, hipStream_t s) { return type_t<Job::Fwd>(p, ffn_cut_up(p.R, p.D, p.F, dtype, false), dtype, s); }
hipError_t launch_ffn_grad(const FfnParams& p, int dtype, hipStream_t s) {
  hipError_t e = type_t<Job::Grad>(p, ffn_cut_up(p.R, p.D, p.F, dtype, p.bias_part != nullptr), dtype, s);
  if (e == hipSuccess && dtype == TTT_DTYPE_F16) {
    const long long blocks = ffn_far_blocks(p.R, p.F);
    hipLaunchKernelGGL(ffn_far_kernel, dim3((unsigned)std::min(blocks, 256LL)), dim3(256), 0, s, p, blocks);
    e = hipGetLastError();
  }
  if (e != hipSuccess || p.bias_part == nullptr) return e;
  return dtype == TTT_DTYPE_BF16 ? bias_t<__bf16>(p, s) : dtype == TTT_DTYPE_F16 ? bias_t<_Float16>(p, s) : bias_t<float>(p, s);
}
hipError_t launch_ffn_dx(const FfnParams& p, int dtype, hipStream_t s) {
  return type_t<Job::Dx>(p, ffn_cut_dx(p.R, p.D, p.F, dtype), dtype, s);
}
hipError_t launch_ffn_dw(const FfnParams& p, int dtype, hipStream_t s) {
  return type_t<Job::Dw>(p, ffn_cut_dw(p.R, p.D, p.F, dtype), dtype, s);
}
hipError_t launch_ffn_planes(const void* from, long long ld, int rows, int width, void* to, int dtype, hipStream_t s) {
  return dtype == TTT_DTYPE_BF16 ? planes_t<__bf16>(from, ld, rows, width, to, s)
         : dtype == TTT_DTYPE_F16 ? planes_t<_Float16>(from, ld, rows, width, to, s)
                                  : planes_t<float>(from, ld, rows, width, to, s);
}

}  // namespace ttt
