// Shared device code of the selective scan's kernels (ttt_scan_walk.hip,
// ttt_scan_bwd.hip): the mathematics of a chunk, operands in planes, LDS layouts.
//
// Per sequence and head, with decay a_t = d_t A (A < 0) and state h [P][N]:
//   h_t = e^{a_t} h_{t-1} + d_t x_t (x) B_t,      y_t = h_t C_t + D x_t
// Over a chunk of Q tokens, with the decays' running sum c_t = a_1 + .. + a_t and
// the state H entering it, this is three matrix products:
//   y_i  = sum_{j<=i} e^{c_i - c_j} d_j (C_i . B_j) x_j + e^{c_i} H C_i + D x_i
//   H'   = e^{c_Q} H + sum_j e^{c_Q - c_j} d_j x_j (x) B_j
// Every exponent is <= 0.  c is summed in 64 bits and kept as two floats: tokens
// that follow a strong decay have differences c_i - c_j far smaller than the sums,
// and the factors they give would otherwise lose what the sums have rounded away.
//
// Matrix operands are bf16 planes whose sum is the value: an input is one plane in
// bf16, two in fp16 and three in fp32, exact in each (8 bits a plane), so a single
// matrix instruction (v_mfma_f32_16x16x32_bf16) and one range serve all types.
// Values formed on the way are fp32 and split into planes where they are
// multiplied: three planes and all products p q with p + q < 3, 2^-24 of the value.
// Fp32 results (states, the gradients of states and parameters) of 16-bit calls are
// as exact as those of fp32 ones.  Where a value leads to bf16 results alone (the masked
// products, the state as the outputs read it, the weights W of the backward) it has
// two, 2^-17 of it: over 1,000 tokens that moves a result by 1.2e-5 of their root mean square
// at most, 1/300 of the largest rounding at the store, and 1 value in 1,000 to its other
// neighbour.  Three there would cost 281 and 295 us, forward and backward of 32,768 tokens of 12
// heads of 64 x 64, and 78 and 96, a prompt of 16,384 of 12 of 64 x 128.  In fp16, whose store
// rounds 8 times finer, two were 1.3e-4 off, a quarter of the store's rounding, and one value in
// 100 went to its other neighbour: it has three (12 heads of 64 x 64: 395 and 415 us).
#pragma once

#include "ttt_ssm.h"

namespace ttt {

struct ScanParams {
  const void *x, *dt, *Bm, *Cm;      // [B*L][ldx], [B*L][lddt], [B*L][ldb], [B*L][ldc]
  const float *A, *D, *dt_bias;      // [H] (D, dt_bias may be null)
  const float* h0;                   // [B][H][P][N] (may be null: zeros)
  void* y;                           // [B][L][H][P]
  float* h_last;                     // [B][H][P][N] (may be null)
  float* states;                     // [B*H][NC][NP][P]: the states entering the chunks, or walking back the
                                     // gradients of those leaving them (may be null)
  float *seg, *seg_decay;            // [B*H][S][P][NP] and [B*H][S]: per segment of the sequence
  long long ldx, lddt, ldb, ldc;
  int B, L, H, G, N;
  int S, per;                        // segments, and chunks in one
  bool joined;                       // the states in `seg` are those entering the segments
  bool softplus, dt_f32;
  // backward
  const void* dy;                    // [B*L][ldy]
  long long ldy;
  const float* gstates;              // the gradients of the states leaving the chunks
  void *dx, *ddt, *dB, *dC;          // [B][L][H][P], [B][L][H], [B][L][G][N]
  float *dBp, *dCp;                  // [splits][B*L][G][N] where a group's heads are split, else null
  float* partial;                    // [3][H][B*NC]: dA, dD, ddt_bias of each chunk
  float *dA, *dD, *ddt_bias;         // [H]
  int splits;
};

hipError_t launch_scan_fwd(const ScanParams& p, int P, int dtype, hipStream_t stream);
// walks back from the last state's gradient (p.h0): the gradients of x (into p.dx), of the states leaving the
// chunks (p.states) and of the initial one (p.h_last)
hipError_t launch_scan_walk_back(const ScanParams& p, int P, int dtype, hipStream_t stream);
hipError_t launch_scan_bwd(const ScanParams& p, int P, int dtype, hipStream_t stream);
struct ScanStepParams {
  const void *x, *dt, *Bm, *Cm;   // [B][ldx], [B][lddt], [B][ldb], [B][ldc]
  const float *A, *D, *dt_bias;   // [H]
  float* h;                       // [B][H][P][N], read and written
  void* y;                        // [B][H][P]
  long long ldx, lddt, ldb, ldc;
  int B, H, P, G, N;
  bool softplus, dt_f32;
};
hipError_t launch_scan_step(const ScanStepParams& p, int dtype, hipStream_t stream);
constexpr int scan_padded(int N) { return N <= 32 ? 32 : N <= 64 ? 64 : 128; }

template <typename T> struct ScanType;
// planes of an input, and of a formed value that leads to results of this type alone
template <> struct ScanType<__bf16> { static constexpr int IN = 1, MID = 2; };
template <> struct ScanType<_Float16> { static constexpr int IN = 2, MID = 3; };
template <> struct ScanType<float> { static constexpr int IN = 3, MID = 3; };
constexpr int kFull = 3;  // planes of a formed value that leads to fp32 results
// tokens of a chunk: 64, or 32 where the backward's planes would not fit in LDS
constexpr int scan_chunk(int dtype, int NP) {
  return dtype == TTT_DTYPE_F32 || (dtype == TTT_DTYPE_F16 && NP == 128) ? 32 : 64;
}
template <typename T, int NP> constexpr int chunk_of() {
  return scan_chunk(ScanType<T>::IN == 3 ? TTT_DTYPE_F32 : ScanType<T>::IN == 2 ? TTT_DTYPE_F16 : TTT_DTYPE_BF16, NP);
}

// The wave's number as a scalar: matrix instructions take no notice of the lanes'
// execution mask, so what decides whether one runs has to be a scalar branch.
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// Workgroups go to the 8 dies in turn, and each die has an L2 of its own: the place of
// workgroup `id` of n such that each die has a run of neighbours, which share rows.
__device__ __forceinline__ unsigned on_xcd(unsigned id, unsigned n) {
  const unsigned die = id & 7, per = n >> 3, rest = n & 7;
  return die * per + min(die, rest) + (id >> 3);
}

// ---------------------------------------------------------------- planes
template <int PL> struct Op {  // one operand of a 32-deep product
  bf8 v[PL];
};
// two values at a time: one conversion instruction a plane, and what it leaves
template <int PL> __device__ __forceinline__ void split2(f2 x, bf2 (&o)[PL]) {
#pragma unroll
  for (int q = 0; q < PL; ++q) {
    o[q] = __builtin_convertvector(x, bf2);
    if (q + 1 < PL) {
      const unsigned u = __builtin_bit_cast(unsigned, o[q]);
      x[0] -= __builtin_bit_cast(float, u << 16);
      x[1] -= __builtin_bit_cast(float, u & 0xffff0000u);
    }
  }
}
template <int PL> __device__ __forceinline__ void split4(f4 x, bf4 (&o)[PL]) {
  bf2 a[PL], b[PL];
  split2<PL>(f2{x[0], x[1]}, a);
  split2<PL>(f2{x[2], x[3]}, b);
#pragma unroll
  for (int q = 0; q < PL; ++q) o[q] = __builtin_shufflevector(a[q], b[q], 0, 1, 2, 3);
}
template <int PL> __device__ __forceinline__ Op<PL> split8(f4 x, f4 y) {
  bf4 a[PL], b[PL];
  split4<PL>(x, a);
  split4<PL>(y, b);
  Op<PL> r;
#pragma unroll
  for (int q = 0; q < PL; ++q) r.v[q] = __builtin_shufflevector(a[q], b[q], 0, 1, 2, 3, 4, 5, 6, 7);
  return r;
}
// 0 where `keep` is false, without a branch around what x comes from
__device__ __forceinline__ float only_if(bool keep, float x) {
  asm("" : "+v"(x));
  return keep ? x : 0.f;
}
// values 4o..4o+3 of an operand
template <int PL> __device__ __forceinline__ f4 join4(const Op<PL>& a, int o) {
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  f4 s = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int q = PL - 1; q >= 0; --q) {
    const bf8 v = a.v[q];
    const bf4 h = o == 0 ? __builtin_shufflevector(v, v, 0, 1, 2, 3) : __builtin_shufflevector(v, v, 4, 5, 6, 7);
    const u2 u = __builtin_bit_cast(u2, h);
    const f4 x = f4{__builtin_bit_cast(float, u[0] << 16), __builtin_bit_cast(float, u[0] & 0xffff0000u),
                    __builtin_bit_cast(float, u[1] << 16), __builtin_bit_cast(float, u[1] & 0xffff0000u)};
    s = q == PL - 1 ? x : s + x;
  }
  return s;
}
// acc[m][n] += sum_k p[m][k] q[n][k], products of planes a and b with a + b < ORDER
template <int ORDER, int PA, int PB> __device__ __forceinline__ void mma(f4& acc, const Op<PA>& p, const Op<PB>& q) {
#pragma unroll
  for (int a = PA - 1; a >= 0; --a)
#pragma unroll
    for (int b = PB - 1; b >= 0; --b)
      if (a + b < ORDER) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p.v[a], q.v[b], acc, 0, 0, 0);
}

// ---------------------------------------------------------------- planes in LDS
// ROWS x COLS values as PL planes of rows, 16 bytes of padding to a row: the 16
// rows of a 16-byte read fall into different banks for COLS = 32, 64 and 128.
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4v lds_s4v;
__device__ __forceinline__ bf4 read_tr(const __bf16* p) {
  return __builtin_bit_cast(bf4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v*)(const_cast<__bf16*>(p))));
}
__device__ __forceinline__ bf8 cat(bf4 a, bf4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

template <int PL, int ROWS, int COLS> struct Planes {
  static constexpr int LD = COLS + 8;
  __bf16 d[PL][ROWS][LD];
  // free index: row; contraction: columns k0 + 8g + e
  __device__ __forceinline__ Op<PL> rows(int r0, int k0) const {
    const int l = lane_id(), g = l >> 4, r = l & 15;
    Op<PL> o;
#pragma unroll
    for (int q = 0; q < PL; ++q) o.v[q] = *reinterpret_cast<const bf8*>(&d[q][r0 + r][k0 + 8 * g]);
    return o;
  }
  // free index r: column c0 + r, or with NAT8 c0 + 8 (r >> 2) + (r & 3);
  // contraction: rows k0 + 4g + e and k0 + 16 + 4g + e (e < 4).
  // (the transposing read: lane 4k + q of a group names row k's columns 4q..4q+3
  // and lane i receives column i of the group's 16 for its four rows)
  template <bool NAT8 = false> __device__ __forceinline__ Op<PL> cols(int k0, int c0) const {
    const int l = lane_id(), g = l >> 4, k = (l & 15) >> 2, c = (l & 3) * (NAT8 ? 8 : 4);
    const int ra = k0 + 4 * g + k, rb = ra + 16;
    Op<PL> o;
#pragma unroll
    for (int q = 0; q < PL; ++q) o.v[q] = cat(read_tr(&d[q][ra][c0 + c]), read_tr(&d[q][rb][c0 + c]));
    return o;
  }
  // four values of row r from column c on
  __device__ __forceinline__ f4 quad(int r, int c) const {
    Op<PL> o;
#pragma unroll
    for (int q = 0; q < PL; ++q) {
      const bf4 v = *reinterpret_cast<const bf4*>(&d[q][r][c]);
      o.v[q] = cat(v, v);
    }
    return join4(o, 0);
  }
};

typedef unsigned u4v __attribute__((ext_vector_type(4)));
// ROWS x COLS values of T on their way from a matrix of rows to planes.  A thread's
// places are the same in every chunk: their offsets are formed once.
template <typename T, int ROWS, int COLS, int NT> struct Stage {
  static constexpr int VE = 16 / (int)sizeof(T), PER = COLS / VE, ALL = ROWS * PER, CNT = (ALL + NT - 1) / NT;
  static_assert(ALL % NT == 0 || CNT == 1, "whole rounds, or some threads without a place");
  u4v v[CNT];
  unsigned off[CNT];  // bytes
  int cols;
  __device__ __forceinline__ static int row(int i) { return (i * NT + (int)threadIdx.x) / PER; }
  __device__ __forceinline__ static int col(int i) { return (i * NT + (int)threadIdx.x) % PER * VE; }
  // rows `ld` apart (ROWS of them within 4 GiB), `cols` columns
  __device__ __forceinline__ void place(long long ld, int n) {
    cols = n;
#pragma unroll
    for (int i = 0; i < CNT; ++i) off[i] = ((unsigned)row(i) * (unsigned)ld + (unsigned)col(i)) * (unsigned)sizeof(T);
  }
  __device__ __forceinline__ static bool has() { return ALL % NT == 0 || (int)threadIdx.x < ALL; }
  __device__ __forceinline__ static u4v get(const char* q, unsigned o) {
    asm volatile("" : "+v"(o));  // 32 bits beside a scalar base: not widened ahead of the loop
    return *reinterpret_cast<const u4v*>(q + o);
  }
  // rows from `p` on, `rows` of them; zeros elsewhere
  __device__ __forceinline__ void load(const T* __restrict__ p, int rows) {
    const char* q = reinterpret_cast<const char*>(p);
    if (rows == ROWS && cols == COLS && ALL % NT == 0) {
#pragma unroll
      for (int i = 0; i < CNT; ++i) v[i] = get(q, off[i]);
    } else {
#pragma unroll
      for (int i = 0; i < CNT; ++i) {
        v[i] = u4v{0, 0, 0, 0};
        if (has() && col(i) < cols && row(i) < rows) v[i] = get(q, off[i]);
      }
    }
  }
  // the loads are done
  __device__ __forceinline__ void settle() {
#pragma unroll
    for (int i = 0; i < CNT; ++i) asm volatile("" : "+v"(v[i]));
  }
  // the sum of a thread's values times those of another
  __device__ __forceinline__ float dot(const Stage& o) const {
    float s = 0.f;
    if (!has()) return s;
    typedef T tv __attribute__((ext_vector_type(VE)));
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const tv a = __builtin_bit_cast(tv, v[i]), b = __builtin_bit_cast(tv, o.v[i]);
#pragma unroll
      for (int e = 0; e < VE; ++e) s = __builtin_fmaf((float)a[e], (float)b[e], s);
    }
    return s;
  }
  template <int PL> __device__ __forceinline__ void store(Planes<PL, ROWS, COLS>& m) const {
    if (!has()) return;
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int r = row(i), c = col(i);
      if constexpr (sizeof(T) == 4) {
        bf4 o[PL];
        split4<PL>(__builtin_bit_cast(f4, v[i]), o);
#pragma unroll
        for (int q = 0; q < PL; ++q) *reinterpret_cast<bf4*>(&m.d[q][r][c]) = o[q];
      } else if constexpr (PL == 1) {
        *reinterpret_cast<u4v*>(&m.d[0][r][c]) = v[i];
      } else {
        const h8 x = __builtin_bit_cast(h8, v[i]);
        const Op<PL> o = split8<PL>(f4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]},
                                    f4{(float)x[4], (float)x[5], (float)x[6], (float)x[7]});
#pragma unroll
        for (int q = 0; q < PL; ++q) *reinterpret_cast<bf8*>(&m.d[q][r][c]) = o.v[q];
      }
    }
  }
};

// ---------------------------------------------------------------- a chunk's decays
// The sum of v over lanes 0..l, by DPP moves: within rows of 16 lanes, then each
// row's total into the rows behind it.
template <int CTRL, int ROWS> __device__ __forceinline__ double dpp_add(double v) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (unsigned)u, CTRL, ROWS, 0xF, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (unsigned)(u >> 32), CTRL, ROWS, 0xF, false);
  return v + __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double lane_sums(double v) {
  v = dpp_add<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
  v = dpp_add<0x112, 0xF>(v);
  v = dpp_add<0x114, 0xF>(v);
  v = dpp_add<0x118, 0xF>(v);
  v = dpp_add<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  return dpp_add<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
}
__device__ __forceinline__ double lane_value(double v, int l) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __builtin_amdgcn_readlane((unsigned)u, l), hi = __builtin_amdgcn_readlane((unsigned)(u >> 32), l);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}

// d_t, the running sum c_t of log2(e) d_t A over the chunk in two floats, and its
// factors from the chunk's start, 2^c_t, and to its end, 2^(c_Q - c_t)
template <int Q, bool WALK = false> struct alignas(16) Decays {  // (read four values at a time)
  float hi[Q], lo[Q], d[Q];
  float head[Q], tail[Q];
  float in[WALK ? Q : 4];  // d_t 2^(c_Q - c_t): what token t adds to the state
  float end;  // 2^c_Q
  float total;  // c_Q
  // one wave, lane t (< Q) with token t's d
  __device__ __forceinline__ void fill(float dt, float A) {
    const int l = lane_id();
    const double c = lane_sums(l < Q ? (double)dt * ((double)A * 1.4426950408889634074) : 0.0);
    const double last = lane_value(c, 63);
    if (l < Q) {
      const float h = (float)c;
      hi[l] = h;
      lo[l] = (float)(c - (double)h);
      d[l] = dt;
      head[l] = __builtin_amdgcn_exp2f(h);
      const float t = __builtin_amdgcn_exp2f((float)(last - c));
      tail[l] = t;
      if (WALK) in[l] = t * dt;
    }
    if (l == 0) {
      total = (float)last;
      end = __builtin_amdgcn_exp2f((float)last);
    }
  }
  __device__ __forceinline__ static f4 four(const float* a, int t) { return *reinterpret_cast<const f4*>(a + t); }
};
// log(1 + e^v), v itself from 20 on (within 2e-9 of it)
__device__ __forceinline__ float softplus_f(float v) { return v > 20.f ? v : log1pf(expf(v)); }
// a step's bits as they are in memory: nothing waits for them until they are decoded
template <typename T> __device__ __forceinline__ unsigned dt_bits(const ScanParams& p, long long row, int h) {
  const long long o = row * p.lddt + h;
  return sizeof(T) == 4 || p.dt_f32 ? static_cast<const unsigned*>(p.dt)[o] : static_cast<const unsigned short*>(p.dt)[o];
}
template <typename T> __device__ __forceinline__ float dt_value(const ScanParams& p, unsigned u, float bias) {
  if constexpr (sizeof(T) == 4)
    return __builtin_bit_cast(float, u) + bias;
  else
    return (p.dt_f32 ? __builtin_bit_cast(float, u) : (float)__builtin_bit_cast(T, (unsigned short)u)) + bias;
}

// ---------------------------------------------------------------- the state in registers
// Wave w holds h[n][p] of its 16 features p = 16w + r as tiles of 16 x 16 (rows n):
// tile 2c + o, row 4g + e is n = 32c + 8g + 4o + e, so that two tiles are an operand
// whose contraction runs over n = 32c + 8g + (0..7), as rows of B and C are read.
template <int NP> struct StateTiles {
  static constexpr int NB = NP / 16, NC2 = NP / 32;
  f4 t[NB];
  __device__ __forceinline__ static int col(int c) { return 32 * c + 8 * (lane_id() >> 4); }
  __device__ __forceinline__ void load(const float* __restrict__ s, int ld, int N, int w) {
    const int r = 16 * w + (lane_id() & 15);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int n = col(i >> 1) + 4 * (i & 1);
      t[i] = f4{0.f, 0.f, 0.f, 0.f};
      if (s != nullptr && n < N) t[i] = *reinterpret_cast<const f4*>(s + (long long)r * ld + n);
    }
  }
  __device__ __forceinline__ void store(float* __restrict__ s, int ld, int N, int w) const {
    const int r = 16 * w + (lane_id() & 15);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int n = col(i >> 1) + 4 * (i & 1);
      if (n < N) *reinterpret_cast<f4*>(s + (long long)r * ld + n) = t[i];
    }
  }
  // as [NP][P]: what the backward reads as operands with contraction over p
  __device__ __forceinline__ void keep(float* __restrict__ s, int P, int w) const {
    const int l = lane_id();
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[(col(i >> 1) + 4 * (i & 1) + e) * P + 16 * w + (l & 15)] = t[i][e];
  }
  template <int PL> __device__ __forceinline__ Op<PL> op(int c) const {
    return split8<PL>(t[2 * c], t[2 * c + 1]);
  }
};
// the tiles (ib, jb), jb <= ib, of a lower triangle of blocks, row by row
__device__ __forceinline__ int tri(int ib, int jb) { return ib * (ib + 1) / 2 + jb; }
__device__ __forceinline__ int tri_row(int t) { return t >= 6 ? 3 : t >= 3 ? 2 : t >= 1 ? 1 : 0; }

}  // namespace ttt
