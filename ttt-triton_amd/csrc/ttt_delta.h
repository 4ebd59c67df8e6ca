// Shared code of the gated delta rule's kernels (ttt_delta_prep.hip, ttt_delta_walk.hip,
// ttt_delta_bwd.hip): the mathematics of a chunk, parameters, layouts.
//
// Per sequence and head, with a state S [P][N], decays a_t = e^{g_t}, and q and k as they
// are or at unit length:
//   S_t = a_t S_{t-1} + u_t (x) k_t,   u_t = b_t (v_t - a_t S_{t-1} k_t),   o_t = s S_t q_t
// Over a chunk of Q tokens, with c_t = g_1 + .. + g_t, F_ij = e^{c_i - c_j} and the state S
// entering it, the values x_t = v_t - a_t S_{t-1} k_t that the state misses solve a
// triangular system:
//   x + A b x = r,   r_i = v_i - e^{c_i} S k_i,   A_ij = F_ij (k_i . k_j) for j < i
// so x = r - Z b r with Z = A - A b Z, which depends on the keys alone.  The rest is products:
//   o_i = s (e^{c_i} S q_i + sum_{j<=i} F_ij (q_i . k_j) b_j x_j)
//   S'  = e^{c_Q} S + sum_j e^{c_Q - c_j} b_j x_j (x) k_j
// and backwards, with M_ij = s F_ij (q_i . k_j) for j <= i and the gradients do, dS':
//   du_j = sum_i M_ij do_i + e^{c_Q - c_j} dS' k_j,   y = du - Z^T b du,   dv = b y
//   dS   = e^{c_Q} dS' + sum_i s e^{c_i} do_i (x) q_i - sum_i e^{c_i} dv_i (x) k_i
// (y is the gradient of r before b: dbeta_i = y_i . x_i, with no division by b.)  Every
// exponent is <= 0; c is summed in 64 bits and kept as two floats, as the scan's.
//
// M and Z take no state: a first launch forms them for all chunks at once
// (ttt_delta_prep.hip) and the walks along the sequences read them (ttt_delta_walk.hip).
// The features of a head do not meet in S: heads of more than 64 features are walked as
// several heads of 64 or 32 that share q, k, g and b ("parts" below).
//
// Operands are bf16 planes and the products of planes those of the scan (ttt_scan.h): three
// planes, 2^-24 of the value, where an fp32 result comes of it (states, the gradients of
// steps, decays, initial states); two where bf16 results alone do (M, the state and u as the outputs
// read them, the masked products of dq and dk), 2^-17.  Three there bring a bf16 call's results from
// 1.3e-4 to 3.2e-5 (of their norm) of those of fp32 arithmetic rounded once, one value in 1,000 to its
// other neighbour, at 613 us for 600 (32,768 tokens of 12 heads of 64 x 64, forward and backward) and 162
// for 154 (a prompt of 16,384); the store's rounding, 1.7e-3, is what either is off by.
#pragma once

#include "ttt_scan.h"

namespace ttt {

struct DeltaParams {
  const void *q, *k, *v;  // [B*L][ldq], [B*L][ldk], [B*L][ldv]
  const void *g, *beta;   // [B*L][ldg], [B*L][ldbeta]
  const float* h0;        // [B][H][P][N] (may be null: zeros); backwards the gradient of the last state
  void* o;                // [B][L][H][P]; backwards dv
  float* h_last;          // [B][H][P][N] (may be null); backwards the gradient of the initial state
  float* tok;             // [B*H][NC] DeltaTok
  float *z, *m;           // [B*H][NC][tiles][64][4]: Z and M by blocks, as tile_at has them
  float* states;          // [B*H*parts][NC][NP][PB]: the states entering the chunks, or walking back the
                          // gradients of those leaving them (may be null)
  float* rows;            // [B*H*parts][NC*Q][PB]: x, or walking back y (may be null)
  float *seg, *trans;     // [B*H*parts][S][NP][PB] and [B*H][S][NP][NP]: per segment of the sequence
  long long ldq, ldk, ldv, ldg, ldbeta;
  int B, L, H, G, N, P;
  int S, per;             // segments, and chunks in one
  float scale;
  bool l2, g_f32, beta_f32;
  // backward
  const void* dO;              // [B*L][lddo]
  long long lddo;
  const float *gstates, *x;    // what the walk back and the forward's walk kept
  void *dq, *dk, *dg, *dbeta;  // [B][L][G][N] and [B][L][H]
  float *dqp, *dkp;            // [H/G][B*L][G][N] where heads share q and k, else null
};
hipError_t launch_delta_fwd(const DeltaParams& p, int dtype, hipStream_t stream);
hipError_t launch_delta_walk_back(const DeltaParams& p, int dtype, hipStream_t stream);
hipError_t launch_delta_prep(const DeltaParams& p, int dtype, hipStream_t stream);
hipError_t launch_delta_bwd(const DeltaParams& p, int dtype, hipStream_t stream);
struct DeltaStepParams {
  const void *q, *k, *v, *g, *beta;  // [B][ldq], ..
  float* h;                          // [B][H][P][N], read and written
  void* o;                           // [B][H][P]
  long long ldq, ldk, ldv, ldg, ldbeta;
  int B, H, P, G, N;
  float scale;
  bool l2, g_f32, beta_f32;
};
hipError_t launch_delta_step(const DeltaStepParams& p, int dtype, hipStream_t stream);

constexpr float kUnitEps = 1e-6f;  // x / sqrt(|x|^2 + eps)
constexpr int kDeltaMaxP = 256;
// features of a part
constexpr int delta_part(int P) { return P % 64 == 0 ? 64 : 32; }
// tokens of a chunk: 64, or 32 where the backward's planes would not fit in LDS
constexpr int delta_chunk(int dtype) { return dtype == TTT_DTYPE_BF16 ? 64 : 32; }
// blocks of 16 x 16 in a chunk's triangle, and operands of 32 contracted tokens
constexpr int delta_tiles(int Q) { return Q == 64 ? 10 : 3; }
constexpr int delta_pairs(int Q) { return Q == 64 ? 6 : 2; }
constexpr int delta_tok_floats(int Q) { return 8 * Q + 4; }

template <typename T> constexpr int kDeltaQ = sizeof(T) == 2 && ScanType<T>::IN == 1 ? 64 : 32;

// A chunk's numbers by token: c as two floats, b, the factors that bring q and k to unit
// length, and what the products with raw rows of q and k take:
//   er = e^c rk,   wr = e^{c_Q - c} rk,   eq = s e^c rq
template <int Q> struct alignas(16) DeltaTok {
  float hi[Q], lo[Q], beta[Q], rk[Q], rq[Q], er[Q], wr[Q], eq[Q];
  float end;  // e^{c_Q}
  float pad[3];
  __device__ __forceinline__ static f4 four(const float* a, int t) { return *reinterpret_cast<const f4*>(a + t); }
};

// Z and M are kept by blocks of 16 x 16 as the forward's operands take them: a row to a lane, four
// columns to its registers.  Walking back the column is a lane's and the rows are contracted: four
// reads of 4 bytes each, 16 bytes apart between the lanes.
template <bool BACK> __device__ __forceinline__ f4 tile_at(const float* p, int t) {
  const int l = lane_id(), g = l >> 4, r = l & 15;
  p += t * 256;
  if constexpr (!BACK) return *reinterpret_cast<const f4*>(p + 4 * l);
  p += (r >> 2) * 64 + 16 * g + (r & 3);
  return f4{p[0], p[4], p[8], p[12]};
}
// A block has its free token to a lane and four contracted ones to a lane's registers.  Two of them are an operand of 32 contracted tokens:
// forwards of row block b, columns 32q.. (q <= b / 2), backwards of column block b, rows 32q..
// (q >= b / 2); the place of an operand among the triangle's:
__device__ __forceinline__ constexpr int pair_at(bool back, int Q, int b, int q) {
  if (Q == 32) return b;
  if (!back) return b < 2 ? b : 2 * b - 2 + q;
  return b < 2 ? 2 * b + q : b + 2;
}
// Whether the block of contracted tokens `in` meets the free block `b`
__device__ __forceinline__ constexpr bool meets(bool back, int b, int in) { return back ? in >= b : in <= b; }

// One of a token's numbers, of H to a row
template <typename T> __device__ __forceinline__ float token_value(const void* p, bool f32, long long o) {
  if constexpr (sizeof(T) == 4)
    return static_cast<const float*>(p)[o];
  else
    return f32 ? static_cast<const float*>(p)[o] : (float)static_cast<const T*>(p)[o];
}
// A decay below e^-1000 is 0 in fp32 either way; bounded, the sums of the tokens behind it
// keep their last bits
__device__ __forceinline__ float bounded_decay(float g) { return g < -1000.f ? -1000.f : g; }

// Whether any value of a wave's tiles is not finite, or so large that their sum is not: no value
// that first_not_finite finds is missed (|.|, so that none takes another's place)
template <int TB> __device__ __forceinline__ bool any_not_finite(const f4 (&t)[TB]) {
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int b = 0; b < TB; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += fabsf(t[b][e]);
  return __ballot(!((s[0] + s[1]) + (s[2] + s[3]) < 3.3895e38f)) != 0;
}
// The first of a column's 16 blocks' rows (tile rows 4g + e of TB tiles, a lane group each)
// whose value is not finite, 16 TB where there is none; the same in the column's four lanes
template <int TB> __device__ __forceinline__ int first_not_finite(const f4 (&t)[TB]) {
  const int g = lane_id() >> 4;
  int first = 16 * TB;
#pragma unroll
  for (int b = TB - 1; b >= 0; --b)
#pragma unroll
    for (int e = 3; e >= 0; --e)
      if (!(fabsf(t[b][e]) < 3.3895e38f)) first = 16 * b + 4 * g + e;
  first = min(first, __shfl_xor(first, 16));
  return min(first, __shfl_xor(first, 32));
}

template <typename K> hipError_t allow_lds(K k, size_t bytes) {
  return bytes <= 65536 ? hipSuccess
                        : hipFuncSetAttribute(reinterpret_cast<const void*>(k),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

}  // namespace ttt
