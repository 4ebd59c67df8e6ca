// extern "C" entry points of the selective state-space operators: host-side
// validation and workspace layout, then launches on the caller's stream.
// Declarations and argument contracts are in include/ttt_amd.h.
#include <stdint.h>

#include <algorithm>

#include "ttt_abi_check.h"
#include "ttt_scan.h"

namespace {

// ---- convolution
int check_conv(int B, int L, int C, int W, int act, int dtype) {
  if (!dtype_ok(dtype)) return TTT_ERR_DTYPE;
  if (B <= 0 || L <= 0 || C <= 0 || W < 2 || W > 4) return TTT_ERR_SHAPE;
  // (the kernels' threads have four channels each and 16 tokens or, where that makes fewer
  // threads than this by far, 8)
  if (L > 0x7fffff00 || C > 1 << 22 || (long long)((L + 18) / 16) * ((C + 3) / 4) > kMaxThreads / B) return TTT_ERR_SHAPE;
  if (act != TTT_ACT_NONE && act != TTT_ACT_SILU) return TTT_ERR_ARG;
  return TTT_OK;
}

// ---- scan
int check_scan(int B, int L, int H, int P, int G, int N, int dtype, int dt_dtype) {
  if (!dtype_ok(dtype) || (dt_dtype != dtype && dt_dtype != TTT_DTYPE_F32)) return TTT_ERR_DTYPE;
  if (B <= 0 || L <= 0 || H <= 0 || G <= 0 || H % G != 0) return TTT_ERR_SHAPE;
  if ((P != 32 && P != 64) || N < 16 || N > 128 || N % 16 != 0) return TTT_ERR_SHAPE;
  if (L > 0x7fffff00 || (long long)B * H > kMaxGrid || H > (1 << 23) / P || G > (1 << 23) / N) return TTT_ERR_SHAPE;
  return TTT_OK;
}
constexpr int kSelfJoined = 8;  // segments whose states the walk's workgroups join themselves
struct ScanPlan {
  int Q, NC, NP, S, per, splits;
  size_t states, seg, decay, partial, split;
};
// Workgroups of the walk that a compute unit holds, by its registers and LDS.  Heads of 64
// with states up to 32 in fp32 need fewer registers walking back: 132 forwards and 116 back.
// (With one workgroup more than is held, and with those that are, us forwards of 32 x 1,024
// tokens of 8 heads of 64 x 32: fp16 69 and 64, fp32 75 and 72; of 16 x 2,048 of 12: 100 and 96, 108
// and 102; of 4 x 4,096 of 12: 61 and 68, 72 and 64.)
int walk_resident(int P, int NP, int dtype, bool back) {
  constexpr signed char t[2][3][3] = {{{5, 3, 5}, {4, 2, 3}, {2, 3, 2}}, {{3, 2, 3}, {3, 2, 3}, {2, 2, 2}}};
  if (back && P == 64 && NP == 32 && dtype == TTT_DTYPE_F32) return 4;
  return t[P == 64][NP == 32 ? 0 : NP == 64 ? 1 : 2][dtype == TTT_DTYPE_BF16 ? 0 : dtype == TTT_DTYPE_F16 ? 1 : 2];
}
// How a scan is cut up.  Segments: a workgroup walks a sequence and head; where that
// makes too few of them, the tokens are shared out as well, whole chunks each, to at
// most the full rounds of the card nearest above three workgroups of 64 features or
// five of 32 a compute unit, 8 segments though, which a workgroup joins by itself.  (Forward
// and backward of 32,768 tokens: 768 at once, 12 heads of 64 x 64 in bf16: 306, 279 and 299 us
// with 3, 4 and 6 segments; 512 at once, in fp16: 469, 439, 413, 423 with 3, 4, 5, 6; 1,024 at
// once, 24 heads of 32 x 64: 406, 383, 362, 383 with 3, 4, 5, 8.)  More segments cost two launches
// and a pass over them all: one round of the card, where 8 do not fill three quarters of it.
// (128 chains of 32 x 64: 139 us with 8, 159 with 11.  Forward of 40,000 tokens of 5 heads of
// 64 x 128 in fp16, 512 at once: 141, 122, 134 and 164 us with 128, 102, 86 and 52 segments; 2 x
// 5,000 of 9 in bf16: 53, 47 and 52 with 40, 27 and 20.)
// Splits: the backward's workgroups have a chunk and go over a group's heads; below
// 512 of them, two a compute unit, the heads are shared out.  (16,384 tokens of 12 heads of
// 64 x 64 in bf16: 157 us forward and backward, 174 with half and 168 with twice as many.)
ScanPlan plan(int B, int L, int H, int P, int G, int N, int dtype, bool back) {
  ScanPlan s;
  s.NP = ttt::scan_padded(N);
  s.Q = ttt::scan_chunk(dtype, s.NP);
  s.NC = (L + s.Q - 1) / s.Q;
  const long long chains = (long long)B * H;
  const int at_once = 256 * walk_resident(P, s.NP, dtype, back), least = P == 64 ? 768 : 1280;
  const int most = (least + at_once - 1) / at_once * at_once;
  long long want = at_once / chains;
  if (want <= kSelfJoined)
    want = std::min<long long>(kSelfJoined, most / chains);
  else if (4 * kSelfJoined * chains >= 3 * at_once)
    want = kSelfJoined;
  want = std::max(1LL, std::min<long long>(s.NC, want));
  s.per = (int)((s.NC + want - 1) / want);
  s.S = (s.NC + s.per - 1) / s.per;
  const long long groups = (long long)B * s.NC * G;
  s.splits = (int)std::min<long long>(H / G, (512 + groups - 1) / groups);
  s.states = (size_t)chains * s.NC * P * s.NP * 4;
  s.seg = s.S > 1 ? (size_t)chains * s.S * P * s.NP * 4 : 0;
  s.decay = s.S > 1 ? up256((size_t)chains * s.S * 4) : 0;
  s.partial = up256((size_t)3 * H * B * s.NC * 4);
  s.split = s.splits > 1 ? (size_t)s.splits * B * L * G * N * 4 : 0;
  return s;
}
// (the backward's workgroups have up to 8 P threads)
bool grid_ok(const ScanPlan& s, int B, int H, int P, int G) {
  return (long long)B * H * s.S <= kMaxThreads / (4 * P) && (long long)B * s.NC <= kMaxGrid &&
         (long long)B * s.NC * G <= kMaxThreads / (8 * P) / s.splits;
}
bool plan_ok(int B, int L, int H, int P, int G, int N, int dtype, bool back, ScanPlan& s) {
  if (check_scan(B, L, H, P, G, N, dtype, dtype) != TTT_OK) return false;
  s = plan(B, L, H, P, G, N, dtype, back);
  return grid_ok(s, B, H, P, G);
}

// ---- layer norm
int check_norm(long long R, int D, float eps, int dtype) {
  if (!dtype_ok(dtype)) return TTT_ERR_DTYPE;
  if (R <= 0 || R > kMaxGrid || D <= 0 || D > ttt::kNormMaxD) return TTT_ERR_SHAPE;
  if (!(eps > 0.0f) || eps > 1.0f) return TTT_ERR_ARG;
  return TTT_OK;
}

}  // namespace

extern "C" {

int ttt_causal_conv_fwd(const void* x, long long ldx, const void* state, const float* weight, const float* bias, int B,
                        int L, int C, int W, int activation, int dtype, void* y, void* state_out, void* stream) {
  const int st = check_conv(B, L, C, W, activation, dtype);
  if (st != TTT_OK) return st;
  if (ldx < C) return TTT_ERR_SHAPE;
  const size_t n = size_of(dtype);
  REQUIRE(x, n);
  REQUIRE(weight, 4);
  REQUIRE(y, n);
  OPTIONAL(state, n);
  OPTIONAL(bias, 4);
  OPTIONAL(state_out, n);
  ttt::ConvParams p{};
  p.x = x;
  p.ldx = ldx;
  p.state = state;
  p.w = weight;
  p.bias = bias;
  p.B = B;
  p.L = L;
  p.C = C;
  p.W = W;
  p.silu = activation == TTT_ACT_SILU;
  p.y = y;
  p.last = state_out;
  return hip_status(ttt::launch_conv_fwd(p, dtype, static_cast<hipStream_t>(stream)));
}

size_t ttt_causal_conv_partial_bytes(int B, int L, int C, int W) {
  if (check_conv(B, L, C, W, TTT_ACT_NONE, TTT_DTYPE_F32) != TTT_OK) return 0;
  return (size_t)ttt::conv_bwd_parts(B, L, C) * (W + 1) * C * sizeof(float);
}

int ttt_causal_conv_bwd(const void* x, long long ldx, const void* state, const float* weight, const float* bias,
                        const void* dy, const void* dstate_out, int B, int L, int C, int W, int activation, int dtype,
                        void* dx, void* dstate, float* dweight, float* dbias, float* partial, size_t partial_bytes,
                        void* stream) {
  const int st = check_conv(B, L, C, W, activation, dtype);
  if (st != TTT_OK) return st;
  if (ldx < C) return TTT_ERR_SHAPE;
  const size_t n = size_of(dtype);
  REQUIRE(x, n);
  REQUIRE(weight, 4);
  REQUIRE(dx, n);
  REQUIRE(dweight, 4);
  OPTIONAL(state, n);
  OPTIONAL(bias, 4);
  OPTIONAL(dy, n);
  OPTIONAL(dstate_out, n);
  OPTIONAL(dstate, n);
  OPTIONAL(dbias, 4);
  if (partial == nullptr || partial_bytes < ttt_causal_conv_partial_bytes(B, L, C, W)) return TTT_ERR_WORKSPACE;
  if (!aligned(partial, 16)) return TTT_ERR_ALIGN;
  ttt::ConvParams p{};
  p.x = x;
  p.ldx = ldx;
  p.state = state;
  p.w = weight;
  p.bias = bias;
  p.dy = dy;
  p.ldy = C;
  p.dlast = dstate_out;
  p.B = B;
  p.L = L;
  p.C = C;
  p.W = W;
  p.silu = activation == TTT_ACT_SILU;
  p.dx = dx;
  p.dstate = dstate;
  p.dw = dweight;
  p.dbias = dbias;
  p.partial = partial;
  return hip_status(ttt::launch_conv_bwd(p, dtype, static_cast<hipStream_t>(stream)));
}

int ttt_causal_conv_step(const void* x, long long ldx, void* state, const float* weight, const float* bias, int B, int C,
                         int W, int activation, int dtype, void* y, void* stream) {
  const int st = check_conv(B, 1, C, W, activation, dtype);
  if (st != TTT_OK) return st;
  if (ldx < C) return TTT_ERR_SHAPE;
  const size_t n = size_of(dtype);
  REQUIRE(x, n);
  REQUIRE(state, n);
  REQUIRE(weight, 4);
  REQUIRE(y, n);
  OPTIONAL(bias, 4);
  ttt::ConvParams p{};
  p.x = x;
  p.ldx = ldx;
  p.last = state;
  p.w = weight;
  p.bias = bias;
  p.B = B;
  p.L = 1;
  p.C = C;
  p.W = W;
  p.silu = activation == TTT_ACT_SILU;
  p.y = y;
  return hip_status(ttt::launch_conv_step(p, dtype, static_cast<hipStream_t>(stream)));
}

size_t ttt_scan_states_bytes(int B, int L, int H, int P, int N, int dtype) {
  ScanPlan s;
  return plan_ok(B, L, H, P, 1, N, dtype, false, s) ? s.states : 0;
}
size_t ttt_scan_workspace_bytes(int B, int L, int H, int P, int N, int dtype) {
  ScanPlan s;
  return plan_ok(B, L, H, P, 1, N, dtype, false, s) ? s.seg + s.decay : 0;
}
size_t ttt_scan_bwd_workspace_bytes(int B, int L, int H, int P, int G, int N, int dtype) {
  ScanPlan s;
  return plan_ok(B, L, H, P, G, N, dtype, true, s) ? up256(s.states) + s.seg + s.decay + s.partial + 2 * s.split : 0;
}

int ttt_scan_fwd(const void* x, long long ldx, const void* dt, long long lddt, const float* A, const void* Bm,
                 long long ldb, const void* Cm, long long ldc, const float* D, const float* dt_bias, const float* h0,
                 int B, int L, int H, int P, int G, int N, int dtype, int dt_dtype, int softplus, void* y,
                 float* h_last, void* states, size_t states_bytes, void* workspace, size_t workspace_bytes,
                 void* stream) {
  int st = check_scan(B, L, H, P, G, N, dtype, dt_dtype);
  if (st != TTT_OK) return st;
  const ScanPlan s = plan(B, L, H, P, G, N, dtype, false);
  if (!grid_ok(s, B, H, P, G)) return TTT_ERR_SHAPE;
  if (lddt < H) return TTT_ERR_SHAPE;
  if ((st = check_row(ldx, (long long)H * P, L, dtype)) != TTT_OK) return st;
  if ((st = check_row(ldb, (long long)G * N, L, dtype)) != TTT_OK) return st;
  if ((st = check_row(ldc, (long long)G * N, L, dtype)) != TTT_OK) return st;
  REQUIRE(x, 16);
  REQUIRE(dt, size_of(dt_dtype));
  REQUIRE(A, 4);
  REQUIRE(Bm, 16);
  REQUIRE(Cm, 16);
  REQUIRE(y, 16);
  OPTIONAL(D, 4);
  OPTIONAL(dt_bias, 4);
  OPTIONAL(h0, 16);
  OPTIONAL(h_last, 16);
  OPTIONAL(states, 16);
  OPTIONAL(workspace, 16);
  if (states != nullptr && states_bytes < s.states) return TTT_ERR_WORKSPACE;
  if (s.S > 1 && (workspace == nullptr || workspace_bytes < s.seg + s.decay)) return TTT_ERR_WORKSPACE;
  ttt::ScanParams p{};
  p.x = x;
  p.ldx = ldx;
  p.dt = dt;
  p.lddt = lddt;
  p.A = A;
  p.Bm = Bm;
  p.ldb = ldb;
  p.Cm = Cm;
  p.ldc = ldc;
  p.D = D;
  p.dt_bias = dt_bias;
  p.h0 = h0;
  p.B = B;
  p.L = L;
  p.H = H;
  p.G = G;
  p.N = N;
  p.softplus = softplus != 0;
  p.dt_f32 = dt_dtype == TTT_DTYPE_F32;
  p.y = y;
  p.h_last = h_last;
  p.states = static_cast<float*>(states);
  p.S = s.S;
  p.per = s.per;
  p.joined = s.S > kSelfJoined;
  if (s.S > 1) {
    p.seg = static_cast<float*>(workspace);
    p.seg_decay = reinterpret_cast<float*>(static_cast<char*>(workspace) + s.seg);
  }
  return hip_status(ttt::launch_scan_fwd(p, P, dtype, static_cast<hipStream_t>(stream)));
}

int ttt_scan_bwd(const void* x, long long ldx, const void* dt, long long lddt, const float* A, const void* Bm,
                 long long ldb, const void* Cm, long long ldc, const float* D, const float* dt_bias, const void* dy,
                 long long ldy, const float* dh_last, const void* states, size_t states_bytes, int B, int L, int H,
                 int P, int G, int N, int dtype, int dt_dtype, int softplus, void* dx, void* ddt, float* dA, void* dB,
                 void* dC, float* dD, float* ddt_bias, float* dh0, void* workspace, size_t workspace_bytes,
                 void* stream) {
  int st = check_scan(B, L, H, P, G, N, dtype, dt_dtype);
  if (st != TTT_OK) return st;
  const ScanPlan s = plan(B, L, H, P, G, N, dtype, true);
  if (!grid_ok(s, B, H, P, G)) return TTT_ERR_SHAPE;
  if (lddt < H) return TTT_ERR_SHAPE;
  if ((st = check_row(ldx, (long long)H * P, L, dtype)) != TTT_OK) return st;
  if ((st = check_row(ldy, (long long)H * P, L, dtype)) != TTT_OK) return st;
  if ((st = check_row(ldb, (long long)G * N, L, dtype)) != TTT_OK) return st;
  if ((st = check_row(ldc, (long long)G * N, L, dtype)) != TTT_OK) return st;
  REQUIRE(x, 16);
  REQUIRE(dt, size_of(dt_dtype));
  REQUIRE(A, 4);
  REQUIRE(Bm, 16);
  REQUIRE(Cm, 16);
  REQUIRE(dy, 16);
  REQUIRE(dx, 16);
  REQUIRE(ddt, size_of(dt_dtype));
  REQUIRE(dA, 4);
  REQUIRE(dB, 16);
  REQUIRE(dC, 16);
  OPTIONAL(D, 4);
  OPTIONAL(dt_bias, 4);
  OPTIONAL(dh_last, 16);
  OPTIONAL(dD, 4);
  OPTIONAL(ddt_bias, 4);
  OPTIONAL(dh0, 16);
  if (states == nullptr || states_bytes < s.states) return TTT_ERR_WORKSPACE;
  if (workspace == nullptr || workspace_bytes < ttt_scan_bwd_workspace_bytes(B, L, H, P, G, N, dtype))
    return TTT_ERR_WORKSPACE;
  if (!aligned(states, 16) || !aligned(workspace, 16)) return TTT_ERR_ALIGN;
  ttt::ScanParams p{};
  p.x = x;
  p.ldx = ldx;
  p.dt = dt;
  p.lddt = lddt;
  p.A = A;
  p.Bm = Bm;
  p.ldb = ldb;
  p.Cm = Cm;
  p.ldc = ldc;
  p.D = D;
  p.dt_bias = dt_bias;
  p.dy = dy;
  p.ldy = ldy;
  p.B = B;
  p.L = L;
  p.H = H;
  p.G = G;
  p.N = N;
  p.softplus = softplus != 0;
  p.dt_f32 = dt_dtype == TTT_DTYPE_F32;
  p.S = s.S;
  p.per = s.per;
  p.joined = s.S > kSelfJoined;
  p.splits = s.splits;
  char* ws = static_cast<char*>(workspace);
  float* gstates = reinterpret_cast<float*>(ws);
  ws += up256(s.states);
  if (s.S > 1) {
    p.seg = reinterpret_cast<float*>(ws);
    p.seg_decay = reinterpret_cast<float*>(ws + s.seg);
    ws += s.seg + s.decay;
  }
  p.partial = reinterpret_cast<float*>(ws);
  ws += s.partial;
  if (s.splits > 1) {
    p.dBp = reinterpret_cast<float*>(ws);
    p.dCp = reinterpret_cast<float*>(ws + s.split);
  }
  const hipStream_t hs = static_cast<hipStream_t>(stream);
  p.h0 = dh_last;
  p.h_last = dh0;
  p.states = gstates;
  p.dx = dx;
  const hipError_t e = ttt::launch_scan_walk_back(p, P, dtype, hs);
  if (e != hipSuccess) return TTT_ERR_HIP;
  p.states = const_cast<float*>(static_cast<const float*>(states));  // read only here
  p.gstates = gstates;
  p.ddt = ddt;
  p.dA = dA;
  p.dB = dB;
  p.dC = dC;
  p.dD = dD;
  p.ddt_bias = ddt_bias;
  return hip_status(ttt::launch_scan_bwd(p, P, dtype, hs));
}

int ttt_scan_step(const void* x, long long ldx, const void* dt, long long lddt, const float* A, const void* Bm,
                  long long ldb, const void* Cm, long long ldc, const float* D, const float* dt_bias, float* h, int B,
                  int H, int P, int G, int N, int dtype, int dt_dtype, int softplus, void* y, void* stream) {
  const int st = check_scan(B, 1, H, P, G, N, dtype, dt_dtype);
  if (st != TTT_OK) return st;
  if (lddt < H || ldx < (long long)H * P || ldb < (long long)G * N || ldc < (long long)G * N) return TTT_ERR_SHAPE;
  if ((long long)B * H * P > kMaxThreads / 32) return TTT_ERR_SHAPE;
  const size_t n = size_of(dtype);
  if (ldb * n % (4 * n) != 0 || ldc * n % (4 * n) != 0) return TTT_ERR_SHAPE;  // four values at a time
  REQUIRE(x, n);
  REQUIRE(dt, size_of(dt_dtype));
  REQUIRE(A, 4);
  REQUIRE(Bm, 4 * n);
  REQUIRE(Cm, 4 * n);
  REQUIRE(h, 16);
  REQUIRE(y, n);
  OPTIONAL(D, 4);
  OPTIONAL(dt_bias, 4);
  ttt::ScanStepParams p{};
  p.x = x;
  p.ldx = ldx;
  p.dt = dt;
  p.lddt = lddt;
  p.A = A;
  p.Bm = Bm;
  p.ldb = ldb;
  p.Cm = Cm;
  p.ldc = ldc;
  p.D = D;
  p.dt_bias = dt_bias;
  p.h = h;
  p.y = y;
  p.B = B;
  p.H = H;
  p.P = P;
  p.G = G;
  p.N = N;
  p.softplus = softplus != 0;
  p.dt_f32 = dt_dtype == TTT_DTYPE_F32;
  return hip_status(ttt::launch_scan_step(p, dtype, static_cast<hipStream_t>(stream)));
}

int ttt_layer_norm_fwd(const void* x, long long ldx, const void* gate, long long ldg, const float* weight,
                       const float* bias, long long R, int D, float eps, int dtype, void* y, float* stats,
                       void* stream) {
  const int st = check_norm(R, D, eps, dtype);
  if (st != TTT_OK) return st;
  if (ldx < D || (gate != nullptr && ldg < D)) return TTT_ERR_SHAPE;
  if ((weight == nullptr) != (bias == nullptr)) return TTT_ERR_NULL;
  const size_t n = size_of(dtype);
  REQUIRE(x, n);
  REQUIRE(y, n);
  OPTIONAL(gate, n);
  OPTIONAL(weight, 4);
  OPTIONAL(bias, 4);
  OPTIONAL(stats, 4);
  ttt::NormParams p{};
  p.x = x;
  p.ldx = ldx;
  p.gate = gate;
  p.ldg = ldg;
  p.w = weight;
  p.b = bias;
  p.R = R;
  p.D = D;
  p.eps = eps;
  p.y = y;
  p.stats = stats;
  return hip_status(ttt::launch_norm_fwd(p, dtype, static_cast<hipStream_t>(stream)));
}

size_t ttt_layer_norm_partial_bytes(long long R, int D) {
  if (check_norm(R, D, 1e-6f, TTT_DTYPE_F32) != TTT_OK) return 0;
  return (size_t)ttt::norm_bwd_parts(R, D) * 2 * D * sizeof(float);
}

int ttt_layer_norm_bwd(const void* x, long long ldx, const void* gate, long long ldg, const float* weight,
                       const float* stats, const void* dy, long long R, int D, int dtype, void* dx, void* dgate,
                       float* dweight, float* dbias, float* partial, size_t partial_bytes, void* stream) {
  const int st = check_norm(R, D, 1e-6f, dtype);
  if (st != TTT_OK) return st;
  if (ldx < D || (gate != nullptr && ldg < D)) return TTT_ERR_SHAPE;
  if ((gate == nullptr) != (dgate == nullptr) || (dweight == nullptr) != (dbias == nullptr)) return TTT_ERR_NULL;
  const size_t n = size_of(dtype);
  REQUIRE(x, n);
  REQUIRE(stats, 4);
  REQUIRE(dy, n);
  REQUIRE(dx, n);
  OPTIONAL(gate, n);
  OPTIONAL(dgate, n);
  OPTIONAL(weight, 4);
  OPTIONAL(dweight, 4);
  OPTIONAL(dbias, 4);
  if (dweight != nullptr) {
    if (partial == nullptr || partial_bytes < ttt_layer_norm_partial_bytes(R, D)) return TTT_ERR_WORKSPACE;
    if (!aligned(partial, 16)) return TTT_ERR_ALIGN;
  }
  ttt::NormParams p{};
  p.x = x;
  p.ldx = ldx;
  p.gate = gate;
  p.ldg = ldg;
  p.w = weight;
  p.stats = const_cast<float*>(stats);  // read only in the backward
  p.dy = dy;
  p.R = R;
  p.D = D;
  p.dx = dx;
  p.dgate = dgate;
  p.dw = dweight;
  p.db = dbias;
  p.partial = dweight != nullptr ? partial : nullptr;
  return hip_status(ttt::launch_norm_bwd(p, dtype, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
