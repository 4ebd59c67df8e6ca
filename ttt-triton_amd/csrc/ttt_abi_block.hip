// extern "C" entry points of a gated delta-rule block's operators: host-side validation
// and workspace layout, then launches on the caller's stream.  Declarations and argument
// contracts are in include/ttt_amd.h.
#include <stdint.h>

#include <algorithm>

#include "ttt_abi_check.h"
#include "ttt_block_norm.h"
#include "ttt_delta.h"
#include "ttt_ffn.h"

namespace {

// ---- gated delta rule
int check_delta(int B, int L, int H, int P, int G, int N, int dtype, int g_dtype, int beta_dtype) {
  if (!dtype_ok(dtype)) return TTT_ERR_DTYPE;
  for (int d : {g_dtype, beta_dtype})
    if (d != dtype && d != TTT_DTYPE_F32) return TTT_ERR_DTYPE;
  if (B <= 0 || L <= 0 || H <= 0 || G <= 0 || H % G != 0) return TTT_ERR_SHAPE;
  if (P < 32 || P > ttt::kDeltaMaxP || P % 32 != 0 || N < 16 || N > 128 || N % 16 != 0) return TTT_ERR_SHAPE;
  if (L > 0x7fffff00 || (long long)B * H > kMaxGrid || H > (1 << 23) / P || G > (1 << 23) / N) return TTT_ERR_SHAPE;
  return TTT_OK;
}
struct DeltaPlan {
  int Q, NC, share, S, per;
  size_t tok, zm, states, rows, qk, seg, trans;
};
// Segments that the tokens are cut into: as many as make the walk quickest.  In units of a chunk's
// walk with outputs (3.6 to 5.9 us with 64 tokens, 2.2 to 3.8 with 32), one without takes 0.7, a
// segment's join 0.3 and two more launches 2; a compute unit holds one workgroup of 64 features or
// of states over 64 wide, else two.  (Kernels of 16,384 tokens of 12 heads of 64 x 64 in bf16: 930 us
// with one, 160 with 20; 32,768 tokens of 16 x 12 heads fill the compute units with one.)
int delta_segments(long long heads, int P, int NP, int NC) {
  const int wide = P % 64 == 0 && NP < 128 ? 64 : 32, places = wide == 64 || NP == 128 ? 256 : 512;
  const auto rounds = [&](long long columns) { return (double)((heads * columns / wide + places - 1) / places); };
  int best = 1;
  double least = rounds(P) * NC;
  for (int want = 2; want <= std::min(NC, 128); ++want) {
    const int per = (NC + want - 1) / want, S = (NC + per - 1) / per;
    const double time = rounds((long long)P * S) * per + rounds((long long)(P + NP) * (S - 1)) * per * 0.7 + 0.3 * S + 2.0;
    if (time < least) {
      least = time;
      best = S;
    }
  }
  return best;
}
DeltaPlan delta_plan(int B, int L, int H, int P, int G, int N, int dtype) {
  DeltaPlan s;
  s.Q = ttt::delta_chunk(dtype);
  s.NC = (L + s.Q - 1) / s.Q;
  s.share = H / G;
  const size_t chunks = (size_t)B * H * s.NC;
  s.tok = up256(chunks * ttt::delta_tok_floats(s.Q) * 4);
  s.zm = chunks * ttt::delta_tiles(s.Q) * 1024;
  s.states = chunks * P * ttt::scan_padded(N) * 4;
  s.rows = chunks * P * s.Q * 4;
  s.qk = s.share > 1 ? (size_t)s.share * B * L * G * N * 4 : 0;
  const int NP = ttt::scan_padded(N), want = delta_segments((long long)B * H, P, NP, s.NC);
  s.per = (s.NC + want - 1) / want;
  s.S = (s.NC + s.per - 1) / s.per;
  s.seg = s.S > 1 ? (size_t)B * H * s.S * NP * P * 4 : 0;
  s.trans = s.S > 1 ? (size_t)B * H * s.S * NP * NP * 4 : 0;
  return s;
}
// (forwards, prep: 256 threads a chunk and head; walk: eight for a column, a feature or one of the identity's, and
// segment; join: up to 32 a feature; where a backward follows its gradients: 512 a chunk and head, and the sums of
// the heads that share q and k: one for four values of both)
bool delta_grid_ok(const DeltaPlan& s, int B, int L, int H, int P, int G, int N, bool train) {
  const long long heads = (long long)B * H;
  if (heads * (P + 128) > kMaxThreads / 8 / s.S || heads * P > kMaxThreads / 32 || heads > kMaxThreads / (train ? 512 : 256) / s.NC)
    return false;
  return !train || s.share == 1 || (long long)B * L * G <= (kMaxThreads - 255) * 2 / N;
}
bool delta_plan_ok(int B, int L, int H, int P, int G, int N, int dtype, bool train, DeltaPlan& s) {
  if (check_delta(B, L, H, P, G, N, dtype, dtype, dtype) != TTT_OK) return false;
  s = delta_plan(B, L, H, P, G, N, dtype);
  return delta_grid_ok(s, B, L, H, P, G, N, train);
}

// ---- norms around a block
int check_block(long long R, int D, int heads, long long ldx, long long ldg, long long ldr, bool gate, bool res,
                const float* w2, int dtype, int res_dtype) {
  if (!dtype_ok(dtype) || (res_dtype != -1 && res_dtype != dtype && res_dtype != TTT_DTYPE_F32)) return TTT_ERR_DTYPE;
  if (R <= 0 || R > kMaxGrid || D <= 0 || D > ttt::kBlockNormMaxD || heads <= 0 || R % heads != 0) return TTT_ERR_SHAPE;
  const long long least = (long long)heads * D;
  if (ldx < least || (gate && ldg < least) || (res && ldr < least)) return TTT_ERR_SHAPE;
  // (a launch has whole wider rows: 2^31 threads are enough for one)
  if ((long long)heads * ttt::block_lanes(D) > 0x7fffffffLL) return TTT_ERR_SHAPE;
  if (w2 != nullptr && res_dtype == -1) return TTT_ERR_ARG;
  return TTT_OK;
}

// ---- gated feed-forward projections
constexpr int kFfnMaxWidth = 1 << 20;  // rows of a tile are reached by 31-bit offsets
int check_ffn(int R, int D, int F, int act, int dtype) {
  if (!dtype_ok(dtype)) return TTT_ERR_DTYPE;
  if (R <= 0 || D <= 0 || F <= 0 || D > kFfnMaxWidth || F > kFfnMaxWidth || R > 0x7fffff00) return TTT_ERR_SHAPE;
  if (act != TTT_ACT_SILU && act != TTT_ACT_GELU) return TTT_ERR_ARG;
  // (tiles of 128 x 128 with 256 threads; planes 8 values a thread)
  const long long n = std::max(2LL * F, (long long)D), m = std::max<long long>(R, 2LL * F + 16);
  if (((m + 127) / 128) * ((n + 127) / 128) > kMaxThreads / 256 / ttt::kFfnMostSplits) return TTT_ERR_SHAPE;
  if (std::max<long long>(R, F) * (ttt::ffn_pad(D) / 8) > kMaxThreads) return TTT_ERR_SHAPE;
  return TTT_OK;
}
struct FfnPlan {
  bool in_place;
  size_t x, w, grad, part, bias, far;
  size_t backward() const { return x + 2 * w + grad + part + bias + far; }
};
FfnPlan ffn_plan(int R, int D, int F, int dtype) {
  FfnPlan s;
  const size_t Dp = ttt::ffn_pad(D), Fp = ttt::ffn_pad(F), planes = ttt::ffn_planes(dtype);
  s.in_place = planes == 1 && D % 8 == 0;
  s.x = s.in_place ? 0 : up256(planes * R * Dp * 2);
  s.w = s.in_place ? 0 : up256(planes * F * Dp * 2);
  s.grad = up256((size_t)ttt::ffn_grad_planes(dtype) * R * 2 * Fp * 2);
  const int of_dx = ttt::ffn_cut_dx(R, D, F, dtype).splits, of_dw = ttt::ffn_cut_dw(R, D, F, dtype).splits;
  const size_t dx = of_dx > 1 ? (size_t)of_dx * R * Dp * 4 : 0, dw = of_dw > 1 ? (size_t)of_dw * 2 * Fp * Dp * 4 : 0;
  s.part = up256(std::max(dx, dw));  // (one after the other)
  s.bias = up256((size_t)ttt::ffn_bias_parts(R, D, F, dtype) * 2 * Fp * 4);
  s.far = dtype == TTT_DTYPE_F16 ? 256 + up256((size_t)ttt::ffn_far_blocks(R, F)) : 0;
  return s;
}
// x, wg and wu as the products read them: in place, or as planes in the workspace
hipError_t ffn_operands(ttt::FfnParams& p, const FfnPlan& s, const void* x, long long ldx, const void* wg, const void* wu,
                        int dtype, char*& ws, hipStream_t stream) {
  const long long es = size_of(dtype);
  if (s.in_place) {
    p.x = {x, ldx * es, 0};
    p.wg = {wg, p.D * es, 0};
    p.wu = {wu, p.D * es, 0};
    return hipSuccess;
  }
  const auto make = [&](ttt::FfnMatrix& m, const void* from, long long ld, int rows, size_t bytes) {
    m = {ws, p.Dp * 2LL, (long long)rows * p.Dp * 2};
    ws += bytes;
    return ttt::launch_ffn_planes(from, ld, rows, p.D, const_cast<void*>(m.p), dtype, stream);
  };
  hipError_t e = make(p.x, x, ldx, p.R, s.x);
  if (e == hipSuccess) e = make(p.wg, wg, p.D, p.F, s.w);
  if (e == hipSuccess) e = make(p.wu, wu, p.D, p.F, s.w);
  return e;
}
int check_ffn_rows(bool in_place, const void* x, long long ldx, const void* wg, const void* wu, int D, int dtype) {
  if (ldx < D) return TTT_ERR_SHAPE;
  const size_t n = in_place ? 16 : size_of(dtype);
  if (in_place && (ldx % 8 != 0 || ldx > (4 << 20) / 2)) return TTT_ERR_SHAPE;
  REQUIRE(x, n);
  REQUIRE(wg, n);
  REQUIRE(wu, n);
  return TTT_OK;
}

}  // namespace

extern "C" {

size_t ttt_ffn_workspace_bytes(int R, int D, int F, int dtype) {
  if (check_ffn(R, D, F, TTT_ACT_SILU, dtype) != TTT_OK || R <= ttt::kFfnFew) return 0;
  const FfnPlan s = ffn_plan(R, D, F, dtype);
  return s.x + 2 * s.w;
}
size_t ttt_ffn_bwd_workspace_bytes(int R, int D, int F, int dtype) {
  if (check_ffn(R, D, F, TTT_ACT_SILU, dtype) != TTT_OK) return 0;
  const FfnPlan s = ffn_plan(R, D, F, dtype);
  return s.backward();
}

int ttt_ffn_fwd(const void* x, long long ldx, const void* wg, const void* wu, const void* bg, const void* bu, int R,
                int D, int F, int activation, int dtype, void* y, void* workspace, size_t workspace_bytes,
                void* stream) {
  int st = check_ffn(R, D, F, activation, dtype);
  if (st != TTT_OK) return st;
  const bool few = R <= ttt::kFfnFew;
  const FfnPlan s = ffn_plan(R, D, F, dtype);
  if ((st = check_ffn_rows(!few && s.in_place, x, ldx, wg, wu, D, dtype)) != TTT_OK) return st;
  const size_t n = size_of(dtype);
  OPTIONAL(bg, n);
  OPTIONAL(bu, n);
  REQUIRE(y, n);
  ttt::FfnParams p{};
  p.bg = bg;
  p.bu = bu;
  p.y = y;
  p.R = R;
  p.D = D;
  p.F = F;
  p.Dp = ttt::ffn_pad(D);
  p.Fp = ttt::ffn_pad(F);
  p.planes = ttt::ffn_planes(dtype);
  p.act = activation;
  const hipStream_t on = static_cast<hipStream_t>(stream);
  if (few) {
    const long long es = size_of(dtype);
    p.x = {x, ldx * es, 0};
    p.wg = {wg, D * es, 0};
    p.wu = {wu, D * es, 0};
    return hip_status(ttt::launch_ffn_few(p, dtype, on));
  }
  const size_t need = s.x + 2 * s.w;
  if (need > 0) {
    if (workspace == nullptr || workspace_bytes < need) return TTT_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return TTT_ERR_ALIGN;
  }
  char* ws = static_cast<char*>(workspace);
  const hipError_t e = ffn_operands(p, s, x, ldx, wg, wu, dtype, ws, on);
  if (e != hipSuccess) return hip_status(e);
  return hip_status(ttt::launch_ffn_fwd(p, dtype, on));
}

int ttt_ffn_bwd(const void* x, long long ldx, const void* wg, const void* wu, const void* bg, const void* bu,
                const void* dy, long long lddy, int R, int D, int F, int activation, int dtype, void* dx, void* dwg,
                void* dwu, void* dbg, void* dbu, void* workspace, size_t workspace_bytes, void* stream) {
  int st = check_ffn(R, D, F, activation, dtype);
  if (st != TTT_OK) return st;
  const FfnPlan s = ffn_plan(R, D, F, dtype);
  if ((st = check_ffn_rows(s.in_place, x, ldx, wg, wu, D, dtype)) != TTT_OK) return st;
  if (lddy < F) return TTT_ERR_SHAPE;
  const size_t n = size_of(dtype);
  OPTIONAL(bg, n);
  OPTIONAL(bu, n);
  REQUIRE(dy, n);
  OPTIONAL(dx, n);
  OPTIONAL(dwg, n);
  OPTIONAL(dwu, n);
  OPTIONAL(dbg, n);
  OPTIONAL(dbu, n);
  if ((dwg == nullptr) != (dwu == nullptr)) return TTT_ERR_ARG;
  if (workspace == nullptr || workspace_bytes < s.backward()) return TTT_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return TTT_ERR_ALIGN;
  ttt::FfnParams p{};
  p.bg = bg;
  p.bu = bu;
  p.dy = dy;
  p.lddy = lddy;
  p.R = R;
  p.D = D;
  p.F = F;
  p.Dp = ttt::ffn_pad(D);
  p.Fp = ttt::ffn_pad(F);
  p.planes = ttt::ffn_planes(dtype);
  p.act = activation;
  p.dx = dx;
  p.dwg = dwg;
  p.dwu = dwu;
  p.dbg = dbg;
  p.dbu = dbu;
  p.bias_parts = ttt::ffn_bias_parts(R, D, F, dtype);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  hipError_t e = ffn_operands(p, s, x, ldx, wg, wu, dtype, ws, on);
  if (e != hipSuccess) return hip_status(e);
  p.grad = {ws, 4LL * p.Fp, (long long)R * 4 * p.Fp};
  ws += s.grad;
  if (s.part > 0) p.part = reinterpret_cast<float*>(ws);
  ws += s.part;
  if (dbg != nullptr || dbu != nullptr) p.bias_part = reinterpret_cast<float*>(ws);
  ws += s.bias;
  if (s.far > 0) {
    p.far = reinterpret_cast<int*>(ws);
    p.over = reinterpret_cast<unsigned char*>(ws + 256);
  }
  e = ttt::launch_ffn_grad(p, dtype, on);
  if (e == hipSuccess && dx != nullptr) e = ttt::launch_ffn_dx(p, dtype, on);
  if (e == hipSuccess && dwg != nullptr) e = ttt::launch_ffn_dw(p, dtype, on);
  return hip_status(e);
}

int ttt_block_norm_fwd(const void* x, long long ldx, const void* gate, long long ldg, const void* residual,
                       long long ldr, const float* w, const float* s, const float* w2, long long R, int D, int heads,
                       float eps, int dtype, int res_dtype, void* r, void* y, float* stats, void* stream) {
  const int st = check_block(R, D, heads, ldx, ldg, ldr, gate != nullptr, residual != nullptr, w2, dtype, res_dtype);
  if (st != TTT_OK) return st;
  if (!(eps > 0.0f) || eps > 1.0f) return TTT_ERR_ARG;
  const size_t n = size_of(dtype), nr = res_dtype == -1 ? n : size_of(res_dtype);
  REQUIRE(x, n);
  OPTIONAL(gate, n);
  if (res_dtype != -1)
    REQUIRE(residual, nr);
  else if (residual != nullptr)
    return TTT_ERR_ARG;
  OPTIONAL(w, 4);
  OPTIONAL(s, 4);
  OPTIONAL(w2, 4);
  REQUIRE(r, nr);
  if (w2 != nullptr) REQUIRE(y, n);
  OPTIONAL(stats, 4);
  ttt::BlockNormParams p{};
  p.x = x;
  p.ldx = ldx;
  p.gate = gate;
  p.ldg = ldg;
  p.res = residual;
  p.ldr = ldr;
  p.w = w;
  p.s = s;
  p.w2 = w2;
  p.R = R;
  p.D = D;
  p.heads = heads;
  p.eps = eps;
  p.r = r;
  p.y = y;
  p.stats = stats;
  return hip_status(ttt::launch_block_norm_fwd(p, dtype, res_dtype, static_cast<hipStream_t>(stream)));
}

size_t ttt_block_norm_partial_bytes(long long R, int D) {
  if (R <= 0 || R > kMaxGrid || D <= 0 || D > ttt::kBlockNormMaxD) return 0;
  return (size_t)ttt::block_norm_parts(R, D) * 3 * D * sizeof(float);
}

int ttt_block_norm_bwd(const void* x, long long ldx, const void* gate, long long ldg, const void* residual,
                       long long ldr, const float* w, const float* s, const float* w2, const float* stats,
                       const void* dr, const void* dy, long long R, int D, int heads, int dtype, int res_dtype,
                       void* dx, void* dgate, void* dresidual, float* dw, float* ds, float* dw2, float* partial,
                       size_t partial_bytes, void* stream) {
  const bool reads = w2 != nullptr;
  const int st = check_block(R, D, heads, ldx, ldg, ldr, gate != nullptr, reads, w2, dtype, res_dtype);
  if (st != TTT_OK) return st;
  const size_t n = size_of(dtype), nr = res_dtype == -1 ? n : size_of(res_dtype);
  REQUIRE(x, n);
  OPTIONAL(gate, n);
  if (reads) REQUIRE(residual, nr);
  OPTIONAL(w, 4);
  OPTIONAL(s, 4);
  OPTIONAL(w2, 4);
  REQUIRE(stats, 4);
  OPTIONAL(dr, nr);
  OPTIONAL(dy, n);
  REQUIRE(dx, n);
  if (gate != nullptr) REQUIRE(dgate, n);
  OPTIONAL(dresidual, nr);
  OPTIONAL(dw, 4);
  OPTIONAL(ds, 4);
  OPTIONAL(dw2, 4);
  if ((dw != nullptr && w == nullptr) || (ds != nullptr && s == nullptr) || (dw2 != nullptr && w2 == nullptr) ||
      (dresidual != nullptr && res_dtype == -1))
    return TTT_ERR_ARG;
  if (dw != nullptr || ds != nullptr || dw2 != nullptr) {
    if (partial == nullptr || partial_bytes < ttt_block_norm_partial_bytes(R, D)) return TTT_ERR_WORKSPACE;
    if (!aligned(partial, 4)) return TTT_ERR_ALIGN;
  }
  ttt::BlockNormParams p{};
  p.x = x;
  p.ldx = ldx;
  p.gate = gate;
  p.ldg = ldg;
  p.res = residual;
  p.ldr = ldr;
  p.w = w;
  p.s = s;
  p.w2 = w2;
  p.stats = const_cast<float*>(stats);
  p.dr = dr;
  p.dy = dy;
  p.R = R;
  p.D = D;
  p.heads = heads;
  p.dx = dx;
  p.dgate = dgate;
  p.dres = dresidual;
  p.dw = dw;
  p.ds = ds;
  p.dw2 = dw2;
  if (dw != nullptr || ds != nullptr || dw2 != nullptr) p.partial = partial;
  return hip_status(ttt::launch_block_norm_bwd(p, dtype, res_dtype, static_cast<hipStream_t>(stream)));
}

size_t ttt_delta_saved_bytes(int B, int L, int H, int P, int N, int dtype) {
  DeltaPlan s;
  return delta_plan_ok(B, L, H, P, 1, N, dtype, true, s) ? s.states + s.rows : 0;
}
size_t ttt_delta_workspace_bytes(int B, int L, int H, int P, int N, int dtype) {
  DeltaPlan s;
  return delta_plan_ok(B, L, H, P, 1, N, dtype, false, s) ? s.tok + 2 * s.zm + s.seg + s.trans : 0;
}
size_t ttt_delta_bwd_workspace_bytes(int B, int L, int H, int P, int G, int N, int dtype) {
  DeltaPlan s;
  return delta_plan_ok(B, L, H, P, G, N, dtype, true, s) ? s.states + s.rows + 2 * s.qk + s.seg : 0;
}

int ttt_delta_fwd(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv,
                  const void* g, long long ldg, const void* beta, long long ldbeta, const float* h0, int B, int L,
                  int H, int P, int G, int N, float scale, int unit, int dtype, int g_dtype, int beta_dtype, void* o,
                  float* h_last, void* saved, size_t saved_bytes, void* workspace, size_t workspace_bytes,
                  void* stream) {
  int st = check_delta(B, L, H, P, G, N, dtype, g_dtype, beta_dtype);
  if (st != TTT_OK) return st;
  const DeltaPlan s = delta_plan(B, L, H, P, G, N, dtype);
  if (!delta_grid_ok(s, B, L, H, P, G, N, saved != nullptr)) return TTT_ERR_SHAPE;
  if (ldg < H || ldbeta < H) return TTT_ERR_SHAPE;
  if ((st = check_row(ldq, (long long)G * N, L, dtype)) != TTT_OK) return st;
  if ((st = check_row(ldk, (long long)G * N, L, dtype)) != TTT_OK) return st;
  if ((st = check_row(ldv, (long long)H * P, L, dtype)) != TTT_OK) return st;
  REQUIRE(q, 16);
  REQUIRE(k, 16);
  REQUIRE(v, 16);
  REQUIRE(g, size_of(g_dtype));
  REQUIRE(beta, size_of(beta_dtype));
  REQUIRE(o, 16);
  OPTIONAL(h0, 16);
  OPTIONAL(h_last, 16);
  OPTIONAL(saved, 16);
  if (saved != nullptr && saved_bytes < s.states + s.rows) return TTT_ERR_WORKSPACE;
  if (workspace == nullptr || workspace_bytes < s.tok + 2 * s.zm + s.seg + s.trans) return TTT_ERR_WORKSPACE;
  OPTIONAL(workspace, 16);
  ttt::DeltaParams p{};
  p.q = q;
  p.k = k;
  p.v = v;
  p.g = g;
  p.beta = beta;
  p.ldq = ldq;
  p.ldk = ldk;
  p.ldv = ldv;
  p.ldg = ldg;
  p.ldbeta = ldbeta;
  p.h0 = h0;
  p.o = o;
  p.h_last = h_last;
  p.B = B;
  p.L = L;
  p.H = H;
  p.G = G;
  p.N = N;
  p.P = P;
  p.scale = scale;
  p.l2 = unit != 0;
  p.g_f32 = g_dtype == TTT_DTYPE_F32;
  p.beta_f32 = beta_dtype == TTT_DTYPE_F32;
  char* ws = static_cast<char*>(workspace);
  p.tok = reinterpret_cast<float*>(ws);
  p.z = reinterpret_cast<float*>(ws + s.tok);
  p.m = reinterpret_cast<float*>(ws + s.tok + s.zm);
  p.S = s.S;
  p.per = s.per;
  if (s.S > 1) {
    p.seg = reinterpret_cast<float*>(ws + s.tok + 2 * s.zm);
    p.trans = reinterpret_cast<float*>(ws + s.tok + 2 * s.zm + s.seg);
  }
  if (saved != nullptr) {
    p.states = static_cast<float*>(saved);
    p.rows = reinterpret_cast<float*>(static_cast<char*>(saved) + s.states);
  }
  const hipError_t e = ttt::launch_delta_prep(p, dtype, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_status(e);
  return hip_status(ttt::launch_delta_fwd(p, dtype, static_cast<hipStream_t>(stream)));
}

int ttt_delta_bwd(const void* q, long long ldq, const void* k, long long ldk, const void* g, long long ldg,
                  const void* beta, long long ldbeta, const void* dO, long long lddo, const float* dh_last,
                  const void* saved, size_t saved_bytes, const void* kept, size_t kept_bytes, int B, int L, int H,
                  int P, int G, int N, float scale, int unit, int dtype, int g_dtype, int beta_dtype, void* dq, void* dk, void* dv, void* dg,
                  void* dbeta, float* dh0, void* workspace, size_t workspace_bytes, void* stream) {
  int st = check_delta(B, L, H, P, G, N, dtype, g_dtype, beta_dtype);
  if (st != TTT_OK) return st;
  const DeltaPlan s = delta_plan(B, L, H, P, G, N, dtype);
  if (!delta_grid_ok(s, B, L, H, P, G, N, true)) return TTT_ERR_SHAPE;
  if (ldg < H || ldbeta < H) return TTT_ERR_SHAPE;
  if ((st = check_row(ldq, (long long)G * N, L, dtype)) != TTT_OK) return st;
  if ((st = check_row(ldk, (long long)G * N, L, dtype)) != TTT_OK) return st;
  if ((st = check_row(lddo, (long long)H * P, L, dtype)) != TTT_OK) return st;
  REQUIRE(q, 16);
  REQUIRE(k, 16);
  REQUIRE(g, size_of(g_dtype));
  REQUIRE(beta, size_of(beta_dtype));
  REQUIRE(dO, 16);
  REQUIRE(saved, 16);
  REQUIRE(kept, 16);
  REQUIRE(dq, 16);
  REQUIRE(dk, 16);
  REQUIRE(dv, 16);
  REQUIRE(dg, size_of(g_dtype));
  REQUIRE(dbeta, size_of(beta_dtype));
  OPTIONAL(dh_last, 16);
  OPTIONAL(dh0, 16);
  if (saved_bytes < s.states + s.rows || kept_bytes < s.tok + 2 * s.zm + s.seg + s.trans)
    return TTT_ERR_WORKSPACE;
  if (workspace == nullptr || workspace_bytes < s.states + s.rows + 2 * s.qk + s.seg) return TTT_ERR_WORKSPACE;
  OPTIONAL(workspace, 16);
  ttt::DeltaParams p{};
  p.q = q;
  p.k = k;
  p.g = g;
  p.beta = beta;
  p.ldq = ldq;
  p.ldk = ldk;
  p.ldg = ldg;
  p.ldbeta = ldbeta;
  p.dO = dO;
  p.lddo = lddo;
  p.h0 = dh_last;
  p.o = dv;
  p.h_last = dh0;
  p.B = B;
  p.L = L;
  p.H = H;
  p.G = G;
  p.N = N;
  p.P = P;
  p.scale = scale;
  p.l2 = unit != 0;
  p.g_f32 = g_dtype == TTT_DTYPE_F32;
  p.beta_f32 = beta_dtype == TTT_DTYPE_F32;
  char* ws = static_cast<char*>(workspace);
  const auto take = [&ws](size_t n) {
    char* at = ws;
    ws += n;
    return at;
  };
  float* const of = const_cast<float*>(static_cast<const float*>(kept));  // read only
  p.tok = of;
  p.z = of + s.tok / 4;
  p.m = of + (s.tok + s.zm) / 4;
  p.states = reinterpret_cast<float*>(take(s.states));
  p.rows = reinterpret_cast<float*>(take(s.rows));
  p.S = s.S;
  p.per = s.per;
  if (s.S > 1) {
    p.seg = reinterpret_cast<float*>(take(s.seg));
    p.trans = of + (s.tok + 2 * s.zm + s.seg) / 4;
  }
  if (s.share > 1) {
    p.dqp = reinterpret_cast<float*>(take(s.qk));
    p.dkp = reinterpret_cast<float*>(take(s.qk));
  }
  const hipStream_t on = static_cast<hipStream_t>(stream);
  const hipError_t e = ttt::launch_delta_walk_back(p, dtype, on);
  if (e != hipSuccess) return hip_status(e);
  p.gstates = p.states;
  p.states = const_cast<float*>(static_cast<const float*>(saved));
  p.x = reinterpret_cast<const float*>(static_cast<const char*>(saved) + s.states);
  p.dq = dq;
  p.dk = dk;
  p.dg = dg;
  p.dbeta = dbeta;
  return hip_status(ttt::launch_delta_bwd(p, dtype, on));
}

int ttt_delta_step(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv,
                   const void* g, long long ldg, const void* beta, long long ldbeta, float* h, int B, int H, int P,
                   int G, int N, float scale, int unit, int dtype, int g_dtype, int beta_dtype, void* o,
                   void* stream) {
  const int st = check_delta(B, 1, H, P, G, N, dtype, g_dtype, beta_dtype);
  if (st != TTT_OK) return st;
  // (up to 32 threads to a feature, and the last workgroup's idle ones)
  if ((long long)B * H > kMaxThreads / 32 / P - 1) return TTT_ERR_SHAPE;
  if (ldg < H || ldbeta < H || ldv < (long long)H * P || ldq < (long long)G * N || ldk < (long long)G * N || ldq % 4 != 0 ||
      ldk % 4 != 0)
    return TTT_ERR_SHAPE;
  const size_t n = size_of(dtype);
  REQUIRE(q, 4 * n);
  REQUIRE(k, 4 * n);
  REQUIRE(v, n);
  REQUIRE(g, size_of(g_dtype));
  REQUIRE(beta, size_of(beta_dtype));
  REQUIRE(h, 16);
  REQUIRE(o, n);
  ttt::DeltaStepParams p{};
  p.q = q;
  p.k = k;
  p.v = v;
  p.g = g;
  p.beta = beta;
  p.ldq = ldq;
  p.ldk = ldk;
  p.ldv = ldv;
  p.ldg = ldg;
  p.ldbeta = ldbeta;
  p.h = h;
  p.o = o;
  p.B = B;
  p.H = H;
  p.P = P;
  p.G = G;
  p.N = N;
  p.scale = scale;
  p.l2 = unit != 0;
  p.g_f32 = g_dtype == TTT_DTYPE_F32;
  p.beta_f32 = beta_dtype == TTT_DTYPE_F32;
  return hip_status(ttt::launch_delta_step(p, dtype, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
