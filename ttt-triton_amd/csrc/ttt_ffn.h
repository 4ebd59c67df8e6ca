// Kernel-side parameter blocks and launchers of the gated feed-forward projections
// (ttt_ffn.hip).  Internal to libttt_amd.so.
#pragma once

#include "ttt_ssm.h"

namespace ttt {

constexpr int kFfnStep = 64;  // contracted values of a step
constexpr int kFfnFew = 64;   // rows up to which a call is one of few rows

// What a product reads: a matrix of 16-bit elements in planes, rows `ld` bytes apart and on 16
// bytes, `plane` bytes between planes
struct FfnMatrix {
  const void* p;
  long long ld, plane;
};
struct FfnParams {
  FfnMatrix x, wg, wu, grad;  // [R][Dp], [F][Dp], [F][Dp], [R][2 Fp]: da and db side by side
  const void *bg, *bu;        // [F], or null
  const void* dy;             // [R][lddy]
  void* y;                    // [R][F]
  void *dx, *dwg, *dwu;       // [R][D], [F][D], [F][D]
  void *dbg, *dbu;            // [F], or null
  float* part;                // [splits][R or 2 Fp][Dp] of dx, or dwg and dwu, where their steps are split
  float* bias_part;           // [bias_parts][2 Fp], or null
  // fp16: whether a value of da or db is past its largest number, in blocks of 16 rows by 32 columns of both
  // and anywhere; `grad` has a second plane for those, read where there are any
  unsigned char* over;
  int* far;
  long long lddy;
  int R, D, F, Dp, Fp;        // widths as the user's and padded to 8
  int planes, act;
  int splits, whole;          // of the product that is launched (FfnCut)
  int bias_parts;
};
// few rows: the operands as the user's, rows of x ldx elements apart
hipError_t launch_ffn_few(const FfnParams& p, int dtype, hipStream_t stream);
hipError_t launch_ffn_fwd(const FfnParams& p, int dtype, hipStream_t stream);
hipError_t launch_ffn_grad(const FfnParams& p, int dtype, hipStream_t stream);  // writes `grad`, `over`, `far`, dbg, dbu
hipError_t launch_ffn_dx(const FfnParams& p, int dtype, hipStream_t stream);
hipError_t launch_ffn_dw(const FfnParams& p, int dtype, hipStream_t stream);
// rows of `width` values `ld` elements apart -> planes of rows padded with zeros to a multiple of 8
hipError_t launch_ffn_planes(const void* from, long long ld, int rows, int width, void* to, int dtype, hipStream_t stream);

constexpr int ffn_pad(int n) { return (n + 7) / 8 * 8; }
constexpr int ffn_planes(int dtype) { return dtype == TTT_DTYPE_F32 ? 3 : 1; }
constexpr int ffn_grad_planes(int dtype) { return dtype == TTT_DTYPE_F16 ? 2 : ffn_planes(dtype); }
constexpr int kFfnFarRows = 16, kFfnFarCols = 32;  // of a block of `over`: what a wave stores at once
constexpr int ffn_far_cols(int F) { return (F + kFfnFarCols - 1) / kFfnFarCols; }
constexpr long long ffn_far_blocks(long long R, int F) { return (R + kFfnFarRows - 1) / kFfnFarRows * ffn_far_cols(F); }

// How a product is cut up: tiles of 256 x 256, a workgroup to a compute unit, or of 128 x 128,
// two; and the steps of 64 contracted values of a tile into shares, whose sums are joined by
// another launch.  Or as many whole rounds of large tiles as there are, and what is left of them,
// less than a round, in four small ones each by another launch.
struct FfnCut {
  bool large;
  int splits;
  int whole;  // large tiles before the small ones, or 0: one size
};
// M x N results (the width of both projections together), `steps` of 64 contracted values, joined
// over `most` shares or fewer, `mixed` where two sizes may be.  In units of a step of a large tile
// (1.7 us at the rate of a large product), a small tile's takes 0.6 with another on the compute unit;
// a tile's start and end take about 5, another launch 2; a join reads and writes its sums at the
// card's bandwidth.  (Large and small: dx of 32,768 rows, 768 by 2,048, in one round of large tiles and one
// of small 262 us, in three of small 294; y of 4,099 rows, 1,024 by 2,731, fp16: 73 and two rounds of large 86.)
inline FfnCut ffn_cut(long long M, long long N, long long steps, int most, bool mixed) {
  FfnCut best{false, 1, 0};
  double least = 0.0;
  for (int large = 0; large < 2; ++large) {
    const long long side = large ? 256 : 128, places = large ? 256 : 512;
    const long long tiles = ((M + side - 1) / side) * ((N + side - 1) / side);
    for (int k = 1; k <= most && (k == 1 || k * 8 <= steps); ++k) {
      const double rounds = (double)((tiles * k + places - 1) / places);
      const double join = k > 1 ? 8.0 + 1e-6 * (double)(M * N) * (k + 1) : 0.0;
      const double time = rounds * ((double)((steps + k - 1) / k) * (large ? 1.0 : 0.6) + 5.0) + join;
      if ((large == 0 && k == 1) || time < least) {
        least = time;
        best = {large != 0, k, 0};
      }
    }
  }
  const long long tiles = ((M + 255) / 256) * ((N + 255) / 256), whole = tiles / 256 * 256;
  if (mixed && whole > 0 && whole < tiles) {
    const double small = (double)((4 * (tiles - whole) + 511) / 512);
    if ((double)(whole / 256) * ((double)steps + 5.0) + small * ((double)steps * 0.6 + 5.0) + 2.0 < least) best = {false, 1, (int)whole};
  }
  return best;
}
constexpr int kFfnMostSplits = 16;
inline long long ffn_steps(long long contracted, int dtype) {
  return (contracted + kFfnStep - 1) / kFfnStep * (dtype == TTT_DTYPE_F32 ? 6 : 1);
}
// (one size with sums of rows, which are by a tile's waves)
inline FfnCut ffn_cut_up(long long R, int D, int F, int dtype, bool sums) {
  return ffn_cut(R, 2LL * F, ffn_steps(ffn_pad(D), dtype), 1, !sums);
}
inline FfnCut ffn_cut_dx(long long R, int D, int F, int dtype) {
  return ffn_cut(R, D, 2 * ffn_steps(ffn_pad(F), dtype), kFfnMostSplits, true);
}
inline FfnCut ffn_cut_dw(long long R, int D, int F, int dtype) {
  return ffn_cut(2LL * ffn_pad(F), D, ffn_steps(R, dtype), kFfnMostSplits, false);
}
// rows of partial sums of the bias gradients: one to a wave's rows
inline int ffn_bias_parts(long long R, int D, int F, int dtype) {
  const long long side = ffn_cut_up(R, D, F, dtype, true).large ? 256 : 128;
  return (int)((R + side - 1) / side) * 2;
}

}  // namespace ttt
