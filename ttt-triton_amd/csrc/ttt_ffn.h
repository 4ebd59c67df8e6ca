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
  float* part;                // [splits][2 Fp][Dp] of dwg and dwu where the rows are split, else null
  float* bias_part;           // [bias_parts][2 Fp], or null
  long long lddy;
  int R, D, F, Dp, Fp;        // widths as the user's and padded to 8
  int planes, act;
  int splits, bias_parts;
};
// few rows: the operands as the user's, rows of x ldx elements apart
hipError_t launch_ffn_few(const FfnParams& p, int dtype, hipStream_t stream);
hipError_t launch_ffn_fwd(const FfnParams& p, int dtype, hipStream_t stream);
hipError_t launch_ffn_grad(const FfnParams& p, int dtype, hipStream_t stream);  // writes `grad`, dbg, dbu
hipError_t launch_ffn_dx(const FfnParams& p, int dtype, hipStream_t stream);
hipError_t launch_ffn_dw(const FfnParams& p, int dtype, hipStream_t stream);
// rows of `width` values `ld` elements apart -> planes of rows padded with zeros to a multiple of 8
hipError_t launch_ffn_planes(const void* from, long long ld, int rows, int width, void* to, int dtype, hipStream_t stream);

constexpr int ffn_pad(int n) { return (n + 7) / 8 * 8; }
constexpr int ffn_planes(int dtype) { return dtype == TTT_DTYPE_F32 ? 3 : 1; }
// Tiles of 256 x 256 where they make three quarters of a workgroup to each compute unit, else of 128 x 128
constexpr bool ffn_large(long long m, long long n) { return ((m + 255) / 256) * ((n + 255) / 256) >= 192; }
// rows of partial sums of the bias gradients: one to a wave's rows
constexpr int ffn_bias_parts(long long R, int F) {
  return ffn_large(R, 2LL * F) ? (int)((R + 255) / 256) * 2 : (int)((R + 127) / 128) * 2;
}
int ffn_splits(int R, int D, int F, int dtype);

}  // namespace ttt
