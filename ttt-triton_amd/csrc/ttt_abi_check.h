// Host-side checks that the C entry points share (ttt_abi_ssm.hip, ttt_abi_block.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/ttt_amd.h"

namespace {

bool dtype_ok(int d) { return d == TTT_DTYPE_F32 || d == TTT_DTYPE_BF16 || d == TTT_DTYPE_F16; }
int size_of(int d) { return d == TTT_DTYPE_F32 ? 4 : 2; }
bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int hip_status(hipError_t e) { return e == hipSuccess ? TTT_OK : TTT_ERR_HIP; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

#define REQUIRE(p, n)                           \
  do {                                          \
    if ((p) == nullptr) return TTT_ERR_NULL;    \
    if (!aligned(p, n)) return TTT_ERR_ALIGN;   \
  } while (0)
#define OPTIONAL(p, n)                                                \
  do {                                                                \
    if ((p) != nullptr && !aligned(p, n)) return TTT_ERR_ALIGN;       \
  } while (0)

constexpr long long kMaxGrid = 0x7fffffffLL;
constexpr long long kMaxThreads = 0xffffffffLL;  // of a launch

// a chunk's rows, up to 64, are reached by 32-bit offsets
int check_row(long long ld, long long least, int L, int dtype) {
  if (ld < least || ld * size_of(dtype) % 16 != 0) return TTT_ERR_SHAPE;
  return L > 1 && ld >= (1LL << 26) / size_of(dtype) ? TTT_ERR_SHAPE : TTT_OK;
}

}  // namespace
