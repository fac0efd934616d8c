// Layout of the paged latent cache, shared by the latent-attention units.
//
// A cached token is 512 latent values and a rotary key of 64. A 16-bit page holds page_size
// rows of 576 elements. An e4m3 page of page_size * 644 bytes holds three parts, each
// contiguous over the page's tokens so that a tile of one part is a plain 2-D box:
//   codes  [page_size][512]  e4m3, one scale per 128
//   rope   [page_size][64]   bf16
//   scales [page_size][4]    UE8M0 exponent bytes: the block's scale is 2^(byte - 127)
// Power-of-two scales make code * scale exact in fp32 and, away from bf16's subnormal range,
// in bf16, so nothing is rounded when a page is read back.
#pragma once

#include "common.cuh"
#include "moe_internal.h"

namespace moe {

constexpr int kLatDim = 512;   // latent values per token (keys and values share them)
constexpr int kRopeDim = 64;   // rotary key values per token
constexpr int kRowDim = kLatDim + kRopeDim;
constexpr int kLatBlk = 128;   // latent values per e4m3 scale
constexpr int kRow8Bytes = kLatDim + 2 * kRopeDim + kLatDim / kLatBlk;  // 644
constexpr int kNopeDim = 128;  // per-head key part without position, and per-head value (expanded form)
constexpr int kQkDim = kNopeDim + kRopeDim;

inline bool cache_fmt_ok(int f) { return f == MOE_DTYPE_BF16 || f == MOE_DTYPE_FP16 || f == MOE_CACHE_E4M3; }
inline bool page_size_ok(int p) { return p == 16 || p == 32 || p == 64 || p == 128; }
inline int64_t cache_page_bytes(int fmt, int page_size) {
  return (int64_t)page_size * (fmt == MOE_CACHE_E4M3 ? kRow8Bytes : 2 * kRowDim);
}

// 2^(code - 127) as fp32; code 0 is 2^-127 (subnormal), code 255 (never written) is infinite.
__device__ __forceinline__ float ue8m0_value(uint32_t code) {
  return code == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(code << 23);
}

}  // namespace moe
