// Paged latent cache: tokens quantised (or copied) as they are written, contexts read back
// as contiguous rows for the expanded form of latent attention. Layout: latent.h.
//
//   write: s_b = 2^ceil(log2(amax_b / 448)) over each 128 latent values (1 for a zero block),
//          code = e4m3(x / s_b), nearest even: x / s_b is exact, so one rounding per value. Values
//          that would round up to 256 * 2^120 = 2^128, beyond fp32 and bf16 alike, take 240 * 2^120:
//          a finite value reads back finite (a larger s_b would not help, 255 has no nearer code).
//          amax_b counts finite values only; an infinity or NaN is stored as e4m3 NaN and
//          reads back as NaN without touching its block's other values. Rotary keys keep
//          their 16 bits (their products carry the position and are 1/9 of the row).
//   read:  code * s_b, exact.
//
// Both only move bytes, so they are bound by HBM at length and by launch latency for the few
// tokens of a decode step. One warp per token: a lane holds 16 consecutive latent values
// (32 bytes in, 16 bytes of codes out), so every access of the warp is one contiguous run of
// 512 or 1024 bytes, a scale block is 8 lanes, and its maximum takes three shuffles. A warp has one row in flight,
// and the read comes to it over cu_lens, the table and the page one after the other. Measured: a write of a prompt piece to
// e4m3 pages and the read of its context 21 us for 56.7 MB (4.7 and 11.9 us on the device, the rest the two calls);
// 29011 rows alone, the call included: e4m3 written in 22.9 us, read in 17.1 (2.3 and 3.0 TB/s), bf16 18.4 and 17.9
// (3.6 and 3.7); an append of a step's tokens 8.4 us, 2.2 of them on the device.
#include "latent.h"

#include <cuda_fp8.h>

namespace moe {
namespace {

constexpr int kCacheThreads = 256;
constexpr float kLargestBack = 0x1.Ep127f;  // 240 * 2^120, see write

template <typename T>
__device__ __forceinline__ void load16(const T* p, bool vec, uint32_t (&w)[8]) {
  if (vec) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(p)), b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = (uint32_t)__ldg(q + 2 * i) | ((uint32_t)__ldg(q + 2 * i + 1) << 16);
  }
}

// vec_lat / vec_rope: the source rows are 16-byte aligned (base and pitch); otherwise they
// are read element by element. Slots below zero are skipped; a slot past the cache records
// MOE_ERR_INVALID_ARG and is skipped.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(kCacheThreads)
latent_cache_write_kernel(const T* __restrict__ latent, int64_t ld_latent, bool vec_lat, const T* __restrict__ k_rope,
                          int64_t ld_rope, bool vec_rope, const int64_t* __restrict__ slots, int64_t n,
                          uint8_t* __restrict__ cache, int64_t num_slots, int page_size, int* status) {
  const int lane = threadIdx.x & 31;
  const int64_t i = ((int64_t)blockIdx.x * kCacheThreads + threadIdx.x) >> 5;
  if (i >= n) return;
  const int64_t slot = __ldg(slots + i);
  uint32_t w[8];
  load16(latent + i * ld_latent + lane * 16, vec_lat, w);
  uint32_t r = 0;  // two rotary values per lane
  const T* rp = k_rope + i * ld_rope + lane * 2;
  if (vec_rope) {
    r = __ldg(reinterpret_cast<const uint32_t*>(rp));
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(rp);
    r = (uint32_t)__ldg(q) | ((uint32_t)__ldg(q + 1) << 16);
  }
  if (slot < 0) return;
  if (slot >= num_slots) {
    if (lane == 0) record_status(status, MOE_ERR_INVALID_ARG);
    return;
  }
  if constexpr (!E4M3) {
    uint8_t* row = cache + slot * (int64_t)(2 * kRowDim);
    uint4* dst = reinterpret_cast<uint4*>(row + lane * 32);
    dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
    dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
    reinterpret_cast<uint32_t*>(row + 2 * kLatDim)[lane] = r;
  } else {
    const int64_t page = slot / page_size;
    const int off = (int)(slot - page * page_size);
    uint8_t* base = cache + page * ((int64_t)page_size * kRow8Bytes);
    float v[16];
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 f = ElemTraits<T>::unpack2(w[j]);
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float a = fabsf(v[j]);
      amax = fmaxf(amax, a < INFINITY ? a : 0.f);  // NaN and infinities left out
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float sc = fp8_block_scale(amax, true);
    uint32_t q[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const uint32_t c = fabsf(v[j]) < INFINITY
                             ? (uint32_t)__nv_cvt_float_to_fp8(fminf(fmaxf(v[j], -kLargestBack), kLargestBack) / sc,
                                                               __NV_SATFINITE, __NV_E4M3)
                             : 0x7Fu;
      q[j >> 2] |= c << (8 * (j & 3));
    }
    reinterpret_cast<uint4*>(base + (int64_t)off * kLatDim)[lane] = make_uint4(q[0], q[1], q[2], q[3]);
    reinterpret_cast<uint32_t*>(base + (int64_t)page_size * kLatDim + off * (2 * kRopeDim))[lane] = r;
    const uint32_t code = __float_as_uint(sc) >> 23;
    uint32_t word = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) word |= __shfl_sync(0xffffffffu, code, 8 * b) << (8 * b);
    if (lane == 0)
      reinterpret_cast<uint32_t*>(base + (int64_t)page_size * (kLatDim + 2 * kRopeDim))[off] = word;
  }
}

// Row i of the output is position i - cu_lens[b] of request b, cu_lens[b] <= i < cu_lens[b + 1];
// rows before cu_lens[0] and past cu_lens[num_seqs] are zeros. A table entry outside the cache, or a position past
// the table, records MOE_ERR_INVALID_ARG and reads as NaN.
template <bool E4M3>
__global__ void __launch_bounds__(kCacheThreads)
latent_cache_read_kernel(const uint8_t* __restrict__ cache, int64_t num_pages, int page_size,
                         const int32_t* __restrict__ table, int64_t ld_table, int table_width,
                         const int32_t* __restrict__ cu_lens, int num_seqs, int64_t total, uint32_t nan_word,
                         uint16_t* __restrict__ latent, uint16_t* __restrict__ k_rope, int* status) {
  const int lane = threadIdx.x & 31;
  const int64_t i = ((int64_t)blockIdx.x * kCacheThreads + threadIdx.x) >> 5;
  if (i >= total) return;
  int lo = 0, hi = num_seqs;  // the request holding row i: the last b with cu_lens[b] <= i
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int64_t)__ldg(cu_lens + mid) <= i) lo = mid; else hi = mid - 1;
  }
  uint4* dst = reinterpret_cast<uint4*>(latent + i * kLatDim) + lane * 2;
  uint32_t* rdst = reinterpret_cast<uint32_t*>(k_rope + i * kRopeDim) + lane;
  if (lo >= num_seqs || (int64_t)__ldg(cu_lens + lo) > i) {  // no request's row
    dst[0] = dst[1] = make_uint4(0u, 0u, 0u, 0u);
    *rdst = 0u;
    return;
  }
  const int64_t pos = i - __ldg(cu_lens + lo);
  const int64_t pi = pos / page_size;
  const int off = (int)(pos - pi * page_size);
  const int64_t page = pi < table_width ? (int64_t)__ldg(table + lo * ld_table + pi) : -1;
  if (page < 0 || page >= num_pages) {
    if (lane == 0) record_status(status, MOE_ERR_INVALID_ARG);
    dst[0] = dst[1] = make_uint4(nan_word, nan_word, nan_word, nan_word);
    *rdst = nan_word;
    return;
  }
  if constexpr (!E4M3) {
    const uint8_t* row = cache + (page * page_size + off) * (int64_t)(2 * kRowDim);
    const uint4* src = reinterpret_cast<const uint4*>(row + lane * 32);
    const uint4 a = __ldg(src), b = __ldg(src + 1);
    const uint32_t r = __ldg(reinterpret_cast<const uint32_t*>(row + 2 * kLatDim) + lane);
    dst[0] = a;
    dst[1] = b;
    *rdst = r;
  } else {
    const uint8_t* base = cache + page * ((int64_t)page_size * kRow8Bytes);
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(base + (int64_t)off * kLatDim) + lane);
    const uint32_t r =
        __ldg(reinterpret_cast<const uint32_t*>(base + (int64_t)page_size * kLatDim + off * (2 * kRopeDim)) + lane);
    const float sc = ue8m0_value(
        __ldg(base + (int64_t)page_size * (kLatDim + 2 * kRopeDim) + off * (kLatDim / kLatBlk) + (lane >> 3)));
    const uint32_t c[4] = {q.x, q.y, q.z, q.w};
    uint32_t o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c[j >> 1] >> (16 * (j & 1))), __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      o[j] = ElemTraits<__nv_bfloat16>::pack2(f.x * sc, f.y * sc);
    }
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
    *rdst = r;
  }
}

}  // namespace
}  // namespace moe

extern "C" int64_t moe_latent_cache_page_bytes(int cache_fmt, int page_size) {
  if (!moe::cache_fmt_ok(cache_fmt) || !moe::page_size_ok(page_size)) return -1;
  return moe::cache_page_bytes(cache_fmt, page_size);
}

extern "C" int moe_latent_cache_write(int dtype, const void* latent, int64_t ld_latent, const void* k_rope,
                                      int64_t ld_rope, const int64_t* slots, int64_t num_tokens, int cache_fmt,
                                      void* cache, int64_t num_pages, int page_size, int* status, void* stream) {
  using namespace moe;
  if (!cache_fmt_ok(cache_fmt) || (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_FP16)) return MOE_ERR_UNSUPPORTED;
  // e4m3 pages keep the rotary keys as bf16
  if (cache_fmt == MOE_CACHE_E4M3 ? dtype != MOE_DTYPE_BF16 : dtype != cache_fmt) return MOE_ERR_UNSUPPORTED;
  if (num_tokens < 0 || num_pages < 0) return MOE_ERR_INVALID_ARG;
  if (!page_size_ok(page_size) || num_pages > INT32_MAX || num_tokens > (int64_t)INT32_MAX) return MOE_ERR_BAD_SHAPE;
  if (num_tokens == 0) return MOE_OK;
  if (!latent || !k_rope || !slots || !cache || ld_latent < 0 || ld_rope < 0) return MOE_ERR_INVALID_ARG;
  if (!aligned16(cache) || (reinterpret_cast<uintptr_t>(latent) & 1u) || (reinterpret_cast<uintptr_t>(k_rope) & 1u) ||
      (reinterpret_cast<uintptr_t>(slots) & 7u))
    return MOE_ERR_INVALID_ARG;
  const int rc = moe_check_device();
  if (rc != MOE_OK) return rc;
  const bool vl = aligned16(latent) && ld_latent % 8 == 0;
  const bool vr = (reinterpret_cast<uintptr_t>(k_rope) & 3u) == 0 && ld_rope % 2 == 0;
  const unsigned blocks = (unsigned)ceil_div(num_tokens * 32, kCacheThreads);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* c = static_cast<uint8_t*>(cache);
  const int64_t ns = num_pages * page_size;
  if (cache_fmt == MOE_CACHE_E4M3)
    latent_cache_write_kernel<__nv_bfloat16, true><<<blocks, kCacheThreads, 0, st>>>(
        static_cast<const __nv_bfloat16*>(latent), ld_latent, vl, static_cast<const __nv_bfloat16*>(k_rope), ld_rope,
        vr, slots, num_tokens, c, ns, page_size, status);
  else  // a 16-bit copy is the same for both types
    latent_cache_write_kernel<__nv_bfloat16, false><<<blocks, kCacheThreads, 0, st>>>(
        static_cast<const __nv_bfloat16*>(latent), ld_latent, vl, static_cast<const __nv_bfloat16*>(k_rope), ld_rope,
        vr, slots, num_tokens, c, ns, page_size, status);
  return cudaGetLastError() == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}

extern "C" int moe_latent_cache_read(int cache_fmt, const void* cache, int64_t num_pages, int page_size,
                                     const int32_t* block_table, int64_t ld_table, int table_width,
                                     const int32_t* cu_lens, int num_seqs, int64_t total, void* latent, void* k_rope,
                                     int* status, void* stream) {
  using namespace moe;
  if (!cache_fmt_ok(cache_fmt)) return MOE_ERR_UNSUPPORTED;
  if (num_pages < 0 || num_seqs < 0 || total < 0 || table_width < 0 || ld_table < 0) return MOE_ERR_INVALID_ARG;
  if (!page_size_ok(page_size) || num_pages > INT32_MAX || total > (int64_t)INT32_MAX) return MOE_ERR_BAD_SHAPE;
  if (total == 0) return MOE_OK;
  if (!cache || !cu_lens || !latent || !k_rope || (num_seqs > 0 && table_width > 0 && !block_table))
    return MOE_ERR_INVALID_ARG;
  if (!aligned16(cache) || !aligned16(latent) || !aligned16(k_rope)) return MOE_ERR_INVALID_ARG;
  const int rc = moe_check_device();
  if (rc != MOE_OK) return rc;
  const unsigned blocks = (unsigned)ceil_div(total * 32, kCacheThreads);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const uint8_t* c = static_cast<const uint8_t*>(cache);
  const uint32_t nan_word = cache_fmt == MOE_DTYPE_FP16 ? 0x7E007E00u : 0x7FC07FC0u;
  if (cache_fmt == MOE_CACHE_E4M3)
    latent_cache_read_kernel<true><<<blocks, kCacheThreads, 0, st>>>(
        c, num_pages, page_size, block_table, ld_table, table_width, cu_lens, num_seqs, total, nan_word,
        static_cast<uint16_t*>(latent), static_cast<uint16_t*>(k_rope), status);
  else
    latent_cache_read_kernel<false><<<blocks, kCacheThreads, 0, st>>>(
        c, num_pages, page_size, block_table, ld_table, table_width, cu_lens, num_seqs, total, nan_word,
        static_cast<uint16_t*>(latent), static_cast<uint16_t*>(k_rope), status);
  return cudaGetLastError() == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}
