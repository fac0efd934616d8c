// Latent attention by rows: one warp per query row, keys one after the other with a running
// maximum and sum, fp32 throughout.
//
//   s_j = scale * q . k_j,  m' = max(m, s_j),  l' = l e^(m - m') + e^(s_j - m'),
//   o' = o e^(m - m') + e^(s_j - m') v_j;  result o / l and m + ln l; a row that sees no key
//   gives zeros and -inf.
// Only visible keys are read, so nothing a masked place holds can reach a result.
#include "latent.h"

#include <cuda_fp8.h>

namespace moe {
namespace {

constexpr int kRowsPerBlock = 4;

// One online-softmax step over a key whose score is s; acc holds this lane's output values.
template <int N>
__device__ __forceinline__ void online_step(float s, const float (&v)[N], float& m, float& l, float (&acc)[N]) {
  const float mn = fmaxf(m, s);
  const float base = mn == -INFINITY ? 0.f : mn;
  const float a = expf(m - base), p = expf(s - base);
  m = mn;
  l = l * a + p;
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = acc[i] * a + p * v[i];
}

// q [B, n_q, H, 576] -> out [B, n_q, H, 512], lse [B, n_q, H]. Lane l holds the elements
// 2 l, 2 l + 1 of every 64.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(32 * kRowsPerBlock)
latent_decode_rows_kernel(const T* __restrict__ q, const uint8_t* __restrict__ cache, int64_t num_pages, int page_size,
                          const int32_t* __restrict__ table, int64_t ld_table, int table_width,
                          const int32_t* __restrict__ lens, int64_t rows, int n_q, int heads, float scale,
                          T* __restrict__ out, float* __restrict__ lse, int* status) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int64_t b = row / ((int64_t)n_q * heads);
  const int s_i = (int)(row / heads % n_q);
  float qv[18];
#pragma unroll
  for (int i = 0; i < 9; ++i) {
    const float2 f = ElemTraits<T>::unpack2(__ldg(reinterpret_cast<const uint32_t*>(q + row * kRowDim) + 32 * i + lane));
    qv[2 * i] = f.x;
    qv[2 * i + 1] = f.y;
  }
  const int64_t cap = (int64_t)table_width * page_size;
  int64_t len = __ldg(lens + b);
  if (len > cap || len < 0) {
    if (lane == 0) record_status(status, MOE_ERR_INVALID_ARG);
    len = len < 0 ? 0 : cap;
  }
  const int64_t seen = len - n_q + 1 + s_i;
  float m = -INFINITY, l = 0.f, acc[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  for (int64_t j = 0; j < seen; ++j) {
    const int64_t page = __ldg(table + b * ld_table + j / page_size);
    const int off = (int)(j % page_size);
    if (page < 0 || page >= num_pages) {
      if (lane == 0) record_status(status, MOE_ERR_INVALID_ARG);
      continue;
    }
    float k[18];
    if constexpr (E4M3) {
      const uint8_t* base = cache + page * ((int64_t)page_size * kRow8Bytes);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint16_t c =
            __ldg(reinterpret_cast<const uint16_t*>(base + (int64_t)off * kLatDim + 64 * i) + lane);
        const float sc =
            ue8m0_value(__ldg(base + (int64_t)page_size * (kLatDim + 2 * kRopeDim) + off * 4 + (i >> 1)));
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)c, __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        k[2 * i] = f.x * sc;
        k[2 * i + 1] = f.y * sc;
      }
      const float2 f = ElemTraits<T>::unpack2(
          __ldg(reinterpret_cast<const uint32_t*>(base + (int64_t)page_size * kLatDim + off * (2 * kRopeDim)) + lane));
      k[16] = f.x;
      k[17] = f.y;
    } else {
      const uint32_t* src = reinterpret_cast<const uint32_t*>(cache + (page * page_size + off) * (int64_t)(2 * kRowDim));
#pragma unroll
      for (int i = 0; i < 9; ++i) {
        const float2 f = ElemTraits<T>::unpack2(__ldg(src + 32 * i + lane));
        k[2 * i] = f.x;
        k[2 * i + 1] = f.y;
      }
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 18; ++i) s = fmaf(qv[i], k[i], s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = k[i];
    online_step(s * scale, v, m, l, acc);
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    reinterpret_cast<uint32_t*>(out + row * kLatDim)[32 * i + lane] =
        ElemTraits<T>::pack2(acc[2 * i] * inv, acc[2 * i + 1] * inv);
  if (lse != nullptr && lane == 0) lse[row] = l > 0.f || l != l ? m + logf(l) : -INFINITY;
}

inline bool al(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace
}  // namespace moe

extern "C" int moe_latent_decode(int dtype, const void* q, int64_t num_seqs, int q_len, int heads, int cache_fmt,
                                 const void* cache, int64_t num_pages, int page_size, const int32_t* block_table,
                                 int64_t ld_table, int table_width, const int32_t* cache_lens, float scale, void* out,
                                 float* lse, void* workspace, size_t workspace_bytes, int* status, void* stream) {
  using namespace moe;
  if (!cache_fmt_ok(cache_fmt) || (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_FP16)) return MOE_ERR_UNSUPPORTED;
  if (cache_fmt == MOE_CACHE_E4M3 ? dtype != MOE_DTYPE_BF16 : dtype != cache_fmt) return MOE_ERR_UNSUPPORTED;
  if (num_seqs < 0 || q_len <= 0 || heads <= 0 || num_pages < 0 || table_width < 0 || ld_table < 0)
    return MOE_ERR_INVALID_ARG;
  if (!page_size_ok(page_size) || num_pages > INT32_MAX || (int64_t)q_len * heads > 65536 ||
      num_seqs > 65535 || (int64_t)table_width * page_size > INT32_MAX)
    return MOE_ERR_BAD_SHAPE;
  if (num_seqs == 0) return MOE_OK;
  if (num_pages == 0) return MOE_ERR_INVALID_ARG;
  if (!q || !cache || !cache_lens || !out || (table_width > 0 && !block_table)) return MOE_ERR_INVALID_ARG;
  if (!al(q, 16) || !al(cache, 16) || !al(out, 16)) return MOE_ERR_INVALID_ARG;
  const size_t need = moe_latent_decode_workspace_bytes(num_seqs, q_len, heads);
  if (workspace_bytes < need || (need > 0 && (!workspace || !al(workspace, 16)))) return MOE_ERR_WORKSPACE;
  const int rc = moe_check_device();
  if (rc != MOE_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t rows = num_seqs * q_len * heads;
  const unsigned blocks = (unsigned)ceil_div(rows, kRowsPerBlock);
  const uint8_t* c = static_cast<const uint8_t*>(cache);
#define MOE_LD(T, F8)                                                                                        \
  latent_decode_rows_kernel<T, F8><<<blocks, 32 * kRowsPerBlock, 0, st>>>(                                   \
      static_cast<const T*>(q), c, num_pages, page_size, block_table, ld_table, table_width, cache_lens, rows, q_len, \
      heads, scale, static_cast<T*>(out), lse, status)
  if (cache_fmt == MOE_CACHE_E4M3) {
    MOE_LD(__nv_bfloat16, true);
  } else {
    const cudaError_t e = launch_latent_decode16(dtype, q, (int)num_seqs, q_len, heads, cache, num_pages, page_size,
                                                 block_table, ld_table, table_width, cache_lens, scale, out, lse,
                                                 workspace, status, st);
    return e == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
  }
#undef MOE_LD
  return cudaGetLastError() == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}
