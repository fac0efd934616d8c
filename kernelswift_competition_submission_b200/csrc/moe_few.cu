// A whole MoE layer for a few tokens (decode): routing, gate/up products with SiLU * mul, down
// products and the weighted sum over the chosen experts, in two kernels.
//
//   a_p   = silu(W1g[e] x_t) * (W1u[e] x_t)      p = (t, e), e one of token t's topk experts
//   out_t = sum_e w_te W2[e] a_te
//
// With a few tokens every chosen expert's weights are read for one or a handful of rows, so
// the layer is bound by the bytes of the hit experts (3 * K * N each). They are read once per 8
// pairs of an expert: with more than 8 tokens on one, again for the next 8. The weights go from
// global memory straight into the registers of mma.sync.m16n8k16 as its A operand (16 weight
// rows x 16 k), the tokens are its 8 columns: no shared memory, no barrier and no token tile
// to fill on that way; a tcgen05 tile would pad 1..8 tokens to a 128-row operand and stage
// every weight byte through shared memory for the same bytes.
//
// The k order inside an MMA is free as long as both operands agree, so a lane takes two 16-byte
// pieces of its row per 128-byte block, 64 bytes apart, and feeds them to 8 (e4m3) or 4 (16-bit)
// MMAs in the order they lie: the four lanes of a row read 64 bytes in a row at a time, whole 32-byte
// sectors (32 consecutive bytes per lane asked for every sector twice). e4m3 codes become fp16 pairs with
// the conversion instruction (moving their bits to bf16 by shifts and masks instead kept the
// integer pipe busier than HBM: 0.53 against 0.58 of its rate in few_up at one token, 0.53 against
// 0.64 in few_down at eight), so bf16 tokens and bf16 a_p rows become fp16 too, each row under
// the power of two that brings its largest magnitude to 2^14 .. 2^15: what lies below 2^-39 of
// that maximum is lost, far under the bf16 rounding of the same row.
//
// few_up:   items of 8 columns of N for a chunk of up to 8 pairs of one expert: rows 0-7 of the A
//           operand are gate rows, rows 8-15 the same up rows, so a lane holds both halves of its
//           SiLU * mul. Every CTA routes all tokens itself (a warp per token), takes an equal run
//           of the items and gives each of its warps an equal run of their k blocks, whatever
//           the number of items; items cut between warps are joined in shared memory in order.
// few_down: one CTA per 16 rows of the output; its warps take consecutive runs of the (chunk, k
//           block) list, add weight * product into their own shared rows in fp32, and the rows are
//           summed in warp order.
// Measured, of the bytes of the hit experts at HBM's 6.55 TB/s: e4m3, E 256, K 7168, N 2048: one token 91 us
// (0.59: 65 up, 31 down, 1.3 to zero the maxima), 11 tokens 710-730 us (0.70-0.72); bf16, E 8, K 4096, N 14336, 6 tokens
// 431-458 us (0.82-0.85). The warps wait for their loads: issue slots are 20 to 38 % busy, the integer pipe 18 to 34 %
// with e4m3 weights. At 11 tokens (E 256) and 8 (E 8) moe_grouped_topk and moe_fused_experts(_fp8) have become faster, at
// 32 tokens 1390 against 1670 us and 516 against 798; at E 64, K 2048, N 1408 they have not at 32 tokens (237 against 216).
// Both give the same bits on every run. Sums are fp32; a_p is rounded once to the tokens' type (the
// layer's other paths do the same).
#include "common.cuh"
#include "moe_internal.h"
#include "routing.cuh"

#include <cuda_fp8.h>

#include <algorithm>

namespace moe {
namespace {

constexpr int kFewMaxTokens = 32;
constexpr int kFewMaxPairs = 512;
constexpr int kFewCols = 8;          // pairs per chunk: the MMA's columns
constexpr int kUpWarps = 12;
constexpr size_t kUpMaxSmem = 160 * 1024;  // with the tokens' fp16 copies, see launch_few
constexpr int kBlkBytes = 128;       // weight bytes of a row per k block

// Written by few_up's first CTA for few_down.
struct FewTables {
  int32_t n_chunks;
  int32_t bad[kFewMaxTokens];                      // token without a valid routing (NaN logits)
  int32_t chunk_expert[kFewMaxPairs];
  int16_t chunk_pair[kFewMaxPairs][kFewCols];      // pair t * topk + slot, -1 for an empty column
  float weight[kFewMaxPairs];                      // by pair
  uint32_t amax[kFewMaxPairs];                     // by pair: largest |a| as float bits (e4m3 weights, bf16 tokens)
};

struct FewRouting {
  const float* logits;
  const float* bias;
  int topk, renormalize, n_group, topk_group, scoring, gmode;
  float scale;
  bool aligned;  // logits and bias on 16 bytes
};

__device__ __forceinline__ uint4 ldg_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                 uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two e4m3 codes (the low half of w) as an fp16 pair; NaN codes stay NaN.
__device__ __forceinline__ uint32_t widen2(uint32_t w) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w, __NV_E4M3);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The power of two that brings a largest magnitude (as float bits) into [2^14, 2^15); 1 for a row of
// zeros and for one that holds infinities or NaN.
__device__ __forceinline__ float row_scale(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23);
  return e == 0 || e == 255 ? 1.0f : __int_as_float(min(max(127 + 14 - (e - 127), 1), 254) << 23);
}

// The tokens' side of one k block: this lane's 32 or 16 values of its column, zeros without one.
// With e4m3 weights the values are wanted in fp16: bf16 ones are scaled and converted.
template <typename T, bool F8>
__device__ __forceinline__ void load_col(const T* p, float scale, uint32_t (&x)[F8 ? 16 : 8]) {
  constexpr int kPart = F8 ? 2 : 1;  // 16-byte pieces that belong to 16 bytes of weights
#pragma unroll
  for (int i = 0; i < 2 * kPart; ++i) {
    const uint4 v = p ? *reinterpret_cast<const uint4*>(p + (i / kPart) * (F8 ? 64 : 32) + (i % kPart) * 8)
                      : make_uint4(0u, 0u, 0u, 0u);
    x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
  }
  if constexpr (F8 && ElemTraits<T>::kFmt == 1) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float lo = __uint_as_float(x[i] << 16) * scale, hi = __uint_as_float(x[i] & 0xFFFF0000u) * scale;
      x[i] = ElemTraits<__half>::pack2(lo, hi);
    }
  }
}

// One 128-byte k block: rows lo (A rows 0-7) and hi (A rows 8-15), two 16-byte pieces each per lane.
template <typename T, bool F8>
__device__ __forceinline__ void block_mma(float (&c)[4], const uint4 (&lo)[2], const uint4 (&hi)[2],
                                          const uint32_t (&x)[F8 ? 16 : 8]) {
  const uint32_t l[8] = {lo[0].x, lo[0].y, lo[0].z, lo[0].w, lo[1].x, lo[1].y, lo[1].z, lo[1].w};
  const uint32_t h[8] = {hi[0].x, hi[0].y, hi[0].z, hi[0].w, hi[1].x, hi[1].y, hi[1].z, hi[1].w};
  if constexpr (F8) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      mma16816<__half>(c, widen2(l[i] & 0xFFFFu), widen2(h[i] & 0xFFFFu), widen2(l[i] >> 16), widen2(h[i] >> 16),
                       x[2 * i], x[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) mma16816<T>(c, l[2 * i], h[2 * i], l[2 * i + 1], h[2 * i + 1], x[2 * i], x[2 * i + 1]);
  }
}

// The same from tokens already in fp16.
__device__ __forceinline__ void load_col16(const __half* p, uint32_t (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 v = p ? *reinterpret_cast<const uint4*>(p + (i / 2) * 64 + (i % 2) * 8) : make_uint4(0u, 0u, 0u, 0u);
    x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
  }
}

// The routing of one token by one warp, as moe_grouped_topk does it.
__device__ __forceinline__ void route_one(const FewRouting& r, int tok, int E, float* w, int32_t* ids,
                                          float* s_choice, RouteScratch* scr) {
  const float* row = r.logits + (int64_t)tok * E;
  const bool grouped = r.topk_group < r.n_group;
  // 256 experts, without groups or in groups of 64 or 32: the register-only rule (1 us less per token)
  if (E == 256 && r.aligned && (!grouped || r.n_group == 4 || r.n_group == 8)) {
#define MOE_ROUTE(LPG)                                                                                             \
  route_token_lanes<8, LPG, false>(row, r.bias, tok, r.topk, r.renormalize, r.n_group, r.topk_group, r.scoring, r.gmode, \
                                   r.scale, w, ids, scr)
    if (grouped && r.n_group == 8) MOE_ROUTE(4);
    else if (grouped) MOE_ROUTE(8);
    else MOE_ROUTE(1);
#undef MOE_ROUTE
  } else if (E <= 64) {
    route_token_general<2, false>(row, r.bias, tok, E, r.topk, r.renormalize, r.n_group, r.topk_group, r.scoring,
                                  r.gmode, r.scale, w, ids, s_choice);
  } else if (E <= 256) {
    route_token_general<8, false>(row, r.bias, tok, E, r.topk, r.renormalize, r.n_group, r.topk_group, r.scoring,
                                  r.gmode, r.scale, w, ids, s_choice);
  } else {
    route_token_general<16, false>(row, r.bias, tok, E, r.topk, r.renormalize, r.n_group, r.topk_group, r.scoring,
                                   r.gmode, r.scale, w, ids, s_choice);
  }
}

struct UpShared {
  RouteScratch scratch[kUpWarps];
  float choice[kUpWarps][kRouteMaxExperts];
  float weight[kFewMaxPairs];
  int32_t id[kFewMaxPairs];
  int32_t count[kRouteMaxExperts];   // pairs of an expert, then its first chunk
  int32_t chunk_expert[kFewMaxPairs];
  int16_t chunk_pair[kFewMaxPairs][kFewCols];
  float scale[kFewMaxTokens];        // by token, e4m3 weights and bf16 tokens
  uint32_t amax[kFewMaxTokens];
  int32_t n_chunks;
  alignas(16) float part[kUpWarps][2][32][4];  // a warp's sums of an item that it did not begin / did not end
};

template <typename T, bool F8>
__global__ void __launch_bounds__(32 * kUpWarps, 1)
few_up_kernel(const T* __restrict__ x, int64_t ld_x, FewRouting rt, const uint8_t* __restrict__ w1,
              const float* __restrict__ w1s, int M, int E, int K, int N, bool staged, T* __restrict__ act, FewTables* tab) {
  extern __shared__ __align__(16) uint8_t smem_up[];
  UpShared& s = *reinterpret_cast<UpShared*>(smem_up);
  constexpr bool kToHalf = F8 && ElemTraits<T>::kFmt == 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int P = M * rt.topk;
  // few tokens are converted once per CTA into shared memory (pitch: 16 bytes more than a row, so that the
  // lanes of two columns take different banks); more of them at every use
  __half* xh = reinterpret_cast<__half*>(smem_up + sizeof(UpShared));
  const int xh_ld = K + 8;
  if constexpr (kToHalf) {
    if (threadIdx.x < M) s.amax[threadIdx.x] = 0u;
    __syncthreads();
    for (int t = 0; t < M; ++t) {
      uint32_t m = 0;
      for (int i = threadIdx.x * 8; i < K; i += blockDim.x * 8) {
        const uint4 v = *reinterpret_cast<const uint4*>(x + (int64_t)t * ld_x + i);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) m = max(m, max(w[j] << 16 & 0x7FFF0000u, w[j] & 0x7FFF0000u));
      }
      m = __reduce_max_sync(0xffffffffu, m);
      if (lane == 0 && m) atomicMax(&s.amax[t], m);
    }
  }
  for (int t = warp; t < M; t += kUpWarps) {
    route_one(rt, t, E, s.weight, s.id, s.choice[warp], &s.scratch[warp]);
    __syncwarp();
  }
  for (int i = threadIdx.x; i < E; i += blockDim.x) s.count[i] = 0;
  for (int i = threadIdx.x; i < kFewMaxPairs * kFewCols / 2; i += blockDim.x)
    reinterpret_cast<uint32_t*>(s.chunk_pair)[i] = 0xFFFFFFFFu;
  __syncthreads();
  if constexpr (kToHalf) {
    if (threadIdx.x < M) s.scale[threadIdx.x] = row_scale(s.amax[threadIdx.x]);
    if (staged)
      for (int t = 0; t < M; ++t) {
        const float sc = row_scale(s.amax[t]);
        for (int i = threadIdx.x * 8; i < K; i += blockDim.x * 8) {
          const uint4 v = *reinterpret_cast<const uint4*>(x + (int64_t)t * ld_x + i);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
          uint32_t o[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            o[j] = ElemTraits<__half>::pack2(__uint_as_float(w[j] << 16) * sc, __uint_as_float(w[j] & 0xFFFF0000u) * sc);
          *reinterpret_cast<uint4*>(xh + t * xh_ld + i) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
  }
  for (int p = threadIdx.x; p < P; p += blockDim.x)
    if (s.id[p] >= 0 && s.id[p] < E) atomicAdd(&s.count[s.id[p]], 1);
  __syncthreads();
  if (warp == 0) {  // exclusive prefix of the experts' chunk counts
    int base = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int n = e0 + lane < E ? (s.count[e0 + lane] + kFewCols - 1) / kFewCols : 0;
      int inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (e0 + lane < E) s.count[e0 + lane] = base + inc - n;
      base += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) s.n_chunks = base;
  }
  __syncthreads();
  for (int p = threadIdx.x; p < P; p += blockDim.x) {
    const int e = s.id[p];
    if (e < 0 || e >= E) continue;
    int r = 0;  // place among the expert's pairs, in pair order
    for (int j = 0; j < p; ++j) r += s.id[j] == e ? 1 : 0;
    const int c = s.count[e] + r / kFewCols;
    s.chunk_expert[c] = e;
    s.chunk_pair[c][r % kFewCols] = (int16_t)p;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int p = threadIdx.x; p < P; p += blockDim.x) tab->weight[p] = s.weight[p];
    for (int i = threadIdx.x; i < s.n_chunks; i += blockDim.x) tab->chunk_expert[i] = s.chunk_expert[i];
    for (int i = threadIdx.x; i < s.n_chunks * kFewCols; i += blockDim.x)
      (&tab->chunk_pair[0][0])[i] = (&s.chunk_pair[0][0])[i];
    for (int t = threadIdx.x; t < M; t += blockDim.x) {
      int bad = 0;
      for (int j = 0; j < rt.topk; ++j) {
        const int e = s.id[t * rt.topk + j];
        bad |= (e < 0 || e >= E) ? 1 : 0;
      }
      tab->bad[t] = bad;
    }
    if (threadIdx.x == 0) tab->n_chunks = s.n_chunks;
  }

  constexpr int kElt = F8 ? 1 : 2;                // weight bytes per element
  constexpr int kBlkElts = kBlkBytes / kElt;      // elements of a k block
  constexpr int kColElts = kBlkElts / 8;          // of them in a lane's 16 bytes
  constexpr int kDepth = 4;                       // k blocks in flight per lane, asked for two at a time: DRAM
                                                  // serves 256 bytes of a row better than 128 (0.81 against 0.72)
  const int g = lane >> 2, t4 = lane & 3;
  const int nkb = K / kBlkElts;
  const int NB = N / 8;
  const int64_t items = (int64_t)s.n_chunks * NB;
  const int64_t row_bytes = (int64_t)K * kElt;
  const int64_t i0 = items * blockIdx.x / gridDim.x, i1 = items * (blockIdx.x + 1) / gridDim.x;
  const int blocks = (int)(i1 - i0) * nkb;
  auto begin_of = [&](int w) { return (int)((int64_t)blocks * w / kUpWarps); };
  const int b0 = begin_of(warp), b1 = begin_of(warp + 1);

  // item `it` (of this CTA): its gate row for this lane; the up row is N rows further on
  auto row_of = [&](int it) {
    const int64_t i = i0 + it;
    const int c = (int)(i / NB), n0 = (int)(i - (int64_t)c * NB) * 8;
    return w1 + ((int64_t)s.chunk_expert[c] * 2 * N + n0 + g) * row_bytes + t4 * 16;
  };
  const int64_t up = (int64_t)N * row_bytes;
  int l_it = b0 / nkb, l_k = b0 - l_it * nkb, left = b1 - b0;  // the next block to load
  const uint8_t* lp = left > 0 ? row_of(l_it) : nullptr;
  uint4 lo[kDepth][2], hi[kDepth][2];
  auto load = [&](int d) {
    const uint8_t* p = lp + (int64_t)l_k * kBlkBytes;
    lo[d][0] = ldg_stream(p);
    lo[d][1] = ldg_stream(p + 64);
    hi[d][0] = ldg_stream(p + up);
    hi[d][1] = ldg_stream(p + up + 64);
    --left;
    if (++l_k == nkb) {
      l_k = 0;
      ++l_it;
      if (left > 0) lp = row_of(l_it);
    }
  };
#pragma unroll
  for (int d = 0; d < kDepth; ++d)
    if (left > 0) load(d);

  int it = b0 / nkb, kb = b0 - it * nkb;
  bool begun = kb == 0;  // this warp has the item from its first block on
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  const T* xp = nullptr;
  const __half* hp = nullptr;
  float xs = 1.0f;
  const float* sg = nullptr;
  const float* su = nullptr;
  auto open_item = [&]() {
    const int64_t i = i0 + it;
    const int c = (int)(i / NB), n0 = (int)(i - (int64_t)c * NB) * 8;
    const int pair = s.chunk_pair[c][g];
    xp = pair >= 0 ? x + (int64_t)(pair / rt.topk) * ld_x + t4 * kColElts : nullptr;
    if constexpr (kToHalf) {
      xs = pair >= 0 ? s.scale[pair / rt.topk] : 1.0f;
      hp = pair >= 0 ? xh + (pair / rt.topk) * xh_ld + t4 * kColElts : nullptr;
    }
    if constexpr (F8) {
      sg = w1s + ((int64_t)s.chunk_expert[c] * (2 * N / 128) + n0 / 128) * (K / 128);
      su = sg + (int64_t)(N / 128) * (K / 128);
    }
  };
  // this lane: row n0 + g of gate (a 0, 1) and up (a 2, 3) for columns 2 t4, 2 t4 + 1
  auto finish = [&](int item, const float (&a)[4]) {
    const int64_t i = i0 + item;
    const int c = (int)(i / NB), n0 = (int)(i - (int64_t)c * NB) * 8;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int pj = s.chunk_pair[c][2 * t4 + j];
      float v = 0.f;
      if (pj >= 0) {
        const float r = kToHalf ? 1.0f / s.scale[pj / rt.topk] : 1.0f;  // a power of two
        const float gate = a[j] * r, upv = a[2 + j] * r;
        const T q = ElemTraits<T>::from_float(gate / (1.0f + expf(-gate)) * upv);
        act[(int64_t)pj * N + n0 + g] = q;
        v = fabsf((float)q);
      }
      if constexpr (kToHalf) {
        // the pair's largest magnitude over the item's 8 rows, then over all items; a maximum needs no order
        uint32_t m = __float_as_uint(v);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (g == 0 && pj >= 0) atomicMax(&tab->amax[pj], m);
      }
    }
  };
  if (b0 < b1) open_item();
  for (int b = b0; b < b1; b += kDepth) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      if (b + d < b1) {
        uint32_t xv[F8 ? 16 : 8];
        bool have = false;
        if constexpr (kToHalf) {
          if (staged) {
            load_col16(hp ? hp + kb * kBlkElts : nullptr, xv);
            have = true;
          }
        }
        if (!have) load_col<T, F8>(xp ? xp + (int64_t)kb * kBlkElts : nullptr, xs, xv);
        if constexpr (F8) {
          float part[4] = {0.f, 0.f, 0.f, 0.f};
          block_mma<T, F8>(part, lo[d], hi[d], xv);
          const float a = __ldg(sg + kb), u = __ldg(su + kb);
          acc[0] = fmaf(a, part[0], acc[0]);
          acc[1] = fmaf(a, part[1], acc[1]);
          acc[2] = fmaf(u, part[2], acc[2]);
          acc[3] = fmaf(u, part[3], acc[3]);
        } else {
          block_mma<T, F8>(acc, lo[d], hi[d], xv);
        }
        if (d & 1) {
          if (left > 0) load(d - 1);
          if (left > 0) load(d);
        }
        if (++kb == nkb) {
          if (begun) finish(it, acc);
          else *reinterpret_cast<float4*>(s.part[warp][0][lane]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j] = 0.f;
          kb = 0;
          ++it;
          begun = true;
          if (b + d + 1 < b1) open_item();
        }
      }
    }
  }
  if (b0 < b1 && kb != 0)
    *reinterpret_cast<float4*>(s.part[warp][begun ? 1 : 0][lane]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  if (b0 < b1 && kb != 0 && begun) {  // this warp began the item: it adds what the next ones have of it
    const int end = (it + 1) * nkb;
    for (int w = warp + 1; w < kUpWarps && begin_of(w) < end; ++w) {
      if (begin_of(w) == begin_of(w + 1)) continue;
      const float4 v = *reinterpret_cast<const float4*>(s.part[w][0][lane]);
      acc[0] += v.x;
      acc[1] += v.y;
      acc[2] += v.z;
      acc[3] += v.w;
    }
    finish(it, acc);
  }
}

template <typename T, bool F8, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, 16 / WARPS)
few_down_kernel(const T* __restrict__ act, const FewTables* __restrict__ tab, const uint8_t* __restrict__ w2,
                const float* __restrict__ w2s, int M, int topk, int K, int N, T* __restrict__ out) {
  extern __shared__ __align__(16) float s_part[];  // [warps][M][16]
  constexpr bool kToHalf = F8 && ElemTraits<T>::kFmt == 1;
  constexpr int kElt = F8 ? 1 : 2;
  constexpr int kBlkElts = kBlkBytes / kElt;
  constexpr int kColElts = kBlkElts / 8;
  constexpr int kDepth = 4;  // k blocks in flight per lane, asked for two at a time
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int h0 = blockIdx.x * 16;
  const int nkb = N / kBlkElts;
  const int64_t row_bytes = (int64_t)N * kElt;
  float* mine = s_part + warp * M * 16;
  for (int i = lane; i < M * 16; i += 32) mine[i] = 0.f;
  __syncwarp();
  const int total = tab->n_chunks * nkb;
  const int b0 = (int)((int64_t)total * warp / WARPS), b1 = (int)((int64_t)total * (warp + 1) / WARPS);

  int lc = b0 / nkb, lk = b0 - lc * nkb, left = b1 - b0;  // the next block to load
  auto row_of = [&](int c) { return w2 + ((int64_t)tab->chunk_expert[c] * K + h0 + g) * row_bytes + t4 * 16; };
  const uint8_t* lp = left > 0 ? row_of(lc) : nullptr;
  uint4 lo[kDepth][2], hi[kDepth][2];
  auto load = [&](int d) {
    const uint8_t* p = lp + (int64_t)lk * kBlkBytes;
    lo[d][0] = ldg_stream(p);
    lo[d][1] = ldg_stream(p + 64);
    hi[d][0] = ldg_stream(p + 8 * row_bytes);
    hi[d][1] = ldg_stream(p + 8 * row_bytes + 64);
    --left;
    if (++lk == nkb) {
      lk = 0;
      ++lc;
      if (left > 0) lp = row_of(lc);
    }
  };
#pragma unroll
  for (int d = 0; d < kDepth; ++d)
    if (left > 0) load(d);

  int c = b0 < b1 ? b0 / nkb : 0, kb = b0 < b1 ? b0 - c * nkb : 0;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  const T* xp = nullptr;
  float xs = 1.0f;
  const float* sp = nullptr;
  auto open_chunk = [&]() {
    const int pair = tab->chunk_pair[c][g];
    xp = pair >= 0 ? act + (int64_t)pair * N + t4 * kColElts : nullptr;
    if constexpr (kToHalf) xs = pair >= 0 ? row_scale(tab->amax[pair]) : 1.0f;
    if constexpr (F8) sp = w2s + ((int64_t)tab->chunk_expert[c] * (K / 128) + h0 / 128) * (N / 128);
  };
  auto close_chunk = [&]() {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int p = tab->chunk_pair[c][2 * t4 + j];
      if (p >= 0) {
        const float r = kToHalf ? 1.0f / row_scale(tab->amax[p]) : 1.0f;  // a power of two
        const float w = tab->weight[p];
        float* o = mine + (p / topk) * 16 + g;
        o[0] += w * (acc[j] * r);
        o[8] += w * (acc[2 + j] * r);
      }
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = 0.f;
  };
  if (b0 < b1) open_chunk();
  for (int b = b0; b < b1; b += kDepth) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      if (b + d < b1) {
        uint32_t xv[F8 ? 16 : 8];
        load_col<T, F8>(xp ? xp + (int64_t)kb * kBlkElts : nullptr, xs, xv);
        if constexpr (F8) {
          float part[4] = {0.f, 0.f, 0.f, 0.f};
          block_mma<T, F8>(part, lo[d], hi[d], xv);
          const float a = __ldg(sp + kb);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j] = fmaf(a, part[j], acc[j]);
        } else {
          block_mma<T, F8>(acc, lo[d], hi[d], xv);
        }
        if (d & 1) {
          if (left > 0) load(d - 1);
          if (left > 0) load(d);
        }
        if (++kb == nkb) {
          close_chunk();
          kb = 0;
          ++c;
          if (b + d + 1 < b1) open_chunk();
        }
      }
    }
  }
  if (b0 < b1 && kb != 0) close_chunk();
  __syncthreads();
  for (int i = threadIdx.x; i < M * 16; i += blockDim.x) {
    float v = 0.f;
    for (int w = 0; w < WARPS; ++w) v += s_part[w * M * 16 + i];
    const int t = i >> 4;
    if (tab->bad[t]) v = __int_as_float(0x7FC00000);
    out[(int64_t)t * K + h0 + (i & 15)] = ElemTraits<T>::from_float(v);
  }
}

inline size_t few_tables_bytes() { return (sizeof(FewTables) + 255) / 256 * 256; }
template <typename T, bool F8>
cudaError_t launch_few(const void* x, int64_t ld_x, const FewRouting& rt, const void* w1, const float* w1s,
                       const void* w2, const float* w2s, int M, int E, int K, int N, void* out, void* ws,
                       cudaStream_t st) {
  FewTables* tab = static_cast<FewTables*>(ws);
  T* act = reinterpret_cast<T*>(static_cast<uint8_t*>(ws) + few_tables_bytes());
  const size_t rows = (size_t)M * (size_t)(K + 8) * 2;
  // A few bf16 tokens become fp16 once per CTA, more of them as they are read. e4m3, E 256, K 7168, N 2048, us, once against
  // as read: 1 token 99/102, 2 169/174, 4 294/305, 6 425/428, but 8 600/551 and 9 664/612, where the copies leave little
  // of the SM's memory to L1; so up to 160 KB with the tables, 6 tokens of that width
  const bool staged = F8 && ElemTraits<T>::kFmt == 1 && sizeof(UpShared) + rows <= kUpMaxSmem;
  const size_t smem = sizeof(UpShared) + (staged ? rows : 0);
  cudaError_t err = ensure_smem_limit(reinterpret_cast<const void*>(few_up_kernel<T, F8>), (int)smem);
  if (err != cudaSuccess) return err;
  if (F8 && ElemTraits<T>::kFmt == 1) {
    err = cudaMemsetAsync(tab->amax, 0, sizeof(uint32_t) * (size_t)M * rt.topk, st);
    if (err != cudaSuccess) return err;
  }
  few_up_kernel<T, F8><<<num_sms(), 32 * kUpWarps, smem, st>>>(
      static_cast<const T*>(x), ld_x, rt, static_cast<const uint8_t*>(w1), w1s, M, E, K, N, staged, act, tab);
  if ((err = cudaGetLastError()) != cudaSuccess) return err;
  // about 16 warps per SM over all CTAs, so that few rows of output still ask for enough bytes at once. Measured
  // with 4, 8 and 16 warps, us: e4m3, K 7168, N 2048, 1 token 31, 34, 40, 11 tokens 245, 254, 269; bf16, K 4096,
  // N 14336, 6 tokens 225, 147, 155; bf16, K 2048, N 1408, 4 tokens of 6 experts 72, 41, 29, 1 token 21, 14, 11
  const int ctas = K / 16;
  const int warps = ctas * 6 > num_sms() * 16 ? 4 : ctas * 12 > num_sms() * 16 ? 8 : 16;
  auto kern = warps == 4 ? few_down_kernel<T, F8, 4> : warps == 8 ? few_down_kernel<T, F8, 8> : few_down_kernel<T, F8, 16>;
  kern<<<(unsigned)ctas, 32 * warps, (size_t)warps * M * 16 * 4, st>>>(act, tab, static_cast<const uint8_t*>(w2), w2s, M,
                                                                      rt.topk, K, N, static_cast<T*>(out));
  return cudaGetLastError();
}

}  // namespace
}  // namespace moe

extern "C" int moe_few_max_tokens(int topk) {
  if (topk <= 0) return 0;
  return moe::kFewMaxPairs / topk < moe::kFewMaxTokens ? moe::kFewMaxPairs / topk : moe::kFewMaxTokens;
}

extern "C" size_t moe_few_workspace_bytes(int64_t num_tokens, int topk, int intermediate_size) {
  if (num_tokens < 0 || topk <= 0 || intermediate_size <= 0) return 0;
  return moe::few_tables_bytes() + 2 * (size_t)num_tokens * (size_t)topk * (size_t)intermediate_size;
}

extern "C" int moe_few_tokens(int dtype, const void* hidden_states, int64_t ld_hidden, const float* gating_output,
                              const float* bias, int weight_e4m3, const void* w1, const float* w1_scale,
                              const void* w2, const float* w2_scale, int64_t num_tokens, int num_experts, int topk,
                              int renormalize, int num_expert_group, int topk_group, int scoring_func,
                              int group_score_mode, float routed_scaling_factor, int hidden_size,
                              int intermediate_size, void* out, void* workspace, size_t workspace_bytes,
                              void* stream) {
  using namespace moe;
  if (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_FP16) return MOE_ERR_UNSUPPORTED;
  if (num_tokens < 0 || num_experts <= 0 || topk <= 0 || num_expert_group <= 0 || topk_group <= 0 ||
      hidden_size <= 0 || intermediate_size <= 0)
    return MOE_ERR_INVALID_ARG;
  if (scoring_func != MOE_SCORING_SOFTMAX && scoring_func != MOE_SCORING_SIGMOID) return MOE_ERR_INVALID_ARG;
  if (group_score_mode != MOE_GROUP_SCORE_MAX && group_score_mode != MOE_GROUP_SCORE_TOP2_SUM)
    return MOE_ERR_INVALID_ARG;
  if (num_experts > kRouteMaxExperts || num_expert_group > 32 || topk > 32) return MOE_ERR_BAD_SHAPE;
  if (num_experts % num_expert_group != 0 || topk_group > num_expert_group) return MOE_ERR_BAD_SHAPE;
  const int epg = num_experts / num_expert_group;
  if (topk > topk_group * epg) return MOE_ERR_BAD_SHAPE;
  if (group_score_mode == MOE_GROUP_SCORE_TOP2_SUM && epg < 2) return MOE_ERR_BAD_SHAPE;
  const int gran = weight_e4m3 ? 128 : 64;
  if (hidden_size % gran || intermediate_size % gran || num_tokens > moe_few_max_tokens(topk)) return MOE_ERR_BAD_SHAPE;
  if (num_tokens == 0) return MOE_OK;
  if (!hidden_states || !gating_output || !w1 || !w2 || !out || !workspace || (weight_e4m3 && (!w1_scale || !w2_scale)))
    return MOE_ERR_INVALID_ARG;
  if (!aligned16(hidden_states) || ld_hidden % 8 || ld_hidden < 0 || !aligned16(w1) || !aligned16(w2) || !aligned16(workspace))
    return MOE_ERR_INVALID_ARG;
  if (workspace_bytes < moe_few_workspace_bytes(num_tokens, topk, intermediate_size)) return MOE_ERR_WORKSPACE;
  const int rc = moe_check_device();
  if (rc != MOE_OK) return rc;
  const FewRouting rt{gating_output, bias,         topk,           renormalize, num_expert_group, topk_group,
                      scoring_func,  group_score_mode, routed_scaling_factor,
                      aligned16(gating_output) && (!bias || aligned16(bias))};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int M = (int)num_tokens;
  cudaError_t err;
#define MOE_FEW(T, F8) \
  launch_few<T, F8>(hidden_states, ld_hidden, rt, w1, w1_scale, w2, w2_scale, M, num_experts, hidden_size, \
                    intermediate_size, out, workspace, st)
  if (dtype == MOE_DTYPE_BF16) err = weight_e4m3 ? MOE_FEW(__nv_bfloat16, true) : MOE_FEW(__nv_bfloat16, false);
  else err = weight_e4m3 ? MOE_FEW(__half, true) : MOE_FEW(__half, false);
#undef MOE_FEW
  return err == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}
