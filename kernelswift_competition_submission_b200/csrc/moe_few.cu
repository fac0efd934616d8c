// A whole MoE layer for a few tokens (decode): routing, gate/up products with SiLU * mul, down
// products and the weighted sum over the chosen experts, in two kernels.
//
//   a_p   = silu(W1g[e] x_t) * (W1u[e] x_t)      p = (t, e), e one of token t's topk experts
//   out_t = sum_e w_te W2[e] a_te
//
// With a few tokens every chosen expert's weights are read for one or a handful of rows, so
// the layer is bound by the bytes of the hit experts (3 * K * N each). The weights go from
// global memory straight into the registers of mma.sync.m16n8k16 as its A operand (16 weight
// rows x 16 k), the tokens are its 8 columns: no shared memory, no barrier and no token tile
// to fill on that way; a tcgen05 tile would pad 1..8 tokens to a 128-row operand and stage
// every weight byte through shared memory for the same bytes.
//
// The k order inside an MMA is free as long as both operands agree, so a lane takes 32
// consecutive bytes of its row per 128-byte block (four lanes read one full line) and feeds
// them to 8 (e4m3) or 4 (16-bit) MMAs in the order they lie. e4m3 codes become 16-bit floats
// by moving their bits: the code's exponent and fraction land in the low end of the wider
// exponent field, which is the value times 2^-120 (bf16) or 2^-8 (fp16) exactly, subnormals
// included; the power goes back exactly in a bf16 multiply, or for fp16 in the block scale.
//
// few_up:   one warp per item (chunk of up to 8 pairs of one expert, 8 columns of N): rows 0-7
//           of the A operand are gate rows, rows 8-15 the same up rows, so a lane holds both
//           halves of its SiLU * mul. Every CTA routes all tokens itself (a warp per token).
// few_down: one CTA per 16 rows of the output; its warps take consecutive runs of the
//           (chunk, k block) list, add weight * product into their own shared rows in fp32,
//           and the rows are summed in warp order: the same bits on every run.
// Sums are fp32; a_p is rounded once to the tokens' type (the layer's other paths do the same).
#include "common.cuh"
#include "moe_internal.h"
#include "routing.cuh"

namespace moe {
namespace {

constexpr int kFewMaxTokens = 32;
constexpr int kFewMaxPairs = 512;
constexpr int kFewCols = 8;          // pairs per chunk: the MMA's columns
constexpr int kUpWarps = 16;
constexpr int kDownWarps = 8;
constexpr int kBlkBytes = 128;       // weight bytes of a row per k block

// Written by few_up's first CTA for few_down.
struct FewTables {
  int32_t n_chunks;
  int32_t bad[kFewMaxTokens];                      // token without a valid routing (NaN logits)
  int32_t chunk_expert[kFewMaxPairs];
  int16_t chunk_pair[kFewMaxPairs][kFewCols];      // pair t * topk + slot, -1 for an empty column
  float weight[kFewMaxPairs];                      // by pair
};

struct FewRouting {
  const float* logits;
  const float* bias;
  int topk, renormalize, n_group, topk_group, scoring, gmode;
  float scale;
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

// Four e4m3 codes -> (codes 0, 2) and (codes 1, 3) as pairs of T. The bit move would turn e4m3
// NaN into 480, so block_mma notes NaN codes per row and the row's results become NaN.
template <typename T> struct Expand8;
template <> struct Expand8<__nv_bfloat16> {
  static constexpr float kScale = 1.0f;
  __device__ static __forceinline__ uint32_t lift(uint32_t w) {  // codes in the high byte of each half
    const uint32_t b = (w & 0x80008000u) | ((w >> 4) & 0x07F007F0u);
    uint32_t r;  // * 2^120
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(b), "r"(0x7B807B80u));
    return r;
  }
};
template <> struct Expand8<__half> {
  static constexpr float kScale = 256.0f;  // joins the block scale
  __device__ static __forceinline__ uint32_t lift(uint32_t w) { return (w & 0x80008000u) | ((w >> 1) & 0x3F803F80u); }
};

// The tokens' side of one k block: 32 or 16 consecutive values of this lane's column.
template <int WORDS>
__device__ __forceinline__ void load_col(const uint8_t* p, uint32_t (&x)[WORDS]) {
#pragma unroll
  for (int i = 0; i < WORDS / 4; ++i) {
    const uint4 v = p ? *reinterpret_cast<const uint4*>(p + 16 * i) : make_uint4(0u, 0u, 0u, 0u);
    x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
  }
}

// One 128-byte k block: rows lo (A rows 0-7) and hi (A rows 8-15), 32 bytes each per lane.
template <typename T, bool F8>
__device__ __forceinline__ void block_mma(float (&c)[4], const uint4 (&lo)[2], const uint4 (&hi)[2],
                                          const uint32_t (&x)[F8 ? 16 : 8], uint32_t& nan_lo, uint32_t& nan_hi) {
  const uint32_t l[8] = {lo[0].x, lo[0].y, lo[0].z, lo[0].w, lo[1].x, lo[1].y, lo[1].z, lo[1].w};
  const uint32_t h[8] = {hi[0].x, hi[0].y, hi[0].z, hi[0].w, hi[1].x, hi[1].y, hi[1].z, hi[1].w};
  if constexpr (F8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      nan_lo |= (l[i] & 0x7F7F7F7Fu) + 0x01010101u;  // bit 7 of a byte: the code was NaN
      nan_hi |= (h[i] & 0x7F7F7F7Fu) + 0x01010101u;
      const uint32_t b0 = __byte_perm(x[2 * i], x[2 * i + 1], 0x5410);  // values 0, 2 of the four
      const uint32_t b1 = __byte_perm(x[2 * i], x[2 * i + 1], 0x7632);  // values 1, 3
      mma16816<T>(c, Expand8<T>::lift(l[i] << 8), Expand8<T>::lift(h[i] << 8), Expand8<T>::lift(l[i]),
                  Expand8<T>::lift(h[i]), b0, b1);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) mma16816<T>(c, l[2 * i], h[2 * i], l[2 * i + 1], h[2 * i + 1], x[2 * i], x[2 * i + 1]);
  }
}

// The quad's four lanes hold one row's k values: a NaN code in any of them makes the row NaN.
__device__ __forceinline__ void poison_rows(float (&acc)[4], uint32_t nan_lo, uint32_t nan_hi) {
  uint32_t f = ((nan_lo & 0x80808080u) ? 1u : 0u) | ((nan_hi & 0x80808080u) ? 2u : 0u);
  f |= __shfl_xor_sync(0xffffffffu, f, 1);
  f |= __shfl_xor_sync(0xffffffffu, f, 2);
  if (f & 1u) acc[0] = acc[1] = __int_as_float(0x7FC00000);
  if (f & 2u) acc[2] = acc[3] = __int_as_float(0x7FC00000);
}

__device__ __forceinline__ void route_one(const FewRouting& r, int tok, int E, float* w, int32_t* ids,
                                          float* s_choice) {
  const float* row = r.logits + (int64_t)tok * E;
  if (E <= 64)
    route_token_general<2, false>(row, r.bias, tok, E, r.topk, r.renormalize, r.n_group, r.topk_group, r.scoring,
                                  r.gmode, r.scale, w, ids, s_choice);
  else if (E <= 256)
    route_token_general<8, false>(row, r.bias, tok, E, r.topk, r.renormalize, r.n_group, r.topk_group, r.scoring,
                                  r.gmode, r.scale, w, ids, s_choice);
  else
    route_token_general<16, false>(row, r.bias, tok, E, r.topk, r.renormalize, r.n_group, r.topk_group, r.scoring,
                                   r.gmode, r.scale, w, ids, s_choice);
}

struct UpShared {
  float choice[kUpWarps][kRouteMaxExperts];
  float weight[kFewMaxPairs];
  int32_t id[kFewMaxPairs];
  int32_t count[kRouteMaxExperts];   // pairs of an expert, then its first chunk
  int32_t chunk_expert[kFewMaxPairs];
  int16_t chunk_pair[kFewMaxPairs][kFewCols];
  int32_t n_chunks;
};

template <typename T, bool F8>
__global__ void __launch_bounds__(32 * kUpWarps, 1)
few_up_kernel(const T* __restrict__ x, int64_t ld_x, FewRouting rt, const uint8_t* __restrict__ w1,
              const float* __restrict__ w1s, int M, int E, int K, int N, T* __restrict__ act, FewTables* tab) {
  extern __shared__ __align__(16) uint8_t smem_up[];
  UpShared& s = *reinterpret_cast<UpShared*>(smem_up);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int P = M * rt.topk;
  for (int t = warp; t < M; t += kUpWarps) {
    route_one(rt, t, E, s.weight, s.id, s.choice[warp]);
    __syncwarp();
  }
  for (int i = threadIdx.x; i < E; i += blockDim.x) s.count[i] = 0;
  for (int i = threadIdx.x; i < kFewMaxPairs * kFewCols / 2; i += blockDim.x)
    reinterpret_cast<uint32_t*>(s.chunk_pair)[i] = 0xFFFFFFFFu;
  __syncthreads();
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
  constexpr int kWords = F8 ? 16 : 8;             // 32-bit words of x per lane and block
  constexpr int kDepth = 3;                       // k blocks in flight per lane
  const int g = lane >> 2, t4 = lane & 3;
  const int nkb = K / kBlkElts;
  const int NB = N / 8;
  const int items = s.n_chunks * NB;
  const int64_t row_bytes = (int64_t)K * kElt;
  for (int it = blockIdx.x * kUpWarps + warp; it < items; it += gridDim.x * kUpWarps) {
    const int c = it / NB, n0 = (it - c * NB) * 8;
    const int e = s.chunk_expert[c];
    const uint8_t* lo_p = w1 + ((int64_t)e * 2 * N + n0 + g) * row_bytes + t4 * 32;
    const uint8_t* hi_p = lo_p + (int64_t)N * row_bytes;
    const int pair = s.chunk_pair[c][g];
    const uint8_t* xp = pair >= 0
                            ? reinterpret_cast<const uint8_t*>(x + (int64_t)(pair / rt.topk) * ld_x) + t4 * (kWords * 4)
                            : nullptr;
    const float* sg = nullptr;
    const float* su = nullptr;
    if constexpr (F8) {
      sg = w1s + ((int64_t)e * (2 * N / 128) + n0 / 128) * (K / 128);
      su = sg + (int64_t)(N / 128) * (K / 128);
    }
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    uint32_t nan_lo = 0, nan_hi = 0;
    uint4 lo[kDepth][2], hi[kDepth][2];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      if (d < nkb) {
        lo[d][0] = ldg_stream(lo_p + d * kBlkBytes);
        lo[d][1] = ldg_stream(lo_p + d * kBlkBytes + 16);
        hi[d][0] = ldg_stream(hi_p + d * kBlkBytes);
        hi[d][1] = ldg_stream(hi_p + d * kBlkBytes + 16);
      }
    }
    for (int kb0 = 0; kb0 < nkb; kb0 += kDepth) {
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        const int kb = kb0 + d;
        if (kb < nkb) {
          uint32_t xv[kWords];
          load_col<kWords>(xp ? xp + (int64_t)kb * (kBlkElts * 2) : nullptr, xv);
          if constexpr (F8) {
            float part[4] = {0.f, 0.f, 0.f, 0.f};
            block_mma<T, F8>(part, lo[d], hi[d], xv, nan_lo, nan_hi);
            const float a = __ldg(sg + kb) * Expand8<T>::kScale, b = __ldg(su + kb) * Expand8<T>::kScale;
            acc[0] = fmaf(a, part[0], acc[0]);
            acc[1] = fmaf(a, part[1], acc[1]);
            acc[2] = fmaf(b, part[2], acc[2]);
            acc[3] = fmaf(b, part[3], acc[3]);
          } else {
            block_mma<T, F8>(acc, lo[d], hi[d], xv, nan_lo, nan_hi);
          }
          const int nx = kb + kDepth;
          if (nx < nkb) {
            lo[d][0] = ldg_stream(lo_p + (int64_t)nx * kBlkBytes);
            lo[d][1] = ldg_stream(lo_p + (int64_t)nx * kBlkBytes + 16);
            hi[d][0] = ldg_stream(hi_p + (int64_t)nx * kBlkBytes);
            hi[d][1] = ldg_stream(hi_p + (int64_t)nx * kBlkBytes + 16);
          }
        }
      }
    }
    if constexpr (F8) poison_rows(acc, nan_lo, nan_hi);
    // this lane: row n0 + g of gate (acc 0, 1) and up (acc 2, 3) for columns 2 t4, 2 t4 + 1
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int pj = s.chunk_pair[c][2 * t4 + j];
      if (pj >= 0) {
        const float gate = acc[j], up = acc[2 + j];
        act[(int64_t)pj * N + n0 + g] = ElemTraits<T>::from_float(gate / (1.0f + expf(-gate)) * up);
      }
    }
  }
}

template <typename T, bool F8>
__global__ void __launch_bounds__(32 * kDownWarps)
few_down_kernel(const T* __restrict__ act, const FewTables* __restrict__ tab, const uint8_t* __restrict__ w2,
                const float* __restrict__ w2s, int M, int topk, int K, int N, T* __restrict__ out) {
  extern __shared__ __align__(16) float s_part[];  // [kDownWarps][M][16]
  constexpr int kElt = F8 ? 1 : 2;
  constexpr int kBlkElts = kBlkBytes / kElt;
  constexpr int kWords = F8 ? 16 : 8;
  constexpr int kDepth = 3;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int h0 = blockIdx.x * 16;
  const int nkb = N / kBlkElts;
  const int64_t row_bytes = (int64_t)N * kElt;
  float* mine = s_part + warp * M * 16;
  for (int i = lane; i < M * 16; i += 32) mine[i] = 0.f;
  __syncwarp();
  const int total = tab->n_chunks * nkb;
  const int b0 = (int)((int64_t)total * warp / kDownWarps), b1 = (int)((int64_t)total * (warp + 1) / kDownWarps);

  int lc = b0 / nkb, lk = b0 - lc * nkb;  // the next block to load
  const uint8_t* lp = nullptr;
  auto row_of = [&](int c) { return w2 + ((int64_t)__ldg(&tab->chunk_expert[c]) * K + h0 + g) * row_bytes + t4 * 32; };
  if (b0 < b1) lp = row_of(lc);
  uint4 lo[kDepth][2], hi[kDepth][2];
  auto load = [&](int d) {
    const uint8_t* p = lp + (int64_t)lk * kBlkBytes;
    lo[d][0] = ldg_stream(p);
    lo[d][1] = ldg_stream(p + 16);
    hi[d][0] = ldg_stream(p + 8 * row_bytes);
    hi[d][1] = ldg_stream(p + 8 * row_bytes + 16);
  };
  int left = b1 - b0;  // blocks not yet loaded
  auto advance = [&]() {
    --left;
    if (++lk == nkb) {
      lk = 0;
      ++lc;
      if (left > 0) lp = row_of(lc);
    }
  };
#pragma unroll
  for (int d = 0; d < kDepth; ++d)
    if (left > 0) { load(d); advance(); }

  int c = b0 < b1 ? b0 / nkb : 0, kb = b0 < b1 ? b0 - c * nkb : 0;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  uint32_t nan_lo = 0, nan_hi = 0;
  const uint8_t* xp = nullptr;
  const float* sp = nullptr;
  auto open_chunk = [&]() {
    const int pair = tab->chunk_pair[c][g];
    xp = pair >= 0 ? reinterpret_cast<const uint8_t*>(act + (int64_t)pair * N) + t4 * (kWords * 4) : nullptr;
    if constexpr (F8) sp = w2s + ((int64_t)tab->chunk_expert[c] * (K / 128) + h0 / 128) * (N / 128);
  };
  auto close_chunk = [&]() {
    if constexpr (F8) {
      poison_rows(acc, nan_lo, nan_hi);
      nan_lo = nan_hi = 0;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int p = tab->chunk_pair[c][2 * t4 + j];
      if (p >= 0) {
        const float w = tab->weight[p];
        float* o = mine + (p / topk) * 16 + g;
        o[0] += w * acc[j];
        o[8] += w * acc[2 + j];
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
        uint32_t xv[kWords];
        load_col<kWords>(xp ? xp + (int64_t)kb * (kBlkElts * 2) : nullptr, xv);
        if constexpr (F8) {
          float part[4] = {0.f, 0.f, 0.f, 0.f};
          block_mma<T, F8>(part, lo[d], hi[d], xv, nan_lo, nan_hi);
          const float a = __ldg(sp + kb) * Expand8<T>::kScale;
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j] = fmaf(a, part[j], acc[j]);
        } else {
          block_mma<T, F8>(acc, lo[d], hi[d], xv, nan_lo, nan_hi);
        }
        if (left > 0) { load(d); advance(); }
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
#pragma unroll
    for (int w = 0; w < kDownWarps; ++w) v += s_part[w * M * 16 + i];
    const int t = i >> 4;
    if (tab->bad[t]) v = __int_as_float(0x7FC00000);
    out[(int64_t)t * K + h0 + (i & 15)] = ElemTraits<T>::from_float(v);
  }
}

inline size_t few_tables_bytes() { return (sizeof(FewTables) + 255) / 256 * 256; }
inline bool al16f(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T, bool F8>
cudaError_t launch_few(const void* x, int64_t ld_x, const FewRouting& rt, const void* w1, const float* w1s,
                       const void* w2, const float* w2s, int M, int E, int K, int N, void* out, void* ws,
                       cudaStream_t st) {
  FewTables* tab = static_cast<FewTables*>(ws);
  T* act = reinterpret_cast<T*>(static_cast<uint8_t*>(ws) + few_tables_bytes());
  cudaError_t err = ensure_smem_limit(reinterpret_cast<const void*>(few_up_kernel<T, F8>), (int)sizeof(UpShared));
  if (err != cudaSuccess) return err;
  few_up_kernel<T, F8><<<num_sms(), 32 * kUpWarps, sizeof(UpShared), st>>>(
      static_cast<const T*>(x), ld_x, rt, static_cast<const uint8_t*>(w1), w1s, M, E, K, N, act, tab);
  if ((err = cudaGetLastError()) != cudaSuccess) return err;
  few_down_kernel<T, F8><<<K / 16, 32 * kDownWarps, (size_t)kDownWarps * M * 16 * 4, st>>>(
      act, tab, static_cast<const uint8_t*>(w2), w2s, M, rt.topk, K, N, static_cast<T*>(out));
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
  if (!al16f(hidden_states) || ld_hidden % 8 || ld_hidden < 0 || !al16f(w1) || !al16f(w2) || !al16f(workspace))
    return MOE_ERR_INVALID_ARG;
  if (workspace_bytes < moe_few_workspace_bytes(num_tokens, topk, intermediate_size)) return MOE_ERR_WORKSPACE;
  const int rc = moe_check_device();
  if (rc != MOE_OK) return rc;
  const FewRouting rt{gating_output, bias,         topk,           renormalize, num_expert_group, topk_group,
                      scoring_func,  group_score_mode, routed_scaling_factor};
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
