// Latent attention over the paged cache, absorbed form, on the tensor cores (tcgen05 + TMEM + TMA).
//
//   s_j = scale q . [c_j, r_j],   o = sum_j softmax_j(s_j) c_j,   c_j 512 wide, r_j 64 wide
// for every query row (request, draft token, head); all rows of a request share the cached rows, so
// a tile is 128 rows (heads of one or several draft tokens) against 128 keys.
//
// A CTA pair (cta_group::2) takes a tile: each CTA holds 64 rows of Q, P and of O, whose 64 x 512 fp32
// sums fill 256 of its 512 TMEM columns (a single CTA with 128 rows would need all of them and have
// no place for the scores). For S = Q K^T each CTA supplies 64 of the 128 keys, for O += P V it
// supplies half of V's columns, so a key's row crosses from L2 to shared memory twice per pair.
//   warps 0-7  softmax: four threads per row with 32 keys each (TMEM gives a warp 32 of the 128 lanes; lanes
//              0-63 hold keys 0-63, lanes 64-127 keys 64-127); running maximum and sum, P into shared memory, O
//              rescaled when the maximum has moved by 2^8
//   warps 8, 10 TMA producers of K and of V: 16 KB slots ([64 keys][128 values]), four for a tile's K and four for
//              its V, the rotary keys in a buffer of their own; each slot is refilled as soon as it has been read
//   warps 11-26 (e4m3 pages) widen the codes that the TMA left in half of a slot to bf16 over the whole slot
//              (exact: the scales are powers of two), eight warps a slot
//   warp 9     MMA issuer (first CTA): QK two tiles ahead of PV, so that the softmax of tile j runs
//              beside PV of j - 1 and QK of j + 1
//
// The (request, row tile, key tile) list is cut into equal runs, one per pair, by lengths read on
// the device: no host copy of the lengths, every pair has the same work, whatever the mix. A
// run that ends inside a request leaves its sum, maximum and unnormalised output in the workspace, and
// a second kernel joins the pieces in key order (the same bits on every run).
//
// Masked places: scores are replaced before the maximum. V meets P = 0 in the MMA and 0 * NaN is
// NaN, so in tiles that some row does not see whole the producer zeroes V past the length and looks
// for non-finite values before the draft tokens; if there is one, the rows are computed again key by
// key over visible keys, while the pair's other waits hold their limit (s_hold).
//
// Measured, 74 requests of 2560 tokens, join included: 16-bit pages 65.5 us with 128 heads (805 TFLOP/s, 0.49 of
// the burst bf16 rate) and 61 us with 16 (3.6 TB/s, 0.54 of HBM); e4m3 pages 118 and 117 us.
// 16-bit pages are bound by what L2 gives the SMs: a tile brings 272 KB into a pair's shared memory (144 KB of K
// and 128 KB of V, all of which lies in the K slots of the two CTAs already) in 2.0 us, over 74 pairs 10 TB/s; asking
// for lines in L2 ahead of the copies made it slower. e4m3 pages are bound by the way of a slot from its copy over the
// widening warps to its MMAs, with every code widened twice, for K and for V.
#include "latent.h"

#include <cuda_fp8.h>

#include <algorithm>

namespace moe {
namespace {

constexpr int kDcTile = 128;          // keys per tile, rows per pair
constexpr int kDcRows = 64;           // rows per CTA
constexpr int kDcSlots = 8;
constexpr int kDcSlotBytes = 16384;   // [64 keys][128 values]
constexpr int kDcMaxPairs = 80;
constexpr int kDcSoftmax = 256;       // threads of the softmax warps
constexpr int kDcThreads = kDcSoftmax + 96;  // 16-bit pages
constexpr int kDcConv = 16;           // e4m3 pages: warps that widen the codes,
constexpr int kDcTeam = 8;            // so many to a slot
constexpr int kDcThreads8 = kDcThreads + 32 * kDcConv;
constexpr float kDcRescaleLog2 = 8.0f;

struct DcSmem {
  static constexpr int kRing = 9 * 8192;                      // after Q: nine [64 rows][64] chunks
  static constexpr int kRope = kRing + kDcSlots * kDcSlotBytes;  // [64 keys][64]
  static constexpr int kP = kRope + 8192;                     // two [64 rows][64 keys] chunks
  static constexpr int kX = kP + 16384;                       // the rows' threads' maxima (two tiles) or sums
  static constexpr int kBars = kX + 2 * kDcSoftmax * 4;
  // full[8], empty[8], raw[8], rope_full, rope_free, q_full, q_free, s_full[2], p_full, pv_done, o_free, mma_done,
  // fix, v_fixed
  static constexpr int kNumBars = 3 * kDcSlots + 12;
  static constexpr int kMisc = kBars + kNumBars * 8;
  static constexpr int kBytes = kMisc + 64;
};

struct DcArgs {
  const void* q;
  const uint8_t* cache;
  const int32_t* table;
  int64_t ld_table;
  const int32_t* lens;
  int64_t num_pages;
  int table_width, page_size, page_shift;
  int num_seqs, n_q, heads, rows, row_tiles;
  int pairs;
  float scale, scale_log2;
  int neg;
  void* out;
  float* lse;
  float* part_o;    // [2 * pairs][part_rows][512]
  float2* part_ml;  // [2 * pairs][part_rows]: maximum (log2 units) and sum
  int part_rows;
  int* status;
};

__device__ __forceinline__ int clamped_len(const DcArgs& a, int b) {
  const int64_t cap = (int64_t)a.table_width << a.page_shift;
  const int64_t n = __ldg(a.lens + b);
  return (int)(n < 0 ? 0 : (n > cap ? cap : n));
}
__device__ __forceinline__ int len_tiles(int len) { return (len + kDcTile - 1) / kDcTile; }

// Key tiles of all requests and row tiles, by one warp.
__device__ __forceinline__ int64_t plan_total(const DcArgs& a) {
  const int lane = threadIdx.x & 31;
  int64_t n = 0;
  for (int b = lane; b < a.num_seqs; b += 32) n += len_tiles(clamped_len(a, b));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n * a.row_tiles;
}
__device__ __forceinline__ int64_t plan_chunk(const DcArgs& a, int64_t total) {
  return max((int64_t)1, (total + a.pairs - 1) / a.pairs);
}

struct DcSeg {
  int b, rt, k0, k1, n, len;  // key tiles [k0, k1) of n
  // the same values, known to be equal over the warp
  __device__ __forceinline__ void uniform() {
    b = __shfl_sync(0xffffffffu, b, 0);
    rt = __shfl_sync(0xffffffffu, rt, 0);
    k0 = __shfl_sync(0xffffffffu, k0, 0);
    k1 = __shfl_sync(0xffffffffu, k1, 0);
    n = __shfl_sync(0xffffffffu, n, 0);
    len = __shfl_sync(0xffffffffu, len, 0);
  }
};
// The segments of one pair's run, in order.
struct DcIter {
  int b;
  int64_t off;   // tiles of request b before the next one
  int64_t left;  // tiles of the run still to come
  __device__ __forceinline__ bool next(const DcArgs& a, DcSeg& s) {
    while (left > 0 && b < a.num_seqs) {
      s.len = clamped_len(a, b);
      s.n = len_tiles(s.len);
      if (off >= (int64_t)s.n * a.row_tiles) {
        off = 0;
        ++b;
        continue;
      }
      s.b = b;
      s.rt = (int)(off / s.n);
      s.k0 = (int)(off - (int64_t)s.rt * s.n);
      s.k1 = (int)min((int64_t)s.n, s.k0 + left);
      off += s.k1 - s.k0;
      left -= s.k1 - s.k0;
      return true;
    }
    return false;
  }
};

// Keys that row r of a request sees.
__device__ __forceinline__ int row_seen(const DcArgs& a, int len, int r) {
  return r >= a.rows ? 0 : max(0, len - a.n_q + 1 + r / a.heads);
}

// One row by a warp, key by key over [kb, ke): maximum and sum in natural units, output unnormalised;
// lane l holds the elements 2 l, 2 l + 1 of every 64.
template <typename T, bool E4M3>
__device__ __noinline__ void decode_row(const DcArgs& a, int b, int r, int kb, int ke, float& m, float& l,
                                        float (&acc)[16]) {
  const int lane = threadIdx.x & 31;
  const uint32_t* q =
      reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q) + ((int64_t)b * a.rows + r) * kRowDim);
  float qv[18];
#pragma unroll
  for (int i = 0; i < 9; ++i) {
    const float2 f = ElemTraits<T>::unpack2(__ldg(q + 32 * i + lane));
    qv[2 * i] = f.x;
    qv[2 * i + 1] = f.y;
  }
  m = -INFINITY;
  l = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  for (int j = kb; j < ke; ++j) {
    const int64_t page = __ldg(a.table + b * a.ld_table + (j >> a.page_shift));
    if (page < 0 || page >= a.num_pages) continue;
    const int off = j & (a.page_size - 1);
    float k[18], s = 0.f;
    if constexpr (E4M3) {
      const uint8_t* base = a.cache + page * ((int64_t)a.page_size * kRow8Bytes);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint16_t c = __ldg(reinterpret_cast<const uint16_t*>(base + (int64_t)off * kLatDim + 64 * i) + lane);
        const float sc =
            ue8m0_value(__ldg(base + (int64_t)a.page_size * (kLatDim + 2 * kRopeDim) + off * 4 + (i >> 1)));
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)c, __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        k[2 * i] = f.x * sc;
        k[2 * i + 1] = f.y * sc;
      }
      const float2 f = ElemTraits<T>::unpack2(
          __ldg(reinterpret_cast<const uint32_t*>(base + (int64_t)a.page_size * kLatDim + off * (2 * kRopeDim)) + lane));
      k[16] = f.x;
      k[17] = f.y;
    } else {
      const uint32_t* src =
          reinterpret_cast<const uint32_t*>(a.cache + (page * a.page_size + off) * (int64_t)(2 * kRowDim));
#pragma unroll
      for (int i = 0; i < 9; ++i) {
        const float2 f = ElemTraits<T>::unpack2(__ldg(src + 32 * i + lane));
        k[2 * i] = f.x;
        k[2 * i + 1] = f.y;
      }
    }
#pragma unroll
    for (int i = 0; i < 18; ++i) s = fmaf(qv[i], k[i], s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= a.scale;
    const float mn = fmaxf(m, s);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float f = expf(m - base), p = expf(s - base);
    m = mn;
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = acc[i] * f + p * k[i];
  }
}

// ---------------------------------------------------------------- e4m3 pages into 16-bit slots
// 8 codes times 2^(e - 127) as bf16: f is bf16 2^min(e - 7, 127) in both halves, f2 what is left of it
// (e above 134 only). The codes' exponent and fraction moved to the low end of bf16's are the value times
// 2^-120, subnormals included, and the multiply rounds nothing. Bit 7 of a byte of `nan`: a NaN code, which
// comes out as 480 here.
__device__ __forceinline__ void widen8(uint2 q, uint32_t f, bool big, uint32_t f2, uint32_t& nan, uint32_t (&o)[4]) {
  const uint32_t c[2] = {q.x, q.y};
  nan |= ((c[0] & 0x7F7F7F7Fu) + 0x01010101u) | ((c[1] & 0x7F7F7F7Fu) + 0x01010101u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = __byte_perm(c[i >> 1], 0u, (i & 1) ? 0x3424 : 0x1404);  // two codes in the high bytes
    const uint32_t b = (w & 0x80008000u) | ((w >> 4) & 0x07F007F0u);
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(o[i]) : "r"(b), "r"(f));
  }
  if (big) {
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(o[i]) : "r"(f2));
  }
}
__device__ __forceinline__ void nan8(uint2 q, uint32_t (&o)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = ((i >> 1) ? q.y : q.x) >> (16 * (i & 1));
    if ((w & 0x7Fu) == 0x7Fu) o[i] = (o[i] & 0xFFFF0000u) | 0x7FC0u;
    if ((w & 0x7F00u) == 0x7F00u) o[i] = (o[i] & 0xFFFFu) | 0x7FC00000u;
  }
}

// Marks a segment in CTA `rank`'s s_bad. The barriers that follow order by CTA scope only, so the mark is released to the
// cluster here, and acquired once per segment by the softmax warps that read it.
__device__ __forceinline__ void flag_bad(const int* flag, uint32_t rank, int mark) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_shared(flag, rank)), "r"(mark) : "memory");
  asm volatile("fence.acq_rel.cluster;" ::: "memory");
}
// Sets a word of CTA `rank`'s s_hold; it orders nothing.
__device__ __forceinline__ void set_hold(const int* word, uint32_t rank, int value) {
  asm volatile("st.relaxed.cluster.shared::cluster.u32 [%0], %1;" ::"r"(mapa_shared(word, rank)), "r"(value) : "memory");
}

template <typename T, bool E4M3>
__global__ void __launch_bounds__(E4M3 ? kDcThreads8 : kDcThreads, 1)
latent_decode_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_c,
                     const __grid_constant__ CUtensorMap map_r, const __grid_constant__ CUtensorMap map_s,
                     const __grid_constant__ DcArgs a) {
  // the swizzled tiles need 1024 bytes, and there is no room to round a base up
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) record_status(a.status, MOE_ERR_UNSUPPORTED);
    return;
  }
  uint8_t* ring = smem + DcSmem::kRing;
  uint8_t* s_p = smem + DcSmem::kP;
  float* s_x = reinterpret_cast<float*>(smem + DcSmem::kX);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + DcSmem::kBars);
  uint64_t* full = bars;                 // first CTA's: both CTAs' copies of a slot (0-3: K, 4-7: V)
  uint64_t* empty = full + kDcSlots;     // each CTA's
  uint64_t* raw = empty + kDcSlots;      // each CTA's, e4m3: codes and scales of a slot
  uint64_t* rope_full = raw + kDcSlots;  // first CTA's
  uint64_t* rope_free = rope_full + 1;   // each CTA's
  uint64_t* q_full = rope_free + 1;      // first CTA's
  uint64_t* q_free = q_full + 1;
  uint64_t* s_full = q_free + 1;         // [2]
  uint64_t* p_full = s_full + 2;         // first CTA's: both CTAs' softmax warps
  uint64_t* pv_done = p_full + 1;
  uint64_t* o_free = pv_done + 1;        // first CTA's: both CTAs' softmax warps
  uint64_t* mma_done = o_free + 1;
  uint64_t* fix = mma_done + 1;
  uint64_t* v_fixed = fix + 1;           // first CTA's: the other CTA has looked at its V
  int* misc = reinterpret_cast<int*>(smem + DcSmem::kMisc);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(misc);
  volatile int* s_abort = misc + 1;
  volatile int* s_bad = misc + 2;        // [2]: segment number + 1 whose V holds a non-finite value
  volatile int* s_badpage = misc + 4;
  int* s_plan = misc + 6;                // request, offset (2 words), tiles (2 words)
  volatile int* s_hold = misc + 12;      // [2]: a CTA of the pair computes rows key by key

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = (int)cluster_id_x();

  if (warp == 0) {
    const int64_t total = plan_total(a), chunk = plan_chunk(a, total);
    const int64_t start = min(total, pair * chunk), left = min(total, start + chunk) - start;
    int64_t base = 0;
    int found = a.num_seqs;
    int64_t off = 0;
    for (int b0 = 0; b0 < a.num_seqs && left > 0; b0 += 32) {
      const int64_t n = b0 + lane < a.num_seqs ? (int64_t)len_tiles(clamped_len(a, b0 + lane)) * a.row_tiles : 0;
      int64_t inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, start < base + inc);
      if (hit) {
        const int src = __ffs(hit) - 1;
        found = b0 + src;
        off = start - base - __shfl_sync(0xffffffffu, inc - n, src);
        break;
      }
      base += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) {
      s_plan[0] = found;
      *reinterpret_cast<int64_t*>(s_plan + 2) = off;
      *reinterpret_cast<int64_t*>(s_plan + 4) = left;
    }
  }
  if (threadIdx.x == 32) {
    for (int s = 0; s < kDcSlots; ++s) { mbar_init(&full[s], E4M3 ? 2 * kDcTeam : 1); mbar_init(&empty[s], 1); mbar_init(&raw[s], 1); }
    mbar_init(rope_full, 1);
    mbar_init(rope_free, 1);
    mbar_init(q_full, 1);
    mbar_init(q_free, 1);
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(p_full, 2 * kDcSoftmax / 32);
    mbar_init(pv_done, 1);
    mbar_init(o_free, 2 * kDcSoftmax / 32);
    mbar_init(mma_done, 1);
    mbar_init(fix, 1);
    mbar_init(v_fixed, 1);
    *s_abort = 0;
    s_bad[0] = s_bad[1] = 0;
    *s_badpage = 0;
    s_hold[0] = s_hold[1] = 0;
    fence_mbar_init();
  }
  if (warp == 9) { tmem_alloc_pair(s_tmem, 512); tmem_relinquish_pair(); }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // barriers of both CTAs are ready
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  constexpr uint32_t kTmemS = 256;  // O: columns 0-127 and 128-255, S: 256-319 and 320-383
  DcIter it{s_plan[0], *reinterpret_cast<int64_t*>(s_plan + 2), *reinterpret_cast<int64_t*>(s_plan + 4)};
  DcSeg sg{};

  if (warp == 8 || warp == 10) {
    // ------------------------------------------------ TMA producers: the warp converged, one lane issues, two
    // slots at a time
    const bool one = elect_one();
    const bool for_v = warp == 10;
    const int slot0 = for_v ? 4 : 0;
    // one copy per slot when a page holds 64 keys, else one per page and 64 values
    const int br = min(a.page_size, 64), ppk = 64 / br;
    const uint32_t full0 = mapa_shared(full, 0);
    int seg = 0;
    uint32_t g = 0, fix_phase = 0;  // g: tiles of the run so far
    bool ok = true;
    // pages of a tile: lane l (l < 8) that of keys 16 l .. 16 l + 15
    auto pages_of = [&](int j) {
      const int64_t pi = ((int64_t)j * kDcTile + (lane & 7) * 16) >> a.page_shift;
      return j < sg.k1 && pi < a.table_width ? __ldg(a.table + sg.b * a.ld_table + pi) : -1;
    };
    // One slot, by the elected lane: 64 keys of tile j (from key half `half`; pg: their pages, by copy), value
    // block blk of 128. 16-bit pages: counted on the first CTA's `full` (whose own arrival expects both CTAs'
    // bytes), or with `local` on this CTA's `fix`. e4m3 pages: as they are, counted on this CTA's raw[], the codes
    // into the second half of the slot, their scale bytes into the first.
    auto copy = [&](int sl, const int (&pg)[4], int half, int j, int blk, bool local) {
      uint8_t* dst = ring + sl * kDcSlotBytes;
      const int row = br == 64 ? (j * kDcTile + half * 64) & (a.page_size - 1) : 0;
      if constexpr (E4M3) {
        mbar_arrive_expect_tx(&raw[sl], 8192 + 256);
        for (int i = 0; i < ppk; ++i) {
          tma_load_3d(&map_c, &raw[sl], dst + 8192 + i * br * 128, blk * 128, row, pg[i]);
          tma_load_3d(&map_s, &raw[sl], dst + i * max(br * 4, 128), row * 4, 0, pg[i]);
        }
      } else {
        if (!local && rank == 0) mbar_arrive_expect_tx(&full[sl], 2 * kDcSlotBytes);
        if (br == 64) {
          if (local) tma_load_4d(&map_c, fix, dst, 0, row, blk * 2, pg[0]);
          else tma_load_4d_pair(&map_c, full0 + sl * 8, dst, 0, row, blk * 2, pg[0]);
        } else {
          for (int i = 0; i < 2 * ppk; ++i) {
            uint8_t* d = dst + (i & 1) * 8192 + (i >> 1) * br * 128;
            if (local) tma_load_4d(&map_c, fix, d, 0, 0, blk * 2 + (i & 1), pg[i >> 1]);
            else tma_load_4d_pair(&map_c, full0 + sl * 8, d, 0, 0, blk * 2 + (i & 1), pg[i >> 1]);
          }
        }
      }
    };
    auto half_pages = [&](int pages, int half, int (&pg)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) pg[i] = __shfl_sync(0xffffffffu, pages, half * 4 + ((i * br) >> 4 & 3));
    };
    auto wait_two = [&](int c) {  // slots c, c + 1 of this warp's four have been read
      return mbar_wait_lanes(lane < 2 ? &empty[slot0 + c + lane] : nullptr, (g & 1u) ^ 1u, a.status, s_abort, s_hold);
    };
    auto load_k = [&](int pages, int j) {
      int pg[4];
      half_pages(pages, (int)rank, pg);
#pragma unroll 1
      for (int c = 0; c < 4; c += 2) {
        if (!wait_two(c)) return false;
        if (one) {
          copy(c, pg, (int)rank, j, c, false);
          copy(c + 1, pg, (int)rank, j, c + 1, false);
        }
        __syncwarp();
      }
      if (!mbar_wait_warp(rope_free, (g & 1u) ^ 1u, a.status, s_abort, s_hold)) return false;
      if (one) {
        const int row = br == 64 ? (j * kDcTile + (int)rank * 64) & (a.page_size - 1) : 0;
        if (rank == 0) mbar_arrive_expect_tx(rope_full, 2 * 8192);
        for (int i = 0; i < ppk; ++i)
          tma_load_3d_pair(&map_r, full0 + 3 * kDcSlots * 8, smem + DcSmem::kRope + i * br * 128, 0, row, pg[i]);
      }
      __syncwarp();
      ++g;
      return true;
    };
    // slot order of V: value block 0 keys 0-63, 64-127, value block 1 keys 0-63, 64-127
    auto load_v = [&](int pages, int j) {
      int pg0[4], pg1[4];
      half_pages(pages, 0, pg0);
      half_pages(pages, 1, pg1);
      const int sure = max(0, sg.len - a.n_q + 1);  // keys that every row sees
      const bool local = !E4M3 && (j + 1) * kDcTile > sure;
      if (local && one) mbar_arrive_expect_tx(fix, 4 * kDcSlotBytes);
#pragma unroll 1
      for (int c = 0; c < 4; c += 2) {
        if (!wait_two(c)) return false;
        if (one) {
          copy(slot0 + c, pg0, 0, j, c + (int)rank, local);
          copy(slot0 + c + 1, pg1, 1, j, c + (int)rank, local);
        }
        __syncwarp();
      }
      ++g;
      if (!local) return true;
      // some row does not see all of this tile: V came in on this CTA's own barrier; zero the rows past the
      // length, look at the rows some query may not see, then hand the slots over
      if (!mbar_wait_warp(fix, fix_phase, a.status, s_abort, s_hold)) return false;
      fix_phase ^= 1;
      uint32_t worst = 0;
      for (int c = 0; c < 4; ++c) {
        uint8_t* base = ring + (slot0 + c) * kDcSlotBytes;
        const int key0 = j * kDcTile + (c & 1) * 64;
        for (int v = max(0, sure - key0) * 16 + lane; v < 64 * 16; v += 32) {  // 16-byte pieces of rows >= sure
          const int row = v >> 4;
          uint4* p = reinterpret_cast<uint4*>(base + ((v >> 3) & 1) * 8192 + row * 128 + (v & 7) * 16);
          if (key0 + row >= sg.len) {
            *p = make_uint4(0u, 0u, 0u, 0u);
          } else {
            const uint4 x = *p;
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int y = 0; y < 4; ++y) worst = max(worst, max(w[y] & 0x7FFFu, (w[y] >> 16) & 0x7FFFu));
          }
        }
      }
      if (__any_sync(0xffffffffu, worst >= (ElemTraits<T>::kFmt == 1 ? 0x7F80u : 0x7C00u)) && lane < 2)
        flag_bad(const_cast<const int*>(s_bad) + (seg & 1), (uint32_t)lane, seg + 1);
      fence_proxy_async_smem();
      __syncwarp();
      if (one) {
        if (rank != 0) mbar_arrive_cluster(mapa_shared(v_fixed, 0));
        else
          for (int c = 0; c < 4; ++c) mbar_arrive(&full[slot0 + c]);
      }
      __syncwarp();
      return true;
    };
    while (ok && it.next(a, sg)) {
      sg.uniform();
      if (for_v) {
        int pg = pages_of(sg.k0);
        for (int j = sg.k0; j < sg.k1 && ok; ++j) {
          const int next = pages_of(j + 1);
          ok = load_v(pg, j);
          pg = next;
        }
      } else {
        // the query rows of the segment before are no longer read
        if (seg > 0 && !mbar_wait_warp(q_free, (seg - 1) & 1, a.status, s_abort, s_hold)) { ok = false; break; }
        if (one) {
          if (rank == 0) mbar_arrive_expect_tx(q_full, 2 * 9 * 8192);
          tma_load_4d_pair(&map_q, mapa_shared(q_full, 0), smem, 0, sg.rt * kDcTile + (int)rank * kDcRows, 0, sg.b);
        }
        __syncwarp();
        int pg = pages_of(sg.k0), pg1 = pages_of(sg.k0 + 1);
        for (int j = sg.k0; j < sg.k1 && ok; ++j) {
          const int pg2 = pages_of(j + 2);
          ok = load_k(pg, j);
          pg = pg1;
          pg1 = pg2;
        }
      }
      ++seg;
    }
    if (!ok) {
      // Copies in flight have to land before the pair may leave. The other CTA's are counted on the first one's
      // barriers, and phases stay open for good where one of the two has stopped, so this warp waits out a time
      // instead: ten thousand times what a copy takes.
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 10000000ull) __nanosleep(1000);
    }
  } else if (warp == 9) {
    if (rank == 0) {
      // ------------------------------------------------ MMA issuer: the warp converged, one lane issues
      constexpr uint32_t kIdescQK = idesc_f16(128, 128, ElemTraits<T>::kFmt);
      constexpr uint32_t kIdescPV = idesc_f16(128, 256, ElemTraits<T>::kFmt) | kIdescBMnMajor;
      const bool one = elect_one();
      int seg = 0, g = 0, n_fixed = 0;  // g: tiles of the run so far
      bool ok = true;
      const uint64_t dq0 = smem_desc_sw128(smem), dk0 = smem_desc_sw128(ring), dp0 = smem_desc_sw128(s_p);
      const uint64_t dv0 = smem_desc_mn_sw128(ring + 4 * kDcSlotBytes, 8192), dr0 = smem_desc_sw128(smem + DcSmem::kRope);
      auto wait_for = [&](uint64_t* bar, uint32_t phase) {
        ok = mbar_wait_warp(bar, phase, a.status, s_abort, s_hold) && ok;
        tc_fence_after();
      };
      // S of the run's tile `tile`; last: nothing reads the segment's Q after it
      auto issue_qk = [&](int tile, bool last) {
        const uint32_t d = tmem + kTmemS + (tile & 1) * 64;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          wait_for(&full[c], tile & 1);
          if (one) {
            const uint64_t da = dq0 + c * (16384 >> 4), db = dk0 + c * (kDcSlotBytes >> 4);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t step = (k >> 2) * (8192 >> 4) + 2 * (k & 3);
              umma_f16_pair(d, da + step, db + step, kIdescQK, (c | k) != 0);
            }
            umma_commit_pair_multicast(&empty[c], 0x3);
          }
          __syncwarp();
        }
        wait_for(rope_full, tile & 1);
        if (one) {
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_f16_pair(d, dq0 + 8 * (8192 >> 4) + 2 * k, dr0 + 2 * k, kIdescQK, 1);
          umma_commit_pair_multicast(rope_free, 0x3);
          umma_commit_pair_multicast(&s_full[tile & 1], 0x3);
          if (last) umma_commit_pair_multicast(q_free, 0x3);
        }
        __syncwarp();
      };
      // a wait that gave up ends the loops at the next tile; until then the MMAs run on what is there
      while (ok && it.next(a, sg)) {
        sg.uniform();
        const int nt = sg.k1 - sg.k0;
        const int sure = max(0, sg.len - a.n_q + 1);
        wait_for(q_full, seg & 1);
        issue_qk(g, nt == 1);
        if (nt > 1) issue_qk(g + 1, nt == 2);
        for (int j = 0; j < nt && ok; ++j) {
          if (j == 0 && seg > 0) wait_for(o_free, (seg - 1) & 1);
          if (!E4M3 && (sg.k0 + j + 1) * kDcTile > sure) {
            wait_for(v_fixed, n_fixed & 1);
            ++n_fixed;
          }
          wait_for(p_full, (g + j) & 1);
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            wait_for(&full[4 + c], (g + j) & 1);
            if (one) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_f16_pair(tmem + (c >> 1) * 128, dp0 + (c & 1) * (8192 >> 4) + 2 * k,
                              dv0 + c * (kDcSlotBytes >> 4) + 128 * k, kIdescPV, (j | (c & 1) | k) != 0);
              umma_commit_pair_multicast(&empty[4 + c], 0x3);
              if (c == 3) umma_commit_pair_multicast(pv_done, 0x3);
            }
            __syncwarp();
          }
          if (j + 2 < nt) issue_qk(g + j + 2, j + 3 == nt);
        }
        g += nt;
        ++seg;
      }
      if (one) umma_commit_pair(mma_done);  // every MMA issued here is done before TMEM is freed
      __syncwarp();
      mbar_wait_warp(mma_done, 0, nullptr, nullptr);
    }
  } else if (E4M3 && warp >= 11) {
    // ------------------------------------------------ e4m3 codes to bf16, in place
    // kDcTeam warps to a slot, the slots of K and V in the order of their products: few warps take long over a
    // slot, and a slot is refilled once per tile, so their time would be the tile's. The TMA leaves the codes of
    // key k where the second half of its bf16 row goes, so eight lanes that take a row's codes and then write
    // both its halves need no other place, and no barrier but their warp's; the scale bytes lie where other
    // rows' first halves go, so the team takes them all before it writes.
    constexpr int kTeams = kDcConv / kDcTeam, kStride = 4 * kDcTeam;   // keys per round of a team
    static_assert(4 % kTeams == 0 && 64 % kStride == 0, "teams share the slots evenly");
    const int team = (warp - 11) / kDcTeam, t = threadIdx.x - kDcThreads;
    const int key_lo = (t >> 3) % kStride, part = t & 7;               // keys key_lo + kStride u, 16 of 128 values
    const uint32_t full0 = mapa_shared(full, 0);
    int seg = 0;
    bool ok = true;
    // this team's slots of K (for_v false) or V of key tile j, the run's tile g
    auto widen = [&](bool for_v, int j, uint32_t g) {
#pragma unroll 1
      for (int c = team; c < 4; c += kTeams) {
        const int slot = for_v ? 4 + c : c;
        const int half = for_v ? (c & 1) : (int)rank, blk = for_v ? (c & 2) + (int)rank : c;
        uint8_t* base = ring + slot * kDcSlotBytes;
        const int first = j * kDcTile + half * 64;
        ok = mbar_wait_warp(&raw[slot], g & 1u, a.status, s_abort, s_hold) && ok;
        // scale bytes: TMA writes start on 128 bytes, with pages of 16 keys a page's 64 bytes are that far apart
        uint32_t scale[64 / kStride];
#pragma unroll
        for (int u = 0; u < 64 / kStride; ++u) {
          const int key = key_lo + kStride * u;
          scale[u] = base[blk + key * 4 + (a.page_size == 16 ? (key >> 4) * 64 : 0)];
        }
        ok = named_bar_and(2 + team, 32 * kDcTeam, ok);
        const int sure = max(0, sg.len - a.n_q + 1);
        bool bad = false;
        const int sw = part >> 2, x = key_lo & 7;
        uint8_t* row = base + sw * 8192 + key_lo * 128;
        // this thread's 32 bytes of chunk part / 4: the two halves in an order that keeps eight lanes on eight banks
        const uint32_t o0 = (uint32_t)((((part & 3) * 2 + sw) ^ x) << 4), o1 = (uint32_t)((((part & 3) * 2 + 1 - sw) ^ x) << 4);
        const uint8_t* src = base + 8192 + key_lo * 128 + part * 16;
#pragma unroll
        for (int u = 0; u < 64 / kStride; ++u) {
          const int key = first + kStride * u + key_lo;
          uint2 q0 = *reinterpret_cast<const uint2*>(src + u * (kStride * 128) + 8 * sw);
          uint2 q1 = *reinterpret_cast<const uint2*>(src + u * (kStride * 128) + 8 - 8 * sw);
          if (key >= sg.len) q0 = q1 = make_uint2(0u, 0u);
          uint32_t v0[4], v1[4], nan = 0;
          const uint32_t f = min(scale[u] + 120u, 254u) * 0x00800080u, f2 = (scale[u] - 7u) * 0x00800080u;
          widen8(q0, f, scale[u] > 134u, f2, nan, v0);
          widen8(q1, f, scale[u] > 134u, f2, nan, v1);
          // above 246 a code may widen to infinity (448 x 2^(e - 127) from 2^128 up)
          if ((nan & 0x80808080u) != 0u || scale[u] > 246u) {
            nan8(q0, v0);
            nan8(q1, v1);
            bad |= key >= sure && key < sg.len;
          }
          __syncwarp();
          *reinterpret_cast<uint4*>(row + u * (kStride * 128) + o0) = make_uint4(v0[0], v0[1], v0[2], v0[3]);
          *reinterpret_cast<uint4*>(row + u * (kStride * 128) + o1) = make_uint4(v1[0], v1[1], v1[2], v1[3]);
        }
        // values that some query may not see must not be NaN or infinite under its P = 0
        if (for_v && __any_sync(0xffffffffu, bad) && lane < 2)
          flag_bad(const_cast<const int*>(s_bad) + (seg & 1), (uint32_t)lane, seg + 1);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(full0 + slot * 8);
      }
    };
    uint32_t g = 0;  // tiles of the run before the segment
    while (ok && it.next(a, sg)) {
      const int nt = sg.k1 - sg.k0;
      widen(false, sg.k0, g);
      if (nt > 1) widen(false, sg.k0 + 1, g + 1);
      for (int i = 0; i < nt && ok; ++i) {
        widen(true, sg.k0 + i, g + i);
        if (i + 2 < nt) widen(false, sg.k0 + i + 2, g + i + 2);
      }
      g += nt;
      ++seg;
    }
  } else {
    // ------------------------------------------------ softmax
    const int half = (warp >> 1) & 1, quarter = warp >> 2;  // keys 64 half + 32 quarter .. + 31 of S; values
                                                            // 256 quarter + 128 half .. + 127 of O
    const int r = (warp & 1) * 32 + lane;                   // row of this CTA
    const uint32_t lane_base = tmem + ((uint32_t)(warp & 3) << 21);
    int seg = 0, g = 0;
    bool ok = true;
    while (ok && it.next(a, sg)) {
      const int row = sg.rt * kDcTile + (int)rank * kDcRows + r;  // row of the request
      const int limit = row_seen(a, sg.len, row);
      float m_ref = -INFINITY, l = 0.f;
      // the segment's pages: a bad one hides its keys (their V arrives as zeros)
      {
        if (threadIdx.x == 0) {
          const int n = __ldg(a.lens + sg.b);
          if (n != sg.len) record_status(a.status, MOE_ERR_INVALID_ARG);
        }
        const int first = (int)(((int64_t)sg.k0 * kDcTile) >> a.page_shift);
        const int last = (int)((min((int64_t)sg.k1 * kDcTile, (int64_t)sg.len) - 1) >> a.page_shift);
        bool bad = false;
        for (int p = first + (int)threadIdx.x; p <= last; p += kDcSoftmax) {
          const int v = __ldg(a.table + sg.b * a.ld_table + p);
          bad |= v < 0 || v >= a.num_pages;
        }
        if (bad) { record_status(a.status, MOE_ERR_INVALID_ARG); *s_badpage = seg + 1; }
        named_bar_sync(1, kDcSoftmax);
      }
      const bool bad_page = *s_badpage == seg + 1;
      for (int j = sg.k0; j < sg.k1; ++j, ++g) {
        // a wait that gave up is carried to the next barrier of the softmax warps, so that all leave together
        ok = mbar_wait(&s_full[g & 1], (g >> 1) & 1, a.status, s_abort, s_hold) && ok;
        tc_fence_after();
        uint32_t raw[32];
        tmem_ld32(lane_base + kTmemS + (g & 1) * 64 + quarter * 32, raw);
        tmem_wait_ld();
        const int key0 = j * kDcTile + half * 64 + quarter * 32;
        const int vis = limit - key0;
        if (a.neg) {
#pragma unroll
          for (int x = 0; x < 32; ++x) raw[x] ^= 0x80000000u;
        }
        if (__any_sync(0xffffffffu, vis < 32)) {
#pragma unroll
          for (int x = 0; x < 32; ++x)
            if (x >= vis) raw[x] = 0xFF800000u;
        }
        if (bad_page) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int64_t pi = ((int64_t)key0 + u * 16) >> a.page_shift;
            const int v = pi < a.table_width ? __ldg(a.table + sg.b * a.ld_table + pi) : -1;
            if (v < 0 || v >= a.num_pages) {
#pragma unroll
              for (int x = 0; x < 16; ++x) raw[u * 16 + x] = 0xFF800000u;
            }
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int x = 0; x < 32; ++x) mx[x & 3] = fmaxf(mx[x & 3], __uint_as_float(raw[x]));
        // the row's other keys are with three other threads; two tiles' maxima in turn
        float* x = s_x + (g & 1) * kDcSoftmax;
        x[threadIdx.x] = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        ok = named_bar_and(1, kDcSoftmax, ok);
        if (!ok) break;
        const float top =
            fmaxf(fmaxf(x[threadIdx.x], x[threadIdx.x ^ 64]), fmaxf(x[threadIdx.x ^ 128], x[threadIdx.x ^ 192])) *
            a.scale_log2;
        const bool move = top > m_ref + kDcRescaleLog2 || m_ref == -INFINITY;
        float f = 1.0f;
        if (move) {
          f = (m_ref == -INFINITY) ? 0.f : ex2(m_ref - top);
          m_ref = top;
          l *= f;
        }
        const float base = m_ref == -INFINITY ? 0.f : m_ref;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p0 = ex2(fmaf(__uint_as_float(raw[2 * e]), a.scale_log2, -base));
          const float p1 = ex2(fmaf(__uint_as_float(raw[2 * e + 1]), a.scale_log2, -base));
          sum[e & 1] += p0;
          sum[2 + (e & 1)] += p1;
          p[e] = ElemTraits<T>::pack2(p0, p1);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if (j > sg.k0) {  // PV of the tile before: its P is read, its O is written
          ok = mbar_wait(pv_done, (g - 1) & 1, a.status, s_abort, s_hold) && ok;
          tc_fence_after();
          if (__any_sync(0xffffffffu, move && f != 1.0f)) {
            const float w = move ? f : 1.0f;
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t o[32];
              tmem_ld32(lane_base + quarter * 128 + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * w);
              tmem_st32(lane_base + quarter * 128 + c * 32, o);
            }
            tmem_wait_st();
          }
        }
        uint8_t* dst = s_p + half * 8192 + r * 128;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *reinterpret_cast<uint4*>(dst + (((quarter * 4 + c) ^ (r & 7)) << 4)) =
              make_uint4(p[4 * c], p[4 * c + 1], p[4 * c + 2], p[4 * c + 3]);
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(p_full, 0));
      }
      ok = ok && mbar_wait(pv_done, (g - 1) & 1, a.status, s_abort, s_hold);
      tc_fence_after();
      // ---------------------------------------------- end of the segment
      ok = named_bar_and(1, kDcSoftmax, ok);  // the maxima of the last tile are read
      if (!ok) break;
      s_x[threadIdx.x] = l;
      named_bar_sync(1, kDcSoftmax);
      // in one order for all four: the same sum
      l = (s_x[r] + s_x[r + 64]) + (s_x[r + 128] + s_x[r + 192]);
      const bool whole = sg.k0 == 0 && sg.k1 == sg.n;
      const int64_t pslot = 2 * pair + (sg.k0 == 0 ? 1 : 0);
      const bool live = row < a.rows;
      asm volatile("fence.acq_rel.cluster;" ::: "memory");  // flag_bad of either CTA, ahead of the products in pv_done
      if (s_bad[seg & 1] == seg + 1) {
        // rows of a long segment take longer than a wait may: the pair's waits are told
        if (threadIdx.x < 2) set_hold(const_cast<const int*>(s_hold) + rank, threadIdx.x, 1);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(o_free, 0));
        for (int rr = warp; rr < kDcRows; rr += kDcSoftmax / 32) {
          const int rw = sg.rt * kDcTile + (int)rank * kDcRows + rr;
          if (rw >= a.rows) break;
          float m, ls, acc[16];
          decode_row<T, E4M3>(a, sg.b, rw, sg.k0 * kDcTile, min(row_seen(a, sg.len, rw), sg.k1 * kDcTile), m, ls, acc);
          const bool some = ls > 0.f || ls != ls;
          if (whole) {
            const int64_t o = (int64_t)sg.b * a.rows + rw;
            const float inv = some ? 1.f / ls : 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + o * kLatDim)[32 * i + lane] =
                  ElemTraits<T>::pack2(acc[2 * i] * inv, acc[2 * i + 1] * inv);
            if (a.lse != nullptr && lane == 0) a.lse[o] = some ? m + logf(ls) : -INFINITY;
          } else {
            const int64_t o = pslot * a.part_rows + (int)rank * kDcRows + rr;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              reinterpret_cast<float2*>(a.part_o + o * kLatDim)[32 * i + lane] = make_float2(acc[2 * i], acc[2 * i + 1]);
            if (lane == 0) a.part_ml[o] = make_float2(m * 1.4426950408889634f, ls);
          }
        }
        named_bar_sync(1, kDcSoftmax);  // all warps' rows
        if (threadIdx.x < 2) set_hold(const_cast<const int*>(s_hold) + rank, threadIdx.x, 0);
      } else {
        const bool some = l > 0.f || l != l;
        const float inv = some ? 1.0f / l : 0.f;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld32(lane_base + quarter * 128 + c * 32, o);
          tmem_wait_ld();
          const int d = quarter * 256 + half * 128 + c * 32;
          if (live) {
            if (whole) {
              uint4* dst =
                  reinterpret_cast<uint4*>(static_cast<T*>(a.out) + ((int64_t)sg.b * a.rows + row) * kLatDim + d);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                uint32_t w[4];
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  w[y] = some ? ElemTraits<T>::pack2(__uint_as_float(o[e * 8 + 2 * y]) * inv,
                                                     __uint_as_float(o[e * 8 + 2 * y + 1]) * inv)
                              : 0u;
                dst[e] = make_uint4(w[0], w[1], w[2], w[3]);
              }
            } else {
              uint4* dst = reinterpret_cast<uint4*>(a.part_o + (pslot * a.part_rows + (int)rank * kDcRows + r) * kLatDim + d);
#pragma unroll
              for (int e = 0; e < 8; ++e) dst[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
          }
        }
        if (live && half == 0 && quarter == 0) {
          if (!whole) a.part_ml[pslot * a.part_rows + (int)rank * kDcRows + r] = make_float2(m_ref, l);
          else if (a.lse != nullptr)
            a.lse[(int64_t)sg.b * a.rows + row] = some ? (m_ref + log2f(l)) * 0.6931471805599453f : -INFINITY;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(o_free, 0));
      }
      named_bar_sync(1, kDcSoftmax);  // s_x is free again
      ++seg;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // no CTA leaves while its peer may use its barriers, shared memory or TMEM
  tc_fence_after();
  if (warp == 9) tmem_dealloc_pair(tmem, 512);
}

// Joins the pieces of requests that several pairs worked on, and writes the rows of empty ones: one
// warp per row, pieces in key order.
template <typename T>
__global__ void __launch_bounds__(128)
latent_decode_join_kernel(const __grid_constant__ DcArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= (int64_t)a.num_seqs * a.rows) return;
  const int b = (int)(row / a.rows), r = (int)(row - (int64_t)b * a.rows), rt = r / kDcTile;
  int64_t total = 0, before = 0;
  for (int i = lane; i < a.num_seqs; i += 32) {
    const int n = len_tiles(clamped_len(a, i));
    total += n;
    before += i < b ? n : 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  const int64_t chunk = plan_chunk(a, total * a.row_tiles);
  const int n = len_tiles(clamped_len(a, b));
  T* out = static_cast<T*>(a.out) + row * kLatDim;
  if (n == 0) {
    for (int i = lane; i < kLatDim / 8; i += 32) reinterpret_cast<uint4*>(out)[i] = make_uint4(0u, 0u, 0u, 0u);
    if (lane == 0) {
      if (a.lse != nullptr) a.lse[row] = -INFINITY;
      if (__ldg(a.lens + b) != 0) record_status(a.status, MOE_ERR_INVALID_ARG);
    }
    return;
  }
  const int64_t g0 = before * a.row_tiles + (int64_t)rt * n;
  const int p0 = (int)(g0 / chunk), p1 = (int)((g0 + n - 1) / chunk);
  if (p0 == p1) return;  // one pair had all of it
  auto place = [&](int p) { return (int64_t)(2 * p + (p == p0 ? 1 : 0)) * a.part_rows + (r - rt * kDcTile); };
  float m = -INFINITY;
  for (int p = p0 + lane; p <= p1; p += 32) m = fmaxf(m, a.part_ml[place(p)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 acc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p = p0; p <= p1; ++p) {
    const int64_t s = place(p);
    const float2 ml = a.part_ml[s];
    if (ml.y == 0.f) continue;  // saw nothing; a NaN sum goes on
    const float w = ex2(ml.x - base);
    l += w * ml.y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 v = reinterpret_cast<const float4*>(a.part_o + s * kLatDim)[32 * i + lane];
      acc[i].x += w * v.x;
      acc[i].y += w * v.y;
      acc[i].z += w * v.z;
      acc[i].w += w * v.w;
    }
  }
  const bool some = l > 0.f || l != l;
  const float inv = some ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    reinterpret_cast<uint2*>(out)[32 * i + lane] =
        make_uint2(ElemTraits<T>::pack2(acc[i].x * inv, acc[i].y * inv), ElemTraits<T>::pack2(acc[i].z * inv, acc[i].w * inv));
  if (lane == 0 && a.lse != nullptr) a.lse[row] = some ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

constexpr int kMaxDev = 64;

// CTA pairs that can be resident at once (a pair needs two SMs of one cluster); asked once per device and kernel.
template <typename K>
cudaError_t resident_pairs(K kern, cudaLaunchConfig_t cfg, int (&cache)[kMaxDev], int* pairs) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev >= 0 && dev < kMaxDev && cache[dev] > 0) {
    *pairs = cache[dev];
    return cudaSuccess;
  }
  cfg.gridDim = dim3((unsigned)num_sms() / 2 * 2, 1, 1);
  int n = 0;
  err = cudaOccupancyMaxActiveClusters(&n, kern, &cfg);
  if (err != cudaSuccess) return err;
  if (n <= 0) return cudaErrorInvalidConfiguration;
  *pairs = std::min(n, kDcMaxPairs);
  if (dev >= 0 && dev < kMaxDev) cache[dev] = *pairs;
  return cudaSuccess;
}

template <typename T, bool E4M3>
cudaError_t launch_decode(int dtype, DcArgs a, cudaStream_t st) {
  CUtensorMap mq, mc, mr, ms;
  const uint64_t row = 2 * kRowDim;
  const uint64_t dq[4] = {64, (uint64_t)a.rows, kRowDim / 64, (uint64_t)a.num_seqs};
  const uint64_t sq[3] = {row, 128, row * (uint64_t)a.rows};
  const uint32_t box_rows = (uint32_t)std::min(a.page_size, 64);
  const uint64_t page8 = (uint64_t)a.page_size * kRow8Bytes;
  bool maps = make_chunks_map(&mq, dtype, a.q, dq, sq, kDcRows, kRowDim / 64);
  if (E4M3) {
    const uint64_t dc[3] = {kLatDim, (uint64_t)a.page_size, (uint64_t)a.num_pages}, sc[2] = {kLatDim, page8};
    const uint64_t dr[3] = {kRopeDim, (uint64_t)a.page_size, (uint64_t)a.num_pages}, sr[2] = {2 * kRopeDim, page8};
    const uint64_t scale_row = (uint64_t)a.page_size * 4;  // a page's scale bytes
    const uint64_t ds[3] = {scale_row, 1, (uint64_t)a.num_pages}, ss[2] = {scale_row, page8};
    maps = maps && make_bytes_map(&mc, a.cache, dc, sc, box_rows, 128) &&
           make_bytes_map(&ms, a.cache + (size_t)a.page_size * (kLatDim + 2 * kRopeDim), ds, ss, 1, box_rows * 4) &&
           make_kmajor_map(&mr, dtype, a.cache + (size_t)a.page_size * kLatDim, 3, dr, sr, box_rows);
  } else {
    const uint64_t dc[4] = {64, (uint64_t)a.page_size, kRowDim / 64, (uint64_t)a.num_pages};
    const uint64_t sc[3] = {row, 128, row * (uint64_t)a.page_size};
    const uint64_t dr[3] = {kRopeDim, (uint64_t)a.page_size, (uint64_t)a.num_pages}, sr[2] = {row, sc[2]};
    maps = maps && make_chunks_map(&mc, dtype, a.cache, dc, sc, box_rows, box_rows == 64 ? 2 : 1) &&
           make_kmajor_map(&mr, dtype, a.cache + 2 * kLatDim, 3, dr, sr, box_rows);
    ms = mc;
  }
  if (!maps) return cudaErrorInvalidValue;
  auto kern = latent_decode_kernel<T, E4M3>;
  cudaError_t err = ensure_smem_limit(reinterpret_cast<const void*>(kern), DcSmem::kBytes);
  if (err != cudaSuccess) return err;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(E4M3 ? kDcThreads8 : kDcThreads, 1, 1);
  cfg.dynamicSmemBytes = DcSmem::kBytes;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  static int pairs_of_device[kMaxDev];
  if ((err = resident_pairs(kern, cfg, pairs_of_device, &a.pairs)) != cudaSuccess) return err;
  cfg.gridDim = dim3(2 * (unsigned)a.pairs, 1, 1);
  if ((err = cudaLaunchKernelEx(&cfg, kern, mq, mc, mr, ms, a)) != cudaSuccess) return err;
  latent_decode_join_kernel<T><<<(unsigned)ceil_div((int64_t)a.num_seqs * a.rows, 4), 128, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace moe

extern "C" size_t moe_latent_decode_workspace_bytes(int64_t num_seqs, int q_len, int heads) {
  if (num_seqs < 0 || q_len <= 0 || heads <= 0) return 0;
  const size_t rows = (size_t)std::min<int64_t>((int64_t)q_len * heads, moe::kDcTile);
  return 2 * (size_t)moe::kDcMaxPairs * rows * (moe::kLatDim * 4 + 8);
}

extern "C" int moe_latent_decode(int dtype, const void* q, int64_t num_seqs, int q_len, int heads, int cache_fmt,
                                 const void* cache, int64_t num_pages, int page_size, const int32_t* block_table,
                                 int64_t ld_table, int table_width, const int32_t* cache_lens, float scale, void* out,
                                 float* lse, void* workspace, size_t workspace_bytes, int* status, void* stream) {
  using namespace moe;
  if (!cache_fmt_ok(cache_fmt) || (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_FP16)) return MOE_ERR_UNSUPPORTED;
  if (cache_fmt == MOE_CACHE_E4M3 ? dtype != MOE_DTYPE_BF16 : dtype != cache_fmt) return MOE_ERR_UNSUPPORTED;
  if (num_seqs < 0 || q_len <= 0 || heads <= 0 || num_pages < 0 || table_width < 0 || ld_table < 0)
    return MOE_ERR_INVALID_ARG;
  if (!page_size_ok(page_size) || num_pages > INT32_MAX || (int64_t)q_len * heads > 65536 || num_seqs > 65535 ||
      (int64_t)table_width * page_size > INT32_MAX - kDcTile)
    return MOE_ERR_BAD_SHAPE;
  if (num_seqs == 0) return MOE_OK;
  if (num_pages == 0 || !q || !cache || !cache_lens || !out || (table_width > 0 && !block_table))
    return MOE_ERR_INVALID_ARG;
  if (!aligned16(q) || !aligned16(cache) || !aligned16(out)) return MOE_ERR_INVALID_ARG;
  if (workspace_bytes < moe_latent_decode_workspace_bytes(num_seqs, q_len, heads) || !workspace || !aligned16(workspace))
    return MOE_ERR_WORKSPACE;
  const int rc = moe_check_device();
  if (rc != MOE_OK) return rc;
  DcArgs a{};
  a.q = q;
  a.cache = static_cast<const uint8_t*>(cache);
  a.table = block_table;
  a.ld_table = ld_table;
  a.lens = cache_lens;
  a.num_pages = num_pages;
  a.table_width = table_width;
  a.page_size = page_size;
  a.page_shift = page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : 7;
  a.num_seqs = (int)num_seqs;
  a.n_q = q_len;
  a.heads = heads;
  a.rows = q_len * heads;
  a.row_tiles = (int)ceil_div(a.rows, kDcTile);
  a.scale = scale;
  // flat softmax for a scale of zero: any scale this small gives scores of zero, and hidden places stay -inf
  a.scale_log2 = scale == 0.f ? 1e-37f : (scale < 0.f ? -scale : scale) * 1.4426950408889634f;
  a.neg = scale < 0.f;
  a.out = out;
  a.lse = lse;
  a.part_rows = std::min(a.rows, kDcTile);
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + 2 * (size_t)kDcMaxPairs * a.part_rows * kLatDim);
  a.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t err = cache_fmt == MOE_CACHE_E4M3   ? launch_decode<__nv_bfloat16, true>(dtype, a, st)
                          : dtype == MOE_DTYPE_BF16 ? launch_decode<__nv_bfloat16, false>(dtype, a, st)
                                                    : launch_decode<__half, false>(dtype, a, st);
  return err == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}
