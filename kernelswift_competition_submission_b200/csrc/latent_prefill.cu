// Latent attention, expanded form, on the tensor cores (tcgen05 + TMEM + TMA).
//
//   s_ij = scale (q_i[0:128] . k_j + q_i[128:192] . r_j),  o_i = sum_j softmax_j(s_ij) v_j
// over the keys j that query i of its request sees; k, v per head, the rotary key r shared.
//
// One CTA takes 256 query rows of one head as two 128-row subtiles and walks the keys 128 at a
// time with a running maximum and sum per row:
//   warps 0-7, 8-15 softmax of subtile 0 / 1, two threads per row with 64 keys each: S from TMEM into
//                   registers, maximum, exp2, row sum in fp32, P as 16-bit pairs back into S's columns
//                   (one thread per row with 128 keys took 2100 clocks of a chain of 4200 per tile)
//   warp 16         TMA producer: K as three [128 keys][64] boxes, V as two [64 keys][128] halves,
//                   16 KB slots in a ring of 8, in the order the MMAs use them
//   warp 17         MMA issuer: S = Q K^T from shared memory, O += P V with P from TMEM and V as it
//                   lies (MN-major)
//   warps 18-19     look at V before its MMAs where a row of the tile may not see a key (see below)
// The MMAs of one subtile run while the other one's softmax does: after PV of subtile i the next
// QK of i is issued at once, so its scores wait for the softmax and not the other way round.
//
// The reference point of a row's exponentials follows its maximum only when that has moved by
// more than 2^8: P then stays below 256 (exact range for both 16-bit types), the sum is fp32, and
// O in TMEM is rescaled a few times per row instead of once per tile. P is rounded to the
// inputs' type for the second product (as wide as V itself; in fp16 the smallest are off by up to 2^-25 of the
// reference's 1); l sums the unrounded values.
//
// Masked places: a score is replaced before the maximum is taken, so keys may hold anything.
// V meets P = 0 in the MMA, and 0 * NaN is NaN, so warps 18-19 zero the V rows past the request's
// end, and look for non-finite values in tiles that some row sees only in part; if there is one,
// the rows of the subtiles that walk the tile are computed again by the softmax warps, key by key over visible
// keys only. A subtile asks for its own tiles alone, and after their look, so its answer does not depend on when
// the other subtile's next V lands.
//
// What bounds it: per 128 keys and CTA the MMAs take 2560 clocks, the exponentials 2048 of the
// 4-per-clock units of each SM quarter, so the two have to overlap all the time, and every fourth pair
// of exponentials is taken off those units by a polynomial. What is left is the chain softmax, PV, QK of each
// subtile (P lies in S's columns): 128 heads of one causal prompt of 7993 tokens take 2500-2570 us (1020-1045 TFLOP/s,
// 0.62-0.63 of the burst bf16 rate), 2.8 us per tile, with the power cap as the clocks' limit. Ragged prompts of up to
// 1777 tokens take 55 us, the longest unit's 14 tiles most of it: units are not split over keys, and start by their place
// in cu_q, not by length.
#include "latent.h"

namespace moe {
namespace {

constexpr int kPfSoftmax = 256;          // softmax threads of a subtile
constexpr int kPfThreads = 2 * kPfSoftmax + 128;
constexpr int kPfTile = 128;             // keys per tile, rows per subtile
constexpr int kPfSlots = 8;
constexpr int kSlotBytes = 16384;
constexpr int kQSubBytes = 3 * 16384;    // a subtile of Q: three [128 rows][64] chunks
constexpr float kRescaleLog2 = 8.0f;
constexpr int kPolyEvery = 4;  // every fourth pair of exponentials by polynomial, beside the exponential units' three.
                               // None, a quarter, a half in turn on one card, us: 7993 tokens of 128 heads 2594, 2555,
                               // 2667; a piece of a context 88.6, 87.5, 90.0; ragged prompts 55.3, 55.1, 55.7

struct PfSmem {
  static constexpr int kRing = 2 * kQSubBytes;
  static constexpr int kX = kRing + kPfSlots * kSlotBytes;  // the rows' threads' maxima or sums
  static constexpr int kBars = kX + 2 * kPfSoftmax * 4;
  // q, full[8], empty[8], s_full[2], p_full[2], o_full[2], v_ok[2], v_raw[2], mma_done
  static constexpr int kNumBars = 1 + 2 * kPfSlots + 11;
  static constexpr int kMisc = kBars + kNumBars * 8;
  static constexpr int kBytes = kMisc + 64;
};

struct PfArgs {
  const void* q;
  int64_t q_st, q_sh;
  const void* kv;
  int64_t kv_st, kv_sh;
  const void* kr;
  int64_t kr_st;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int num_seqs;
  int64_t tq, tk;
  int heads, units;
  float scale;       // natural units, for the row-by-row path
  float scale_log2;  // |scale| * log2(e), above zero
  int neg;           // scale below zero: scores change sign first
  int causal;
  void* out;
  float* lse;
  int* status;
};

// 2^x of two values x <= 2^7 without the exponential unit: x = n + f with n the nearest integer, 2^f by its
// degree-4 polynomial of least relative error on [-1/2, 1/2] (2.7e-6 in fp32; a weighted least-squares fit at
// Chebyshev nodes iterated to equal extrema), times 2^n made from n's bits. n stops at -127, whose bits are
// those of zero: -inf and everything below 2^-126 give 0, NaN stays NaN.
__device__ __forceinline__ void exp2_poly_pair(float& y0, float& y1, float x0, float x1) {
  asm("{\n\t.reg .f32 a, b, c, d;\n\t.reg .b32 m, n;\n\t.reg .b64 x, t, f, p, k, s;\n\t"
      "max.NaN.f32 a, %2, 0fC2FE0000;\n\tmax.NaN.f32 b, %3, 0fC2FE0000;\n\t"  // -127
      "mov.b64 x, {a, b};\n\t"
      "mov.b64 k, 0x4B4000004B400000;\n\tadd.rn.f32x2 t, x, k;\n\t"            // 1.5 * 2^23: n in the low bits
      "mov.b64 {m, n}, t;\n\t"
      "mov.b64 k, 0xCB400000CB400000;\n\tadd.rn.f32x2 f, t, k;\n\t"
      "mov.b64 k, 0xBF800000BF800000;\n\tfma.rn.f32x2 f, f, k, x;\n\t"         // f = x - n
      "mov.b64 {c, d}, f;\n\t"
      "mov.b64 p, {%4, %4};\n\tmov.b64 k, {%5, %5};\n\tfma.rn.f32x2 p, p, f, k;\n\t"
      "mov.b64 k, {%6, %6};\n\tfma.rn.f32x2 p, p, f, k;\n\t"
      "mov.b64 k, {%7, %7};\n\tfma.rn.f32x2 p, p, f, k;\n\t"
      "mov.b64 k, {%8, %8};\n\tfma.rn.f32x2 p, p, f, k;\n\t"
      "shl.b32 m, m, 23;\n\tadd.s32 m, m, 0x3F800000;\n\tshl.b32 n, n, 23;\n\tadd.s32 n, n, 0x3F800000;\n\t"
      "mov.b64 s, {m, n};\n\tmul.rn.f32x2 p, p, s;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "=f"(y0), "=f"(y1)
      : "f"(x0), "f"(x1), "f"(0.009570101276040077f), "f"(0.05591785907745361f), "f"(0.240247443318367f),
        "f"(0.6931217908859253f), "f"(0.9999992847442627f));
}

// One row by a warp, key by key, over the keys it sees: fp32, online softmax. Lane l holds
// elements l, l + 32, ... of the 192 and of the 128.
template <typename T>
__device__ __noinline__ void prefill_row(const PfArgs& a, int64_t t, int h, int64_t k0, int64_t seen) {
  const int lane = threadIdx.x & 31;
  const T* q = static_cast<const T*>(a.q) + t * a.q_st + h * a.q_sh;
  float qv[6];
#pragma unroll
  for (int i = 0; i < 6; ++i) qv[i] = ElemTraits<T>::unpack2(*reinterpret_cast<const uint16_t*>(q + 32 * i + lane)).x;
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int64_t j = 0; j < seen; ++j) {
    const T* kp = static_cast<const T*>(a.kv) + (k0 + j) * a.kv_st + h * a.kv_sh;
    const T* rp = static_cast<const T*>(a.kr) + (k0 + j) * a.kr_st;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      const T* p = i < 4 ? kp + 32 * i : rp + 32 * (i - 4);
      s = fmaf(qv[i], ElemTraits<T>::unpack2(*reinterpret_cast<const uint16_t*>(p + lane)).x, s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= a.scale;
    const float mn = fmaxf(m, s);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float f = expf(m - base), p = expf(s - base);
    m = mn;
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      acc[i] = acc[i] * f +
               p * ElemTraits<T>::unpack2(*reinterpret_cast<const uint16_t*>(kp + kNopeDim + 32 * i + lane)).x;
  }
  const bool some = l > 0.f || l != l;
  const float inv = some ? 1.f / l : 0.f;
  const int64_t row = t * a.heads + h;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    static_cast<T*>(a.out)[row * kNopeDim + 32 * i + lane] = ElemTraits<T>::from_float(acc[i] * inv);
  if (a.lse != nullptr && lane == 0) a.lse[row] = some ? m + logf(l) : -INFINITY;
}

template <typename T>
__global__ void __launch_bounds__(kPfThreads, 1)
latent_prefill_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv,
                      const __grid_constant__ CUtensorMap map_kr, const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ PfArgs a) {
  // the swizzled tiles need 1024 bytes, and there is no room to round a base up
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) record_status(a.status, MOE_ERR_UNSUPPORTED);
    return;
  }
  uint8_t* ring = smem + PfSmem::kRing;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + PfSmem::kBars);
  uint64_t* q_full = bars;
  uint64_t* full = bars + 1;
  uint64_t* empty = full + kPfSlots;
  uint64_t* s_full = empty + kPfSlots;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* v_ok = o_full + 2;
  uint64_t* v_raw = v_ok + 2;
  uint64_t* mma_done = v_raw + 2;
  int* misc = reinterpret_cast<int*>(smem + PfSmem::kMisc);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(misc);
  volatile int* s_abort = misc + 1;
  volatile int* s_bad = misc + 2;  // [2]: a V tile that the subtile walks holds a non-finite value
  int* s_unit = misc + 4;  // request, tile
  volatile int* s_look = misc + 6;  // [2]: a subtile's tiles from the first that is looked at, less one

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int h = blockIdx.x / a.units;
  const int unit = a.units - 1 - (blockIdx.x - h * a.units);

  // which request and tile: prefix of ceil(rows / 256); the rows before cu_q[0] and those past
  // cu_q[num_seqs] are together one more request without keys
  const int64_t lead = min((int64_t)max(__ldg(a.cu_q), 0), a.tq);
  if (warp == 0) {
    int base = 0, found = -1, tile = 0;
    for (int b0 = 0; b0 <= a.num_seqs && found < 0; b0 += 32) {
      const int b = b0 + lane;
      int n = 0;
      if (b <= a.num_seqs) {
        const int64_t lo = min((int64_t)max(__ldg(a.cu_q + b), 0), a.tq);
        const int64_t hi = b < a.num_seqs ? min((int64_t)max(__ldg(a.cu_q + b + 1), 0), a.tq) : a.tq + lead;
        n = hi > lo ? (int)((hi - lo + 255) / 256) : 0;
      }
      int inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, unit < base + inc);
      if (hit) {
        const int src = __ffs(hit) - 1;
        found = b0 + src;
        tile = unit - base - __shfl_sync(0xffffffffu, inc - n, src);
      }
      base += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) { s_unit[0] = found; s_unit[1] = tile; }
  }
  if (threadIdx.x == 32) {
    mbar_init(q_full, 1);
    for (int s = 0; s < kPfSlots; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], kPfSoftmax); mbar_init(&o_full[i], 1); mbar_init(&v_ok[i], 64); mbar_init(&v_raw[i], 2); }
    mbar_init(mma_done, 1);
    *s_abort = 0;
    s_bad[0] = s_bad[1] = 0;
    fence_mbar_init();
  }
  __syncthreads();
  const int req = s_unit[0];
  if (req < 0) return;  // past the last unit: nothing allocated, nothing in flight
  const int64_t q_lo = min((int64_t)max(__ldg(a.cu_q + req), 0), a.tq);
  const int64_t q_hi = req < a.num_seqs ? min((int64_t)max(__ldg(a.cu_q + req + 1), 0), a.tq) : a.tq + lead;
  const int nq = (int)(q_hi - q_lo);
  int64_t k_lo = 0;
  int nk = 0;
  if (req < a.num_seqs) {
    k_lo = min((int64_t)max(__ldg(a.cu_k + req), 0), a.tk);
    const int64_t k_hi = min((int64_t)max(__ldg(a.cu_k + req + 1), 0), a.tk);
    nk = k_hi > k_lo ? (int)(k_hi - k_lo) : 0;
  }
  const int row0 = s_unit[1] * 256;
  // keys seen by row i of the request, and the tiles each subtile walks
  auto seen = [&](int i) { return i >= nq ? 0 : (a.causal ? max(0, nk - nq + 1 + i) : nk); };
  int n_tiles[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int last = min(row0 + i * kPfTile + kPfTile, nq) - 1;  // the subtile's last row
    n_tiles[i] = last >= row0 + i * kPfTile ? (seen(last) + kPfTile - 1) / kPfTile : 0;
  }
  const int n_max = max(n_tiles[0], n_tiles[1]);
  // tile j needs its V looked at when some row that walks it does not see all of it; row 0's
  // limit is the smallest, and the last tile may run past the request
  const int sure = min(nk, a.causal ? max(0, nk - nq + 1 + row0) : nk) / kPfTile;  // tiles all rows see whole

  if (n_max > 0) {
    if (threadIdx.x < 2) s_look[threadIdx.x] = (threadIdx.x ? n_tiles[1] : n_tiles[0]) - 1 - sure;
    if (warp == 17) { tmem_alloc(s_tmem, 512); tmem_relinquish(); }
    tc_fence_before();
  }
  __syncthreads();
  if (n_max == 0) {
    if (warp < 8) {  // 256 rows
      const int i = row0 + threadIdx.x;
      if (i < nq) {
        // past the last request the rows go on at 0
        const int64_t row = (q_lo + i < a.tq ? q_lo + i : q_lo + i - a.tq) * a.heads + h;
        uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * kNopeDim);
#pragma unroll
        for (int c = 0; c < 16; ++c) o[c] = make_uint4(0u, 0u, 0u, 0u);
        if (a.lse != nullptr) a.lse[row] = -INFINITY;
      }
    }
    return;
  }
  tc_fence_after();
  const uint32_t tmem = *s_tmem;

  if (warp == 16) {
    // ------------------------------------------------ TMA producer: the warp converged, one lane issues
    const bool one = elect_one();
    if (one) {
      tma_prefetch_desc(&map_kv);
      tma_prefetch_desc(&map_kr);
      tma_prefetch_desc(&map_v);
      mbar_arrive_expect_tx(q_full, 2 * kQSubBytes);
      for (int i = 0; i < 2; ++i)
        for (int c = 0; c < 3; ++c)
          tma_load_3d(&map_q, q_full, smem + i * kQSubBytes + c * 16384, c * 64, (int)q_lo + row0 + i * kPfTile, h);
    }
    __syncwarp();
    int slot = 0;
    uint32_t phase = 0, issued = 0, issued_parity = 0, raw_issued = 0, raw_parity = 0;
    bool ok = true;
    for (int j = 0; j < n_max && ok; ++j) {
      const int kt = (int)k_lo + j * kPfTile;
#pragma unroll
      for (int c = 0; c < 5; ++c) {
        if (ok) {
          ok = mbar_wait_warp(&empty[slot], phase ^ 1, a.status, s_abort);
          if (ok) {
            uint8_t* dst = ring + slot * kSlotBytes;
            // V that warps 18-19 look at arrives at a barrier of its own, which they see in every phase; its slot
            // is passed on at once and the MMAs wait for v_ok. (Had they waited for the slots' barriers, of
            // which they see V's phases only, a K copy that lands after the V behind it would leave the next phase's
            // parity looking complete.)
            const bool look = c >= 3 && j >= sure;
            const int n = (j - sure) & 1;
            if (one) {
              uint64_t* bar = look ? &v_raw[n] : &full[slot];
              mbar_arrive_expect_tx(bar, kSlotBytes);
              if (look) mbar_arrive(&full[slot]);
              if (c < 2) tma_load_3d(&map_kv, bar, dst, c * 64, kt, h);
              else if (c == 2) tma_load_2d(&map_kr, bar, dst, 0, kt);
              else tma_load_4d(&map_v, bar, dst, 0, kt + (c - 3) * 64, 2, h);
            }
            __syncwarp();
            if (look) {
              raw_issued |= 1u << n;
              raw_parity = (raw_parity & ~(1u << n)) | ((uint32_t)((j - sure) >> 1 & 1) << n);
            }
            issued |= 1u << slot;
            issued_parity = (issued_parity & ~(1u << slot)) | (phase << slot);
            if (++slot == kPfSlots) { slot = 0; phase ^= 1; }
          }
        }
      }
    }
    if (!ok) {  // wait (bounded) for the copies in flight before the CTA may leave
      mbar_wait_warp(q_full, 0, nullptr, nullptr);
      for (int s = 0; s < kPfSlots; ++s)
        if ((issued >> s) & 1u) mbar_wait_warp(&full[s], (issued_parity >> s) & 1u, nullptr, nullptr);
      for (int n = 0; n < 2; ++n)
        if ((raw_issued >> n) & 1u) mbar_wait_warp(&v_raw[n], (raw_parity >> n) & 1u, nullptr, nullptr);
    }
  } else if (warp == 17) {
    // ------------------------------------------------ MMA issuer: the warp converged, one lane issues
    constexpr uint32_t kIdescQK = idesc_f16(128, 128, ElemTraits<T>::kFmt);
    constexpr uint32_t kIdescPV = idesc_f16(128, 128, ElemTraits<T>::kFmt) | kIdescBMnMajor;
    const bool one = elect_one();
    const uint64_t dq0 = smem_desc_sw128(smem), dk0 = smem_desc_sw128(ring), dv0 = smem_desc_mn_sw128(ring, 8192);
    bool ok = true;
    int kslot = 0, vslot = 3;  // ring position of the tile's K (three slots) and V (two)
    uint32_t kphase = 0, vphase = 0;
    auto at = [](int s) { return s >= kPfSlots ? s - kPfSlots : s; };
    // one lane issues: S of subtile i from the K at kslot; `last`: no later user of this K
    auto issue_qk = [&](int i, bool last) {
#pragma unroll
      for (int c = 0; c < 3; ++c) {
        const uint64_t da = dq0 + i * (kQSubBytes >> 4) + c * (16384 >> 4);
        const uint64_t db = dk0 + (uint32_t)at(kslot + c) * (kSlotBytes >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_f16(tmem + i * 128, da + 2 * k, db + 2 * k, kIdescQK, (c | k) != 0);
      }
      umma_commit(&s_full[i]);
      if (last)
        for (int c = 0; c < 3; ++c) umma_commit(&empty[at(kslot + c)]);
    };
    auto issue_pv = [&](int i, bool first, bool fin, bool last) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint64_t db = dv0 + (uint32_t)at(vslot + c) * (kSlotBytes >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f16_ts(tmem + 256 + i * 128, tmem + i * 128 + (c * 4 + k) * 8, db + 128 * k, kIdescPV,
                      !first || (c | k) != 0);
      }
      if (fin) umma_commit(&o_full[i]);
      if (last)
        for (int c = 0; c < 2; ++c) umma_commit(&empty[at(vslot + c)]);
    };
    auto forward = [&](int& s, uint32_t& ph) {
      s += 5;
      if (s >= kPfSlots) { s -= kPfSlots; ph ^= 1; }
    };
    // Everything that PV of a subtile and its next QK need is waited for at once (a wait costs about 125 clocks
    // when all is there, and a subtile's softmax, PV and QK are one chain): lanes 0-1 V, 2 its check where there is one, 3 P, 4-6 K.
    // A wait that gave up ends the loop at the next tile; until then the MMAs run on what is there.
    auto wait_all = [&](int j, int i, bool pv, bool qk) {
      uint64_t* bar = nullptr;
      uint32_t ph = 0;
      if (pv && lane < 2) {
        bar = &full[at(vslot + lane)];
        ph = vslot + lane >= kPfSlots ? vphase ^ 1 : vphase;
      } else if (pv && lane == 2 && j >= sure) {
        bar = &v_ok[(j - sure) & 1];
        ph = ((j - sure) >> 1) & 1;
      } else if (pv && lane == 3) {
        bar = &p_full[i];
        ph = j & 1;
      } else if (qk && lane >= 4 && lane < 7) {
        bar = &full[at(kslot + lane - 4)];
        ph = kslot + lane - 4 >= kPfSlots ? kphase ^ 1 : kphase;
      }
      ok = mbar_wait_lanes(bar, ph, a.status, s_abort) && ok;
      tc_fence_after();
    };
    ok = mbar_wait_warp(q_full, 0, a.status, s_abort);
    wait_all(0, 0, false, true);
    if (one) {
      if (n_tiles[0] > 0) issue_qk(0, n_tiles[1] == 0);
      if (n_tiles[1] > 0) issue_qk(1, true);
    }
    __syncwarp();
    forward(kslot, kphase);
    for (int j = 0; j < n_max && ok; ++j) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool pv = j < n_tiles[i], qk = j + 1 < n_tiles[i];
        if (pv || qk) {
          wait_all(j, i, pv, qk);
          if (one) {
            if (pv) issue_pv(i, j == 0, j + 1 == n_tiles[i], i == 1 || n_tiles[1] <= j);
            if (qk) issue_qk(i, i == 1 || n_tiles[1] <= j + 1);
          }
          __syncwarp();
        }
      }
      forward(vslot, vphase);
      forward(kslot, kphase);
    }
    if (one) umma_commit(mma_done);  // every MMA issued here is done before TMEM is freed
    __syncwarp();
    mbar_wait_warp(mma_done, 0, nullptr, nullptr);
  } else if (warp >= 18) {
    // ------------------------------------------------ V where a row may not see a key
    // Two such tiles in turn: the ring holds no more than two tiles' V.
    const int vt = threadIdx.x - (2 * kPfSoftmax + 64);  // 0 .. 63: a key row of each half
    for (int j = sure; j < n_max; ++j) {
      if (!mbar_wait(&v_raw[(j - sure) & 1], ((j - sure) >> 1) & 1, a.status, s_abort)) break;
      bool wrote = false;
#pragma unroll 1
      for (int c = 3; c < 5; ++c) {
        const int idx = 5 * j + c;
        uint8_t* base = ring + (idx % kPfSlots) * kSlotBytes + vt * 128;
        const bool past = j * kPfTile + (c - 3) * 64 + vt >= nk;
        uint32_t worst = 0;
#pragma unroll
        for (int d = 0; d < 2; ++d) {
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            // any order of the row's eight 16-byte pieces will do; this one spreads the banks
            uint4* p = reinterpret_cast<uint4*>(base + d * 8192 + ((x ^ (vt & 7)) << 4));
            if (past) {
              *p = make_uint4(0u, 0u, 0u, 0u);
            } else {
              const uint4 v = *p;
              const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                worst = max(worst, max(w[y] & 0x7FFFu, (w[y] >> 16) & 0x7FFFu));
              }
            }
          }
        }
        if (worst >= (ElemTraits<T>::kFmt == 1 ? 0x7F80u : 0x7C00u)) {
          if (j < n_tiles[0]) s_bad[0] = 1;
          if (j < n_tiles[1]) s_bad[1] = 1;
        }
        wrote |= past;
      }
      if (wrote) fence_proxy_async_smem();
      mbar_arrive(&v_ok[(j - sure) & 1]);
    }
  } else {
    // ------------------------------------------------ softmax, two threads per row
    const int sub = warp >> 3, half = (warp >> 2) & 1;   // keys 64 half .. + 63 of S, values 64 half .. + 63 of O
    const int r = (warp & 3) * 32 + lane;                // row of the subtile
    const int i_row = row0 + sub * kPfTile + r;          // row of the request
    const int limit = seen(i_row);
    const int n_t = sub ? n_tiles[1] : n_tiles[0];
    const uint32_t lane_base = tmem + ((uint32_t)(warp & 3) << 21);  // 32 lanes per warp
    const uint32_t t_s = lane_base + sub * 128, t_o = lane_base + 256 + sub * 128 + half * 64;
    float* x_max = reinterpret_cast<float*>(smem + PfSmem::kX) + sub * kPfSoftmax;
    float* x_sum = x_max;
    const int x_me = half * kPfTile + r;
    float m_ref = -INFINITY, l = 0.f;  // in log2 units of the scaled scores
    bool ok = true;
    for (int j = 0; j < n_t; ++j) {
      // a wait that gave up is carried to the next barrier of the subtile's warps, so that all leave together
      ok = mbar_wait(&s_full[sub], j & 1, a.status, s_abort) && ok;
      tc_fence_after();
      uint32_t raw[2][32];
#pragma unroll
      for (int c = 0; c < 2; ++c) tmem_ld32(t_s + half * 64 + c * 32, raw[c]);
      tmem_wait_ld();
      if (a.neg) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int x = 0; x < 32; ++x) raw[c][x] ^= 0x80000000u;
      }
      const int vis = limit - j * kPfTile - half * 64;  // of this thread's keys, those that the row sees
      if (__any_sync(0xffffffffu, vis < 64)) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int x = 0; x < 32; ++x)
            if (c * 32 + x >= vis) raw[c][x] = 0xFF800000u;
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int x = 0; x < 32; x += 2)
          mx[(x >> 1) & 3] = fmaxf(fmaxf(mx[(x >> 1) & 3], __uint_as_float(raw[c][x])), __uint_as_float(raw[c][x + 1]));
      // The row's two threads exchange their maxima. The place is free: this tile's scores follow the P that
      // every thread gave after it had read the last ones.
      x_max[x_me] = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      ok = named_bar_and(1 + sub, kPfSoftmax, ok);
      if (!ok) break;
      const float top = fmaxf(x_max[r], x_max[kPfTile + r]) * a.scale_log2;
      const bool move = top > m_ref + kRescaleLog2 || m_ref == -INFINITY;
      float f = 1.0f;
      if (move) {
        f = (m_ref == -INFINITY) ? 0.f : ex2(m_ref - top);
        m_ref = top;
        l *= f;
      }
      if (j > 0 && __any_sync(0xffffffffu, move && f != 1.0f)) {
        // this tile's scores are there, so the PV of the tile before it has finished
        const float g = move ? f : 1.0f;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[16];
          tmem_ld16(t_o + c * 16, o);
          tmem_wait_ld();
#pragma unroll
          for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * g);
          tmem_st16(t_o + c * 16, o);
        }
      }
      const float base = m_ref == -INFINITY ? 0.f : m_ref;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      // P takes the place of S's first 64 columns, which the row's other thread has read before the barrier
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t p[16];
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          float p0, p1;
          fma_pair(p0, p1, __uint_as_float(raw[c][2 * x]), __uint_as_float(raw[c][2 * x + 1]), a.scale_log2, -base);
          if (x % kPolyEvery == kPolyEvery - 1) {
            exp2_poly_pair(p0, p1, p0, p1);
          } else {
            p0 = ex2(p0);
            p1 = ex2(p1);
          }
          add_pair(sum[2 * (x & 1)], sum[2 * (x & 1) + 1], p0, p1);
          p[x] = ElemTraits<T>::pack2(p0, p1);
        }
        tmem_st16(t_s + half * 32 + c * 16, p);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[sub]);
    }
    if (n_t > 0) ok = mbar_wait(&o_full[sub], 0, a.status, s_abort) && ok;
    // The look at the subtile's last tile, and with it at all before: its s_bad no longer changes. (The other
    // subtile walks one tile more at most, on the other barrier, so this phase is the barrier's latest.)
    const int looked = s_look[sub];
    if (looked >= 0) ok = mbar_wait(&v_ok[looked & 1], (looked >> 1) & 1, a.status, s_abort) && ok;
    tc_fence_after();
    ok = named_bar_and(1 + sub, kPfSoftmax, ok);  // the last maxima are read
    if (half == 1) x_sum[r] = l;
    named_bar_sync(1 + sub, kPfSoftmax);
    if (half == 0) {
      l += x_sum[r];
      x_sum[r] = l;
    }
    named_bar_sync(1 + sub, kPfSoftmax);
    l = x_sum[r];
    const bool live = i_row < nq;
    const int64_t row = (q_lo + i_row) * a.heads + h;
    if (s_bad[sub]) {
      if (ok)
        for (int rr = warp & 7; rr < kPfTile; rr += kPfSoftmax / 32) {
          const int i = row0 + sub * kPfTile + rr;
          if (i < nq) prefill_row<T>(a, q_lo + i, h, k_lo, seen(i));
        }
    } else {
      const bool some = l > 0.f || l != l;
      const float inv = some ? 1.0f / l : 0.f;
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        uint32_t o[32];
        if (n_t > 0) {
          tmem_ld32(t_o + c * 32, o);
          tmem_wait_ld();
        }
        if (live) {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * kNopeDim + half * 64 + c * 32);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint32_t w[4];
#pragma unroll
            for (int y = 0; y < 4; ++y)
              w[y] = some ? ElemTraits<T>::pack2(__uint_as_float(o[x * 8 + 2 * y]) * inv,
                                                 __uint_as_float(o[x * 8 + 2 * y + 1]) * inv)
                          : 0u;
            dst[x] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (live && half == 0 && a.lse != nullptr)
        a.lse[row] = some ? (m_ref + log2f(l)) * 0.6931471805599453f : -INFINITY;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 17) {
    tc_fence_after();
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T>
cudaError_t launch_prefill(int dtype, PfArgs a, cudaStream_t st) {
  CUtensorMap mq, mkv, mkr, mv;
  const uint64_t dq[3] = {(uint64_t)kQkDim, (uint64_t)a.tq, (uint64_t)a.heads};
  const uint64_t sq[2] = {(uint64_t)a.q_st * 2, (uint64_t)a.q_sh * 2};
  const uint64_t dkv[3] = {2 * (uint64_t)kNopeDim, (uint64_t)a.tk, (uint64_t)a.heads};
  const uint64_t skv[2] = {(uint64_t)a.kv_st * 2, (uint64_t)a.kv_sh * 2};
  const uint64_t dkr[2] = {(uint64_t)kRopeDim, (uint64_t)a.tk};
  const uint64_t skr[1] = {(uint64_t)a.kr_st * 2};
  if (!make_kmajor_map(&mq, dtype, a.q, 3, dq, sq, kPfTile)) return cudaErrorInvalidValue;
  if (a.tk > 0) {
    // V: both 64-value chunks of 64 keys in one box
    const uint64_t dv[4] = {64, (uint64_t)a.tk, 4, (uint64_t)a.heads};
    const uint64_t sv[3] = {(uint64_t)a.kv_st * 2, 128, (uint64_t)a.kv_sh * 2};
    if (!make_kmajor_map(&mkv, dtype, a.kv, 3, dkv, skv, kPfTile) ||
        !make_kmajor_map(&mkr, dtype, a.kr, 2, dkr, skr, kPfTile) || !make_chunks_map(&mv, dtype, a.kv, dv, sv, 64, 2))
      return cudaErrorInvalidValue;
  } else {
    mkv = mkr = mv = mq;  // no key tile is ever loaded
  }
  cudaError_t err = ensure_smem_limit(reinterpret_cast<const void*>(latent_prefill_kernel<T>), PfSmem::kBytes);
  if (err != cudaSuccess) return err;
  latent_prefill_kernel<T><<<(unsigned)((int64_t)a.units * a.heads), kPfThreads, PfSmem::kBytes, st>>>(mq, mkv, mkr, mv,
                                                                                                        a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace moe

extern "C" int moe_latent_prefill(int dtype, const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* kv,
                                  int64_t kv_stride_t, int64_t kv_stride_h, const void* k_rope, int64_t kr_stride_t,
                                  const int32_t* cu_q, const int32_t* cu_k, int num_seqs, int64_t total_q,
                                  int64_t total_k, int heads, float scale, int causal, void* out, float* lse,
                                  int* status, void* stream) {
  using namespace moe;
  if (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_FP16) return MOE_ERR_UNSUPPORTED;
  if (num_seqs < 0 || total_q < 0 || total_k < 0 || heads <= 0) return MOE_ERR_INVALID_ARG;
  if (total_q > INT32_MAX - 512 || total_k > INT32_MAX - 512 || heads > 65535 || num_seqs > 65535)
    return MOE_ERR_BAD_SHAPE;
  if (total_q == 0) return MOE_OK;
  if (!q || !cu_q || !cu_k || !out || (total_k > 0 && (!kv || !k_rope))) return MOE_ERR_INVALID_ARG;
  if (!aligned16(q) || !aligned16(kv) || !aligned16(k_rope) || !aligned16(out)) return MOE_ERR_INVALID_ARG;
  // 16-byte TMA strides above zero; the stride of a dimension of one is not used
  int64_t st[5] = {total_q > 1 ? q_stride_t : 8, heads > 1 ? q_stride_h : 8, total_k > 1 ? kv_stride_t : 8,
                   heads > 1 ? kv_stride_h : 8, total_k > 1 ? kr_stride_t : 8};
  for (int i = 0; i < 5; ++i)
    if (st[i] <= 0 || st[i] % 8 || st[i] >= (int64_t)1 << 38) return MOE_ERR_BAD_SHAPE;
  const int64_t units = total_q / 256 + num_seqs + 1;
  if (units * heads > INT32_MAX) return MOE_ERR_BAD_SHAPE;
  const int rc = moe_check_device();
  if (rc != MOE_OK) return rc;
  PfArgs a{q,     st[0], st[1], kv,     st[2],   st[3],   k_rope,  st[4],      cu_q, cu_k,
           num_seqs, total_q, total_k, heads, (int)units, scale, 0.f, scale < 0.f, causal != 0, out,
           lse,   status};
  // flat softmax for a scale of zero: any scale this small gives scores of zero, and hidden places stay -inf
  a.scale_log2 = scale == 0.f ? 1e-37f : (scale < 0.f ? -scale : scale) * 1.4426950408889634f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = dtype == MOE_DTYPE_BF16 ? launch_prefill<__nv_bfloat16>(dtype, a, s)
                                                  : launch_prefill<__half>(dtype, a, s);
  return err == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}
