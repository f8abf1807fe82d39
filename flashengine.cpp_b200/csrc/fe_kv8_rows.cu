// Multi-row paged attention (chunked prefill, speculative verify, draft
// blocks) over the 8-bit KV cache on the 5th-generation tensor cores. No
// counterpart in the reference, whose pools are 16-bit; semantics as
// fe_attn_run over the cache's values code * 2^exponent.
//
// Mathematics as in fe_kv8_decode.cu: with s the score in base-2 units, v the
// V scale of the key's block, the weights are w = 2^(s + v - m) with m the
// running maximum of s + v, O = sum w code_v, l = sum w 2^-v, out = O / l.
//  * S = Q K^T runs on tcgen05 kind::f8f6f4 with the K codes as they lie in
//    the cache and each query row as two e4m3 parts (high part and residual)
//    scaled by a power of two: two fp8 products take the tensor core the time
//    of one 16-bit product, and K needs no conversion.
//  * O = W V runs on kind::f16 with the weights in f16 (11 bits, kept between
//    2^-9 and 2^15 around the running maximum, so that the codes' 4 bits
//    dominate the error) and V's codes converted to f16, exactly, by a
//    warpgroup. Splitting the weights into two e4m3 parts instead would feed V
//    raw, but costs five conversions a pair of weights (about 14 clocks of a
//    warp) in the softmax warps, which are what bounds this kernel, against
//    the one that f16 takes; converting V costs the spare warpgroup about 250
//    clocks a tile.
//
// One persistent CTA per SM, sixteen warps. An item is 128 packed query rows
// (row p = query row p / G, head kvh*G + p % G) of one sequence and KV head
// against a range of keys, in tiles of 128 keys (64 for head_dim 256).
//  warps 0-7   softmax, as in fe_prefill_tc.cu: a thread per packed row, the
//              two groups take half a tile's keys each, trade maxima through
//              shared memory and keep one O, rescaled lazily in TMEM.
//  warp 8/11   producers of K (with the tiles' scale exponents) and of V.
//  warp 9      issues S into one of three TMEM slots; owns TMEM.
//  warp 10     issues O += W V once both groups wrote their half of W over
//              the slot.
//  warps 12-15 convert: V tiles to f16 (rows past the end become zeros, so
//              nothing that lies there reaches O), and the next item's query
//              rows to their two parts.
// The softmax warps take 184 registers, the others 72 (setmaxnreg: 256 x 184 +
// 256 x 72 = the launch's 512 x 128). All hand-offs are mbarriers; every wait
// is bounded.
#include <mutex>

#include "fe_attn_common.cuh"
#include "fe_kv8_attn.h"
#include "fe_kv8_common.cuh"
#include "fe_tcgen05.cuh"

namespace fe {
namespace {

constexpr int kThreads = 16 * 32;
constexpr int kKWarp = 8, kSWarp = 9, kPvWarp = 10, kVWarp = 11, kConvWarp = 12;
constexpr int kSlots = 3;      // S / W slots in TMEM
constexpr int kKStages = 3;    // raw K tiles
constexpr int kV8Stages = 2;   // raw V tiles
constexpr int kV16Stages = 2;  // V tiles in f16
constexpr int kExpRing = 8;    // tiles of scale factors; K runs at most 6 ahead
constexpr uint32_t kTmemCols = 512;
constexpr float kRescale = 8.f;  // O is rescaled when the maximum grew by 2^8
constexpr float kBias = 7.f;     // weights are kept times 2^7: at most 2^15

template <int D>
struct Cfg {
  static constexpr int kM = 128;
  static constexpr int kN = D == 128 ? 128 : 64;       // keys per tile
  static constexpr int kHalfN = kN / 2;
  static constexpr int kPieces = kN / kTileTokens;
  static constexpr int kHalfBlocks = kPieces / 2;      // scale blocks of a group's half
  static constexpr int kBoxes = D / 128;               // 128-code boxes per row
  static constexpr int kQBox = kM * 128;               // 128 rows x 128 codes
  static constexpr int kQPart = kBoxes * kQBox;
  static constexpr int kQBytes = 2 * kQPart;
  static constexpr int kQBufs = D == 128 ? 2 : 1;
  // raw tiles: [8-key group][box][8 rows x 128 B]; f16 V: [8-key group][64-dim
  // box][8 rows x 128 B]; all in 128-byte swizzle
  static constexpr int kPiece8 = kTileTokens * D;
  static constexpr int kGroup8 = 8 * D;
  static constexpr int kTile8 = kN * D;
  static constexpr int kGroup16 = 16 * D;
  static constexpr int kTile16 = 2 * kTile8;
  static constexpr int kOffK = kQBufs * kQBytes;
  static constexpr int kOffV8 = kOffK + kKStages * kTile8;
  static constexpr int kOffV16 = kOffV8 + kV8Stages * kTile8;
  static constexpr int kOffMax = kOffV16 + kV16Stages * kTile16;  // [tile parity][group][row]
  static constexpr int kOffSum = kOffMax + 2 * 2 * kM * 4;        // [item parity][group][row]
  static constexpr int kOffRow = kOffSum + 2 * 2 * kM * 4;        // [Q buffer][row] score factors
  static constexpr int kOffExp = kOffRow + 2 * kM * 4;            // [ring][8] float4
  static constexpr int kOffBar = kOffExp + kExpRing * 8 * 16;
  static constexpr int kNumBars = 2 + 2 + 1 + 1 + 2 * kKStages + 2 * kV8Stages + 2 * kV16Stages +
                                  kSlots + kSlots + 2 * kSlots + kExpRing + 8 + 1;
  static constexpr int kSmem = kOffBar + kNumBars * 8 + 32;
  static constexpr uint32_t kOCol = D == 128 ? kSlots * kN : 256;
  static constexpr int kGroupDims = D / 2;  // O dims a softmax group rescales and stores
  static_assert(kSmem <= 232448, "shared memory budget");
  static_assert(kSlots * kN <= int(kOCol) && kOCol + D <= 512, "TMEM budget");
};

__device__ __forceinline__ void mma_f8_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// wait_bounded_short, inlined: a call would keep ptxas from giving the two
// halves of the kernel their own register counts.
__device__ __forceinline__ bool wait_bounded_inl(uint64_t* bar, uint32_t parity,
                                                 volatile int* abort_flag) {
  if (mbar_try_wait_short(bar, parity)) return true;
  const uint64_t t0 = global_ns();
  for (;;) {
    if (mbar_try_wait_short(bar, parity)) return true;
    if (*abort_flag) return false;
    if (global_ns() - t0 > kWaitLimitNs) {
      *abort_flag = 1;
      return false;
    }
  }
}

__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile int* flags,
                                              bool& aborted) {
  if (aborted) return false;
  if (!wait_bounded_inl(bar, parity, flags)) aborted = true;
  return !aborted;
}
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* flags,
                                          bool& aborted) {
  wait_or_abort(bar, parity, flags, aborted);
  if (__any_sync(0xffffffffu, aborted)) aborted = true;
  return !aborted;
}

// Sixteen codes to f16, in order.
__device__ __forceinline__ void codes_to_h2(const uint4& v, uint4& lo, uint4& hi) {
  lo = make_uint4(e4m3x2_to_h2(v.x), e4m3x2_hi_to_h2(v.x), e4m3x2_to_h2(v.y),
                  e4m3x2_hi_to_h2(v.y));
  hi = make_uint4(e4m3x2_to_h2(v.z), e4m3x2_hi_to_h2(v.z), e4m3x2_to_h2(v.w),
                  e4m3x2_hi_to_h2(v.w));
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    kv8_rows_kernel(const __grid_constant__ CUtensorMap kmap,
                    const __grid_constant__ CUtensorMap vmap, const Kv8Args<T> ka) {
  using C = Cfg<D>;
  constexpr int kM = C::kM, kN = C::kN, kHalfN = C::kHalfN, kPieces = C::kPieces;
  const AttnArgs<T>& a = ka.a;
  extern __shared__ __align__(16) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* q_full = bars;                        // [buffer] both parts written
  uint64_t* q_empty = q_full + 2;                 // [buffer] S done, row factors read
  uint64_t* o_free = q_empty + 2;
  uint64_t* l_done = o_free + 1;
  uint64_t* k_full = l_done + 1;
  uint64_t* k_empty = k_full + kKStages;
  uint64_t* v8_full = k_empty + kKStages;
  uint64_t* v8_empty = v8_full + kV8Stages;
  uint64_t* v16_full = v8_empty + kV8Stages;
  uint64_t* v16_empty = v16_full + kV16Stages;
  uint64_t* s_full = v16_empty + kV16Stages;      // [slot] S written
  uint64_t* s_free = s_full + kSlots;             // [slot] the PV that read it is done
  uint64_t* p_full = s_free + kSlots;             // [slot*2 + group] W written
  uint64_t* e_full = p_full + 2 * kSlots;         // [ring] scale factors written
  uint64_t* max_bar = e_full + kExpRing;          // [tile parity*4 + quad]
  uint64_t* drain = max_bar + 8;                  // every MMA issued is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kNumBars);
  volatile int* flags = reinterpret_cast<volatile int*>(tmem_slot + 2);
  float* xmax = reinterpret_cast<float*>(smem + C::kOffMax);
  float* xsum = reinterpret_cast<float*>(smem + C::kOffSum);
  float* row_f = reinterpret_cast<float*>(smem + C::kOffRow);
  float4* ring = reinterpret_cast<float4*>(smem + C::kOffExp);  // {K factor, v, 2^-v, -}

  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const MetaHeader* hdr = reinterpret_cast<const MetaHeader*>(a.meta);
  const int view = a.view;
  if (static_cast<int>(blockIdx.x) >= hdr->grid[view]) return;
  const int32_t* cta_off = reinterpret_cast<const int32_t*>(a.meta + hdr->cta_off_off[view]);
  const WorkItem* items = reinterpret_cast<const WorkItem*>(a.meta + hdr->items_off[view]);
  const SeqInfo* seqs = reinterpret_cast<const SeqInfo*>(a.meta + hdr->seqs_off);
  const int32_t* pages = reinterpret_cast<const int32_t*>(a.meta + hdr->pages_off);
  const int it0 = cta_off[blockIdx.x], it1 = cta_off[blockIdx.x + 1];
  if (it0 >= it1) return;
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) raise_device_error(a.err, FE_DEVERR_SMEM_ALIGN);
    return;
  }

  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(&q_full[b], 4);   // one arrival per converter warp
      mbar_init(&q_empty[b], 9);  // the S issuer's commit, the softmax warps
    }
    mbar_init(o_free, 256);
    mbar_init(l_done, 256);
    for (int s = 0; s < kKStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < kV8Stages; ++s) {
      mbar_init(&v8_full[s], 1);
      mbar_init(&v8_empty[s], 4);
    }
    for (int s = 0; s < kV16Stages; ++s) {
      mbar_init(&v16_full[s], 4);
      mbar_init(&v16_empty[s], 1);
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_free[s], 1);
    }
    for (int b = 0; b < 2 * kSlots; ++b) mbar_init(&p_full[b], 4);
    for (int b = 0; b < kExpRing; ++b) mbar_init(&e_full[b], 1);
    for (int b = 0; b < 8; ++b) mbar_init(&max_bar[b], 64);
    mbar_init(drain, 2);
    flags[0] = 0;
    flags[1] = 0;
    fence_barrier_init();
  }
  if (warp == kSWarp) {
    tc::tmem_alloc(tmem_slot, kTmemCols);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  bool aborted = false;
  // q and the pools belong to earlier kernels until here
  pdl_wait();

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == kKWarp || warp == kVWarp) {
      // ---------------------------------------------------------- producers
      const bool is_v = warp == kVWarp;
      const CUtensorMap* map = is_v ? &vmap : &kmap;
      uint64_t* full = is_v ? v8_full : k_full;
      uint64_t* empty = is_v ? v8_empty : k_empty;
      const uint32_t stages = is_v ? kV8Stages : kKStages;
      uint8_t* region = smem + (is_v ? C::kOffV8 : C::kOffK);
      if (lane == 0) prefetch_tensormap(map);
      uint32_t g = 0;
      for (int it = it0; it < it1 && !aborted; ++it) {
        const WorkItem w = items[it];
        const SeqInfo si = seqs[w.seq];
        const int npieces = w.kt1 - w.kt0;
        const int ntiles = (npieces + kPieces - 1) / kPieces;
        // Slot of 16-token piece i; the lanes hold 32 pieces and ask for the
        // next 32 before they are needed. The K producer also holds its
        // pieces' K and V exponents.
        auto piece_slot = [&](int i) -> int {
          if (i >= npieces) return -1;
          const int t0 = (w.kt0 + i) * kTileTokens;
          return __ldg(pages + si.page_off + t0 / a.page) * a.page + (t0 % a.page);
        };
        auto piece_exps = [&](int slot) -> int {
          if (is_v || slot < 0) return 127 | 127 << 8;
          const int64_t at = int64_t(slot / kKv8Block) * ka.hkv + w.kvh;
          return ka.k_exp[at] | ka.v_exp[at] << 8;
        };
        int cur = piece_slot(lane), nxt = piece_slot(32 + lane);
        int ecur = piece_exps(cur), enxt = piece_exps(nxt);
        for (int j = 0; j < ntiles && !aborted; ++j, ++g) {
          const int pb = (kPieces * j) & 31;
          if (j > 0 && pb == 0) {
            cur = nxt;
            ecur = enxt;
            nxt = piece_slot(kPieces * j + 32 + lane);
            enxt = piece_exps(nxt);
          }
          const int pieces = min(kPieces, npieces - kPieces * j);
          const uint32_t st = g % stages;
          int sl[kPieces];
#pragma unroll
          for (int u = 0; u < kPieces; ++u) sl[u] = __shfl_sync(0xffffffffu, cur, pb + u);
          int good = 1;
          if (lane == 0 && !wait_or_abort(&empty[st], ((g / stages) & 1u) ^ 1u, flags, aborted))
            good = 0;
          if (!__shfl_sync(0xffffffffu, good, 0)) {
            aborted = true;
            break;
          }
          if (!is_v) {
            // this tile's factors (the softmax is done with the tile kExpRing
            // back: the S three tiles back has completed, which waited for
            // the PV of the tile six back)
            if (lane >= pb && lane < pb + kPieces) {
              const int ke = exp_clamp(ecur & 0xff), ve = exp_clamp(ecur >> 8);
              ring[(g % kExpRing) * 8 + lane - pb] =
                  make_float4(exp_scale(ke), float(ve - 127), exp_scale(254 - ve), 0.f);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&e_full[g % kExpRing]);
          }
          if (lane == 0) {
            mbar_arrive_expect_tx(&full[st], pieces * C::kPiece8);
            uint8_t* dst = region + st * C::kTile8;
#pragma unroll
            for (int u = 0; u < kPieces; ++u)
              if (u < pieces)
                tma_load_4d(dst + u * C::kPiece8, map, &full[st], 0, 0, w.kvh * C::kBoxes,
                            sl[u] >> 3);
          }
        }
      }
      if (lane == 0) {
        if (aborted) raise_device_error(a.err, FE_DEVERR_TIMEOUT);
        // the last load into each stage has landed before the CTA may exit
        for (uint32_t t = g > stages ? g - stages : 0; t < g; ++t)
          wait_bounded_inl(&full[t % stages], (t / stages) & 1u, flags + 1);
      }
    } else if (warp == kSWarp || warp == kPvWarp) {
      // -------------------------------------------------------- MMA issuers
      if (lane == 0) {
        constexpr uint32_t idesc_s = tc::idesc_f16(0, false, false, kM, kN);  // e4m3 = 0
        constexpr uint32_t idesc_o = tc::idesc_f16(0, false, true, kM, D);    // f16 = 0
        const uint64_t q_desc0 = tc::smem_desc_sw128(smem_u32(smem), 16, 1024);
        const uint64_t k_desc0 =
            tc::smem_desc_sw128(smem_u32(smem + C::kOffK), 16, C::kGroup8);
        const uint64_t v_desc0 =
            tc::smem_desc_sw128(smem_u32(smem + C::kOffV16), 1024, C::kGroup16);
        uint32_t n = 0;  // tiles issued
        int unit = 0;
        for (int it = it0; it < it1 && !aborted; ++it, ++unit) {
          const WorkItem w = items[it];
          const int ntiles = (w.kt1 - w.kt0 + kPieces - 1) / kPieces;
          if (warp == kSWarp) {
            const int qb = unit % C::kQBufs;
            if (!wait_or_abort(&q_full[qb], (unit / C::kQBufs) & 1u, flags, aborted)) break;
            const uint64_t q_desc = q_desc0 + uint64_t((qb * C::kQBytes) >> 4);
            for (int t = 0; t < ntiles && !aborted; ++t, ++n) {
              const int slot = n % kSlots;
              const uint32_t st = n % kKStages;
              if (!wait_or_abort(&s_free[slot], ((n / kSlots) & 1u) ^ 1u, flags, aborted)) break;
              if (!wait_or_abort(&k_full[st], (n / kKStages) & 1u, flags, aborted)) break;
              tc::fence_after_sync();
              const uint64_t k_desc = k_desc0 + uint64_t((st * C::kTile8) >> 4);
#pragma unroll
              for (int part = 0; part < 2; ++part)
#pragma unroll
                for (int kk = 0; kk < D / 32; ++kk) {
                  const int box = kk >> 2, ko = (kk & 3) * 32;
                  mma_f8_ss(tmem + slot * kN,
                            q_desc + uint64_t((part * C::kQPart + box * C::kQBox + ko) >> 4),
                            k_desc + uint64_t((box * 1024 + ko) >> 4), idesc_s,
                            part + kk > 0 ? 1u : 0u);
                }
              tc::commit(&s_full[slot]);
              tc::commit(&k_empty[st]);
            }
            if (!aborted) tc::commit(&q_empty[qb]);
          } else {
            for (int t = 0; t < ntiles && !aborted; ++t, ++n) {
              const int slot = n % kSlots;
              const uint32_t st = n % kV16Stages;
              // O is free once both groups stored the last item's output
              if (t == 0 && unit > 0 &&
                  !wait_or_abort(o_free, (unit - 1) & 1, flags, aborted))
                break;
              if (!wait_or_abort(&v16_full[st], (n / kV16Stages) & 1u, flags, aborted)) break;
              if (!wait_or_abort(&p_full[slot * 2], (n / kSlots) & 1u, flags, aborted)) break;
              if (!wait_or_abort(&p_full[slot * 2 + 1], (n / kSlots) & 1u, flags, aborted)) break;
              tc::fence_after_sync();
              const uint64_t v_desc = v_desc0 + uint64_t((st * C::kTile16) >> 4);
#pragma unroll
              for (int kk = 0; kk < kN / 16; ++kk) {
                const int gi = kk / (kHalfN / 16), kg = kk % (kHalfN / 16);
                tc::mma_f16_ts(tmem + C::kOCol, tmem + slot * kN + gi * kHalfN + kg * 8,
                               v_desc + uint64_t((kk * 2 * C::kGroup16) >> 4), idesc_o,
                               t + kk > 0 ? 1u : 0u);
              }
              tc::commit(&s_free[slot]);
              tc::commit(&v16_empty[st]);
            }
          }
        }
        if (aborted) raise_device_error(a.err, FE_DEVERR_TIMEOUT);
        tc::commit(drain);
        wait_bounded_inl(drain, 0, flags + 1);
      }
    } else {
      // ---------------------------------------------------------- converters
      const int tid = threadIdx.x - kConvWarp * 32;
      const int G = a.G;
      // Query rows of item `u` (the CTA's u-th): a thread per packed row, its
      // scale from the row's largest magnitude, two parts, the row's factor
      // from products to base-2 scores.
      auto convert_q = [&](int u) {
        if (it0 + u >= it1) return;
        const int qb = u % C::kQBufs;
        if (!wait_warp(&q_empty[qb], ((u / C::kQBufs) & 1u) ^ 1u, flags, aborted)) return;
        const WorkItem w = items[it0 + u];
        const SeqInfo si = seqs[w.seq];
        const int p = w.rb0 * kRowBlock + tid;
        const bool valid = p < si.qrows * G;
        const uint4* src = reinterpret_cast<const uint4*>(
            a.q + (valid ? (static_cast<int64_t>(si.q_row0 + p / G) * a.hq + w.kvh * G + p % G) * D
                         : 0));
        float amax = 0.f;
        if (valid) {
#pragma unroll 4
          for (int c = 0; c < D / 8; ++c) {
            const uint4 v = __ldg(src + c);
            const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = unpack2<T>(x[e]);
              if (fabsf(f.x) < INFINITY) amax = fmaxf(amax, fabsf(f.x));
              if (fabsf(f.y) < INFINITY) amax = fmaxf(amax, fabsf(f.y));
            }
          }
        }
        const int e = kv8_query_exp(amax);
        const float up = exp_scale(254 - e);
        row_f[qb * kM + tid] = exp_scale(e) * a.scale_log2;
        uint8_t* dst = smem + qb * C::kQBytes + (tid >> 3) * 1024 + (tid & 7) * 128;
#pragma unroll 2
        for (int c = 0; c < D / 16; ++c) {  // 16 codes
          uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
          if (valid) {
            const uint4 x = __ldg(src + 2 * c), y = __ldg(src + 2 * c + 1);
            kv8_split_query<T>(make_uint2(x.x, x.y), up, hi.x, lo.x);
            kv8_split_query<T>(make_uint2(x.z, x.w), up, hi.y, lo.y);
            kv8_split_query<T>(make_uint2(y.x, y.y), up, hi.z, lo.z);
            kv8_split_query<T>(make_uint2(y.z, y.w), up, hi.w, lo.w);
          }
          uint8_t* at = dst + (c >> 3) * C::kQBox + (((c & 7) ^ (tid & 7)) << 4);
          *reinterpret_cast<uint4*>(at) = hi;
          *reinterpret_cast<uint4*>(at + C::kQPart) = lo;
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[qb]);
      };
      convert_q(0);
      uint32_t n = 0;
      for (int u = 0; it0 + u < it1 && !aborted; ++u) {
        const WorkItem w = items[it0 + u];
        const SeqInfo si = seqs[w.seq];
        const int npieces = w.kt1 - w.kt0;
        const int ntiles = (npieces + kPieces - 1) / kPieces;
        // the next item's queries: after the item's second tile where a second
        // buffer takes them, else after its last (the buffer is then waiting
        // for S of tiles whose V is converted)
        const int q_after = C::kQBufs == 2 ? min(1, ntiles - 1) : ntiles - 1;
        for (int t = 0; t < ntiles; ++t, ++n) {
          const uint32_t s8 = n % kV8Stages, s16 = n % kV16Stages;
          if (!wait_warp(&v8_full[s8], (n / kV8Stages) & 1u, flags, aborted)) break;
          if (!wait_warp(&v16_empty[s16], ((n / kV16Stages) & 1u) ^ 1u, flags, aborted)) break;
          const uint8_t* from = smem + C::kOffV8 + s8 * C::kTile8;
          uint8_t* to = smem + C::kOffV16 + s16 * C::kTile16;
          const int valid = min(si.length - (w.kt0 + kPieces * t) * kTileTokens,
                                (npieces - kPieces * t) * kTileTokens);
          constexpr int kRowChunks = D / 16;
          constexpr int kPer = kN * kRowChunks / 128;
#pragma unroll 4
          for (int k = 0; k < kPer; ++k) {
            const int i = tid + k * 128;
            const int c = i % kRowChunks, r = i / kRowChunks;
            uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
            if (r < valid)
              codes_to_h2(*reinterpret_cast<const uint4*>(
                              from + (r >> 3) * C::kGroup8 + (c >> 3) * 1024 + (r & 7) * 128 +
                              (((c & 7) ^ (r & 7)) << 4)),
                          lo, hi);
            // dims 16c .. 16c + 15: chunks 2c and 2c + 1 of 64-dim box c / 4.
            // Lanes of odd boxes store their second chunk first, so that the
            // eight lanes of a row use all banks.
            uint8_t* at = to + (r >> 3) * C::kGroup16 + (c >> 2) * 1024 + (r & 7) * 128;
            const int odd = (c >> 2) & 1;
            const int ch = (2 * c) & 7;
            *reinterpret_cast<uint4*>(at + (((ch + odd) ^ (r & 7)) << 4)) = odd ? hi : lo;
            *reinterpret_cast<uint4*>(at + (((ch + 1 - odd) ^ (r & 7)) << 4)) = odd ? lo : hi;
          }
          tc::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&v8_empty[s8]);
            mbar_arrive(&v16_full[s16]);
          }
          if (t == q_after) convert_q(u + 1);
        }
      }
      if (aborted && lane == 0) raise_device_error(a.err, FE_DEVERR_TIMEOUT);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    // ------------------------------------------------ softmax and epilogue
    constexpr int kGD = C::kGroupDims, kHB = C::kHalfBlocks;
    const int gi = warp >= 4 ? 1 : 0;
    const int quad = warp & 3;
    const int r = quad * 32 + lane;  // packed row = TMEM lane
    const uint32_t lane_addr = tmem + (uint32_t(quad * 32) << 16);
    const uint32_t o_dims = lane_addr + C::kOCol + gi * kGD;
    const int G = a.G;
    const bool causal = view == 1;
    uint32_t n = 0;  // tiles processed
    int unit = 0;
    for (int it = it0; it < it1 && !aborted; ++it, ++unit) {
      const WorkItem w = items[it];
      const SeqInfo si = seqs[w.seq];
      const int npieces = w.kt1 - w.kt0;
      const int ntiles = (npieces + kPieces - 1) / kPieces;
      const int P = si.qrows * G;
      const int p = w.rb0 * kRowBlock + r;
      const bool row_valid = p < P;
      // keys this row sees in this item
      int lim = (causal && row_valid) ? si.length - si.qrows + p / G + 1 : si.length;
      lim = min(lim, w.kt1 * kTileTokens);
      const int qb = unit % C::kQBufs;
      if (!wait_warp(&q_full[qb], (unit / C::kQBufs) & 1u, flags, aborted)) break;
      const float rf = row_f[qb * kM + r];
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_empty[qb]);
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < ntiles; ++j, ++n) {
        const int slot = n % kSlots;
        const uint32_t half_addr = lane_addr + slot * kN + gi * kHalfN;
        if (!wait_warp(&e_full[n % kExpRing], (n / kExpRing) & 1u, flags, aborted)) break;
        float kf[kHB], vf[kHB], vi[kHB];
#pragma unroll
        for (int b = 0; b < kHB; ++b) {
          const float4 x = ring[(n % kExpRing) * 8 + gi * kHB + b];
          kf[b] = x.x * rf;
          vf[b] = x.y;
          vi[b] = x.z;
        }
        if (!wait_warp(&s_full[slot], (n / kSlots) & 1u, flags, aborted)) break;
        tc::fence_after_sync();
        const int tkey = (w.kt0 + kPieces * j) * kTileTokens + gi * kHalfN;
        float s[kHalfN];
#pragma unroll
        for (int c = 0; c < kHalfN; c += 32)
          tc::ld_32x32b_x32(half_addr + c, *reinterpret_cast<uint32_t(*)[32]>(&s[c]));
        tc::wait_ld();
        if (tkey + kHalfN > lim) {
#pragma unroll
          for (int c = 0; c < kHalfN; ++c)
            if (tkey + c >= lim) s[c] = -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < kHB; ++b) {
          const float* x = s + 16 * b;
          const float m0 = fmax3(x[0], x[1], x[2]), m1 = fmax3(x[3], x[4], x[5]),
                      m2 = fmax3(x[6], x[7], x[8]), m3 = fmax3(x[9], x[10], x[11]),
                      m4 = fmax3(x[12], x[13], x[14]);
          const float mb = fmax3(fmax3(m0, m1, m2), fmax3(m3, m4, x[15]), -INFINITY);
          mx = fmaxf(mx, fmaf(mb, kf[b], vf[b]));
        }
        {
          // trade maxima with the other warp of these rows; the buffer of a
          // tile parity is rewritten only after the partner passed the
          // exchange of the tile in between
          const int b = n & 1;
          float* xm = xmax + b * 2 * kM;
          xm[gi * kM + r] = mx;
          mbar_arrive(&max_bar[b * 4 + quad]);
          if (!wait_warp(&max_bar[b * 4 + quad], (n >> 1) & 1u, flags, aborted)) break;
          mx = fmaxf(mx, xm[(gi ^ 1) * kM + r]);
        }
        const float m_new = fmaxf(m_used, mx);
        // both groups see the same maxima and take the same decisions
        const bool grow = m_new > m_used + kRescale;
        if (__any_sync(0xffffffffu, grow)) {
          const float alpha = grow ? fast_exp2(m_used - m_new) : 1.f;
          if (j > 0) {
            // wait for the last PV into O, then rescale this group's dims
            if (!wait_warp(&s_free[(n - 1) % kSlots], ((n - 1) / kSlots) & 1u, flags, aborted))
              break;
            tc::fence_after_sync();
#pragma unroll
            for (int c2 = 0; c2 < kGD / 32; ++c2) {
              float ov[32];
              tc::ld_32x32b_x32(o_dims + c2 * 32, *reinterpret_cast<uint32_t(*)[32]>(&ov[0]));
              tc::wait_ld();
#pragma unroll
              for (int c = 0; c < 32; ++c) ov[c] *= alpha;
              tc::st_32x32b_x32(o_dims + c2 * 32, *reinterpret_cast<uint32_t(*)[32]>(&ov[0]));
            }
          }
          l *= alpha;
          if (grow) m_used = m_new;
        }
        const float m_sub = (m_used == -INFINITY ? 0.f : m_used) - kBias;
#pragma unroll
        for (int h = 0; h < kHalfN / 32; ++h) {
          uint32_t pk[16];
#pragma unroll
          for (int b2 = 0; b2 < 2; ++b2) {
            const int b = 2 * h + b2;
            const float2 sc2 = make_float2(kf[b], kf[b]);
            const float off = vf[b] - m_sub;
            const float2 off2 = make_float2(off, off);
            float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float2 x =
                  fma2(make_float2(s[16 * b + 2 * e], s[16 * b + 2 * e + 1]), sc2, off2);
              const float2 pp = make_float2(fast_exp2(x.x), fast_exp2(x.y));
              if (e & 1)
                sum1 = add2(sum1, pp);
              else
                sum0 = add2(sum0, pp);
              pk[8 * b2 + e] = pack2<__half>(pp.x, pp.y);
            }
            l = fmaf((sum0.x + sum0.y) + (sum1.x + sum1.y), vi[b], l);
          }
          tc::st_32x32b_x16(half_addr + 16 * h, pk);
        }
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[slot * 2 + gi]);
      }
      if (aborted) break;
      // the item's last PV
      if (ntiles > 0 &&
          !wait_warp(&s_free[(n - 1) % kSlots], ((n - 1) / kSlots) & 1u, flags, aborted))
        break;
      float* xs = xsum + (unit & 1) * 2 * kM;
      xs[gi * kM + r] = l;
      mbar_arrive(l_done);
      if (!wait_warp(l_done, unit & 1, flags, aborted)) break;
      tc::fence_after_sync();
      const float lsum = l + xs[(gi ^ 1) * kM + r];
      const float inv = 1.f / lsum;
      const bool split = w.part >= 0;
      const int rows_rec = min(P, w.rb0 * kRowBlock + kM) - w.rb0 * kRowBlock;
      float* rec = split ? a.partials + w.part : nullptr;
      T* dst = row_valid && !split
                   ? a.out + (static_cast<int64_t>(si.q_row0 + p / G) * a.hq + w.kvh * G + p % G) *
                                 D + gi * kGD
                   : nullptr;
      if (split && row_valid && gi == 0) {
        rec[rows_rec * D + r] = m_used;
        rec[rows_rec * (D + 1) + r] = lsum;
      }
#pragma unroll
      for (int c2 = 0; c2 < kGD / 32; ++c2) {
        float o[32];
        tc::ld_32x32b_x32(o_dims + c2 * 32, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
        tc::wait_ld();
        if (dst) {
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            uint4 pk;
            pk.x = pack2<T>(o[8 * v + 0] * inv, o[8 * v + 1] * inv);
            pk.y = pack2<T>(o[8 * v + 2] * inv, o[8 * v + 3] * inv);
            pk.z = pack2<T>(o[8 * v + 4] * inv, o[8 * v + 5] * inv);
            pk.w = pack2<T>(o[8 * v + 6] * inv, o[8 * v + 7] * inv);
            *reinterpret_cast<uint4*>(dst + c2 * 32 + 8 * v) = pk;
          }
        } else if (split && row_valid) {
          float* row = rec + r * D + gi * kGD + c2 * 32;
#pragma unroll
          for (int v = 0; v < 8; ++v)
            *reinterpret_cast<float4*>(row + 4 * v) =
                make_float4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
        }
      }
      // O and this item's sums have been read: the next item may reuse them
      tc::fence_before_sync();
      mbar_arrive(o_free);
    }
    if (aborted && lane == 0) raise_device_error(a.err, FE_DEVERR_TIMEOUT);
  }

  tc::fence_before_sync();
  __syncthreads();
  if (warp == kSWarp) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
}

template <typename T, int D>
int launch(const CUtensorMap& kmap, const CUtensorMap& vmap, const Kv8Args<T>& args, int grid,
           cudaStream_t stream) {
  static std::once_flag once;
  static cudaError_t attr_err = cudaSuccess;
  std::call_once(once, [] {
    attr_err = cudaFuncSetAttribute(kv8_rows_kernel<T, D>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem);
  });
  if (attr_err != cudaSuccess) return cuda_fail(attr_err, "kv8_rows_kernel attribute");
  FE_CUDA_TRY(launch_pdl(kv8_rows_kernel<T, D>, dim3(grid), dim3(kThreads), Cfg<D>::kSmem, stream,
                         kmap, vmap, args));
  return FE_OK;
}

template <typename T>
int dispatch(int dim, const CUtensorMap& kmap, const CUtensorMap& vmap, const void* args, int grid,
             cudaStream_t stream) {
  const auto& a = *static_cast<const Kv8Args<T>*>(args);
  if (dim == kWideHeadDim) return launch<T, kWideHeadDim>(kmap, vmap, a, grid, stream);
  return launch<T, kHeadDim>(kmap, vmap, a, grid, stream);
}

}  // namespace

int kv8_rows_launch(int dtype, int dim, const CUtensorMap& kmap, const CUtensorMap& vmap,
                    const void* args, int grid, cudaStream_t stream) {
  if (dtype == FE_DTYPE_BF16)
    return dispatch<__nv_bfloat16>(dim, kmap, vmap, args, grid, stream);
  return dispatch<__half>(dim, kmap, vmap, args, grid, stream);
}

}  // namespace fe
