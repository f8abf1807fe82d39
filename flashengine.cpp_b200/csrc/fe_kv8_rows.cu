// Multi-row paged attention (chunked prefill, speculative verify, draft
// blocks) over the 8-bit KV cache on the 5th-generation tensor cores. No
// counterpart in the reference, whose pools are 16-bit; semantics as
// fe_attn_run over the cache's values code * 2^exponent.
//
// Mathematics as in fe_kv8_decode.cu: with s the score in base-2 units, v the
// V scale of the key's block, the weights are w = 2^(s + v - m) with m the
// running maximum of s + v, O = sum w code_v, l = sum w 2^-v, out = O / l.
//  * S = Q K^T runs on tcgen05 kind::f8f6f4 with the K codes as they lie in
//    the cache and each query row scaled by a power of two and split into e4m3
//    parts, each the rounding of what the ones before leave: two for bf16,
//    three for f16. They hold an element exactly down to 2^-9 (bf16) or 2^-6
//    (f16) of the row's largest, and smaller ones to 2^-17.8 of the largest:
//    the last part's subnormals end there. An fp8 product takes the tensor core
//    half the time of a 16-bit one, and K needs no conversion.
//  * O = W V runs on kind::f16 with the weights in f16 and V's codes converted
//    to f16, exactly, by a warpgroup. A weight is kept times 2^7 relative to a
//    running maximum (of s + v) that moves once it is exceeded by 2^8, so the
//    row's largest is stored between 2^7 and 2^15: 11 bits for weights down to
//    2^-21 of it at least, fewer below, none under 2^-32. (The kernels over the
//    16-bit cache keep a half and its residual, about 16 bits; a code of V holds
//    its value to 2^-4.) Splitting the weights into e4m3 parts instead
//    would feed V raw, but costs five conversions a pair of weights in the
//    softmax warps, which are what bounds this kernel, against the one that f16
//    takes.
//
// One persistent CTA per SM, twenty warps. An item is 128 packed query rows
// (row p = query row p / G, head kvh*G + p % G) of one sequence and KV head
// against a range of keys, in tiles of 128 keys (64 for head_dim 256).
//  warps 0-7   softmax, two groups of four warps, a thread per packed row; the
//              groups take alternate tiles, so that one's exponentials run
//              while the other loads scores, finds its maximum or waits. The
//              running maximum passes from tile to tile through shared memory;
//              there is one O, rescaled in TMEM when the maximum has grown by
//              2^8. Each group keeps the sum of its own tiles' weights, and
//              goes on to the next item's tiles while this one is stored.
//  warp 8/11   producers of K (with the tiles' scale exponents) and of V.
//  warp 9      issues S into one of three TMEM slots; owns TMEM.
//  warp 10     issues O += W V once the tile's group wrote W over the slot.
//  warps 12-15 convert V tiles to f16 (rows past the end become zeros, so
//              nothing that lies there reaches O).
//  warps 16-19 split the next items' query rows into their parts and store the
//              items' outputs (by the softmax warps, between items, 120 us
//              against 114 below, and 79 against 68 for 148 blocks of 32 rows
//              over 512 keys).
// All hand-offs are mbarriers; every wait is bounded.
//
// Measured on a B200: 128 blocks of 16 bf16 rows, 32 query heads over 4 KV
// heads of 128 dims, 2064 to 2560 keys each, no mask: 112 us, 690 TFLOP/s and
// 3.0 TB/s (twice that many bytes in a 16-bit cache); 131 us when it runs for
// seconds, at the 1000 W power cap and 1.69 GHz. About 1.3 us for a tile
// of 128 keys and 2.5 us for an item beside its tiles. Neither the tensor pipe
// (40 % busy) nor the exponentials (40 %) nor the issue slots (50 %) bound it:
// without the exponentials 107 us, without 7/8 of the PV products 110, with one
// part of the queries 112, without all three 102. Nor do the loads: a third V
// stage and a fourth K stage in place of the second query buffer change
// nothing on long items. What bounds it is the ring S -> softmax -> PV -> S of
// dependent steps over three TMEM slots, which take all columns beside O.
// Built, measured and not kept (the same case, at 112 to 129 us): V loaded by
// the converting warps two tiles ahead, 215 us (the fence for the asynchronous
// proxy waits for the loads in flight); V stages of half a tile, 155; all 128
// scores in registers with the S slot freed early, 152; S and W in separate
// TMEM halves in turn, 122 to 126; scores loaded 16 keys ahead in either pass
// or both, 2 to 5 % slower; one pass over the scores with the maximum of the
// group's tile before (and corrections where it is exceeded), three softmax
// groups, items' descriptions in shared memory: no change.
#include <mutex>
#include <type_traits>

#include "fe_attn_common.cuh"
#include "fe_kv8_attn.h"
#include "fe_kv8_common.cuh"
#include "fe_tcgen05.cuh"

namespace fe {
namespace {

constexpr int kThreads = 20 * 32;
constexpr int kKWarp = 8, kSWarp = 9, kPvWarp = 10, kVWarp = 11, kConvWarp = 12,
              kQWarp = 16;
constexpr int kSlots = 3;      // S / W slots in TMEM
constexpr int kV16Stages = 2;  // V tiles in f16
constexpr int kExpRing = 8;    // tiles of scale factors; K runs at most 6 ahead
constexpr uint32_t kTmemCols = 512;
constexpr float kRescale = 8.f;  // O is rescaled when the maximum grew by 2^8
constexpr float kBias = 7.f;     // weights are kept times 2^7: at most 2^15
constexpr float kFar = 1 << 20;  // maxima beyond (unit 2^-3 and more) are subtracted apart

template <typename T, int D>
struct Cfg {
  static constexpr bool kHalf = std::is_same<T, __half>::value;
  static constexpr int kM = 128;
  static constexpr int kN = D == 128 ? 128 : 64;       // keys per tile
  static constexpr int kPieces = kN / kTileTokens;     // = scale blocks of a tile
  static constexpr int kBoxes = D / 128;               // 128-code boxes per row
  static constexpr int kParts = kHalf ? 3 : 2;         // e4m3 parts of a query
  static constexpr int kQBox = kM * 128;               // 128 rows x 128 codes
  static constexpr int kQPart = kBoxes * kQBox;
  static constexpr int kQBytes = kParts * kQPart;
  // What the 208 KiB of operands hold: two f16 V tiles, the query parts (twice
  // for bf16 with 128 dims: the next item's rows are converted while this
  // one's tiles run; with one buffer, while the softmax finishes the last
  // tiles, whose S no longer needs it) and raw tiles, of which V's wait longer
  // (for their load, then for the conversion).
  static constexpr int kQBufs = D == 128 && !kHalf ? 2 : 1;
  static constexpr int kKStages = D == 128 ? 3 : (kHalf ? 2 : 3);
  static constexpr int kV8Stages = D == 128 ? (kHalf ? 3 : 2) : (kHalf ? 1 : 2);
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
  static constexpr int kOffMax = kOffV16 + kV16Stages * kTile16;  // [tile parity][row]
  static constexpr int kOffSum = kOffMax + 2 * kM * 4;            // [sum|maximum][group][row]
  static constexpr int kOffRow = kOffSum + 2 * 2 * kM * 4;        // [Q buffer][row] score factors
  static constexpr int kOffExp = kOffRow + 2 * kM * 4;            // [ring][8] float4
  static constexpr int kOffBar = kOffExp + kExpRing * 8 * 16;
  static constexpr int kNumBars = 2 + 2 + 1 + 1 + 2 * kKStages + 2 * kV8Stages + 2 * kV16Stages +
                                  kSlots + kSlots + kSlots + kExpRing + 8 + 1;
  static constexpr int kSmem = kOffBar + kNumBars * 8 + 32;
  static constexpr uint32_t kOCol = D == 128 ? kSlots * kN : 256;
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

__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile int* flags,
                                              bool& aborted) {
  if (aborted) return false;
  if (!wait_bounded_short(bar, parity, flags)) aborted = true;
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
  using C = Cfg<T, D>;
  constexpr int kM = C::kM, kN = C::kN, kPieces = C::kPieces;
  constexpr int kKStages = C::kKStages, kV8Stages = C::kV8Stages;
  const AttnArgs<T>& a = ka.a;
  extern __shared__ __align__(16) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* q_full = bars;                        // [buffer] an item's query parts written
  uint64_t* q_empty = q_full + 2;                 // [buffer] its S done, its row factors read
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
  uint64_t* p_full = s_free + kSlots;             // [slot] W written
  uint64_t* e_full = p_full + kSlots;             // [ring] scale factors written
  uint64_t* max_bar = e_full + kExpRing;          // [tile parity*4 + quad] maxima published
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
  // A CTA without work waits as well: a grid that ended before the one it
  // follows would let the next one start beside that.
  if (static_cast<int>(blockIdx.x) >= hdr->grid[view]) {
    pdl_wait();
    return;
  }
  const int32_t* cta_off = reinterpret_cast<const int32_t*>(a.meta + hdr->cta_off_off[view]);
  const WorkItem* items = reinterpret_cast<const WorkItem*>(a.meta + hdr->items_off[view]);
  const SeqInfo* seqs = reinterpret_cast<const SeqInfo*>(a.meta + hdr->seqs_off);
  const int32_t* pages = reinterpret_cast<const int32_t*>(a.meta + hdr->pages_off);
  const int it0 = cta_off[blockIdx.x], it1 = cta_off[blockIdx.x + 1];
  if (it0 >= it1) {
    pdl_wait();
    return;
  }
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) raise_device_error(a.err, FE_DEVERR_SMEM_ALIGN);
    pdl_wait();
    return;
  }

  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(&q_full[b], 4);   // one arrival per converter warp
      mbar_init(&q_empty[b], 9);  // the S issuer's commit, the softmax warps
    }
    mbar_init(o_free, 128);  // the storing warps
    mbar_init(l_done, 8);    // the softmax warps
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
      mbar_init(&p_full[s], 4);
    }
    for (int b = 0; b < kExpRing; ++b) mbar_init(&e_full[b], 1);
    for (int b = 0; b < 8; ++b) mbar_init(&max_bar[b], 1);
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
        // Slot of 16-token piece i. A lane looks after one piece of a batch of
        // 32: its slot is asked for two batches ahead; in the K producer, the K
        // and V exponents of its block one batch ahead.
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
        int cur = 0, nxt = piece_slot(lane), nxt2 = piece_slot(32 + lane);
        int ecur = 0, enxt = piece_exps(nxt);
        for (int j = 0; j < ntiles && !aborted; ++j, ++g) {
          const int pb = (kPieces * j) & 31;
          if (pb == 0) {
            cur = nxt;
            ecur = enxt;
            nxt = nxt2;
            enxt = piece_exps(nxt);
            nxt2 = piece_slot(kPieces * j + 64 + lane);
          }
          const int pieces = min(kPieces, npieces - kPieces * j);
          const uint32_t st = g % stages;
          int good = 1;
          if (lane == 0 && !wait_or_abort(&empty[st], ((g / stages) & 1u) ^ 1u, flags, aborted))
            good = 0;
          if (!__shfl_sync(0xffffffffu, good, 0)) {
            aborted = true;
            break;
          }
          const int mine = lane - pb;  // this lane's piece of the tile
          if (!is_v && mine >= 0 && mine < kPieces) {
            // this tile's factors (the softmax is done with the tile kExpRing
            // back: the S three tiles back has completed, which waited for
            // the PV of the tile six back)
            const int ke = exp_clamp(ecur & 0xff), ve = exp_clamp(ecur >> 8);
            ring[(g % kExpRing) * 8 + mine] =
                make_float4(exp_scale(ke), float(ve - 127), exp_scale(254 - ve), 0.f);
          }
          if (lane == 0) mbar_arrive_expect_tx(&full[st], pieces * C::kPiece8);
          __syncwarp();
          if (!is_v && lane == 0) mbar_arrive(&e_full[g % kExpRing]);
          if (mine >= 0 && mine < pieces)
            tma_load_4d(region + st * C::kTile8 + mine * C::kPiece8, map, &full[st], 0, 0,
                        w.kvh * C::kBoxes, cur >> 3);
        }
      }
      if (lane == 0) {
        if (aborted) raise_device_error(a.err, FE_DEVERR_TIMEOUT);
        // the last load into each stage has landed before the CTA may exit
        for (uint32_t t = g > stages ? g - stages : 0; t < g; ++t)
          wait_bounded_short(&full[t % stages], (t / stages) & 1u, flags + 1);
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
              for (int part = 0; part < C::kParts; ++part)
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
              // O is free once the last item's output is stored
              if (t == 0 && unit > 0 &&
                  !wait_or_abort(o_free, (unit - 1) & 1, flags, aborted))
                break;
              if (!wait_or_abort(&v16_full[st], (n / kV16Stages) & 1u, flags, aborted)) break;
              if (!wait_or_abort(&p_full[slot], (n / kSlots) & 1u, flags, aborted)) break;
              tc::fence_after_sync();
              const uint64_t v_desc = v_desc0 + uint64_t((st * C::kTile16) >> 4);
#pragma unroll
              for (int kk = 0; kk < kN / 16; ++kk) {
                tc::mma_f16_ts(tmem + C::kOCol, tmem + slot * kN + kk * 8,
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
        wait_bounded_short(drain, 0, flags + 1);
      }
    } else if (warp >= kQWarp) {
      // --------------------------------------------- query conversion, output
      // Rows of the CTA's u-th item: D / 16 lanes a row, 16 elements each.
      // fetch_q copies the 16-bit rows into the item's buffer (zeros past the
      // sequence), 16-byte chunk k of row r to position k % 8 (swizzled) of
      // box k / 8; convert_q replaces a row by its parts in place (the row
      // takes as many bytes as two of them), and sets the row's factor from
      // products to base-2 scores.
      const int G = a.G, nitems = it1 - it0;
      constexpr int kLanes = D / 16, kStep = 32 / kLanes;
      const int qc = lane % kLanes;  // 16 elements, or codes of a part
      const int q_r0 = (warp - kQWarp) * 32 + lane / kLanes;
      const int q_odd = (qc >> 2) & 1;  // odd boxes second chunk first: no bank conflicts
      const int step_row = kStep / G, step_head = kStep % G;
      auto q_at = [&](int u, int r, int k) {
        return smem + (u % C::kQBufs) * C::kQBytes + (k >> 3) * C::kQBox + (r >> 3) * 1024 +
               (r & 7) * 128 + (((k & 7) ^ (r & 7)) << 4);
      };
      auto fetch_q = [&](int u, const WorkItem& w, const SeqInfo& si) {
        int row = (w.rb0 * kRowBlock + q_r0) / G, head = (w.rb0 * kRowBlock + q_r0) % G;
        const T* base =
            a.q + (static_cast<int64_t>(si.q_row0) * a.hq + w.kvh * G) * D + 16 * qc;
#pragma unroll 2
        for (int r = q_r0; r < (q_r0 | 31) + 1; r += kStep) {
          const bool valid = row < si.qrows;
          const T* src = valid ? base + (static_cast<int64_t>(row) * a.hq + head) * D : a.q;
          row += step_row;
          head += step_head;
          if (head >= G) {
            head -= G;
            ++row;
          }
#pragma unroll
          for (int x = 0; x < 2; ++x)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                             smem_u32(q_at(u, r, 2 * qc + x))),
                         "l"(src + 8 * x), "r"(valid ? 16 : 0)
                         : "memory");
        }
      };
      auto convert_q = [&](int u) {
        asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 2
        for (int r = q_r0; r < (q_r0 | 31) + 1; r += kStep) {
          uint4 x = *reinterpret_cast<const uint4*>(q_at(u, r, 2 * qc + q_odd));
          uint4 y = *reinterpret_cast<const uint4*>(q_at(u, r, 2 * qc + 1 - q_odd));
          if (q_odd) {
            const uint4 z = x;
            x = y;
            y = z;
          }
          const uint32_t v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
          uint32_t m2 = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) m2 = max_abs2(m2, v[e], T());
          const float2 mf = unpack2<T>(m2);
          float amax = fmaxf(mf.x, mf.y);
#pragma unroll
          for (int o = kLanes / 2; o; o >>= 1)
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
          const int e = kv8_query_exp(amax);
          // a row that holds an infinity has no defined softmax
          const float up = amax == INFINITY ? NAN : exp_scale(254 - e);
          if (qc == 0) row_f[(u % C::kQBufs) * kM + r] = exp_scale(e) * a.scale_log2;
          uint32_t part[C::kParts][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t four[C::kParts];
            kv8_split_query<T, C::kParts>(v[2 * i], v[2 * i + 1], up, four);
#pragma unroll
            for (int k = 0; k < C::kParts; ++k) part[k][i] = four[k];
          }
          __syncwarp();  // every lane of the row has read its elements
#pragma unroll
          for (int k = 0; k < C::kParts; ++k)
            *reinterpret_cast<uint4*>(q_at(u, r, qc) + k * C::kQPart) =
                make_uint4(part[k][0], part[k][1], part[k][2], part[k][3]);
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[u % C::kQBufs]);
      };
      // Output of the CTA's u-th item, once its last PV is done: the next
      // item's tiles are on their way in the other warps meanwhile.
      uint32_t n_end = 0;  // tiles of the items stored
      auto store_o = [&](int u) {
        const WorkItem w = items[it0 + u];
        const SeqInfo si = seqs[w.seq];
        n_end += (w.kt1 - w.kt0 + kPieces - 1) / kPieces;
        const uint32_t nl = n_end - 1;
        const int quad = warp - kQWarp, r = quad * 32 + lane;
        const int P = si.qrows * G, p = w.rb0 * kRowBlock + r;
        const bool row_valid = p < P, split = w.part >= 0;
        const int rows_rec = min(P, w.rb0 * kRowBlock + kM) - w.rb0 * kRowBlock;
        float* rec = split ? a.partials + w.part : nullptr;
        T* dst = row_valid && !split
                     ? a.out + (static_cast<int64_t>(si.q_row0 + p / G) * a.hq + w.kvh * G +
                                p % G) * D
                     : nullptr;
        if (!wait_warp(l_done, u & 1, flags, aborted)) return;
        // (the last tile's S waited for the slot's PV before)
        if (!wait_warp(&s_free[nl % kSlots], (nl / kSlots) & 1u, flags, aborted)) return;
        tc::fence_after_sync();
        // the group of the last tile has the item's maximum
        const float* sums = xsum + r;
        const float* maxs = xsum + 2 * kM + r;
        const int own = (nl & 1) * kM, other = kM - own;
        const float m_item = maxs[own], m_other = maxs[other];
        float l_other = sums[other];
        if (m_other != m_item) l_other *= fast_exp2(m_other - m_item);
        const float lsum = sums[own] + l_other;
        const float inv = 1.f / lsum;
        if (split && row_valid) {
          rec[rows_rec * D + r] = m_item;
          rec[rows_rec * (D + 1) + r] = lsum;
        }
        const uint32_t o_addr = tmem + (uint32_t(quad * 32) << 16) + C::kOCol;
#pragma unroll 2
        for (int c2 = 0; c2 < D / 32; ++c2) {
          float o[32];
          tc::ld_32x32b_x32(o_addr + c2 * 32, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
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
            float* row = rec + r * D + c2 * 32;
#pragma unroll
            for (int v = 0; v < 8; ++v)
              *reinterpret_cast<float4*>(row + 4 * v) =
                  make_float4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
          }
        }
        // O and this item's sums have been read: the next item may reuse them
        tc::fence_before_sync();
        mbar_arrive(o_free);
      };
      WorkItem w = items[it0];
      SeqInfo si = seqs[w.seq];
      for (int u = 0; u <= nitems && !aborted; ++u) {
        if (u < nitems) {
          if (!wait_warp(&q_empty[u % C::kQBufs], ((u / C::kQBufs) & 1u) ^ 1u, flags, aborted))
            break;
          fetch_q(u, w, si);
          if (u + 1 < nitems) {  // in flight with this item's rows
            w = items[it0 + u + 1];
            si = seqs[w.seq];
          }
          convert_q(u);
        }
        if (u > 0) store_o(u - 1);
      }
      if (aborted && lane == 0) raise_device_error(a.err, FE_DEVERR_TIMEOUT);
    } else {
      // ---------------------------------------------------------- V conversion
      const int tid = threadIdx.x - kConvWarp * 32;
      // A thread's part of a V tile: chunk vc (16 codes) of rows vr, vr +
      // kRowStep, ..., whose addresses are constants apart. Codes 16 vc ..
      // become chunks 2 vc and 2 vc + 1 of the f16 rows (64-dim box vc / 4);
      // threads of odd boxes store their second chunk first, so that the
      // eight threads of a row use all banks.
      constexpr int kRowChunks = D / 16, kRowStep = 128 / kRowChunks, kPer = kN / kRowStep;
      constexpr int kFromStep = kRowStep * D, kToStep = kRowStep * D * 2;
      static_assert(kRowStep % 8 == 0, "whole 8-key groups between a thread's rows");
      const int vc = tid % kRowChunks, vr = tid / kRowChunks;
      const bool odd = (vc >> 2) & 1;
      const uint8_t* v_from = smem + C::kOffV8 + (vr >> 3) * C::kGroup8 + (vc >> 3) * 1024 +
                              (vr & 7) * 128 + (((vc & 7) ^ (vr & 7)) << 4);
      uint8_t* v_to =
          smem + C::kOffV16 + (vr >> 3) * C::kGroup16 + (vc >> 2) * 1024 + (vr & 7) * 128;
      const int at0 = ((((2 * vc) & 7) + odd) ^ (vr & 7)) << 4;
      const int at1 = ((((2 * vc) & 7) + 1 - odd) ^ (vr & 7)) << 4;
      uint32_t n = 0;
      for (int u = 0; it0 + u < it1 && !aborted; ++u) {
        const WorkItem w = items[it0 + u];
        const SeqInfo si = seqs[w.seq];
        const int npieces = w.kt1 - w.kt0;
        const int ntiles = (npieces + kPieces - 1) / kPieces;
        for (int t = 0; t < ntiles; ++t, ++n) {
          const uint32_t s8 = n % kV8Stages, s16 = n % kV16Stages;
          if (!wait_warp(&v8_full[s8], (n / kV8Stages) & 1u, flags, aborted)) break;
          if (!wait_warp(&v16_empty[s16], ((n / kV16Stages) & 1u) ^ 1u, flags, aborted)) break;
          const int valid = min(si.length - (w.kt0 + kPieces * t) * kTileTokens,
                                (npieces - kPieces * t) * kTileTokens);
          const uint8_t* from = v_from + s8 * C::kTile8;
          uint8_t* to = v_to + s16 * C::kTile16;
          if (valid >= kN) {
#pragma unroll 4
            for (int k = 0; k < kPer; ++k) {
              uint4 lo, hi, c = *reinterpret_cast<const uint4*>(from + k * kFromStep);
              if (odd) c = make_uint4(c.z, c.w, c.x, c.y);
              codes_to_h2(c, lo, hi);
              *reinterpret_cast<uint4*>(to + at0 + k * kToStep) = lo;
              *reinterpret_cast<uint4*>(to + at1 + k * kToStep) = hi;
            }
          } else {
#pragma unroll 1
            for (int k = 0; k < kPer; ++k) {
              uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
              if (vr + k * kRowStep < valid)
                codes_to_h2(*reinterpret_cast<const uint4*>(from + k * kFromStep), lo, hi);
              *reinterpret_cast<uint4*>(to + at0 + k * kToStep) = odd ? hi : lo;
              *reinterpret_cast<uint4*>(to + at1 + k * kToStep) = odd ? lo : hi;
            }
          }
          tc::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&v8_empty[s8]);
            mbar_arrive(&v16_full[s16]);
          }
        }
      }
      if (aborted && lane == 0) raise_device_error(a.err, FE_DEVERR_TIMEOUT);
    }
  } else {
    // ------------------------------------------------------------- softmax
    const int gi = warp >= 4 ? 1 : 0;
    const int quad = warp & 3;
    const int r = quad * 32 + lane;  // packed row = TMEM lane
    const uint32_t lane_addr = tmem + (uint32_t(quad * 32) << 16);
    const int G = a.G;
    const bool causal = view == 1;
    uint32_t n0 = 0;  // the item's first tile
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
      // the maximum this group's weight sum l refers to
      float m_used = -INFINITY, l = 0.f;
      for (int j = (gi ^ n0) & 1; j < ntiles; j += 2) {
        const uint32_t n = n0 + j;
        const int slot = n % kSlots;
        const uint32_t s_addr = lane_addr + slot * kN;
        const float4* fac = ring + (n % kExpRing) * 8;
        if (!wait_warp(&e_full[n % kExpRing], (n / kExpRing) & 1u, flags, aborted)) break;
        if (!wait_warp(&s_full[slot], (n / kSlots) & 1u, flags, aborted)) break;
        tc::fence_after_sync();
        const int tkey = (w.kt0 + kPieces * j) * kTileTokens;
        // Scores pass twice through registers, 32 keys at a time: for the
        // maximum, and for the weights. (All 128 at once need 200 registers
        // and four times the code; the instruction fetch of the kernel's many
        // kinds of warps then bounds it.)
        float mx = -INFINITY;
#pragma unroll 1
        for (int h = 0; h < kN; h += 32) {
          float s[32];
          tc::ld_32x32b_x32(s_addr + h, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
          tc::wait_ld();
          if (__any_sync(0xffffffffu, tkey + h + 32 > lim)) {
            // hidden keys become -inf, in TMEM too
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (tkey + h + c >= lim) s[c] = -INFINITY;
            tc::st_32x32b_x32(s_addr + h, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
          }
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const float* x = s + 16 * b;
            const float4 f = fac[h / 16 + b];
            const float m0 = fmax3(x[0], x[1], x[2]), m1 = fmax3(x[3], x[4], x[5]),
                        m2 = fmax3(x[6], x[7], x[8]), m3 = fmax3(x[9], x[10], x[11]),
                        m4 = fmax3(x[12], x[13], x[14]);
            mx = fmaxf(mx, fmaf(fmaxf(fmax3(m0, m1, m2), fmax3(m3, m4, x[15])), f.x * rf, f.y));
          }
        }
        tc::wait_st();
        // the maximum so far comes from the tile before and goes to the next;
        // it moves only when it grows by more than 2^8 (or from nothing)
        // (an item's first tile only waits, so that the group of the tile before
        // has read what this one overwrites)
        float m_prev = -INFINITY;
        if (n > 0) {
          if (!wait_warp(&max_bar[((n - 1) & 1) * 4 + quad], ((n - 1) >> 1) & 1u, flags, aborted))
            break;
          if (j > 0) m_prev = xmax[((n - 1) & 1) * kM + r];
        }
        const float m_top = fmaxf(m_prev, mx);
        const bool grow = m_top > m_prev + kRescale;
        const float m_now = grow ? m_top : m_prev;
        xmax[(n & 1) * kM + r] = m_now;
        __syncwarp();
        if (lane == 0) mbar_arrive(&max_bar[(n & 1) * 4 + quad]);
        if (m_now != m_used) {
          l *= fast_exp2(m_used - m_now);
          m_used = m_now;
        }
        if (j > 0 && __any_sync(0xffffffffu, grow)) {
          // wait for the last PV into O, then rescale it
          const float alpha = grow ? fast_exp2(m_prev - m_now) : 1.f;
          if (!wait_warp(&s_free[(n - 1) % kSlots], ((n - 1) / kSlots) & 1u, flags, aborted))
            break;
          tc::fence_after_sync();
#pragma unroll 1
          for (int c2 = 0; c2 < D / 16; ++c2) {
            uint32_t ov[16];
            tc::ld_32x32b_x16(lane_addr + C::kOCol + c2 * 16, ov);
            tc::wait_ld();
#pragma unroll
            for (int c = 0; c < 16; ++c) ov[c] = __float_as_uint(__uint_as_float(ov[c]) * alpha);
            tc::st_32x32b_x16(lane_addr + C::kOCol + c2 * 16, ov);
          }
        }
        const float m_ref = m_now == -INFINITY ? 0.f : m_now, m_sub = m_ref - kBias;
        // Scores so large that one fma with the maximum would leave a rounding
        // beyond a half's range (from |s| = 2^23 on): s + v rounded as in the
        // maximum, and the difference taken then. In a loop of its own, as small
        // as it gets: shared with the one below it cost 2 % of a call.
        if (__builtin_expect(__any_sync(0xffffffffu, fabsf(m_ref) > kFar), 0)) {
#pragma unroll 1
          for (int h = 0; h < kN; h += 16) {
            uint32_t s[16], pk[8];
            tc::ld_32x32b_x16(s_addr + h, s);
            tc::wait_ld();
            const float4 f = fac[h / 16];
            const float fs = f.x * rf;
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float w = fast_exp2(fmaf(__uint_as_float(s[e]), fs, f.y) - m_ref + kBias);
              sum += w;
              s[e] = __float_as_uint(w);
            }
            l = fmaf(sum, f.z, l);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              pk[e] = pack2<__half>(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]));
            tc::st_32x32b_x8(s_addr + h / 2, pk);
          }
        } else {
#pragma unroll 1
          for (int h = 0; h < kN; h += 32) {
            float s[32];
            tc::ld_32x32b_x32(s_addr + h, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
            tc::wait_ld();
            uint32_t pk[16];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const float4 f = fac[h / 16 + b];
              const float fs = f.x * rf, off = f.y - m_sub;
              const float2 sc2 = make_float2(fs, fs), off2 = make_float2(off, off);
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
                pk[8 * b + e] = pack2<__half>(pp.x, pp.y);
              }
              l = fmaf((sum0.x + sum0.y) + (sum1.x + sum1.y), f.z, l);
            }
            // (weights of 32 keys take 16 columns: never ones still to be read)
            tc::st_32x32b_x16(s_addr + h / 2, pk);
          }
        }
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[slot]);
      }
      if (aborted) break;
      n0 += ntiles;
      // this group's sum and the maximum it refers to, once the item before is
      // stored
      if (unit > 0 && !wait_warp(o_free, (unit - 1) & 1, flags, aborted)) break;
      xsum[gi * kM + r] = l;
      xsum[(2 + gi) * kM + r] = m_used;
      __syncwarp();
      if (lane == 0) mbar_arrive(l_done);
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
                                    cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<T, D>::kSmem);
  });
  if (attr_err != cudaSuccess) return cuda_fail(attr_err, "kv8_rows_kernel attribute");
  constexpr int kSmem = Cfg<T, D>::kSmem;
  FE_CUDA_TRY(launch_pdl(kv8_rows_kernel<T, D>, dim3(grid), dim3(kThreads), kSmem, stream, kmap,
                         vmap, args));
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
