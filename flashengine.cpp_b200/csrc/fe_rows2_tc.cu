// Row kernel of shared-prefix plans at head_dim 128: packed query rows against
// a KV head's keys on the 5th-generation tensor cores, two streams of scores a
// CTA.
//
// Reference behaviour: Cambridgebit/FlashEngine.cpp src/flashinfer_attention.cu:35-44
// (multi-row requests of a paged kernel) with the arithmetic of
// src/portable_gpu_ops.cpp:39-44.
//
// The mathematics is that of fe_prefill_tc.cu: S = Q K^T, an online base-2
// softmax with a lazy rescale, O += P V with P as a 16-bit high part and its
// 16-bit residual. What differs is the shape of the work. There the two softmax
// groups share the rows of one 128-row tile, trade their half-row maxima every
// tile, and one O serves both. Here every group has a stream of its own: its S,
// its O, one thread a row over all 128 keys of a tile, nothing to trade while
// keys remain. The tensor pipe alternates between the streams,
//     P V of stream 0, its next S, P V of stream 1, its next S, ...
// so that one group exponentiates while the other's products run.
//  * An item of more than 128 rows (up to 256) gives each stream 128 of them;
//    every K and V tile is loaded once for both.
//  * An item of up to 128 rows gives both streams the same rows and each half of
//    every tile's keys; at its end the streams' states are joined: both groups
//    read both O's (warps q and q + 4 own the same TMEM lanes), each half of the
//    dims.
// A 256-row item's 128-key tile costs 2 S and 4 P V products of 128 x 128 x 128,
// about 3100 cycles of the tensor pipe; a group's softmax of a tile (16384
// exponentials on one SM's 16 a cycle, packed arithmetic beside them) hides
// behind the other's 1550.
//
// One persistent CTA per SM, three warpgroups:
//  warps 0-3, 4-7  softmax of stream 0 and 1;
//  warps 8 / 11    producers of K (and Q) / of V: eight 16-token page pieces a
//                  tile, one TMA box each, into 2 K and 2 V stages of 32 KiB
//                  (S runs two steps ahead, so that a K stage is refilled two
//                  before it is read);
//  warps 9 / 10    issue of a stream's S and P V products (one elected thread
//                  each); warp 9 owns the TMEM.
// All hand-offs are mbarriers; every wait is bounded.
#include "fe_attn_common.cuh"
#include "fe_tcgen05.cuh"

namespace fe {

int rows2_launch(int dtype, const CUtensorMap& kmap, const CUtensorMap& vmap,
                 const CUtensorMap& qmap, const void* args, int grid, cudaStream_t stream);

namespace {

constexpr int kD = kHeadDim;
constexpr int kM = 128;  // rows of a stream
constexpr int kN = 128;  // keys of a tile
constexpr int kHalf = kN / 2;
constexpr int kPieces = kN / kTileTokens;
constexpr int kKStages = 2, kVStages = 2, kQBufs = 2;
constexpr int kThreads = 12 * 32;
constexpr int kKWarp = 8, kMmaWarp = 9, kVWarp = 11;  // MMA: 9 and 10, a stream each
constexpr int kBoxes = kD / 64;
constexpr int kQBox = kM * 128;            // 128 rows x 64 dims
constexpr int kQBytes = kBoxes * kQBox;    // 32 KiB
constexpr int kPieceBytes = kTileTokens * kD * 2;
constexpr int kGroupBytes = 8 * kD * 2;
constexpr int kTile = kPieces * kPieceBytes;  // 32 KiB
constexpr int kOffK = kQBufs * kQBytes;
constexpr int kOffV = kOffK + kKStages * kTile;
constexpr int kOffOut = kOffV + kVStages * kTile;  // [softmax warp][32 rows][128 B]
constexpr int kOffX = kOffOut + 8 * 4096;         // [stream][m, l][row]
constexpr int kOffBar = kOffX + 2 * 2 * kM * 4;
// q_full[2], q_empty[2], k_full[2], k_empty[2], v_full[2], v_empty[2],
// s_full[2][2], pv_done[2][2], p_full[2][2], o_full[2], o_free[2], x_full, drain
constexpr int kBars = 4 + 2 * kKStages + 2 * kVStages + 16 + 2;
constexpr int kSmem = kOffBar + kBars * 8 + 32;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kOCol = 2 * kN;  // O of stream i at kOCol + i * 128
constexpr float kRescaleThreshold = 8.f;
static_assert(kSmem <= 232448, "shared memory budget");

template <typename T>
struct Fmt;
template <>
struct Fmt<__half> {
  static constexpr int v = 0;
};
template <>
struct Fmt<__nv_bfloat16> {
  static constexpr int v = 1;
};

template <typename T>
__device__ __forceinline__ float2 hi_as_float(uint32_t h);
template <>
__device__ __forceinline__ float2 hi_as_float<__nv_bfloat16>(uint32_t h) {
  return make_float2(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 hi_as_float<__half>(uint32_t h) {
  return unpack2<__half>(h);
}

// Bounded wait of a whole warp, a barrier a lane (shared-memory addresses):
// false when one did not complete within kWaitLimitNs, or another warp gave up,
// so that every warp of the CTA winds down. Time is looked at every 4096 polls
// only: a poll that fails suspends the warp for a while anyway.
__device__ __forceinline__ bool poll(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

__device__ __noinline__ bool give_up(uint64_t& since, volatile int* flags) {
  const uint64_t now = global_ns();
  if (since == 0) since = now;
  if (now - since > kWaitLimitNs) *flags = 1;
  return __any_sync(0xffffffffu, *flags != 0);
}

__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* flags,
                                          bool& aborted) {
  uint64_t since = 0;
  uint32_t n = 0;
  while (!__all_sync(0xffffffffu, poll(bar, parity))) {
    if ((++n & 4095u) == 0 && give_up(since, flags)) {
      aborted = true;
      return false;
    }
  }
  return true;
}

// Bounded wait of one thread.
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile int* flags,
                                              bool& aborted) {
  if (aborted) return false;
  if (!wait_bounded_short(bar, parity, flags)) aborted = true;
  return !aborted;
}

// The same value in every lane, known as such to the compiler.
__device__ __forceinline__ int uniform(int x) { return __reduce_max_sync(0xffffffffu, x); }

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(p));
  return p != 0;
}

// What all roles derive from an item. A stream walks it in steps of 64 keys: both
// halves of every tile of a pair, else the stream's half of every tile.
struct Shape {
  int pieces, tiles;
  bool pair;  // two row tiles
  __device__ __forceinline__ explicit Shape(const WorkItem& w)
      : pieces(w.kt1 - w.kt0), tiles((pieces + kPieces - 1) / kPieces),
        pair(w.nrb * kRowBlock > kM) {}
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    paged_rows2_kernel(const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap,
                       const __grid_constant__ CUtensorMap qmap, const AttnArgs<T> a) {
  extern __shared__ __align__(16) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBar);
  uint64_t* q_full = bars;
  uint64_t* q_empty = q_full + 2;
  uint64_t* k_full = q_empty + 2;
  uint64_t* k_empty = k_full + kKStages;
  uint64_t* v_full = k_empty + kKStages;
  uint64_t* v_empty = v_full + kVStages;
  // [stream * 2 + slot]: a stream's steps take its two slots in turn
  uint64_t* s_full = v_empty + kVStages;  // S written
  uint64_t* pv_done = s_full + 4;         // P V done
  uint64_t* p_full = pv_done + 4;          // P written, O rescaled
  uint64_t* o_full = p_full + 4;          // [stream]: the item's last P V done
  uint64_t* o_free = o_full + 2;          // [stream]: O read
  uint64_t* x_full = o_free + 2;          // both streams' (m, l) written
  uint64_t* drain = x_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBars);
  volatile int* flags = reinterpret_cast<volatile int*>(tmem_slot + 2);
  auto at = [&](const uint64_t* bar) { return smem_u32(bar); };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const MetaHeader* hdr = reinterpret_cast<const MetaHeader*>(a.meta);
  const int view = a.view;
  int it0 = 0, it1 = 0;
  if (static_cast<int>(blockIdx.x) < hdr->grid[view]) {
    const int32_t* cta_off = reinterpret_cast<const int32_t*>(a.meta + hdr->cta_off_off[view]);
    it0 = cta_off[blockIdx.x];
    it1 = cta_off[blockIdx.x + 1];
  }
  if (it0 >= it1) {  // nothing to do, but not before the grid ahead is done
    pdl_wait();
    return;
  }
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) raise_device_error(a.err, FE_DEVERR_SMEM_ALIGN);
    pdl_wait();
    return;
  }
  const WorkItem* items = reinterpret_cast<const WorkItem*>(a.meta + hdr->items_off[view]);
  const SeqInfo* seqs = reinterpret_cast<const SeqInfo*>(a.meta + hdr->seqs_off);
  const int32_t* pages = reinterpret_cast<const int32_t*>(a.meta + hdr->pages_off);

  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(&q_full[b], 1);
      mbar_init(&q_empty[b], 2);  // as k_empty and v_empty: one commit per stream
      for (int h = 2 * b; h < 2 * b + 2; ++h) {
        mbar_init(&s_full[h], 1);
        mbar_init(&pv_done[h], 1);
        mbar_init(&p_full[h], 4);  // one arrival per warp of the group
      }
      mbar_init(&o_full[b], 1);
      mbar_init(&o_free[b], 8);  // eight warps, or four that arrive twice
    }
    for (int s = 0; s < kKStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 2);
    }
    for (int s = 0; s < kVStages; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 2);
    }
    mbar_init(x_full, 256);
    mbar_init(drain, 2);  // one commit per issuing warp
    flags[0] = 0;
    flags[1] = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tc::tmem_alloc(tmem_slot, kTmemCols);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  bool aborted = false;
  pdl_wait();  // q and the pools belong to earlier kernels until here
  // Only now: the key kernel, launched behind this one, starts beside it on the SMs
  // that this grid leaves free, and so behind whatever this grid has waited for.
  pdl_trigger();

  if (warp >= 8) {
    if (warp == kKWarp || warp == kVWarp) {
      // -------------------------------------------------------- producers
      const bool is_v = warp == kVWarp;
      const CUtensorMap* map = is_v ? &vmap : &kmap;
      uint64_t* full = is_v ? v_full : k_full;
      uint64_t* empty = is_v ? v_empty : k_empty;
      const int stages = is_v ? kVStages : kKStages;
      uint8_t* region = smem + (is_v ? kOffV : kOffK);
      // Q tiles by TMA when a tile is whole query rows (G divides 128) inside the
      // rows the Q map covers, else by the warp's lanes
      const bool q_tma = (kM % a.G) == 0 && a.q_map_rows > 0;
      if (lane == 0) {
        prefetch_tensormap(map);
        if (!is_v && q_tma) prefetch_tensormap(&qmap);
      }
      uint32_t g = 0, qn = 0;  // tiles loaded, Q tiles loaded
      for (int it = it0; it < it1 && !aborted; ++it) {
        const WorkItem w = items[it];
        const SeqInfo si = seqs[w.seq];
        const Shape sh(w);
        if (!is_v) {
          const int G = a.G, P = si.qrows * G;
          for (int x = 0; x < (sh.pair ? 2 : 1) && !aborted; ++x, ++qn) {
            // packed row p = query row p / G, head kvh*G + p % G: 128/G query rows x
            // G heads x 64 dims per box (rows past the sequence are other sequences'
            // q or zero fill; their output is never stored)
            const int b = qn % kQBufs;
            uint8_t* dst = smem + b * kQBytes;
            const int p0 = w.rb0 * kRowBlock + x * kM;
            const bool tma_tile =
                q_tma && si.q_row0 + (min(P, p0 + kM) - 1) / G < a.q_map_rows;
            int good = 1;
            if (lane == 0) {
              if (!wait_or_abort(&q_empty[b], ((qn / kQBufs) & 1u) ^ 1u, flags, aborted)) {
                good = 0;
              } else if (tma_tile) {
                mbar_arrive_expect_tx(&q_full[b], kQBytes);
#pragma unroll
                for (int y = 0; y < kBoxes; ++y)
                  tma_load_3d(dst + y * kQBox, &qmap, &q_full[b], 64 * y, w.kvh * G,
                              si.q_row0 + p0 / G);
              }
            }
            if (!__shfl_sync(0xffffffffu, good, 0)) {
              aborted = true;
              break;
            }
            if (!tma_tile) {
              // copied by the lanes into the swizzled K-major tile (zeros past the
              // sequence), then published
              constexpr int kChunks = kD / 8;
              for (int i = lane; i < kM * kChunks; i += 32) {
                const int r = i / kChunks, c = i % kChunks, pr = p0 + r;
                uint4 val = make_uint4(0, 0, 0, 0);
                if (pr < P)
                  val = __ldg(reinterpret_cast<const uint4*>(
                                a.q + (static_cast<int64_t>(si.q_row0 + pr / G) * a.hq +
                                       w.kvh * G + pr % G) * kD) + c);
                *reinterpret_cast<uint4*>(dst + (c >> 3) * kQBox + r * 128 +
                                          (((c & 7) ^ (r & 7)) << 4)) = val;
              }
              tc::fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) mbar_arrive(&q_full[b]);
            }
          }
        }
        // Slot of 16-token piece `i` of the item; lanes fetch 32 pieces at a time and
        // the next 32 are requested before they are needed.
        auto piece_slot = [&](int i) -> int {
          if (i >= sh.pieces) return 0;
          const int t0 = (w.kt0 + i) * kTileTokens;
          return __ldg(pages + si.page_off + t0 / a.page) * a.page + (t0 % a.page);
        };
        int cur = piece_slot(lane), nxt = piece_slot(32 + lane);
        for (int j = 0; j < sh.tiles && !aborted; ++j, ++g) {
          const int pb = (kPieces * j) & 31;
          if (j > 0 && pb == 0) {
            cur = nxt;
            nxt = piece_slot(kPieces * j + 32 + lane);
          }
          const int pieces = min(kPieces, sh.pieces - kPieces * j);
          const int st = g % stages;
          int sl[kPieces];
#pragma unroll
          for (int u = 0; u < kPieces; ++u) sl[u] = __shfl_sync(0xffffffffu, cur, pb + u);
          int good = 1;
          if (lane == 0) {
            if (!wait_or_abort(&empty[st], ((g / stages) & 1u) ^ 1u, flags, aborted)) {
              good = 0;
            } else {
              mbar_arrive_expect_tx(&full[st], pieces * kPieceBytes);
              uint8_t* dst = region + st * kTile;
#pragma unroll
              for (int u = 0; u < kPieces; ++u)
                if (u < pieces)
                  tma_load_4d(dst + u * kPieceBytes, map, &full[st], 0, 0, w.kvh * kBoxes,
                              sl[u] >> 3);
            }
          }
          if (!__shfl_sync(0xffffffffu, good, 0)) {
            aborted = true;
            break;
          }
        }
      }
      if (lane == 0) {
        if (aborted) raise_device_error(a.err, FE_DEVERR_TIMEOUT);
        // The last load into each buffer has landed before the CTA may exit
        // (consumed ones return at once; bounded for an aborted run).
        for (uint32_t t = g > uint32_t(stages) ? g - stages : 0; t < g; ++t)
          wait_bounded_short(&full[t % stages], (t / stages) & 1u, flags + 1);
        if (!is_v)
          for (uint32_t t = qn > kQBufs ? qn - kQBufs : 0; t < qn; ++t)
            wait_bounded_short(&q_full[t % kQBufs], (t / kQBufs) & 1u, flags + 1);
      }
    } else {
      // ------------------------------------------- MMA issuers, one a stream
      // A warp walks its stream's schedule whole and one elected thread issues:
      // descriptors and counters then stay in uniform registers (issued by one thread
      // under `lane == 0`, eight products took 700 to 1200 cycles of moving
      // descriptors where they run for 512). An event is the P V product of a step and,
      // behind it, the S of the step after the next, in the slot that it frees: MMAs of
      // one thread execute in order. All that an event waits for is polled at once, a
      // barrier a lane. Both streams wait for every Q, K and V tile and both release
      // it, whoever reads it: a barrier that a warp waits for is then never more than
      // one phase ahead of or behind it, which a wait by parity needs.
      const int i = warp - kMmaWarp;
      constexpr uint32_t idesc_s = tc::idesc_f16(Fmt<T>::v, false, false, kM, kHalf);
      constexpr uint32_t idesc_o = tc::idesc_f16(Fmt<T>::v, false, true, kM, kD);
      // Descriptors of the first buffers; the 14-bit start-address field (address >>
      // 4) is advanced by plain addition. K: K-major, 8-key groups kGroupBytes
      // apart, each next 64 dims at +1 KiB. V: MN-major, 64-dim boxes 1 KiB apart
      // (leading), 8-key groups kGroupBytes apart (stride), 16 keys per piece.
      const uint64_t q_desc0 = tc::smem_desc_sw128(smem_u32(smem), 16, 1024);
      const uint64_t k_desc0 = tc::smem_desc_sw128(smem_u32(smem + kOffK), 16, kGroupBytes);
      const uint64_t v_desc0 = tc::smem_desc_sw128(smem_u32(smem + kOffV), 1024, kGroupBytes);
      const uint32_t tm = uniform(tmem);
      const uint32_t s_col = tm + i * kN, o_col = tm + kOCol + i * kD;
      const uint32_t b_qf = at(q_full), b_kf = at(k_full), b_vf = at(v_full),
                     b_of = at(o_free + i), b_pf = at(p_full + 2 * i);
      const int i0 = uniform(it0), i1 = uniform(it1);
      uint32_t base = 0, qn = 0, gs = 0;  // tiles, Q tiles and steps before the item
      int unit = 0;
      for (int it = i0; it < i1 && !aborted; ++it, ++unit) {
        const Shape loaded(items[it]);
        const int tiles = uniform(loaded.tiles);
        const int pair = uniform(loaded.pair ? 1 : 0);
        const int steps = tiles << pair;
        const uint32_t qb = (qn + (pair ? i : 0)) % kQBufs;
        const uint64_t q_desc = q_desc0 + uint64_t((qb * kQBytes) >> 4);
#pragma unroll 1
        for (int e = -2; e < steps; ++e) {
          const bool next = e + 2 < steps;
          const uint32_t g = gs + e + 2, slot = g & 1u;  // of the step e + 2, and of e
          const uint32_t vg = base + (e >> pair), vst = vg % kVStages;
          const uint32_t kg = base + ((e + 2) >> pair), kst = kg % kKStages;
          const int vhalf = pair ? e & 1 : i;  // a pair's steps e and e + 2: the same half
          uint32_t bar = b_kf + 8 * kst;
          uint32_t parity = (kg / kKStages) & 1u;
          if (e < 0) {  // the item's first two S
            if (!next) continue;
            if (lane >= 1 && lane <= 1 + pair) {
              const uint32_t qt = qn + lane - 1;
              bar = b_qf + 8 * (qt % kQBufs);
              parity = (qt / kQBufs) & 1u;
            }
          } else if (lane == 1) {
            bar = b_vf + 8 * vst;
            parity = (vg / kVStages) & 1u;
          } else if (lane == 2 && unit > 0) {
            // O belongs to the softmax groups until they have stored the last item
            bar = b_of;
            parity = (unit - 1) & 1u;
          } else if (lane != 3 || !next) {
            bar = b_pf + 8 * slot;
            parity = ((g - 2) >> 1) & 1u;
          }
          if (!wait_warp(bar, parity, flags, aborted)) break;
          tc::fence_after_sync();
          const uint32_t p_col = s_col + slot * kHalf;
          const uint64_t vh =
              v_desc0 + uint64_t((vst * kTile + vhalf * (kPieces / 2) * kPieceBytes) >> 4);
          const uint64_t kh =
              k_desc0 + uint64_t((kst * kTile + vhalf * (kPieces / 2) * kPieceBytes) >> 4);
          const uint32_t more = e > 0 ? 1u : 0u;
          if (elect_one()) {
            if (e >= 0) {  // O += P V of the step
#pragma unroll
              for (int part = 0; part < 2; ++part)
#pragma unroll
                for (int kk = 0; kk < kHalf / 16; ++kk)
                  tc::mma_f16_ts(o_col, p_col + part * (kHalf / 2) + kk * 8,
                                 vh + uint64_t((kk * kPieceBytes) >> 4), idesc_o,
                                 part + kk == 0 ? more : 1u);
              tc::commit(&pv_done[2 * i + slot]);
              if (!pair || vhalf) tc::commit(&v_empty[vst]);
              if (e + 1 == steps) tc::commit(&o_full[i]);
            }
            if (next) {  // S of the step after the next
#pragma unroll
              for (int kk = 0; kk < kD / 16; ++kk) {
                const int box = kk >> 2, ko = (kk & 3) * 32;
                tc::mma_f16(p_col, q_desc + uint64_t((box * kQBox + ko) >> 4),
                            kh + uint64_t((box * 1024 + ko) >> 4), idesc_s, kk > 0 ? 1u : 0u);
              }
              tc::commit(&s_full[2 * i + slot]);
              if (!pair || vhalf) tc::commit(&k_empty[kst]);
              if (e + 3 == steps) {
                tc::commit(&q_empty[qn % kQBufs]);
                if (pair) tc::commit(&q_empty[(qn + 1) % kQBufs]);
              }
            }
          }
          __syncwarp();
        }
        base += tiles;
        qn += 1 + pair;
        gs += steps;
      }
      if (aborted && lane == 0) raise_device_error(a.err, FE_DEVERR_TIMEOUT);
      // TMEM is released only after every MMA issued here has completed.
      if (elect_one()) tc::commit(drain);
      __syncwarp();
      wait_bounded_short(drain, 0, flags + 1);
    }
  } else {
    // -------------------------------------------------- softmax / epilogue
    const int gi = warp >= 4 ? 1 : 0;  // the group's stream
    const int quad = warp & 3;
    const int r = quad * 32 + lane;  // row of the tile = TMEM lane
    const uint32_t lane_addr = tmem + (uint32_t(quad * 32) << 16);
    const uint32_t s_addr = lane_addr + gi * kN;
    const uint32_t o_addr = lane_addr + kOCol + gi * kD;
    const int G = a.G;
    uint32_t base = 0, gs = 0, nx = 0;  // tiles, steps and joined items before this one
    int unit = 0;
    for (int it = it0; it < it1 && !aborted; ++it, ++unit) {
      const WorkItem w = items[it];
      const SeqInfo si = seqs[w.seq];
      const Shape sh(w);
      const int P = si.qrows * G;
      const int p0 = w.rb0 * kRowBlock;
      const int p = p0 + (sh.pair ? gi * kM : 0) + r;
      const bool row_valid = p < P;
      // keys this row sees in this item: the mask's (none for items of a prefix, key_mode
      // 2), cut at the end of the item's pieces
      int lim = view == 1 && w.key_mode == 0 && row_valid ? si.length - si.qrows + p / G + 1
                                                          : si.length;
      lim = min(lim, w.kt1 * kTileTokens);
      // m stays -inf until the first unmasked key (its weights are 0)
      float m = -INFINITY, l = 0.f;
      const int steps = sh.tiles << (sh.pair ? 1 : 0);
#pragma unroll 1
      for (int step = 0; step < steps; ++step) {
        const uint32_t g = gs + step, slot = g & 1u;
        const int kt = sh.pair ? step >> 1 : step, half = sh.pair ? step & 1 : gi;
        const int t0 = (w.kt0 + kPieces * kt) * kTileTokens + half * kHalf;
        if (!wait_warp(at(&s_full[2 * gi + slot]), (g >> 1) & 1u, flags, aborted)) break;
        tc::fence_after_sync();
        const uint32_t half_addr = s_addr + slot * kHalf;
        float s[kHalf];
#pragma unroll
        for (int x = 0; x < kHalf; x += 32)
          tc::ld_32x32b_x32(half_addr + x, *reinterpret_cast<uint32_t(*)[32]>(&s[x]));
        tc::wait_ld();
        const int room = lim - t0;  // keys that the row sees here
        if (room < kHalf) {
#pragma unroll
          for (int x = 0; x < kHalf; ++x)
            if (x >= room) s[x] = -INFINITY;
        }
        float mx8[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) mx8[e] = fmax3(s[e], s[8 + e], s[16 + e]);
#pragma unroll
        for (int x = 24; x < kHalf - 8; x += 16)
#pragma unroll
          for (int e = 0; e < 8; ++e) mx8[e] = fmax3(mx8[e], s[x + e], s[x + 8 + e]);
#pragma unroll
        for (int e = 0; e < 8; ++e) mx8[e] = fmaxf(mx8[e], s[kHalf - 8 + e]);
        const float mx = fmaxf(fmax3(mx8[0], mx8[1], mx8[2]),
                               fmax3(fmax3(mx8[3], mx8[4], mx8[5]), mx8[6], mx8[7]));
        const float m_new = fmaxf(m, mx * a.scale_log2);
        // lazily: O and l keep the old maximum until it grew by 2^8 (true for a row's
        // first finite maximum too)
        const bool grow = m_new > m + kRescaleThreshold;
        if (__any_sync(0xffffffffu, grow)) {
          const float alpha = grow ? fast_exp2(m - m_new) : 1.f;
          if (step > 0) {
            // the P V before this one has completed (its slot's earlier one had before this
            // slot's S: the barrier is at most one phase short)
            if (!wait_warp(at(&pv_done[2 * gi + (slot ^ 1)]), ((g - 1) >> 1) & 1u, flags, aborted))
              break;
            tc::fence_after_sync();
#pragma unroll 1
            for (int c2 = 0; c2 < kD / 16; ++c2) {
              float ov[16];
              tc::ld_32x32b_x16(o_addr + c2 * 16, *reinterpret_cast<uint32_t(*)[16]>(&ov[0]));
              tc::wait_ld();
#pragma unroll
              for (int x = 0; x < 16; ++x) ov[x] *= alpha;
              tc::st_32x32b_x16(o_addr + c2 * 16, *reinterpret_cast<uint32_t(*)[16]>(&ov[0]));
            }
          }
          l *= alpha;
          if (grow) m = m_new;
        }
        const float m_sub = m == -INFINITY ? 0.f : m;
        // V rows of this half past the sequence end or past the loaded pieces are zeroed
        // (the pool may hold NaN there; unloaded rows hold an older tile). The stage's
        // earlier tile landed before the P V that made room for this S, so its full
        // barrier is at most one phase short of this tile's.
        const int valid = min(si.length - t0, (sh.pieces - kPieces * kt) * kTileTokens - half * kHalf);
        if (valid < kHalf) {
          const uint32_t vg = base + kt;
          const int st = vg % kVStages;
          if (!wait_warp(at(&v_full[st]), (vg / kVStages) & 1u, flags, aborted)) break;
          uint8_t* vb = smem + kOffV + st * kTile;
          const int r0 = max(valid, 0), nch = (kHalf - r0) * 8;  // 16-byte chunks per box
#pragma unroll 1
          for (int i = r; i < kBoxes * nch; i += kM) {
            const int box = i / nch, rem = i % nch;
            const int row = half * kHalf + r0 + rem / 8, ch = rem % 8;
            *reinterpret_cast<uint4*>(vb + (row >> 3) * kGroupBytes + box * 1024 +
                                      (row & 7) * 128 + (ch << 4)) = make_uint4(0, 0, 0, 0);
          }
          tc::fence_proxy_async_smem();
        }
        // P = exp2(S * scale - m) over its own S columns: the 16-bit high part in the
        // first 32, the residual in the others
        float2 l4[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f),
                        make_float2(0.f, 0.f)};
        const float2 sc2 = make_float2(a.scale_log2, a.scale_log2);
        const float2 nm2 = make_float2(-m_sub, -m_sub);
#pragma unroll
        for (int h = 0; h < kHalf / 32; ++h) {  // 32 keys -> 16 high + 16 residual columns
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 x = fma2(make_float2(s[32 * h + 2 * e], s[32 * h + 2 * e + 1]), sc2, nm2);
            const float2 pp = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            l4[e & 3] = add2(l4[e & 3], pp);
            hi[e] = pack2<T>(pp.x, pp.y);
            const float2 res = sub2(pp, hi_as_float<T>(hi[e]));
            lo[e] = pack2<T>(res.x, res.y);
          }
          tc::st_32x32b_x16(half_addr + 16 * h, hi);
          tc::st_32x32b_x16(half_addr + kHalf / 2 + 16 * h, lo);
        }
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * gi + slot]);
        l += ((l4[0].x + l4[0].y) + (l4[1].x + l4[1].y)) +
             ((l4[2].x + l4[2].y) + (l4[3].x + l4[3].y));
      }
      gs += steps;
      if (aborted) break;
      base += sh.tiles;
      const int rows_rec = min(P - p0, w.nrb * kRowBlock);
      float* rec = w.part >= 0 ? a.partials + w.part : nullptr;
      // What a thread holds of its row, 128 bytes at `x`, goes through shared memory (16-
      // byte chunks swizzled by the row), so that a store of the warp covers whole
      // lines of four rows and not a piece of 32 (5 us an item before). `dst` is row 0's
      // place of the warp; rows [0, live) are stored.
      uint8_t* stage = smem + kOffOut + warp * 4096;
      const int wrow0 = p0 + (sh.pair ? gi * kM : 0) + quad * 32;  // the warp's first packed row
      const int live = min(32, P - wrow0);
      auto put = [&](const uint4 (&x)[8], auto&& dst) {
        __syncwarp();
#pragma unroll
        for (int v = 0; v < 8; ++v)
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((v ^ (lane & 7)) << 4)) = x[v];
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const int row = 4 * q + (lane >> 3), c = lane & 7;
          const uint4 y =
              *reinterpret_cast<const uint4*>(stage + row * 128 + ((c ^ (row & 7)) << 4));
          if (row < live) *reinterpret_cast<uint4*>(dst(row) + c * 16) = y;
        }
      };
      // Dims dim0 .. +31, unscaled, to the record.
      auto put_record = [&](int dim0, const float (&o)[32]) {
        uint4 x[8];
#pragma unroll
        for (int v = 0; v < 8; ++v)
          x[v] = make_uint4(__float_as_uint(o[4 * v]), __float_as_uint(o[4 * v + 1]),
                            __float_as_uint(o[4 * v + 2]), __float_as_uint(o[4 * v + 3]));
        put(x, [&](int row) {
          return reinterpret_cast<uint8_t*>(
              rec + static_cast<int64_t>(wrow0 - p0 + row) * kD + dim0);
        });
      };
      // Dims dim0 .. +63 in 16 bits to the output.
      auto put_out = [&](int dim0, const uint4 (&x)[8]) {
        put(x, [&](int row) {
          const int pr = wrow0 + row;
          return reinterpret_cast<uint8_t*>(
              a.out + (static_cast<int64_t>(si.q_row0 + pr / G) * a.hq + w.kvh * G + pr % G) * kD +
              dim0);
        });
      };
      auto pack32 = [&](const float (&o)[32], float f, uint4* x) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[v].x = pack2<T>(o[8 * v + 0] * f, o[8 * v + 1] * f);
          x[v].y = pack2<T>(o[8 * v + 2] * f, o[8 * v + 3] * f);
          x[v].z = pack2<T>(o[8 * v + 4] * f, o[8 * v + 5] * f);
          x[v].w = pack2<T>(o[8 * v + 6] * f, o[8 * v + 7] * f);
        }
      };
      if (sh.pair) {
        if (!wait_warp(at(&o_full[gi]), unit & 1u, flags, aborted)) break;
        tc::fence_after_sync();
        if (rec && row_valid) {
          rec[rows_rec * kD + (p - p0)] = m;
          rec[rows_rec * (kD + 1) + (p - p0)] = l;
        }
        const float inv = 1.f / l;
#pragma unroll 1
        for (int c2 = 0; c2 < kD / 64; ++c2) {
          uint4 x[8];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float o[32];
            tc::ld_32x32b_x32(o_addr + c2 * 64 + h * 32,
                              *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
            tc::wait_ld();
            if (rec)
              put_record(c2 * 64 + h * 32, o);
            else
              pack32(o, inv, x + 4 * h);
          }
          if (!rec) put_out(c2 * 64, x);
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cnt(&o_free[gi], 2);
      } else {
        // join the streams: (m, l) through shared memory, then each group half of the
        // dims of both O's
        if (!wait_warp(at(&o_full[gi]), unit & 1u, flags, aborted)) break;
        // (the next item's write comes behind its o_full, which comes behind both
        // groups' o_free of this item: nobody still reads)
        float* x = reinterpret_cast<float*>(smem + kOffX);
        x[gi * 2 * kM + r] = m;
        x[gi * 2 * kM + kM + r] = l;
        mbar_arrive(x_full);
        if (!wait_warp(at(x_full), nx & 1u, flags, aborted)) break;
        ++nx;
        // (the other group has seen its stream's end: the phase is complete)
        if (!wait_warp(at(&o_full[gi ^ 1]), unit & 1u, flags, aborted)) break;
        tc::fence_after_sync();
        const float m0 = x[r], l0 = x[kM + r], m1 = x[2 * kM + r], l1 = x[3 * kM + r];
        const float mj = fmaxf(m0, m1), mb = mj == -INFINITY ? 0.f : mj;
        const float f0 = fast_exp2(m0 - mb), f1 = fast_exp2(m1 - mb);
        const float lj = l0 * f0 + l1 * f1;
        if (rec && row_valid && gi == 0) {
          rec[rows_rec * kD + r] = mj;
          rec[rows_rec * (kD + 1) + r] = lj;
        }
        const float inv = 1.f / lj;
        uint4 y[8];
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2) {
          const int dim0 = gi * 64 + c2 * 32;
          float o[32], o1[32];
          tc::ld_32x32b_x32(lane_addr + kOCol + dim0, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
          tc::ld_32x32b_x32(lane_addr + kOCol + kD + dim0,
                            *reinterpret_cast<uint32_t(*)[32]>(&o1[0]));
          tc::wait_ld();
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = o[c] * f0 + o1[c] * f1;
          if (rec)
            put_record(dim0, o);
          else
            pack32(o, inv, y + 4 * c2);
        }
        if (!rec) put_out(gi * 64, y);
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&o_free[0]);
          mbar_arrive(&o_free[1]);
        }
      }
    }
    if (aborted && lane == 0) raise_device_error(a.err, FE_DEVERR_TIMEOUT);
  }

  tc::fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
}

template <typename T>
int launch_t(const CUtensorMap& kmap, const CUtensorMap& vmap, const CUtensorMap& qmap,
             const void* args, int grid, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  FE_CUDA_TRY(allow_smem(paged_rows2_kernel<T>, kSmem, done));
  FE_CUDA_TRY(launch_pdl(paged_rows2_kernel<T>, dim3(grid), dim3(kThreads), kSmem, stream, kmap,
                         vmap, qmap, *static_cast<const AttnArgs<T>*>(args)));
  return FE_OK;
}

}  // namespace

int rows2_launch(int dtype, const CUtensorMap& kmap, const CUtensorMap& vmap,
                 const CUtensorMap& qmap, const void* args, int grid, cudaStream_t stream) {
  return dtype == FE_DTYPE_BF16
             ? launch_t<__nv_bfloat16>(kmap, vmap, qmap, args, grid, stream)
             : launch_t<__half>(kmap, vmap, qmap, args, grid, stream);
}

}  // namespace fe
