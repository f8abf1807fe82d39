// Paged decode attention over the 8-bit KV cache (sm_100a): sequences whose
// query rows x GQA group fit one 16-row block. No counterpart in the
// reference, whose pools are 16-bit; semantics as fe_attn_run (the arithmetic
// of Cambridgebit/FlashEngine.cpp src/portable_gpu_ops.cpp:39-44) over the
// cache's values code * 2^exponent.
//
// Mathematics. With s(t) the score in base-2 units, 2^v(t) the V scale of the
// token's block and m a running maximum of s + v (not of s), the kernel keeps
//   w(t) = 2^(s(t) + v(t) - m),  O = sum w(t) code_v(t),  l = sum w(t) 2^-v(t)
// and the output is O / l: V's scales cost one addition per 16 tokens, K's one
// factor per 16 tokens. Both products run on mma.m16n8k16 in f16 with fp32
// accumulation: the codes become halves, exactly, in registers (one conversion
// for two codes); queries are halves times a power of two per row (f16 as they
// are, bf16 exactly down to 2^-29 of the row's largest); weights are halves
// times 2^15, so that they keep 11 bits down to 2^-29 of the largest.
// mma.m16n8k32 on the codes themselves, with the other operand in two or three
// 8-bit parts, was built and measured first: on a B200 one takes 21 to 29
// clocks a warp and SM quarter when its operands change (the 16-bit one 10), a
// step of this kernel 3200 clocks, and it was bound by them and not by HBM.
//
// Roundings. A weight's 11 bits are fewer than the about 16 that the kernels
// over the 16-bit cache keep (a half and its residual): its share of the
// output moves by at most 2^-11, where a code of V holds its value to 2^-4 and
// an output in f16 is rounded to 2^-11 itself, and a second half would cost
// every PV product again. m refers to weight times V scale, so the 11 bits are
// there for weights down to 2^-29 of the row's largest such product, fewer
// below, none under 2^-40; l sums the unrounded weights in fp32.
//
// B200 design, as fe_decode.cu: bound by HBM traffic. One persistent CTA per
// SM with 8 consumer warps and a producer warp; an item is (sequence, group
// of H KV heads, range of 16-token tiles), a step is two tiles (32 tokens, the
// K of one PV product) of all H heads, fetched with one TMA box per tile for
// K and one for V into a ring of 128-192 KiB. The tiles' scale exponents are
// gathered by the producer's lanes a batch ahead and travel with the stage; a
// stage's loads go out before its exponents are stored, so that an item's
// first do not wait for them (64 sequences of 512 to 4096 keys: 47.0 -> 45.7
// us).
// Measured on a B200 with 8 KV heads of 128 dims, merge included: 64 bf16
// sequences of 2 to 32 Ki keys, 64 query heads, 219 us = 6.4 TB/s (0.98 of a
// device-to-device copy's rate); of 512 to 4096 keys, 32 heads, 44.7 us = 4.9
// TB/s (the rest: launch, first loads, the merge and the cut's ends); 4
// sequences of up to 1000 keys, 9.5 us (a chain of dependent latencies). Two KV
// heads of 256 dims, 16 heads, 512 to 4096 keys: 33 us = 3.4 TB/s.
// Nine warps leave 168 registers a thread, of which ptxas spills 96 to 112
// bytes at 128 dims, 72 at 256.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "fe_attn_common.cuh"
#include "fe_kv8_attn.h"
#include "fe_kv8_common.cuh"

namespace fe {
namespace {

constexpr int kConsumers = 8;
constexpr int kThreads = (kConsumers + 1) * 32;
constexpr int kStepTiles = 2;
constexpr int kStepTokens = kStepTiles * kTileTokens;
constexpr int kBoxBytes = kTileTokens * 128;  // 16 rows x 128 codes
constexpr float kWeightBits = 15.f;           // weights are kept times 2^15 (a half holds 2^16)
constexpr float kFar = 1 << 20;               // maxima of a unit of 2^-3 and more

// Warps of a CTA: group = (head, half of the packed rows), kWh = 8 / groups
// warps of a group take steps j, j + kWh, ...; the stage count is a multiple
// of kWh, so a stage's previous user among them is the warp itself and a
// parity wait can never be a phase ahead.
template <int H, int D>
struct Cfg {
  static constexpr int kBoxes = D / 128;
  static constexpr int kTileBytes = H * D * kTileTokens;        // one of K or V
  static constexpr int kStageBytes = 2 * kStepTiles * kTileBytes;
  static constexpr int kStages = (D == 128 && H == 8) ? 3 : (128 * 1024) / kStageBytes;
  static constexpr int kNT = D == 128 ? 2 : 1;                  // most 8-row column tiles a warp
  static constexpr int kSlotFloats = 8 * kNT * (D + 4);
  static constexpr int kCombBytes = H == 8 ? 0 : (kConsumers / 2) * kSlotFloats * 4;
  static constexpr int kExpOff = kStages * kStageBytes + kCombBytes;
  static constexpr int kExpBytes = 2 * kStepTiles * 8;          // [tile][K|V][8 heads]
  static constexpr int kBarOff = kExpOff + kStages * kExpBytes;
  static constexpr int kSmem = 1024 + kBarOff + 2 * kStages * 8 + 16;
  static_assert(kSmem <= 232448, "shared memory budget");
  static_assert(H == 8 || kStages % (kConsumers / H) == 0, "see above");
};

// 8*NT packed rows (columns of the products) of one KV head of D dims.
// Fragment layout: the tokens of a tile are the M side of S^T = K Q^T, dims
// the M side of O^T = V^T W^T. A 32-bit word of K holds dims 4cq .. 4cq + 3 of
// a 16-dim chunk (cq = lane % 4); its halves are k elements 2cq, 2cq + 1 and
// 2cq + 8, 2cq + 9 of a product over that chunk, and Q's words are picked to
// match. O row i of m-tile mt is dim 16 mt + 2 i (i < 8) or 16 mt + 2 (i - 8)
// + 1: the byte pairs that a transposed 16-bit load of 8-bit V delivers.
template <typename T, int NT, int D>
struct State {
  static constexpr int kMT = D / 16;  // 16-dim chunks: k-steps of S^T, m-tiles of O^T
  uint32_t qf[NT][kMT][2];
  float f[NT][2];  // base-2 score units per raw product, per column of this lane
  int lim[NT][2];
  int lim_min;
  float m[NT][2], l[NT][2];
  float o[NT][kMT][4];

  __device__ __forceinline__ void init(const T* q, int hq, const SeqInfo& si, int head0, int G,
                                       bool causal, float scale_log2, int key_end, int lane,
                                       int col0) {
    const int r8 = lane >> 2, cq = lane & 3;
    const int P = si.qrows * G;
    const int length = min(si.length, key_end);
    lim_min = length;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int p = col0 + nt * 8 + r8;
      const T* qp = p < P ? q + (static_cast<int64_t>(si.q_row0 + p / G) * hq + head0 + p % G) * D
                          : nullptr;
#pragma unroll
      for (int c = 0; c < kMT; ++c) {
        uint2 raw = make_uint2(0u, 0u);
        if (qp) raw = __ldg(reinterpret_cast<const uint2*>(qp + 16 * c + 4 * cq));
        qf[nt][c][0] = raw.x;
        qf[nt][c][1] = raw.y;
      }
      float mine = scale_log2;
      if constexpr (!std::is_same<T, __half>::value) {
        // into f16's range: the row's largest magnitude to [2^14, 2^15)
        float amax = 0.f;
#pragma unroll
        for (int c = 0; c < kMT; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float2 v = unpack2<T>(qf[nt][c][x]);
            if (fabsf(v.x) < INFINITY) amax = fmaxf(amax, fabsf(v.x));
            if (fabsf(v.y) < INFINITY) amax = fmaxf(amax, fabsf(v.y));
          }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // (at least 2^-60: products of smaller rows stay normal numbers)
        const int e = max((__float_as_int(amax) >> 23) - 14, 67);
        const float up = exp_scale(254 - e);
#pragma unroll
        for (int c = 0; c < kMT; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float2 v = unpack2<T>(qf[nt][c][x]);
            qf[nt][c][x] = pack2<__half>(v.x * up, v.y * up);
          }
        mine *= exp_scale(e);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        f[nt][c] = __shfl_sync(0xffffffffu, mine, (2 * cq + c) * 4);
        const int pc = col0 + nt * 8 + 2 * cq + c;
        lim[nt][c] = (causal && pc < P)
                         ? min(length, si.length - si.qrows + pc / G + 1) : length;
        lim_min = min(lim_min, lim[nt][c]);
        m[nt][c] = -INFINITY;
        l[nt][c] = 0.f;
      }
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt)
        o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.f;
    }
  }

  // One step: the 32 tokens from `tbase` on; ka, va: shared addresses of this
  // head's boxes of the first tile, the second tile's `tile_bytes` further;
  // ke, ve: the two tiles' scale exponents (clamped, biased); `length`: keys
  // of the item.
  __device__ __forceinline__ void step(uint32_t ka, uint32_t va, uint32_t tile_bytes,
                                       const int (&ke)[2], const int (&ve)[2], int tbase,
                                       int length, int lane) {
    const int r8 = lane >> 2, cq = lane & 3, mi = lane >> 3, li = lane & 7;
    // ---- S^T = K Q^T, the two tiles' products alternating
    float s[2][NT][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[u][nt][0] = s[u][nt][1] = s[u][nt][2] = s[u][nt][3] = 0.f;
    const uint32_t krow = ka + (li + ((mi & 1) << 3)) * 128;
#pragma unroll
    for (int c2 = 0; c2 < kMT / 2; ++c2) {
      const int c = 2 * c2 + (mi >> 1);  // 16-code chunk of the row, 8 per box
      const uint32_t at = krow + (c >> 3) * kBoxBytes + (((c & 7) ^ li) << 4);
      uint32_t w[2][4];  // tokens r8, r8 + 8 of chunk 2 c2, then of chunk 2 c2 + 1
#pragma unroll
      for (int u = 0; u < 2; ++u)
        ldmatrix_x4(at + u * tile_bytes, w[u][0], w[u][1], w[u][2], w[u][3]);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t af[4] = {e4m3x2_to_h2(w[u][2 * x]), e4m3x2_to_h2(w[u][2 * x + 1]),
                                  e4m3x2_hi_to_h2(w[u][2 * x]), e4m3x2_hi_to_h2(w[u][2 * x + 1])};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma_16816<__half>(s[u][nt], af, qf[nt][2 * c2 + x][0], qf[nt][2 * c2 + x][1]);
        }
    }
    // ---- hide keys past each column's limit
    if (tbase + kStepTokens > lim_min) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (tbase + u * kTileTokens + r8 + (e >> 1) * 8 >= lim[nt][e & 1])
              s[u][nt][e] = -INFINITY;
    }
    // ---- weights: columns are held by the 8 lanes with the same lane % 4
    const float kf[2] = {exp_scale(ke[0]), exp_scale(ke[1])};
    const float vf[2] = {float(ve[0] - 127), float(ve[1] - 127)};
    const float vi[2] = {exp_scale(254 - ve[0]), exp_scale(254 - ve[1])};
    float al[NT][2];
    bool moved = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; ++u)
          mx = fmaxf(mx, fmaf(fmaxf(s[u][nt][c], s[u][nt][2 + c]), kf[u] * f[nt][c], vf[u]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float mn = fmaxf(m[nt][c], mx);
        const float base = mn == -INFINITY ? 0.f : mn;
        moved |= mn > m[nt][c];
        al[nt][c] = fast_exp2(m[nt][c] - base);
        m[nt][c] = mn;
        float add = 0.f;
        // s + v rounded as in the maximum, and the difference taken then: at the
        // largest score it is 0 whatever the scores' size (one fma with v - base
        // would leave that sum's rounding, beyond a half's range from |s| = 2^23
        // on). At 256 dims only where it is needed: there the two additions take
        // 64 sequences of 512 to 4096 keys from 32.6 to 33.6 us, at 128 from 45.2
        // to 44.7.
        const bool apart = D == 128 || __any_sync(0xffffffffu, fabsf(base) > kFar);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float ft = kf[u] * f[nt][c], off = vf[u] + kWeightBits - base;
          float x0, x1;
          if (apart) {
            x0 = fmaf(s[u][nt][c], ft, vf[u]) - base + kWeightBits;
            x1 = fmaf(s[u][nt][2 + c], ft, vf[u]) - base + kWeightBits;
          } else {
            x0 = fmaf(s[u][nt][c], ft, off);
            x1 = fmaf(s[u][nt][2 + c], ft, off);
          }
          const float w0 = fast_exp2(x0), w1 = fast_exp2(x1);
          s[u][nt][c] = w0;
          s[u][nt][2 + c] = w1;
          add = fmaf(w0 + w1, vi[u], add);
        }
        l[nt][c] = fmaf(l[nt][c], al[nt][c], add);
      }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) {
          o[nt][mt][0] *= al[nt][0];
          o[nt][mt][1] *= al[nt][1];
          o[nt][mt][2] *= al[nt][0];
          o[nt][mt][3] *= al[nt][1];
        }
    }
    // ---- W^T as B fragments
    uint32_t bw[2][NT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          bw[u][nt][x] = movmatrix_trans(pack2<__half>(s[u][nt][2 * x], s[u][nt][2 * x + 1]));
    // ---- codes of V rows past the end are zeroed (anything may lie there,
    // and 0 * NaN would poison O): bytes of tokens 2cq and 2cq + 1, twice
    uint32_t vm[2][2] = {{0xffffffffu, 0xffffffffu}, {0xffffffffu, 0xffffffffu}};
    if (tbase + kStepTokens > length) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int t = tbase + u * kTileTokens + 8 * x + 2 * cq;
          vm[u][x] = (t < length ? 0x00ff00ffu : 0u) | (t + 1 < length ? 0xff00ff00u : 0u);
        }
    }
    // ---- O^T += V^T W^T, two m-tiles at a time
    const uint32_t vrow = va + (mi >> 1) * tile_bytes + (li + ((mi & 1) << 3)) * 128;
#pragma unroll
    for (int m0 = 0; m0 < kMT; m0 += 2) {
      uint32_t a[2][2][4];  // [m-tile][tile]
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int mt = m0 + i;
        uint32_t w[2][2];  // [tile][tokens 0-7, 8-15], dims 16 mt ..
        ldmatrix_x4_trans(vrow + (mt >> 3) * kBoxBytes + (((mt & 7) ^ li) << 4), w[0][0], w[0][1],
                          w[1][0], w[1][1]);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            // both tokens of the even dim, then both of the odd dim
            const uint32_t y = __byte_perm(w[u][x], 0, 0x3120) & vm[u][x];
            a[i][u][2 * x] = e4m3x2_to_h2(y);
            a[i][u][2 * x + 1] = e4m3x2_hi_to_h2(y);
          }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma_16816<__half>(o[nt][m0 + i], a[i][u], bw[u][nt][0], bw[u][nt][1]);
    }
  }

  __device__ __forceinline__ void reduce_l() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 4);
        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 8);
        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 16);
      }
  }

  // (O, m, l) of every column as merge rows of D + 4 floats; a column's dims
  // in order.
  __device__ __forceinline__ void stash(float* rows, int lane) const {
    const int r8 = lane >> 2, cq = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float* row = rows + (nt * 8 + 2 * cq + c) * (D + 4);
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
          *reinterpret_cast<float2*>(row + 16 * mt + 2 * r8) =
              make_float2(o[nt][mt][c], o[nt][mt][2 + c]);
        if (r8 == 0) {
          row[D] = m[nt][c];
          row[D + 1] = l[nt][c];
        }
      }
  }
  __device__ __forceinline__ void absorb(const float* rows, int lane) {
    const int r8 = lane >> 2, cq = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float* row = rows + (nt * 8 + 2 * cq + c) * (D + 4);
        const float mo = row[D], lo = row[D + 1];
        const float mn = fmaxf(m[nt][c], mo);
        const float base = mn == -INFINITY ? 0.f : mn;
        const float as = fast_exp2(m[nt][c] - base), ao = fast_exp2(mo - base);
        m[nt][c] = mn;
        l[nt][c] = l[nt][c] * as + lo * ao;
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) {
          const float2 x = *reinterpret_cast<const float2*>(row + 16 * mt + 2 * r8);
          o[nt][mt][c] = o[nt][mt][c] * as + x.x * ao;
          o[nt][mt][2 + c] = o[nt][mt][2 + c] * as + x.y * ao;
        }
      }
  }
};

template <typename T, int H, int D, int NT>
__device__ __forceinline__ void run_item(const Kv8Args<T>& ka, const WorkItem& wi,
                                         const SeqInfo& si, int halves, uint8_t* stages,
                                         const uint8_t* exps, uint64_t* full, uint64_t* empty,
                                         volatile int* flags, float* comb, int w, int lane,
                                         uint32_t& g, bool& aborted) {
  using C = Cfg<H, D>;
  const AttnArgs<T>& a = ka.a;
  const int G = a.G;
  const int P = si.qrows * G;
  const int groups = H * halves;
  const int kwh = kConsumers / groups;
  const int grp = w % groups, sub = w / groups;
  const int hh = grp % H, col0 = (grp / H) * 8;
  const int head0 = (wi.kvh + hh) * G;
  const int key_end = wi.kt1 * kTileTokens;
  State<T, NT, D> st;
  st.init(a.q, a.hq, si, head0, G, a.view == 1, a.scale_log2, key_end, lane, col0);
  const int length = min(si.length, key_end);

  const int nsteps = (wi.kt1 - wi.kt0 + kStepTiles - 1) / kStepTiles;
  for (int j = sub; j < nsteps; j += kwh) {
    const uint32_t gg = g + j;
    const int s = gg % C::kStages;
    if (aborted || flags[0] || !wait_bounded(&full[s], (gg / C::kStages) & 1u, flags)) {
      aborted = true;
      break;
    }
    const uint8_t* ex = exps + s * C::kExpBytes + hh;
    const int ke[2] = {exp_clamp(ex[0]), exp_clamp(ex[16])};
    const int ve[2] = {exp_clamp(ex[8]), exp_clamp(ex[24])};
    // stage: K tile 0, K tile 1, V tile 0, V tile 1, each [head][box][16 rows]
    const uint32_t base = smem_u32(stages + s * C::kStageBytes) + hh * C::kBoxes * kBoxBytes;
    st.step(base, base + kStepTiles * C::kTileBytes, C::kTileBytes, ke, ve,
            (wi.kt0 + j * kStepTiles) * kTileTokens, length, lane);
    __syncwarp();
    if (lane == 0) mbar_arrive_cnt(&empty[s], kwh);
  }
  g += nsteps;
  st.reduce_l();

  if constexpr (H < 8) {
    // fold the group's states pairwise: round `step` leaves warps 0..step-1
    constexpr int kSlot = C::kSlotFloats;
    for (int step = kwh >> 1; step >= 1; step >>= 1) {
      if (sub >= step && sub < 2 * step)
        st.stash(comb + ((sub - step) * groups + grp) * kSlot, lane);
      named_barrier_sync(1, kConsumers * 32);
      if (sub < step) st.absorb(comb + (sub * groups + grp) * kSlot, lane);
      named_barrier_sync(1, kConsumers * 32);
    }
  }
  if (sub != 0 || aborted) return;

  const int r8 = lane >> 2, cq = lane & 3;
  const int R = H * P;  // rows of the item's record: head-major, then packed row
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int p = col0 + nt * 8 + 2 * cq + c;
      if (p >= P) continue;
      if (wi.group < 0) {
        const float inv = 1.f / st.l[nt][c];
        T* dst = a.out + (static_cast<int64_t>(si.q_row0 + p / G) * a.hq + head0 + p % G) * D;
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt)
          *reinterpret_cast<uint32_t*>(dst + 16 * mt + 2 * r8) =
              pack2<T>(st.o[nt][mt][c] * inv, st.o[nt][mt][2 + c] * inv);
      } else {
        float* rec = a.partials + wi.part;
        float* row = rec + (hh * P + p) * D;
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt)
          *reinterpret_cast<float2*>(row + 16 * mt + 2 * r8) =
              make_float2(st.o[nt][mt][c], st.o[nt][mt][2 + c]);
        if (r8 == 0) {
          rec[R * D + hh * P + p] = st.m[nt][c];
          rec[R * (D + 1) + hh * P + p] = st.l[nt][c];
        }
      }
    }
}

template <typename T, int H, int D>
__global__ void __launch_bounds__(kThreads, 1)
    kv8_decode_kernel(const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap, const Kv8Args<T> ka) {
  using C = Cfg<H, D>;
  const AttnArgs<T>& a = ka.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* stages = smem;
  float* comb = reinterpret_cast<float*>(smem + C::kStages * C::kStageBytes);
  uint8_t* exps = smem + C::kExpOff;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* empty = full + C::kStages;
  volatile int* flags = reinterpret_cast<volatile int*>(empty + C::kStages);

  pdl_trigger();  // the merge kernel may be scheduled; it waits for this grid
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const MetaHeader* hdr = reinterpret_cast<const MetaHeader*>(a.meta);
  constexpr int kList = 2;  // decode work list
  // A CTA without work waits as well: a grid that ended before the one it
  // follows would let the next one start beside that.
  if (static_cast<int>(blockIdx.x) >= hdr->grid[kList]) {
    pdl_wait();
    return;
  }
  const int32_t* cta_off = reinterpret_cast<const int32_t*>(a.meta + hdr->cta_off_off[kList]);
  const WorkItem* items = reinterpret_cast<const WorkItem*>(a.meta + hdr->items_off[kList]);
  const SeqInfo* seqs = reinterpret_cast<const SeqInfo*>(a.meta + hdr->seqs_off);
  const int32_t* pages = reinterpret_cast<const int32_t*>(a.meta + hdr->pages_off);
  const int it0 = cta_off[blockIdx.x], it1 = cta_off[blockIdx.x + 1];
  if (it0 >= it1) {
    pdl_wait();
    return;
  }

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kConsumers);
    }
    flags[0] = 0;
    fence_barrier_init();
  }
  __syncthreads();

  if (warp == kConsumers) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      prefetch_tensormap(&kmap);
      prefetch_tensormap(&vmap);
    }
    // A lane looks after one tile of a batch of 32: its first slot (from the
    // page list, asked for two batches ahead) and the H + H exponents of its
    // block (one batch ahead).
    auto tile_slot = [&](const WorkItem& w, const SeqInfo& si, int j) -> int {
      if (j >= w.kt1) return 0;
      const int t0 = j * kTileTokens;
      return __ldg(pages + si.page_off + t0 / a.page) * a.page + (t0 % a.page);
    };
    struct Exps {
      uint64_t k, v;
    };
    auto tile_exps = [&](const WorkItem& w, int slot) -> Exps {
      const int64_t at = int64_t(slot / kKv8Block) * ka.hkv + w.kvh;
      Exps e;
      if constexpr (H == 8) {
        e.k = *reinterpret_cast<const uint64_t*>(ka.k_exp + at);
        e.v = *reinterpret_cast<const uint64_t*>(ka.v_exp + at);
      } else if constexpr (H == 4) {
        e.k = *reinterpret_cast<const uint32_t*>(ka.k_exp + at);
        e.v = *reinterpret_cast<const uint32_t*>(ka.v_exp + at);
      } else if constexpr (H == 2) {
        e.k = *reinterpret_cast<const uint16_t*>(ka.k_exp + at);
        e.v = *reinterpret_cast<const uint16_t*>(ka.v_exp + at);
      } else {
        e.k = ka.k_exp[at];
        e.v = ka.v_exp[at];
      }
      return e;
    };
    // The first two batches' slots of an item, and its first batch's exponents,
    // are asked for while the item before it streams (they are four dependent
    // loads). Page ids are the plan's metadata: the first item's are fetched
    // before waiting for the kernel that owns the pools.
    struct Head {
      WorkItem w;
      SeqInfo si;
      int slot, slot2;
      Exps e;
    };
    Head cur, next;
    auto head_slots = [&](int it, Head& h) {
      h.w = items[it];
      h.si = seqs[h.w.seq];
      h.slot = tile_slot(h.w, h.si, h.w.kt0 + lane);
      h.slot2 = tile_slot(h.w, h.si, h.w.kt0 + 32 + lane);
    };
    head_slots(it0, next);
    pdl_wait();
    next.e = tile_exps(next.w, next.slot);
    uint32_t g = 0;
    bool ok = true;
    for (int it = it0; it < it1 && ok; ++it) {
      cur = next;
      const int box = cur.w.kvh * C::kBoxes;
      // steps of this item to issue before looking at the next one
      int before = min(C::kStages, (cur.w.kt1 - cur.w.kt0 + kStepTiles - 1) / kStepTiles);
      for (int j0 = cur.w.kt0; j0 < cur.w.kt1 && ok; j0 += 32) {
        const int n = min(32, cur.w.kt1 - j0);
        const int slot = cur.slot;
        const Exps e = cur.e;
        cur.slot = cur.slot2;
        cur.e = tile_exps(cur.w, cur.slot);
        cur.slot2 = tile_slot(cur.w, cur.si, j0 + 64 + lane);
        for (int jj = 0; jj < n; jj += kStepTiles) {
          const int s0 = __shfl_sync(0xffffffffu, slot, jj);
          const int s1 = __shfl_sync(0xffffffffu, slot, jj + 1);
          const int s = g % C::kStages;
          int good = 1;
          if (lane == 0 && (flags[0] || !wait_bounded(&empty[s], ((g / C::kStages) & 1u) ^ 1u, flags)))
            good = 0;
          good = __shfl_sync(0xffffffffu, good, 0);
          if (!good) {
            ok = false;
            break;
          }
          // the loads first: the exponents of an item's first batch may still
          // be on their way
          if (lane == 0) {
            const int tiles = min(kStepTiles, n - jj);
            mbar_expect_tx(&full[s], tiles * 2 * C::kTileBytes);
            uint8_t* st = stages + s * C::kStageBytes;
            tma_load_3d(st, &kmap, &full[s], 0, s0, box);
            if (tiles == 2) tma_load_3d(st + C::kTileBytes, &kmap, &full[s], 0, s1, box);
            st += kStepTiles * C::kTileBytes;
            tma_load_3d(st, &vmap, &full[s], 0, s0, box);
            if (tiles == 2) tma_load_3d(st + C::kTileBytes, &vmap, &full[s], 0, s1, box);
          }
          if ((lane & ~1) == jj) {
            uint64_t* dst = reinterpret_cast<uint64_t*>(exps + s * C::kExpBytes + (lane & 1) * 16);
            dst[0] = e.k;
            dst[1] = e.v;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[s]);
          ++g;
          if (--before == 0 && it + 1 < it1) {
            head_slots(it + 1, next);
            next.e = tile_exps(next.w, next.slot);
          }
        }
      }
    }
    if (!ok && lane == 0) {
      raise_device_error(a.err, FE_DEVERR_TIMEOUT);
      flags[0] = 1;
      const uint32_t pending = g < C::kStages ? g : C::kStages;
      for (uint32_t k = 1; k <= pending; ++k) {
        const uint32_t gg = g - k;
        volatile int never = 0;
        (void)wait_bounded(&full[gg % C::kStages], (gg / C::kStages) & 1u, &never);
      }
    }
    return;
  }

  // -------------------------------------------------------------- consumers
  pdl_wait();  // q and the split workspace belong to earlier kernels until here
  uint32_t g = 0;
  bool aborted = false;
  WorkItem wi_next = items[it0];
  SeqInfo si_next = seqs[wi_next.seq];
  for (int it = it0; it < it1; ++it) {
    const WorkItem wi = wi_next;
    const SeqInfo si = si_next;
    if (it + 1 < it1) {  // in flight while this item runs
      wi_next = items[it + 1];
      si_next = seqs[wi_next.seq];
    }
    const bool many = si.qrows * a.G > 8;
    if constexpr (D == 128) {
      if (many)
        run_item<T, H, D, 2>(ka, wi, si, 1, stages, exps, full, empty, flags, comb, warp, lane, g,
                             aborted);
      else
        run_item<T, H, D, 1>(ka, wi, si, 1, stages, exps, full, empty, flags, comb, warp, lane, g,
                             aborted);
    } else {
      // 256 dims leave registers for 8 packed rows a warp: more are two groups
      run_item<T, H, D, 1>(ka, wi, si, many ? 2 : 1, stages, exps, full, empty, flags, comb, warp,
                           lane, g, aborted);
    }
  }
  if (aborted && lane == 0) raise_device_error(a.err, FE_DEVERR_TIMEOUT);
}

template <typename T, int H, int D>
int launch(const CUtensorMap& kmap, const CUtensorMap& vmap, const Kv8Args<T>& args, int grid,
           cudaStream_t stream) {
  using C = Cfg<H, D>;
  static std::once_flag once;
  static cudaError_t attr_err = cudaSuccess;
  std::call_once(once, [] {
    attr_err = cudaFuncSetAttribute(kv8_decode_kernel<T, H, D>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  if (attr_err != cudaSuccess) return cuda_fail(attr_err, "kv8_decode_kernel attribute");
  FE_CUDA_TRY(launch_pdl(kv8_decode_kernel<T, H, D>, dim3(grid), dim3(kThreads), C::kSmem, stream,
                         kmap, vmap, args));
  return FE_OK;
}

template <typename T>
int dispatch(int dim, int heads, const CUtensorMap& kmap, const CUtensorMap& vmap,
             const Kv8Args<T>& a, int grid, cudaStream_t stream) {
  if (dim == kWideHeadDim)
    return heads == 2 ? launch<T, 2, kWideHeadDim>(kmap, vmap, a, grid, stream)
                      : launch<T, 1, kWideHeadDim>(kmap, vmap, a, grid, stream);
  switch (heads) {
    case 8: return launch<T, 8, kHeadDim>(kmap, vmap, a, grid, stream);
    case 4: return launch<T, 4, kHeadDim>(kmap, vmap, a, grid, stream);
    case 2: return launch<T, 2, kHeadDim>(kmap, vmap, a, grid, stream);
    default: return launch<T, 1, kHeadDim>(kmap, vmap, a, grid, stream);
  }
}

// ---------------------------------------------------------------------------
// Merge of split units' records (O[rows][D], m[rows], l[rows], as in
// fe_decode.cu): out = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i.
// `per_row` warps of a block share a row, each taking every per_row-th piece
// with up to eight O vectors in flight, and join through shared memory: one
// long sequence has a record per CTA, and a warp that walked 128 of them alone
// took longer than the attention. per_row follows from the unit's pieces alone,
// not from the launch, so that the sums' order, and with it the bits, are the
// same for a plan of the host and one of the device with the same cuts.
// gridDim.x blocks stride over the units, gridDim.y over a unit's rows.
// ---------------------------------------------------------------------------
constexpr int kMergeWarps = 8;

// One warp a row up to eight pieces, then as many as leave each about eight.
// Whole calls in us on a B200 with always one, this rule, always eight:
// a sequence of 8192 keys 21.8, 9.9, 11.0; 64 of 512 to 4096 keys 45.7,
// 45.4, 52.6; a 1024-row chunk over 8192 keys 156.6, 156.3, 203.5.
__host__ __device__ __forceinline__ int merge_log2_warps(int pieces) {
  return (pieces > 8) + (pieces > 16) + (pieces > 32);
}
static_assert(kMergeWarps == 8, "merge_log2_warps");

template <typename T, int D>
__global__ void __launch_bounds__(kMergeWarps * 32)
    kv8_merge_kernel(const AttnArgs<T> a, int list) {
  constexpr int kV = D / 128;  // float4 per lane
  __shared__ float4 part[kMergeWarps][32 * kV];
  __shared__ float2 stat[kMergeWarps];
  pdl_trigger();
  // the metadata is older than the kernel that wrote the records
  const MetaHeader* hdr = reinterpret_cast<const MetaHeader*>(a.meta);
  const int n = hdr->n_groups[list];
  const SplitGroup* groups = reinterpret_cast<const SplitGroup*>(a.meta + hdr->groups_off[list]);
  const SeqInfo* seqs = reinterpret_cast<const SeqInfo*>(a.meta + hdr->seqs_off);
  SplitGroup g{};
  SeqInfo si{};
  if (static_cast<int>(blockIdx.x) < n) {
    g = groups[blockIdx.x];
    if (g.nsplit >= 2) si = seqs[g.seq];
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int lg = merge_log2_warps(g.nsplit), per_row = 1 << lg;
  int sub = warp & (per_row - 1), rows = kMergeWarps >> lg;
  pdl_wait();
  for (int u = blockIdx.x; u < n; u += gridDim.x) {
    if (u != static_cast<int>(blockIdx.x)) {
      g = groups[u];
      if (g.nsplit >= 2) si = seqs[g.seq];
      lg = merge_log2_warps(g.nsplit);
      per_row = 1 << lg;
      sub = warp & (per_row - 1);
      rows = kMergeWarps >> lg;
    }
    if (g.nsplit < 2) continue;  // placeholder ids of the row lists
    const int rph = g.rows_per_head > 0 ? g.rows_per_head : si.qrows * a.G;
    for (int r0 = blockIdx.y * rows; r0 < g.rows; r0 += gridDim.y * rows) {
      const int r = r0 + (warp >> lg);
      float M = -INFINITY, L = 0.f;
      float4 acc[kV];
#pragma unroll
      for (int v = 0; v < kV; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < g.rows) {
        const float* base = a.partials + g.part0;
        // the warp's pieces, 32 at a time: sub, sub + per_row, ..
        for (int s0 = sub; s0 < g.nsplit; s0 += 32 * per_row) {
          const int s = s0 + lane * per_row;
          float m = -INFINITY, l = 0.f;
          if (s < g.nsplit) {
            const float* rec = base + int64_t(s) * g.rec_floats;
            m = __ldcg(rec + g.rows * D + r);
            l = __ldcg(rec + g.rows * (D + 1) + r);
          }
          // the first O vectors are in flight with them
          constexpr int kPre = 8 / kV;
          const int count = min(32, (g.nsplit - s0 + per_row - 1) >> lg);
          float4 pre[kPre][kV];
#pragma unroll
          for (int j = 0; j < kPre; ++j)
            if (j < count) {
              const float* rec = base + int64_t(s0 + j * per_row) * g.rec_floats;
#pragma unroll
              for (int v = 0; v < kV; ++v)
                pre[j][v] = __ldcg(reinterpret_cast<const float4*>(rec + r * D + v * 128 + lane * 4));
            }
          float top = m;
#pragma unroll
          for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const float M_new = fmaxf(M, top);
          const float ref = M_new == -INFINITY ? 0.f : M_new;
          const float old = fast_exp2(M - ref);  // 0 from nothing
          const float w = fast_exp2(m - ref);
          float lw = l * w;
#pragma unroll
          for (int o = 16; o; o >>= 1) lw += __shfl_xor_sync(0xffffffffu, lw, o);
          L = fmaf(L, old, lw);
          M = M_new;
#pragma unroll
          for (int v = 0; v < kV; ++v) {
            acc[v].x *= old;
            acc[v].y *= old;
            acc[v].z *= old;
            acc[v].w *= old;
          }
          auto add = [&](const float4 (&x)[kV], float wj) {
#pragma unroll
            for (int v = 0; v < kV; ++v) {
              acc[v].x = fmaf(x[v].x, wj, acc[v].x);
              acc[v].y = fmaf(x[v].y, wj, acc[v].y);
              acc[v].z = fmaf(x[v].z, wj, acc[v].z);
              acc[v].w = fmaf(x[v].w, wj, acc[v].w);
            }
          };
#pragma unroll
          for (int j = 0; j < kPre; ++j) {
            const float wj = __shfl_sync(0xffffffffu, w, j);
            if (j < count) add(pre[j], wj);
          }
#pragma unroll 4
          for (int j = kPre; j < count; ++j) {
            const float* rec = base + int64_t(s0 + j * per_row) * g.rec_floats;
            float4 x[kV];
#pragma unroll
            for (int v = 0; v < kV; ++v)
              x[v] = __ldcg(reinterpret_cast<const float4*>(rec + r * D + v * 128 + lane * 4));
            add(x, __shfl_sync(0xffffffffu, w, j));
          }
        }
      }
      if (per_row > 1) {
#pragma unroll
        for (int v = 0; v < kV; ++v) part[warp][v * 32 + lane] = acc[v];
        if (lane == 0) stat[warp] = make_float2(M, L);
        __syncthreads();
        if (sub == 0) {
          float top = M;
          for (int k = 1; k < per_row; ++k) top = fmaxf(top, stat[warp + k].x);
          const float ref = top == -INFINITY ? 0.f : top;
          float w = fast_exp2(M - ref);
          L *= w;
#pragma unroll
          for (int v = 0; v < kV; ++v)
            acc[v] = make_float4(acc[v].x * w, acc[v].y * w, acc[v].z * w, acc[v].w * w);
          for (int k = 1; k < per_row; ++k) {
            w = fast_exp2(stat[warp + k].x - ref);
            L = fmaf(stat[warp + k].y, w, L);
#pragma unroll
            for (int v = 0; v < kV; ++v) {
              const float4 x = part[warp + k][v * 32 + lane];
              acc[v].x = fmaf(x.x, w, acc[v].x);
              acc[v].y = fmaf(x.y, w, acc[v].y);
              acc[v].z = fmaf(x.z, w, acc[v].z);
              acc[v].w = fmaf(x.w, w, acc[v].w);
            }
          }
        }
        __syncthreads();
      }
      if (sub == 0 && r < g.rows) {
        const float inv = 1.f / L;
        const int p = g.row0 + r % rph;
        T* dst = a.out + (static_cast<int64_t>(si.q_row0 + p / a.G) * a.hq +
                          (g.kvh + r / rph) * a.G + p % a.G) * D + lane * 4;
#pragma unroll
        for (int v = 0; v < kV; ++v)
          store4<T>(dst + v * 128, acc[v].x * inv, acc[v].y * inv, acc[v].z * inv,
                    acc[v].w * inv);
      }
    }
  }
}

template <typename T>
int merge_launch(int dim, int list, const AttnArgs<T>& a, int units, int rows, int pieces,
                 int max_blocks, cudaStream_t stream, bool pdl) {
  // blocks for the rows of the most split unit
  const int per_block = kMergeWarps >> merge_log2_warps(pieces);
  const dim3 grid(units, std::min((rows + per_block - 1) / per_block,
                                  std::max(1, max_blocks / units)));
  auto kernel = dim == kWideHeadDim ? kv8_merge_kernel<T, kWideHeadDim>
                                    : kv8_merge_kernel<T, kHeadDim>;
  if (pdl) {
    FE_CUDA_TRY(launch_pdl(kernel, grid, dim3(kMergeWarps * 32), 0, stream, a, list));
  } else {
    kernel<<<grid, kMergeWarps * 32, 0, stream>>>(a, list);
    FE_CUDA_TRY(cudaGetLastError());
  }
  return FE_OK;
}

}  // namespace

int kv8_merge_launch(int dtype, int dim, int list, const void* args, int units, int rows,
                     int pieces, int max_blocks, cudaStream_t stream, bool pdl) {
  if (units <= 0) return FE_OK;
  if (dtype == FE_DTYPE_BF16)
    return merge_launch(dim, list, *static_cast<const AttnArgs<__nv_bfloat16>*>(args), units, rows,
                        pieces, max_blocks, stream, pdl);
  return merge_launch(dim, list, *static_cast<const AttnArgs<__half>*>(args), units, rows, pieces,
                      max_blocks, stream, pdl);
}

int kv8_decode_launch(int dtype, int dim, int heads, const CUtensorMap& kmap,
                      const CUtensorMap& vmap, const void* args, int grid, cudaStream_t stream) {
  if (dtype == FE_DTYPE_BF16)
    return dispatch(dim, heads, kmap, vmap, *static_cast<const Kv8Args<__nv_bfloat16>*>(args),
                    grid, stream);
  return dispatch(dim, heads, kmap, vmap, *static_cast<const Kv8Args<__half>*>(args), grid,
                  stream);
}

}  // namespace fe
