// 8-bit KV cache operators around the attention: append (rotation,
// quantisation and scatter in one launch), gather of whole sequences back to
// 16 bits, and block copies of forked sequences. No counterpart in the
// reference, whose pools are 16-bit (src/cuda_model.cpp:60); slot semantics,
// rotation and roundings follow fe_kv_append / fe_rope.
#include <cstring>
#include <mutex>
#include <string>

#include "fe_kv8_common.cuh"

namespace fe {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kQHeads = 4;  // query heads per thread of an append

// Four values as two fp32 pairs.
struct Quad {
  float2 x, y;
};

// A rotation pair in fp32, each product and sum rounded separately as fe_rope
// does (the packed fp32 instructions were not: ptxas fused them).
__device__ __forceinline__ void rotate1(float& a, float& b, float c, float s) {
  const float x = a;
  a = __fsub_rn(__fmul_rn(x, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(x, s));
}
__device__ __forceinline__ void rotate4(Quad& a, Quad& b, const float* cos, const float* sin) {
  const float4 c = *reinterpret_cast<const float4*>(cos);
  const float4 s = *reinterpret_cast<const float4*>(sin);
  rotate1(a.x.x, b.x.x, c.x, s.x);
  rotate1(a.x.y, b.x.y, c.y, s.y);
  rotate1(a.y.x, b.y.x, c.z, s.z);
  rotate1(a.y.y, b.y.y, c.w, s.w);
}

template <typename T>
__device__ __forceinline__ Quad unpack4(uint2 v) {
  return Quad{unpack2<T>(v.x), unpack2<T>(v.y)};
}

__device__ __forceinline__ float max4(float m, const Quad& q) {
  return fmaxf(fmaxf(fmaxf(m, fabsf(q.x.x)), fmaxf(fabsf(q.x.y), fabsf(q.y.x))), fabsf(q.y.y));
}
// The same over finite values only.
__device__ __forceinline__ float max4_finite(float m, const Quad& q) {
  const float v[4] = {fabsf(q.x.x), fabsf(q.x.y), fabsf(q.y.x), fabsf(q.y.y)};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (v[i] < INFINITY) m = fmaxf(m, v[i]);
  return m;
}

__device__ __forceinline__ uint32_t codes4(const Quad& q, float inv) {
  const float2 s = make_float2(inv, inv);
  const float2 x = mul2(q.x, s), y = mul2(q.y, s);
  return e4m3x2(x.x, x.y) | e4m3x2(y.x, y.y) << 16;
}

// Biased exponent of the smallest power of two s with amax <= 448 s (448 is
// the largest e4m3 value, 1.75 * 2^8): amax's exponent less 8, one more when
// its mantissa is above 1.75; within the limits of an append.
__device__ __forceinline__ int needed_exp(float amax) {
  return exp_clamp(((__float_as_int(amax) + 0x1fffff) >> 23) - 8);
}

struct AppendArgs {
  const void* q;
  void* q_out;
  const void* k;
  const void* v;
  uint8_t* k_codes;
  uint8_t* v_codes;
  uint8_t* k_exp;
  uint8_t* v_exp;
  const int64_t* slots;
  const int64_t* pos;   // null when nothing is rotated
  const float* cache;
  int rows, hq, hkv, rot, max_positions;
  int64_t cache_slots;  // below 2^31
  int kv_blocks;        // blocks of the kv part; the rest rotate queries
  bool apart;           // its blocks take K and V in turn
  unsigned int* err;
};

// ---------------------------------------------------------------------------
// Append. Work of the kv part: a RUN, the adjacent rows whose slots lie in one
// scale block in increasing order (rows that are skipped do not end it), for
// one KV head, is one warp's: it takes the largest finite magnitude of the
// (rotated) values of K, and of V, joins each with the block's old exponent
// when earlier tokens are kept, and writes the codes; when a scale grows, the
// kept tokens' codes are rounded to the new one. So every (block, head) has
// one writer per call and nothing is atomic.
//
// A warp looks at a window of W rows for run starts (W = 1: a decode step
// gives each row its own warps; W = 16: a prompt's rows, whose runs are mostly
// whole blocks, are covered by one warp per 16 rows and head instead of 16
// warps of which 15 find nothing; W = 4 between them); a small step takes K and
// V by warps of their own. The 32 lanes read the slots of rows w - 1
// .. w + 30: the row before the window, the window, and what its last run can
// reach; only among skipped rows does a run need more (the two loops over
// rows). All of a run's K and V rows (8 KiB at head_dim 128) are in flight to
// shared memory before the first is used.
//
// The query part rotates q into q_out, a thread per (row, kQHeads heads, 4 + 4
// dims): the heads share the row's cos / sin.
// Both parts are bound by memory traffic on prompts and by a chain of three
// loads (slot and position, row and cos / sin, store) on decode steps.
// Measured on a B200, bf16, 32 query and 8 KV heads of 128 dims, all rotated:
// 64 Ki rows of 16 prompts 286 us = 5.3 TB/s (0.81 of a device-to-device copy's
// rate; 402 us with rows in registers and runs found by a warp a row); 64 rows
// of 64 sequences 3.5 us, 4 rows 3.2 us. Query and KV blocks in turn instead of
// one after the other, and KV rows held in fp32 registers, measured 305 and 342
// us against 301 and 290. 64 Ki rows of 16 query and 2 KV heads of 256 dims:
// 484 us = 2.8 TB/s, 0.42 of the copy's rate (a warp's stage of 16 KiB leaves
// one block an SM, and the query part is launched with it).
// ---------------------------------------------------------------------------

// The m-th row of a run: rows are adjacent and slots consecutive (dense), or
// lane m holds its row, its token of the block and its position.
struct Run {
  bool dense;
  int row0, len, kept, blk;
  int row_m, off_m, pos_m;
};

// A warp's staged rows of one head, [16][D]. Rows wait in shared memory and
// not in registers: the loops over them stay loops, and 24 warps an SM fit.
template <int D>
struct Stage {
  static constexpr int kBytes = kKv8Block * D * 2;
  static constexpr int kUnits = D / 8;     // a unit is 4 + 4 dims of a row
  static constexpr int kRows = 256 / D;    // rows per pass of a warp
};

template <int D>
__device__ __forceinline__ void stage_rows(uint8_t* to, const void* from, int hkv, int h,
                                           const Run& run, int lane) {
  using S = Stage<D>;
  const int sub = lane / S::kUnits, c = lane % S::kUnits;  // 16 bytes of a row
  const uint8_t* base = static_cast<const uint8_t*>(from) + (int64_t(h) * D + 8 * c) * 2;
  for (int i = 0; i < run.len; i += S::kRows) {
    const int t = i + sub;
    const int row = run.dense ? run.row0 + t : __shfl_sync(0xffffffffu, run.row_m, t & 31);
    if (t < run.len)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                       smem_u32(to + t * (D * 2) + 16 * c)),
                   "l"(base + int64_t(row) * hkv * (D * 2))
                   : "memory");
  }
}

// Quantise the staged rows into block run.blk of one head. kRot: `rot` dims
// are rotated (the lanes that `turn`). kFull: a whole block of adjacent rows,
// as most of a prompt's are, without the checks of the others (a third of the
// instructions, which are what bounds the kv part). Values are formed twice,
// for the maximum and for the codes.
template <typename T, int D, bool kRot, bool kFull>
__device__ __forceinline__ void quantise_rows(const uint8_t* stage, const Run& run,
                                              const float* cache, int rot, int e0, int e1,
                                              bool turn, uint8_t* codes, uint8_t* exps, int old,
                                              int hkv, int h, int lane) {
  using S = Stage<D>;
  constexpr int kRows = S::kRows, kStep = kFull ? 4 : 1;
  const int sub = lane / S::kUnits, u = lane % S::kUnits;
  const int len = kFull ? kKv8Block : run.len;
  const uint8_t* from = stage + sub * (D * 2);
  auto raw = [&](int i, uint2& lo, uint2& hi) {
    lo = *reinterpret_cast<const uint2*>(from + i * (D * 2) + 2 * e0);
    hi = *reinterpret_cast<const uint2*>(from + i * (D * 2) + 2 * e1);
  };
  auto values = [&](int i, Quad& a, Quad& b) {
    uint2 lo, hi;
    raw(i, lo, hi);
    a = unpack4<T>(lo);
    b = unpack4<T>(hi);
    if (kRot) {
      const int p = __shfl_sync(0xffffffffu, run.pos_m, (i + sub) & 31);
      if (turn && (kFull || i + sub < len)) {
        const float* at = cache + int64_t(p) * rot + e0;
        rotate4(a, b, at, at + rot / 2);
      }
    }
  };
  float amax = 0.f;
  if (kRot) {
#pragma unroll kStep
    for (int i = 0; i < len; i += kRows) {
      Quad a, b;
      values(i, a, b);
      if (kFull || i + sub < len) amax = max4(max4(amax, a), b);
    }
  } else {
    uint32_t m = 0;
#pragma unroll kStep
    for (int i = 0; i < len; i += kRows) {
      uint2 lo, hi;
      raw(i, lo, hi);
      if (kFull || i + sub < len)
        m = max_abs2(max_abs2(max_abs2(max_abs2(m, lo.x, T()), lo.y, T()), hi.x, T()), hi.y, T());
    }
    const float2 f = unpack2<T>(m);
    amax = fmaxf(f.x, f.y);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (amax == INFINITY) {  // infinities saturate: once more without them
    amax = 0.f;
#pragma unroll 1
    for (int i = 0; i < len; i += kRows) {
      Quad a, b;
      values(i, a, b);
      if (i + sub < len) amax = max4_finite(max4_finite(amax, a), b);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  }
  int e = needed_exp(amax);
  // the kept tokens' scale as every reader takes it: a byte outside the limits
  // is the nearest within
  const int was = exp_clamp(old);
  if (run.kept) e = max(e, was);
  const float inv = exp_scale(254 - e);
  const int64_t tok = int64_t(hkv) * D;  // bytes from one token to the next
  uint8_t* block = codes + int64_t(run.blk) * kKv8Block * tok + h * D;
  if (kFull) {
    uint8_t* dst = block + sub * tok;
#pragma unroll kStep
    for (int i = 0; i < len; i += kRows, dst += kRows * tok) {
      Quad a, b;
      values(i, a, b);
      *reinterpret_cast<uint32_t*>(dst + e0) = codes4(a, inv);
      *reinterpret_cast<uint32_t*>(dst + e1) = codes4(b, inv);
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < len; i += kRows) {
      const int t = i + sub;
      const int off = run.dense ? run.kept + t : __shfl_sync(0xffffffffu, run.off_m, t & 31);
      Quad a, b;
      values(i, a, b);
      if (t < len) {
        uint8_t* dst = block + off * tok;
        *reinterpret_cast<uint32_t*>(dst + e0) = codes4(a, inv);
        *reinterpret_cast<uint32_t*>(dst + e1) = codes4(b, inv);
      }
    }
  }
  if (run.kept && e > was) {
    // the kept tokens move to the larger scale: 8 codes per lane and pass
    const float down = exp_scale(was - e + 127);
    for (int t = sub; t < run.kept; t += kRows) {
      uint2* w = reinterpret_cast<uint2*>(block + t * tok) + u;
      uint2 c = *w;
      uint32_t* cw = &c.x;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 a = unpack2<__half>(e4m3x2_to_h2(cw[j]));
        const float2 b = unpack2<__half>(e4m3x2_hi_to_h2(cw[j]));
        cw[j] = e4m3x2(a.x * down, a.y * down) | e4m3x2(b.x * down, b.y * down) << 16;
      }
      *w = c;
    }
  }
  if (lane == 0 && (!run.kept || e != old))
    exps[int64_t(run.blk) * hkv + h] = static_cast<uint8_t>(e);
}

// do_k, do_v: one of them or both are this warp's.
template <typename T, int D, bool kFull>
__device__ __forceinline__ void append_run(const AppendArgs& a, const Run& run, int h, bool do_k,
                                           bool do_v, uint8_t* stage, int lane) {
  using S = Stage<D>;
  uint8_t* stage_v = stage + (do_k ? S::kBytes : 0);
  if (do_k) stage_rows<D>(stage, a.k, a.hkv, h, run, lane);
  asm volatile("cp.async.commit_group;" ::: "memory");
  if (do_v) stage_rows<D>(stage_v, a.v, a.hkv, h, run, lane);
  asm volatile("cp.async.commit_group;" ::: "memory");
  const int rot_units = a.rot / 8;
  const int u = lane % S::kUnits;
  const bool turn = u < rot_units;
  const int e0 = turn ? 4 * u : a.rot + 8 * (u - rot_units), e1 = e0 + (turn ? a.rot / 2 : 4);
  int old_k = 0, old_v = 0;
  if (run.kept) {
    old_k = a.k_exp[int64_t(run.blk) * a.hkv + h];
    old_v = a.v_exp[int64_t(run.blk) * a.hkv + h];
  }
  if (do_k) {
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    if (a.pos)
      quantise_rows<T, D, true, kFull>(stage, run, a.cache, a.rot, e0, e1, turn, a.k_codes,
                                       a.k_exp, old_k, a.hkv, h, lane);
    else
      quantise_rows<T, D, false, kFull>(stage, run, nullptr, 0, e0, e1, false, a.k_codes, a.k_exp,
                                        old_k, a.hkv, h, lane);
  }
  if (do_v) {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    quantise_rows<T, D, false, kFull>(stage_v, run, nullptr, 0, e0, e1, false, a.v_codes, a.v_exp,
                                      old_v, a.hkv, h, lane);
  }
  __syncwarp();  // the stage may be refilled
}

template <typename T, int D, int W>
__global__ void __launch_bounds__(kThreads, D == 128 ? 3 : 1) kv8_append_kernel(const AppendArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  pdl_trigger();
  pdl_wait();  // q, k, v come from, and the pools are read by, earlier kernels
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kUnits = D / 8;  // a unit is 4 + 4 dims of a head
  if (static_cast<int>(blockIdx.x) >= a.kv_blocks) {
    // ------------------------------------------------------------- queries
    const int r = a.rot / 2, rot_units = a.rot / 8;
    const int per_row = (a.hq + kQHeads - 1) / kQHeads * kUnits;
    const int64_t total = int64_t(a.rows) * per_row;
    const int64_t i =
        int64_t(blockIdx.x - a.kv_blocks) * kThreads + threadIdx.x;
    if (i < total) {
      const int row = static_cast<int>(i / per_row);
      const int rem = static_cast<int>(i - int64_t(row) * per_row);
      const int u = rem % kUnits, h0 = rem / kUnits * kQHeads;
      const bool turn = u < rot_units;
      const int e0 = turn ? 4 * u : a.rot + 8 * (u - rot_units), e1 = turn ? e0 + r : e0 + 4;
      const int64_t base = (int64_t(row) * a.hq + h0) * D;
      const T* src = static_cast<const T*>(a.q) + base;
      T* dst = static_cast<T*>(a.q_out) + base;
      uint2 lo[kQHeads], hi[kQHeads];
#pragma unroll
      for (int h = 0; h < kQHeads; ++h)
        if (h0 + h < a.hq) {
          lo[h] = *reinterpret_cast<const uint2*>(src + h * D + e0);
          hi[h] = *reinterpret_cast<const uint2*>(src + h * D + e1);
        }
      const float* cs = nullptr;
      if (a.pos) {
        const int64_t p = a.pos[row];
        if (p < 0 || p >= a.max_positions) {
          if (rem == 0) raise_device_error(a.err, FE_DEVERR_POS_RANGE);
          return;
        }
        if (turn) cs = a.cache + p * a.rot + e0;
      }
#pragma unroll
      for (int h = 0; h < kQHeads; ++h)
        if (h0 + h < a.hq) {
          if (cs) {
            Quad x = unpack4<T>(lo[h]), y = unpack4<T>(hi[h]);
            rotate4(x, y, cs, cs + r);
            lo[h] = make_uint2(pack2<T>(x.x.x, x.x.y), pack2<T>(x.y.x, x.y.y));
            hi[h] = make_uint2(pack2<T>(y.x.x, y.x.y), pack2<T>(y.y.x, y.y.y));
          }
          *reinterpret_cast<uint2*>(dst + h * D + e0) = lo[h];
          *reinterpret_cast<uint2*>(dst + h * D + e1) = hi[h];
        }
    }
    return;
  }
  // -------------------------------------------------------------- keys, values
  // `lanes_h` warps share a window's heads; a block has 8 / lanes_h windows
  const int lanes_h = min(a.hkv, kWarps), windows = kWarps / lanes_h;
  if (warp >= windows * lanes_h) return;
  const bool apart = W == 1 && a.apart;
  const bool do_k = !apart || !(blockIdx.x & 1), do_v = !apart || (blockIdx.x & 1);
  const int64_t w0l = (int64_t(apart ? blockIdx.x / 2 : blockIdx.x) * windows + warp / lanes_h) * W;
  if (w0l >= a.rows) return;
  const int w0 = static_cast<int>(w0l);
  const int h0 = warp % lanes_h;

  // slot of a row, or -1 where it is skipped
  auto slot_of = [&](int row, int& p, unsigned& bad) -> int {
    const int64_t s = a.slots[row];
    if (s < 0) return -1;
    if (s >= a.cache_slots) bad |= FE_DEVERR_SLOT_RANGE;
    if (a.pos) {
      const int64_t q = a.pos[row];
      if (q < 0 || q >= a.max_positions) bad |= FE_DEVERR_POS_RANGE;
      p = static_cast<int>(q);
    }
    return bad ? -1 : static_cast<int>(s);
  };
  const int my = w0 - 1 + lane;  // this lane's row
  int slot = -1, p = 0;
  unsigned bad = 0;
  if (my >= 0 && my < a.rows) slot = slot_of(my, p, bad);
  if (h0 == 0 && do_k && bad && lane >= 1 && lane <= W) raise_device_error(a.err, bad);
  const unsigned good = __ballot_sync(0xffffffffu, slot >= 0);
  const unsigned below = good & ((1u << lane) - 1u);
  int prev = __shfl_sync(0xffffffffu, slot, below ? 31 - __clz(below) : 0);
  if (!below) prev = -1;
  const int lowest = __ffs(good) - 1;
  if (lowest >= 1 && lowest <= W)  // the row before is skipped: look further back
    for (int c = w0 - 2; c >= 0; c -= 32) {
      unsigned bits = 0;
      int q = 0;
      const int s = c >= lane ? slot_of(c - lane, q, bits) : -1;
      const unsigned any = __ballot_sync(0xffffffffu, s >= 0);
      if (any) {
        const int near = __shfl_sync(0xffffffffu, s, __ffs(any) - 1);
        if (lane == lowest) prev = near;
        break;
      }
    }
  const bool joins =
      slot >= 0 && prev >= 0 && slot / kKv8Block == prev / kKv8Block && slot > prev;
  const unsigned heads = __ballot_sync(0xffffffffu, slot >= 0 && !joins);
  unsigned starts = heads & static_cast<unsigned>(((uint64_t(1) << W) - 1) << 1);

  while (starts) {
    const int b = __ffs(starts) - 1;
    starts &= starts - 1;
    // the run's rows: lane m < len has row, slot and position of the m-th
    const unsigned next = heads & ~((2u << b) - 1u);
    unsigned members = good & ~((1u << b) - 1u);
    if (next) members &= (1u << (__ffs(next) - 1)) - 1u;
    Run run;
    run.len = __popc(members);
    const bool adjacent = (members >> b) == (1u << run.len) - 1u;  // b >= 1: len < 32
    const int at = adjacent ? (b + lane) & 31 : static_cast<int>(__fns(members, 0, lane + 1)) & 31;
    run.row0 = w0 - 1 + b;
    run.row_m = w0 - 1 + at;
    int slot_m = __shfl_sync(0xffffffffu, slot, at);
    run.pos_m = __shfl_sync(0xffffffffu, p, at);
    int last = __shfl_sync(0xffffffffu, slot_m, run.len - 1);
    bool more = !next;  // skipped rows may have pushed the run past the lanes
    for (int c = w0 + 31; more && c < a.rows && last % kKv8Block != kKv8Block - 1; c += 32) {
      unsigned bits = 0;
      int q = 0;
      const int s = c + lane < a.rows ? slot_of(c + lane, q, bits) : -1;
      for (unsigned g = __ballot_sync(0xffffffffu, s >= 0); g; g &= g - 1) {
        const int l = __ffs(g) - 1;
        const int sl = __shfl_sync(0xffffffffu, s, l), ql = __shfl_sync(0xffffffffu, q, l);
        more = sl / kKv8Block == last / kKv8Block && sl > last;
        if (!more) break;
        if (lane == run.len) {
          run.row_m = c + l;
          slot_m = sl;
          run.pos_m = ql;
        }
        ++run.len;
        last = sl;
      }
    }
    run.blk = last / kKv8Block;
    run.off_m = slot_m % kKv8Block;
    run.kept = __shfl_sync(0xffffffffu, run.off_m, 0);
    const int last_row = __shfl_sync(0xffffffffu, run.row_m, run.len - 1);
    run.dense = last_row - run.row0 == run.len - 1 &&
                last % kKv8Block - run.kept == run.len - 1;
    uint8_t* stage = smem + warp * (apart ? 1 : 2) * Stage<D>::kBytes;
    for (int h = h0; h < a.hkv; h += lanes_h) {
      if (W > 1 && run.dense && run.len == kKv8Block)
        append_run<T, D, true>(a, run, h, do_k, do_v, stage, lane);
      else
        append_run<T, D, false>(a, run, h, do_k, do_v, stage, lane);
    }
  }
}

// ---------------------------------------------------------------------------
// Gather: blockIdx.y = sequence; a warp takes kTok tokens, every lane's
// 16-code chunks of them in flight together. Bound by memory traffic: 64
// sequences of 512 to 4096 tokens, 8 heads of 128 dims to bf16, 68.4 us = 5.6
// TB/s (0.86 of a device-to-device copy's rate, whose reads and writes are
// equal parts; here two thirds are writes). Four blocks an SM against three,
// by registers: 72 against 85 us.
// ---------------------------------------------------------------------------
constexpr int kGatherTok = 4;

template <typename T>
__global__ void __launch_bounds__(kThreads, 4)
    kv8_gather_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps,
                      T* __restrict__ out, const int32_t* __restrict__ kv,
                      const int32_t* __restrict__ pages, const int32_t* __restrict__ last,
                      const int32_t* __restrict__ row_offset, int page, int hkv, int dim,
                      int64_t cache_slots, int64_t out_rows, int num_pages, unsigned int* err) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.y;
  const int p0 = __ldg(kv + b), p1 = __ldg(kv + b + 1);
  if (p1 <= p0) return;
  const int tail = __ldg(last + b);
  const int off = __ldg(row_offset + b);
  int len;
  {
    const int64_t tokens = (int64_t(p1) - p0 - 1) * page + tail;
    // its pages within the list, its rows within `out`
    const bool bad = tail < 1 || tail > page || tokens > INT32_MAX / 2 || p0 < 0 ||
                     p1 > num_pages || off < 0 || tokens > out_rows - off;
    if (bad) {
      if (threadIdx.x == 0 && blockIdx.x == 0) raise_device_error(err, FE_DEVERR_PAGE_RANGE);
      return;
    }
    len = static_cast<int>(tokens);
  }
  const int64_t orow = off;
  const int lane = threadIdx.x & 31;
  const int chunks = hkv * dim / 16;
  const int step = gridDim.x * kWarps * kGatherTok;
  for (int t0 = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * kGatherTok; t0 < len; t0 += step) {
    int slot[kGatherTok];  // below 2^31, -1: nothing to do
#pragma unroll
    for (int i = 0; i < kGatherTok; ++i) {
      const int t = t0 + i;
      slot[i] = -1;
      if (t < len) {
        const int64_t s = int64_t(__ldg(pages + p0 + t / page)) * page + t % page;
        if (s >= 0 && s < cache_slots)
          slot[i] = static_cast<int>(s);
        else if (lane == 0)
          raise_device_error(err, FE_DEVERR_PAGE_RANGE);
      }
    }
    for (int c = lane; c < chunks; c += 32) {
      const int h = c * 16 / dim;
      uint4 v[kGatherTok];
      int e[kGatherTok];
#pragma unroll
      for (int i = 0; i < kGatherTok; ++i)
        if (slot[i] >= 0) {
          v[i] = __ldg(reinterpret_cast<const uint4*>(codes) + int64_t(slot[i]) * chunks + c);
          e[i] = __ldg(exps + int64_t(slot[i] / kKv8Block) * hkv + h);
        }
#pragma unroll
      for (int i = 0; i < kGatherTok; ++i)
        if (slot[i] >= 0) {
          const float s = exp_scale(exp_clamp(e[i]));
          const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
          uint32_t o[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 s2 = make_float2(s, s);
            const float2 lo = mul2(unpack2<__half>(e4m3x2_to_h2(w[j])), s2);
            const float2 hi = mul2(unpack2<__half>(e4m3x2_hi_to_h2(w[j])), s2);
            o[2 * j] = pack2<T>(lo.x, lo.y);
            o[2 * j + 1] = pack2<T>(hi.x, hi.y);
          }
          uint4* dst = reinterpret_cast<uint4*>(out + (orow + t0 + i) * (int64_t(chunks) * 16)) +
                       2 * c;
          dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
          dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
        }
    }
  }
}

// ---------------------------------------------------------------------------
// Block copy: blockIdx.y = copy, blockIdx.z = layer * 2 + (K|V). A page's
// first ntok tokens are one contiguous range of codes; their scales are the
// first ceil(ntok / 16) rows of the page's scales (a partly copied block
// keeps its source's scale). Bound by memory traffic, once it outlasts the
// launch: 64 pages in 48 layers with 4 heads of 128 dims 14.8 us = 3.9 TB/s.
// ---------------------------------------------------------------------------
struct Kv8Table {
  uint8_t* codes[2 * FE_MAX_LAYERS];
  uint8_t* exps[2 * FE_MAX_LAYERS];
};

constexpr int kCopyUnroll = 4;

__global__ void __launch_bounds__(kThreads)
    kv8_copy_kernel(const __grid_constant__ Kv8Table t, const int32_t* __restrict__ src,
                    const int32_t* __restrict__ dst, const int32_t* __restrict__ ntok, int page,
                    int hkv, int chunks_per_row, int num_pages_total, unsigned int* err) {
  pdl_trigger();
  pdl_wait();
  const int c = blockIdx.y;
  const int s = __ldg(src + c), d = __ldg(dst + c), n = __ldg(ntok + c);
  if (s < 0 || s >= num_pages_total || d < 0 || d >= num_pages_total || n < 0 || n > page) {
    if (threadIdx.x == 0 && blockIdx.x == 0)
      raise_device_error(err, n < 0 || n > page ? FE_DEVERR_NTOK_RANGE : FE_DEVERR_PAGE_RANGE);
    return;
  }
  uint4* pool = reinterpret_cast<uint4*>(t.codes[blockIdx.z]);
  const int64_t page_chunks = int64_t(page) * chunks_per_row;
  const uint4* from = pool + s * page_chunks;
  uint4* to = pool + d * page_chunks;
  const int64_t total = int64_t(n) * chunks_per_row;
  const int64_t stride = int64_t(gridDim.x) * blockDim.x;
  const int64_t me = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  for (int64_t base = me; base < total; base += stride * kCopyUnroll) {
    uint4 val[kCopyUnroll];
#pragma unroll
    for (int k = 0; k < kCopyUnroll; ++k)
      if (base + k * stride < total) val[k] = from[base + k * stride];
#pragma unroll
    for (int k = 0; k < kCopyUnroll; ++k)
      if (base + k * stride < total) to[base + k * stride] = val[k];
  }
  uint8_t* exps = t.exps[blockIdx.z];
  const int64_t rows = page / kKv8Block;
  const int64_t bytes = int64_t((n + kKv8Block - 1) / kKv8Block) * hkv;
  for (int64_t i = me; i < bytes; i += stride)
    exps[d * rows * hkv + i] = exps[s * rows * hkv + i];
}

template <typename T, int D>
int launch_append(AppendArgs& a, cudaStream_t stream) {
  // Up to 2 Ki (row, head) pairs two warps each, one for K and one for V; up to
  // 8 Ki one; a warp per 4 rows and head up to 32 Ki, per 16 beyond. us on a
  // B200 with 8 heads:
  //   sequences x rows  64x1 16x16 512x1 16x61 1024x1 16x125 2048x1 16x253 16x1021
  //   two warps          3.5   7.9   8.5  12.7   15.5   25.5     37     45     173
  //   one warp           3.9  10.3   7.5  13.3   11.7   20.2     27     32     124
  //   per 4 rows         9.7  12.2  12.3  12.5   12.9   15.7     26     22      80
  //   per 16 rows       32.5  12.2  35.4  15.2   37.1   18.3     47     22      76
  // (8 rows: 64 Ki rows of 16 prompts 297 against 289.)
  const int64_t pairs = int64_t(a.rows) * a.hkv;
  const int w = pairs > 32768 ? 16 : pairs > 8192 ? 4 : 1;
  a.apart = pairs <= 2048;
  const int64_t windows = (int64_t(a.rows) + w - 1) / w;
  const int per_block = a.hkv < kWarps ? kWarps / a.hkv : 1;
  const int64_t kvb = (windows + per_block - 1) / per_block * (a.apart ? 2 : 1);
  const int64_t qb = (int64_t(a.rows) * ((a.hq + kQHeads - 1) / kQHeads) * (D / 8) + kThreads - 1) /
               kThreads;
  if (kvb > INT32_MAX - qb) return fail(FE_ERR_CAPACITY, "fe_kv8_append: too many rows");
  a.kv_blocks = static_cast<int>(kvb);
  const dim3 grid(static_cast<unsigned>(kvb + qb));
  constexpr int kSmem = kWarps * 2 * Stage<D>::kBytes;
  static std::once_flag once;
  static cudaError_t attr_err = cudaSuccess;
  std::call_once(once, [] {
    for (auto kernel : {kv8_append_kernel<T, D, 16>, kv8_append_kernel<T, D, 4>,
                        kv8_append_kernel<T, D, 1>})
      if (attr_err == cudaSuccess)
        attr_err =
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  });
  if (attr_err != cudaSuccess) return cuda_fail(attr_err, "kv8_append_kernel attribute");
  auto kernel = w == 16  ? kv8_append_kernel<T, D, 16>
                : w == 4 ? kv8_append_kernel<T, D, 4>
                         : kv8_append_kernel<T, D, 1>;
  FE_CUDA_TRY(launch_pdl(kernel, grid, dim3(kThreads), a.apart ? kSmem / 2 : kSmem, stream, a));
  return FE_OK;
}

bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

}  // namespace
}  // namespace fe

using namespace fe;

extern "C" {

int fe_kv8_append(const void* q, void* q_out, const void* k, const void* v, uint8_t* k_codes,
                  uint8_t* v_codes, uint8_t* k_exp, uint8_t* v_exp, const int64_t* slots,
                  const int64_t* pos, const float* cache, int rows, int hq, int hkv, int dim,
                  int rotary_dim, int max_positions, int dtype, int64_t cache_slots,
                  void* stream) {
  if (!valid_dtype(dtype)) return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv8_append: bad dtype");
  if (rows < 0 || hq < 0 || hkv <= 0 || cache_slots <= 0 || cache_slots % kKv8Block != 0)
    return fail(FE_ERR_INVALID_ARGUMENT,
                "fe_kv8_append: sizes out of range (cache_slots a multiple of 16)");
  if (dim != 128 && dim != 256)
    return fail(FE_ERR_UNSUPPORTED, "fe_kv8_append: head_dim must be 128 or 256");
  if (rotary_dim < 0 || rotary_dim > dim || rotary_dim % 8 != 0)
    return fail(FE_ERR_UNSUPPORTED,
                "fe_kv8_append: rotary_dim must be a multiple of 8, at most head_dim");
  if (rotary_dim > 0 && max_positions <= 0)
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv8_append: max_positions <= 0");
  if (cache_slots > INT32_MAX)
    return fail(FE_ERR_CAPACITY, "fe_kv8_append: cache_slots above 2^31");
  if (rows == 0) return FE_OK;
  if (!k || !v || !k_codes || !v_codes || !k_exp || !v_exp || !slots ||
      (hq > 0 && (!q || !q_out)) || (rotary_dim > 0 && (!pos || !cache)))
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv8_append: null pointer");
  if (!aligned16(k) || !aligned16(v) || !aligned8(q) || !aligned8(q_out) || !aligned8(k_codes) ||
      !aligned8(v_codes) || !aligned16(cache))
    return fail(FE_ERR_INVALID_ARGUMENT,
                "fe_kv8_append: k, v and the cache must be 16-byte, q and codes 8-byte aligned");
  AppendArgs a{q, q_out, k, v, k_codes, v_codes, k_exp, v_exp, slots,
               rotary_dim > 0 ? pos : nullptr, cache, rows, hq, hkv, rotary_dim, max_positions,
               cache_slots, 0, false, device_error_word()};
  auto s = static_cast<cudaStream_t>(stream);
  if (dtype == FE_DTYPE_BF16)
    return dim == 128 ? launch_append<__nv_bfloat16, 128>(a, s)
                      : launch_append<__nv_bfloat16, 256>(a, s);
  return dim == 128 ? launch_append<__half, 128>(a, s) : launch_append<__half, 256>(a, s);
}

int fe_kv8_gather(const uint8_t* codes, const uint8_t* exps, void* out, const int32_t* kv,
                  const int32_t* pages, const int32_t* last, const int32_t* row_offset, int batch,
                  int max_len, int page, int hkv, int dim, int dtype, int64_t cache_slots,
                  void* stream) {
  return fe_kv8_gather_within(codes, exps, out, INT64_MAX, kv, pages, INT32_MAX, last, row_offset,
                              batch, max_len, page, hkv, dim, dtype, cache_slots, stream);
}

int fe_kv8_gather_within(const uint8_t* codes, const uint8_t* exps, void* out, int64_t out_rows,
                         const int32_t* kv, const int32_t* pages, int num_pages,
                         const int32_t* last, const int32_t* row_offset, int batch, int max_len,
                         int page, int hkv, int dim, int dtype, int64_t cache_slots,
                         void* stream) {
  if (!valid_dtype(dtype)) return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv8_gather: bad dtype");
  if (batch < 0 || max_len < 0 || page <= 0 || page % kKv8Block != 0 || hkv <= 0 || dim <= 0 ||
      cache_slots <= 0 || cache_slots % kKv8Block != 0 || out_rows < 0 || num_pages < 0)
    return fail(FE_ERR_INVALID_ARGUMENT,
                "fe_kv8_gather: bad sizes (page and cache_slots multiples of 16)");
  if (dim % 16 != 0 || int64_t(hkv) * dim > INT32_MAX / 2)
    return fail(FE_ERR_UNSUPPORTED, "fe_kv8_gather: head_dim must be a multiple of 16");
  if (batch == 0 || max_len == 0) return FE_OK;
  if (batch > 65535) return fail(FE_ERR_CAPACITY, "fe_kv8_gather: at most 65535 sequences");
  if (cache_slots > INT32_MAX)
    return fail(FE_ERR_CAPACITY, "fe_kv8_gather: cache_slots above 2^31");
  if (!codes || !exps || !out || !kv || !pages || !last || !row_offset)
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv8_gather: null pointer");
  if (!aligned16(codes) || !aligned16(out))
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv8_gather: buffers must be 16-byte aligned");
  const int per_block = kWarps * kGatherTok;
  int64_t bx = (int64_t(max_len) + per_block - 1) / per_block;
  if (bx > 4096) bx = 4096;  // warps stride over longer sequences
  const dim3 grid(static_cast<unsigned>(bx), batch);
  auto s = static_cast<cudaStream_t>(stream);
  if (dtype == FE_DTYPE_BF16)
    FE_CUDA_TRY(launch_pdl(kv8_gather_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, s, codes,
                           exps, static_cast<__nv_bfloat16*>(out), kv, pages, last, row_offset,
                           page, hkv, dim, cache_slots, out_rows, num_pages,
                           device_error_word()));
  else
    FE_CUDA_TRY(launch_pdl(kv8_gather_kernel<__half>, grid, dim3(kThreads), 0, s, codes, exps,
                           static_cast<__half*>(out), kv, pages, last, row_offset, page, hkv, dim,
                           cache_slots, out_rows, num_pages, device_error_word()));
  return FE_OK;
}

int fe_kv8_copy_blocks(void* const* k_codes, void* const* v_codes, void* const* k_exps,
                       void* const* v_exps, int num_layers, const int32_t* src,
                       const int32_t* dst, const int32_t* ntok, int num_copies, int page, int hkv,
                       int dim, int num_pages_total, void* stream) {
  if (num_layers < 0 || num_layers > FE_MAX_LAYERS)
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv8_copy_blocks: num_layers out of range");
  if (num_copies < 0 || page <= 0 || page % kKv8Block != 0 || hkv <= 0 || dim <= 0 ||
      num_pages_total <= 0)
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv8_copy_blocks: bad sizes (page a multiple of 16)");
  if (dim % 16 != 0 || int64_t(hkv) * dim > INT32_MAX / 2)
    return fail(FE_ERR_UNSUPPORTED, "fe_kv8_copy_blocks: head_dim must be a multiple of 16");
  if (num_copies == 0 || num_layers == 0) return FE_OK;
  if (num_copies > 65535)
    return fail(FE_ERR_CAPACITY, "fe_kv8_copy_blocks: at most 65535 copies per call");
  if (!k_codes || !v_codes || !k_exps || !v_exps || !src || !dst || !ntok)
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv8_copy_blocks: null pointer");
  Kv8Table t;
  std::memset(&t, 0, sizeof(t));
  for (int l = 0; l < num_layers; ++l) {
    if (!k_codes[l] || !v_codes[l] || !k_exps[l] || !v_exps[l] || !aligned16(k_codes[l]) ||
        !aligned16(v_codes[l]))
      return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv8_copy_blocks: pool pointers must be non-null, "
                                           "codes 16-byte aligned");
    t.codes[2 * l] = static_cast<uint8_t*>(k_codes[l]);
    t.codes[2 * l + 1] = static_cast<uint8_t*>(v_codes[l]);
    t.exps[2 * l] = static_cast<uint8_t*>(k_exps[l]);
    t.exps[2 * l + 1] = static_cast<uint8_t*>(v_exps[l]);
  }
  const int chunks = hkv * dim / 16;
  int64_t bx = (int64_t(page) * chunks + kThreads * kCopyUnroll - 1) / (kThreads * kCopyUnroll);
  if (bx > 1024) bx = 1024;
  const dim3 grid(static_cast<unsigned>(bx), num_copies, num_layers * 2);
  FE_CUDA_TRY(launch_pdl(kv8_copy_kernel, grid, dim3(kThreads), 0,
                         static_cast<cudaStream_t>(stream), t, src, dst, ntok, page, hkv, chunks,
                         num_pages_total, device_error_word()));
  return FE_OK;
}

}  // extern "C"
