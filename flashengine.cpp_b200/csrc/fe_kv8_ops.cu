// 8-bit KV cache operators around the attention: append (rotation,
// quantisation and scatter in one launch), gather of whole sequences back to
// 16 bits, and block copies of forked sequences. No counterpart in the
// reference, whose pools are 16-bit (src/cuda_model.cpp:60); slot semantics,
// rotation and roundings follow fe_kv_append / fe_rope.
#include <cstring>
#include <string>

#include "fe_kv8_common.cuh"

namespace fe {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kQHeads = 4;  // query heads per thread of an append

__device__ __forceinline__ float2 to_float2(uint32_t v, __half) {
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}
__device__ __forceinline__ float2 to_float2(uint32_t v, __nv_bfloat16) {
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
}

// Four rotation pairs a[i], b[i] in fp32, each product and sum rounded
// separately as fe_rope does.
__device__ __forceinline__ void rotate4(float* a, float* b, const float (&c)[4],
                                        const float (&s)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = a[i], y = b[i];
    a[i] = __fsub_rn(__fmul_rn(x, c[i]), __fmul_rn(y, s[i]));
    b[i] = __fadd_rn(__fmul_rn(y, c[i]), __fmul_rn(x, s[i]));
  }
}

template <typename T>
__device__ __forceinline__ void unpack4(float* x, uint2 v) {
  const float2 a = to_float2(v.x, T()), b = to_float2(v.y, T());
  x[0] = a.x;
  x[1] = a.y;
  x[2] = b.x;
  x[3] = b.y;
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
  int64_t cache_slots;
  int kv_blocks;        // blocks of the kv part; the rest rotate queries
  unsigned int* err;
};

// ---------------------------------------------------------------------------
// Append. Work of the kv part: a RUN, the adjacent rows whose slots lie in one
// scale block in increasing order (rows that are skipped do not end it), for
// one KV head of K or of V, is one warp's: it holds the (rotated) values in
// fp32 registers, takes their largest finite magnitude, joins it with the
// block's old exponent when earlier tokens are kept, and writes the codes;
// when the scale grows, the kept tokens' codes are rounded to the new one. So
// every (block, head) has one writer per call and nothing is atomic.
//
// A warp looks at a window of W rows for run starts (W = 1: a decode step
// gives each row its own warp; W = 16: a prompt's rows, whose runs are mostly
// whole blocks, are covered by one warp per 16 rows instead of 16 warps of
// which 15 find nothing). The 32 lanes read the slots of rows w - 1 .. w + 30:
// the row before the window, the window, and what its last run can reach;
// only among skipped rows does a run need more (the two loops over rows).
//
// The query part rotates q into q_out, a thread per (row, kQHeads heads, 4 + 4
// dims): the heads share the row's cos / sin.
// Both parts are bound by memory traffic on prompts and by a chain of three
// loads (slot and position, row and cos / sin, store) on decode steps.
// ---------------------------------------------------------------------------
template <typename T, int D, int W>
__global__ void __launch_bounds__(kThreads, D == 128 ? 3 : 2) kv8_append_kernel(const AppendArgs a) {
  pdl_trigger();
  pdl_wait();  // q, k, v come from, and the pools are read by, earlier kernels
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = a.rot / 2;
  const int rot_units = a.rot / 8;
  constexpr int kUnits = D / 8;  // a unit is 4 + 4 dims of a head
  if (static_cast<int>(blockIdx.x) >= a.kv_blocks) {
    // ------------------------------------------------------------- queries
    const int groups = (a.hq + kQHeads - 1) / kQHeads;
    const int64_t per_row = int64_t(groups) * kUnits;
    const int64_t total = a.rows * per_row;
    const int64_t step = int64_t(gridDim.x - a.kv_blocks) * kThreads;
    for (int64_t i = int64_t(blockIdx.x - a.kv_blocks) * kThreads + threadIdx.x; i < total;
         i += step) {
      const int row = static_cast<int>(i / per_row);
      const int rem = static_cast<int>(i - row * per_row);
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
      float cs[4], sn[4];
      if (a.pos) {
        const int64_t p = a.pos[row];
        if (p < 0 || p >= a.max_positions) {
          if (rem == 0) raise_device_error(a.err, FE_DEVERR_POS_RANGE);
          continue;
        }
        if (turn) {
          const float* at = a.cache + p * a.rot + e0;
          *reinterpret_cast<float4*>(cs) = *reinterpret_cast<const float4*>(at);
          *reinterpret_cast<float4*>(sn) = *reinterpret_cast<const float4*>(at + r);
        }
      }
#pragma unroll
      for (int h = 0; h < kQHeads; ++h)
        if (h0 + h < a.hq) {
          if (turn && a.pos) {
            float x[4], y[4];
            unpack4<T>(x, lo[h]);
            unpack4<T>(y, hi[h]);
            rotate4(x, y, cs, sn);
            lo[h] = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
            hi[h] = make_uint2(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]));
          }
          *reinterpret_cast<uint2*>(dst + h * D + e0) = lo[h];
          *reinterpret_cast<uint2*>(dst + h * D + e1) = hi[h];
        }
    }
    return;
  }
  // -------------------------------------------------------------- keys, values
  const int64_t job = int64_t(blockIdx.x) * kWarps + warp;
  const int jobs_per_window = 2 * a.hkv;
  const int64_t window = job / jobs_per_window;
  const int which = static_cast<int>(job - window * jobs_per_window);
  const int64_t w0 = window * W;
  if (w0 >= a.rows) return;
  const bool is_v = which >= a.hkv;
  const int h = is_v ? which - a.hkv : which;
  uint8_t* codes = is_v ? a.v_codes : a.k_codes;
  uint8_t* exps = is_v ? a.v_exp : a.k_exp;
  const T* src = static_cast<const T*>(is_v ? a.v : a.k);
  const bool turning = !is_v && a.pos != nullptr;

  // slot of a row, or -1 where it is skipped
  auto slot_of = [&](int64_t row, int64_t& p, unsigned& bad) -> int64_t {
    const int64_t s = a.slots[row];
    if (s < 0) return -1;
    if (s >= a.cache_slots) bad |= FE_DEVERR_SLOT_RANGE;
    if (a.pos) {
      p = a.pos[row];
      if (p < 0 || p >= a.max_positions) bad |= FE_DEVERR_POS_RANGE;
    }
    return bad ? -1 : s;
  };
  const int64_t my = w0 - 1 + lane;  // this lane's row
  int64_t slot = -1, p = 0;
  unsigned bad = 0;
  if (my >= 0 && my < a.rows) slot = slot_of(my, p, bad);
  if (which == 0 && bad && lane >= 1 && lane <= W) raise_device_error(a.err, bad);
  const unsigned good = __ballot_sync(0xffffffffu, slot >= 0);
  const unsigned below = good & ((1u << lane) - 1u);
  int64_t prev = __shfl_sync(0xffffffffu, slot, below ? 31 - __clz(below) : 0);
  if (!below) prev = -1;
  const int lowest = __ffs(good) - 1;
  if (lowest >= 1 && lowest <= W)  // the row before is skipped: look further back
    for (int64_t c = w0 - 2; c >= 0; c -= 32) {
      unsigned bits = 0;
      int64_t q = 0;
      const int64_t s = c >= lane ? slot_of(c - lane, q, bits) : -1;
      const unsigned any = __ballot_sync(0xffffffffu, s >= 0);
      if (any) {
        const int64_t near = __shfl_sync(0xffffffffu, s, __ffs(any) - 1);
        if (lane == lowest) prev = near;
        break;
      }
    }
  const bool joins =
      slot >= 0 && prev >= 0 && slot / kKv8Block == prev / kKv8Block && slot > prev;
  const unsigned heads = __ballot_sync(0xffffffffu, slot >= 0 && !joins);
  unsigned starts = heads & static_cast<unsigned>(((uint64_t(1) << W) - 1) << 1);

  constexpr int kRows = 256 / D;               // rows per pass of the warp
  constexpr int kPasses = kKv8Block / kRows;
  const int sub = lane / kUnits, u = lane % kUnits;
  const bool turn = u < rot_units;
  const int e0 = turn ? 4 * u : a.rot + 8 * (u - rot_units), e1 = turn ? e0 + r : e0 + 4;
  while (starts) {
    const int b = __ffs(starts) - 1;
    starts &= starts - 1;
    // the run's rows: lane m < len has row and slot of the m-th
    const unsigned next = heads & ~((2u << b) - 1u);
    unsigned members = good & ~((1u << b) - 1u);
    if (next) members &= (1u << (__ffs(next) - 1)) - 1u;
    int len = __popc(members);
    const bool dense = (members >> b) == (len == 32 ? ~0u : (1u << len) - 1u);
    const int at = dense ? (b + lane) & 31 : static_cast<int>(__fns(members, 0, lane + 1)) & 31;
    int64_t row_m = w0 - 1 + at, slot_m = __shfl_sync(0xffffffffu, slot, at),
            pos_m = __shfl_sync(0xffffffffu, p, at);
    int64_t last = __shfl_sync(0xffffffffu, slot_m, len - 1);
    if (!next) {  // skipped rows may have pushed the run past the lanes
      bool more = true;
      for (int64_t c = w0 + 31; more && c < a.rows && last % kKv8Block != kKv8Block - 1; c += 32) {
        unsigned bits = 0;
        int64_t q = 0;
        const int64_t s = c + lane < a.rows ? slot_of(c + lane, q, bits) : -1;
        for (unsigned g = __ballot_sync(0xffffffffu, s >= 0); g && more; g &= g - 1) {
          const int l = __ffs(g) - 1;
          const int64_t sl = __shfl_sync(0xffffffffu, s, l), ql = __shfl_sync(0xffffffffu, q, l);
          more = sl / kKv8Block == last / kKv8Block && sl > last;
          if (!more) break;
          if (lane == len) {
            row_m = c + l;
            slot_m = sl;
            pos_m = ql;
          }
          ++len;
          last = sl;
        }
      }
    }
    const int64_t blk = last / kKv8Block;
    const int off_m = static_cast<int>(slot_m % kKv8Block);
    const int kept = __shfl_sync(0xffffffffu, off_m, 0);
    const int old = kept ? exps[blk * a.hkv + h] : 0;
    // all rows of the run in flight, then the rotation and the maximum
    uint2 lo[kPasses], hi[kPasses];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int t = i * kRows + sub;
      const int64_t rt = __shfl_sync(0xffffffffu, row_m, t & 31);
      if (t < len) {
        const T* row = src + (rt * a.hkv + h) * D;
        lo[i] = *reinterpret_cast<const uint2*>(row + e0);
        hi[i] = *reinterpret_cast<const uint2*>(row + e1);
      }
    }
    // (the second time for the codes: rotating again costs less than keeping
    // the fp32 values, 64 registers a lane, would in warps per SM)
    auto turned = [&](int i, float (&x)[8]) {
      const int64_t pt = __shfl_sync(0xffffffffu, pos_m, (i * kRows + sub) & 31);
      if (i * kRows + sub < len) {
        unpack4<T>(x, lo[i]);
        unpack4<T>(x + 4, hi[i]);
        if (turning && turn) {
          const float* at = a.cache + pt * a.rot + e0;
          float cs[4], sn[4];
          *reinterpret_cast<float4*>(cs) = *reinterpret_cast<const float4*>(at);
          *reinterpret_cast<float4*>(sn) = *reinterpret_cast<const float4*>(at + r);
          rotate4(x, x + 4, cs, sn);
        }
      }
    };
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      if (i * kRows >= len) break;
      float x[8];
      turned(i, x);
      if (i * kRows + sub < len) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float m = fabsf(x[e]);
          if (m < INFINITY) amax = fmaxf(amax, m);  // infinities saturate, NaN stays
        }
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    int e = needed_exp(amax);
    if (kept) e = min(max(e, old), kKv8MaxExp);
    const float inv = exp_scale(254 - e);
    uint8_t* block = codes + (blk * kKv8Block * a.hkv + h) * D;
    const int64_t tok = int64_t(a.hkv) * D;  // bytes from one token to the next
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      if (i * kRows >= len) break;
      const int t = i * kRows + sub;
      const int off = __shfl_sync(0xffffffffu, off_m, t & 31);
      float x[8];
      turned(i, x);
      if (t < len) {
        uint8_t* dst = block + off * tok;
        const uint32_t c0 = e4m3x2(x[0] * inv, x[1] * inv) | e4m3x2(x[2] * inv, x[3] * inv) << 16;
        const uint32_t c1 = e4m3x2(x[4] * inv, x[5] * inv) | e4m3x2(x[6] * inv, x[7] * inv) << 16;
        *reinterpret_cast<uint32_t*>(dst + e0) = c0;
        *reinterpret_cast<uint32_t*>(dst + e1) = c1;
      }
    }
    if (kept && e > old) {
      // the kept tokens move to the larger scale: 8 codes per lane and pass
      const float down = exp_scale(max(old - e + 127, 1));
      for (int t = sub; t < kept; t += kRows) {
        uint2* w = reinterpret_cast<uint2*>(block + t * tok) + u;
        uint2 c = *w;
        uint32_t* cw = &c.x;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t l = e4m3x2_to_h2(cw[j]), g = e4m3x2_hi_to_h2(cw[j]);
          const float2 fl = unpack2<__half>(l), fg = unpack2<__half>(g);
          cw[j] = e4m3x2(fl.x * down, fl.y * down) | e4m3x2(fg.x * down, fg.y * down) << 16;
        }
        *w = c;
      }
    }
    if (lane == 0 && (!kept || e != old)) exps[blk * a.hkv + h] = static_cast<uint8_t>(e);
  }
}

// ---------------------------------------------------------------------------
// Gather: blockIdx.y = sequence; a warp takes kTok tokens, every lane's
// 16-code chunks of them in flight together. Bound by memory traffic.
// ---------------------------------------------------------------------------
constexpr int kGatherTok = 4;

template <typename T>
__global__ void __launch_bounds__(kThreads)
    kv8_gather_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps,
                      T* __restrict__ out, const int32_t* __restrict__ kv,
                      const int32_t* __restrict__ pages, const int32_t* __restrict__ last,
                      const int32_t* __restrict__ row_offset, int page, int hkv, int dim,
                      int64_t cache_slots, unsigned int* err) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.y;
  const int p0 = __ldg(kv + b), p1 = __ldg(kv + b + 1);
  if (p1 <= p0) return;
  const int len = (p1 - p0 - 1) * page + __ldg(last + b);
  const int64_t orow = __ldg(row_offset + b);
  const int lane = threadIdx.x & 31;
  const int chunks = hkv * dim / 16;
  const int step = gridDim.x * kWarps * kGatherTok;
  for (int t0 = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * kGatherTok; t0 < len; t0 += step) {
    int64_t slot[kGatherTok];
#pragma unroll
    for (int i = 0; i < kGatherTok; ++i) {
      const int t = t0 + i;
      slot[i] = t < len ? int64_t(__ldg(pages + p0 + t / page)) * page + t % page : -1;
      if (t < len && (slot[i] < 0 || slot[i] >= cache_slots)) {
        if (lane == 0) raise_device_error(err, FE_DEVERR_PAGE_RANGE);
        slot[i] = -1;
      }
    }
    for (int c = lane; c < chunks; c += 32) {
      const int h = c * 16 / dim;
      uint4 v[kGatherTok];
      int e[kGatherTok];
#pragma unroll
      for (int i = 0; i < kGatherTok; ++i)
        if (slot[i] >= 0) {
          v[i] = __ldg(reinterpret_cast<const uint4*>(codes) + slot[i] * chunks + c);
          e[i] = __ldg(exps + slot[i] / kKv8Block * hkv + h);
        }
#pragma unroll
      for (int i = 0; i < kGatherTok; ++i)
        if (slot[i] >= 0) {
          const float s = exp_scale(exp_clamp(e[i]));
          const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
          uint32_t o[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 lo = unpack2<__half>(e4m3x2_to_h2(w[j]));
            const float2 hi = unpack2<__half>(e4m3x2_hi_to_h2(w[j]));
            o[2 * j] = pack2<T>(lo.x * s, lo.y * s);
            o[2 * j + 1] = pack2<T>(hi.x * s, hi.y * s);
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
// keeps its source's scale).
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
  // One warp per row and head up to 64 Ki of them, a warp per 16 rows beyond (prompts).
  const bool wide = int64_t(a.rows) * 2 * a.hkv > 65536;
  const int64_t windows = wide ? (int64_t(a.rows) + 15) / 16 : a.rows;
  const int64_t kvb = (windows * 2 * a.hkv + kWarps - 1) / kWarps;
  int64_t qb = (int64_t(a.rows) * ((a.hq + kQHeads - 1) / kQHeads) * (D / 8) + kThreads - 1) /
               kThreads;
  if (qb > 148 * 64) qb = 148 * 64;
  if (kvb > INT32_MAX - qb) return fail(FE_ERR_CAPACITY, "fe_kv8_append: too many rows");
  a.kv_blocks = static_cast<int>(kvb);
  const dim3 grid(static_cast<unsigned>(kvb + qb));
  if (wide)
    FE_CUDA_TRY(launch_pdl(kv8_append_kernel<T, D, 16>, grid, dim3(kThreads), 0, stream, a));
  else
    FE_CUDA_TRY(launch_pdl(kv8_append_kernel<T, D, 1>, grid, dim3(kThreads), 0, stream, a));
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
  if (rows == 0) return FE_OK;
  if (!k || !v || !k_codes || !v_codes || !k_exp || !v_exp || !slots ||
      (hq > 0 && (!q || !q_out)) || (rotary_dim > 0 && (!pos || !cache)))
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv8_append: null pointer");
  if (!aligned8(k) || !aligned8(v) || !aligned8(q) || !aligned8(q_out) || !aligned8(k_codes) ||
      !aligned8(v_codes) || !aligned16(cache))
    return fail(FE_ERR_INVALID_ARGUMENT,
                "fe_kv8_append: q, k, v and codes must be 8-byte, the cache 16-byte aligned");
  AppendArgs a{q, q_out, k, v, k_codes, v_codes, k_exp, v_exp, slots,
               rotary_dim > 0 ? pos : nullptr, cache, rows, hq, hkv, rotary_dim, max_positions,
               cache_slots, 0, device_error_word()};
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
  if (!valid_dtype(dtype)) return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv8_gather: bad dtype");
  if (batch < 0 || max_len < 0 || page <= 0 || page % kKv8Block != 0 || hkv <= 0 || dim <= 0 ||
      cache_slots <= 0)
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv8_gather: bad sizes (page a multiple of 16)");
  if (dim % 16 != 0 || int64_t(hkv) * dim > INT32_MAX / 2)
    return fail(FE_ERR_UNSUPPORTED, "fe_kv8_gather: head_dim must be a multiple of 16");
  if (batch == 0 || max_len == 0) return FE_OK;
  if (batch > 65535) return fail(FE_ERR_CAPACITY, "fe_kv8_gather: at most 65535 sequences");
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
                           page, hkv, dim, cache_slots, device_error_word()));
  else
    FE_CUDA_TRY(launch_pdl(kv8_gather_kernel<__half>, grid, dim3(kThreads), 0, s, codes, exps,
                           static_cast<__half*>(out), kv, pages, last, row_offset, page, hkv, dim,
                           cache_slots, device_error_word()));
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
