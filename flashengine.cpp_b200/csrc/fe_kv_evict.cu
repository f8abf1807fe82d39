// Eviction from the paged cache by accumulated attention weight: selection of
// the tokens to keep, per sequence and KV head, and their compaction to the
// front of the sequence. No counterpart in the reference, whose cache drops
// whole sequences only (Cambridgebit/FlashEngine.cpp src/scheduler.cpp:6-29).
//
// Both kernels take device metadata (a captured graph replays them for later
// steps) and check what they read of it: a sequence or token that reaches past
// its lists or the pool is skipped and flagged.
#include <algorithm>
#include <string>

#include "fe_common.cuh"

namespace fe {
namespace {

constexpr int kSelThreads = 512;
constexpr int kSelList = 2048;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048;
// most CTAs a list, most CTAs for which lists are divided, fewest tokens a CTA
constexpr int kSelCluster = 8, kSelCtas = 296, kSelPart = 4096;
constexpr int kRankBatch = 128;  // sequences that are taken longest first
constexpr int kSelRoom = 128 << 10;  // tokens whose classes fit in shared memory

// A score as an unsigned number of the same order; NaN below everything.
__device__ __forceinline__ uint32_t ordered(float x) {
  const int b = __float_as_int(x + 0.f);  // -0 and +0 tie
  return x != x ? 0u : static_cast<uint32_t>(b ^ ((b >> 31) | static_cast<int>(0x80000000u)));
}

struct SeqTable {
  const int32_t* kv;
  const int32_t* pages;
  const int32_t* last;
  int num_pages, page;
  int64_t cache_slots;
};

// Pages [p0, p1) and length of sequence b; false when they reach past the
// list or are no sequence.
__device__ __forceinline__ bool sequence(const SeqTable& t, int b, int& p0, int& n) {
  p0 = __ldg(t.kv + b);
  const int p1 = __ldg(t.kv + b + 1), ln = __ldg(t.last + b);
  n = 0;
  if (p0 < 0 || p1 <= p0 || p1 > t.num_pages || ln < 1 || ln > t.page) return false;
  const int64_t len = static_cast<int64_t>(p1 - p0 - 1) * t.page + ln;
  if (len > INT32_MAX - 127) return false;  // (room for rounding up)
  n = static_cast<int>(len);
  return true;
}

// Slot of token t of the sequence at p0, -1 for a page outside the pool.
__device__ __forceinline__ int64_t slot_of(const SeqTable& s, int p0, int t) {
  const int pg = __ldg(s.pages + p0 + t / s.page);
  const int64_t first = static_cast<int64_t>(pg) * s.page;
  return pg < 0 || first + s.page > s.cache_slots ? -1 : first + t % s.page;
}

// Exclusive sum over the block of one value a thread; `total` for everyone.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the last call's sums have been read
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) {
    const int s = warp_sums[w];
    before += w < warp ? s : 0;
    total += s;
  }
  return before + x - v;
}

// The CTAs of a cluster share a list: rank, size, a barrier of all their threads, and
// loads from another CTA's shared memory.
struct Cluster {
  uint32_t rank, size;
  __device__ __forceinline__ Cluster() {
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  }
  __device__ __forceinline__ void sync() const {
    if (size == 1) {
      __syncthreads();
    } else {
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
  }
  __device__ __forceinline__ static uint32_t at(const void* p, uint32_t r) {
    uint32_t addr;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(r));
    return addr;
  }
};

// The bin from the top in which the left-th key lies: (bin, keys still wanted
// of it), for the whole cluster. hist holds kBins bins in each of its CTAs, all
// written before a cluster barrier.
__device__ __forceinline__ int2 find_bin(const Cluster& cl, const int* hist, int left,
                                         int* warp_sums, int* found) {
  constexpr int kPer = kBins / kSelThreads;
  static_assert(kPer == 4, "a thread reads its bins as one vector");
  const int tid = threadIdx.x;
  const int4* at = reinterpret_cast<const int4*>(hist) + (kSelThreads - 1 - tid);
  int4 x = *at;
  if (cl.size > 1) {
    for (uint32_t r = 1; r < cl.size; ++r) {  // the others, each CTA from its own neighbour on
      uint32_t other = cl.rank + r;
      if (other >= cl.size) other -= cl.size;
      int4 y;
      asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w)
                   : "r"(Cluster::at(at, other)));
      x.x += y.x;
      x.y += y.y;
      x.z += y.z;
      x.w += y.w;
    }
  }
  const int mine[kPer] = {x.w, x.z, x.y, x.x};
  int total;
  int above = block_scan(x.x + x.y + x.z + x.w, warp_sums, total);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (above < left && left <= above + mine[i]) {
      found[0] = kBins - 1 - (tid * kPer + i);
      found[1] = left - above;
    }
    above += mine[i];
  }
  __syncthreads();
  const int2 r = make_int2(found[0], found[1]);
  __syncthreads();  // found may be written again
  return r;
}

// One CTA, or a cluster of them, per (sequence, KV head). The `want` best of the
// tokens between sink and the recent ones are found by a radix select over their ordered scores:
// a histogram of the first 11 bits gives the bin in which the want-th key lies;
// a second sweep over the scores notes for every token whether it is above that
// bin and lists the keys within; two more histograms (11 and 10 bits) over the
// list give the threshold and how many of the tokens equal to it are kept, the
// lowest indexes first; then the kept tokens are written in order from the notes.
// Scores are read four tokens at a time (pages are multiples of 16), each twice;
// a note is a byte per four tokens (above the threshold, at it). A sequence of
// more than `room` tokens is read again for the output, and so is one whose bin
// has more than kSelList keys (equal or close scores). 64 sequences of 4 to 36 Ki
// tokens, 8 heads: 43 us (40 where the L2 holds the scores already). That is latency
// before all: a CTA's sweeps follow one another behind barriers, each load of
// scores behind that of its page, with three CTAs an SM, and eight lists of 32k tokens
// on an empty GPU take 26 us with a CTA each. Warps issue in 46 % of the slots
// (24.5 M instructions, 115 a token counting all lanes and phases), 57 % on the SM
// with the most. Measured before: 75 us with all keys in shared memory and one CTA an
// SM, 52 with a byte's tokens written at a time and a branch a token, 79 with 256
// threads, 65 with 1024.
__global__ void __launch_bounds__(kSelThreads, 3)
    select_kernel(const float* __restrict__ scores, const SeqTable table,
                  int32_t* __restrict__ kept, int batch, int hkv, int budget, int sink,
                  int recent, int room, bool ranked, unsigned int* err) {
  extern __shared__ uint32_t notes32[];  // notes, four a word
  __shared__ __align__(16) int hist[kBins], hist1[kBins], hist2[kBins];
  __shared__ uint2 list[kSelList];  // key, token
  __shared__ int warp_sums[kSelWarps];
  __shared__ __align__(8) int counts[2];
  __shared__ int found[2], listed, ranks[kRankBatch];
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < kBins; i += kSelThreads) hist[i] = hist1[i] = hist2[i] = 0;
  if (tid == 0) listed = 0;
  const Cluster cl;
  const int lists_at = blockIdx.x / cl.size;
  pdl_wait();  // the scores come from, and the lists may come from, earlier kernels
  int b = lists_at / hkv, p0, n;
  const int h = lists_at % hkv;
  if (ranked) {  // the b-th longest sequence
    if (tid < kRankBatch) {
      int len = -1;
      if (tid < batch && !sequence(table, tid, p0, len)) len = 0;
      ranks[tid] = len;
    }
    __syncthreads();
    if (tid < batch) {
      const int len = ranks[tid];
      int longer = 0;
      for (int j = 0; j < batch; ++j) longer += ranks[j] > len || (ranks[j] == len && j < tid);
      if (longer == b) found[0] = tid;
    }
    __syncthreads();
    b = found[0];
  }
  int32_t* out = kept + (static_cast<int64_t>(b) * hkv + h) * budget;
  const int all_tid = cl.rank * kSelThreads + tid, all_threads = cl.size * kSelThreads;
  if (!sequence(table, b, p0, n)) {
    if (tid == 0 && h == 0) raise_device_error(err, FE_DEVERR_PAGE_RANGE);
    for (int i = all_tid; i < budget; i += all_threads) out[i] = -1;
    return;
  }
  if (n <= budget) {
    for (int i = all_tid; i < budget; i += all_threads) out[i] = i < n ? i : -1;
    return;
  }
  const int end = n - recent, want = budget - sink - recent;
  for (int i = all_tid; i < sink; i += all_threads) out[i] = i;
  for (int i = all_tid; i < recent; i += all_threads) out[budget - recent + i] = end + i;
  if (want == 0) return;
  const float* sc = scores + static_cast<int64_t>(h) * table.cache_slots;
  const int per16 = table.page / 16;
  // the page of tokens 4g .. 4g + 3, whose slots are adjacent, and their scores
  const int num_pages = static_cast<int>(table.cache_slots / table.page);
  uint8_t* notes = reinterpret_cast<uint8_t*>(notes32);  // of group 4 * wa on
  auto page_of = [&](int g) {
    return __ldg(table.pages + p0 + (per16 == 1 ? g >> 2 : (g >> 2) / per16));
  };
  auto load4 = [&](int g, int pg) -> float4 {
    if (static_cast<unsigned>(pg) >= static_cast<unsigned>(num_pages)) {
      raise_device_error(err, FE_DEVERR_PAGE_RANGE);
      const float least = __uint_as_float(0xffffffffu);
      return make_float4(least, least, least, least);
    }
    const int in = per16 == 1 ? g & 3 : g - (g >> 2) / per16 * per16 * 4;
    return __ldg(reinterpret_cast<const float4*>(sc + static_cast<int64_t>(pg) * table.page) + in);
  };
  auto keys = [&](const float4& x) {
    return make_uint4(ordered(x.x), ordered(x.y), ordered(x.z), ordered(x.w));
  };
  // this CTA's stretch of groups, in whole words of notes: [ga, gb), words from wa on
  const int first_word = sink / 16, end_word = (end + 15) / 16;
  const int part = (end_word - first_word + cl.size - 1) / cl.size;
  const int wa = min(end_word, first_word + static_cast<int>(cl.rank) * part);
  const int wb = min(end_word, wa + part);
  const int ga = max(4 * wa, sink / 4), gb = min(4 * wb, (end + 3) / 4);
  const bool noted = (wb - wa) * 16 <= room;
  if (noted && tid == 0 && wa < wb) {  // (the sweeps write the notes of [ga, gb) only)
    notes32[0] = 0;
    notes32[wb - 1 - wa] = 0;
  }
  // f(i, key) for the tokens 4g + i of a group that lie between sink and end
  auto each = [&](int g, const uint4& x, auto&& f) {
    const uint32_t v[4] = {x.x, x.y, x.z, x.w};
    // (the first and the last group may lie across the bounds)
    const int from = max(sink - 4 * g, 0), to = min(end - 4 * g, 4);
    if (to - from == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f(i, v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i >= from && i < to) f(i, v[i]);
    }
  };
  // groups in flight a thread; the pages of the next ones are there by then
  constexpr int kAhead = 2;
  auto sweep = [&](auto&& f) {
    int pg[kAhead];
    int g0 = ga + tid;
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      pg[u] = g0 + u * kSelThreads < gb ? page_of(g0 + u * kSelThreads) : 0;
    for (; g0 < gb; g0 += kAhead * kSelThreads) {
      float4 x[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (g0 + u * kSelThreads < gb) x[u] = load4(g0 + u * kSelThreads, pg[u]);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int g = g0 + (kAhead + u) * kSelThreads;
        if (g < gb) pg[u] = page_of(g);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (g0 + u * kSelThreads < gb) f(g0 + u * kSelThreads, keys(x[u]));
    }
  };
  __syncthreads();
  sweep([&](int g, const uint4& x) {
    each(g, x, [&](int, uint32_t k) { atomicAdd(&hist[k >> 21], 1); });
  });
  cl.sync();
  int2 at = find_bin(cl, hist, want, warp_sums, found);
  uint32_t prefix = static_cast<uint32_t>(at.x) << 21;
  int left = at.y;  // of the keys that begin with prefix
  const uint32_t bin_end = prefix | ((1u << 21) - 1);
  // ---- the rest of the threshold's bits, over the keys of its bin
  sweep([&](int g, const uint4& x) {
    uint32_t note = 0;
    each(g, x, [&](int i, uint32_t k) {
      note |= (k > bin_end ? 1u : k >= prefix ? 16u : 0u) << i;
    });
    const uint32_t in_bin = note >> 4;
    if (noted) notes[g - 4 * wa] = note & 15u;
    if (in_bin) {
      int at = atomicAdd(&listed, __popc(in_bin));
      const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!(in_bin >> i & 1)) continue;
        atomicAdd(&hist1[(v[i] >> 10) & 2047], 1);
        if (at < kSelList) list[at] = make_uint2(v[i], 4 * g + i);
        ++at;
      }
    }
  });
  cl.sync();
  const bool whole = listed <= kSelList;  // the list holds the bin
  const int count = min(listed, kSelList);
  at = find_bin(cl, hist1, left, warp_sums, found);
  prefix |= static_cast<uint32_t>(at.x) << 10;
  left = at.y;
  if (whole) {
    for (int i = tid; i < count; i += kSelThreads)
      if ((list[i].x >> 10) == (prefix >> 10)) atomicAdd(&hist2[list[i].x & 1023], 1);
  } else {
    sweep([&](int g, const uint4& x) {
      each(g, x, [&](int, uint32_t k) {
        if ((k >> 10) == (prefix >> 10)) atomicAdd(&hist2[k & 1023], 1);
      });
    });
  }
  cl.sync();
  at = find_bin(cl, hist2, left, warp_sums, found);
  prefix |= static_cast<uint32_t>(at.x);
  left = at.y;
  // ---- the notes against the threshold itself: bits 0-3 above it, 4-7 at it
  auto judge = [&](int g, const uint4& x) -> uint32_t {
    uint32_t note = 0;
    each(g, x, [&](int i, uint32_t k) {
      note |= (k > prefix ? 1u : k == prefix ? 16u : 0u) << i;
    });
    return note;
  };
  if (noted && whole) {
    for (int i = tid; i < count; i += kSelThreads) {
      const uint2 e = list[i];
      const uint32_t bit = (e.x > prefix ? 1u : e.x == prefix ? 16u : 0u) << (e.y & 3);
      const int g = (static_cast<int>(e.y) >> 2) - 4 * wa;
      if (bit) atomicOr(&notes32[g >> 2], bit << (8 * (g & 3)));
    }
  } else if (noted) {
    sweep([&](int g, const uint4& x) { notes[g - 4 * wa] = judge(g, x); });
  }
  __syncthreads();
  // ---- kept tokens in order: a warp owns a stretch of the groups, a lane four of
  // them at a time: sixteen tokens, bit t of `mg` / `me` token t above / at it
  const int per = ((wb - wa + kSelWarps - 1) / kSelWarps + 31) / 32 * 32;
  const int w0 = min(wb, wa + warp * per), w1 = min(wb, w0 + per);
  auto word = [&](int w, uint32_t& mg, uint32_t& me) {
    uint32_t x = 0;
    if (noted) {
      x = notes32[w - wa];
    } else {
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        const int g = 4 * w + i;
        if (g >= ga && g < gb) x |= judge(g, keys(load4(g, page_of(g)))) << (8 * i);
      }
    }
    auto nibbles = [](uint32_t y) {  // the low half of each byte, packed
      y &= 0x0f0f0f0fu;
      y |= y >> 4;
      return (y & 0xffu) | (y >> 8 & 0xff00u);
    };
    mg = nibbles(x);
    me = nibbles(x >> 4);
  };
  int gt = 0, eq = 0;
  for (int w = w0 + lane; w < w1; w += 32) {
    uint32_t mg, me;
    word(w, mg, me);
    gt += __popc(mg);
    eq += __popc(me);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    gt += __shfl_xor_sync(0xffffffffu, gt, o);
    eq += __shfl_xor_sync(0xffffffffu, eq, o);
  }
  int total_gt, total;
  int gt0 = block_scan(lane == 0 ? gt : 0, warp_sums, total_gt);
  int eq0 = block_scan(lane == 0 ? eq : 0, warp_sums, total);
  gt0 = __shfl_sync(0xffffffffu, gt0, 0);
  eq0 = __shfl_sync(0xffffffffu, eq0, 0);
  if (cl.size > 1) {  // what the CTAs before this one keep
    if (tid == 0) counts[0] = total_gt;
    if (tid == 0) counts[1] = total;
    cl.sync();
    for (uint32_t r = 0; r < cl.rank; ++r) {
      int x, y;
      asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];"
                   : "=r"(x), "=r"(y)
                   : "r"(Cluster::at(counts, r)));
      gt0 += x;
      eq0 += y;
    }
  }
  for (int wbase = w0; wbase < w1; wbase += 32) {
    const int w = wbase + lane;
    uint32_t mg = 0, me = 0;
    if (w < w1) word(w, mg, me);
    // counts of the lanes before: both in one sum (512 of each at most)
    const int mine = __popc(mg) | __popc(me) << 16;
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += y;
    }
    const int all = __shfl_sync(0xffffffffu, before, 31);
    before -= mine;
    int at_g = gt0 + (before & 0xffff), at_e = eq0 + (before >> 16);
    for (uint32_t m = mg | me; m; m &= m - 1) {
      const int t = __ffs(m) - 1;
      const bool same = me >> t & 1;
      if (!same || at_e < left) out[sink + at_g + min(at_e, left)] = 16 * w + t;
      at_g += !same;
      at_e += same;
    }
    gt0 += all & 0xffff;
    eq0 += all >> 16;
  }
  if (cl.size > 1) cl.sync();  // the others have read this CTA's shared memory
}

// ---------------------------------------------------------------------------
// compaction: for every sequence and KV head, the K and V rows and the score
// of token kept[j] move to token j, for every j before the list's first entry
// below 0. A CTA walks the list of one (sequence, head) in order, for one slice
// of the row's 16-byte chunks (slices give one sequence's move more CTAs). A
// table of the source and destination slots of kTableTokens tokens is made
// first, so that the moves wait for no index. Each step moves rows *
// kMoveUnroll tokens: all of them are read before any is written, and the
// sources of later steps lie at or past their own index (kept[j] >= j, checked),
// which no earlier step writes; so the move works in place.
// ---------------------------------------------------------------------------
constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 4;
constexpr int kTableTokens = kMoveThreads;

struct MoveArgs {
  uint4* k;
  uint4* v;
  float* scores;
  const int32_t* kept;
  SeqTable src, dst;
  int in_place;
  int hkv, budget, chunks;  // chunks: 16-byte chunks of a K (or V) row
  int slice;                // chunks of a CTA's slice, of K and of V each
  unsigned int* err;
};

__global__ void __launch_bounds__(kMoveThreads) compact_kernel(const MoveArgs a) {
  __shared__ int2 table[2][kTableTokens];  // source and destination slot, -1: no move
  __shared__ int ends[2][kMoveThreads / 32];  // a warp's first entry below 0
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x / a.hkv, h = blockIdx.x % a.hkv;
  const int lanes = 2 * a.slice;  // threads of a token
  const int row = threadIdx.x / lanes, c = threadIdx.x % lanes;
  const int rows = kMoveThreads / lanes;
  const bool idle = row >= rows;  // threads left over where lanes does not divide the block
  const bool is_v = c >= a.slice;
  const int chunk = blockIdx.y * a.slice + (is_v ? c - a.slice : c);
  const bool scoring = blockIdx.y == 0 && c == 0 && a.scores != nullptr;
  uint4* pool = (is_v ? a.v : a.k) + h * a.chunks + chunk;
  const int64_t slot_chunks = static_cast<int64_t>(a.hkv) * a.chunks;
  float* sc = a.scores + (a.scores ? static_cast<int64_t>(h) * a.src.cache_slots : 0);
  int p0, n, d0, dn;
  bool good = sequence(a.src, b, p0, n);
  if (a.in_place) {
    d0 = p0;
    dn = n;
  } else {
    d0 = __ldg(a.dst.kv + b);
    const int d1 = __ldg(a.dst.kv + b + 1);
    good &= d0 >= 0 && d1 >= d0 && d1 <= a.dst.num_pages;
    dn = good ? static_cast<int>(min(static_cast<int64_t>(d1 - d0) * a.src.page,
                                     static_cast<int64_t>(INT32_MAX)))
              : 0;
  }
  if (!good) {
    if (threadIdx.x == 0 && h == 0 && blockIdx.y == 0)
      raise_device_error(a.err, FE_DEVERR_PAGE_RANGE);
    return;
  }
  const int32_t* kept = a.kept + static_cast<int64_t>(blockIdx.x) * a.budget;
  int next = static_cast<int>(threadIdx.x) < a.budget ? __ldg(kept + threadIdx.x) : -1;
  int buf = 0;
  for (int base = 0; base < a.budget; base += kTableTokens, buf ^= 1) {
    const int j = base + threadIdx.x;
    bool bad = false;
    {
      const int t = next;
      const int jn = j + kTableTokens;
      next = jn < a.budget ? __ldg(kept + jn) : -1;
      int2 e = make_int2(-1, -1);
      if (t >= 0 && !(a.in_place && t == j)) {
        if (t < n && j < dn && (!a.in_place || t > j)) {
          e.x = static_cast<int>(slot_of(a.src, p0, t));
          e.y = static_cast<int>(slot_of(a.in_place ? a.src : a.dst, d0, j));
        }
        bad = e.x < 0 || e.y < 0;
        if (bad) e = make_int2(-1, -1);
      }
      table[buf][threadIdx.x] = e;
      const unsigned none = __ballot_sync(0xffffffffu, t < 0);  // (also past the budget)
      if ((threadIdx.x & 31) == 0)
        ends[buf][threadIdx.x >> 5] = none ? j + __ffs(none) - 1 : INT32_MAX;
    }
    // (Two buffers: this barrier also keeps the table before the last in use.)
    const bool moves = __syncthreads_or(table[buf][threadIdx.x].x >= 0);
    int end = INT32_MAX;  // the list ends at its first entry below 0
#pragma unroll
    for (int w = 0; w < kMoveThreads / 32; ++w) end = min(end, ends[buf][w]);
    if (bad && j < end && blockIdx.y == 0) raise_device_error(a.err, FE_DEVERR_PAGE_RANGE);
    // where nothing of these tokens moves: a prefix that stays
    const int count = moves ? min(kTableTokens, end - base) : 0;
    for (int j0 = 0; j0 < count; j0 += rows * kMoveUnroll) {
      int2 e[kMoveUnroll];
      uint4 x[kMoveUnroll];
      float s[kMoveUnroll];
#pragma unroll
      for (int u = 0; u < kMoveUnroll; ++u) {
        const int j = j0 + u * rows + row;
        e[u] = !idle && j < count ? table[buf][j] : make_int2(-1, -1);
        if (e[u].x < 0) continue;
        x[u] = pool[e[u].x * slot_chunks];
        if (scoring) s[u] = sc[e[u].x];
      }
      __syncthreads();  // everything of this step has been read
#pragma unroll
      for (int u = 0; u < kMoveUnroll; ++u) {
        if (e[u].x < 0) continue;
        pool[e[u].y * slot_chunks] = x[u];
        if (scoring) sc[e[u].y] = s[u];
      }
    }
    if (end < base + kTableTokens) break;
  }
}

int check_lists(const char* what, const int32_t* kv, const int32_t* pages, const int32_t* last,
                int num_pages, int batch, int hkv, int page, int budget, int64_t cache_slots) {
  const std::string name = what;
  if (batch < 0 || hkv <= 0 || budget < 0 || num_pages < 0)
    return fail(FE_ERR_INVALID_ARGUMENT, name + ": sizes out of range");
  if (page <= 0 || page % 16 != 0)
    return fail(FE_ERR_UNSUPPORTED, name + ": page must be a multiple of 16");
  if (cache_slots <= 0 || cache_slots % page != 0 || cache_slots >= INT32_MAX)
    return fail(FE_ERR_INVALID_ARGUMENT,
                name + ": cache_slots must be whole pages, below 2^31");
  if (int64_t(batch) * hkv > INT32_MAX)
    return fail(FE_ERR_CAPACITY, name + ": batch x hkv too large");
  // (the kernels' indexes of an entry go a block's threads past the last)
  if (budget > (1 << 30)) return fail(FE_ERR_CAPACITY, name + ": budget above 2^30");
  if (batch > 0 && budget > 0 && (!kv || !pages || !last))
    return fail(FE_ERR_INVALID_ARGUMENT, name + ": null pointer");
  return FE_OK;
}

}  // namespace
}  // namespace fe

using namespace fe;

extern "C" {

int fe_kv_select(const float* scores, const int32_t* kv, const int32_t* pages, int num_pages,
                 const int32_t* last, int32_t* kept, int batch, int max_len, int hkv, int page,
                 int budget, int sink, int recent, int64_t cache_slots, void* stream) {
  int rc = check_lists("fe_kv_select", kv, pages, last, num_pages, batch, hkv, page, budget,
                       cache_slots);
  if (rc != FE_OK) return rc;
  if (sink < 0 || recent < 0 || int64_t(sink) + recent > budget)
    return fail(FE_ERR_INVALID_ARGUMENT,
                "fe_kv_select: sink and recent must be non-negative and fit the budget");
  if (max_len < 0) return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv_select: max_len < 0");
  if (batch == 0 || budget == 0) return FE_OK;
  if (!scores || !kept) return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv_select: null pointer");
  if (!aligned16(scores))
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv_select: scores must be 16-byte aligned");
  if (!aligned4(kept))
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv_select: kept must be 4-byte aligned");
  const SeqTable table{kv, pages, last, num_pages, page, cache_slots};
  auto s = static_cast<cudaStream_t>(stream);
  static std::atomic<uint64_t> done{0};
  FE_CUDA_TRY(allow_smem(select_kernel, kSelRoom / 4, done));
  // more lists than SMs: the longest first, so that the last to end are short. Not
  // for large batches, where a CTA's look at all lengths costs more than it gives.
  const int lists = batch * hkv;
  const bool ranked = batch <= kRankBatch && lists > 148;
  // few long lists: a cluster of CTAs each, of at least kSelPart tokens a CTA (8 lists
  // of 32k tokens 25.7 us with one CTA each, 16.6 with eight; of 8k 11.0 with one,
  // 11.7 with four, 16.1 with eight; 512 lists 40 us with one, 53 with two)
  int cluster = 1;
  while (cluster < kSelCluster && lists * cluster * 2 <= kSelCtas &&
         max_len >= 2 * cluster * kSelPart)
    cluster *= 2;
  const int room = std::min(std::min(max_len / cluster, kSelRoom) + 32, kSelRoom);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(lists * cluster);
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(room + 15) / 16 * 4;
  cfg.stream = s;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  FE_CUDA_TRY(cudaLaunchKernelEx(&cfg, select_kernel, scores, table, kept, batch, hkv, budget,
                                 sink, recent, room, ranked, device_error_word()));
  return FE_OK;
}

int fe_kv_compact(void* k_pool, void* v_pool, float* scores, const int32_t* kept,
                  const int32_t* kv, const int32_t* pages, int num_pages, const int32_t* last,
                  const int32_t* dst_kv, const int32_t* dst_pages, int num_dst_pages, int batch,
                  int hkv, int dim, int page, int budget, int dtype, int64_t cache_slots,
                  void* stream) {
  if (!valid_dtype(dtype)) return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv_compact: bad dtype");
  int rc = check_lists("fe_kv_compact", kv, pages, last, num_pages, batch, hkv, page, budget,
                       cache_slots);
  if (rc != FE_OK) return rc;
  if (dim <= 0 || dim % 8 != 0 || dim > 512)
    return fail(FE_ERR_UNSUPPORTED, "fe_kv_compact: dim must be a multiple of 8, at most 512");
  if ((dst_kv == nullptr) != (dst_pages == nullptr) || num_dst_pages < 0)
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv_compact: dst_kv and dst_pages go together");
  if (batch == 0 || budget == 0) return FE_OK;
  if (!k_pool || !v_pool || !kept)
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv_compact: null pointer");
  if (!aligned16(k_pool) || !aligned16(v_pool))
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv_compact: pools must be 16-byte aligned");
  if (!aligned4(scores) || !aligned4(kept))
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv_compact: scores and kept must be 4-byte aligned");
  MoveArgs a{};
  a.k = static_cast<uint4*>(k_pool);
  a.v = static_cast<uint4*>(v_pool);
  a.scores = scores;
  a.kept = kept;
  a.src = SeqTable{kv, pages, last, num_pages, page, cache_slots};
  a.dst = SeqTable{dst_kv, dst_pages, nullptr, num_dst_pages, page, cache_slots};
  a.in_place = dst_kv == nullptr;
  a.hkv = hkv;
  a.budget = budget;
  a.chunks = dim / 8;
  a.err = device_error_word();
  // slices of whole 32-byte sectors while there are fewer CTAs than SMs take
  const int64_t lists = int64_t(batch) * hkv;
  a.slice = a.chunks;
  while (a.slice % 4 == 0 && lists * (a.chunks / a.slice) < 512) a.slice /= 2;
  FE_CUDA_TRY(launch_pdl(compact_kernel, dim3(static_cast<unsigned>(lists), a.chunks / a.slice),
                         dim3(kMoveThreads), 0, static_cast<cudaStream_t>(stream), a));
  return FE_OK;
}

}  // extern "C"
