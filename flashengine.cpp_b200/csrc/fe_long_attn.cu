// Attention for long shared prompts over the paged cache: sequences that begin
// with the same pages (the prefix read once for all of them), and attention
// that scores every cached key by the weight it got. No counterpart in the
// reference, whose attention reads each sequence's pages by itself
// (Cambridgebit/FlashEngine.cpp src/flashinfer_attention.cu:35-44).
//
// Both run over the lists of fe_long_plan.h: up to 16 packed rows by the key kernel
// (fe_keys.cu; at head_dim 256 the decode kernel, fe_decode.cu), more rows of the
// shared plans by a row kernel (fe_rows2_tc.cu; at 256 fe_prefill_tc.cu). Scored plans
// cut their rows into blocks of 16 and run no row kernel. A record holds, for each of
// its rows, m = the largest base-2 score of its keys, l = sum 2^(s - m) and
// O = sum 2^(s - m) v; records of disjoint keys join as
//   m = max m_i, l = sum l_i 2^(m_i - m), out = sum O_i 2^(m_i - m) / l.
// The weight of a key with score s is then 2^(s - m) / l. (2^(s - (m + log2 l)) loses
// log2 l to the rounding of m + log2 l where scores are large: with |m| = 2^23 the
// weights of equal keys are up to 4 % off, with 2^28 each of 700 weighs 1.)
#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <string>
#include <vector>

#include "fe_attn_common.cuh"
#include "fe_long_plan.h"
#include "fe_tensor_maps.h"

namespace fe {

int decode_ext_launch(int dtype, int heads, const CUtensorMap& kmap, const CUtensorMap& vmap,
                      bool per_head_tma, const void* args, int grid, cudaStream_t stream);
int keys_launch(int dtype, const CUtensorMap& kmap, const CUtensorMap& vmap, const void* args,
                int grid, bool beside, cudaStream_t stream);
int rows2_launch(int dtype, const CUtensorMap& kmap, const CUtensorMap& vmap,
                 const CUtensorMap& qmap, const void* args, int grid, cudaStream_t stream);
int prefill_tc_ext_launch(int dtype, const CUtensorMap& kmap, const CUtensorMap& vmap,
                          const CUtensorMap& qmap, const void* args, int grid,
                          cudaStream_t stream);

namespace {

constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;
constexpr int kScoreThreads = 128;

// The records of one row: n of them, rec_floats apart.
struct Records {
  const float* first;
  int n, rec_floats, rows, row;
};

// Unit and record row of packed row p (of P a KV head) for KV head h.
template <int D>
__device__ __forceinline__ int unit_of(int unit, int blocks, int p, int P, int h, int H,
                                       int& row) {
  if (blocks > 0) {
    row = p % row_item_rows(D);
    return unit + h * blocks + p / row_item_rows(D);
  }
  row = (h % H) * P + p;
  return unit + h / H;
}

__device__ __forceinline__ Records records_of(const UnitRec& u, const float* partials, int row) {
  return Records{partials + u.part0, u.n, u.rec_floats, u.rows, row};
}

template <int D>
__device__ __forceinline__ const float* record(const Records& a, const Records& b, int i,
                                               int& rows, int& row) {
  const bool second = i >= a.n;
  rows = second ? b.rows : a.rows;
  row = second ? b.row : a.row;
  return second ? b.first + static_cast<int64_t>(i - a.n) * b.rec_floats
                : a.first + static_cast<int64_t>(i) * a.rec_floats;
}

// One warp joins the records of one row and stores its 16-bit output. What
// bounds it is the way to the L2 and back, so the loads of kStep records, their
// (m, l) among them, go out together.
template <typename T, int D, int kStep>
__device__ __forceinline__ void join_row(const Records& a, const Records& b, int lane, T* out,
                                         float2* norm) {
  constexpr int kV = D / 128;  // float4 vectors per lane
  const int n = a.n + b.n;
  float4 acc[kV];
#pragma unroll
  for (int v = 0; v < kV; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  float M = -INFINITY, L = 0.f;
  for (int s0 = 0; s0 < n; s0 += kStep) {
    float m[kStep], l[kStep];
    float4 x[kStep][kV];
#pragma unroll
    for (int j = 0; j < kStep; ++j) {
      m[j] = -INFINITY;
      l[j] = 0.f;
#pragma unroll
      for (int v = 0; v < kV; ++v) x[j][v] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s0 + j < n) {
        int rows, row;
        const float* rec = record<D>(a, b, s0 + j, rows, row);
        m[j] = __ldcg(rec + rows * D + row);
        l[j] = __ldcg(rec + rows * (D + 1) + row);
#pragma unroll
        for (int v = 0; v < kV; ++v)
          x[j][v] = __ldcg(reinterpret_cast<const float4*>(rec + row * D + v * 128 + lane * 4));
      }
    }
    float top = M;
#pragma unroll
    for (int j = 0; j < kStep; ++j) top = fmaxf(top, m[j]);
    const float base = top == -INFINITY ? 0.f : top;
    const float resc = M == -INFINITY ? 0.f : fast_exp2(M - base);
    M = top;
    L *= resc;
#pragma unroll
    for (int v = 0; v < kV; ++v) {
      acc[v].x *= resc;
      acc[v].y *= resc;
      acc[v].z *= resc;
      acc[v].w *= resc;
    }
#pragma unroll
    for (int j = 0; j < kStep; ++j) {
      if (s0 + j >= n) break;
      const float w = fast_exp2(m[j] - base);
      L = fmaf(l[j], w, L);
#pragma unroll
      for (int v = 0; v < kV; ++v) {
        acc[v].x = fmaf(x[j][v].x, w, acc[v].x);
        acc[v].y = fmaf(x[j][v].y, w, acc[v].y);
        acc[v].z = fmaf(x[j][v].z, w, acc[v].z);
        acc[v].w = fmaf(x[j][v].w, w, acc[v].w);
      }
    }
  }
  const float inv = 1.f / L;
#pragma unroll
  for (int v = 0; v < kV; ++v)
    store4<T>(out + v * 128 + lane * 4, acc[v].x * inv, acc[v].y * inv, acc[v].z * inv,
              acc[v].w * inv);
  if (norm && lane == 0) *norm = make_float2(M, inv);
}

// The records of query row w / hq, head w % hq: the plan's metadata alone, complete
// before the kernels ahead began.
template <typename T, int D>
__device__ __forceinline__ void find_records(const AttnArgs<T>& a, int64_t w, Records& own,
                                             Records& pre) {
  const MetaHeader* hdr = reinterpret_cast<const MetaHeader*>(a.meta);
  const int r = static_cast<int>(w / a.hq), head = static_cast<int>(w % a.hq);
  const int H = hdr->dec_heads, h = head / a.G;
  own = pre = Records{nullptr, 0, 0, 0, 0};
  if (r >= hdr->rows) return;
  const RowInfo x = reinterpret_cast<const RowInfo*>(a.meta + hdr->row_info_off)[r];
  const UnitRec* units = reinterpret_cast<const UnitRec*>(a.meta + hdr->unit_off[a.view]);
  int row;
  if (x.own_unit >= 0) {
    const int u = unit_of<D>(x.own_unit, x.own_blocks, x.own_p + head % a.G, x.own_rows, h, H,
                             row);
    own = records_of(units[u], a.partials, row);
  }
  if (x.pre_unit >= 0) {
    const int u = unit_of<D>(x.pre_unit, x.pre_blocks, x.pre_p + head % a.G, x.pre_rows, h, H,
                             row);
    pre = records_of(units[u], a.partials, row);
  }
}

// One warp per query row and head; norms (scored plans): where (m, 1 / l) of each
// goes, [rows, hq]. A warp has kStep records in flight: with few pairs of row and
// head all warps are resident and four shorten each one's chain of loads; with many
// what counts are loads in flight an SM, and two leave registers for more warps.
// Whole calls in us with four and with two at head_dim 128: 4 rows of 16 heads 7.2
// and 7.8, 128 rows of 32 heads 21.6 and 22.6, 64 rows of 64 heads 68.0 and 68.3,
// 2048 rows of 32 heads (many pairs) 113.1 and 111.5.
constexpr int kManyPairs = 148 * 48;

template <typename T, int D, int kStep>
__global__ void __launch_bounds__(kJoinThreads, kStep == 2 && D == kHeadDim ? 5 : 4)
    join_kernel(const AttnArgs<T> a, float2* norms) {
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * kJoinWarps + (threadIdx.x >> 5);
  Records own, pre;
  find_records<T, D>(a, w, own, pre);
  pdl_wait();
  if (own.n > 0)  // else written by its unit
    join_row<T, D, kStep>(own, pre, lane, a.out + w * D, norms ? norms + w : nullptr);
}

template <typename T, int D>
int launch_join(const AttnArgs<T>& a, int rows, float2* norms, cudaStream_t s) {
  const int64_t pairs = int64_t(rows) * a.hq;
  const int grid = static_cast<int>((pairs + kJoinWarps - 1) / kJoinWarps);
  auto kernel = pairs > kManyPairs ? join_kernel<T, D, 2> : join_kernel<T, D, 4 * kHeadDim / D>;
  FE_CUDA_TRY(launch_pdl(kernel, dim3(grid), dim3(kJoinThreads), 0, s, a, norms));
  return FE_OK;
}

template <typename T>
int launch_join(const AttnArgs<T>& a, int dim, int rows, float2* norms, cudaStream_t s) {
  return dim == kWideHeadDim ? launch_join<T, kWideHeadDim>(a, rows, norms, s)
                             : launch_join<T, kHeadDim>(a, rows, norms, s);
}

// Scored plans, behind the join: the weights of kScoreChunk keys of one KV head
// at a time, 2^(raw score - m) / l summed over the packed rows in order, go to the
// keys' scores. Grid: chunks x KV heads.
__global__ void __launch_bounds__(kScoreThreads, 8)
    score_kernel(const uint8_t* __restrict__ meta, const float* __restrict__ raw_scores,
                 const float2* __restrict__ norms, float* __restrict__ scores, int hq, int hkv,
                 int page, int64_t cache_slots) {
  constexpr int kPer = kScoreChunk / kScoreThreads;  // keys a thread
  pdl_trigger();
  const MetaHeader* hdr = reinterpret_cast<const MetaHeader*>(meta);
  const ScoreChunk* chunks = reinterpret_cast<const ScoreChunk*>(meta + hdr->chunk_off);
  const SeqInfo* seqs = reinterpret_cast<const SeqInfo*>(meta + hdr->seqs_off);
  const int64_t* sink = reinterpret_cast<const int64_t*>(meta + hdr->sink_off);
  const int32_t* pages = reinterpret_cast<const int32_t*>(meta + hdr->pages_off);
  const int total = hdr->n_chunks, G = hq / hkv, h = blockIdx.y;
  float* out = scores + h * cache_slots;
  bool waited = false;
  for (int e = blockIdx.x; e < total; e += gridDim.x) {
    const ScoreChunk c = chunks[e];
    float w[kPer];
    int64_t at[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      w[i] = 0.f;
      const int t = c.t0 + i * kScoreThreads + threadIdx.x;
      const unsigned pg = static_cast<unsigned>(t) / static_cast<unsigned>(page);
      at[i] = t < c.length ? static_cast<int64_t>(__ldg(pages + c.page_off + pg)) * page +
                                 (t - static_cast<int>(pg) * page)
                           : -1;
    }
    SeqInfo si = seqs[c.block0];
    int64_t raw0 = sink[c.block0];
    if (!waited) pdl_wait();
    waited = true;
    float old[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int t = c.t0 + i * kScoreThreads + threadIdx.x;
      old[i] = at[i] >= 0 && t < c.fresh ? out[at[i]] : 0.f;
    }
    for (int j = 0;;) {
      if (c.t0 < si.length) {  // else the block's rows do not see this far
        const int P = si.qrows * G, cols = (P + 1) & ~1;
        const int tiles = (si.length + kTileTokens - 1) / kTileTokens;
        const float* raw = raw_scores + raw0 + static_cast<int64_t>(h) * tiles * kTileTokens * cols;
        const float2* row = norms + static_cast<int64_t>(si.q_row0) * hq + h * G;
        const float* at_key = raw + static_cast<int64_t>(c.t0 + threadIdx.x) * cols;
        const int stride = kScoreThreads * cols;
        int g = 0;  // packed row p is head g of the query row that `row` points at
        for (int p = 0; p < P; p += 4, at_key += 4) {  // four rows' scores of a key at once
          float2 c4[4];  // (m, 1 / l) of the four rows
          float2 s0[kPer], s1[kPer];
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            s0[i] = s1[i] = make_float2(-INFINITY, -INFINITY);
            if (c.t0 + i * kScoreThreads + static_cast<int>(threadIdx.x) < si.length) {
              const float2* x = reinterpret_cast<const float2*>(at_key + i * stride);
              s0[i] = __ldcg(x);
              if (p + 2 < P) s1[i] = __ldcg(x + 1);
            }
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            c4[r] = p + r < P ? __ldcg(row + g) : make_float2(INFINITY, 0.f);
            if (++g == G) {
              g = 0;
              row += hq;
            }
          }
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            w[i] = fmaf(fast_exp2(s0[i].x - c4[0].x), c4[0].y, w[i]);
            if (p + 1 < P) w[i] = fmaf(fast_exp2(s0[i].y - c4[1].x), c4[1].y, w[i]);
            if (p + 2 < P) w[i] = fmaf(fast_exp2(s1[i].x - c4[2].x), c4[2].y, w[i]);
            if (p + 3 < P) w[i] = fmaf(fast_exp2(s1[i].y - c4[3].x), c4[3].y, w[i]);
          }
        }
      }
      if (++j >= c.blocks) break;
      si = seqs[c.block0 + j];
      raw0 = sink[c.block0 + j];
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (at[i] >= 0) out[at[i]] = old[i] + w[i];
  }
  if (!waited) pdl_wait();
}

}  // namespace
}  // namespace fe

using namespace fe;

// What a step's kernels read and write of the plan: its lists, and records of up to
// `floats`.
struct LongSpace {
  uint8_t* meta = nullptr;
  float* partials = nullptr;
  int64_t floats = 0;
};

struct fe_long_plan {
  PlanConfig cfg{};
  int dtype = 0;
  bool scored = false, host_only = false;
  bool keys = false;  // the decode list is the key kernel's
  int device = -1;
  // The first serves most steps; later, larger ones the steps with more query rows.
  // None is freed before the plan, as a captured run keeps the one that it was
  // captured with, and a step takes the first that it fits, so that a graph's later
  // steps come to the same one.
  std::vector<LongSpace> spaces;
  size_t space = 0;  // of the last prepare
  size_t meta_cap = 0;
  float* d_sink = nullptr;
  float2* d_norms = nullptr;  // scored plans: (m, 1 / l) of each query row and head
  int64_t max_rows = 0;
  int64_t sink_floats = 0;
  // pinned staging, double-buffered
  uint8_t* h_meta[2] = {nullptr, nullptr};
  size_t h_cap[2] = {0, 0};
  cudaEvent_t h_ev[2] = {nullptr, nullptr};
  bool h_used[2] = {false, false};
  int h_idx = 0;
  bool prepared = false, fixed_grid = false, graph_shape_set = false;
  int graph_batch = 0, graph_rows = 0;
  LongResult last;
  // tensor maps of the pools last seen (row kernel, decode kernel)
  CUtensorMap kmap_tc, vmap_tc, kmap_dec, vmap_dec;
  const void* kmap_ptr = nullptr;
  const void* vmap_ptr = nullptr;
  bool per_head_tma = false;
};

namespace {

constexpr int kKeyWarps = 8;  // CTAs (of one warp) of the key kernel an SM
constexpr int64_t kLongPartialFloats = int64_t(64) << 20;  // 256 MiB

void destroy_long(fe_long_plan* p) {
  if (!p) return;
  if (!p->host_only) {
    for (int i = 0; i < 2; ++i) {
      if (p->h_ev[i]) {
        cudaEventSynchronize(p->h_ev[i]);
        cudaEventDestroy(p->h_ev[i]);
      }
      if (p->h_meta[i]) cudaFreeHost(p->h_meta[i]);
    }
    for (const LongSpace& x : p->spaces) {
      if (x.meta) cudaFree(x.meta);
      if (x.partials) cudaFree(x.partials);
    }
    if (p->d_sink) cudaFree(p->d_sink);
    if (p->d_norms) cudaFree(p->d_norms);
  }
  delete p;
}

cudaError_t add_space(fe_long_plan* p, int64_t floats) {
  LongSpace x;
  x.floats = floats;
  cudaError_t e = cudaMalloc(&x.partials, sizeof(float) * floats);
  if (e == cudaSuccess) e = cudaMalloc(&x.meta, p->meta_cap);
  if (e == cudaSuccess) try {
      p->spaces.push_back(x);
      return e;
    } catch (const std::bad_alloc&) {
      e = cudaErrorMemoryAllocation;
    }
  if (x.meta) cudaFree(x.meta);
  if (x.partials) cudaFree(x.partials);
  return e;
}

int create_long(const char* what, int hq, int hkv, int dim, int page, int max_batch,
                int max_pages, int dtype, int num_blocks, bool scored, int64_t max_keys,
                int host_ctas, fe_long_plan** plan_out) {
  const std::string name = what;
  if (!plan_out) return fail(FE_ERR_INVALID_ARGUMENT, name + ": plan_out is null");
  *plan_out = nullptr;
  if (!valid_dtype(dtype)) return fail(FE_ERR_INVALID_ARGUMENT, name + ": bad dtype");
  if (dim != kHeadDim && dim != kWideHeadDim)
    return fail(FE_ERR_UNSUPPORTED, name + ": head_dim must be 128 or 256");
  if (hq <= 0 || hkv <= 0 || hq % hkv != 0 || hq / hkv > kRowBlock || hkv > 32767)
    return fail(FE_ERR_UNSUPPORTED, name + ": need hq % hkv == 0 and hq/hkv <= 16");
  if (page <= 0 || page % kTileTokens != 0)
    return fail(FE_ERR_UNSUPPORTED, name + ": page must be a multiple of 16");
  if (max_batch <= 0 || max_pages <= 0 || num_blocks <= 0 || max_keys < 0)
    return fail(FE_ERR_INVALID_ARGUMENT, name + ": sizes must be positive");
  if (int64_t(num_blocks + int64_t(1)) * page >= INT32_MAX)
    return fail(FE_ERR_INVALID_ARGUMENT, name + ": (num_blocks+1)*page overflows");
  if (int64_t(max_batch) * max_pages >= INT32_MAX / 4)
    return fail(FE_ERR_CAPACITY, name + ": max_batch*max_pages too large");
  const int G = hq / hkv;
  if (max_keys > (int64_t(1) << 40) / (int64_t(hkv) * (G + 1)))
    return fail(FE_ERR_CAPACITY, name + ": max_keys too large");
  int sms = host_ctas;
  int dev = -1;
  if (!host_ctas) {
    FE_CUDA_TRY(cudaGetDevice(&dev));
    int major = 0;
    FE_CUDA_TRY(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
    FE_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    if (major != 10) return fail(FE_ERR_NO_DEVICE, name + ": needs an sm_100 (B200) device");
  }
  auto* p = new (std::nothrow) fe_long_plan();
  if (!p) return fail(FE_ERR_INVALID_ARGUMENT, name + ": out of host memory");
  p->host_only = host_ctas > 0;
  p->dtype = dtype;
  p->scored = scored;
  p->device = dev;
  PlanConfig& c = p->cfg;
  c.hq = hq;
  c.hkv = hkv;
  c.dim = dim;
  c.page = page;
  c.max_batch = max_batch;
  c.max_pages = max_pages;
  c.num_blocks = num_blocks;
  c.grid_cap = c.dec_grid_cap = sms;
  c.dec_heads = 8;
  while (hkv % c.dec_heads) c.dec_heads >>= 1;
  if (dim == kWideHeadDim) c.dec_heads = hkv % 2 == 0 ? 2 : 1;
  p->keys = dim == kHeadDim;
  if (p->keys) {
    c.dec_heads = 1;
    c.dec_grid_cap = kKeyWarps * sms;
  }
  c.row_group_blocks = 8;
  c.row_tile = dim == kWideHeadDim ? 4 : 8;
  // measured: a 128-key tile of the two-stream kernel 2.0 us for 256 rows, 1.4 us for
  // 128; of the head_dim 256 kernel (64 keys) 1.6 us; an item about 4 us more
  c.row_weight[0] = dim == kHeadDim ? 6 : 8;
  c.row_weight[1] = 12;
  c.row_item_tiles = 20;  // in fifths of a microsecond, as the weights
  c.row_pair_blocks = dim == kHeadDim ? 8 : 0;
  c.row_min_piece = 2;
  c.elem_bytes = 2;
  c.dec_min_tiles = 4;
  const size_t list_heads = 3 * (4 * size_t(c.dec_grid_cap + 1) + 64) + 4096;
  if (scored) {
    // every query row of a key or score is rounded up to an even number of columns
    p->sink_floats = max_keys * hkv * (G + (G & 1));
    // What max_keys lets a step have. Query rows: each sees a block of 16 keys at
    // least, and the i-th of a sequence i keys, so that R rows of B sequences have
    // R^2 / 2 B of them. Row blocks: full ones, and one more a sequence. Items: a
    // block's KV heads, and a cut at the end of each CTA's share.
    const double pairs = double(max_keys) * (G + (G & 1)) / G;
    p->max_rows = std::min<int64_t>(max_keys / kTileTokens,
                                    int64_t(std::sqrt(2.0 * max_batch * pairs)) + 1);
    const int64_t blocks = std::min(p->max_rows, p->max_rows / (kRowBlock / G) + max_batch);
    const int64_t units = std::min<int64_t>(blocks * (hkv / c.dec_heads), 1 << 28);
    c.max_groups = static_cast<int>(units);
    c.max_items = static_cast<int>(units + c.dec_grid_cap);
    c.partial_capacity = INT32_MAX;  // offsets of records; the workspace grows (hold_records)
    // decode list, units twice, row blocks, query rows, chunks, pages
    p->meta_cap = size_t(c.max_items) * (sizeof(WorkItem) + sizeof(KeyItem)) +
                  size_t(units) * (sizeof(SplitGroup) + 2 * sizeof(UnitRec)) +
                  size_t(blocks) * (sizeof(SeqInfo) + 8) + size_t(p->max_rows) * sizeof(RowInfo) +
                  sizeof(ScoreChunk) * size_t(max_batch) *
                      (size_t(max_pages) * page / kScoreChunk + 1) +
                  4 * size_t(max_batch) * max_pages + list_heads;
    p->meta_cap = std::min(p->meta_cap, size_t(INT32_MAX));  // offsets within it
  } else {
    c.max_items = c.max_groups = static_cast<int>(std::min<int64_t>(
        std::max<int64_t>(int64_t(max_batch) * hkv * 64, 8192), 1 << 20));
    c.partial_capacity = kLongPartialFloats;
    // lists (cta offsets, items, groups) three times, units twice, sequences and
    // prefixes, query rows, pages
    const size_t n = c.max_items;
    p->meta_cap = n * sizeof(KeyItem) + 3 * n * (sizeof(WorkItem) + sizeof(SplitGroup)) +
                  2 * sizeof(UnitRec) * n + n * (sizeof(SeqInfo) + 8) + sizeof(RowInfo) * 16 * n +
                  2 * size_t(max_batch) * sizeof(SeqInfo) + 4 * size_t(max_batch) * max_pages +
                  list_heads;
  }
  *plan_out = p;
  if (p->host_only) return FE_OK;
  cudaError_t e = add_space(p, kLongPartialFloats);
  if (e == cudaSuccess) e = cudaMemset(p->spaces[0].meta, 0, sizeof(MetaHeader));
  if (e == cudaSuccess && p->sink_floats > 0)
    e = cudaMalloc(&p->d_sink, sizeof(float) * p->sink_floats);
  if (e == cudaSuccess && p->max_rows > 0)
    e = cudaMalloc(&p->d_norms, sizeof(float2) * p->max_rows * hq);
  for (int i = 0; i < 2 && e == cudaSuccess; ++i) {
    p->h_cap[i] = std::min<size_t>(p->meta_cap, size_t(256) << 10);  // grows with the steps
    e = cudaMallocHost(&p->h_meta[i], p->h_cap[i]);
    if (e == cudaSuccess) e = cudaEventCreateWithFlags(&p->h_ev[i], cudaEventDisableTiming);
  }
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  if (e != cudaSuccess) {
    destroy_long(p);
    *plan_out = nullptr;
    return cuda_fail(e, (name + ": workspace allocation").c_str());
  }
  return FE_OK;
}

// The space for a step: by the records that it needs, those of a graph's later steps
// (as many query rows, cut in other places) among them. Nothing of the plan's
// current step changes.
int find_space(fe_long_plan* p, const LongResult& res, int batch, int rows, int graph,
               const std::string& name, size_t& space) {
  const PlanConfig& c = p->cfg;
  int64_t need = res.partial_floats;
  if (graph) {
    const int64_t per = kRowBlock / (c.hq / c.hkv), H = c.dec_heads;
    const int64_t units = std::min<int64_t>(rows, rows / per + batch) * (c.hkv / H);
    need = int64_t(rows) * c.hq * (c.dim + 2) + 3 * (units + c.dec_grid_cap) +
           int64_t(c.dec_grid_cap) * H * kRowBlock * (c.dim + 2);
    need = std::min<int64_t>(need, INT32_MAX);
  }
  for (space = 0; space < p->spaces.size(); ++space)
    if (need <= p->spaces[space].floats) return FE_OK;
  const cudaError_t e = add_space(
      p, std::min<int64_t>(std::max(need, 2 * p->spaces.back().floats), INT32_MAX));
  if (e != cudaSuccess) return cuda_fail(e, (name + ": workspace of more query rows").c_str());
  return FE_OK;
}

// Upload a step's metadata and take it as the plan's current one.
int install(fe_long_plan* p, LongResult& res, size_t space, int batch, int rows, int graph,
            const std::string& name, void* stream) {
  if (res.meta.size() > p->meta_cap)
    return fail(FE_ERR_CAPACITY, name + ": metadata exceeds workspace");
  if (!p->host_only) {
    auto s = static_cast<cudaStream_t>(stream);
    const int i = p->h_idx;
    if (p->h_used[i]) FE_CUDA_TRY(cudaEventSynchronize(p->h_ev[i]));
    if (res.meta.size() > p->h_cap[i]) {
      uint8_t* more = nullptr;
      const size_t cap = std::min(p->meta_cap, 2 * res.meta.size());
      FE_CUDA_TRY(cudaMallocHost(&more, cap));
      cudaFreeHost(p->h_meta[i]);
      p->h_meta[i] = more;
      p->h_cap[i] = cap;
    }
    std::memcpy(p->h_meta[i], res.meta.data(), res.meta.size());
    FE_CUDA_TRY(cudaMemcpyAsync(p->spaces[space].meta, p->h_meta[i], res.meta.size(),
                                cudaMemcpyHostToDevice, s));
    FE_CUDA_TRY(cudaEventRecord(p->h_ev[i], s));
    p->h_used[i] = true;
    p->h_idx ^= 1;
  }
  p->last = std::move(res);
  p->space = space;
  p->prepared = true;
  p->fixed_grid = graph != 0;
  if (graph) {
    p->graph_shape_set = true;
    p->graph_batch = batch;
    p->graph_rows = rows;
  }
  return FE_OK;
}

int check_prepare(const fe_long_plan* p, bool scored, int batch, int rows, int graph,
                  const std::string& name) {
  if (!p) return fail(FE_ERR_INVALID_ARGUMENT, name + ": plan is null");
  if (p->scored != scored)
    return fail(FE_ERR_INVALID_ARGUMENT, name + ": a plan of the other kind");
  if (graph && p->graph_shape_set && (p->graph_batch != batch || p->graph_rows != rows))
    return fail(FE_ERR_INVALID_ARGUMENT, name + ": graph plan batch/rows changed since capture");
  return FE_OK;
}

int check_run(const fe_long_plan* p, bool scored, const std::string& name) {
  if (!p) return fail(FE_ERR_INVALID_ARGUMENT, name + ": plan is null");
  if (p->host_only) return fail(FE_ERR_INVALID_ARGUMENT, name + ": host-only plan");
  if (p->scored != scored)
    return fail(FE_ERR_INVALID_ARGUMENT, name + ": a plan of the other kind");
  if (!p->prepared) return fail(FE_ERR_INVALID_ARGUMENT, name + ": plan not prepared");
  int dev = 0;
  FE_CUDA_TRY(cudaGetDevice(&dev));
  if (dev != p->device)
    return fail(FE_ERR_INVALID_ARGUMENT, name + ": the plan is for another device");
  return FE_OK;
}

int check_buffers(const void* q, const void* k_pool, const void* v_pool, const void* out,
                  const std::string& name) {
  if (!q || !k_pool || !v_pool || !out)
    return fail(FE_ERR_INVALID_ARGUMENT, name + ": null pointer");
  if (!aligned16(q) || !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(out))
    return fail(FE_ERR_INVALID_ARGUMENT, name + ": buffers must be 16-byte aligned");
  return FE_OK;
}

// Tensor maps of the pools, encoded once per address.
int maps(fe_long_plan* p, const void* k_pool, const void* v_pool) {
  const PlanConfig& c = p->cfg;
  const int64_t slots = int64_t(c.num_blocks + 1) * c.page;
  if (k_pool == p->kmap_ptr && v_pool == p->vmap_ptr) return FE_OK;
  p->kmap_ptr = p->vmap_ptr = nullptr;
  p->per_head_tma = false;
  if (encode_decode_map(&p->kmap_dec, k_pool, p->dtype, c.hkv, c.dim, c.dec_heads, slots) !=
          FE_OK ||
      encode_decode_map(&p->vmap_dec, v_pool, p->dtype, c.hkv, c.dim, c.dec_heads, slots) !=
          FE_OK) {
    if (p->keys) return FE_ERR_CUDA;
    p->per_head_tma = true;
    int rc = encode_pool_map(&p->kmap_dec, k_pool, p->dtype, c.hkv, c.dim, slots);
    if (rc == FE_OK) rc = encode_pool_map(&p->vmap_dec, v_pool, p->dtype, c.hkv, c.dim, slots);
    if (rc != FE_OK) return rc;
  }
  int rc = encode_tc_map(&p->kmap_tc, k_pool, p->dtype, c.hkv, c.dim, slots);
  if (rc == FE_OK) rc = encode_tc_map(&p->vmap_tc, v_pool, p->dtype, c.hkv, c.dim, slots);
  if (rc != FE_OK) return rc;
  p->kmap_ptr = k_pool;
  p->vmap_ptr = v_pool;
  return FE_OK;
}

template <typename T>
AttnArgs<T> long_args(const fe_long_plan* p, const void* q, void* out, int view, int q_map_rows) {
  AttnArgs<T> a{};
  a.meta = p->spaces[p->space].meta;
  a.q = static_cast<const T*>(q);
  a.out = static_cast<T*>(out);
  a.partials = p->spaces[p->space].partials;
  a.err = device_error_word();
  a.hq = p->cfg.hq;
  a.G = p->cfg.hq / p->cfg.hkv;
  a.page = p->cfg.page;
  a.view = view;
  a.scale_log2 = 1.4426950408889634f / sqrtf(float(p->cfg.dim));
  a.q_map_rows = q_map_rows;
  a.sink = p->d_sink;
  return a;
}

int launch_decode(fe_long_plan* p, const void* args, int grid, bool beside, cudaStream_t s) {
  if (p->keys) return keys_launch(p->dtype, p->kmap_dec, p->vmap_dec, args, grid, beside, s);
  return decode_ext_launch(p->dtype, p->cfg.dec_heads, p->kmap_dec, p->vmap_dec, p->per_head_tma,
                           args, grid, s);
}

template <typename T>
int run_shared(fe_long_plan* p, const void* q, void* out, int view, cudaStream_t s) {
  const PlanConfig& c = p->cfg;
  const int grid_rows = p->fixed_grid ? c.grid_cap : p->last.grid[view];
  const int grid_dec = p->fixed_grid ? c.dec_grid_cap : p->last.grid[2];
  const int G = c.hq / c.hkv;
  CUtensorMap qmap;
  std::memset(&qmap, 0, sizeof(qmap));  // unused when G does not divide 128
  int q_map_rows = 0;
  if (grid_rows > 0 && 128 % G == 0 && p->last.rows > 0) {
    int rc = encode_q_map(&qmap, q, p->dtype, c.hq, c.dim, p->last.rows, G);
    if (rc != FE_OK) return rc;
    q_map_rows = p->last.rows;
  }
  const AttnArgs<T> a = long_args<T>(p, q, out, view, q_map_rows);
  if (grid_rows > 0) {
    int rc = c.dim == kHeadDim
                 ? rows2_launch(p->dtype, p->kmap_tc, p->vmap_tc, qmap, &a, grid_rows, s)
                 : prefill_tc_ext_launch(p->dtype, p->kmap_tc, p->vmap_tc, qmap, &a, grid_rows,
                                         s);
    if (rc != FE_OK) return rc;
  }
  if (grid_dec > 0) {
    int rc = launch_decode(p, &a, grid_dec, grid_rows > 0, s);
    if (rc != FE_OK) return rc;
  }
  if (p->fixed_grid || p->last.merge[view])
    return launch_join<T>(a, c.dim, p->last.rows, nullptr, s);
  return FE_OK;
}

template <typename T>
int run_scored(fe_long_plan* p, const void* q, float* scores, void* out, cudaStream_t s) {
  const PlanConfig& c = p->cfg;
  const int grid_dec = p->fixed_grid ? c.dec_grid_cap : p->last.grid[2];
  const AttnArgs<T> a = long_args<T>(p, q, out, 1, 0);
  int rc = launch_decode(p, &a, grid_dec, false, s);
  if (rc != FE_OK) return rc;
  rc = launch_join<T>(a, c.dim, p->last.rows, p->d_norms, s);
  if (rc != FE_OK) return rc;
  // a graph's launch has to do for later steps of more keys: the CTAs stride
  const int most = std::max(1, 16 * c.grid_cap / c.hkv);
  const dim3 grid(p->fixed_grid ? most : std::max(1, std::min(p->last.n_chunks, most)), c.hkv);
  FE_CUDA_TRY(launch_pdl(score_kernel, grid, dim3(kScoreThreads), 0, s,
                         static_cast<const uint8_t*>(a.meta),
                         static_cast<const float*>(p->d_sink),
                         static_cast<const float2*>(p->d_norms), scores, c.hq, c.hkv, c.page,
                         int64_t(c.num_blocks + 1) * c.page));
  return FE_OK;
}

}  // namespace

extern "C" {

int fe_shared_plan_create(int hq, int hkv, int dim, int page, int max_batch, int max_pages,
                          int dtype, int num_blocks, fe_long_plan** plan_out) {
  return create_long("fe_shared_plan_create", hq, hkv, dim, page, max_batch, max_pages, dtype,
                     num_blocks, false, 0, 0, plan_out);
}

int fe_scored_plan_create(int hq, int hkv, int dim, int page, int max_batch, int max_pages,
                          int dtype, int num_blocks, int64_t max_keys, fe_long_plan** plan_out) {
  return create_long("fe_scored_plan_create", hq, hkv, dim, page, max_batch, max_pages, dtype,
                     num_blocks, true, max_keys, 0, plan_out);
}

int fe_long_plan_create_host(int hq, int hkv, int dim, int page, int max_batch, int max_pages,
                             int dtype, int num_blocks, int scored, int64_t max_keys, int grid_cap,
                             fe_long_plan** plan_out) {
  if (grid_cap <= 0) return fail(FE_ERR_INVALID_ARGUMENT, "grid_cap must be positive");
  return create_long("fe_long_plan_create_host", hq, hkv, dim, page, max_batch, max_pages, dtype,
                     num_blocks, scored != 0, max_keys, grid_cap, plan_out);
}

int fe_long_plan_destroy(fe_long_plan* plan) {
  destroy_long(plan);
  return FE_OK;
}

int fe_shared_plan_prepare(fe_long_plan* p, const int32_t* qo, const int32_t* kv,
                           const int32_t* pages, const int32_t* last, const int32_t* group_off,
                           const int32_t* shared, int groups, int batch, int rows, int graph,
                           void* stream) {
  const std::string name = "fe_shared_plan_prepare";
  int rc = check_prepare(p, false, batch, rows, graph, name);
  if (rc != FE_OK) return rc;
  LongResult res;
  std::string err;
  try {
    rc = build_shared_plan(p->cfg, p->keys, qo, kv, pages, last, group_off, shared, groups, batch,
                           rows, graph != 0, res, err);
  } catch (const std::bad_alloc&) {
    return fail(FE_ERR_CAPACITY, name + ": out of host memory");
  }
  if (rc != FE_OK) return fail(rc, name + ": " + err);
  return install(p, res, 0, batch, rows, graph, name, stream);
}

int fe_scored_plan_prepare(fe_long_plan* p, const int32_t* qo, const int32_t* kv,
                           const int32_t* pages, const int32_t* last, const int32_t* fresh,
                           int batch, int rows, int graph, void* stream) {
  const std::string name = "fe_scored_plan_prepare";
  int rc = check_prepare(p, true, batch, rows, graph, name);
  if (rc != FE_OK) return rc;
  if (rows > p->max_rows)
    return fail(FE_ERR_CAPACITY, name + ": query rows x keys exceed the plan's max_keys");
  LongResult res;
  size_t space = 0;
  std::string err;
  try {
    rc = build_scored_plan(p->cfg, p->keys, qo, kv, pages, last, fresh, batch, rows, graph != 0,
                           p->sink_floats, res, err);
    if (rc == FE_OK && !p->host_only) {
      rc = find_space(p, res, batch, rows, graph, name, space);
      if (rc != FE_OK) return rc;
    }
  } catch (const std::bad_alloc&) {
    return fail(FE_ERR_CAPACITY, name + ": out of host memory");
  }
  if (rc != FE_OK) return fail(rc, name + ": " + err);
  return install(p, res, space, batch, rows, graph, name, stream);
}

int fe_shared_attn_run(fe_long_plan* p, const void* q, const void* k_pool, const void* v_pool,
                       void* out, int causal, void* stream) {
  const std::string name = "fe_shared_attn_run";
  int rc = check_run(p, false, name);
  if (rc != FE_OK || p->last.rows == 0) return rc;
  rc = check_buffers(q, k_pool, v_pool, out, name);
  if (rc == FE_OK) rc = maps(p, k_pool, v_pool);
  if (rc != FE_OK) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  return p->dtype == FE_DTYPE_BF16 ? run_shared<__nv_bfloat16>(p, q, out, causal ? 1 : 0, s)
                                   : run_shared<__half>(p, q, out, causal ? 1 : 0, s);
}

int fe_scored_attn_run(fe_long_plan* p, const void* q, const void* k_pool, const void* v_pool,
                       float* scores, void* out, void* stream) {
  const std::string name = "fe_scored_attn_run";
  int rc = check_run(p, true, name);
  if (rc != FE_OK || p->last.rows == 0) return rc;
  rc = check_buffers(q, k_pool, v_pool, out, name);
  if (rc != FE_OK) return rc;
  if (!scores) return fail(FE_ERR_INVALID_ARGUMENT, name + ": null pointer");
  if (!aligned4(scores))
    return fail(FE_ERR_INVALID_ARGUMENT, name + ": scores must be 4-byte aligned");
  rc = maps(p, k_pool, v_pool);
  if (rc != FE_OK) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  return p->dtype == FE_DTYPE_BF16 ? run_scored<__nv_bfloat16>(p, q, scores, out, s)
                                   : run_scored<__half>(p, q, scores, out, s);
}

int fe_long_plan_get_info(const fe_long_plan* p, fe_long_plan_info* info) {
  if (!p || !info) return fail(FE_ERR_INVALID_ARGUMENT, "fe_long_plan_get_info: null pointer");
  std::memset(info, 0, sizeof(*info));
  if (!p->prepared) return FE_OK;
  info->rows = p->last.rows;
  info->shared_groups = p->last.groups_shared;
  info->shared_tiles = p->last.shared_tiles;
  info->row_ctas = p->last.grid[1];
  info->decode_ctas = p->last.grid[2];
  info->partial_floats = p->last.partial_floats;
  info->weight_floats = p->last.sink_floats;
  return FE_OK;
}

int fe_long_plan_debug_meta(const fe_long_plan* p, void* dst, int64_t cap, int64_t* bytes) {
  if (!p || !bytes) return fail(FE_ERR_INVALID_ARGUMENT, "null pointer");
  *bytes = static_cast<int64_t>(p->last.meta.size());
  if (dst && cap > 0)
    std::memcpy(dst, p->last.meta.data(), static_cast<size_t>(std::min<int64_t>(cap, *bytes)));
  return FE_OK;
}

}  // extern "C"
