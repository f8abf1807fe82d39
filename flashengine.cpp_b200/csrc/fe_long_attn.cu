// Attention for long shared prompts over the paged cache: sequences that begin
// with the same pages (the prefix read once for all of them), and attention
// that scores every cached key by the weight it got. No counterpart in the
// reference, whose attention reads each sequence's pages by itself
// (Cambridgebit/FlashEngine.cpp src/flashinfer_attention.cu:35-44).
//
// Both run the decode kernel (fe_decode.cu) and the row kernel
// (fe_prefill_tc.cu) over the lists of fe_long_plan.h. A record holds, for each
// of its rows, m = the largest base-2 score of its keys, l = sum 2^(s - m) and
// O = sum 2^(s - m) v; records of disjoint keys join as
//   m = max m_i, l = sum l_i 2^(m_i - m), out = sum O_i 2^(m_i - m) / l.
// The weight of a key with score s is then 2^(s - m - log2 l).
#include <algorithm>
#include <cstring>
#include <new>
#include <string>

#include "fe_attn_common.cuh"
#include "fe_long_plan.h"
#include "fe_tensor_maps.h"

namespace fe {

int decode_ext_launch(int dtype, int dim, int heads, const CUtensorMap& kmap,
                      const CUtensorMap& vmap, bool per_head_tma, const void* args, int grid,
                      cudaStream_t stream);
int prefill_tc_ext_launch(int dtype, int dim, const CUtensorMap& kmap, const CUtensorMap& vmap,
                          const CUtensorMap& qmap, const void* args, int grid,
                          cudaStream_t stream);

namespace {

constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;

// The records of one row: nsplit of them, rec_floats apart.
struct Records {
  const float* first;  // split 0's record
  int n, rec_floats, rows, row;
};

__device__ __forceinline__ const SplitGroup* group_of(const MetaHeader* hdr, const uint8_t* meta,
                                                      int view, int unit, int row_units) {
  const int g = reinterpret_cast<const int32_t*>(meta + hdr->unit_off[view])[unit];
  if (g < 0) return nullptr;
  return reinterpret_cast<const SplitGroup*>(
             meta + hdr->groups_off[unit < row_units ? view : 2]) + g;
}

// Records of packed row p (of P) of KV head h in the units that start at
// `unit`; n = 0 where the unit wrote its output itself.
__device__ __forceinline__ Records records_of(const MetaHeader* hdr, const uint8_t* meta,
                                              const float* partials, int view, int unit,
                                              int blocks, int p, int P, int h) {
  Records r{nullptr, 0, 0, 0, 0};
  if (unit < 0) return r;
  const int H = hdr->dec_heads;
  int row;
  if (blocks > 0) {
    unit += h * blocks + p / 128;
    row = p % 128;
  } else {
    unit += h / H;
    row = (h % H) * P + p;
  }
  const int row_units = hdr->chunk_tiles;
  const SplitGroup* g = group_of(hdr, meta, view, unit, row_units);
  if (!g) return r;
  r.first = partials + g->part0;
  r.n = g->nsplit;
  r.rec_floats = g->rec_floats;
  r.rows = g->rows;
  r.row = row;
  return r;
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

// One warp joins the records of one row and stores its 16-bit output.
template <typename T, int D>
__device__ __forceinline__ void join_row(const Records& a, const Records& b, int lane, T* out) {
  constexpr int kV = D / 128;  // float4 vectors per lane
  const int n = a.n + b.n;
  float4 acc[kV];
#pragma unroll
  for (int v = 0; v < kV; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  float M = -INFINITY, L = 0.f;
  for (int s0 = 0; s0 < n; s0 += 32) {
    float m = -INFINITY, l = 0.f;
    if (s0 + lane < n) {
      int rows, row;
      const float* rec = record<D>(a, b, s0 + lane, rows, row);
      m = __ldcg(rec + rows * D + row);
      l = __ldcg(rec + rows * (D + 1) + row);
    }
    float mc = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) mc = fmaxf(mc, __shfl_xor_sync(0xffffffffu, mc, o));
    const float M_new = fmaxf(M, mc);
    const float base = M_new == -INFINITY ? 0.f : M_new;
    const float resc = M == -INFINITY ? 0.f : fast_exp2(M - base);
    M = M_new;
    const float w = s0 + lane < n ? fast_exp2(m - base) : 0.f;
    float lw = l * w;
#pragma unroll
    for (int o = 16; o; o >>= 1) lw += __shfl_xor_sync(0xffffffffu, lw, o);
    L = L * resc + lw;
#pragma unroll
    for (int v = 0; v < kV; ++v) {
      acc[v].x *= resc;
      acc[v].y *= resc;
      acc[v].z *= resc;
      acc[v].w *= resc;
    }
    const int c = min(32, n - s0);
#pragma unroll 4
    for (int j = 0; j < c; ++j) {
      int rows, row;
      const float* rec = record<D>(a, b, s0 + j, rows, row);
      const float wj = __shfl_sync(0xffffffffu, w, j);
#pragma unroll
      for (int v = 0; v < kV; ++v) {
        const float4 x =
            __ldcg(reinterpret_cast<const float4*>(rec + row * D + v * 128 + lane * 4));
        acc[v].x = fmaf(x.x, wj, acc[v].x);
        acc[v].y = fmaf(x.y, wj, acc[v].y);
        acc[v].z = fmaf(x.z, wj, acc[v].z);
        acc[v].w = fmaf(x.w, wj, acc[v].w);
      }
    }
  }
  const float inv = 1.f / L;
#pragma unroll
  for (int v = 0; v < kV; ++v)
    store4<T>(out + v * 128 + lane * 4, acc[v].x * inv, acc[v].y * inv, acc[v].z * inv,
              acc[v].w * inv);
}

// Warp `w` of the joining warps: query row w / hq, head w % hq.
template <typename T, int D>
__device__ __forceinline__ void join_warp(const AttnArgs<T>& a, int64_t w, int lane) {
  const MetaHeader* hdr = reinterpret_cast<const MetaHeader*>(a.meta);
  const int r = static_cast<int>(w / a.hq), head = static_cast<int>(w % a.hq);
  if (r >= hdr->rows) return;
  const int s = reinterpret_cast<const int32_t*>(a.meta + hdr->row_seq_off)[r];
  const MergeSeq m = reinterpret_cast<const MergeSeq*>(a.meta + hdr->merge_off)[s];
  const int h = head / a.G, p = (r - m.q_row0) * a.G + head % a.G;
  const Records own = records_of(hdr, a.meta, a.partials, a.view, m.own_unit, m.own_blocks, p,
                                 m.qrows * a.G, h);
  if (own.n == 0) return;  // written by its unit
  const Records pre = records_of(hdr, a.meta, a.partials, a.view, m.pre_unit, m.pre_blocks,
                                 m.pre_row0 + p, m.pre_rows, h);
  join_row<T, D>(own, pre, lane, a.out + (static_cast<int64_t>(r) * a.hq + head) * D);
}

// Shared-prefix plans: one warp per query row and head.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const AttnArgs<T> a) {
  pdl_trigger();
  pdl_wait();
  join_warp<T, D>(a, static_cast<int64_t>(blockIdx.x) * kJoinWarps + (threadIdx.x >> 5),
                  threadIdx.x & 31);
}

// Scored plans: the first `join_ctas` CTAs join rows as above, the others give
// the weights of kScoreChunk keys of one KV head at a time to the scores.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
    score_kernel(const AttnArgs<T> a, float* __restrict__ scores, int hkv, int64_t cache_slots,
                 int join_ctas) {
  constexpr int kPer = kScoreChunk / kJoinThreads;  // keys a thread
  __shared__ float lse[kRowBlock];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (static_cast<int>(blockIdx.x) < join_ctas) {
    join_warp<T, D>(a, static_cast<int64_t>(blockIdx.x) * kJoinWarps + warp, lane);
    return;
  }
  const MetaHeader* hdr = reinterpret_cast<const MetaHeader*>(a.meta);
  const ScoreChunk* chunks = reinterpret_cast<const ScoreChunk*>(a.meta + hdr->chunk_off);
  const SeqInfo* seqs = reinterpret_cast<const SeqInfo*>(a.meta + hdr->seqs_off);
  const MergeSeq* merge = reinterpret_cast<const MergeSeq*>(a.meta + hdr->merge_off);
  const int64_t* sink = reinterpret_cast<const int64_t*>(a.meta + hdr->sink_off);
  const int32_t* pages = reinterpret_cast<const int32_t*>(a.meta + hdr->pages_off);
  const int64_t total = static_cast<int64_t>(hdr->n_chunks) * hkv;
  for (int64_t e = blockIdx.x - join_ctas; e < total; e += gridDim.x - join_ctas) {
    const ScoreChunk c = chunks[e / hkv];
    const int h = static_cast<int>(e % hkv);
    float w[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) w[i] = 0.f;
    for (int j = c.block0; j < c.block0 + c.blocks; ++j) {
      const SeqInfo si = seqs[j];
      if (c.t0 >= si.length) continue;  // the block's rows do not see this far
      const int P = si.qrows * a.G, cols = (P + 1) & ~1;
      __syncthreads();  // the last block's sums have been read
      for (int p = warp; p < P; p += kJoinWarps) {
        const Records r =
            records_of(hdr, a.meta, a.partials, a.view, merge[j].own_unit, 0, p, P, h);
        float M = -INFINITY, L = 0.f;
        for (int s = lane; s < r.n; s += 32) {
          const float* rec = r.first + static_cast<int64_t>(s) * r.rec_floats;
          const float m = __ldcg(rec + r.rows * D + r.row);
          const float l = __ldcg(rec + r.rows * (D + 1) + r.row);
          const float mn = fmaxf(M, m), base = mn == -INFINITY ? 0.f : mn;
          L = L * fast_exp2(M - base) + l * fast_exp2(m - base);
          M = mn;
        }
        float top = M;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        L *= fast_exp2(M - (top == -INFINITY ? 0.f : top));
#pragma unroll
        for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        if (lane == 0) lse[p] = top + log2f(L);
      }
      __syncthreads();
      const int tiles = (si.length + kTileTokens - 1) / kTileTokens;
      const float* raw = a.sink + sink[j] + static_cast<int64_t>(h) * tiles * kTileTokens * cols;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int t = c.t0 + i * kJoinThreads + threadIdx.x;
        if (t >= si.length) continue;
        const float2* s2 = reinterpret_cast<const float2*>(raw + static_cast<int64_t>(t) * cols);
        for (int p = 0; p < P; p += 2) {
          const float2 s = __ldcg(s2 + p / 2);
          w[i] += fast_exp2(s.x - lse[p]);
          if (p + 1 < P) w[i] += fast_exp2(s.y - lse[p + 1]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int t = c.t0 + i * kJoinThreads + threadIdx.x;
      if (t >= c.length) continue;
      const int64_t slot =
          static_cast<int64_t>(__ldg(pages + c.page_off + t / a.page)) * a.page + t % a.page;
      float* at = scores + h * cache_slots + slot;
      *at = t >= c.fresh ? w[i] : *at + w[i];
    }
  }
}

}  // namespace
}  // namespace fe

using namespace fe;

struct fe_long_plan {
  PlanConfig cfg{};
  int dtype = 0;
  bool scored = false, host_only = false;
  int device = -1;
  uint8_t* d_meta = nullptr;
  size_t meta_cap = 0;
  float* d_partials = nullptr;
  float* d_sink = nullptr;
  int64_t sink_floats = 0;
  // pinned staging, double-buffered
  uint8_t* h_meta[2] = {nullptr, nullptr};
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
    if (p->d_meta) cudaFree(p->d_meta);
    if (p->d_partials) cudaFree(p->d_partials);
    if (p->d_sink) cudaFree(p->d_sink);
  }
  delete p;
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
  c.row_group_blocks = 8;
  c.row_tile = dim == kWideHeadDim ? 4 : 8;
  c.row_item_tiles = 2;
  c.elem_bytes = 2;
  c.dec_min_tiles = 8;
  c.max_items = c.max_groups = static_cast<int>(std::min<int64_t>(
      std::max<int64_t>(int64_t(max_batch) * hkv * 64, 8192), 1 << 20));
  c.partial_capacity = kLongPartialFloats;
  // every query row of a key or score is rounded up to an even number of columns
  p->sink_floats = scored ? max_keys * hkv * (G + (G & 1)) : 0;
  // lists (cta offsets, items, groups) three times, units twice, row blocks and
  // their tables, query rows, chunks, pages
  const size_t n = c.max_items;
  p->meta_cap = 3 * (n * (sizeof(WorkItem) + sizeof(SplitGroup)) + 4 * size_t(sms + 1) + 64) +
                2 * 4 * n + n * (sizeof(SeqInfo) + sizeof(MergeSeq) + 8) + 4 * 16 * n +
                2 * size_t(max_batch) * (sizeof(SeqInfo) + sizeof(MergeSeq)) +
                sizeof(ScoreChunk) * size_t(max_batch) *
                    (size_t(max_pages) * page / kScoreChunk + 1) +
                4 * size_t(max_batch) * max_pages + 4096;
  *plan_out = p;
  if (p->host_only) return FE_OK;
  cudaError_t e = cudaMalloc(&p->d_partials, sizeof(float) * c.partial_capacity);
  if (e == cudaSuccess) e = cudaMalloc(&p->d_meta, p->meta_cap);
  if (e == cudaSuccess) e = cudaMemset(p->d_meta, 0, sizeof(MetaHeader));
  if (e == cudaSuccess && p->sink_floats > 0)
    e = cudaMalloc(&p->d_sink, sizeof(float) * p->sink_floats);
  for (int i = 0; i < 2 && e == cudaSuccess; ++i) {
    e = cudaMallocHost(&p->h_meta[i], p->meta_cap);
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

// Upload a step's metadata and take it as the plan's current one.
int install(fe_long_plan* p, LongResult& res, int batch, int rows, int graph,
            const std::string& name, void* stream) {
  if (res.meta.size() > p->meta_cap)
    return fail(FE_ERR_CAPACITY, name + ": metadata exceeds workspace");
  if (!p->host_only) {
    auto s = static_cast<cudaStream_t>(stream);
    const int i = p->h_idx;
    if (p->h_used[i]) FE_CUDA_TRY(cudaEventSynchronize(p->h_ev[i]));
    std::memcpy(p->h_meta[i], res.meta.data(), res.meta.size());
    FE_CUDA_TRY(
        cudaMemcpyAsync(p->d_meta, p->h_meta[i], res.meta.size(), cudaMemcpyHostToDevice, s));
    FE_CUDA_TRY(cudaEventRecord(p->h_ev[i], s));
    p->h_used[i] = true;
    p->h_idx ^= 1;
  }
  p->last = std::move(res);
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
  a.meta = p->d_meta;
  a.q = static_cast<const T*>(q);
  a.out = static_cast<T*>(out);
  a.partials = p->d_partials;
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

int join_ctas(const fe_long_plan* p) {
  return static_cast<int>((int64_t(p->last.rows) * p->cfg.hq + kJoinWarps - 1) / kJoinWarps);
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
    int rc = prefill_tc_ext_launch(p->dtype, c.dim, p->kmap_tc, p->vmap_tc, qmap, &a, grid_rows, s);
    if (rc != FE_OK) return rc;
  }
  if (grid_dec > 0) {
    int rc = decode_ext_launch(p->dtype, c.dim, c.dec_heads, p->kmap_dec, p->vmap_dec,
                               p->per_head_tma, &a, grid_dec, s);
    if (rc != FE_OK) return rc;
  }
  if (p->fixed_grid || p->last.merge[view]) {
    auto kernel = c.dim == kWideHeadDim ? join_kernel<T, kWideHeadDim> : join_kernel<T, kHeadDim>;
    FE_CUDA_TRY(launch_pdl(kernel, dim3(join_ctas(p)), dim3(kJoinThreads), 0, s, a));
  }
  return FE_OK;
}

template <typename T>
int run_scored(fe_long_plan* p, const void* q, float* scores, void* out, cudaStream_t s) {
  const PlanConfig& c = p->cfg;
  const int grid_dec = p->fixed_grid ? c.dec_grid_cap : p->last.grid[2];
  const AttnArgs<T> a = long_args<T>(p, q, out, 1, 0);
  int rc = decode_ext_launch(p->dtype, c.dim, c.dec_heads, p->kmap_dec, p->vmap_dec,
                             p->per_head_tma, &a, grid_dec, s);
  if (rc != FE_OK) return rc;
  const int joins = join_ctas(p);
  // a graph's launch has to do for later steps of more keys: the CTAs stride
  const int64_t most = int64_t(8) * c.grid_cap;
  const int64_t work = int64_t(p->last.n_chunks) * c.hkv;
  const int more = static_cast<int>(p->fixed_grid ? most : std::min(work, most));
  auto kernel = c.dim == kWideHeadDim ? score_kernel<T, kWideHeadDim> : score_kernel<T, kHeadDim>;
  FE_CUDA_TRY(launch_pdl(kernel, dim3(joins + more), dim3(kJoinThreads), 0, s, a, scores, c.hkv,
                         int64_t(c.num_blocks + 1) * c.page, joins));
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
    rc = build_shared_plan(p->cfg, qo, kv, pages, last, group_off, shared, groups, batch, rows,
                           graph != 0, res, err);
  } catch (const std::bad_alloc&) {
    return fail(FE_ERR_CAPACITY, name + ": out of host memory");
  }
  if (rc != FE_OK) return fail(rc, name + ": " + err);
  return install(p, res, batch, rows, graph, name, stream);
}

int fe_scored_plan_prepare(fe_long_plan* p, const int32_t* qo, const int32_t* kv,
                           const int32_t* pages, const int32_t* last, const int32_t* fresh,
                           int batch, int rows, int graph, void* stream) {
  const std::string name = "fe_scored_plan_prepare";
  int rc = check_prepare(p, true, batch, rows, graph, name);
  if (rc != FE_OK) return rc;
  LongResult res;
  std::string err;
  try {
    rc = build_scored_plan(p->cfg, qo, kv, pages, last, fresh, batch, rows, graph != 0,
                           p->sink_floats, res, err);
  } catch (const std::bad_alloc&) {
    return fail(FE_ERR_CAPACITY, name + ": out of host memory");
  }
  if (rc != FE_OK) return fail(rc, name + ": " + err);
  return install(p, res, batch, rows, graph, name, stream);
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
