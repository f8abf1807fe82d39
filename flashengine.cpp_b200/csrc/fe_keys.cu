// Key kernel of the plans for long shared prompts at head_dim 128: up to 16
// packed query rows against a KV head's keys, one warp a piece of the work.
//
// Reference behaviour: Cambridgebit/FlashEngine.cpp src/flashinfer_attention.cu:35-44
// with the arithmetic of src/portable_gpu_ops.cpp:39-44.
//
// The keys that are a sequence's own behind a shared prefix are few: the decode
// kernel's items (all KV heads of a sequence, eight warps that merge through
// shared memory) then spend most of their time on their beginning and end (128
// sequences of up to 257 own keys and 4 KV heads 26 us, mostly two or three
// items one after the other on each of 55 SMs). Here a piece is one (sequence,
// KV head) and a range of 16-key tiles, and one warp works through its pieces
// alone: it fetches K and V tiles (4 KiB each, one TMA box) into a ring of its
// own, does their products and writes a partial record. Eight such warps, each a
// CTA, fit an SM; a step's tiles are cut evenly across all of them, so that short
// pieces run side by side and long streams keep 192 KiB an SM in flight.
#include "fe_attn_common.cuh"
#include "fe_long_plan.h"

namespace fe {

int keys_launch(int dtype, const CUtensorMap& kmap, const CUtensorMap& vmap, const void* args,
                int grid, bool beside, cudaStream_t stream);

namespace {

constexpr int kStages = 3;
constexpr int kKBytes = 2 * kHalfBytes;       // one head's 16 keys
constexpr int kStageBytes = 2 * kKBytes;
constexpr int kSmem = kStages * kStageBytes + kStages * 8 + 8;

template <typename T>
__device__ __forceinline__ T to_elem(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 to_elem<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half to_elem<__half>(float x) {
  return __float2half_rn(x);
}

// Past the L1, as TMA reads K and V: nothing here depends on its being clean.
__device__ __forceinline__ uint32_t ld_l2(const void* p) {
  return __ldcg(reinterpret_cast<const uint32_t*>(p));
}

// D += A B on one 16 x 8 x 16 product; no side effects, so that the compiler
// may order products and loads by their operands.
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4],
                                                   uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                            uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A row block's softmax state, as KeyState (fe_attn_common.cuh): S^T = K Q^T with
// the 16 keys on the product's M side, O^T = V^T P^T, P as a 16-bit high part and
// its residual. One warp works alone here, two on an SM's quarter, so a tile's
// time is the length of its chain of dependent steps: the tile's fragments are
// loaded ahead of their products, S is summed in two chains, and O is rescaled
// only where a row's maximum grew by more than 2^8.
template <typename T, int NT>
struct RowState {
  uint32_t qb[NT][8][2];  // Q^T as B fragments: column lane/4 (+8 nt)
  int lim[NT][2];         // visible-key limit of this lane's columns
  int lim_min;
  float m[NT][2], l[NT][2];
  float o[NT][8][4];

  __device__ __forceinline__ void init(const T* q, int hq, const SeqInfo& si, int head0, int G,
                                       bool causal, int lane) {
    const int r8 = lane >> 2, cq = lane & 3, P = si.qrows * G;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int p = nt * 8 + r8;
      const T* qp = p < P ? q + (static_cast<int64_t>(si.q_row0 + p / G) * hq + head0 + p % G) *
                                    kHeadDim
                          : nullptr;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        qb[nt][kk][0] = qp ? ld_l2(qp + kk * 16 + 2 * cq) : 0u;
        qb[nt][kk][1] = qp ? ld_l2(qp + kk * 16 + 8 + 2 * cq) : 0u;
      }
    }
    lim_min = si.length;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int p = nt * 8 + 2 * cq + e;
        lim[nt][e] = causal && p < P ? si.length - si.qrows + p / G + 1 : si.length;
        lim_min = min(lim_min, lim[nt][e]);
        m[nt][e] = -INFINITY;
        l[nt][e] = 0.f;
      }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.f;
  }

  // One 16-token tile at `k` and `v`, starting at token `tbase`; raw scores also to
  // sink[key * cols + column] where sink is given.
  __device__ __forceinline__ void tile(uint32_t k, uint32_t v, int tbase, int length,
                                       float scale_log2, int lane, float* sink, int cols) {
    const int r8 = lane >> 2, cq = lane & 3, mi = lane >> 3, li = lane & 7;
    // ---- S^T = K Q^T, even and odd k-steps apart
    float sc[NT][4], odd[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[nt][e] = odd[nt][e] = 0.f;
    uint32_t f[8][4];
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      const int tok = li + ((mi & 1) << 3);
      const int c = 2 * kk + (mi >> 1);  // 16-byte chunk of the row (8 per 64-dim box)
      ldmatrix_x4(k + (c >> 3) * kHalfBytes + tok * 128 + (((c & 7) ^ li) << 4), f[kk][0],
                  f[kk][1], f[kk][2], f[kk][3]);
    }
#pragma unroll
    for (int kk = 0; kk < 8; kk += 2)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma<T>(sc[nt], f[kk], qb[nt][kk][0], qb[nt][kk][1]);
        mma<T>(odd[nt], f[kk + 1], qb[nt][kk + 1][0], qb[nt][kk + 1][1]);
      }
    // V's fragments are on their way while the weights are made
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      const int tok = li + ((mi >> 1) << 3);
      const int c = 2 * mt + (mi & 1);
      ldmatrix_x4_trans(v + (c >> 3) * kHalfBytes + tok * 128 + (((c & 7) ^ li) << 4), f[mt][0],
                        f[mt][1], f[mt][2], f[mt][3]);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[nt][e] = (sc[nt][e] + odd[nt][e]) * scale_log2;
    // ---- mask keys past each column's limit (causal) or the sequence end
    if (tbase + kTileTokens > lim_min) {
      const int t0 = tbase + r8, t1 = t0 + 8;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (t0 >= lim[nt][e]) sc[nt][e] = -INFINITY;
          if (t1 >= lim[nt][e]) sc[nt][2 + e] = -INFINITY;
        }
    }
    if (sink) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int col = nt * 8 + 2 * cq;
        if (col < cols) {
          *reinterpret_cast<float2*>(sink + r8 * cols + col) = make_float2(sc[nt][0], sc[nt][1]);
          *reinterpret_cast<float2*>(sink + (r8 + 8) * cols + col) =
              make_float2(sc[nt][2], sc[nt][3]);
        }
      }
    }
    // ---- online softmax per column; the 8 lanes sharing lane%4 hold a column
    float mx[NT][2];
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[nt][e] = fmaxf(sc[nt][e], sc[nt][2 + e]);
        grow |= mx[nt][e] > m[nt][e] + 8.f;  // (true for a column's first finite score)
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = mx[nt][e];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const float mn = fmaxf(m[nt][e], x);
          const float al = fast_exp2(m[nt][e] - (mn == -INFINITY ? 0.f : mn));
          m[nt][e] = mn;
          l[nt][e] *= al;
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            o[nt][mt][e] *= al;
            o[nt][mt][2 + e] *= al;
          }
        }
    }
    // ---- P^T as B fragments (high part + residual), transposed with movmatrix
    uint32_t bh[NT][2], bl[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float base = m[nt][e] == -INFINITY ? 0.f : m[nt][e];
        sc[nt][e] = fast_exp2(sc[nt][e] - base);
        sc[nt][2 + e] = fast_exp2(sc[nt][2 + e] - base);
        l[nt][e] += sc[nt][e] + sc[nt][2 + e];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t x = pack2<T>(sc[nt][2 * h], sc[nt][2 * h + 1]);
        const float2 y = unpack2<T>(x);
        bh[nt][h] = movmatrix_trans(x);
        bl[nt][h] = movmatrix_trans(pack2<T>(sc[nt][2 * h] - y.x, sc[nt][2 * h + 1] - y.y));
      }
    }
    // ---- V rows past the sequence end are zeroed in the fragments (the pool may
    // hold anything there; 0 * NaN would poison O)
    if (tbase + kTileTokens > length) {
      const int ta = tbase + 2 * cq;
      const uint32_t v0 = (ta < length ? 0x0000ffffu : 0u) | (ta + 1 < length ? 0xffff0000u : 0u);
      const uint32_t v1 =
          (ta + 8 < length ? 0x0000ffffu : 0u) | (ta + 9 < length ? 0xffff0000u : 0u);
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        f[mt][0] &= v0;
        f[mt][1] &= v0;
        f[mt][2] &= v1;
        f[mt][3] &= v1;
      }
    }
    // ---- O^T += V^T P^T (16 dims per m-tile)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) mma<T>(o[nt][mt], f[mt], bh[nt][0], bh[nt][1]);
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) mma<T>(o[nt][mt], f[mt], bl[nt][0], bl[nt][1]);
    }
  }

  // Sum each column's l over the 8 lanes that share it.
  __device__ __forceinline__ void reduce_l() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4);
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8);
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
      }
  }
};

// The warp's ring: tiles of its items in order, fetched ahead of their use. An
// item's place and the slots of its first tiles are loaded one and two items
// before they are needed, so that going on to the next waits for nothing.
struct Ring {
  const KeyItem* items;
  const int32_t* pages;
  const CUtensorMap* kmap;
  const CUtensorMap* vmap;
  uint8_t* stages;
  uint64_t* full;
  int it, it1;     // item of the next tile to fetch
  int page;
  int kvh, page_off, j, j1;            // the item: head, pages, next tile, end
  int base, slot;                      // lane l holds the slot of tile base + l
  int kvh_n, page_off_n, j_n, j1_n, slot_n;  // the item behind it
  uint32_t issued;

  __device__ __forceinline__ int slot_at(int off, int t, int end) const {
    if (t >= end) return 0;
    const int t0 = t * kTileTokens;
    return __ldg(pages + off + t0 / page) * page + t0 % page;
  }
  __device__ __forceinline__ void look(int item) {  // at the item behind
    if (item >= it1) return;
    const int4 a = __ldg(reinterpret_cast<const int4*>(items + item));
    const int4 b = __ldg(reinterpret_cast<const int4*>(items + item) + 1);
    page_off_n = a.w;
    kvh_n = b.x;
    j_n = b.z;
    j1_n = b.w;
  }
  __device__ __forceinline__ void next(int lane) {
    ++it;
    kvh = kvh_n;
    page_off = page_off_n;
    base = j = j_n;
    j1 = j1_n;
    slot = slot_n;
    look(it + 1);
  }
  __device__ __forceinline__ void open(int first, int lane) {
    it = first - 1;
    page_off_n = kvh_n = j_n = j1_n = slot_n = 0;
    look(first);
    slot_n = slot_at(page_off_n, j_n + lane, j1_n);
    next(lane);
  }
  __device__ __forceinline__ void issue(int lane) {
    if (it >= it1) return;
    if (j - base == 32) {
      base = j;
      slot = slot_at(page_off, j + lane, j1);
    }
    const int s0 = __shfl_sync(0xffffffffu, slot, j - base);
    const int st = issued % kStages;
    if (lane == 0) {
      mbar_arrive_expect_tx(&full[st], kStageBytes);
      uint8_t* dst = stages + st * kStageBytes;
      tma_load_3d(dst, kmap, &full[st], 0, s0, 2 * kvh);
      tma_load_3d(dst + kKBytes, vmap, &full[st], 0, s0, 2 * kvh);
    }
    // (j - base is small again only behind the item's first tile)
    if (j == base && it + 1 < it1) slot_n = slot_at(page_off_n, j_n + lane, j1_n);
    ++issued;
    if (++j == j1) next(lane);
  }
};

// One piece: the row block's packed rows against tiles [kt0, kt1) of the head.
template <typename T, int NT>
__device__ __forceinline__ bool piece(const AttnArgs<T>& a, const KeyItem& wi, Ring& ring,
                                      uint32_t& g, volatile int* flag, int lane) {
  const SeqInfo si{wi.q_row0, wi.qrows, wi.length, wi.page_off};
  const int G = a.G, P = si.qrows * G, head0 = wi.kvh * G;
  // items of a shared prefix (key_mode 2) are seen whole by every row
  const bool causal = a.view == 1 && wi.key_mode == 1;
  RowState<T, NT> ks;
  ks.init(a.q, a.hq, si, head0, G, causal, lane);
  const int cols = (P + 1) & ~1;
  float* sink = nullptr;  // raw scores: [KV head][key tile][16 keys][cols] per sequence
  if (a.sink) {
    const MetaHeader* hdr = reinterpret_cast<const MetaHeader*>(a.meta);
    const int64_t* off = reinterpret_cast<const int64_t*>(a.meta + hdr->sink_off);
    const int tiles = (si.length + kTileTokens - 1) / kTileTokens;
    sink = a.sink + off[wi.seq] + static_cast<int64_t>(wi.kvh) * tiles * (kTileTokens * cols);
  }
  for (int jt = wi.kt0; jt < wi.kt1; ++jt, ++g) {
    const int s = g % kStages;
    if (!__all_sync(0xffffffffu, wait_bounded(&ring.full[s], (g / kStages) & 1u, flag)))
      return false;
    const uint32_t k = smem_u32(ring.stages + s * kStageBytes);
    ks.tile(k, k + kKBytes, jt * kTileTokens, si.length, a.scale_log2, lane,
            sink ? sink + static_cast<int64_t>(jt) * (kTileTokens * cols) : nullptr, cols);
    __syncwarp();  // the stage has been read by every lane
    ring.issue(lane);
  }
  ks.reduce_l();
  const int r8 = lane >> 2, cq = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int p = nt * 8 + 2 * cq + e;
      if (p >= P) continue;
      if (wi.group < 0) {
        const float inv = 1.f / ks.l[nt][e];
        T* dst = a.out +
                 (static_cast<int64_t>(si.q_row0 + p / G) * a.hq + head0 + p % G) * kHeadDim;
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
          dst[16 * mt + r8] = to_elem<T>(ks.o[nt][mt][e] * inv);
          dst[16 * mt + r8 + 8] = to_elem<T>(ks.o[nt][mt][2 + e] * inv);
        }
      } else {
        float* rec = a.partials + wi.part;
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
          rec[p * kHeadDim + 16 * mt + r8] = ks.o[nt][mt][e];
          rec[p * kHeadDim + 16 * mt + r8 + 8] = ks.o[nt][mt][2 + e];
        }
        if (r8 == 0) {
          rec[P * kHeadDim + p] = ks.m[nt][e];
          rec[P * (kHeadDim + 1) + p] = ks.l[nt][e];
        }
      }
    }
  return true;
}

template <typename T>
__global__ void __launch_bounds__(32)
    paged_keys_kernel(const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap, const AttnArgs<T> a, int beside) {
  extern __shared__ __align__(16) uint8_t smem[];
  pdl_trigger();
  const int lane = threadIdx.x;
  const MetaHeader* hdr = reinterpret_cast<const MetaHeader*>(a.meta);
  int it0 = 0, it1 = 0;
  if (static_cast<int>(blockIdx.x) < hdr->grid[2]) {
    const int32_t* cta_off = reinterpret_cast<const int32_t*>(a.meta + hdr->cta_off_off[2]);
    it0 = cta_off[blockIdx.x];
    it1 = cta_off[blockIdx.x + 1];
  }
  if (it0 >= it1) {  // nothing to do, but the grid does not end before the one ahead
    if (!beside || blockIdx.x == 0) pdl_wait();
    return;
  }
  if (smem_u32(smem) & 1023u) {  // the swizzle's atoms
    if (lane == 0) raise_device_error(a.err, FE_DEVERR_SMEM_ALIGN);
    pdl_wait();
    return;
  }
  Ring ring;
  ring.items = reinterpret_cast<const KeyItem*>(a.meta + hdr->key_items_off);
  ring.pages = reinterpret_cast<const int32_t*>(a.meta + hdr->pages_off);
  ring.kmap = &kmap;
  ring.vmap = &vmap;
  ring.stages = smem;
  ring.full = reinterpret_cast<uint64_t*>(smem + kStages * kStageBytes);
  volatile int* flag = reinterpret_cast<volatile int*>(ring.full + kStages);
  ring.it1 = it1;
  ring.page = a.page;
  ring.issued = 0;
  if (lane == 0) {
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
    for (int s = 0; s < kStages; ++s) mbar_init(&ring.full[s], 1);
    *flag = 0;
    fence_barrier_init();
  }
  __syncwarp();
  ring.open(it0, lane);
  // q, the pools and the records belong to earlier kernels until here. `beside`: the
  // grid ahead is the row kernel, which lets this one start once it has waited for
  // those itself, and which shares nothing with it but the kernel that joins their
  // records; that one waits for this grid, so the row kernel's end is awaited last.
  if (!beside) pdl_wait();
  for (int s = 0; s < kStages; ++s) ring.issue(lane);
  uint32_t g = 0;
  bool ok = true;
  for (int it = it0; it < it1 && ok; ++it) {
    const KeyItem wi = ring.items[it];
    ok = wi.qrows * a.G <= 8 ? piece<T, 1>(a, wi, ring, g, flag, lane)
                             : piece<T, 2>(a, wi, ring, g, flag, lane);
    ok = __all_sync(0xffffffffu, ok);
  }
  if (beside) pdl_wait();
  if (!ok) {
    if (lane == 0) raise_device_error(a.err, FE_DEVERR_TIMEOUT);
    // what was fetched has landed before the CTA exits (bounded)
    volatile int never = 0;
    for (uint32_t k = g; k < ring.issued; ++k)
      (void)wait_bounded(&ring.full[k % kStages], (k / kStages) & 1u, &never);
  }
}

template <typename T>
int launch_t(const CUtensorMap& kmap, const CUtensorMap& vmap, const void* args, int grid,
             bool beside, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  FE_CUDA_TRY(allow_smem(paged_keys_kernel<T>, kSmem, done));
  FE_CUDA_TRY(launch_pdl(paged_keys_kernel<T>, dim3(grid), dim3(32), kSmem, stream, kmap, vmap,
                         *static_cast<const AttnArgs<T>*>(args), beside ? 1 : 0));
  return FE_OK;
}

}  // namespace

int keys_launch(int dtype, const CUtensorMap& kmap, const CUtensorMap& vmap, const void* args,
                int grid, bool beside, cudaStream_t stream) {
  return dtype == FE_DTYPE_BF16 ? launch_t<__nv_bfloat16>(kmap, vmap, args, grid, beside, stream)
                                : launch_t<__half>(kmap, vmap, args, grid, beside, stream);
}

}  // namespace fe
