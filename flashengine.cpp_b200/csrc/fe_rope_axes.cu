// Rotary embedding with several position axes (time, height and width of an
// image's or video's patches), alone and fused with the K/V append. No
// counterpart in the reference, whose rope has one position a row
// (Cambridgebit/FlashEngine.cpp src/cuda_kernels.cu:19-23).
//
// Pair j of a head, (x[j], x[j + r]) with r = rotary_dim / 2, turns by the
// cos / sin of cache row pos[axis(j)][row], column j: the rotation of fe_rope,
// with a cache row of its own for each pair's axis and the same roundings, so
// that equal positions on all axes give fe_rope's bits.
//
// HBM-bound: 4 bytes of q and 8 of k and v per element (in and out) and one
// cos / sin row a token.
#include <algorithm>
#include <string>

#include "fe_attn_common.cuh"
#include "fe_rope_common.cuh"

namespace fe {
namespace {

constexpr int kMaxAxes = FE_MAX_AXES;
constexpr int kMaxPairs = 256;
constexpr int kAxesThreads = 256;

// Axis of each pair, a kernel argument (the caller's list lives on the host).
struct __align__(16) AxisMap {
  uint8_t axis[kMaxPairs];
};

struct AxesArgs {
  const int64_t* slots;
  const int64_t* pos;  // [axes][rows]
  const float* cache;
  unsigned int* err;
  int64_t cache_slots;
  int rows, axes, hq, hkv, dim, rot, max_positions;
};

// The row's position on each axis; false (and flagged by `who`) when one lies
// outside the cache.
__device__ __forceinline__ bool row_positions(const AxesArgs& a, int row, int (&p)[kMaxAxes],
                                              bool who) {
  bool good = true;
#pragma unroll
  for (int x = 0; x < kMaxAxes; ++x) {
    const int64_t v = x < a.axes ? __ldg(a.pos + static_cast<int64_t>(x) * a.rows + row) : 0;
    good &= v >= 0 && v < a.max_positions;
    p[x] = static_cast<int>(v);
  }
  if (!good && who) raise_device_error(a.err, FE_DEVERR_POS_RANGE);
  return good;
}

__device__ __forceinline__ int pick(const int (&p)[kMaxAxes], int axis) {
  return axis == 0 ? p[0] : axis == 1 ? p[1] : axis == 2 ? p[2] : p[3];
}

// Any dim and rotary_dim that are multiples of 4: a thread owns two adjacent
// pairs (or four unrotated dims) of a head, as in fe_rope's plain form.
template <typename T>
__global__ void __launch_bounds__(kAxesThreads)
    rope_axes_kernel(T* __restrict__ q, const T* k, const T* __restrict__ v, T* k_out,
                     T* __restrict__ kc, T* __restrict__ vc, const AxesArgs a, const AxisMap map) {
  using V = typename Pair2<T>::V;
  pdl_trigger();
  pdl_wait();  // q, k, v come from, and the pools are read by, earlier kernels
  const int per_head = a.dim / 4, heads = a.hq + a.hkv;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (idx >= static_cast<int64_t>(a.rows) * heads * per_head) return;
  const int jp = static_cast<int>(idx % per_head);
  const int head = static_cast<int>((idx / per_head) % heads);
  const int row = static_cast<int>(idx / (static_cast<int64_t>(per_head) * heads));
  int p[kMaxAxes];
  if (!row_positions(a, row, p, jp == 0 && head == 0)) return;
  const bool rotating = jp < a.rot / 4;
  const int i0 = rotating ? jp : (a.rot + 4 * (jp - a.rot / 4)) / 2;
  const int i1 = rotating ? (a.rot / 2 + 2 * jp) / 2 : i0 + 1;
  float2 c = make_float2(0.f, 0.f), s = c;
  if (rotating) {
    const int j = 2 * jp, r = a.rot / 2;
    const float* c0 = a.cache + static_cast<int64_t>(pick(p, map.axis[j])) * a.rot + j;
    const float* c1 = a.cache + static_cast<int64_t>(pick(p, map.axis[j + 1])) * a.rot + j + 1;
    c = make_float2(__ldg(c0), __ldg(c1));
    s = make_float2(__ldg(c0 + r), __ldg(c1 + r));
  }
  if (head < a.hq) {
    if (!rotating) return;  // q's unrotated dims stay as they are
    V* base = reinterpret_cast<V*>(q + (static_cast<int64_t>(row) * a.hq + head) * a.dim);
    V lo = base[i0], hi = base[i1];
    rotate<T>(lo, hi, c, s);
    base[i0] = lo;
    base[i1] = hi;
    return;
  }
  const int h = head - a.hq;
  const int64_t off = (static_cast<int64_t>(row) * a.hkv + h) * a.dim;
  const V* kb = reinterpret_cast<const V*>(k + off);
  V lo = kb[i0], hi = kb[i1];
  if (rotating) rotate<T>(lo, hi, c, s);
  if (k_out && (rotating || k_out != k)) {
    V* ko = reinterpret_cast<V*>(k_out + off);
    ko[i0] = lo;
    ko[i1] = hi;
  }
  if (!kc) return;
  const int64_t slot = __ldg(a.slots + row);
  if (slot < 0) return;
  if (slot >= a.cache_slots) {
    if (jp == 0 && h == 0) raise_device_error(a.err, FE_DEVERR_SLOT_RANGE);
    return;
  }
  const int64_t dst = (slot * a.hkv + h) * a.dim;
  V* kd = reinterpret_cast<V*>(kc + dst);
  kd[i0] = lo;
  kd[i1] = hi;
  const V* vb = reinterpret_cast<const V*>(v + off);
  V* vd = reinterpret_cast<V*>(vc + dst);
  vd[i0] = vb[i0];
  vd[i1] = vb[i1];
}

// 16-byte form, for rotary_dim a multiple of 16, dim a multiple of 8 and
// 16-byte aligned buffers. A head is `units` units: unit u < rot/16 owns the
// eight pairs 8u .. 8u+7 (two 16-byte chunks), the others an unrotated chunk.
// A thread keeps its unit and walks the heads hl, hl + hl_count, ... two at a
// time. The row's cos / sin, each pair's from the cache row of its own axis, are
// gathered into shared memory by asynchronous copies one row ahead (three
// buffers: the barrier before a row's use also ends the use of the row before
// the last), so that a pair's axis costs one 4-byte copy a row and not one load
// a head.
constexpr int kRowBufs = 3;
// From this many rows the ring of bulk copies is used (us by threads and by the
// ring, head_dim 128, all dims rotated): 4096 rows of 4 + 1 heads 8.7 and 9.9, of
// 16 + 1 heads 17.8 and 13.0, of 32 + 8 heads 23.0 and 20.3; 2048 rows of those 5.4 and
// 8.0, 9.3 and 8.6, 11.5 and 12.2; 32k rows of 4 + 1 heads 50.7 and 46.1, of 16 + 1
// heads 170 and 69. With fewer dims rotated the ring moves the rest of q as well,
// which the threads skip, and is the faster one all the same: 64k rows of 32 + 8 heads
// of 128 with 64 rotated 365 and 284, with 32 rotated 559 and 282, of 16 + 2 heads of
// 256 with 64 rotated 352 and 240.
constexpr int kBulkRows = 4096;
constexpr int kBulkSmem = 112 * 1024;

template <typename T>
__global__ void __launch_bounds__(kAxesThreads)
    rope_axes_vec_kernel(T* __restrict__ q, const T* k, const T* __restrict__ v, T* k_out,
                         T* __restrict__ kc, T* __restrict__ vc, const AxesArgs a,
                         const AxisMap map, int units, int hl_count) {
  using V = typename Pair2<T>::V;
  union Chunk {
    uint4 u;
    V v[4];
  };
  extern __shared__ __align__(16) float turns[];  // [kRowBufs][rot]: cos, then sin
  pdl_trigger();
  pdl_wait();  // q, k, v come from, and the pools are read by, earlier kernels
  const int heads = a.hq + a.hkv;
  const int hl = threadIdx.x / units, u = threadIdx.x - hl * units;
  const bool idle = hl >= hl_count;
  const int rot_units = a.rot / 16, r = a.rot / 2;
  const bool rotating = u < rot_units;
  const int e0 = rotating ? 8 * u : a.rot + 8 * (u - rot_units);
  const int e1 = e0 + r;  // the partners (rotating)
  const int first = blockIdx.x * hl_count + hl, step = gridDim.x * hl_count;
  auto gather = [&](int row, int buf) {
    for (int i = threadIdx.x; i < a.rot; i += blockDim.x) {
      const int j = i < r ? i : i - r;
      const int64_t p = __ldg(a.pos + static_cast<int64_t>(map.axis[j]) * a.rows + row);
      // a row that is out of range is skipped below; its copies stay in bounds
      const float* src = a.cache + (p >= 0 && p < a.max_positions ? p : 0) * a.rot + i;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(turns + buf * a.rot + i)),
                   "l"(src)
                   : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int buf = 0;
  if (static_cast<int>(blockIdx.y) < a.rows) gather(blockIdx.y, 0);
  for (int row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const int ahead = buf == kRowBufs - 1 ? 0 : buf + 1;
    Chunk lo[2], hi[2], vlo[2], vhi[2];
    auto load = [&](int h0) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int head = h0 + x * step;
        if (idle || head >= heads || (head < a.hq && !rotating)) continue;
        const T* src = head < a.hq ? q + (static_cast<int64_t>(row) * a.hq + head) * a.dim
                                   : k + (static_cast<int64_t>(row) * a.hkv + head - a.hq) * a.dim;
        lo[x].u = *reinterpret_cast<const uint4*>(src + e0);
        if (rotating) hi[x].u = *reinterpret_cast<const uint4*>(src + e1);
        if (head >= a.hq && kc) {
          const T* vs = v + (static_cast<int64_t>(row) * a.hkv + head - a.hq) * a.dim;
          vlo[x].u = *reinterpret_cast<const uint4*>(vs + e0);
          if (rotating) vhi[x].u = *reinterpret_cast<const uint4*>(vs + e1);
        }
      }
    };
    load(first);
    int p[kMaxAxes];
    const bool good = row_positions(a, row, p, threadIdx.x == 0 && blockIdx.x == 0);
    int64_t slot = kc ? __ldg(a.slots + row) : -1;
    if (slot >= a.cache_slots) {
      if (threadIdx.x == 0 && blockIdx.x == 0 && good)
        raise_device_error(a.err, FE_DEVERR_SLOT_RANGE);
      slot = -1;
    }
    if (row + static_cast<int>(gridDim.y) < a.rows)
      gather(row + gridDim.y, ahead);
    else
      asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    const float* cs = turns + buf * a.rot + 8 * u;
    buf = ahead;
    if (!good) continue;
    float4 c[2], s[2];
    if (rotating) {
      c[0] = *reinterpret_cast<const float4*>(cs);
      c[1] = *reinterpret_cast<const float4*>(cs + 4);
      s[0] = *reinterpret_cast<const float4*>(cs + r);
      s[1] = *reinterpret_cast<const float4*>(cs + r + 4);
    }
    for (int h0 = first;;) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int head = h0 + x * step;
        if (idle || head >= heads || (head < a.hq && !rotating)) continue;
        if (rotating)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 cc = c[i >> 1], ss = s[i >> 1];
            rotate<T>(lo[x].v[i], hi[x].v[i],
                      i & 1 ? make_float2(cc.z, cc.w) : make_float2(cc.x, cc.y),
                      i & 1 ? make_float2(ss.z, ss.w) : make_float2(ss.x, ss.y));
          }
        if (head < a.hq) {
          T* dst = q + (static_cast<int64_t>(row) * a.hq + head) * a.dim;
          *reinterpret_cast<uint4*>(dst + e0) = lo[x].u;
          *reinterpret_cast<uint4*>(dst + e1) = hi[x].u;
          continue;
        }
        const int h = head - a.hq;
        const int64_t off = (static_cast<int64_t>(row) * a.hkv + h) * a.dim;
        if (k_out && (rotating || k_out != k)) {
          *reinterpret_cast<uint4*>(k_out + off + e0) = lo[x].u;
          if (rotating) *reinterpret_cast<uint4*>(k_out + off + e1) = hi[x].u;
        }
        if (slot < 0) continue;
        const int64_t dst = (slot * a.hkv + h) * a.dim;
        *reinterpret_cast<uint4*>(kc + dst + e0) = lo[x].u;
        *reinterpret_cast<uint4*>(vc + dst + e0) = vlo[x].u;
        if (rotating) {
          *reinterpret_cast<uint4*>(kc + dst + e1) = hi[x].u;
          *reinterpret_cast<uint4*>(vc + dst + e1) = vhi[x].u;
        }
      }
      h0 += 2 * step;
      if (h0 >= heads) break;
      load(h0);
    }
  }
}

// Many rows: a CTA walks rows through a ring of shared-memory stages. A stage
// holds a row's q, k and v, brought by bulk copies several rows ahead; the threads
// turn q and k in place, and bulk copies take q back, k and v to their pool rows (and
// k to k_out), while the next rows are already there. Loads and stores are then
// in flight all the time, where a thread that loads, turns and stores its row
// itself keeps the memory waiting. The cos / sin come as in the kernel above, two
// rows ahead, and their positions and the slot four rows ahead. 64k rows of 32 + 8
// heads of 128, 1.6 GB: 258 us, 6.4 TB/s (426 us by the kernel above). A row's
// steps follow one another behind two barriers, so it is the CTAs of an SM that
// overlap, as many as their stages leave room for: five of 64 threads and three
// stages, where three of 256 threads and five stages took 328 us, two with eight
// stages 437 us. Short rows take a warp a CTA (16 + 1 heads: 69 us, 75 with two
// warps), long ones four (64 + 8 heads: 213 us, 248 with two).
constexpr uint32_t kStages = 3;
constexpr int kMetaBufs = 8;
// (what lies between the stages and `turns`, which is read 16 bytes at a time)
static_assert((kStages + 1 + kMetaBufs * (kMaxAxes + 1)) % 2 == 0, "turns: 16-byte aligned");

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst),
               "r"(smem_u32(src)), "r"(bytes)
               : "memory");
}

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads)
    rope_axes_bulk_kernel(T* __restrict__ q, const T* k, const T* __restrict__ v, T* k_out,
                          T* __restrict__ kc, T* __restrict__ vc, const AxesArgs a,
                          const AxisMap map, uint32_t stages) {
  using V = typename Pair2<T>::V;
  union Chunk {
    uint4 u;
    V v[4];
  };
  extern __shared__ __align__(128) uint8_t ring[];
  pdl_trigger();
  const uint32_t qb = a.hq * a.dim * 2, kb = a.hkv * a.dim * 2;
  const uint32_t stage_bytes = qb + kb + (kc ? kb : 0);
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + stages * stage_bytes);
  volatile int* flag = reinterpret_cast<volatile int*>(full + kStages);
  int64_t* meta = reinterpret_cast<int64_t*>(full + kStages + 1);
  float* turns = reinterpret_cast<float*>(meta + kMetaBufs * (kMaxAxes + 1));  // [kRowBufs][rot]
  if (threadIdx.x == 0) {
    for (int s = 0; s < static_cast<int>(stages); ++s) mbar_init(&full[s], 1);
    *flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  pdl_wait();  // q, k, v come from, and the pools are read by, earlier kernels
  const int rot_units = a.rot / 16, r = a.rot / 2, heads = a.hq + a.hkv;
  auto fetch = [&](int64_t row, int s) {  // one thread
    uint8_t* st = ring + s * stage_bytes;
    mbar_arrive_expect_tx(&full[s], stage_bytes);
    if (qb) bulk_load(st, q + row * a.hq * a.dim, qb, &full[s]);
    bulk_load(st + qb, k + row * a.hkv * a.dim, kb, &full[s]);
    if (kc) bulk_load(st + qb + kb, v + row * a.hkv * a.dim, kb, &full[s]);
  };
  // positions and slot of a row, four rows ahead: [row % kMetaBufs][kMaxAxes + 1]
  auto meta_ahead = [&](int64_t row, uint32_t n) {
    if (threadIdx.x <= kMaxAxes && row < a.rows) {
      const int64_t* src = nullptr;
      if (static_cast<int>(threadIdx.x) < a.axes)
        src = a.pos + static_cast<int64_t>(threadIdx.x) * a.rows + row;
      else if (threadIdx.x == kMaxAxes && kc)
        src = a.slots + row;
      if (src)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(
                         smem_u32(meta + n % kMetaBufs * (kMaxAxes + 1) + threadIdx.x)),
                     "l"(src)
                     : "memory");
    }
  };
  auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
  // its cos / sin, two rows ahead
  auto gather = [&](int64_t row, uint32_t n) {
    if (row >= a.rows) return;
    const int64_t* m = meta + n % kMetaBufs * (kMaxAxes + 1);
    float* dst = turns + n % kRowBufs * a.rot;
    for (int i = threadIdx.x; i < a.rot; i += kThreads) {
      const int64_t p = m[map.axis[i < r ? i : i - r]];
      // a row that is out of range is skipped below; its copies stay in bounds
      const float* src = a.cache + (p >= 0 && p < a.max_positions ? p : 0) * a.rot + i;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst + i)), "l"(src)
                   : "memory");
    }
  };
  const int64_t step = gridDim.x;
  int64_t fetched = blockIdx.x;        // next row to fetch (thread 0)
  uint32_t nf = 0, n = 0;              // rows fetched, rows done
  if (threadIdx.x == 0)
    for (; nf < stages - 1 && fetched < a.rows; fetched += step, ++nf)
      fetch(fetched, nf);
  for (uint32_t i = 0; i < 4; ++i) meta_ahead(blockIdx.x + i * step, i);
  commit();
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  for (uint32_t i = 0; i < 2; ++i) {
    gather(blockIdx.x + i * step, i);
    commit();
  }
  bool ok = true;
  for (int64_t row = blockIdx.x; row < a.rows; row += step, ++n) {
    const uint32_t s = n % stages;
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    ok = wait_bounded(&full[s], (n / stages) & 1u, flag);
    if (!__syncthreads_and(ok)) {  // (and what came by cp.async is there for everyone)
      ok = false;
      break;
    }
    gather(row + 2 * step, n + 2);
    meta_ahead(row + 4 * step, n + 4);
    commit();
    const int64_t* m = meta + n % kMetaBufs * (kMaxAxes + 1);
    bool good = true;
    for (int i = 0; i < a.axes; ++i) good &= m[i] >= 0 && m[i] < a.max_positions;
    const float* cs = turns + n % kRowBufs * a.rot;
    uint8_t* st = ring + s * stage_bytes;
    if (good) {
      for (int t = threadIdx.x; t < heads * rot_units; t += kThreads) {
        const int head = t / rot_units, u = t - head * rot_units;
        uint4* x = reinterpret_cast<uint4*>(st + head * a.dim * 2) + u;
        uint4* y = x + r / 8;
        const float* c = cs + 8 * u;
        Chunk lo, hi;
        lo.u = *x;
        hi.u = *y;
        const float4 c0 = *reinterpret_cast<const float4*>(c);
        const float4 c1 = *reinterpret_cast<const float4*>(c + 4);
        const float4 s0 = *reinterpret_cast<const float4*>(c + r);
        const float4 s1 = *reinterpret_cast<const float4*>(c + r + 4);
        rotate<T>(lo.v[0], hi.v[0], make_float2(c0.x, c0.y), make_float2(s0.x, s0.y));
        rotate<T>(lo.v[1], hi.v[1], make_float2(c0.z, c0.w), make_float2(s0.z, s0.w));
        rotate<T>(lo.v[2], hi.v[2], make_float2(c1.x, c1.y), make_float2(s1.x, s1.y));
        rotate<T>(lo.v[3], hi.v[3], make_float2(c1.z, c1.w), make_float2(s1.z, s1.w));
        *x = lo.u;
        *y = hi.u;
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
      int64_t slot = kc ? m[kMaxAxes] : -1;
      if (!good) raise_device_error(a.err, FE_DEVERR_POS_RANGE);
      if (good && slot >= a.cache_slots) {
        raise_device_error(a.err, FE_DEVERR_SLOT_RANGE);
        slot = -1;
      }
      if (good) {
        if (qb) bulk_store(q + row * a.hq * a.dim, st, qb);
        if (k_out) bulk_store(k_out + row * a.hkv * a.dim, st + qb, kb);
        if (slot >= 0) {
          bulk_store(kc + slot * a.hkv * a.dim, st + qb, kb);
          bulk_store(vc + slot * a.hkv * a.dim, st + qb + kb, kb);
        }
      }
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      // the stage of the row before this one is free once its stores have read it
      if (fetched < a.rows) {
        asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        fetch(fetched, nf % stages);
        fetched += step;
        ++nf;
      }
    }
  }
  if (threadIdx.x == 0) {
    if (!ok) {
      raise_device_error(a.err, FE_DEVERR_TIMEOUT);
      volatile int never = 0;
      for (uint32_t t = n; t < nf; ++t)  // what was fetched has landed (bounded)
        (void)wait_bounded(&full[t % stages], (t / stages) & 1u, &never);
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
}

template <typename T>
int launch_axes(void* q, const void* k, const void* v, void* k_out, void* kc, void* vc,
                const AxesArgs& a, const AxisMap& map, cudaStream_t stream) {
  T* tq = static_cast<T*>(q);
  const T* tk = static_cast<const T*>(k);
  const T* tv = static_cast<const T*>(v);
  T *to = static_cast<T*>(k_out), *tkc = static_cast<T*>(kc), *tvc = static_cast<T*>(vc);
  const int heads = a.hq + a.hkv;
  const int units = a.rot / 16 + (a.dim - a.rot) / 8;
  if (a.rot % 16 == 0 && a.dim % 8 == 0 && aligned16(q) && aligned16(k) && aligned16(v) &&
      aligned16(k_out) && aligned16(kc) && aligned16(vc) && aligned16(a.cache) &&
      units <= kAxesThreads) {
    // heads of a row over as few blocks as fit, evenly
    const int most = kAxesThreads / units;
    const int passes = (heads + most - 1) / most;
    const int hl = (heads + passes - 1) / passes;
    const int vec_threads = (hl * units + 31) / 32 * 32;
    const int stage = (heads + (kc ? a.hkv : 0)) * a.dim * 2;
    const int smem = static_cast<int>(kStages) * stage +
                     8 * (kStages + 1 + kMetaBufs * (kMaxAxes + 1)) + 4 * kRowBufs * a.rot;
    if (a.rows >= kBulkRows && smem <= kBulkSmem) {
      static std::atomic<uint64_t> done[3];
      const int i = stage <= 5120 ? 0 : stage <= 14336 ? 1 : 2;
      auto kernel = i == 0   ? rope_axes_bulk_kernel<T, 32>
                    : i == 1 ? rope_axes_bulk_kernel<T, 64>
                             : rope_axes_bulk_kernel<T, 128>;
      FE_CUDA_TRY(allow_smem(kernel, kBulkSmem, done[i]));
      const int per_sm = std::min(40, 225 * 1024 / (smem + 1024));
      FE_CUDA_TRY(launch_pdl(kernel, dim3(std::min(a.rows, 148 * per_sm)), dim3(32 << i), smem,
                             stream, tq, tk, tv, to, tkc, tvc, a, map, kStages));
      return FE_OK;
    }
    const int gx = a.rows < 1024 ? passes : (passes + 1) / 2;
    // a row a block while there are few; then blocks that walk the rows, as many
    // as are resident
    const int resident = 148 * std::max(1, 65536 / (80 * vec_threads));  // by registers
    const int gy = a.rows < 1024 ? a.rows : std::min(a.rows, std::max(1, resident / gx));
    FE_CUDA_TRY(launch_pdl(rope_axes_vec_kernel<T>, dim3(gx, gy), dim3(vec_threads),
                           sizeof(float) * kRowBufs * a.rot, stream, tq, tk, tv, to, tkc, tvc, a,
                           map, units, hl));
    return FE_OK;
  }
  const int64_t total = static_cast<int64_t>(a.rows) * heads * (a.dim / 4);
  const int64_t blocks = (total + kAxesThreads - 1) / kAxesThreads;
  if (blocks > INT32_MAX) return fail(FE_ERR_CAPACITY, "fe_rope_axes: too many rows");
  FE_CUDA_TRY(launch_pdl(rope_axes_kernel<T>, dim3(static_cast<int>(blocks)), dim3(kAxesThreads),
                         0, stream, tq, tk, tv, to, tkc, tvc, a, map));
  return FE_OK;
}

int run_axes(const char* what, void* q, const void* k, const void* v, void* k_out, void* k_pool,
             void* v_pool, const int64_t* slots, const int64_t* pos, int axes,
             const uint8_t* pair_axis, const float* cache, int rows, int hq, int hkv, int dim,
             int rot, int max_positions, int dtype, int64_t cache_slots, bool append,
             void* stream) {
  const std::string name = what;
  if (!valid_dtype(dtype)) return fail(FE_ERR_INVALID_ARGUMENT, name + ": bad dtype");
  if (rows < 0 || hq < 0 || hkv <= 0 || dim <= 0 || max_positions <= 0)
    return fail(FE_ERR_INVALID_ARGUMENT, name + ": sizes out of range");
  if (axes < 1 || axes > kMaxAxes)
    return fail(FE_ERR_UNSUPPORTED, name + ": 1 to 4 axes");
  if (dim % 4 != 0 || rot < 0 || rot > dim || rot % 4 != 0 || rot > 2 * kMaxPairs)
    return fail(FE_ERR_UNSUPPORTED, name + ": dim and rotary_dim must be multiples of 4, "
                                           "rotary_dim <= dim and <= 512");
  // (row and element indexes of a step ahead stay within 31 bits)
  if (rows > (1 << 30) || (int64_t(hq) + hkv) * dim > (1 << 24))
    return fail(FE_ERR_CAPACITY, name + ": at most 2^30 rows of 2^24 elements");
  if (rot > 0 && !pair_axis) return fail(FE_ERR_INVALID_ARGUMENT, name + ": pair_axis is null");
  AxisMap map{};
  for (int j = 0; j < rot / 2; ++j) {
    if (pair_axis[j] >= axes)
      return fail(FE_ERR_INVALID_ARGUMENT, name + ": a pair's axis is not below `axes`");
    map.axis[j] = pair_axis[j];
  }
  if (rows == 0) return FE_OK;
  if (!k || !pos || (rot > 0 && !cache) || (hq > 0 && !q))
    return fail(FE_ERR_INVALID_ARGUMENT, name + ": null pointer");
  if (append && (!v || !k_pool || !v_pool || !slots))
    return fail(FE_ERR_INVALID_ARGUMENT, name + ": null pointer");
  if (append && cache_slots <= 0)
    return fail(FE_ERR_INVALID_ARGUMENT, name + ": cache_slots <= 0");
  for (const void* p : {static_cast<const void*>(q), k, v, static_cast<const void*>(k_out),
                        static_cast<const void*>(k_pool), static_cast<const void*>(v_pool),
                        static_cast<const void*>(cache)})
    if (reinterpret_cast<uintptr_t>(p) & 3u)
      return fail(FE_ERR_INVALID_ARGUMENT, name + ": buffers must be 4-byte aligned");
  if ((reinterpret_cast<uintptr_t>(pos) | reinterpret_cast<uintptr_t>(slots)) & 7u)
    return fail(FE_ERR_INVALID_ARGUMENT, name + ": pos and slots must be 8-byte aligned");
  const AxesArgs a{slots, pos, cache, device_error_word(), cache_slots, rows, axes, hq, hkv, dim,
                   rot, max_positions};
  auto s = static_cast<cudaStream_t>(stream);
  if (dtype == FE_DTYPE_BF16)
    return launch_axes<__nv_bfloat16>(q, k, v, k_out, k_pool, v_pool, a, map, s);
  return launch_axes<__half>(q, k, v, k_out, k_pool, v_pool, a, map, s);
}

}  // namespace
}  // namespace fe

using namespace fe;

extern "C" {

int fe_rope_axes(void* q, void* k, const int64_t* pos, int axes, const uint8_t* pair_axis,
                 const float* cache, int rows, int hq, int hkv, int dim, int rotary_dim,
                 int max_positions, int dtype, void* stream) {
  return run_axes("fe_rope_axes", q, k, nullptr, k, nullptr, nullptr, nullptr, pos, axes,
                  pair_axis, cache, rows, hq, hkv, dim, rotary_dim, max_positions, dtype, 0, false,
                  stream);
}

int fe_rope_axes_append(void* q, const void* k, const void* v, void* k_out, void* k_pool,
                        void* v_pool, const int64_t* slots, const int64_t* pos, int axes,
                        const uint8_t* pair_axis, const float* cache, int rows, int hq, int hkv,
                        int dim, int rotary_dim, int max_positions, int dtype,
                        int64_t cache_slots, void* stream) {
  return run_axes("fe_rope_axes_append", q, k, v, k_out, k_pool, v_pool, slots, pos, axes,
                  pair_axis, cache, rows, hq, hkv, dim, rotary_dim, max_positions, dtype,
                  cache_slots, true, stream);
}

}  // extern "C"
