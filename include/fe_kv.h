/*
 * fe_kv.h — C ABI of the B200 (sm_100a) paged-KV hot path for FlashEngine.cpp.
 *
 * Drop-in for the KV and attention operators behind the reference's CUDA
 * DeviceModel (Cambridgebit/FlashEngine.cpp include/fe/native_cuda.hpp:6-14):
 * K/V append through the slot mapping, paged GQA attention (decode, chunked
 * prefill, speculative verify) over per-sequence block tables, plus a
 * block-copy / copy-on-write operator the reference does not have.
 *
 * Conventions
 *  - Every entry point returns an fe_status; 0 (FE_OK) is success. No C++
 *    exception crosses this boundary. fe_last_error() returns a detail string
 *    for the calling thread's most recent failure.
 *  - `stream` is a cudaStream_t passed as void* (0 = legacy default stream),
 *    the same convention as the reference's `void* stream`.
 *  - Element data are fp16 or bf16 (`dtype`: FE_DTYPE_F16 / FE_DTYPE_BF16).
 *    `bf16` in the shim (fe_native_cuda.hpp) maps to FE_DTYPE_BF16.
 *  - KV pools are laid out as in the reference (src/cuda_model.cpp:60):
 *    [num_blocks + 1, page, hkv, dim], i.e. a flat [cache_slots, hkv*dim]
 *    with cache_slots = (num_blocks + 1) * page. The last page
 *    (index num_blocks) is the graph-padding page and is never handed to a
 *    request.
 *  - Device pointers unless stated "host".
 */
#ifndef FE_KV_H_
#define FE_KV_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FE_KV_ABI_VERSION 1

typedef enum fe_status {
  FE_OK = 0,
  FE_ERR_INVALID_ARGUMENT = 1, /* bad shape, null pointer, unsupported combination */
  FE_ERR_CAPACITY = 2,         /* batch/pages/work beyond the plan's fixed capacity */
  FE_ERR_CONTEXT = 3,          /* a sequence's length < its query rows, or > max context */
  FE_ERR_CUDA = 4,             /* a CUDA runtime call failed (detail in fe_last_error) */
  FE_ERR_UNSUPPORTED = 5,      /* head_dim / page size / group size not compiled */
  FE_ERR_DEVICE = 6,           /* a kernel recorded an error (e.g. out-of-range slot) */
  FE_ERR_NO_DEVICE = 7         /* no usable sm_100 device */
} fe_status;

typedef enum fe_dtype { FE_DTYPE_F16 = 0, FE_DTYPE_BF16 = 1 } fe_dtype;

/* Bits reported by fe_device_errors(). */
#define FE_DEVERR_SLOT_RANGE 0x1u  /* append: slot >= cache_slots (row skipped) */
#define FE_DEVERR_PAGE_RANGE 0x2u  /* copy/clear: page index out of range (copy skipped) */
#define FE_DEVERR_NTOK_RANGE 0x4u  /* copy: ntok outside [0, page] (copy skipped) */
#define FE_DEVERR_TIMEOUT 0x8u     /* attention: a pipeline wait exceeded its bound */
#define FE_DEVERR_SMEM_ALIGN 0x10u /* attention: dynamic shared memory not 1 KiB aligned (launch skipped) */
#define FE_DEVERR_POS_RANGE 0x20u  /* rope: position outside [0, max_positions) (row skipped) */
#define FE_DEVERR_PLAN 0x40u       /* device-side prepare: invalid step or capacity (plan emptied) */

const char* fe_status_string(int status);
const char* fe_last_error(void);
int fe_abi_version(void);

/* Read and clear the device-side error bits of the current device (see
 * FE_DEVERR_*). Synchronises `stream`. */
int fe_device_errors(void* stream, uint32_t* bits_out);

/* ------------------------------------------------------------------------
 * K/V append. Replaces fe::cuda::store (include/fe/native_cuda.hpp:14;
 * src/cuda_kernels.cu:24 store_kernel and :34 its launcher).
 *   k, v:        [rows, width] new post-RoPE keys / values (width = hkv*dim)
 *   k_pool/v_pool: [cache_slots, width]
 *   slots:       int64 [rows] (device); slot < 0 rows are skipped (graph
 *                padding, as the reference CUDA kernel does); a slot
 *                >= cache_slots is skipped and raises FE_DEVERR_SLOT_RANGE.
 * Bit-exact copy. width must be a multiple of 8 elements (16 bytes).
 * ------------------------------------------------------------------------ */
int fe_kv_append(const void* k, const void* v, void* k_pool, void* v_pool, const int64_t* slots,
                 int rows, int width, int dtype, int cache_slots, void* stream);

/* ------------------------------------------------------------------------
 * Block copy / copy-on-write. No reference counterpart: the reference
 * shares only whole published pages and never copies one
 * (src/scheduler.cpp:6-29). For each copy c and each layer l, token rows
 * [0, ntok[c]) of page src[c] are copied onto page dst[c] in both
 * k_pools[l] and v_pools[l] (ntok = page copies a whole block; a smaller
 * ntok is the copy-on-write of a shared partial tail block).
 *   k_pools, v_pools: HOST arrays of num_layers device pool pointers
 *                     (num_layers <= FE_MAX_LAYERS)
 *   src, dst, ntok:   int32 [num_copies] (device)
 * Source and destination pages of one call must not overlap.
 * ------------------------------------------------------------------------ */
#define FE_MAX_LAYERS 128
int fe_kv_copy_blocks(void* const* k_pools, void* const* v_pools, int num_layers,
                      const int32_t* src, const int32_t* dst, const int32_t* ntok, int num_copies,
                      int page, int width, int num_pages_total, int dtype, void* stream);

/* Copy lists for forked sequences (no reference counterpart; HOST memory
 * only, needs no GPU). The reference shares only whole published pages and
 * recomputes the rest of a shared prefix by prefill (src/scheduler.cpp:6-29);
 * a fork that copies KV instead gives, for each fork f, the parent's block
 * table parent_tables[parent_off[f] .. parent_off[f+1]), the child's table
 * child_tables[child_off[f] .. child_off[f+1]) as the scheduler assigned it
 * (the parent's full pages it shares, then pages of its own) and the
 * length fork_len[f] of the prefix the child continues from. For every page
 * j < ceil(fork_len/page) the child does not share, one copy entry
 * (src = parent[j], dst = child[j], ntok = the prefix tokens on that page:
 * page, or fork_len % page for the tail) is written to src/dst/ntok, ready
 * for fe_kv_copy_blocks, which must run before either sequence appends.
 * Rejected with FE_ERR_INVALID_ARGUMENT: a shared page that is not full (both
 * sequences would append into it: the copy-on-write case), a child page that
 * is one of the parent's pages at another position, a fork length beyond
 * either table. FE_ERR_CAPACITY when the copies exceed `capacity`.
 * *num_copies receives the number of entries written. */
int fe_kv_fork_copies(int num_forks, const int32_t* parent_tables, const int32_t* parent_off,
                      const int32_t* child_tables, const int32_t* child_off,
                      const int64_t* fork_len, int page, int32_t* src, int32_t* dst,
                      int32_t* ntok, int capacity, int* num_copies);

/* Zero-fill whole pages (e.g. the graph-padding page num_blocks, which the
 * reference gets from at::zeros at start-up, src/cuda_model.cpp:60).
 *   pools: HOST array of num_pools device pool pointers
 *   pages: int32 [num_pages] (device) */
int fe_kv_clear_pages(void* const* pools, int num_pools, const int32_t* pages, int num_pages,
                      int page, int width, int num_pages_total, int dtype, void* stream);

/* Gather the KV of whole sequences into a dense buffer: the index_select
 * of the reference ATen path (src/portable_gpu_ops.cpp:40) without its
 * padding to max_context. Token t of sequence b is read from slot
 * pages[kv[b] + t/page]*page + t%page, and written to row
 * kv_row_offset[b] + t of `out` ([sum of lengths, width]).
 *   kv, pages, last, kv_row_offset: int32 (device), as in prepare. */
int fe_kv_gather(const void* pool, void* out, const int32_t* kv, const int32_t* pages,
                 const int32_t* last, const int32_t* row_offset, int batch, int max_len, int page,
                 int width, int dtype, void* stream);

/* ------------------------------------------------------------------------
 * Eviction from the paged cache by accumulated attention weight (no reference
 * counterpart). Scores are fp32 [hkv, cache_slots], one for each cached token
 * and KV head, as fe_scored_attn_run accumulates them. Both calls take DEVICE
 * metadata: kv [batch+1], pages [num_pages] (kv[batch] of them are used) and
 * last [batch] as in fe_attn_plan_prepare. A sequence that reaches past the
 * page list, or a page past the pool, is skipped (its kept entries are -1) and
 * raises FE_DEVERR_PAGE_RANGE. A budget of at most 2^30 tokens.
 *
 * fe_kv_select: the tokens to keep, int32 kept [batch, hkv, budget], ascending.
 * Of a sequence of more than `budget` tokens each KV head keeps the first `sink`,
 * the last `recent`, and of the others those with the highest scores, `budget`
 * in all; of equal scores (-0 and +0 are equal) the lowest token indexes win,
 * NaN is below every number. A shorter sequence keeps all of its tokens, and -1
 * fills the rest. max_len sizes the launch: sequences of up to max_len tokens
 * (and up to 131072) are read twice, longer ones several times. A page that lies
 * outside the pool counts as NaN.
 *
 * fe_kv_compact: for each KV head, the K and V row and (scores not NULL) the
 * score of token kept[b, h, j] become those of token j of the sequence, for
 * every j before the first -1. With dst_kv / dst_pages NULL in place: kept[b, h,
 * j] >= j has to hold (an ascending list's does), and the sequence goes on with
 * as many tokens as were kept; what its slots past them held is unspecified.
 * Otherwise the tokens go to the pages dst_pages[dst_kv[b] ..], none of which
 * may be among the source pages of any sequence of the call: the source keeps
 * its tokens. A page that is written belongs to one sequence. Entries that break
 * these bounds are skipped and raise FE_DEVERR_PAGE_RANGE. dim a multiple of 8,
 * at most 512; pools and scores 16-byte aligned; cache_slots whole pages.
 * ------------------------------------------------------------------------ */
int fe_kv_select(const float* scores, const int32_t* kv, const int32_t* pages, int num_pages,
                 const int32_t* last, int32_t* kept, int batch, int max_len, int hkv, int page,
                 int budget, int sink, int recent, int64_t cache_slots, void* stream);
int fe_kv_compact(void* k_pool, void* v_pool, float* scores, const int32_t* kept,
                  const int32_t* kv, const int32_t* pages, int num_pages, const int32_t* last,
                  const int32_t* dst_kv, const int32_t* dst_pages, int num_dst_pages, int batch,
                  int hkv, int dim, int page, int budget, int dtype, int64_t cache_slots,
                  void* stream);

/* ------------------------------------------------------------------------
 * Rotary embedding. Replaces fe::cuda::rope (include/fe/native_cuda.hpp:13;
 * src/cuda_kernels.cu:19-23 rope_kernel and :33 its launcher), bit-exact:
 * with r = rotary_dim / 2, for each head and pair (j, j + r), j < r, with
 * c = cache[pos*rotary_dim + j] and s = cache[pos*rotary_dim + r + j] (fp32
 * cache [max_positions, rotary_dim], cos then sin), x[j] = a*c - b*s and
 * x[j + r] = b*c + a*s, each product and sum rounded to fp32 separately, the
 * result rounded to the 16-bit type. rotary_dim = dim is the reference's
 * rope; rotary_dim < dim rotates only the leading dims (the partial rotary of
 * Qwen3.5 full-attention layers, src/hybrid_model.cpp:44) and leaves the rest.
 *   q: [rows, hq, dim], k: [rows, hkv, dim] (rotated in place; hq may be 0)
 *   pos: int64 [rows] (device). A position outside [0, max_positions) leaves
 *        its row unrotated and raises FE_DEVERR_POS_RANGE (the reference
 *        reads out of bounds there).
 * dim and rotary_dim multiples of 4, rotary_dim <= dim; q/k 4-byte aligned,
 * cache 8-byte aligned.
 * ------------------------------------------------------------------------ */
int fe_rope(void* q, void* k, const int64_t* pos, const float* cache, int rows, int hq, int hkv,
            int dim, int rotary_dim, int max_positions, int dtype, void* stream);

/* Fused RoPE + K/V append (one launch): rotates q in place, and writes the
 * rotated keys and the values to the pools through the slot mapping exactly
 * as fe_rope followed by fe_kv_append would (slot < 0 skipped, slot >=
 * cache_slots skipped and flagged). k and v ([rows, hkv, dim]) are read
 * only; when k_out is not NULL the rotated keys are also written there (k_out
 * may equal k). Pools are [cache_slots, hkv*dim]. */
int fe_rope_append(void* q, const void* k, const void* v, void* k_out, void* k_pool,
                   void* v_pool, const int64_t* slots, const int64_t* pos, const float* cache,
                   int rows, int hq, int hkv, int dim, int rotary_dim, int max_positions,
                   int dtype, int64_t cache_slots, void* stream);

/* ------------------------------------------------------------------------
 * Rotary embedding with several position axes (no reference counterpart:
 * its rope has one position a row). As fe_rope and fe_rope_append, but pair j
 * of a head, (x[j], x[j + rotary_dim/2]), turns by the cache row of its own
 * axis: pos is int64 [axes, rows], and pair_axis[j] (HOST, rotary_dim/2 bytes,
 * read by the call) names the axis of pair j, e.g. time, height and width of an
 * image's patches, in sections or taking turns. Equal positions on all axes
 * give fe_rope's bits. A row with a position outside [0, max_positions) on any
 * axis is skipped (rotation and append) and raises FE_DEVERR_POS_RANGE.
 * axes 1 .. 4, rotary_dim <= 512; else as fe_rope.
 * ------------------------------------------------------------------------ */
#define FE_MAX_AXES 4
int fe_rope_axes(void* q, void* k, const int64_t* pos, int axes, const uint8_t* pair_axis,
                 const float* cache, int rows, int hq, int hkv, int dim, int rotary_dim,
                 int max_positions, int dtype, void* stream);
int fe_rope_axes_append(void* q, const void* k, const void* v, void* k_out, void* k_pool,
                        void* v_pool, const int64_t* slots, const int64_t* pos, int axes,
                        const uint8_t* pair_axis, const float* cache, int rows, int hq, int hkv,
                        int dim, int rotary_dim, int max_positions, int dtype,
                        int64_t cache_slots, void* stream);

/* ------------------------------------------------------------------------
 * Greedy speculative acceptance. Replaces fe::cuda::accept
 * (include/fe/native_cuda.hpp:15; src/cuda_kernels.cu:25 accept_kernel and
 * :35 its launcher). For each row b: m = the number of leading draft tokens
 * draft[b, i] equal to verify[b, i]; out[b, 0..m) = those drafts,
 * out[b, m] = verify[b, m], out[b, k+1] = m + 1; out[b, m+1..k] untouched.
 *   draft: int64 [batch, k], verify: int64 [batch, k+1], out: int64 [batch, k+2]
 * ------------------------------------------------------------------------ */
int fe_accept(const int64_t* draft, const int64_t* verify, int64_t* out, int batch, int k,
              void* stream);

/* ------------------------------------------------------------------------
 * Paged attention plan. Replaces fe::cuda::create_plan / destroy_plan /
 * prepare_plan (include/fe/native_cuda.hpp:7-9; src/flashinfer_attention.cu:22-34).
 * ------------------------------------------------------------------------ */
typedef struct fe_attn_plan fe_attn_plan;

/* head_dim 128 (as src/flashinfer_attention.cu:23 requires) or 256 (the
 * full-attention layers of hybrid and DFlash draft models, which the reference
 * serves through ATen with any head_dim: src/hybrid_model.cpp:98,
 * src/block_draft.cpp:38); page a multiple of 16; hq a multiple of hkv with
 * hq/hkv <= 16.
 * max_pages = per-sequence page capacity (the reference passes
 * ceil(max_model_len/page)+1, src/cuda_model.cpp:118). Allocates the plan's
 * fixed device workspaces on the current device. */
int fe_attn_plan_create(int hq, int hkv, int dim, int page, int max_batch, int max_pages,
                        int dtype, int num_blocks, fe_attn_plan** plan_out);
int fe_attn_plan_destroy(fe_attn_plan* plan);

/* Per-step metadata, HOST pointers (as fe::cuda::prepare_plan):
 *   qo[batch+1]   query-row prefix sums (rows per sequence: 1 = decode,
 *                 k+1 = verify, chunk = prefill)
 *   kv[batch+1]   page-count prefix sums into `pages`
 *   pages[kv[batch]] physical page ids, each in [0, num_blocks]
 *   last[batch]   tokens in each sequence's last page, 1..page
 * length_b = (kv[b+1]-kv[b]-1)*page + last[b] keys; query row r of
 * sequence b is its (r - qo[b])-th of qrows_b = qo[b+1]-qo[b] rows.
 * Builds the work list on the host and uploads it with one async copy on
 * `stream` into fixed device buffers, so a CUDA graph that captured
 * fe_attn_run replays correctly after any later prepare (graph != 0 only
 * asserts that the row count is unchanged). */
int fe_attn_plan_prepare(fe_attn_plan* plan, const int32_t* qo, const int32_t* kv,
                         const int32_t* pages, const int32_t* last, int batch, int rows, int graph,
                         void* stream);

/* Paged GQA attention. Replaces fe::cuda::attention
 * (include/fe/native_cuda.hpp:10; src/flashinfer_attention.cu:35-44).
 *   q, out: [rows, hq, dim]; k_pool, v_pool: [cache_slots, hkv, dim]
 *           (dim = the plan's head_dim, 128 or 256)
 *   causal != 0: row i of a sequence with qrows rows sees keys
 *                t <= length - qrows + i (bottom-right aligned);
 *   causal == 0: every row sees t < length (DFlash draft / block verify).
 * Scale 1/sqrt(dim); fp32 accumulation; output rounded to nearest even.
 * A step prepared outside graph mode that mixes decode rows with multi-row
 * sequences may run its two kernels side by side: the multi-row kernel on a
 * stream the plan owns, forked from `stream` by an event and joined back
 * before the call returns, so the call is ordered on `stream` as usual (and
 * a capture of `stream` records the fork and the join). */
int fe_attn_run(fe_attn_plan* plan, const void* q, const void* k_pool, const void* v_pool,
                void* out, int causal, void* stream);

/* fe_attn_run restricted to some of the prepared work: FE_ATTN_LISTS_DECODE
 * (the rows that run on the decode kernel, and their split-K merge) and/or
 * FE_ATTN_LISTS_ROWS (multi-row sequences on the tcgen05 kernel).
 * fe_attn_run is FE_ATTN_LISTS_ALL. Calling the two parts back to back on one
 * stream does the same work as one fe_attn_run (used to time each kernel). */
#define FE_ATTN_LISTS_DECODE 1
#define FE_ATTN_LISTS_ROWS 2
#define FE_ATTN_LISTS_ALL 3
int fe_attn_run_lists(fe_attn_plan* plan, const void* q, const void* k_pool, const void* v_pool,
                      void* out, int causal, int lists, void* stream);

/* Decode attention that allocates nothing. No counterpart in the reference:
 * it is for callers that cannot call cudaMalloc where they run attention
 * (hosts that give all free device memory to their own pool allocator at
 * start-up, so a later allocation fails; hot loops where an allocation,
 * which may synchronise the device, is not allowed). Same arithmetic as
 * fe_attn_run for one query row per sequence, but no plan: kv, pages and
 * last are DEVICE int32 arrays laid out as in fe_attn_plan_prepare, and the
 * work split is derived on the device.
 * head_dim 128 only: q and out are [batch, hq, 128], row b of q/out belongs
 * to sequence b; pools are [cache_slots, hkv, 128].
 * Split-K scratch is a fixed 16 MiB (+64 KiB counters) array inside the
 * library that every GPU loading it holds until exit; batch x KV-head groups
 * beyond 16384 is rejected with FE_ERR_CAPACITY, and batches whose split
 * records would not fit that array run every sequence unsplit (same
 * results, less parallelism for long contexts). The first call on a device
 * resolves that array's device address and sets kernel attributes — make it
 * before any stream capture. Calls share the array: sequential calls are
 * safe, calls that overlap on the GPU race. Out-of-range page ids or last
 * values are reported through fe_device_errors. */
int fe_paged_decode_noalloc(const void* q, const void* k_pool, const void* v_pool, void* out,
                            const int32_t* kv, const int32_t* pages, const int32_t* last,
                            int batch, int hq, int hkv, int page, int num_blocks, int max_pages,
                            int dtype, void* stream);

/* ------------------------------------------------------------------------
 * 8-bit KV cache (no reference counterpart: the reference's pools are
 * 16-bit, src/cuda_model.cpp:60). Keys and values are e4m3 codes
 * [cache_slots, hkv, dim] with one power-of-two scale per block of
 * FE_KV8_BLOCK consecutive slots and KV head, stored as its biased exponent,
 * uint8 [cache_slots / FE_KV8_BLOCK, hkv]:
 *   value = code * 2^(exponent - 127).
 * Half the bytes of a 16-bit pool (and 1/16 byte per 128 for the scales), so
 * half the attention traffic and twice the tokens; slots, block tables, page
 * lists and plans are as for the 16-bit pools. page is a multiple of 16.
 *
 * What a cache holds is set by fe_kv8_append: exponents within 2^-32 .. 2^64
 * (bytes 95 .. 191; attention, gather and an append that keeps a block's
 * tokens read a byte outside as the nearest of these, so pages never written to
 * are harmless beyond a sequence's end), codes of magnitude up to 448, NaN
 * where the input was NaN.
 * ------------------------------------------------------------------------ */
#define FE_KV8_BLOCK 16

/* Rotation, quantisation and append in one launch. q [rows, hq, dim] is
 * rotated into q_out (which may be q; hq may be 0) exactly as by fe_rope; k is
 * rotated the same way, in fp32 and not rounded before it is quantised; v is
 * taken as it is. rotary_dim = 0 rotates nothing (pos and cache may be NULL; q
 * is copied).
 * A RUN is a sequence of adjacent rows (skipped ones aside) whose slots lie in
 * one block, in increasing order. Per KV head, and for K and V apart, a run's
 * scale is the smallest power of two s with |x| <= 448 s for its largest
 * finite magnitude |x|, no smaller than the block's present scale when the run
 * does not begin at the block's first slot: the tokens before it are kept, and
 * their codes are rounded to the new scale when it grew (exact but for codes
 * that become subnormal). Tokens of the block after the run are not kept: an append at
 * slot n leaves slots n + 1 .. of its block undefined (they hold rejected
 * drafts at most; the next append overwrites them). Codes are rounded to
 * nearest even; infinities saturate, NaN stays NaN.
 * A block's scale falls only when its first slot is written again: a rejected
 * draft that was far larger than the accepted tokens of its block leaves them
 * at the scale that it needed, with the bits that were left to them there.
 * A call has at most one run in a block (every step's slot mapping does: a
 * sequence's rows are adjacent and in order): two would race for its scale,
 * and that block's contents are then unspecified.
 *   slots: int64 [rows]; < 0: skipped; >= cache_slots: skipped,
 *          FE_DEVERR_SLOT_RANGE. pos: int64 [rows]; outside [0,
 *          max_positions): the row's k, v and q are skipped,
 *          FE_DEVERR_POS_RANGE.
 * dim 128 or 256; rotary_dim a multiple of 8; cache_slots a multiple of 16,
 * below 2^31; k, v and the cos / sin cache 16-byte, q and codes 8-byte
 * aligned. */
int fe_kv8_append(const void* q, void* q_out, const void* k, const void* v, uint8_t* k_codes,
                  uint8_t* v_codes, uint8_t* k_exp, uint8_t* v_exp, const int64_t* slots,
                  const int64_t* pos, const float* cache, int rows, int hq, int hkv, int dim,
                  int rotary_dim, int max_positions, int dtype, int64_t cache_slots,
                  void* stream);

/* fe_kv_gather from an 8-bit pool: the values, rounded to the 16-bit `dtype`
 * (bf16 holds every one exactly). A page id that reaches past cache_slots
 * leaves its token unwritten and raises FE_DEVERR_PAGE_RANGE, a `last` outside
 * [1, page] or a negative list entry its sequence. cache_slots is a multiple of
 * 16. max_len sizes the launch: longer sequences are covered by striding, 0
 * gathers nothing. Neither the rows of `out` nor the entries of `pages` are
 * known to fe_kv8_gather: rows row_offset[b] .. + length of sequence b have to
 * lie in `out`, and kv[batch] page ids in `pages`. fe_kv8_gather_within is told
 * both, and skips a sequence that reaches past either (FE_DEVERR_PAGE_RANGE). */
int fe_kv8_gather(const uint8_t* codes, const uint8_t* exps, void* out, const int32_t* kv,
                  const int32_t* pages, const int32_t* last, const int32_t* row_offset, int batch,
                  int max_len, int page, int hkv, int dim, int dtype, int64_t cache_slots,
                  void* stream);
int fe_kv8_gather_within(const uint8_t* codes, const uint8_t* exps, void* out, int64_t out_rows,
                         const int32_t* kv, const int32_t* pages, int num_pages,
                         const int32_t* last, const int32_t* row_offset, int batch, int max_len,
                         int page, int hkv, int dim, int dtype, int64_t cache_slots,
                         void* stream);

/* fe_kv_copy_blocks for 8-bit pools: token rows [0, ntok[c]) of page src[c]
 * onto page dst[c], and the scales of the blocks they lie in, in every layer's
 * K and V pool (HOST arrays of num_layers device pointers). Works on the lists
 * of fe_kv_fork_copies. */
int fe_kv8_copy_blocks(void* const* k_codes, void* const* v_codes, void* const* k_exps,
                       void* const* v_exps, int num_layers, const int32_t* src,
                       const int32_t* dst, const int32_t* ntok, int num_copies, int page, int hkv,
                       int dim, int num_pages_total, void* stream);

/* Attention over 8-bit pools. A plan of fe_kv8_plan_create is prepared by the
 * same calls as any other (fe_attn_plan_prepare, _prepare_device,
 * fe_step_prepare_device), serves fe_kv8_attn_run only, and is destroyed by
 * fe_attn_plan_destroy; dtype is that of q and out. The host's prepare cuts
 * the lists of both kernels across CTAs by keys and by their measured costs.
 * The device's prepares cut the decode list alike (the same bits), and deal the
 * items of more packed rows whole: few long blocks take longer by them (one of
 * 32 rows over 8192 keys with 4 KV heads 88 us, 19 by the host's lists, 28 by
 * those with graph = 1).
 * fe_kv8_attn_run is fe_attn_run over the values of the codes: the same masks
 * (every query row sees at least one key: a prepared sequence has no fewer
 * keys than query rows), scale 1/sqrt(dim), fp32 softmax and accumulation,
 * output rounded to nearest even. Queries of sequences of up to 16 packed rows
 * (rows x hq / hkv) enter the product as they are (f16, and bf16 down to 2^-29
 * of the row's largest element); with more packed rows in two (bf16) or three
 * (f16) e4m3 parts, which hold an element exactly down to 2^-9 (bf16) or 2^-6
 * (f16) of the row's largest, and smaller ones to 2^-17.8 of the largest.
 * Softmax weights enter the second product as f16, fewer bits than the about 16
 * of fe_attn_run: 11 down to 2^-29 (up to 16 packed rows) or 2^-21 (more) of
 * the row's largest weight times V scale, fewer below, none under 2^-40 or
 * 2^-32; their sum is over the unrounded weights.
 * A query row that holds an infinity or NaN gives NaN. NaN in a key reaches
 * the rows that see it. NaN in a value reaches its dim of the rows that see it
 * and may reach that dim of the sequence's rows it is masked from (weight 0
 * times NaN, as in fe_attn_run); nothing past a sequence's end reaches any
 * row. Exponent arrays are aligned to gcd(hkv, 8) bytes (2 at most for dim
 * 256), all other buffers to 16. */
int fe_kv8_plan_create(int hq, int hkv, int dim, int page, int max_batch, int max_pages, int dtype,
                       int num_blocks, fe_attn_plan** plan_out);
int fe_kv8_attn_run(fe_attn_plan* plan, const void* q, const uint8_t* k_codes,
                    const uint8_t* v_codes, const uint8_t* k_exp, const uint8_t* v_exp, void* out,
                    int causal, void* stream);

/* ------------------------------------------------------------------------
 * Attention for long shared prompts (no reference counterpart: the reference
 * reads every sequence's pages by itself, src/flashinfer_attention.cu:35-44).
 * Two kinds of plans over the 16-bit pools, of one handle type; head_dim, heads,
 * pages and capacities as for fe_attn_plan_create, metadata (HOST) and `graph` as
 * for fe_attn_plan_prepare. Prepare uploads to fixed buffers with one async copy
 * on `stream`: a graph that captured a run replays for later prepares of the same
 * batch and rows. A plan has one workspace (256 MiB of partial records; a scored
 * plan's steps of many rows may get a larger one of their own): its runs must not
 * overlap on the GPU. Scale 1/sqrt(dim), fp32 softmax and accumulation, softmax
 * weights of about 16 bits in the second product (in f16, whose numbers end at
 * 2^-24, to 2^-25 of a row's largest weight), output rounded to nearest even, as
 * fe_attn_run.
 * ------------------------------------------------------------------------ */
typedef struct fe_long_plan fe_long_plan;
int fe_long_plan_destroy(fe_long_plan* plan);

/* Shared prefixes. Sequences group_off[g] .. group_off[g+1]-1 (HOST, runs of
 * consecutive sequences that cover the batch) begin with the same shared[g]
 * pages: prepare checks that they do (FE_ERR_INVALID_ARGUMENT). The result is
 * fe_attn_run's over the full lists (causal as there); K and V of the prefix
 * are read once for the rows of the whole group. groups = 0: nothing is
 * shared. A prefix is taken as far as it is whole pages before every member's
 * query rows, and not at all where sharing it saves too little (a single
 * member, a short prefix, members whose query rows fill the row kernel's tiles by
 * themselves). */
int fe_shared_plan_create(int hq, int hkv, int dim, int page, int max_batch, int max_pages,
                          int dtype, int num_blocks, fe_long_plan** plan_out);
int fe_shared_plan_prepare(fe_long_plan* plan, const int32_t* qo, const int32_t* kv,
                           const int32_t* pages, const int32_t* last, const int32_t* group_off,
                           const int32_t* shared, int groups, int batch, int rows, int graph,
                           void* stream);
int fe_shared_attn_run(fe_long_plan* plan, const void* q, const void* k_pool, const void* v_pool,
                       void* out, int causal, void* stream);
/* The groups of a batch from its page lists (HOST memory only, needs no GPU):
 * neighbours whose first min_pages pages or more are the same. Of all ways to cut
 * the batch into such groups the one that saves the most is taken, the sum of
 * (members - 1) x pages in common: a sequence that has little in common with its
 * neighbours stays out of their groups. kv [batch+1] has to begin with 0 and not to
 * decrease (FE_ERR_INVALID_ARGUMENT), and pages to hold kv[batch] entries.
 * group_off [batch+1] and shared [batch] receive the *num_groups groups. */
int fe_kv_shared_prefixes(const int32_t* kv, const int32_t* pages, int batch, int min_pages,
                          int32_t* group_off, int32_t* shared, int* num_groups);

/* Scored attention: causal attention as fe_attn_run's, and for every key t that
 * a sequence's query rows see, scores[h, slot(t)] (fp32 [hkv, cache_slots], on
 * the device) grows by the softmax weights that KV head h's query heads gave it,
 * summed in fp32 in a fixed order. The last fresh[b] keys of sequence b (HOST,
 * NULL: as many as it has query rows, those that this step appended) have no
 * score yet: theirs is set instead. A page may be listed once only
 * (FE_ERR_INVALID_ARGUMENT: scores of a shared page would be added to by two
 * CTAs). max_keys, at creation: the most query rows x keys of a step, each
 * sequence's keys rounded up to a multiple of 16, summed over the sequences; the
 * plan holds hkv * (hq / hkv rounded up to even) fp32 raw scores for each. A step
 * within it is served, whatever its rows: the first with more than 2^26 / (hq *
 * (dim + 2)) of them, or such a graph prepare, allocates a larger workspace
 * (records of 2^31 floats are the most). A step beyond it fails with
 * FE_ERR_CAPACITY. A query row with an infinity or NaN
 * gives its keys NaN. */
int fe_scored_plan_create(int hq, int hkv, int dim, int page, int max_batch, int max_pages,
                          int dtype, int num_blocks, int64_t max_keys, fe_long_plan** plan_out);
int fe_scored_plan_prepare(fe_long_plan* plan, const int32_t* qo, const int32_t* kv,
                           const int32_t* pages, const int32_t* last, const int32_t* fresh,
                           int batch, int rows, int graph, void* stream);
int fe_scored_attn_run(fe_long_plan* plan, const void* q, const void* k_pool, const void* v_pool,
                       float* scores, void* out, void* stream);

/* Host-side numbers of the last prepare. */
typedef struct fe_long_plan_info {
  int rows, shared_groups;   /* groups whose prefix is read once */
  int row_ctas, decode_ctas; /* CTAs of the two kernels (causal) */
  int64_t shared_tiles;      /* 16-key tiles (x KV heads) that sharing saves reading */
  int64_t partial_floats, weight_floats;
} fe_long_plan_info;
int fe_long_plan_get_info(const fe_long_plan* plan, fe_long_plan_info* info);

/* ------------------------------------------------------------------------
 * Device-side step preparation (no reference counterpart: replaces the host
 * loops of CudaModel::prepare, src/cuda_model.cpp:131-142, and the host
 * planning plus pageable H2D copies of prepare_plan,
 * src/flashinfer_attention.cu:29-34). Every array argument is DEVICE memory
 * and nothing is read back on the host, so both calls can be captured in a
 * CUDA graph together with the append and attention: a decode or verify
 * step then replays with no host work at all.
 *
 * Both leave the plan in graph mode (the attention kernels launch at full
 * width; batch and rows must stay those of the first graph prepare). The
 * work lists are built on the device by one kernel on `stream`: the decode
 * list is the host planner's exact-cut list item for item (identical split
 * points, bit-identical outputs); prefill/verify units (never split) are
 * dealt to the CTAs by cost, longest first, in snake order (at most 8192 such
 * units). Invalid metadata or exceeded capacity does not fail the call (it
 * is not seen on the host): the plan is emptied, attention writes nothing,
 * and FE_DEVERR_PLAN is raised (fe_device_errors).
 * ------------------------------------------------------------------------ */
/* The caller's device metadata, in the layout of fe_attn_plan_prepare. */
int fe_attn_plan_prepare_device(fe_attn_plan* plan, const int32_t* qo, const int32_t* kv,
                                const int32_t* pages, const int32_t* last, int batch, int rows,
                                void* stream);
/* The slot mapping too (CudaModel::prepare): sequence b (b < batch) writes
 * rows_per_seq tokens at positions starts[b] .. starts[b]+rows_per_seq-1
 * through its block-table row block_tables[b*table_stride ...] (int32 page
 * ids, at least ceil((starts[b]+rows_per_seq)/page) of them). starts[b] < 0
 * marks a padding entry of a graph bucket: slot -1 (the append skips it),
 * position j, the dummy page num_blocks, last = rows_per_seq (as
 * src/cuda_model.cpp:138). Writes slots[batch*rows_per_seq] and
 * positions[batch*rows_per_seq] (int64, device) for fe_kv_append / fe_rope*,
 * and plans attention over qo[b] = b*rows_per_seq, the first
 * ceil(length/page) pages of each row, last = (length-1) % page + 1. */
int fe_step_prepare_device(fe_attn_plan* plan, const int32_t* block_tables, int table_stride,
                           const int32_t* starts, int batch, int rows_per_seq, int64_t* slots,
                           int64_t* positions, void* stream);

/* Introspection of the last prepare (host-side numbers, no sync; after a
 * device-side prepare the item counts read -1). */
typedef struct fe_attn_plan_info {
  int batch, rows;
  int decode_items, prefill_items; /* work items queued for the two kernels */
  int split_sequences;             /* (sequence, kv head) pairs split over > 1 item */
  int chunk_tiles;                 /* key tiles (16 tokens) per decode item */
  int grid_ctas;                   /* persistent CTAs launched by fe_attn_run */
  int64_t kv_tokens;               /* sum of sequence lengths */
} fe_attn_plan_info;
int fe_attn_plan_get_info(const fe_attn_plan* plan, fe_attn_plan_info* info);

/* ------------------------------------------------------------------------
 * Test hooks (no reference counterpart): exercise the host planner without
 * a GPU.
 * ------------------------------------------------------------------------ */
/* A plan with no device state; fe_attn_plan_prepare() then only validates
 * and builds the work list, for `grid_cap` persistent CTAs. */
int fe_attn_plan_create_host(int hq, int hkv, int dim, int page, int max_batch, int max_pages,
                             int dtype, int num_blocks, int grid_cap, fe_attn_plan** plan_out);
int fe_kv8_plan_create_host(int hq, int hkv, int dim, int page, int max_batch, int max_pages,
                            int dtype, int num_blocks, int grid_cap, fe_attn_plan** plan_out);
int fe_long_plan_create_host(int hq, int hkv, int dim, int page, int max_batch, int max_pages,
                             int dtype, int num_blocks, int scored, int64_t max_keys, int grid_cap,
                             fe_long_plan** plan_out);
int fe_long_plan_debug_meta(const fe_long_plan* plan, void* dst, int64_t cap, int64_t* bytes);
/* Copy the packed work-list metadata of the last prepare into `dst` (at most
 * `cap` bytes); *bytes receives its full size. Layout: fe_attn_plan.h. */
int fe_attn_plan_debug_meta(const fe_attn_plan* plan, void* dst, int64_t cap, int64_t* bytes);
/* Copy the plan's DEVICE metadata (what the kernels read; at most `cap`
 * bytes) into host memory `dst`; synchronises `stream`. */
int fe_attn_plan_debug_device_meta(const fe_attn_plan* plan, void* dst, int64_t cap, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FE_KV_H_ */
