// Tensor maps of the attention kernels over 16-bit pools and queries
// (fe_attn.cu).
#pragma once

#include "fe_common.cuh"

namespace fe {

// K or V pool for the tcgen05 row kernel: boxes of a 16-token piece of a head.
int encode_tc_map(CUtensorMap* map, const void* pool, int dtype, int hkv, int dim,
                  int64_t cache_slots);
// Queries of the row kernel: boxes of 128 packed rows x 64 dims.
int encode_q_map(CUtensorMap* map, const void* q, int dtype, int hq, int dim, int rows, int G);
// K or V pool for the decode kernel, one head's 64 dims or all heads a box.
int encode_pool_map(CUtensorMap* map, const void* pool, int dtype, int hkv, int dim,
                    int64_t cache_slots);
int encode_decode_map(CUtensorMap* map, const void* pool, int dtype, int hkv, int dim, int heads,
                      int64_t cache_slots);

}  // namespace fe
