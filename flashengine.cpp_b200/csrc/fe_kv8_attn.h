// Launch interface of the attention kernels over the 8-bit KV cache, shared by
// the plan (fe_attn.cu) and the two kernels (fe_kv8_decode.cu, fe_kv8_rows.cu),
// and the row kernel's conversion of a query row to e4m3 parts.
#pragma once

#include "fe_attn_common.cuh"
#include "fe_kv8_common.cuh"

namespace fe {

template <typename T>
struct Kv8Args {
  AttnArgs<T> a;  // as for the 16-bit kernels
  const uint8_t* k_exp;
  const uint8_t* v_exp;
  int hkv;
};

int kv8_decode_launch(int dtype, int dim, int heads, const CUtensorMap& kmap,
                      const CUtensorMap& vmap, const void* args, int grid, cudaStream_t stream);
// Merge the split units of a work list: `units` of them (an upper bound under a
// fixed launch geometry) of at most `rows` record rows; `pieces`: records of the
// most split unit, or an estimate (it sizes the grid only); at most about
// `max_blocks` blocks.
int kv8_merge_launch(int dtype, int dim, int list, const void* args, int units, int rows,
                     int pieces, int max_blocks, cudaStream_t stream, bool pdl);
int kv8_rows_launch(int dtype, int dim, const CUtensorMap& kmap, const CUtensorMap& vmap,
                    const void* args, int grid, cudaStream_t stream);

// Scale exponent (biased) of a query row with largest finite magnitude amax:
// the row is scaled into (224, 448], so its parts use e4m3's whole range. At
// least 2^-60: products of rows smaller than that stay normal numbers.
__device__ __forceinline__ int kv8_query_exp(float amax) {
  return min(max(((__float_as_int(amax) + 0x1fffff) >> 23) - 8, 67), 247);
}

// Four query elements times `up` as e4m3 codes, part by part: each holds the
// rounding of what the parts before it leave (exact in fp32).
template <typename T, int kParts>
__device__ __forceinline__ void kv8_split_query(uint32_t v0, uint32_t v1, float up,
                                                uint32_t (&part)[kParts]) {
  const float2 up2 = make_float2(up, up);
  float2 x = mul2(unpack2<T>(v0), up2), y = mul2(unpack2<T>(v1), up2);
#pragma unroll
  for (int k = 0; k < kParts; ++k) {
    const uint32_t c0 = e4m3x2(x.x, x.y), c1 = e4m3x2(y.x, y.y);
    part[k] = c0 | c1 << 16;
    if (k + 1 < kParts) {
      x = sub2(x, unpack2<__half>(e4m3x2_to_h2(c0)));
      y = sub2(y, unpack2<__half>(e4m3x2_to_h2(c1)));
    }
  }
}

}  // namespace fe
