// Arguments shared by the cross attention kernels: cross_attention.cu (CUDA
// cores, any type and alignment, and the choice between the kernels) and
// cross_attention_tc.cu (tcgen05, 16-bit types, many rows).
#pragma once

#include "transformer.cuh"

namespace spkv2 {

struct AttnArgs {
  const void *q, *k, *v;
  void *out;
  const int32_t *lengths;
  const uint8_t *key_mask;
  int64_t qs[3], ks[3], vs[3], os[3];  // batch, token, head
  int64_t mask_stride;
  int batch, queries, keys, kv_heads, group, width;
  int rows;        // queries * group
  int row_tiles;   // per (batch, key head)
  float scale_log2;
};

__device__ __forceinline__ int entry_keys(const AttnArgs &p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.keys) : p.keys;
}

// Whether the tensor-core kernel takes these arguments: 16-bit elements, width
// a multiple of 8 up to 128, rows on 16-byte boundaries, a positive scale.
bool cross_tc_serves(const AttnArgs &a, int32_t dtype);
int cross_tc(const AttnArgs &a, int32_t dtype, cudaStream_t s);

}  // namespace spkv2
