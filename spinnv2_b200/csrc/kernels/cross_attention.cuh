// Arguments shared by the cross attention kernels: cross_attention.cu (CUDA
// cores, any type and alignment, and the choice between the kernels),
// cross_attention_tc.cu (tcgen05, 16-bit types, many rows),
// cross_attention_step.cu (mma.sync, 16-bit types, few rows) and
// cross_attention_f32.cu (mma.sync, fp32 by three TF32 passes).
#pragma once

#include "tcgen05.cuh"
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
  FastDiv group_div;
};

// Element offset of a row (query * group + head in the group) of q or out, from the
// entry's start.
__device__ __forceinline__ int64_t row_offset(const AttnArgs &p, const int64_t (&st)[3], int hk, int row) {
  const uint32_t qi = p.group_div.div(uint32_t(row));
  return int64_t(qi) * st[1] + (int64_t(hk) * p.group + (uint32_t(row) - qi * uint32_t(p.group))) * st[2];
}

__device__ __forceinline__ int entry_keys(const AttnArgs &p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.keys) : p.keys;
}

// The end of a long mask: one past its last key that counts, searched from behind, 16
// keys a thread at a time, by all of a block's threads.  Its own function, so that its
// instructions lie outside the path of calls that do not search (12 heads x 77 rows
// over 196 masked keys: 8.5 us inlined, 8.2 so).
template <int THREADS>
__device__ __noinline__ int mask_end(const uint8_t *mask, int keys, int tid) {
  __shared__ int s_last;
  if (tid == 0) s_last = 0;
  constexpr int SPAN = THREADS * 16;
  int last = 0;
  for (int end = keys; end > 0; end -= SPAN) {
    bool in[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int j = end - SPAN + k * THREADS + tid;
      in[k] = j >= 0 && mask[j] != 0;
    }
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if (in[k]) last = end - SPAN + k * THREADS + tid + 1;
    if (__syncthreads_or(last)) break;
  }
  last = __reduce_max_sync(0xffffffffu, last);
  if ((tid & 31) == 0 && last) atomicMax(&s_last, last);
  __syncthreads();
  return s_last;
}

// The keys of entry b that have to be read.  Images padded to one grid end in keys that
// do not count (bf16, 4 x 200 rows x 16/4 heads, grids within 60 x 60: 37.8 us reading
// every key, 18.5 so; 8 x 2 rows x 16/8 heads within 43 x 87: 38.1 and 29.8).  Masks of
// under 512 keys are a few steps at most and are not searched.
template <int THREADS>
__device__ __forceinline__ int counted_keys(const AttnArgs &p, int b, int tid) {
  const int keys = entry_keys(p, b);
  if (!p.key_mask || keys < 512) return keys;
  return mask_end<THREADS>(p.key_mask + b * p.mask_stride, keys, tid);
}

// Tensor map of keys or values as {width, key, head, entry}, 128-byte swizzle,
// boxes of 64 columns x `box_keys` keys.
struct KvMap {
  CUtensorMap map;
  int heads_step, batch_step;  // 0: one head or entry for all (stride 0)
};

inline bool encode_kv(KvMap *m, const AttnArgs &a, const void *base, const int64_t (&st)[3], int box_keys) {
  m->heads_step = st[2] != 0 && a.kv_heads > 1;
  m->batch_step = st[0] != 0 && a.batch > 1;
  const cuuint64_t dims[4] = {cuuint64_t(a.width), cuuint64_t(a.keys), cuuint64_t(m->heads_step ? a.kv_heads : 1),
                              cuuint64_t(m->batch_step ? a.batch : 1)};
  const cuuint64_t any = (cuuint64_t(a.width) * 2 + 15) / 16 * 16;
  const cuuint64_t strides[3] = {a.keys > 1 ? cuuint64_t(st[1]) * 2 : any, m->heads_step ? cuuint64_t(st[2]) * 2 : any,
                                 m->batch_step ? cuuint64_t(st[0]) * 2 : any};
  const cuuint32_t box[4] = {64, cuuint32_t(box_keys), 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return tc::encode_fn()(&m->map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void *>(base), dims, strides, box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether the tensor-core kernels take these arguments: 16-bit elements, width
// a multiple of 8 up to 128, rows on 16-byte boundaries, a positive scale.
bool cross_tc_serves(const AttnArgs &a, int32_t dtype);
int cross_tc(const AttnArgs &a, int32_t dtype, cudaStream_t s);
int cross_step(const AttnArgs &a, int32_t dtype, cudaStream_t s);  // a.rows <= 32
int cross_f32(const AttnArgs &a, cudaStream_t s);  // fp32, a.width <= 128

}  // namespace spkv2
