// int8 x int8 product with a scale for each token and each channel:
//
//   y[i, j] = act(float(sum_k a[i, k] w[j, k]) * a_scale[i] * w_scale[j] + bias[j])
//
// The sum is exact in int32 (|a|, |w| <= 128 and k <= 131071).
#include "transformer.cuh"

namespace spkv2 {

namespace {

using namespace xf;

constexpr int64_t kMaxK = 131071;  // 128 * 128 * k stays below 2^31

struct LinearArgs {
  const int8_t *a, *w;
  const float *a_scale, *w_scale, *bias;
  void *y;
  int64_t m, n, a_stride, w_stride, y_stride;
  int k, act;
};

__device__ __forceinline__ float linear_value(int acc, float sa, float sw, float bias, int act) {
  return apply_act(fmaf(float(acc) * sa, sw, bias), act);
}

// CUDA cores (dp4a), any alignment: 64 x 64 tile, 64 of k a step, a 4 x 4
// patch for each of 256 threads.
constexpr int kST = 64, kSK = 64, kSPitch = kSK + 4;

template <class T>
__global__ void __launch_bounds__(256) linear_simt_kernel(LinearArgs p) {
  __shared__ __align__(16) int8_t sa[kST][kSPitch];
  __shared__ __align__(16) int8_t sw[kST][kSPitch];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int64_t n_tiles = ceil_div(p.n, kST);
  const int64_t m0 = int64_t(blockIdx.x) / n_tiles * kST, n0 = int64_t(blockIdx.x) % n_tiles * kST;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < p.k; k0 += kSK) {
#pragma unroll
    for (int i = 0; i < kST * kSK / 256; ++i) {
      const int e = tid + i * 256, r = e / kSK, c = e % kSK;
      const bool kin = k0 + c < p.k;
      sa[r][c] = kin && m0 + r < p.m ? p.a[(m0 + r) * p.a_stride + k0 + c] : int8_t(0);
      sw[r][c] = kin && n0 + r < p.n ? p.w[(n0 + r) * p.w_stride + k0 + c] : int8_t(0);
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kSK; c += 4) {
      int av[4], wv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        av[i] = *reinterpret_cast<const int *>(&sa[ty * 4 + i][c]);
        wv[i] = *reinterpret_cast<const int *>(&sw[tx + 16 * i][c]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(av[i], wv[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty * 4 + i;
    if (m >= p.m) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx + 16 * j;
      if (n >= p.n) continue;
      static_cast<T *>(p.y)[m * p.y_stride + n] = from_f32<T>(
          linear_value(acc[i][j], p.a_scale[m], p.w_scale[n], p.bias ? p.bias[n] : 0.0f, p.act));
    }
  }
}

}  // namespace

}  // namespace spkv2

using namespace spkv2;
using namespace spkv2::xf;

extern "C" int spkv2_cuda_linear_i8(const Spkv2LinearI8 *a, void *stream) {
  if (!a || a->m < 0 || a->n < 0 || a->k < 0) return -1;
  if (a->m == 0 || a->n == 0) return 0;
  if (!a->y || !a->a_scale || !a->w_scale || (a->k > 0 && (!a->a || !a->w))) return -1;
  if (a->a_stride < 0 || a->w_stride < 0 || overlaps(a->y_stride, a->m, a->n)) return -1;
  if (a->activation < SPKV2_CUDA_ACT_NONE || a->activation > SPKV2_CUDA_ACT_SILU) return -1;
  if (!elem_bytes(a->dtype) || a->k > kMaxK || a->m > INT32_MAX || a->n > INT32_MAX) return SPKV2_ERR_UNSUPPORTED;
  const LinearArgs p = {a->a, a->w, a->a_scale, a->w_scale, a->bias, a->y, a->m, a->n, a->a_stride, a->w_stride,
                        a->y_stride, int(a->k), a->activation};
  const int64_t tiles = ceil_div(a->m, kST) * ceil_div(a->n, kST);
  if (tiles > INT32_MAX) return SPKV2_ERR_UNSUPPORTED;
  return by_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    linear_simt_kernel<T><<<unsigned(tiles), 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return cuda_status(cudaGetLastError());
  });
}
