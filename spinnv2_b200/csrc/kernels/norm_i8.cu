// Root-mean-square norm with the residual's addition and int8 output, the
// int8 codes of a tensor's rows, and the values that codes stand for.
//
//   s = x + r,  y = s w / sqrt(mean(s^2) + eps),  scale = max|y| / 127,
//   code = rne(y / scale)
//
// The factor 1 / sqrt(..) is common to a row, so it cancels in the codes:
//   code = rne(s w * (127 / max|s w|)),  scale = max|s w| / sqrt(..) / 127,
// and both reductions (sum of s^2, max |s w|) run in one pass over the row.
// Quantising without the norm is the same with r = 0, w = 1 and no factor.
//
// |s w| is compared by its bits: as an unsigned number, without the sign, a
// NaN is above infinity and infinity above every finite value, so the
// maximum itself says whether the row is finite.
#include "transformer.cuh"

namespace spkv2 {

namespace {

using namespace xf;

constexpr int kThreads = 256;
constexpr int64_t kMaxWidth = int64_t(1) << 24;

struct RowArgs {
  const void *x, *residual, *weight;
  void *sum;
  int8_t *codes;
  float *scale;
  int64_t rows, width;
  int64_t x_stride, residual_stride, sum_stride, codes_stride;
  float eps;
};

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The factor that takes |s w| to codes.  127 / amax overflows where amax is
// below 2^-121 or so; values that small are scaled up by 2^64, exactly, first.
struct CodeScale {
  float pre, inv;
};
__device__ __forceinline__ CodeScale code_scale(float amax) {
  CodeScale c;
  c.pre = amax < 1e-30f ? 18446744073709551616.0f : 1.0f;
  c.inv = amax > 0.0f ? 127.0f / (amax * c.pre) : 0.0f;
  return c;
}
__device__ __forceinline__ int8_t code_of(float v, CodeScale c) { return sat_rne_i8(v * c.pre * c.inv, -127); }

// One block per row; the row is read twice, the second time from L2.
template <class T, bool NORM>
__global__ void __launch_bounds__(kThreads) row_codes_kernel(RowArgs p) {
  __shared__ float s_sum[kThreads / 32];
  __shared__ uint32_t s_max[kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x;
  const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
  const T *r = NORM && p.residual ? static_cast<const T *>(p.residual) + row * p.residual_stride : nullptr;
  const T *w = static_cast<const T *>(p.weight);
  float ss = 0.0f;
  uint32_t mx = 0;
  for (int64_t i = tid; i < p.width; i += kThreads) {
    float s = to_f32(x[i]);
    if (r) s += to_f32(r[i]);
    ss = fmaf(s, s, ss);
    mx = max(mx, abs_bits(NORM ? s * to_f32(w[i]) : s));
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    ss += __shfl_xor_sync(0xffffffffu, ss, o);
    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  if (lane == 0) {
    s_sum[warp] = ss;
    s_max[warp] = mx;
  }
  __syncthreads();
  ss = 0.0f;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) {
    ss += s_sum[i];
    mx = max(mx, s_max[i]);
  }
  const bool finite = mx < 0x7f800000u;
  const float amax = __uint_as_float(mx);
  const CodeScale c = code_scale(finite ? amax : 0.0f);
  if (tid == 0) {
    const float f = NORM && amax > 0.0f ? 1.0f / sqrtf(ss / float(p.width) + p.eps) : 1.0f;
    p.scale[row] = finite ? amax * f / 127.0f : __uint_as_float(0x7fc00000u);
  }
  T *sum = NORM && p.sum ? static_cast<T *>(p.sum) + row * p.sum_stride : nullptr;
  int8_t *codes = p.codes + row * p.codes_stride;
  for (int64_t i = tid; i < p.width; i += kThreads) {
    float s = to_f32(x[i]);
    if (r) s += to_f32(r[i]);
    codes[i] = finite ? code_of(NORM ? s * to_f32(w[i]) : s, c) : int8_t(0);
    if (sum) sum[i] = from_f32<T>(s);
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads)
    row_values_kernel(const int8_t *__restrict__ codes, const float *__restrict__ scale, T *__restrict__ y, int64_t width,
                      int64_t codes_stride, int64_t y_stride) {
  const int64_t row = blockIdx.x;
  const float s = scale[row];
  for (int64_t i = threadIdx.x; i < width; i += kThreads)
    y[row * y_stride + i] = from_f32<T>(float(codes[row * codes_stride + i]) * s);
}

template <bool NORM>
int launch_rows(const RowArgs &a, int32_t dtype, cudaStream_t s) {
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    row_codes_kernel<T, NORM><<<unsigned(a.rows), kThreads, 0, s>>>(a);
    return cuda_status(cudaGetLastError());
  });
}

bool bad_extent(int64_t rows, int64_t width) { return rows < 0 || rows > INT32_MAX || width < 1 || width > kMaxWidth; }

}  // namespace

}  // namespace spkv2

using namespace spkv2;
using namespace spkv2::xf;

extern "C" int spkv2_cuda_rms_norm_i8(const Spkv2RmsNormI8 *a, void *stream) {
  if (!a || bad_extent(a->rows, a->width)) return -1;
  if (a->rows == 0) return 0;
  if (!a->x || !a->weight || !a->codes || !a->scale || !(a->eps >= 0.0f)) return -1;
  if (a->x_stride < 0 || (a->residual && a->residual_stride < 0) || overlaps(a->codes_stride, a->rows, a->width) ||
      (a->sum && overlaps(a->sum_stride, a->rows, a->width)))
    return -1;
  if (!elem_bytes(a->dtype)) return SPKV2_ERR_UNSUPPORTED;
  RowArgs p = {a->x,     a->residual, a->weight,   a->sum,      a->codes,           a->scale,      a->rows,
               a->width, a->x_stride, a->residual_stride, a->sum_stride, a->codes_stride, a->eps};
  return launch_rows<true>(p, a->dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int spkv2_cuda_quantize_rows_i8(const Spkv2QuantizeRowsI8 *a, void *stream) {
  if (!a || bad_extent(a->rows, a->width)) return -1;
  if (a->rows == 0) return 0;
  if (!a->x || !a->codes || !a->scale || a->x_stride < 0 || overlaps(a->codes_stride, a->rows, a->width)) return -1;
  if (!elem_bytes(a->dtype)) return SPKV2_ERR_UNSUPPORTED;
  RowArgs p = {a->x, nullptr, nullptr, nullptr, a->codes, a->scale, a->rows, a->width, a->x_stride, 0, 0,
               a->codes_stride, 0.0f};
  return launch_rows<false>(p, a->dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int spkv2_cuda_dequantize_rows_i8(const Spkv2DequantizeRowsI8 *a, void *stream) {
  if (!a || bad_extent(a->rows, a->width)) return -1;
  if (a->rows == 0) return 0;
  if (!a->codes || !a->scale || !a->y || a->codes_stride < 0 || overlaps(a->y_stride, a->rows, a->width)) return -1;
  return by_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    row_values_kernel<T><<<unsigned(a->rows), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        a->codes, a->scale, static_cast<T *>(a->y), a->width, a->codes_stride, a->y_stride);
    return cuda_status(cudaGetLastError());
  });
}
