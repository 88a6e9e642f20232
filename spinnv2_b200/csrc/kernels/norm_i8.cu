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

// N elements in one access.
template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// A row's scale (its first thread writes it) and the factor of its codes.
template <bool NORM>
__device__ __forceinline__ CodeScale finish_row(const RowArgs &p, int64_t row, float ss, uint32_t mx, bool &finite, bool writes) {
  finite = mx < 0x7f800000u;
  const float amax = __uint_as_float(mx);
  if (writes) {
    const float f = NORM && amax > 0.0f ? 1.0f / sqrtf(ss / float(p.width) + p.eps) : 1.0f;
    p.scale[row] = finite ? amax * f / 127.0f : __uint_as_float(0x7fc00000u);
  }
  return code_scale(finite ? amax : 0.0f);
}

// Bound by memory: every element is read once, kept in registers (EPT a thread)
// through the row's two reductions, and its code written once.  A thread owns
// units of 16 bytes of x (U elements), t, t + tpr, ..: which element is added
// where does not depend on alignment, so neither do the bits of the result.
//
// STAGED: rows that do not start on 16-byte boundaries, or end inside a unit.
// They are read element by element in order, a warp's 32 side by side, and pass
// through shared memory (as fp32 sums) to the threads that own them; reading the
// units themselves element by element would touch each line eight times.
//
// The residual's sum is written by the thread that read both parts, so it may
// take their place.  tpr (32 .. 1024, a power of two) threads a row; rows of less
// than 128 threads share a block.
template <class T, bool NORM, int EPT, bool STAGED>
__global__ void __launch_bounds__(1024) row_codes_kernel(RowArgs p, int tpr, bool vec_codes) {
  constexpr int U = 16 / sizeof(T), N = EPT / U;
  extern __shared__ __align__(16) float staged[];
  __shared__ float s_sum[32];
  __shared__ uint32_t s_max[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = threadIdx.x & (tpr - 1), wpr = tpr >> 5;
  const int64_t row = int64_t(blockIdx.x) * (blockDim.x / tpr) + threadIdx.x / tpr;
  const bool real = row < p.rows;
  const int width = int(p.width);
  const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
  const T *r = static_cast<const T *>(p.residual) + row * p.residual_stride;
  const T *w = static_cast<const T *>(p.weight);
  T *sum = static_cast<T *>(p.sum) + row * p.sum_stride;
  float v[N][U];
  float ss = 0.0f;
  uint32_t mx = 0;
  if (STAGED) {
    float *mine = staged + threadIdx.x / tpr * ((width + U - 1) / U * U);
    constexpr int B = 8;  // loads in flight
    for (int c0 = t; real && c0 < width; c0 += B * tpr) {
      float s[B];
#pragma unroll
      for (int k = 0; k < B; ++k) s[k] = c0 + k * tpr < width ? to_f32(x[c0 + k * tpr]) : 0.0f;
      if (NORM && p.residual) {
#pragma unroll
        for (int k = 0; k < B; ++k) s[k] += c0 + k * tpr < width ? to_f32(r[c0 + k * tpr]) : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < B; ++k) {
        const int c = c0 + k * tpr;
        if (c >= width) break;
        if (NORM && p.sum) sum[c] = from_f32<T>(s[k]);
        mine[c] = s[k];
      }
    }
    if (real && t < (width + U - 1) / U * U - width) mine[width + t] = 0.0f;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (t + i * tpr) * U;
#pragma unroll
      for (int e = 0; e < U; e += 4) {
        const float4 f = real && c < width ? *reinterpret_cast<const float4 *>(mine + c + e) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        v[i][e] = f.x, v[i][e + 1] = f.y, v[i][e + 2] = f.z, v[i][e + 3] = f.w;
      }
    }
  } else {
    Vec<T, U> xv[N], rv[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (t + i * tpr) * U;
      if (real && c < width) {
        xv[i] = *reinterpret_cast<const Vec<T, U> *>(x + c);
        if (NORM && p.residual) rv[i] = *reinterpret_cast<const Vec<T, U> *>(r + c);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (t + i * tpr) * U;
      const bool in = real && c < width;
      Vec<T, U> sv;
#pragma unroll
      for (int e = 0; e < U; ++e) {
        float s = in ? to_f32(xv[i].v[e]) : 0.0f;
        if (NORM && p.residual && in) s += to_f32(rv[i].v[e]);
        if (NORM) sv.v[e] = from_f32<T>(s);
        v[i][e] = s;
      }
      if (NORM && p.sum && in) *reinterpret_cast<Vec<T, U> *>(sum + c) = sv;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (t + i * tpr) * U;
    if (NORM && real && c < width) {
      Vec<T, U> wv;
      if (STAGED) {
#pragma unroll
        for (int e = 0; e < U; ++e) wv.v[e] = c + e < width ? w[c + e] : from_f32<T>(0.0f);
      } else {
        wv = *reinterpret_cast<const Vec<T, U> *>(w + c);
      }
#pragma unroll
      for (int e = 0; e < U; ++e) {
        ss = fmaf(v[i][e], v[i][e], ss);
        v[i][e] *= to_f32(wv.v[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < U; ++e) mx = max(mx, abs_bits(v[i][e]));
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    if (NORM) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  if (wpr > 1) {
    if (lane == 0) {
      s_sum[warp] = ss;
      s_max[warp] = mx;
    }
    __syncthreads();
    const int first = warp & ~(wpr - 1);
    ss = lane < wpr ? s_sum[first + lane] : 0.0f;
    mx = lane < wpr ? s_max[first + lane] : 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      if (NORM) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
  }
  if (!real) return;
  bool finite;
  const CodeScale cs = finish_row<NORM>(p, row, ss, mx, finite, t == 0);
  int8_t *codes = p.codes + row * p.codes_stride;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (t + i * tpr) * U;
    if (c >= width) break;
    Vec<int8_t, U> q;
#pragma unroll
    for (int e = 0; e < U; ++e) q.v[e] = finite ? code_of(v[i][e], cs) : int8_t(0);
    if (!STAGED || (vec_codes && c + U <= width)) {
      *reinterpret_cast<Vec<int8_t, U> *>(codes + c) = q;
    } else {
#pragma unroll
      for (int e = 0; e < U; ++e)
        if (c + e < width) codes[c + e] = q.v[e];
    }
  }
}

// Rows wider than the registers of a block (32 elements a thread): one block a
// row, which is read twice, the second time from L2; the sum is written in the
// second pass, as it may take x's or the residual's place.
template <class T, bool NORM>
__global__ void __launch_bounds__(1024) wide_codes_kernel(RowArgs p) {
  __shared__ float s_sum[32];
  __shared__ uint32_t s_max[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
  const int64_t row = blockIdx.x;
  const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
  const T *r = NORM && p.residual ? static_cast<const T *>(p.residual) + row * p.residual_stride : nullptr;
  const T *w = static_cast<const T *>(p.weight);
  float ss = 0.0f;
  uint32_t mx = 0;
#pragma unroll 4
  for (int64_t i = tid; i < p.width; i += threads) {
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
  ss = s_sum[lane];
  mx = s_max[lane];
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    ss += __shfl_xor_sync(0xffffffffu, ss, o);
    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  bool finite;
  const CodeScale c = finish_row<NORM>(p, row, ss, mx, finite, tid == 0);
  T *sum = NORM && p.sum ? static_cast<T *>(p.sum) + row * p.sum_stride : nullptr;
  int8_t *codes = p.codes + row * p.codes_stride;
#pragma unroll 4
  for (int64_t i = tid; i < p.width; i += threads) {
    float s = to_f32(x[i]);
    if (r) s += to_f32(r[i]);
    codes[i] = finite ? code_of(NORM ? s * to_f32(w[i]) : s, c) : int8_t(0);
    if (sum) sum[i] = from_f32<T>(s);
  }
}

// VW codes a thread; chunks of all rows in one list.
template <class T, int VW>
__global__ void __launch_bounds__(256)
    row_values_kernel(const int8_t *__restrict__ codes, const float *__restrict__ scale, T *__restrict__ y, uint32_t chunks,
                      FastDiv per_row, int64_t codes_stride, int64_t y_stride) {
  for (uint32_t i = blockIdx.x * 256u + threadIdx.x; i < chunks; i += gridDim.x * 256u) {
    const uint32_t row = per_row.div(i), c = (i - row * per_row.d) * VW;
    const float s = __ldg(scale + row);
    const Vec<int8_t, VW> q = *reinterpret_cast<const Vec<int8_t, VW> *>(codes + int64_t(row) * codes_stride + c);
    T *to = y + int64_t(row) * y_stride + c;
    constexpr int S = VW * sizeof(T) > 16 ? 16 / sizeof(T) : VW;  // elements of a store
#pragma unroll
    for (int k = 0; k < VW; k += S) {
      Vec<T, S> o;
#pragma unroll
      for (int e = 0; e < S; ++e) o.v[e] = from_f32<T>(float(q.v[k + e]) * s);
      *reinterpret_cast<Vec<T, S> *>(to + k) = o;
    }
  }
}

template <class T, bool NORM, int EPT, bool STAGED>
int launch_ept(const RowArgs &a, int tpr, bool vec_codes, cudaStream_t s) {
  const int threads = std::max(tpr, 128), rpb = threads / tpr;
  constexpr int U = 16 / sizeof(T);
  const size_t smem = STAGED ? size_t(rpb) * (size_t(a.width) + U - 1) / U * U * 4 : 0;
  if (STAGED)
    if (const int rc = allow_smem<row_codes_kernel<T, NORM, EPT, STAGED>>(32768 * 4)) return rc;
  row_codes_kernel<T, NORM, EPT, STAGED><<<unsigned(ceil_div(a.rows, rpb)), threads, smem, s>>>(a, tpr, vec_codes);
  return cuda_status(cudaGetLastError());
}

template <class T, bool NORM, bool STAGED>
int launch_row(const RowArgs &a, bool vec_codes, cudaStream_t s) {
  // Eight elements a thread for rows of one block's 256 threads, 16 beyond (less
  // synchronisation for the same loads in flight), 32 where 1024 threads need them.
  const int64_t per = a.width <= 2048 ? 8 : a.width <= 16384 ? 16 : 32;
  int tpr = 32;
  while (tpr * per < a.width) tpr *= 2;
  if (per == 8) return launch_ept<T, NORM, 8, STAGED>(a, tpr, vec_codes, s);
  return per == 16 ? launch_ept<T, NORM, 16, STAGED>(a, tpr, vec_codes, s) : launch_ept<T, NORM, 32, STAGED>(a, tpr, vec_codes, s);
}

// The most elements (a power of two up to `most`) that rows can be accessed by:
// their starts, `base` and `stride` in elements, are multiples of them, and the
// width holds a whole number.
int vector_width(int most, int64_t width, uintptr_t base, int64_t stride) {
  int vw = most;
  while (vw > 1 && (uintptr_t(width) | base | uintptr_t(stride)) % uintptr_t(vw) != 0) vw /= 2;
  return vw;
}

template <bool NORM>
int launch_rows(const RowArgs &a, int32_t dtype, cudaStream_t s) {
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (a.width > 32768) {
      wide_codes_kernel<T, NORM><<<unsigned(a.rows), 1024, 0, s>>>(a);
      return cuda_status(cudaGetLastError());
    }
    constexpr int U = 16 / sizeof(T);
    auto apart = [&](const void *base, int64_t stride) { return !aligned16(base) || (a.rows > 1 && stride % U != 0); };
    const bool vec_codes = reinterpret_cast<uintptr_t>(a.codes) % U == 0 && (a.rows == 1 || a.codes_stride % U == 0);
    if (!vec_codes || a.width % U != 0 || apart(a.x, a.x_stride) || apart(a.residual, a.residual_stride) ||
        apart(a.sum, a.sum_stride) || !aligned16(a.weight))
      return launch_row<T, NORM, true>(a, vec_codes, s);
    return launch_row<T, NORM, false>(a, vec_codes, s);
  });
}

template <class T, int VW>
int launch_values(const Spkv2DequantizeRowsI8 *a, cudaStream_t s) {
  const int64_t per_row = a->width / VW, chunks = per_row * a->rows;
  if (chunks > INT32_MAX) return SPKV2_ERR_UNSUPPORTED;
  // Several chunks a thread once all SMs are full (eight blocks each).
  const unsigned grid = unsigned(std::min<int64_t>(ceil_div(chunks, 256), int64_t(sm_count()) * 64));
  row_values_kernel<T, VW><<<grid, 256, 0, s>>>(a->codes, a->scale, static_cast<T *>(a->y), uint32_t(chunks),
                                                FastDiv(uint32_t(per_row)), a->codes_stride, a->y_stride);
  return cuda_status(cudaGetLastError());
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
    // Stores of 16 bytes at most: y's alignment beyond them does not matter.
    constexpr int64_t size = sizeof(T);
    const bool many = a->rows > 1;
    int vw = vector_width(16, a->width, reinterpret_cast<uintptr_t>(a->codes), many ? a->codes_stride : 0);
    const int vy = vector_width(16 / int(size), a->width, reinterpret_cast<uintptr_t>(a->y) / size, many ? a->y_stride : 0);
    if (vy < 16 / int(size)) vw = std::min(vw, vy);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (vw) {
      case 16: return launch_values<T, 16>(a, s);
      case 8: return launch_values<T, 8>(a, s);
      case 4: return launch_values<T, 4>(a, s);
      case 2: return launch_values<T, 2>(a, s);
      default: return launch_values<T, 1>(a, s);
    }
  });
}
