// Root-mean-square norm with the residual's addition and int8 output, the
// int8 codes of a tensor's rows, and the values that codes stand for.
//
//   s = x + r,  y = s w / sqrt(mean(s^2) + eps),  scale = max|y| / 127,
//   code = rne(y / scale)
//
// The factor 1 / sqrt(..) is common to a row, so it cancels in the codes:
//   code = rne(s w * (127 / max|s w|)),  scale = max|s w| / sqrt(..) / 127,
// and both reductions (sum of s^2, max |s w|) run in one pass over the row.
// Quantising without the norm is the same with r = 0, w = 1 and no factor.  Rows
// whose squares leave fp32's range are scaled by a power of two first.
//
// The maximum keeps a NaN, so it says by itself whether the row is finite.
#include "tcgen05.cuh"
#include "transformer.cuh"

namespace spkv2 {

namespace {

using namespace xf;
using namespace tc;

constexpr int64_t kMaxWidth = int64_t(1) << 24, kMostWidth = 16384;  // of a call; of rows kept in registers
constexpr int kPerThread = 16;  // elements; with 8 the synchronisation costs more (40000 x 512 in bf16: 29 us, with 16 24 us)

struct RowArgs {
  const void *x, *residual, *weight;
  void *sum;
  int8_t *codes;
  float *scale;
  int64_t rows, width;
  int64_t x_stride, residual_stride, sum_stride, codes_stride;
  float eps;
};

// The larger of two magnitudes; a NaN stays.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// What takes s w to codes: code = rne(v * pre * inv).  127 / amax overflows where
// amax is below 2^-121 or so; values that small are scaled up by pre = 2^64,
// exactly, first.  Both are 0 for rows of zeros and rows that are not finite.
struct CodeScale {
  float pre, inv;
};
__device__ __forceinline__ CodeScale code_scale(float amax) {
  CodeScale c;
  c.pre = amax < 1e-30f ? 18446744073709551616.0f : 1.0f;
  c.inv = amax > 0.0f ? 127.0f / (amax * c.pre) : 0.0f;
  return c;
}
// |v| <= amax, so v * inv rounds to at most 127 in magnitude, and adding 1.5 * 2^23
// rounds it to the nearest even integer, which lands in the sum's low byte in
// two's complement.
__device__ __forceinline__ uint32_t code_bits(float v, float inv) { return __float_as_uint(fmaf(v, inv, 12582912.0f)); }
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// N elements in one access.
template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// 16 bytes of elements as fp32 and back, two elements of 16 bits a step: taken one
// by one out of a struct they cost a row kernel three times the instructions.
__device__ __forceinline__ void expand(const uint4 &u, float (&f)[4], float) {
  f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void expand(const uint4 &u, float (&f)[8], __nv_bfloat16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
__device__ __forceinline__ void expand(const uint4 &u, float (&f)[8], __half) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    f[2 * i] = v.x, f[2 * i + 1] = v.y;
  }
}
__device__ __forceinline__ uint4 contract(const float (&f)[4], float) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
__device__ __forceinline__ uint4 contract(const float (&f)[8], __nv_bfloat16) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t *>(&v);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 contract(const float (&f)[8], __half) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t *>(&v);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Values of a row whose sum of squares may leave fp32's range, or lose bits at its
// lower end, are taken as s / 2^x instead, x the exponent of the largest |s| among
// them: no square of those overflows, nor a product with a weight, and what
// underflows is too small to matter.  Inside the range |s| < 2^30.
__device__ __forceinline__ bool out_of_range(float ss) { return !(ss >= 0x1p-90f && ss <= 0x1p60f); }
__device__ __forceinline__ int exponent_of(float top) { return ilogbf(top) + 1; }
// 2^n for |n| up to 298 as two factors.
struct TwoTo {
  float a, b;
  __device__ __forceinline__ explicit TwoTo(int n) : a(scalbnf(1.0f, n / 2)), b(scalbnf(1.0f, n - n / 2)) {}
  __device__ __forceinline__ float of(float v) const { return v * a * b; }
};

// The scale of a row whose ss and amax are of s / 2^x.
__device__ __noinline__ float scale_from(float ss, float amax, int x, int64_t width, float eps) {
  if (!(amax < INFINITY)) return __uint_as_float(0x7fc00000u);
  if (amax == 0.0f) return 0.0f;
  const double mean = scalbn(double(ss) / double(width), 2 * x) + double(eps);
  return float(scalbn(double(amax), x) / sqrt(mean) / 127.0);
}

// A row's scale (its first thread writes it) and the factor of its codes.
template <bool NORM>
__device__ __forceinline__ CodeScale finish_row(const RowArgs &p, int64_t row, float ss, float amax, bool &finite, bool writes) {
  finite = amax < INFINITY;
  if (writes) {
    const float f = NORM && amax > 0.0f ? 1.0f / sqrtf(ss / float(p.width) + p.eps) : 1.0f;
    p.scale[row] = finite ? amax * f / 127.0f : __uint_as_float(0x7fc00000u);
  }
  return code_scale(finite ? amax : 0.0f);
}

__host__ __device__ __forceinline__ int stage_at(int e, int u) { return e + e / u; }
__host__ __device__ __forceinline__ int stage_floats(int width, int u) { return stage_at((width + u - 1) / u * u, u); }

// The threads of one row of a block; at most two rows of a block have several warps.
// (The barrier's number is a constant: one in a register reserves all sixteen, and
// fewer blocks fit an SM.)
__device__ __forceinline__ void row_barrier(int row, int threads) {
  if (row == 0)
    asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
  else
    asm volatile("bar.sync 2, %0;" ::"r"(threads) : "memory");
}
constexpr int kNoValues = -1024, kShift = 1024;  // exponent of a thread that has only zeros; makes exponents positive

// Bound by memory: every element is read once, kept in registers (16 a thread)
// through the row's two reductions, and its code written once.  A block for each
// row (or a few) and no more: blocks that stay, load the next row ahead and keep
// the weights need registers that cost more loads in flight than they save
// (16384 x 4096 in bf16: 147 us, without 96 us).
//
// A thread owns units of 16 bytes of x (U elements), t, t + tpr, ..: which element
// is added where depends on the width alone, not on alignment or the number of
// rows, so neither do the bits of the result.
//
// STAGED: rows that do not start on 16-byte boundaries, or end inside a unit.
// They are read in the 16-byte pieces that memory has, and pass through shared
// memory (as fp32 sums) to the threads that own the units.  One word of padding a
// unit: a warp's accesses to the same place of 32 units fall into 32 banks.
//
// The residual's sum is written by the thread that read both parts, so it may
// take their place.  rpb rows a block: one row of any number of warps, or several
// of a power of two of threads.
template <class T, bool NORM, bool STAGED>
__global__ void __launch_bounds__(1024)
    row_codes_kernel(RowArgs p, int tpr, int rpb, bool vec_codes, bool vec_weight) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int U = 16 / sizeof(T), N = kPerThread / U;
  extern __shared__ __align__(16) float staged[];
  __shared__ float s_sum[32], s_max[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = rpb > 1 ? threadIdx.x / tpr : 0, t = threadIdx.x - sub * tpr, wpr = tpr >> 5;
  const int width = int(p.width);
  const T *w = static_cast<const T *>(p.weight);
  float *mine = staged + sub * stage_floats(width, U);

  auto weights = [&](int c) {
    Vec<T, U> wv;
    if (!STAGED || (vec_weight && c + U <= width)) wv = *reinterpret_cast<const Vec<T, U> *>(w + c);
    else
#pragma unroll
      for (int e = 0; e < U; ++e) wv.v[e] = c + e < width ? w[c + e] : from_f32<T>(0.0f);
    return *reinterpret_cast<const uint4 *>(&wv);
  };
  // A row's pieces: `head` elements before its first 16-byte boundary, whole
  // units, and the rest from `tail` on.  Where the residual or the sum have their
  // boundaries elsewhere, all elements count as head.
  const uint4 none = make_uint4(0, 0, 0, 0);
  uint4 xv[N], rv[N], wv[N];
  T xe, re;
  int head = 0, units = (width + U - 1) / U, tail = width;
  const int64_t row = int64_t(blockIdx.x) * rpb + sub;
  const bool real = row < p.rows;
  const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
  const T *r = static_cast<const T *>(p.residual) + row * p.residual_stride;
  T *sum = static_cast<T *>(p.sum) + row * p.sum_stride;
  if (real) {
    if (STAGED) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(x);
      const uintptr_t sum_at = reinterpret_cast<uintptr_t>(sum);
      const bool same = !NORM || ((!p.residual || ((at ^ reinterpret_cast<uintptr_t>(r)) & 15) == 0) &&
                                  (!p.sum || ((at ^ sum_at) & 15) == 0));
      head = same ? min(int((16 - (at & 15)) & 15) / int(sizeof(T)), width) : width;
      units = (width - head) / U;
      tail = head + units * U;
      if (t < head + width - tail) {
        const int e = t < head ? t : t - head + tail;
        xe = x[e];
        if (NORM && p.residual) re = r[e];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int k = t + i * tpr;
    const bool in = real && k < units;
    xv[i] = in ? *reinterpret_cast<const uint4 *>(x + head + k * U) : none;
    if (NORM && p.residual) rv[i] = in ? *reinterpret_cast<const uint4 *>(r + head + k * U) : none;
  }
  // Held from here on, the weights would cost staged fp32 rows spills (9000 x 2647: 74
  // us, read where they are used 62).
  constexpr bool HOLDS = NORM && !(STAGED && sizeof(T) == 4);
  auto unit_weights = [&](int i) { return (t + i * tpr) * U < width ? weights((t + i * tpr) * U) : none; };
  if (HOLDS) {
#pragma unroll
    for (int i = 0; i < N; ++i) wv[i] = unit_weights(i);
  }
  float v[N][U];
  auto unstage = [&] {  // this thread's units; zeros past the width
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (t + i * tpr) * U;
#pragma unroll
      for (int e = 0; e < U; ++e) v[i][e] = real && c < width ? mine[(t + i * tpr) * (U + 1) + e] : 0.0f;
    }
  };
  if (STAGED) {
    // Places of a unit's elements: element head + k U + e lies at k (U + 1) + place[e].
    int place[U];
#pragma unroll
    for (int e = 0; e < U; ++e) place[e] = stage_at(head + e, U);
    if (real) {
      for (int c = t; c < head + width - tail; c += tpr) {
        const int e = c < head ? c : c - head + tail;
        float s;
        if (c == t) {
          s = to_f32(xe);
          if (NORM && p.residual) s += to_f32(re);
        } else {
          s = to_f32(x[e]);
          if (NORM && p.residual) s += to_f32(r[e]);
        }
        if (NORM && p.sum) sum[e] = from_f32<T>(s);
        mine[stage_at(e, U)] = s;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int k = t + i * tpr;
        if (k >= units) break;
        float s[U];
        expand(xv[i], s, T{});
        if (NORM && p.residual) {
          float add[U];
          expand(rv[i], add, T{});
#pragma unroll
          for (int e = 0; e < U; ++e) s[e] += add[e];
        }
#pragma unroll
        for (int e = 0; e < U; ++e) mine[k * (U + 1) + place[e]] = s[e];
        if (NORM && p.sum) *reinterpret_cast<uint4 *>(sum + head + k * U) = contract(s, T{});
      }
      if (t < (width + U - 1) / U * U - width) mine[stage_at(width + t, U)] = 0.0f;
    }
    __syncthreads();
    unstage();
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (t + i * tpr) * U;
      expand(xv[i], v[i], T{});
      if (NORM && p.residual) {
        float add[U];
        expand(rv[i], add, T{});
#pragma unroll
        for (int e = 0; e < U; ++e) v[i][e] += add[e];
      }
      if (NORM && p.sum && real && c < width) *reinterpret_cast<uint4 *>(sum + c) = contract(v[i], T{});
    }
  }
  float ss = 0.0f, mx = 0.0f;
  auto weigh = [&](const uint4 &raw, float (&f)[U]) {  // a unit's products
    if (NORM) {
      float wf[U];
      expand(raw, wf, T{});
#pragma unroll
      for (int e = 0; e < U; ++e) f[e] *= wf[e];
    }
#pragma unroll
    for (int e = 0; e < U; ++e) mx = max_nan(mx, fabsf(f[e]));
  };
  // A thread whose values leave the range scales its own; an infinite ss says so to the
  // others of the row, who follow below.  It needs s once more: staged rows have it in
  // shared memory, the others form their products after the test.
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (NORM) {
#pragma unroll
      for (int e = 0; e < U; ++e) ss = fmaf(v[i][e], v[i][e], ss);
    }
    if (!NORM || STAGED) weigh(NORM && !HOLDS ? unit_weights(i) : wv[i], v[i]);
  }
  int x_exp = 0;
  float own = ss;
  if (NORM && out_of_range(ss)) {
    if (STAGED) unstage();
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < U; ++e) top = max_nan(top, fabsf(v[i][e]));
    own = 0.0f;
    if (top > 0.0f && top < INFINITY) {
      x_exp = exponent_of(top);
      const TwoTo down(-x_exp);
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < U; ++e) {
          v[i][e] = down.of(v[i][e]);
          own = fmaf(v[i][e], v[i][e], own);
        }
      ss = INFINITY;
    } else if (top == 0.0f) {
      x_exp = kNoValues;
    } else {
      ss = 0.0f;
    }
    mx = top < INFINITY ? 0.0f : __uint_as_float(0x7fc00000u);
    if (STAGED) {
#pragma unroll
      for (int i = 0; i < N; ++i) weigh(unit_weights(i), v[i]);
    }
  }
  if (NORM && !STAGED) {
#pragma unroll
    for (int i = 0; i < N; ++i) weigh(wv[i], v[i]);
  }
  auto join = [&](float &sum, float &top, bool again) {
    for (int o = min(tpr, 32) / 2; o; o >>= 1) {
      if (NORM) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (wpr <= 1) return;
    if (again) row_barrier(sub, tpr);  // the sums before have been read
    if (lane == 0) {
      s_sum[warp] = sum;
      s_max[warp] = top;
    }
    if (again)
      row_barrier(sub, tpr);
    else
      __syncthreads();
    const int w0 = sub * wpr;
    sum = lane < wpr ? s_sum[w0 + lane] : 0.0f;
    top = lane < wpr ? s_max[w0 + lane] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      if (NORM) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
  };
  float amax = mx;
  join(ss, amax, false);
  bool scaled = false;
  if (NORM) {
    scaled = ss == INFINITY;
    if (__any_sync(0xffffffffu, scaled)) {  // the warps of one row, or rows that share a warp
      float unused = 0.0f, row_exp = float(x_exp + kShift);  // not below 0, where the maximum starts
      join(unused, row_exp, true);
      const TwoTo down(x_exp + kShift - int(row_exp));
      float row_ss = down.of(down.of(own)), row_max = down.of(mx);
      join(row_ss, row_max, true);
      if (scaled) {
        ss = row_ss, amax = row_max;
        x_exp = int(row_exp) - kShift;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int e = 0; e < U; ++e) v[i][e] = down.of(v[i][e]);
      }
    }
  }
  if (!real) return;
  bool finite;
  const CodeScale cs = finish_row<NORM>(p, row, ss, amax, finite, t == 0 && !scaled);
  if (NORM && scaled && t == 0) p.scale[row] = scale_from(ss, amax, x_exp, p.width, p.eps);
  int8_t *codes = p.codes + row * p.codes_stride;
  if (cs.pre != 1.0f || !finite) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < U; ++e) v[i][e] = finite ? v[i][e] * cs.pre : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (t + i * tpr) * U;
    if (c >= width) break;
    uint32_t q[U / 4];
#pragma unroll
    for (int e = 0; e < U; e += 4)
      q[e / 4] = pack4(code_bits(v[i][e], cs.inv), code_bits(v[i][e + 1], cs.inv), code_bits(v[i][e + 2], cs.inv),
                       code_bits(v[i][e + 3], cs.inv));
    if (!STAGED || (vec_codes && c + U <= width)) {
      *reinterpret_cast<Vec<uint32_t, U / 4> *>(codes + c) = *reinterpret_cast<Vec<uint32_t, U / 4> *>(q);
    } else {
#pragma unroll
      for (int e = 0; e < U; ++e)
        if (c + e < width) codes[c + e] = int8_t(q[e / 4] >> (8 * (e & 3)));
    }
  }
}

// A block's sums and maxima, joined for all of its threads.
__device__ __forceinline__ void join_block(float &ss, float &mx, float *s_sum, float *s_max) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    ss += __shfl_xor_sync(0xffffffffu, ss, o);
    mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
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
    mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
}

// A wide row whose sums left the range: all of it again, from s / 2^x.
template <class T>
__device__ __noinline__ void wide_row_scaled(RowArgs p, int64_t row, float *s_sum, float *s_max) {
  const int tid = threadIdx.x, threads = blockDim.x;
  const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
  const T *r = p.residual ? static_cast<const T *>(p.residual) + row * p.residual_stride : nullptr;
  const T *w = static_cast<const T *>(p.weight);
  auto value = [&](int64_t i) { return r ? to_f32(x[i]) + to_f32(r[i]) : to_f32(x[i]); };
  float ss = 0.0f, mx = 0.0f;
  for (int64_t i = tid; i < p.width; i += threads) mx = max_nan(mx, fabsf(value(i)));
  __syncthreads();  // the sums before have been read
  join_block(ss, mx, s_sum, s_max);
  const int x_exp = mx > 0.0f && mx < INFINITY ? exponent_of(mx) : 0;
  if (mx < INFINITY) {
    ss = mx = 0.0f;
    for (int64_t i = tid; i < p.width; i += threads) {
      const float s = scalbnf(value(i), -x_exp);
      ss = fmaf(s, s, ss);
      mx = max_nan(mx, fabsf(s * to_f32(w[i])));
    }
    __syncthreads();
    join_block(ss, mx, s_sum, s_max);
  }
  if (tid == 0) p.scale[row] = scale_from(ss, mx, x_exp, p.width, p.eps);
  const bool finite = mx < INFINITY;
  const CodeScale c = code_scale(finite ? mx : 0.0f);
  T *sum = p.sum ? static_cast<T *>(p.sum) + row * p.sum_stride : nullptr;
  int8_t *codes = p.codes + row * p.codes_stride;
  for (int64_t i = tid; i < p.width; i += threads) {
    const float s = value(i);
    codes[i] = finite ? int8_t(code_bits(scalbnf(s, -x_exp) * to_f32(w[i]) * c.pre, c.inv)) : int8_t(0);
    if (sum) sum[i] = from_f32<T>(s);
  }
}

// Rows wider than kMostWidth, the registers of a block: one block a row, which is read
// twice, the second time from L2; the sum is written in the second pass, as it may take
// x's or the residual's place.
template <class T, bool NORM>
__global__ void __launch_bounds__(1024, 2) wide_codes_kernel(RowArgs p) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float s_sum[32];
  __shared__ float s_max[32];
  const int tid = threadIdx.x, threads = blockDim.x;
  const int64_t row = blockIdx.x;
  const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
  const T *r = NORM && p.residual ? static_cast<const T *>(p.residual) + row * p.residual_stride : nullptr;
  const T *w = static_cast<const T *>(p.weight);
  float ss = 0.0f;
  float mx = 0.0f;
#pragma unroll 4
  for (int64_t i = tid; i < p.width; i += threads) {
    float s = to_f32(x[i]);
    if (r) s += to_f32(r[i]);
    ss = fmaf(s, s, ss);
    mx = max_nan(mx, fabsf(NORM ? s * to_f32(w[i]) : s));
  }
  join_block(ss, mx, s_sum, s_max);
  if (NORM && out_of_range(ss)) {
    wide_row_scaled<T>(p, row, s_sum, s_max);
    return;
  }
  bool finite;
  const CodeScale c = finish_row<NORM>(p, row, ss, mx, finite, tid == 0);
  T *sum = NORM && p.sum ? static_cast<T *>(p.sum) + row * p.sum_stride : nullptr;
  int8_t *codes = p.codes + row * p.codes_stride;
#pragma unroll 4
  for (int64_t i = tid; i < p.width; i += threads) {
    float s = to_f32(x[i]);
    if (r) s += to_f32(r[i]);
    codes[i] = finite ? int8_t(code_bits((NORM ? s * to_f32(w[i]) : s) * c.pre, c.inv)) : int8_t(0);
    if (sum) sum[i] = from_f32<T>(s);
  }
}

// The pieces of a matrix's rows in one list, a thread each: fn(row, piece of the row).
// The list is counted in 32 bits, so it holds at most `most` rows at a time: all of
// them, but for some 2^31 pieces and more.
struct Pieces {
  int64_t rows;
  uint32_t most;
  FastDiv per_row;
  Pieces(int64_t n, int64_t each) : rows(n), most(uint32_t(std::min<int64_t>(n, INT32_MAX / each))), per_row(uint32_t(each)) {}
  // 256 threads a block; several pieces a thread once all SMs are full (eight blocks each).
  unsigned grid() const { return unsigned(std::min<int64_t>(ceil_div(int64_t(most) * per_row.d, 256), int64_t(sm_count()) * 64)); }
};
template <class F>
__device__ __forceinline__ void for_pieces(const Pieces &p, F &&fn) {
  for (int64_t row0 = 0; row0 < p.rows; row0 += p.most) {
    const uint32_t count = uint32_t(min(int64_t(p.most), p.rows - row0)) * p.per_row.d;
    for (uint32_t i = blockIdx.x * 256u + threadIdx.x; i < count; i += gridDim.x * 256u) {
      const uint32_t row = p.per_row.div(i);
      fn(row0 + row, i - row * p.per_row.d);
    }
  }
}

// VW codes a thread.
template <class T, int VW>
__global__ void __launch_bounds__(256)
    row_values_kernel(const int8_t *__restrict__ codes, const float *__restrict__ scale, T *__restrict__ y, Pieces pieces,
                      int64_t codes_stride, int64_t y_stride) {
  pdl_launch_dependents();
  pdl_wait();
  for_pieces(pieces, [&](int64_t row, uint32_t piece) {
    const uint32_t c = piece * VW;
    const float s = __ldg(scale + row);
    const Vec<int8_t, VW> q = *reinterpret_cast<const Vec<int8_t, VW> *>(codes + row * codes_stride + c);
    T *to = y + row * y_stride + c;
    constexpr int S = VW * sizeof(T) > 16 ? 16 / sizeof(T) : VW;  // elements of a store
#pragma unroll
    for (int k = 0; k < VW; k += S) {
      Vec<T, S> o;
#pragma unroll
      for (int e = 0; e < S; ++e) o.v[e] = from_f32<T>(float(q.v[k + e]) * s);
      *reinterpret_cast<Vec<T, S> *>(to + k) = o;
    }
  });
}

// The same where rows of y do not lie on 16-byte boundaries, or end inside one: a
// thread writes the 16 bytes between two boundaries (or, first and last in a row,
// what there is of them) from codes that start anywhere.
template <class T>
__global__ void __launch_bounds__(256)
    row_values_shifted_kernel(const int8_t *__restrict__ codes, const float *__restrict__ scale, T *__restrict__ y, int width,
                              Pieces pieces, int64_t codes_stride, int64_t y_stride, bool vec_codes) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int U = 16 / sizeof(T);
  for_pieces(pieces, [&](int64_t row, uint32_t k) {
    T *to = y + row * y_stride;
    const int8_t *from = codes + row * codes_stride;
    const int head = int((16 - (reinterpret_cast<uintptr_t>(to) & 15)) & 15) / int(sizeof(T));
    const int c = k == 0 ? 0 : head + int(k - 1) * U, end = min(k == 0 ? head : c + U, width);
    if (c >= end) return;
    const float s = __ldg(scale + row);
    if (k > 0 && c + U <= width) {
      Vec<T, U> o;
      // The codes from aligned words, where all of them lie inside the row.
      const int w0 = c & ~3, shift = (c & 3) * 8;
      if (vec_codes && w0 + U + 4 <= width) {
        uint32_t w[U / 4 + 1];
#pragma unroll
        for (int i = 0; i <= U / 4; ++i) w[i] = *reinterpret_cast<const uint32_t *>(from + w0 + 4 * i);
#pragma unroll
        for (int e = 0; e < U; ++e)
          o.v[e] = from_f32<T>(float(int8_t(__funnelshift_r(w[e / 4], w[e / 4 + 1], shift) >> (8 * (e & 3)))) * s);
      } else {
#pragma unroll
        for (int e = 0; e < U; ++e) o.v[e] = from_f32<T>(float(from[c + e]) * s);
      }
      *reinterpret_cast<Vec<T, U> *>(to + c) = o;
    } else {
      for (int e = c; e < end; ++e) to[e] = from_f32<T>(float(from[e]) * s);
    }
  });
}

template <class T, bool NORM, bool STAGED>
int launch_row(const RowArgs &a, bool vec_codes, cudaStream_t s) {
  constexpr auto kern = row_codes_kernel<T, NORM, STAGED>;
  constexpr int U = 16 / sizeof(T);
  // One row of as many warps as it needs, or several of a power of two of threads.
  int tpr = int(ceil_div(ceil_div(a.width, U), kPerThread / U)), rpb = 1;
  if (tpr <= 64) {
    int up = 8;
    while (up < tpr) up *= 2;
    tpr = up, rpb = 128 / up;
  } else {
    tpr = (tpr + 31) / 32 * 32;
  }
  const size_t smem = STAGED ? size_t(rpb) * stage_floats(int(a.width), U) * 4 : 0;
  if (STAGED)
    if (const int rc = allow_smem<kern>(stage_floats(kMostWidth, U) * 4)) return rc;
  return cuda_status(launch_kernel(kern, unsigned(ceil_div(a.rows, rpb)), unsigned(tpr * rpb), smem, s, 1, a, tpr, rpb, vec_codes,
                                   aligned16(a.weight)));
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
    if (a.width > kMostWidth) {
      return cuda_status(launch_kernel(wide_codes_kernel<T, NORM>, unsigned(a.rows), 1024u, 0, s, 1, a));
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
  const Pieces pieces(a->rows, a->width / VW);
  return cuda_status(launch_kernel(row_values_kernel<T, VW>, pieces.grid(), 256u, 0, s, 1, a->codes, a->scale, static_cast<T *>(a->y),
                                   pieces, a->codes_stride, a->y_stride));
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
  if (!on_bytes(elem_bytes(a->dtype), a->x, a->residual, a->weight, a->sum) || !on_bytes(4, a->scale)) return -1;
  RowArgs p = {a->x,     a->residual, a->weight,   a->sum,      a->codes,           a->scale,      a->rows,
               a->width, a->x_stride, a->residual_stride, a->sum_stride, a->codes_stride, a->eps};
  return launch_rows<true>(p, a->dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int spkv2_cuda_quantize_rows_i8(const Spkv2QuantizeRowsI8 *a, void *stream) {
  if (!a || bad_extent(a->rows, a->width)) return -1;
  if (a->rows == 0) return 0;
  if (!a->x || !a->codes || !a->scale || a->x_stride < 0 || overlaps(a->codes_stride, a->rows, a->width)) return -1;
  if (!elem_bytes(a->dtype)) return SPKV2_ERR_UNSUPPORTED;
  if (!on_bytes(elem_bytes(a->dtype), a->x) || !on_bytes(4, a->scale)) return -1;
  RowArgs p = {a->x, nullptr, nullptr, nullptr, a->codes, a->scale, a->rows, a->width, a->x_stride, 0, 0,
               a->codes_stride, 0.0f};
  return launch_rows<false>(p, a->dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int spkv2_cuda_dequantize_rows_i8(const Spkv2DequantizeRowsI8 *a, void *stream) {
  if (!a || bad_extent(a->rows, a->width)) return -1;
  if (a->rows == 0) return 0;
  if (!a->codes || !a->scale || !a->y || a->codes_stride < 0 || overlaps(a->y_stride, a->rows, a->width)) return -1;
  if (!elem_bytes(a->dtype)) return SPKV2_ERR_UNSUPPORTED;
  if (!on_bytes(elem_bytes(a->dtype), a->y) || !on_bytes(4, a->scale)) return -1;
  return by_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    // Stores of 16 bytes at most: y's alignment beyond them does not matter.
    constexpr int64_t size = sizeof(T);
    const bool many = a->rows > 1;
    const int vw = vector_width(16, a->width, reinterpret_cast<uintptr_t>(a->codes), many ? a->codes_stride : 0);
    const int vy = vector_width(16 / int(size), a->width, reinterpret_cast<uintptr_t>(a->y) / size, many ? a->y_stride : 0);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (std::min(vw, vy) < 16 / int(size)) {
      const Pieces pieces(a->rows, 1 + ceil_div(a->width, 16 / size));
      return cuda_status(launch_kernel(row_values_shifted_kernel<T>, pieces.grid(), 256u, 0, s, 1, a->codes, a->scale,
                                       static_cast<T *>(a->y), int(a->width), pieces, a->codes_stride, a->y_stride,
                                       reinterpret_cast<uintptr_t>(a->codes) % 4 == 0 && (!many || a->codes_stride % 4 == 0)));
    }
    if (vw == 16) return launch_values<T, 16>(a, s);
    if (size == 2 || vw == 8) return launch_values<T, 8>(a, s);
    return launch_values<T, 4>(a, s);
  });
}
