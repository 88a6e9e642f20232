// Cross attention in fp32 on the tensor cores (mma.sync, TF32 in three passes).
//
// An fp32 value x is split into hi = x rounded to TF32 and lo = x - hi, which is
// exact and fits TF32 up to 2^-22 of x, and a product into hi hi + hi lo + lo hi;
// what is left out is 2^-22 of it.  The MMA cuts its sums off where fp32 would round
// them, which adds up over long chains (2e-6 of the answer); so a sum takes four
// (scores) or eight (answers) MMAs from zero and is then added up in fp32 registers,
// and the small cross products have sums of their own.
//
// A CTA of four warps passes over the keys in tiles of 64.  W warps (1, 2 or 4)
// share 16 of the CTA's 64 / W rows and take 64 / W of a tile's keys each, with
// their own m, l and O, joined at the end: more where 64 rows a CTA would leave SMs
// idle or most of the rows empty.
// Keys and values have one buffer each: the next tile's keys load while this
// tile's probabilities and values are multiplied, and its values during the next
// scores.  The scores' accumulators are the next product's A operand: its columns
// t and t + 4 stand for keys 2 t and 2 t + 1 of eight, in both operands.
//
// An infinite value has no low part (inf - inf), and one next to the largest has an
// infinite high part, so their products, though defined, come out as NaN.  Where such
// values count, rows with an answer that is not finite are taken again by plain fp32
// products.
//
// With too few row tiles for the SMs the CTAs of a cluster divide the keys, as in
// the other kernels.  Bound by the MMAs and what splits their operands: 40 TFLOP/s of
// answers (4 x 1024 x 16 heads, 1024 keys, width 128: 865 us; on CUDA cores 1339 us),
// three TF32 MMAs each.
#include "cross_attention.cuh"

namespace spkv2 {

namespace {

using namespace xf;
using namespace tc;

constexpr int kKeys = 64, kThreads = 128, kMaxCluster = 8;

template <int D, int W>
struct F32Smem {
  static constexpr int rows = 64 / W;
  float k[kKeys][D + 4];  // at the end, with v: O, [64][D]
  float v[kKeys][D + 4];
  float q[rows][D + 4];
  float m[64], l[64];  // of the warps' 16 rows
  float cm[64], cl[64];  // of the CTA's rows, joined
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// x = hi + lo, both as TF32 operands (the low bits of lo are dropped by the MMA).
__device__ __forceinline__ void split(float x, uint32_t &hi, uint32_t &lo) {
  const float h = tf32_rna(x);
  hi = __float_as_uint(h);
  lo = __float_as_uint(x - h);
}

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// G accumulators by one A operand and G B operands: the large products into c, the
// cross products, 2^-11 of them, into their own sums.
template <int G>
__device__ __forceinline__ void mma3(float (&c)[G][4], float (&cross)[G][4], const float (&a)[4], const float (&b)[G][2]) {
  uint32_t ah[4], al[4], bh[G][2], bl[G][2];
#pragma unroll
  for (int e = 0; e < 4; ++e) split(a[e], ah[e], al[e]);
#pragma unroll
  for (int n = 0; n < G; ++n) {
    split(b[n][0], bh[n][0], bl[n][0]);
    split(b[n][1], bh[n][1], bl[n][1]);
  }
#pragma unroll
  for (int n = 0; n < G; ++n) mma(c[n], ah, bh[n]);
#pragma unroll
  for (int n = 0; n < G; ++n) mma(cross[n], al, bh[n]);
#pragma unroll
  for (int n = 0; n < G; ++n) mma(cross[n], ah, bl[n]);
}

// 4-byte async copy global -> shared; bytes = 0 writes zeros.
__device__ __forceinline__ void cp_async4(void *dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}

// A value whose high part is infinite.
__device__ __forceinline__ bool unsplittable(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u >= 0x7f7ff000u && u <= 0x7f800000u;
}

// One row by plain fp32 products, by a warp: `q` in shared memory, `mask` of its entry
// or null, `out` its place.  Keys pass twice, once for m and l and once for the answer,
// so that no sum is larger than the values that it weighs.
template <int D>
__device__ __noinline__ void plain_row(const float *q, const float *k, const float *v, float *out, int64_t k_stride, int64_t v_stride,
                                       const uint8_t *mask, int keys, int width, float scale_log2) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  auto counts = [&](int j) { return !mask || mask[j] != 0; };
  auto score = [&](int j) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 32 * i < width) s = fmaf(q[lane + 32 * i], k[j * k_stride + lane + 32 * i], s);
#pragma unroll
    for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    return s * scale_log2;
  };
  float m = -INFINITY, l = 0.0f;
  for (int j = 0; j < keys; ++j) {
    if (!counts(j)) continue;
    const float s = score(j), top = fmaxf(m, s), use = top == -INFINITY ? 0.0f : top;
    l = l * exp2f(m - use) + exp2f(s - use);
    m = top;
  }
  const float use = m == -INFINITY ? 0.0f : m;
  float o[N] = {};
  for (int j = 0; j < keys; ++j) {
    if (!counts(j)) continue;
    const float p = exp2f(score(j) - use) / l;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 32 * i < width) o[i] = fmaf(p, v[j * v_stride + lane + 32 * i], o[i]);
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (lane + 32 * i < width) out[lane + 32 * i] = l != 0.0f ? o[i] : 0.0f;
}

template <int D, int W>
__global__ void __launch_bounds__(kThreads, D == 128 ? 2 : W == 4 ? 4 : 3) cross_f32_kernel(AttnArgs a, int csize, bool vec, bool vec_q, bool vec_out) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  using S = F32Smem<D, W>;
  S &sm = *reinterpret_cast<S *>(smem_raw);
  __shared__ uint32_t s_again[2];  // rows of the CTA with an answer that is not finite
  constexpr int KW = 64 / W, NT = KW / 8;  // keys of a warp in a tile, in eights
  constexpr int G = NT < 4 ? NT : 4;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (tid < 2) s_again[tid] = 0;
  const int rank = csize > 1 ? int(cluster_rank()) : 0;
  int item = int(blockIdx.x) / csize;
  const int r0 = item % a.row_tiles * S::rows;
  item /= a.row_tiles;
  const int hk = item % a.kv_heads, b = item / a.kv_heads;
  const float *q = static_cast<const float *>(a.q) + b * a.qs[0];
  const float *k = static_cast<const float *>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const float *v = static_cast<const float *>(a.v) + b * a.vs[0] + hk * a.vs[2];
  const int keys = counted_keys<kThreads>(a, b, tid), tiles = (keys + kKeys - 1) / kKeys;
  const int tile0 = int(int64_t(tiles) * rank / csize), tile1 = int(int64_t(tiles) * (rank + 1) / csize);

  // A tile's keys or values; zeros for keys that do not count and beyond the width.
  auto load = [&](float (*to)[D + 4], const float *from, int64_t stride, int tile) {
    if (vec) {
#pragma unroll 4
      for (int e = tid * 4; e < kKeys * D; e += kThreads * 4) {
        const int r = e / D, c = e % D, j = tile * kKeys + r;
        const bool in = j < keys && c < a.width && (!a.key_mask || a.key_mask[b * a.mask_stride + j] != 0);
        cp_async16(&to[r][c], in ? from + j * stride + c : from, in ? 16u : 0u);
      }
    } else {
#pragma unroll 4
      for (int e = tid; e < kKeys * D; e += kThreads) {
        const int r = e / D, c = e % D, j = tile * kKeys + r;
        const bool in = j < keys && c < a.width && (!a.key_mask || a.key_mask[b * a.mask_stride + j] != 0);
        cp_async4(&to[r][c], in ? from + j * stride + c : from, in ? 4u : 0u);
      }
    }
  };
  if (vec_q) {
#pragma unroll 4
    for (int e = tid * 4; e < S::rows * D; e += kThreads * 4) {
      const int r = e / D, c = e % D, row = r0 + r;
      const bool in = row < a.rows && c < a.width;
      cp_async16(&sm.q[r][c], in ? q + row_offset(a, a.qs, hk, row) + c : q, in ? 16u : 0u);
    }
  } else {
#pragma unroll 4
    for (int e = tid; e < S::rows * D; e += kThreads) {
      const int r = e / D, c = e % D, row = r0 + r;
      const bool in = row < a.rows && c < a.width;
      cp_async4(&sm.q[r][c], in ? q + row_offset(a, a.qs, hk, row) + c : q, in ? 4u : 0u);
    }
  }
  if (tile0 < tile1) load(sm.k, k, a.ks[1], tile0);
  cp_async_commit();
  if (tile0 < tile1) load(sm.v, v, a.vs[1], tile0);
  cp_async_commit();

  const int qr = warp / W * 16, key0 = warp % W * KW;  // this warp's rows and keys of a tile
  float o[D / 8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {};
  for (int tile = tile0; tile < tile1; ++tile) {
    uint64_t bits = ~uint64_t(0);  // which of the tile's keys count
    const int j0 = tile * kKeys;
    if (a.key_mask || j0 + kKeys > keys) {
      bits = 0;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int j = j0 + w * 32 + lane;
        bool in = j < keys;
        if (in && a.key_mask) in = a.key_mask[b * a.mask_stride + j] != 0;
        bits |= uint64_t(__ballot_sync(0xffffffffu, in)) << (32 * w);
      }
    }
    const int live = keys - j0 - key0;  // this warp's keys of the tile end here: eights beyond are skipped
    cp_async_wait<1>();  // the keys; the values may still be on their way
    __syncthreads();
    float s[NT][4] = {};
#pragma unroll
    for (int n = 0; n < NT; n += G) {
      if (n * 8 >= live) break;
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 32) {
        float sum[G][4] = {}, cross[G][4] = {};
#pragma unroll
        for (int c = c0; c < c0 + 32; c += 8) {
          const float av[4] = {sm.q[qr + g][c + t], sm.q[qr + g + 8][c + t], sm.q[qr + g][c + t + 4], sm.q[qr + g + 8][c + t + 4]};
          float bv[G][2];
#pragma unroll
          for (int i = 0; i < G; ++i) {
            bv[i][0] = sm.k[key0 + (n + i) * 8 + g][c + t];
            bv[i][1] = sm.k[key0 + (n + i) * 8 + g][c + t + 4];
          }
          mma3<G>(sum, cross, av, bv);
        }
#pragma unroll
        for (int i = 0; i < G; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n + i][e] += sum[i][e] + cross[i][e];
      }
    }
    __syncthreads();  // everybody has read the keys
    if (tile + 1 < tile1) load(sm.k, k, a.ks[1], tile + 1);
    cp_async_commit();

    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = (bits >> (key0 + n * 8 + 2 * t + (e & 1))) & 1;
        s[n][e] = in ? s[n][e] * a.scale_log2 : -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
      }
    bool rise[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
      rise[h] = top[h] > m[h] + 8.0f;  // from m = -inf: any score
    }
    if (__any_sync(0xffffffffu, rise[0] || rise[1])) {
      float f[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f[h] = rise[h] ? ex2(m[h] - top[h]) : 1.0f;
        if (rise[h]) m[h] = top[h];
        l[h] *= f[h];
      }
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] *= f[e >> 1];
    }
    const float use[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = ex2(s[n][e] - use[e >> 1]);
        l[e >> 1] += s[n][e];
      }
    cp_async_wait<1>();  // the values; the next keys may still be on their way
    __syncthreads();
#pragma unroll
    for (int d = 0; d < D / 8; d += 4) {
      float sum[4][4] = {}, cross[4][4] = {};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (n * 8 >= live) break;
        const float pv[4] = {s[n][0], s[n][2], s[n][1], s[n][3]};  // columns t and t + 4: keys 2 t and 2 t + 1
        const int j = key0 + n * 8 + 2 * t;
        float bv[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bv[i][0] = sm.v[j][(d + i) * 8 + g];
          bv[i][1] = sm.v[j + 1][(d + i) * 8 + g];
        }
        mma3<4>(sum, cross, pv, bv);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d + i][e] += sum[i][e] + cross[i][e];
    }
    __syncthreads();  // everybody has read the values
    if (tile + 1 < tile1) load(sm.v, v, a.vs[1], tile + 1);
    cp_async_commit();
  }
  cp_async_wait<0>();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
  }
  auto out_row = [&](int row) { return static_cast<float *>(a.out) + b * a.os[0] + row_offset(a, a.os, hk, row); };
  // Rows with an answer that is not finite, once more where a value that counts cannot be
  // split.  A NaN among the keys is in every answer, and leaves nothing to mend.
  auto mend = [&] {
    if (!(s_again[0] | s_again[1])) return;
    const uint8_t *mask = a.key_mask ? a.key_mask + b * a.mask_stride : nullptr;
    bool found = false, nan = false;
    for (int e = tid; e < S::rows * D; e += kThreads) found |= unsplittable(sm.q[e / D][e % D]);
    for (int j = warp; j < keys; j += kThreads / 32) {
      if (mask && mask[j] == 0) continue;
      for (int c = lane; c < a.width; c += 32) {
        const float x = k[j * a.ks[1] + c];
        found |= unsplittable(x) || unsplittable(v[j * a.vs[1] + c]);
        nan |= x != x;
      }
    }
    if (!__syncthreads_or(found) || __syncthreads_or(nan)) return;
    for (int r = warp; r < S::rows; r += kThreads / 32)
      if ((s_again[r >> 5] >> (r & 31)) & 1)
        plain_row<D>(sm.q[r], k, v, out_row(r0 + r), a.ks[1], a.vs[1], mask, keys, a.width, a.scale_log2);
  };
  if (W == 1 && csize == 1) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = r0 + qr + h * 8 + g;
      if (row >= a.rows) continue;
      const float inv = l[h] != 0.0f ? 1.0f / l[h] : 0.0f;
      float *out = out_row(row), size[4] = {};  // sums that are finite only if all answers are
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        const int c = n * 8 + 2 * t;
        const float x = o[n][2 * h] * inv, y = o[n][2 * h + 1] * inv;
        size[n & 3] += fabsf(x) + fabsf(y);
        if (vec_out) {
          if (c < a.width) *reinterpret_cast<float2 *>(out + c) = make_float2(x, y);
        } else {
          if (c < a.width) out[c] = x;
          if (c + 1 < a.width) out[c + 1] = y;
        }
      }
      if (!(size[0] + size[1] + size[2] + size[3] < INFINITY)) atomicOr(&s_again[(qr + h * 8 + g) >> 5], 1u << ((qr + h * 8 + g) & 31));
    }
    __syncthreads();
    mend();
    return;
  }
  auto put = [&](int r, int c, float x) {
    if (c >= a.width) return;
    out_row(r0 + r)[c] = x;
    if (!(fabsf(x) < INFINITY)) atomicOr(&s_again[r >> 5], 1u << (r & 31));
  };
  __syncthreads();  // the last values have been read: O goes over keys and values
  float *part = &sm.k[0][0];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = warp * 16 + h * 8 + g;
    if (t == 0) {
      sm.m[r] = m[h];
      sm.l[r] = l[h];
    }
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
      *reinterpret_cast<float2 *>(part + r * D + n * 8 + 2 * t) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
  }
  __syncthreads();
  auto weight = [](float mw, float top) { return mw == -INFINITY ? 0.0f : ex2(mw - top); };
  const int used = min(S::rows, a.rows - r0) * D;
  // Row r is rows r % 16 of the W warps from r / 16 * W on; joined in warp order into
  // the first one's place.
  auto place = [](int r) { return r / 16 * W * 16 + r % 16; };
  if (W > 1) {
    for (int e = tid; e < used; e += kThreads) {
      const int r = e / D, c = e % D, at = place(r);
      float top = sm.m[at], acc = 0.0f, sum = 0.0f;
#pragma unroll
      for (int w = 1; w < W; ++w) top = fmaxf(top, sm.m[at + w * 16]);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = weight(sm.m[at + w * 16], top);
        acc = fmaf(part[(at + w * 16) * D + c], f, acc);
        sum = fmaf(sm.l[at + w * 16], f, sum);
      }
      if (csize == 1) {
        put(r, c, sum != 0.0f ? acc / sum : 0.0f);
      } else {
        part[at * D + c] = acc;
        if (c == 0) {
          sm.cm[r] = top;
          sm.cl[r] = sum;
        }
      }
    }
  }
  if (csize > 1) {
    const float *cm = W > 1 ? sm.cm : sm.m, *cl = W > 1 ? sm.cl : sm.l;
    __syncwarp();
    cluster_sync();
    for (int e = rank * kThreads + tid; e < used; e += csize * kThreads) {
      const int r = e / D, c = e % D;
      float mk[kMaxCluster], lk[kMaxCluster], ok[kMaxCluster], top = -INFINITY, acc = 0.0f, sum = 0.0f;
#pragma unroll
      for (int n = 0; n < kMaxCluster; ++n) {
        if (n >= csize) break;
        mk[n] = __uint_as_float(ld_cluster(map_rank(&cm[r], n)));
        lk[n] = __uint_as_float(ld_cluster(map_rank(&cl[r], n)));
        ok[n] = __uint_as_float(ld_cluster(map_rank(&part[place(r) * D + c], n)));
        top = fmaxf(top, mk[n]);
      }
#pragma unroll
      for (int n = 0; n < kMaxCluster; ++n) {
        if (n >= csize) break;
        const float f = weight(mk[n], top);
        acc = fmaf(ok[n], f, acc);
        sum = fmaf(lk[n], f, sum);
      }
      put(r, c, sum != 0.0f ? acc / sum : 0.0f);
    }
    __syncwarp();
    cluster_sync();  // the peers have read this CTA's sums, and every answer is written
  } else {
    __syncthreads();
  }
  mend();  // two CTAs of a cluster may mend one row; they write the same bits
}

template <int D, int W>
int launch(AttnArgs a, int csize, cudaStream_t s) {
  using S = F32Smem<D, W>;
  static_assert(sizeof(S::k) + sizeof(S::v) >= 64 * D * 4, "O takes the place of keys and values");
  a.row_tiles = int(ceil_div(a.rows, S::rows));
  const int64_t blocks = int64_t(a.row_tiles) * a.kv_heads * a.batch;
  if (blocks * csize > INT32_MAX) return SPKV2_ERR_UNSUPPORTED;
  if (const int rc = allow_smem<cross_f32_kernel<D, W>>(sizeof(S))) return rc;
  auto rows16 = [](const void *base, const int64_t (&st)[3]) {
    return aligned16(base) && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0;
  };
  const bool vec = a.width % 4 == 0 && rows16(a.k, a.ks) && rows16(a.v, a.vs);
  const bool vec_q = a.width % 4 == 0 && rows16(a.q, a.qs);
  const bool vec_out = a.width % 2 == 0 && on_bytes(8, a.out) && a.os[0] % 2 == 0 && a.os[1] % 2 == 0 && a.os[2] % 2 == 0;
  return cuda_status(launch_kernel(cross_f32_kernel<D, W>, unsigned(blocks * csize), unsigned(kThreads), sizeof(S), s, csize, a,
                                   csize, vec, vec_q, vec_out));
}

// Warps a row and CTAs a cluster by an estimate of the time in microseconds, fitted
// to sweeps of both over ten sizes (over sixteen, the choice took at most 16 % longer
// than the best, for thirteen at most 1 %): a tile takes its warps `wait` + `work` / W one after another, and an SM
// `share` + `full` / W of its throughput; a cluster of eight is slow to start where
// there are more CTAs than SMs.
template <int D>
int launch_rows(const AttnArgs &a, cudaStream_t s) {
  constexpr double wait = D == 32 ? 1.5 : D == 64 ? 3.1 : 3.6, work = D == 32 ? 0.7 : D == 64 ? 1.6 : 5.2;
  constexpr double share = D == 32 ? 0.3 : D == 64 ? 0.7 : 1.4, full = D == 32 ? 2.2 : D == 64 ? 2.6 : 5.5;
  const double sms = sm_count();
  const int64_t tiles = ceil_div(a.keys, kKeys);
  int best_w = 1, best_c = 1;
  double best = 1e30;
  for (int w = 1; w <= 4; w *= 2)
    for (int c = 1; c <= kMaxCluster && (c == 1 || tiles >= c); c *= 2) {
      const double ctas = double(ceil_div(a.rows, 64 / w)) * a.kv_heads * a.batch * c, each = double(ceil_div(tiles, c));
      const double start = c == 1 ? 0.0 : c == 2 ? 1.0 : c == 4 ? 2.0 : 3.0 + 3.0 * std::max(0.0, ctas / sms - 1.0);
      const double time = start + std::max(3.0 + each * (wait + work / w), ctas * each * (share + full / w) / sms);
      if (time < best) best = time, best_w = w, best_c = c;
    }
  if (best_w == 4) return launch<D, 4>(a, best_c, s);
  return best_w == 2 ? launch<D, 2>(a, best_c, s) : launch<D, 1>(a, best_c, s);
}

}  // namespace

int cross_f32(const AttnArgs &a, cudaStream_t s) {
  if (a.width <= 32) return launch_rows<32>(a, s);
  return a.width <= 64 ? launch_rows<64>(a, s) : launch_rows<128>(a, s);
}

}  // namespace spkv2
