// Attention of queries to an encoder's keys and values of another length:
//
//   o_i = sum_j p_ij v_j,  p_i = softmax over the keys that count of scale <q_i, k_j>
//
// No causal order, so the queries of one entry and all the query heads that
// share a key head attend to the same keys: they are laid out as one list of
// rows, r = query * group + (head in the group), and a tile of rows reads
// each key and value once for all of them.
//
// The keys pass once, in tiles, with each row's running maximum m and sum l:
// a tile's scores raise m to m', the sums so far shrink by exp(m - m'), and
// the result is divided by l at the end.  Exponents are taken in base 2, with
// scale * log2(e) as the factor.  A key that does not count has score -inf and
// is read as zeros, so that what lies there (NaN included) has no influence;
// a row without keys keeps l = 0 and is written as 0.
#include "cross_attention.cuh"

namespace spkv2 {

namespace {

using namespace xf;
using namespace tc;

// ------------------------------------------------------------ CUDA cores
// What the tensor-core kernels do not take: widths over 128, and 16-bit types of odd
// width or alignment or with a scale that is not positive.  Exact fp32 products.
// 16 R rows x 64 keys a step, 256 threads; a thread holds scores for R rows x 4 keys
// and sums for R rows x D / 16 columns.  The 16 threads of a row group are half a
// warp.  Bound by issue and the FMA pipe with four rows a thread (25 TFLOP/s at width
// 128); with few rows by shared memory, which every warp reads whole for its two
// rows.  With too few row tiles for the SMs the CTAs of a cluster divide the keys and
// join their m, l and O through distributed shared memory, in CTA order.
constexpr int kKeys = 64, kMaxCluster = 8;

template <int D, int R>
struct SimtSmem {
  static constexpr int rows = 16 * R;
  float k[kKeys][D + 4];  // at the end O, [row][D]
  float v[kKeys][D];
  float q[rows][D + 4];
  float p[rows][kKeys + 4];
  float m[rows], l[rows];
  int valid[kKeys];
};

// Four elements of a row as fp32, in one access.
__device__ __forceinline__ float4 load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
template <class T>
__device__ __forceinline__ float4 load4(const T *p) {
  const uint2 u = *reinterpret_cast<const uint2 *>(p);
  const T *e = reinterpret_cast<const T *>(&u);
  return make_float4(to_f32(e[0]), to_f32(e[1]), to_f32(e[2]), to_f32(e[3]));
}

// The first `left` of four elements, one by one; zeros behind them.
template <class T>
__device__ __forceinline__ float4 load_up_to4(const T *p, int left) {
  return make_float4(to_f32(p[0]), left > 1 ? to_f32(p[1]) : 0.0f, left > 2 ? to_f32(p[2]) : 0.0f, left > 3 ? to_f32(p[3]) : 0.0f);
}

template <class T, int D, int R>
__global__ void __launch_bounds__(256) cross_simt_kernel(AttnArgs a, int csize, bool vec) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  using S = SimtSmem<D, R>;
  S &sm = *reinterpret_cast<S *>(smem_raw);
  static_assert(S::rows <= kKeys, "O takes the place of the keys");
  constexpr int CPT = D / 16;  // columns of a thread: tx * CW + 16 * CW * c
  constexpr int CW = CPT < 4 ? CPT : 4;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  pdl_launch_dependents();
  pdl_wait();
  const int rank = csize > 1 ? int(cluster_rank()) : 0;
  int t = int(blockIdx.x) / csize;
  const int r0 = t % a.row_tiles * S::rows;
  t /= a.row_tiles;
  const int hk = t % a.kv_heads, b = t / a.kv_heads;
  const T *q = static_cast<const T *>(a.q) + b * a.qs[0];
  const T *k = static_cast<const T *>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const T *v = static_cast<const T *>(a.v) + b * a.vs[0] + hk * a.vs[2];
  const int keys = entry_keys(a, b), tiles = (keys + kKeys - 1) / kKeys;
  const int tile0 = int(int64_t(tiles) * rank / csize), tile1 = int(int64_t(tiles) * (rank + 1) / csize);
  auto out_row = [&](int row) {
    return static_cast<T *>(a.out) + b * a.os[0] + row_offset(a, a.os, hk, row);
  };

  // A tile's keys and values, four elements of a row a piece: into registers, and
  // from there into shared memory once the last tile's readers are done.  Up to 64
  // columns the registers last to load a tile while the one before is computed.
  constexpr bool AHEAD = D <= 64;
  constexpr int PIECES = kKeys * D / 4 / 256, HELD = AHEAD ? PIECES : 1;
  float4 kr[HELD], vr[HELD];
  bool counts[HELD];
  auto piece = [&](int n, int &r, int &c) {
    const int e = (tid + n * 256) * 4;
    r = e / D, c = e % D;
  };
  auto fetch = [&](int tile, int n, float4 &kf, float4 &vf, bool &in) {
    int r, c;
    piece(n, r, c);
    const int j = tile * kKeys + r;
    in = j < keys && (!a.key_mask || a.key_mask[b * a.mask_stride + j] != 0);
    kf = vf = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (!in || c >= a.width) return;
    const T *kp = k + j * a.ks[1] + c, *vp = v + j * a.vs[1] + c;
    if (vec) {
      kf = load4(kp);
      vf = load4(vp);
    } else {
      kf = load_up_to4(kp, a.width - c);
      vf = load_up_to4(vp, a.width - c);
    }
  };
  auto put = [&](int n, const float4 &kf, const float4 &vf, bool in) {
    int r, c;
    piece(n, r, c);
    *reinterpret_cast<float4 *>(&sm.k[r][c]) = kf;
    *reinterpret_cast<float4 *>(&sm.v[r][c]) = vf;
    if (c == 0) sm.valid[r] = in;
  };
  if (AHEAD && tile0 < tile1) {
#pragma unroll
    for (int n = 0; n < HELD; ++n) fetch(tile0, n, kr[n], vr[n], counts[n]);
  }
#pragma unroll 4
  for (int e = tid * 4; e < S::rows * D; e += 1024) {
    const int r = e / D, c = e % D, row = r0 + r;
    float4 val = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (row < a.rows && c < a.width) {
      const T *qp = q + row_offset(a, a.qs, hk, row) + c;
      val = vec ? load4(qp) : load_up_to4(qp, a.width - c);
    }
    *reinterpret_cast<float4 *>(&sm.q[r][c]) = val;
  }
  float o[R][CPT] = {}, m[R], l[R] = {};
#pragma unroll
  for (int i = 0; i < R; ++i) m[i] = -INFINITY;

  for (int tile = tile0; tile < tile1; ++tile) {
    __syncthreads();  // the last tile's readers are done
    if (AHEAD) {
#pragma unroll
      for (int n = 0; n < HELD; ++n) put(n, kr[n], vr[n], counts[n]);
    } else {
#pragma unroll 4
      for (int n = 0; n < PIECES; ++n) {
        float4 kf, vf;
        bool in;
        fetch(tile, n, kf, vf, in);
        put(n, kf, vf, in);
      }
    }
    __syncthreads();
    if (AHEAD && tile + 1 < tile1) {
#pragma unroll
      for (int n = 0; n < HELD; ++n) fetch(tile + 1, n, kr[n], vr[n], counts[n]);
    }
    float s[R][4] = {};
#pragma unroll 4
    for (int c = 0; c < D; c += 4) {
      float4 qv[R], kv[4];
#pragma unroll
      for (int i = 0; i < R; ++i) qv[i] = *reinterpret_cast<const float4 *>(&sm.q[ty * R + i][c]);
#pragma unroll
      for (int j = 0; j < 4; ++j) kv[j] = *reinterpret_cast<const float4 *>(&sm.k[tx + 16 * j][c]);
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[i][j] = fmaf(qv[i].x, kv[j].x, s[i][j]);
          s[i][j] = fmaf(qv[i].y, kv[j].y, s[i][j]);
          s[i][j] = fmaf(qv[i].z, kv[j].z, s[i][j]);
          s[i][j] = fmaf(qv[i].w, kv[j].w, s[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float mx = m[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = sm.valid[tx + 16 * j] ? s[i][j] * a.scale_log2 : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int w = 8; w; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      const float use = mx == -INFINITY ? 0.0f : mx;
      const float shrink = exp2f(m[i] - use);
      m[i] = mx;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = exp2f(s[i][j] - use);
        sum += e;
        sm.p[ty * R + i][tx + 16 * j] = e;
      }
      l[i] = l[i] * shrink + sum;  // this thread's keys only; joined at the end
#pragma unroll
      for (int c = 0; c < CPT; ++c) o[i][c] *= shrink;
    }
    __syncwarp();  // a row's 16 threads are in one warp
#pragma unroll 2
    for (int j = 0; j < kKeys; j += 4) {
      float4 pv[R];
#pragma unroll
      for (int i = 0; i < R; ++i) pv[i] = *reinterpret_cast<const float4 *>(&sm.p[ty * R + i][j]);
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
#pragma unroll
        for (int c = 0; c < CPT; c += CW) {
          float vv[CW];
#pragma unroll
          for (int w = 0; w < CW; ++w) vv[w] = sm.v[j + jj][tx * CW + 16 * c + w];
#pragma unroll
          for (int i = 0; i < R; ++i) {
            const float e = jj == 0 ? pv[i].x : jj == 1 ? pv[i].y : jj == 2 ? pv[i].z : pv[i].w;
#pragma unroll
            for (int w = 0; w < CW; ++w) o[i][c + w] = fmaf(e, vv[w], o[i][c + w]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int w = 8; w; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
  if (csize == 1) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int row = r0 + ty * R + i;
      if (row >= a.rows) continue;
      const float inv = l[i] != 0.0f ? 1.0f / l[i] : 0.0f;
      T *out = out_row(row);
#pragma unroll
      for (int c = 0; c < CPT; ++c) {
        const int col = tx * CW + 16 * (c / CW * CW) + c % CW;
        if (col < a.width) out[col] = from_f32<T>(o[i][c] * inv);
      }
    }
    return;
  }
  __syncthreads();  // the last tile's readers are done: O takes the keys' place
  float *part = &sm.k[0][0];
#pragma unroll
  for (int i = 0; i < R; ++i) {
#pragma unroll
    for (int c = 0; c < CPT; ++c) part[(ty * R + i) * D + tx * CW + 16 * (c / CW * CW) + c % CW] = o[i][c];
    if (tx == 0) {
      sm.m[ty * R + i] = m[i];
      sm.l[ty * R + i] = l[i];
    }
  }
  cluster_sync();
  const int used = min(S::rows, a.rows - r0) * D;
  for (int e = rank * 256 + tid; e < used; e += csize * 256) {
    const int r = e / D, c = e % D;
    float mk[kMaxCluster], lk[kMaxCluster], ok[kMaxCluster], top = -INFINITY, acc = 0.0f, sum = 0.0f;
#pragma unroll
    for (int n = 0; n < kMaxCluster; ++n) {
      if (n >= csize) break;
      mk[n] = __uint_as_float(ld_cluster(map_rank(&sm.m[r], n)));
      lk[n] = __uint_as_float(ld_cluster(map_rank(&sm.l[r], n)));
      ok[n] = __uint_as_float(ld_cluster(map_rank(&part[e], n)));
      top = fmaxf(top, mk[n]);
    }
#pragma unroll
    for (int n = 0; n < kMaxCluster; ++n) {
      if (n >= csize) break;
      const float f = mk[n] == -INFINITY ? 0.0f : exp2f(mk[n] - top);
      acc = fmaf(ok[n], f, acc);
      sum = fmaf(lk[n], f, sum);
    }
    if (c < a.width) out_row(r0 + r)[c] = from_f32<T>(sum != 0.0f ? acc / sum : 0.0f);
  }
  cluster_sync();  // the peers have read this CTA's sums
}

template <class T, int D, int R>
int launch_simt(AttnArgs a, cudaStream_t s) {
  using S = SimtSmem<D, R>;
  a.row_tiles = int(ceil_div(a.rows, S::rows));
  const int64_t blocks = int64_t(a.row_tiles) * a.kv_heads * a.batch;
  if (const int rc = allow_smem<cross_simt_kernel<T, D, R>>(sizeof(S))) return rc;
  auto fours = [](const void *base, const int64_t (&st)[3]) {
    return reinterpret_cast<uintptr_t>(base) % (4 * sizeof(T)) == 0 && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0;
  };
  const bool vec = a.width % 4 == 0 && fours(a.q, a.qs) && fours(a.k, a.ks) && fours(a.v, a.vs);
  // Divide the keys while a CTA keeps a tile and the CTAs are fewer than two an SM.
  int csize = 1;
  while (csize < kMaxCluster && blocks * csize * 2 <= 2 * sm_count() && ceil_div(a.keys, kKeys) >= 2 * csize) csize *= 2;
  if (blocks * csize > INT32_MAX) return SPKV2_ERR_UNSUPPORTED;
  return cuda_status(launch_kernel(cross_simt_kernel<T, D, R>, unsigned(blocks * csize), 256u, sizeof(S), s, csize, a, csize, vec));
}

// Sixteen rows a tile where they are all there are, else 64.
template <class T, int D>
int launch_rows(const AttnArgs &a, cudaStream_t s) {
  return a.rows <= 16 ? launch_simt<T, D, 1>(a, s) : launch_simt<T, D, 4>(a, s);
}

}  // namespace

}  // namespace spkv2

using namespace spkv2;
using namespace spkv2::xf;

extern "C" int spkv2_cuda_cross_attention(const Spkv2CrossAttention *x, void *stream) {
  if (!x || x->batch < 0 || x->queries < 0 || x->keys < 0 || x->kv_heads < 1 || x->heads < 1 ||
      x->heads % x->kv_heads != 0 || x->width < 1)
    return -1;
  if (x->batch == 0 || x->queries == 0) return 0;
  if (!x->q || !x->out || (x->keys > 0 && (!x->k || !x->v))) return -1;
  for (int i = 0; i < 3; ++i)
    if (x->q_stride[i] < 0 || x->k_stride[i] < 0 || x->v_stride[i] < 0 || x->out_stride[i] < 0) return -1;
  const int64_t extent[3] = {x->batch, x->queries, x->heads};
  for (int i = 0; i < 3; ++i)
    if (extent[i] > 1 && x->out_stride[i] == 0) return -1;  // one place for several answers
  if (x->key_mask && x->mask_stride < 0) return -1;
  if (!isfinite(x->scale)) return -1;
  const int group = x->heads / x->kv_heads;
  if (!elem_bytes(x->dtype) || x->width > 256 || x->batch > INT32_MAX || x->keys > INT32_MAX - 1024 ||
      x->queries > (INT32_MAX - 1024) / group)
    return SPKV2_ERR_UNSUPPORTED;
  if (!on_bytes(elem_bytes(x->dtype), x->q, x->k, x->v, x->out) || !on_bytes(4, x->lengths)) return -1;
  AttnArgs a = {};
  a.q = x->q, a.k = x->k, a.v = x->v, a.out = x->out, a.lengths = x->lengths, a.key_mask = x->key_mask;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = x->q_stride[i], a.ks[i] = x->k_stride[i], a.vs[i] = x->v_stride[i], a.os[i] = x->out_stride[i];
  }
  a.mask_stride = x->mask_stride;
  a.batch = int(x->batch), a.queries = int(x->queries), a.keys = int(x->keys);
  a.kv_heads = x->kv_heads, a.group = group, a.width = x->width;
  a.rows = a.queries * group;
  a.group_div = FastDiv(uint32_t(group));
  a.scale_log2 = x->scale * 1.4426950408889634f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cross_tc_serves(a, x->dtype)) return a.rows <= 32 ? cross_step(a, x->dtype, s) : cross_tc(a, x->dtype, s);
  if (x->dtype == SPKV2_DTYPE_FP32 && a.width <= 128) return cross_f32(a, s);
  return by_type(x->dtype, [&](auto t) {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2) {
      if (a.width <= 32) return launch_rows<T, 32>(a, s);
      if (a.width <= 64) return launch_rows<T, 64>(a, s);
      if (a.width <= 128) return launch_rows<T, 128>(a, s);
    }
    return launch_rows<T, 256>(a, s);
  });
}
