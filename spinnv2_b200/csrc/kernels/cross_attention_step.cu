// Cross attention for few rows (a decoding step): 16-bit types, at most 32 rows
// (queries x heads of a group) for a key head.
//
// Bound by reading K and V once.  Each warp streams its own chunks of 16 keys
// through its own TMA ring and keeps its own m, l and O, so warps never wait
// for one another until the keys are through; the 16-row MMA fragments
// (mma.sync m16n8k16) are padding for one query, but a chunk's 8 KB costs more
// time in HBM than in them.  The scores' accumulator layout is the layout of
// the next MMA's A operand, so P stays in registers.
//
// The keys of one entry and key head are divided among the CTAs of a cluster
// and, chunk by chunk, among a CTA's warps.  At the end the warps' (m, l, O) are
// joined in shared memory, then the CTAs' through distributed shared memory, in
// a fixed order.  As in the other kernels m lags the maximum by at most 2^8.
#include "cross_attention.cuh"
#include "tcgen05.cuh"

namespace spkv2 {

namespace {

using namespace xf;
using namespace tc;

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kChunk = 16;  // keys

template <int D, int MT>
struct Step {
  static constexpr int halves = D / 64;
  static constexpr int half_bytes = kChunk * 128;            // 64 columns of a chunk
  static constexpr int stage_bytes = 2 * halves * half_bytes;  // K and V
  static constexpr int stages = D == 128 ? 3 : 6;
  static constexpr int part_bytes = MT * 16 * D * 4;  // a warp's O at the end, over its ring
  // A warp's ring, for a warp with `chunks` chunks: short ones leave room for more
  // CTAs on the SM.
  static constexpr int ring_bytes(int chunks) {
    const int ring = (chunks < stages ? chunks : stages) * stage_bytes;
    return ring < part_bytes ? part_bytes : ring;
  }
};

__device__ int g_step_status;  // role code of the last bounded wait that gave up

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <class T>
struct Mma;
template <>
struct Mma<__half> {
  static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
};
template <>
struct Mma<__nv_bfloat16> {
  static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
};

template <class T, int D, int MT>
__global__ void __launch_bounds__(kThreads, MT == 1 ? (D == 64 ? 4 : 3) : 2)
    cross_step_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, AttnArgs a,
                      int k_heads_step, int k_batch_step, int v_heads_step, int v_batch_step, int csize, int ring_bytes) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using S = Step<D, MT>;
  constexpr int R = MT * 16;
  __shared__ uint64_t full_bar[kWarps][S::stages];
  __shared__ float s_m[kWarps][R], s_l[kWarps][R];
  __shared__ float c_m[R], c_l[R];
  __shared__ volatile int abort_flag;
  int *status = &g_step_status;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = csize > 1 ? int(cluster_rank()) : 0;
  const int item = int(blockIdx.x) / csize;
  const int hk = item % a.kv_heads, b = item / a.kv_heads;
  uint8_t *ring = smem + warp * ring_bytes;
  if (lane == 0)
    for (int s = 0; s < S::stages; ++s) mbar_init(&full_bar[warp][s], 1);
  if (tid == 0) abort_flag = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();

  const int keys = counted_keys<kThreads>(a, b, tid);
  const int chunks = (keys + kChunk - 1) / kChunk;
  const int first = int(int64_t(chunks) * rank / csize) + warp;
  const int last = int(int64_t(chunks) * (rank + 1) / csize);  // this warp's chunks: first, first + 4, .. below last
  const int mine = last > first ? (last - first + kWarps - 1) / kWarps : 0;
  auto load = [&](int n) {  // one lane: this warp's n-th chunk
    const int slot = n % S::stages, j0 = (first + n * kWarps) * kChunk;
    uint8_t *st = ring + slot * S::stage_bytes;
    mbar_arrive_expect_tx(&full_bar[warp][slot], S::stage_bytes);
#pragma unroll
    for (int h = 0; h < S::halves; ++h) {
      tma_load_4d(st + h * S::half_bytes, &kmap, h * 64, j0, hk * k_heads_step, b * k_batch_step, &full_bar[warp][slot]);
      tma_load_4d(st + (S::halves + h) * S::half_bytes, &vmap, h * 64, j0, hk * v_heads_step, b * v_batch_step,
                  &full_bar[warp][slot]);
    }
  };
  if (elect_one())
    for (int n = 0; n < S::stages && n < mine; ++n) load(n);
  __syncwarp();

  // Fragments: a lane holds rows g and g + 8 of a 16-row tile, columns 2 t,
  // 2 t + 1 (and + 8) of each 16.
  const int g = lane >> 2, t = lane & 3;
  uint32_t qf[MT][D / 16][4];
  {
    const T *q = static_cast<const T *>(a.q) + b * a.qs[0];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = mt * 16 + half * 8 + g;
        const T *src = q + row_offset(a, a.qs, hk, row);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int c = k * 16 + e * 8 + 2 * t;
            qf[mt][k][e * 2 + half] = row < a.rows && c < a.width ? __ldg(reinterpret_cast<const uint32_t *>(src + c)) : 0u;
          }
      }
  }
  float o[MT][D / 8][4] = {};
  float m[MT][2], l[MT][2] = {};
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) m[mt][0] = m[mt][1] = -INFINITY;

  const uint32_t ring_addr = smem_u32(ring);
  int n = 0;
  for (; n < mine; ++n) {
    const int slot = n % S::stages, j0 = (first + n * kWarps) * kChunk;
    uint32_t bits = 0xffffu;
    if (a.key_mask || j0 + kChunk > keys) {
      const int j = j0 + (lane & 15);
      bool in = j < keys;
      if (in && a.key_mask) in = a.key_mask[b * a.mask_stride + j] != 0;
      bits = __ballot_sync(0xffffffffu, in) & 0xffffu;
    }
    if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[warp][slot], (n / S::stages) & 1, &abort_flag, status, 2))) break;
    const uint32_t ks = ring_addr + slot * S::stage_bytes, vs = ks + S::halves * S::half_bytes;
    if (bits != 0xffffu) {
      // Values that do not count meet p = 0 in the MMA: they must be finite.
      for (uint32_t off = ~bits & 0xffffu; off; off &= off - 1)
        if (lane < S::halves * 8)
          *reinterpret_cast<uint4 *>(ring + slot * S::stage_bytes + (S::halves + (lane >> 3)) * S::half_bytes +
                                     (__ffs(off) - 1) * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
      __syncwarp();
    }
    // Scores of 16 keys: two 8-key accumulators a row tile.
    float s[MT][2][4] = {};
    {
      const int r = (lane & 7) + ((lane >> 4) << 3), cs = (lane >> 3) & 1;  // key row, 8-column half of this lane's address
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t kf[4];
        const int c = (k & 3) * 2 + cs;
        ldmatrix4(ks + (k >> 2) * S::half_bytes + r * 128 + ((c ^ (r & 7)) << 4), kf);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          Mma<T>::run(s[mt][0], qf[mt][k], kf[0], kf[1]);
          Mma<T>::run(s[mt][1], qf[mt][k], kf[2], kf[3]);
        }
      }
    }
    if (bits != 0xffffu) {
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!((bits >> (nt * 8 + 2 * t + (e & 1))) & 1))
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) s[mt][nt][e] = -INFINITY;
    }
    uint32_t pf[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float top[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float x = fmaxf(fmaxf(s[mt][0][2 * half], s[mt][0][2 * half + 1]), fmaxf(s[mt][1][2 * half], s[mt][1][2 * half + 1]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        top[half] = x * a.scale_log2;
      }
      const bool rise0 = top[0] > m[mt][0] + 8.0f, rise1 = top[1] > m[mt][1] + 8.0f;
      if (__any_sync(0xffffffffu, rise0 || rise1)) {
        const float f0 = rise0 ? ex2(m[mt][0] - top[0]) : 1.0f, f1 = rise1 ? ex2(m[mt][1] - top[1]) : 1.0f;
        if (rise0) m[mt][0] = top[0];
        if (rise1) m[mt][1] = top[1];
        l[mt][0] *= f0;
        l[mt][1] *= f1;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          o[mt][c][0] *= f0;
          o[mt][c][1] *= f0;
          o[mt][c][2] *= f1;
          o[mt][c][3] *= f1;
        }
      }
      const float u0 = m[mt][0] == -INFINITY ? 0.0f : m[mt][0], u1 = m[mt][1] == -INFINITY ? 0.0f : m[mt][1];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const float p0 = ex2(fmaf(s[mt][nt][0], a.scale_log2, -u0)), p1 = ex2(fmaf(s[mt][nt][1], a.scale_log2, -u0));
        const float p2 = ex2(fmaf(s[mt][nt][2], a.scale_log2, -u1)), p3 = ex2(fmaf(s[mt][nt][3], a.scale_log2, -u1));
        l[mt][0] += p0 + p1;
        l[mt][1] += p2 + p3;
        pf[mt][nt * 2] = Mma<T>::pack(p0, p1);
        pf[mt][nt * 2 + 1] = Mma<T>::pack(p2, p3);
      }
    }
    {
      const int r = lane & 15, cs = lane >> 4;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {  // 16 columns of V
        uint32_t vf[4];
        const int c = (k & 3) * 2 + cs;
        ldmatrix4_t(vs + (k >> 2) * S::half_bytes + r * 128 + ((c ^ (r & 7)) << 4), vf);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          Mma<T>::run(o[mt][2 * k], pf[mt], vf[0], vf[1]);
          Mma<T>::run(o[mt][2 * k + 1], pf[mt], vf[2], vf[3]);
        }
      }
    }
    if (bits != 0xffffu) fence_proxy_async();  // the zeros above precede the next load into this slot
    __syncwarp();
    if (n + S::stages < mine && elect_one()) load(n + S::stages);
  }
  if (n < mine && lane == 0) {  // giving up: what was issued lands (bounded) before shared memory goes away
    for (int k = n; k < n + S::stages && k < mine; ++k) {
      const long long t0 = clock64();
      while (!mbar_try_wait(&full_bar[warp][k % S::stages], (k / S::stages) & 1) && clock64() - t0 < kWaitCycles) {
      }
    }
  }
  // The warps' sums, each over its own ring.
  float *part = reinterpret_cast<float *>(ring);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float x = l[mt][half];
      x += __shfl_xor_sync(0xffffffffu, x, 1);
      x += __shfl_xor_sync(0xffffffffu, x, 2);
      if (t == 0) {
        s_m[warp][mt * 16 + half * 8 + g] = m[mt][half];
        s_l[warp][mt * 16 + half * 8 + g] = x;
      }
#pragma unroll
      for (int c = 0; c < D / 8; ++c)
        *reinterpret_cast<float2 *>(part + (mt * 16 + half * 8 + g) * D + c * 8 + 2 * t) =
            make_float2(o[mt][c][2 * half], o[mt][c][2 * half + 1]);
    }
  }
  __syncthreads();
  // Joined in warp order; into warp 0's place.
  const int used = min(R, a.rows) * D;
  auto weight = [](float mw, float top) { return mw == -INFINITY ? 0.0f : ex2(mw - top); };
  for (int e = tid; e < used; e += kThreads) {
    const int r = e / D;
    const float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
    float acc = 0.0f, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = weight(s_m[w][r], top);
      // A warp without keys has sums of 0; one whose maximum is not finite has NaN.
      acc += reinterpret_cast<float *>(smem + w * ring_bytes)[e] * f;
      sum += s_l[w][r] * f;
    }
    if (csize == 1) {
      const int c = e % D;
      if (c < a.width && !abort_flag) {
        static_cast<T *>(a.out)[b * a.os[0] + row_offset(a, a.os, hk, r) + c] = from_f32<T>(sum != 0.0f ? acc / sum : 0.0f);
      }
    } else {
      reinterpret_cast<float *>(smem)[e] = acc;
      if (e % D == 0) {
        c_m[r] = top;
        c_l[r] = sum;
      }
    }
  }
  if (csize > 1) {
    __syncwarp();
    cluster_sync();
    for (int e = rank * kThreads + tid; e < used; e += csize * kThreads) {
      const int r = e / D, c = e % D;
      float top = -INFINITY;
      for (int k = 0; k < csize; ++k) top = fmaxf(top, __uint_as_float(ld_cluster(map_rank(&c_m[r], k))));
      float acc = 0.0f, sum = 0.0f;
      for (int k = 0; k < csize; ++k) {
        const float f = weight(__uint_as_float(ld_cluster(map_rank(&c_m[r], k))), top);
        acc += __uint_as_float(ld_cluster(map_rank(smem + e * 4, k))) * f;
        sum += __uint_as_float(ld_cluster(map_rank(&c_l[r], k))) * f;
      }
      if (c < a.width && !abort_flag) {
        static_cast<T *>(a.out)[b * a.os[0] + row_offset(a, a.os, hk, r) + c] = from_f32<T>(sum != 0.0f ? acc / sum : 0.0f);
      }
    }
    __syncwarp();
    cluster_sync();  // the peers have read this CTA's sums
  }
}

template <class T, int D, int MT>
int launch(const AttnArgs &a, cudaStream_t s) {
  using S = Step<D, MT>;
  if (const int rc = allow_smem<cross_step_kernel<T, D, MT>>(size_t(kWarps) * S::ring_bytes(S::stages) + 1024)) return rc;
  KvMap k, v;
  if (!encode_kv(&k, a, a.k, a.ks, kChunk) || !encode_kv(&v, a, a.v, a.vs, kChunk)) return SPKV2_ERR_CUDA;
  const int64_t items = int64_t(a.batch) * a.kv_heads;
  auto warp_chunks = [&](int c) { return int(ceil_div(ceil_div(a.keys, kChunk), int64_t(c) * kWarps)); };
  // Divide the keys while the CTAs are at most two an SM and a warp keeps more
  // than two chunks.  More CTAs than that only queue, and a cluster costs its CTAs
  // a start together and two barriers: 512 entries and heads of 500 keys (width
  // 64) take 21 us undivided, 24 by two, 27 by four; 16 of 4096 keys 34 us, 19,
  // 12, and 9 by eight.
  int csize = 1;
  while (csize < 8 && items * csize <= sm_count() && warp_chunks(csize) > 2) csize *= 2;
  if (items * csize > INT32_MAX) return SPKV2_ERR_UNSUPPORTED;
  const int ring = S::ring_bytes(warp_chunks(csize));
  return cuda_status(launch_kernel(cross_step_kernel<T, D, MT>, unsigned(items * csize), kThreads, size_t(kWarps) * ring + 1024, s,
                                   csize, k.map, v.map, a, k.heads_step, k.batch_step, v.heads_step, v.batch_step, csize, ring));
}

template <class T>
int launch_type(const AttnArgs &a, cudaStream_t s) {
  if (a.width <= 64) return a.rows <= 16 ? launch<T, 64, 1>(a, s) : launch<T, 64, 2>(a, s);
  return a.rows <= 16 ? launch<T, 128, 1>(a, s) : launch<T, 128, 2>(a, s);
}

}  // namespace

int cross_step(const AttnArgs &a, int32_t dtype, cudaStream_t s) {
  return dtype == SPKV2_DTYPE_FP16 ? launch_type<__half>(a, s) : launch_type<__nv_bfloat16>(a, s);
}

int cross_step_status(int *code) { return take_status(g_step_status, code); }

}  // namespace spkv2
