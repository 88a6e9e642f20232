// Cross attention on the tensor cores (tcgen05, 16-bit types): many rows.
//
// A CTA owns two tiles of 128 rows (or one) of one entry and key head and passes
// over the keys in tiles of 128:
//   S = Q K^T   128 x 128 fp32 in TMEM, Q and K from shared memory (K-major)
//   P = exp2(S * scale * log2(e) - m), rounded to the inputs' type, written
//       back over S's columns in TMEM
//   O += P V    A = P from TMEM, V from shared memory as it lies in memory
//               (N-major)
// The two tiles alternate: while the softmax warps of one work, the tensor
// core runs the other's P V and its next Q K^T.  m is a row's running maximum,
// lagging: O and the sum l are rescaled only when the true maximum has risen
// by more than 2^8 over m, which bounds P by 256 and makes the rescaling (a
// TMEM round trip of the whole O tile) rare.  The result does not depend on m.
//
// Warps 0-3 (and 4-7): the softmax of tile 0 (and 1), a row per thread; then a
// warp for the TMA loads of K and V, one that issues the MMAs, and two that fill
// the group of four.  P is rounded once, as both operands of an MMA have one
// type; the sums stay in fp32.
#include "cross_attention.cuh"
#include "tcgen05.cuh"

namespace spkv2 {

namespace {

using namespace xf;
using namespace tc;

constexpr int kTile = 128;  // rows of a tile, keys of a step
constexpr int kHalf = kTile * 128;  // bytes of 64 columns of a tile

// TILES: row tiles of a CTA: two, with one CTA per SM, or one with two CTAs.
template <int D, int TILES>
struct Shape {
  static constexpr int halves = D / 64;
  static constexpr int tile_bytes = halves * kHalf;
  // Ring of K and V tiles: what fits beside Q (two CTAs share an SM's 227 KB).
  static constexpr int slots = TILES == 2 ? (D == 128 ? 4 : 6) : (D == 128 ? 2 : 4);
  static constexpr size_t smem = size_t(TILES + slots) * tile_bytes + 1024;
  static constexpr int soft_warps = 4 * TILES;
  static constexpr int threads = (soft_warps + 4) * 32;
  static constexpr uint32_t tmem_cols = TILES == 2 ? 512 : 256;
  // Registers of a thread: the launch gives every group of four warps the same
  // number (168 and 128, the most that fit); the softmax groups take what the
  // last group can spare.
  static constexpr int soft_regs = TILES == 2 ? 216 : 200, other_regs = TILES == 2 ? 72 : 56;
  static_assert(TILES * soft_regs + other_regs == (TILES + 1) * (TILES == 2 ? 168 : 128), "the launch's registers");
};

__device__ int g_cross_status;  // role code of the last bounded wait that gave up

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two floats in one 64-bit register, their fused multiply-add and sum in one
// instruction each.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(f32x2 v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
template <class T>
__device__ __forceinline__ void store8(T *to, const float (&v)[8]) {
  *reinterpret_cast<uint4 *>(to) =
      make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}

constexpr int kMaxCluster = 8;

// Which of the 32 W keys from j0 on count, a bit each; all lanes of a warp get
// the same.
template <int W>
__device__ __forceinline__ void key_bits(const AttnArgs &a, int b, int keys, int j0, int lane, uint32_t (&bits)[W]) {
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int j = j0 + w * 32 + lane;
    bool in = j < keys;
    if (in && a.key_mask) in = a.key_mask[b * a.mask_stride + j] != 0;
    bits[w] = __ballot_sync(0xffffffffu, in);
  }
}

template <class T, int D, int TILES>
__global__ void __launch_bounds__(Shape<D, TILES>::threads, 3 - TILES)
    cross_tc_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                    const __grid_constant__ CUtensorMap vmap, AttnArgs a, bool q_tma,
                    int k_heads_step, int k_batch_step, int v_heads_step, int v_batch_step, int csize) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using S = Shape<D, TILES>;
  constexpr int SOFT = S::soft_warps;
  uint8_t *ring = smem + TILES * S::tile_bytes;
  __shared__ uint64_t full_bar[S::slots], empty_bar[S::slots], q_bar, s_bar[TILES], p_bar[TILES][2], o_bar[TILES], done_bar;
  __shared__ float s_m[TILES * kTile], s_l[TILES * kTile];  // for the cluster's join
  __shared__ uint32_t tmem_holder;
  __shared__ volatile int abort_flag;
  int *status = &g_cross_status;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = csize > 1 ? int(cluster_rank()) : 0;
  int t = int(blockIdx.x) / csize;
  const int r0 = t % a.row_tiles * (TILES * kTile);
  t /= a.row_tiles;
  const int hk = t % a.kv_heads, b = t / a.kv_heads;
  const int tiles = TILES == 2 && a.rows - r0 > kTile ? 2 : 1;  // tiles with rows

  if (tid == 0) {
    for (int s = 0; s < S::slots; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(&q_bar, q_tma ? 1 : SOFT);
    mbar_init(&done_bar, 1);
    for (int i = 0; i < TILES; ++i) {
      mbar_init(&s_bar[i], 1);
      mbar_init(&p_bar[i][0], 4);
      mbar_init(&p_bar[i][1], 4);
      mbar_init(&o_bar[i], 1);
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == SOFT + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_holder)),
                 "r"(S::tmem_cols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;
  pdl_launch_dependents();
  pdl_wait();

  const int keys = counted_keys<S::threads>(a, b, tid);
  const int all_steps = (keys + kTile - 1) / kTile;  // divided among the CTAs of the cluster
  const int step0 = int(int64_t(all_steps) * rank / csize), steps = int(int64_t(all_steps) * (rank + 1) / csize) - step0;
  // TMEM columns: scores (and P) of tile i at 128 i, sums of tile i behind them.
  auto s_col = [&](int i) { return tmem + uint32_t(i * kTile); };
  auto o_col = [&](int i) { return tmem + uint32_t(TILES * kTile + i * D); };

  // A CTA without steps loads no Q: it writes its zeros over Q's place without a wait,
  // for peers that multiply them by 0, and what landed there later would reach them.
  float *part = reinterpret_cast<float *>(smem);  // O for the cluster's join, [tile][column][row], over Q, K and V
  auto out_row = [&](int row) {
    return static_cast<T *>(a.out) + b * a.os[0] + row_offset(a, a.os, hk, row);
  };

  if (warp < SOFT) {
    // ---------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::soft_regs));
    const int i = warp >> 2, quarter = warp & 3;
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    if (!q_tma && steps > 0) {  // this warp's 32 rows of Q, swizzled for the MMA; 16-byte chunks
      const T *q = static_cast<const T *>(a.q) + b * a.qs[0];
      constexpr int CH = D / 8, RPI = 32 / CH;  // chunks of a row, rows of an iteration
      const int c = lane % CH;
      constexpr int B = 8;  // loads in flight
#pragma unroll
      for (int k0 = 0; k0 < 32 / RPI; k0 += B) {
        uint4 v[B];
#pragma unroll
        for (int k = 0; k < B; ++k) {
          const int row = r0 + i * kTile + quarter * 32 + (k0 + k) * RPI + lane / CH;
          v[k] = make_uint4(0, 0, 0, 0);
          if (row < a.rows && c * 8 < a.width)
            v[k] = __ldg(reinterpret_cast<const uint4 *>(q + row_offset(a, a.qs, hk, row) + c * 8));
        }
#pragma unroll
        for (int k = 0; k < B; ++k) {
          const int rr = quarter * 32 + (k0 + k) * RPI + lane / CH;
          *reinterpret_cast<uint4 *>(smem + i * S::tile_bytes + (c >> 3) * kHalf + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = v[k];
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_bar);
    }
    const int r = quarter * 32 + lane, row = r0 + i * kTile + r;
    float m = -INFINITY, l = 0.0f;
    bool ok = i < tiles;
    for (int j = 0; j < steps && ok; ++j) {
      const int j0 = (step0 + j) * kTile;
      const bool masked = a.key_mask || j0 + kTile > keys;
      uint32_t bits[kTile / 32], all = ~0u;
      if (masked) key_bits<kTile / 32>(a, b, keys, j0, lane, bits);
      ok = __all_sync(0xffffffffu, mbar_wait(&s_bar[i], j & 1, &abort_flag, status, 4));
      if (!ok) break;
      tc_fence_after();
      float s[kTile];
#pragma unroll
      for (int c = 0; c < kTile; c += 32) {
        uint32_t v[32];
        tmem_ld32_async(s_col(i) + lanes + uint32_t(c), v);
#pragma unroll
        for (int k = 0; k < 32; ++k) s[c + k] = __uint_as_float(v[k]);
      }
      tmem_wait_ld();
#pragma unroll
      for (int k = 0; k < kTile; ++k) asm volatile("" : "+f"(s[k]));  // not read before the wait
      if (masked) {
#pragma unroll
        for (int w = 0; w < kTile / 32; ++w) all &= bits[w];
      }
      if (all != ~0u) {
#pragma unroll
        for (int k = 0; k < kTile; ++k) s[k] = (bits[k >> 5] >> (k & 31)) & 1 ? s[k] : -INFINITY;
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int k = 0; k < kTile; k += 2) mx[(k >> 1) & 3] = fmaxf(mx[(k >> 1) & 3], fmaxf(s[k], s[k + 1]));
      float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      top *= a.scale_log2;
      const bool rise = top > m + 8.0f;  // from m = -inf: any score
      if (__any_sync(0xffffffffu, rise)) {
        const float shrink = rise ? ex2(m - top) : 1.0f;  // 0 from m = -inf
        if (rise) m = top;
        l *= shrink;
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t v[32];
            tmem_ld32(o_col(i) + lanes + uint32_t(c), v);
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * shrink);
            tmem_st32(o_col(i) + lanes + uint32_t(c), v);
          }
        }
      }
      const float use = m == -INFINITY ? 0.0f : m;
      const f32x2 factor = pair(a.scale_log2, a.scale_log2), shift = pair(-use, -use);
      f32x2 sum[2] = {pair(0.0f, 0.0f), pair(0.0f, 0.0f)};
#pragma unroll
      for (int c = 0; c < kTile; c += 64) {
        uint32_t p[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const f32x2 x = fma2(pair(s[c + 2 * k], s[c + 2 * k + 1]), factor, shift);
          float e0, e1;
          unpair(x, e0, e1);
          e0 = ex2(e0);
          e1 = ex2(e1);
          sum[k & 1] = add2(sum[k & 1], pair(e0, e1));
          p[k] = pack2<T>(e0, e1);
        }
        tmem_st32(s_col(i) + lanes + uint32_t(c / 2), p);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_bar[i][c / 64]);  // the MMAs of these 64 keys may start
      }
      float l0, l1;
      unpair(add2(sum[0], sum[1]), l0, l1);
      l += l0 + l1;
    }
    // ---------------------------------------------------------- result
    if (i < tiles) {
      if (steps > 0 && ok) ok = __all_sync(0xffffffffu, mbar_wait(&o_bar[i], 0, &abort_flag, status, 4));
      tc_fence_after();
      if (csize > 1) {
        s_m[i * kTile + r] = m;
        s_l[i * kTile + r] = l;
      }
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;
      T *out = out_row(row);
      if (ok) {
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t v[32] = {};
          if (steps > 0) tmem_ld32(o_col(i) + lanes + uint32_t(c), v);
          if (csize > 1) {
#pragma unroll
            for (int k = 0; k < 32; ++k) part[(i * D + c + k) * kTile + r] = __uint_as_float(v[k]);
          } else if (row < a.rows) {
#pragma unroll
            for (int k = 0; k < 32; k += 8)
              if (c + k < a.width) {
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = __uint_as_float(v[k + e]) * inv;
                store8<T>(out + c + k, w);
              }
          }
        }
      }
    }
  } else if (warp != SOFT + 1) {
    // ---------------------------------------------------------- K and V tiles
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::other_regs));
    if (warp == SOFT && elect_one()) {
      if (q_tma && steps > 0) {
        mbar_arrive_expect_tx(&q_bar, uint32_t(tiles * S::tile_bytes));
        for (int i = 0; i < tiles; ++i)
          for (int h = 0; h < S::halves; ++h)
            tma_load_4d(smem + i * S::tile_bytes + h * kHalf, &qmap, h * 64, hk * a.group, (r0 + i * kTile) / a.group, b, &q_bar);
      }
      int it = 0;
      bool ok = true;
      for (int j = 0; j < steps && ok; ++j) {
        for (int kv = 0; kv < 2; ++kv, ++it) {
          const int slot = it % S::slots;
          ok = mbar_wait(&empty_bar[slot], ((it / S::slots) & 1) ^ 1, &abort_flag, status, 2);
          if (!ok) break;
          mbar_arrive_expect_tx(&full_bar[slot], S::tile_bytes);
          for (int h = 0; h < S::halves; ++h)
            tma_load_4d(ring + slot * S::tile_bytes + h * kHalf, kv ? &vmap : &kmap, h * 64, (step0 + j) * kTile,
                        hk * (kv ? v_heads_step : k_heads_step), b * (kv ? v_batch_step : k_batch_step), &full_bar[slot]);
        }
      }
      // What was issued has landed before shared memory goes away.
      if (q_tma && steps > 0) {
        const long long t0 = clock64();
        while (!mbar_try_wait(&q_bar, 0) && clock64() - t0 < kWaitCycles) {
        }
      }
      for (int k = it > S::slots ? it - S::slots : 0; k < it; ++k) {
        const long long t0 = clock64();
        while (!mbar_try_wait(&full_bar[k % S::slots], (k / S::slots) & 1) && clock64() - t0 < kWaitCycles) {
        }
      }
    }
  } else {
    // ---------------------------------------------------------- MMA
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::other_regs));
    constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t id_s = (1u << 4) | (kType << 7) | (kType << 10) | (uint32_t(kTile >> 3) << 17) | (uint32_t(kTile >> 4) << 24);
    constexpr uint32_t id_o = (1u << 4) | (kType << 7) | (kType << 10) | (1u << 16) | (uint32_t(D >> 3) << 17) | (uint32_t(kTile >> 4) << 24);
    auto landed = [&](int it) {
      return __all_sync(0xffffffffu, mbar_wait(&full_bar[it % S::slots], (it / S::slots) & 1, &abort_flag, status, 3));
    };
    auto scores = [&](int i, int slot) {  // S_i = Q_i K^T
      const uint64_t dq = smem_desc(smem + i * S::tile_bytes), dk = smem_desc(ring + slot * S::tile_bytes);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint64_t off = uint64_t((k >> 2) * kHalf + (k & 3) * 32) >> 4;
        mma_f16(s_col(i), dq + off, dk + off, id_s, k > 0 ? 1u : 0u);
      }
    };
    bool ok = steps > 0 && __all_sync(0xffffffffu, mbar_wait(&q_bar, 0, &abort_flag, status, 3));
    if (ok) {
      ok = landed(0);
      if (ok && elect_one()) {
        tc_fence_after();
        for (int i = 0; i < tiles; ++i) {
          scores(i, 0);
          mma_commit(&s_bar[i]);
        }
        mma_commit(&empty_bar[0]);
      }
    }
    for (int j = 0; j < steps && ok; ++j) {
      const int vs = (2 * j + 1) % S::slots, kn = (2 * j + 2) % S::slots;
      uint32_t bits[4] = {~0u, ~0u, ~0u, ~0u};
      const int j0 = (step0 + j) * kTile;
      if (a.key_mask || j0 + kTile > keys) key_bits<4>(a, b, keys, j0, lane, bits);
      ok = landed(2 * j + 1);
      if (!ok) break;
      if ((bits[0] & bits[1] & bits[2] & bits[3]) != 0xffffffffu) {
        // Values that do not count meet p = 0 in the MMA: they must be finite.
        constexpr int CH = S::halves * 8, KPI = 32 / CH;  // 16-byte chunks of a key, keys of an iteration
        const int c = lane % CH;
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int k = lane / CH; k < 32; k += KPI)
            if (!((bits[w] >> k) & 1))
              *reinterpret_cast<uint4 *>(ring + vs * S::tile_bytes + (c >> 3) * kHalf + (w * 32 + k) * 128 + (c & 7) * 16) =
                  make_uint4(0, 0, 0, 0);
        fence_proxy_async();
        __syncwarp();
      }
      for (int i = 0; i < tiles && ok; ++i) {
        const uint64_t dv = smem_desc_mn(ring + vs * S::tile_bytes, kHalf);
        for (int half = 0; half < 2 && ok; ++half) {
          ok = __all_sync(0xffffffffu, mbar_wait(&p_bar[i][half], j & 1, &abort_flag, status, 7));
          if (ok && elect_one()) {
            tc_fence_after();
#pragma unroll
            for (int k = half * 4; k < half * 4 + 4; ++k)  // 16 keys: 8 columns of P, 16 rows of V
              mma_f16_ta(o_col(i), s_col(i) + uint32_t(k * 8), dv + (uint64_t(k * 16 * 128) >> 4), id_o, (j | k) ? 1u : 0u);
          }
        }
        if (ok && i == 0 && j + 1 < steps) ok = landed(2 * j + 2);
        if (!ok) break;
        if (elect_one()) {
          if (i == tiles - 1) mma_commit(&empty_bar[vs]);
          if (j + 1 < steps) {
            scores(i, kn);
            mma_commit(&s_bar[i]);
            if (i == tiles - 1) mma_commit(&empty_bar[kn]);
          } else {
            mma_commit(&o_bar[i]);
          }
        }
        __syncwarp();
      }
    }
    if (lane == 0) {  // every issued MMA has finished before TMEM is freed, also after a wait that gave up
      mma_commit(&done_bar);
      const long long t0 = clock64();
      while (!mbar_try_wait(&done_bar, 0) && clock64() - t0 < kWaitCycles) {
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncwarp();
  if (csize > 1) {
    // ------------------------------------------------------------ join
    // Each CTA takes kTile / csize rows of each tile; a row's D columns are
    // divided among csize threads.  CTA order, so the same bits every time.
    cluster_sync();
    if (warp < SOFT && (warp >> 2) < tiles && !abort_flag) {
      const int i = warp >> 2, rows = kTile / csize, w = tid & (kTile - 1);
      const int r = rank * rows + w % rows, cols = D / csize, c0 = w / rows * cols, row = r0 + i * kTile + r;
      float f[kMaxCluster], top = -INFINITY, sum = 0.0f;
      for (int k = 0; k < csize; ++k) top = fmaxf(top, __uint_as_float(ld_cluster(map_rank(&s_m[i * kTile + r], k))));
#pragma unroll
      for (int k = 0; k < kMaxCluster; ++k) {
        f[k] = 0.0f;
        if (k >= csize) continue;
        const float mk = __uint_as_float(ld_cluster(map_rank(&s_m[i * kTile + r], k)));
        f[k] = mk == -INFINITY ? 0.0f : ex2(mk - top);
        sum += __uint_as_float(ld_cluster(map_rank(&s_l[i * kTile + r], k))) * f[k];
      }
      const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
      if (row < a.rows) {
        T *out = out_row(row);
        for (int c = c0; c < c0 + cols && c < a.width; c += 8) {
          float acc[8] = {};
#pragma unroll
          for (int k = 0; k < kMaxCluster; ++k) {
            if (k >= csize) continue;
            const uint32_t from = map_rank(&part[(i * D + c) * kTile + r], k);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = fmaf(__uint_as_float(ld_cluster(from + e * kTile * 4)), f[k], acc[e]);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] *= inv;
          store8<T>(out + c, acc);
        }
      }
    }
    __syncwarp();
    cluster_sync();  // the peers have read this CTA's sums
  } else {
    __syncthreads();
  }
  if (warp == SOFT + 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::tmem_cols));
  }
}

// Q as {width, head, token, entry}: where the heads of a group divide the 128 rows
// of a tile, the tile is a box of group heads x 128 / group tokens, in the order of
// the rows.
bool encode_q(CUtensorMap *map, const AttnArgs &a) {
  const int64_t heads = int64_t(a.kv_heads) * a.group, most = int64_t(1) << 38;
  if (kTile % a.group != 0) return false;
  if ((heads > 1 && a.qs[2] <= 0) || (a.queries > 1 && a.qs[1] <= 0) || (a.batch > 1 && a.qs[0] <= 0)) return false;
  if (a.qs[0] >= most || a.qs[1] >= most || a.qs[2] >= most) return false;
  const cuuint64_t any = (cuuint64_t(a.width) * 2 + 15) / 16 * 16;
  const cuuint64_t dims[4] = {cuuint64_t(a.width), cuuint64_t(heads), cuuint64_t(a.queries), cuuint64_t(a.batch)};
  const cuuint64_t strides[3] = {heads > 1 ? cuuint64_t(a.qs[2]) * 2 : any, a.queries > 1 ? cuuint64_t(a.qs[1]) * 2 : any,
                                 a.batch > 1 ? cuuint64_t(a.qs[0]) * 2 : any};
  const cuuint32_t box[4] = {64, cuuint32_t(a.group), cuuint32_t(kTile / a.group), 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void *>(a.q), dims, strides, box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int D, int TILES>
int launch(AttnArgs a, cudaStream_t s) {
  using S = Shape<D, TILES>;
  static_assert(size_t(TILES) * D * kTile * 4 <= S::smem - 1024, "the join's sums reuse the operands' memory");
  a.row_tiles = int(ceil_div(a.rows, TILES * kTile));
  const int64_t blocks = int64_t(a.row_tiles) * a.kv_heads * a.batch;
  if (const int rc = allow_smem<cross_tc_kernel<T, D, TILES>>(S::smem)) return rc;
  KvMap k, v;
  if (!encode_kv(&k, a, a.k, a.ks, kTile) || !encode_kv(&v, a, a.v, a.vs, kTile)) return SPKV2_ERR_CUDA;
  CUtensorMap qmap = {};
  const bool q_tma = encode_q(&qmap, a);
  // Too few tiles for the SMs: divide the keys, down to two steps a CTA.
  int csize = 1;
  if (TILES == 1)
    while (csize < kMaxCluster && blocks * csize * 2 <= 2 * sm_count() && ceil_div(a.keys, kTile) >= 4 * csize) csize *= 2;
  if (blocks * csize > INT32_MAX) return SPKV2_ERR_UNSUPPORTED;
  return cuda_status(launch_kernel(cross_tc_kernel<T, D, TILES>, unsigned(blocks * csize), S::threads, S::smem, s, csize, qmap,
                                   k.map, v.map, a, q_tma, k.heads_step, k.batch_step, v.heads_step, v.batch_step, csize));
}

template <class T, int D>
int launch_tiles(const AttnArgs &a, cudaStream_t s) {
  // Two tiles for long passes over the keys that fill the SMs; else two CTAs an SM,
  // so that one works while the other starts or ends (width 128, 16 x 16 heads x
  // 1024 rows: 4096 keys 455 us against 492, 1024 keys 177 us against 167, 256 keys
  // 98 against 82).
  const int64_t blocks = ceil_div(a.rows, 2 * kTile) * a.kv_heads * a.batch;
  return a.rows > kTile && blocks >= sm_count() && a.keys >= 2048 ? launch<T, D, 2>(a, s) : launch<T, D, 1>(a, s);
}

bool rows_aligned(const void *base, const int64_t (&st)[3]) {
  return aligned16(base) && st[0] % 8 == 0 && st[1] % 8 == 0 && st[2] % 8 == 0;
}

// Strides that a tensor map can hold.
bool mappable(const AttnArgs &a, const int64_t (&st)[3]) {
  const int64_t most = int64_t(1) << 38;
  return (a.keys == 1 || st[1] > 0) && st[0] < most && st[1] < most && st[2] < most;
}

}  // namespace

bool cross_tc_serves(const AttnArgs &a, int32_t dtype) {
  return elem_bytes(dtype) == 2 && a.width <= 128 && a.width % 8 == 0 && a.keys > 0 && a.scale_log2 > 0.0f && encode_fn() &&
         rows_aligned(a.q, a.qs) && rows_aligned(a.k, a.ks) && rows_aligned(a.v, a.vs) && rows_aligned(a.out, a.os) &&
         mappable(a, a.ks) && mappable(a, a.vs);
}

int cross_tc(const AttnArgs &a, int32_t dtype, cudaStream_t s) {
  if (dtype == SPKV2_DTYPE_FP16) return a.width <= 64 ? launch_tiles<__half, 64>(a, s) : launch_tiles<__half, 128>(a, s);
  return a.width <= 64 ? launch_tiles<__nv_bfloat16, 64>(a, s) : launch_tiles<__nv_bfloat16, 128>(a, s);
}

int cross_tc_status(int *code) { return take_status(g_cross_status, code); }

}  // namespace spkv2
