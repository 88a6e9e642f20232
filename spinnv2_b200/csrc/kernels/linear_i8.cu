// int8 x int8 product with a scale for each token and each channel:
//
//   y[i, j] = act(float(sum_k a[i, k] w[j, k]) * a_scale[i] * w_scale[j] + bias[j])
//
// The sum is exact in int32 (|a|, |w| <= 128 and k <= 131071).
#include "tcgen05.cuh"
#include "transformer.cuh"

namespace spkv2 {

namespace {

using namespace xf;
using namespace tc;

constexpr int64_t kMaxK = 131071;              // 128 * 128 * k stays below 2^31
constexpr int64_t kMostRows = INT32_MAX - 1024;  // tile coordinates stay 32-bit numbers

struct LinearArgs {
  const int8_t *a, *w;
  const float *a_scale, *w_scale, *bias;
  void *y;
  int64_t m, n, a_stride, w_stride, y_stride;
  int k, act;
  int y_tma;  // y can be stored by TMA
};

// The activations of a Conv, but for ReLU of a NaN, which stays one here: the scale of
// a row that was not finite has to show in what is made of it.
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act) {
  if (act == SPKV2_CUDA_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = v[j] <= 0.0f ? 0.0f : v[j];
  } else {
    apply_act_n<N>(v, act);
  }
}

__device__ __forceinline__ float linear_value(int acc, float sa, float sw, float bias, int act) {
  float v[1] = {fmaf(float(acc) * sa, sw, bias)};
  activate<1>(v, act);
  return v[0];
}

// CUDA cores (dp4a), any alignment: 64 x 64 tile, 64 of k a step, a 4 x 4
// patch for each of 256 threads.
constexpr int kST = 64, kSK = 64, kSPitch = kSK + 4;

template <class T>
__global__ void __launch_bounds__(256) linear_simt_kernel(LinearArgs p) {
  pdl_launch_dependents();
  pdl_wait();
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

// ------------------------------------------------------------ tensor cores
// Both kernels compute the transposed tile: the 128 rows of an MMA are output
// CHANNELS (weight rows) and its columns are tokens.  A TMEM lane is then a
// channel, so a thread keeps its channel's scale and bias in registers, the 32
// lanes of a warp store 32 neighbouring channels of one token, and a few
// tokens cost a few columns, not 128 rows.  K steps are 128 bytes, four MMAs
// of K = 32; TMA fills what lies beyond k, n and m with zeros.
constexpr int kBP = 128;                 // channels of a CTA's tile
constexpr int kBK = 128;                 // int8 elements of a K step
constexpr int kPBytes = kBP * kBK;

__device__ int g_linear_status;  // role code of the last bounded wait that gave up

// Codes of the bounded waits: 2 TMA producer, 3 MMA issuer, 4 epilogue, 7
// accumulator hand-off.

// The TMA loads issued into a ring of stages have landed (a bounded wait each,
// at most the last `stages` of `issued`): shared memory must not go away first.
__device__ __forceinline__ void drain_loads(uint64_t *full_bar, int stages, uint32_t issued) {
  for (uint32_t it = issued > uint32_t(stages) ? issued - uint32_t(stages) : 0; it < issued; ++it) {
    const long long t0 = clock64();
    while (!mbar_try_wait(&full_bar[it % uint32_t(stages)], (it / uint32_t(stages)) & 1) && clock64() - t0 < kWaitCycles) {
    }
  }
}

// Four channels n .. n + 3 of one token, scaled and stored; `vec`: all four
// exist and their place is aligned for one store.
template <class T>
__device__ __forceinline__ void store4(const LinearArgs &p, const int4 acc, int64_t m, int64_t n, float sa, const float (&sw)[4],
                                       const float (&bias)[4], bool vec, bool real) {
  float v[4] = {fmaf(float(acc.x) * sa, sw[0], bias[0]), fmaf(float(acc.y) * sa, sw[1], bias[1]),
                fmaf(float(acc.z) * sa, sw[2], bias[2]), fmaf(float(acc.w) * sa, sw[3], bias[3])};
  activate<4>(v, p.act);
  T *y = static_cast<T *>(p.y) + m * p.y_stride + n;
  if (vec) {
    struct alignas(4 * sizeof(T)) Four {
      T v[4];
    };
    Four f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f.v[e] = from_f32<T>(v[e]);
    if (real) *reinterpret_cast<Four *>(y) = f;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (real && n + e < p.n) y[e] = from_f32<T>(v[e]);
  }
}
template <class T>
__device__ __forceinline__ bool vec4_out(const LinearArgs &p, int64_t n) {
  return n + 4 <= p.n && p.y_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(p.y) & (4 * sizeof(T) - 1)) == 0;
}
__device__ __forceinline__ void load_channels(const LinearArgs &p, int64_t n, float (&sw)[4], float (&bias)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    sw[e] = n + e < p.n ? __ldg(p.w_scale + n + e) : 0.0f;
    bias[e] = p.bias && n + e < p.n ? __ldg(p.bias + n + e) : 0.0f;
  }
}

// A warp's chunk of accumulators: COLS tokens from m on of channel n (a lane
// each; n0 the warp's first).  Where rows of y lie on 16-byte boundaries the
// chunk goes through one of the warp's BUFS buffers of 32 tokens x 32 channels
// and one TMA store, which takes the stores off the warps: 32 two-byte stores a
// lane made the epilogue longer than a tile's MMAs (12544 x 256 x 2048 in bf16:
// 31 us, with TMA stores 18.4 us).  `mine`: the
// scale of token m + lane; `count`: the chunks this warp has stored.
__device__ __forceinline__ float token_scale(const LinearArgs &p, int64_t m) { return m < p.m ? __ldg(p.a_scale + m) : 0.0f; }

template <class T, int COLS, int BUFS>
__device__ __forceinline__ void store_chunk(const LinearArgs &p, const CUtensorMap *ymap, T *buffers, int &count,
                                            const uint32_t (&acc)[32], int64_t n0, int64_t m, int lane, float mine, float sw, float bias) {
  const int64_t n = n0 + lane;
  float v[32];
#pragma unroll
  for (int j = 0; j < COLS; ++j) v[j] = fmaf(float(int(acc[j])) * __shfl_sync(0xffffffffu, mine, j), sw, bias);
  if (p.act != SPKV2_CUDA_ACT_NONE) activate<32>(v, p.act);
  if (COLS == 32 && p.y_tma) {
    if (n0 >= p.n) return;
    T *buf = buffers + (count & (BUFS - 1)) * 1024;
    if (lane == 0) {  // the last store from this buffer has read it
      if (BUFS == 2)
        tma_store_wait_read1();
      else
        tma_store_wait_read0();
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < COLS; ++j) buf[j * 32 + lane] = from_f32<T>(v[j]);
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) tma_store_2d(ymap, int(n0), int(m), buf);
    ++count;
    return;
  }
  if (n >= p.n) return;
  const int cnt = int(min(int64_t(COLS), p.m - m));
  T *y = static_cast<T *>(p.y) + m * p.y_stride + n;
#pragma unroll
  for (int j = 0; j < COLS; ++j)
    if (j < cnt) y[j * p.y_stride] = from_f32<T>(v[j]);
}

constexpr int kSplitThreads = 192;

// Columns c0 .. c1 - 1 of the cluster's partial sums part[column][channel], added
// up and stored: a warp per column, four channels a lane, four columns' loads
// from every CTA in flight.
template <class T>
__device__ __forceinline__ void join_columns(const LinearArgs &p, const int32_t *part, int64_t n0, int64_t m0, int c0, int c1,
                                             int csize, int warp, int lane) {
  constexpr int WARPS = kSplitThreads / 32, U = 4;
  const int64_t n = n0 + lane * 4;
  float sw[4], bias[4];
  load_channels(p, n, sw, bias);
  const int end = int(min(int64_t(c1), p.m - m0));  // columns past m are padding
  const bool vec = vec4_out<T>(p, n);
  for (int c = c0 + warp; c < end; c += WARPS * U) {
    int4 sum[U] = {};
    float sa[U];
#pragma unroll
    for (int u = 0; u < U; ++u) sa[u] = c + u * WARPS < end ? __ldg(p.a_scale + m0 + c + u * WARPS) : 0.0f;
#pragma unroll 2
    for (int r = 0; r < csize; ++r)
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + u * WARPS < end) {
          const int4 v = ld_cluster4(map_rank(part + (c + u * WARPS) * kBP + lane * 4, uint32_t(r)));
          sum[u].x += v.x, sum[u].y += v.y, sum[u].z += v.z, sum[u].w += v.w;
        }
#pragma unroll
    for (int u = 0; u < U; ++u)
      store4<T>(p, sum[u], m0 + c + u * WARPS, n, sa[u], sw, bias, vec, c + u * WARPS < end);
  }
}

// Few tiles: one tile of 128 channels x BN tokens per cluster, whose CTAs
// divide k.  Each CTA leaves its int32 sums in its own shared memory and
// takes BN / cluster columns of everybody's: integer sums, so the order does
// not matter, and nothing passes through global memory.  Warps 0-3 epilogue,
// 4 TMA producer, 5 MMA.
constexpr int split_stages(int bn) { return bn >= 256 ? 4 : bn == 128 ? 6 : bn == 64 ? 8 : 10; }
constexpr size_t split_smem(int bn) { return size_t(split_stages(bn)) * (kPBytes + bn * kBK) + 1024; }

template <class T, int BN>
__global__ void __launch_bounds__(kSplitThreads, 1)
    linear_split_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap amap,
                        const __grid_constant__ CUtensorMap ymap, LinearArgs p, int n_tiles, int num_kb, int csize) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int STAGES = split_stages(BN);
  constexpr int STAGE = kPBytes + BN * kBK;
  constexpr uint32_t kTmemCols = BN < 32 ? 32 : BN;
  static_assert(STAGES * STAGE >= BN * kBP * 4, "the partial sums reuse the operand stages");
  __shared__ uint64_t full_bar[STAGES], empty_bar[STAGES], acc_bar;
  __shared__ uint32_t tmem_holder;
  __shared__ volatile int abort_flag;
  int *status = &g_linear_status;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = csize > 1 ? int(cluster_rank()) : 0;
  const int tile = int(blockIdx.x) / csize;
  const int64_t n0 = int64_t(tile % n_tiles) * kBP, m0 = int64_t(tile / n_tiles) * BN;
  const int kb0 = int(int64_t(num_kb) * rank / csize), kb1 = int(int64_t(num_kb) * (rank + 1) / csize);

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(&acc_bar, 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_holder)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;
  pdl_launch_dependents();
  pdl_wait();

  const uint32_t trow = tmem + (uint32_t(warp * 32) << 16);
  int32_t *part = reinterpret_cast<int32_t *>(smem);  // [column][channel]
  bool landed = false;
  if (warp < 4) {
    landed = __all_sync(0xffffffffu, mbar_wait(&acc_bar, 0, &abort_flag, status, 4));
    tc_fence_after();
    if (landed && csize == 1) {
      const int64_t n = n0 + warp * 32 + lane;
      const float sw = n < p.n ? __ldg(p.w_scale + n) : 0.0f;
      const float bias = p.bias && n < p.n ? __ldg(p.bias + n) : 0.0f;
      int count = 0;
#pragma unroll 1
      for (int c = 0; c < BN; c += 32) {
        if (m0 + c >= p.m) break;
        uint32_t acc[32];
        tmem_ld32(trow + uint32_t(c), acc);
        store_chunk<T, BN < 32 ? BN : 32, 2>(p, &ymap, reinterpret_cast<T *>(part) + warp * 2048, count, acc, n0 + warp * 32, m0 + c,
                                          lane, token_scale(p, m0 + c + lane), sw, bias);
      }
      if (lane == 0) tma_store_wait_all();
    } else if (landed) {
#pragma unroll 1
      for (int c = 0; c < BN; c += 32) {
        uint32_t acc[32];
        tmem_ld32(trow + uint32_t(c), acc);
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j < BN) part[(c + j) * kBP + warp * 32 + lane] = int32_t(acc[j]);
      }
    }
  } else if (warp == 4) {
    if (elect_one()) {
      int it = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int s = it % STAGES;
        if (!mbar_wait(&empty_bar[s], ((it / STAGES) & 1) ^ 1, &abort_flag, status, 2)) break;
        uint8_t *st = smem + s * STAGE;
        mbar_arrive_expect_tx(&full_bar[s], STAGE);
        tma_load_2d(st, &wmap, kb * kBK, int(n0), &full_bar[s]);
        tma_load_2d(st + kPBytes, &amap, kb * kBK, int(m0), &full_bar[s]);
      }
      drain_loads(full_bar, STAGES, uint32_t(it));
    }
  } else if (elect_one()) {
    constexpr uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(BN >> 3) << 17) | (uint32_t(kBP >> 4) << 24);
    for (int kb = kb0; kb < kb1; ++kb) {
      const int it = kb - kb0, s = it % STAGES;
      if (!mbar_wait(&full_bar[s], (it / STAGES) & 1, &abort_flag, status, 3)) break;
      tc_fence_after();
      const uint64_t da = smem_desc(smem + s * STAGE), db = smem_desc(smem + s * STAGE + kPBytes);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        mma_i8(tmem, da + kk * 2, db + kk * 2, idesc, (kb > kb0 || kk > 0) ? 1u : 0u);
      mma_commit(&empty_bar[s]);
    }
    mma_commit(&acc_bar);  // completes once every MMA issued above has
  }
  __syncwarp();
  if (csize > 1) {
    cluster_sync();
    if (!abort_flag) join_columns<T>(p, part, n0, m0, rank * (BN / csize), (rank + 1) * (BN / csize), csize, warp, lane);
    __syncwarp();
    cluster_sync();  // the peers have read this CTA's sums
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    if (lane == 0) {  // every issued MMA has finished before TMEM is freed (also after a wait that gave up)
      const long long t0 = clock64();
      while (!mbar_try_wait(&acc_bar, 0) && clock64() - t0 < kWaitCycles) {
      }
    }
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

// Many tiles: persistent CTA pairs, tiles of 256 channels x 256 tokens.  Each
// CTA holds its 128 channels and 128 of the tokens, so a K step brings it 32 KB
// for 256 x 256 x 128 products (a lone CTA would need 48 KB for half of them,
// more than L2 can give every SM).  Two accumulator buffers in TMEM: a tile's
// epilogue runs under the next tile's MMAs.  Warps 0-15 epilogue (64 columns of a
// TMEM lane quarter each: with 8 warps the chain of loads, conversions and
// stores of a chunk was longer than the MMAs of a tile of small k, 12544 x 256 x
// 2048 in bf16 22 us, with 16 18.4 us), 16 TMA producer, 17 MMA (in the leader).
constexpr int kPairN = 256;
constexpr int kPairEpi = 16, kPairThreads = (kPairEpi + 2) * 32;  // epilogue warps
constexpr int kPairCols = kPairN * 4 / kPairEpi;  // columns of an epilogue warp
constexpr int kPairStage = kPBytes + kPairN / 2 * kBK;
constexpr int pair_stages(int elem) { return kPairEpi * elem > 32 ? 5 : 6; }
constexpr size_t pair_smem(int elem) { return size_t(pair_stages(elem)) * kPairStage + size_t(kPairEpi * elem) * 1024 + 1024; }

template <class T>
__global__ void __launch_bounds__(kPairThreads, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap amap,
                       const __grid_constant__ CUtensorMap ymap, LinearArgs p, int n_tiles, int tiles, int num_kb) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int STAGES = pair_stages(sizeof(T));
  __shared__ uint64_t full_bar[STAGES], empty_bar[STAGES], accf_bar[2], acce_bar[2];
  __shared__ uint32_t tmem_holder;
  __shared__ volatile int abort_flag;
  int *status = &g_linear_status;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = int(cluster_rank());
  const int tile0 = int(cluster_id_x()), tstep = int(cluster_count_x());
  const int my_tiles = tile0 < tiles ? (tiles - 1 - tile0) / tstep + 1 : 0;

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);   // (leader) both CTAs' operands have landed
      mbar_init(&empty_bar[s], 1);  // the leader's MMAs have read the stage
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accf_bar[b], 1);
      mbar_init(&acce_bar[b], 2 * kPairEpi);  // one arrival per epilogue warp of both CTAs
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kPairEpi + 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_holder)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers exist before any remote arrival
  tc_fence_after();
  const uint32_t tmem = tmem_holder;
  pdl_launch_dependents();
  pdl_wait();

  if (warp < kPairEpi) {
    const int quarter = warp & 3, col0 = (warp >> 2) * kPairCols;
    T *buffers = reinterpret_cast<T *>(smem + STAGES * kPairStage) + warp * 1024;
    int count = 0;
    for (int ti = 0; ti < my_tiles; ++ti) {
      const int t = tile0 + ti * tstep, ab = ti & 1;
      const int64_t n = int64_t(t % n_tiles) * 2 * kBP + rank * kBP + quarter * 32 + lane;
      const int64_t m0 = int64_t(t / n_tiles) * kPairN;
      const float sw = n < p.n ? __ldg(p.w_scale + n) : 0.0f;
      const float bias = p.bias && n < p.n ? __ldg(p.bias + n) : 0.0f;
      float mine[kPairCols / 32];
#pragma unroll
      for (int k = 0; k < kPairCols / 32; ++k) mine[k] = token_scale(p, m0 + col0 + k * 32 + lane);
      if (!__all_sync(0xffffffffu, mbar_wait(&accf_bar[ab], (ti >> 1) & 1, &abort_flag, status, 4))) break;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < kPairCols / 32; ++k) {
        const int c = col0 + k * 32;
        uint32_t acc[32];
        tmem_ld32(tmem + (uint32_t(quarter * 32) << 16) + uint32_t(ab * kPairN + c), acc);
        if (k == kPairCols / 32 - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_rank_tmem(&acce_bar[ab], 0);
        }
        if (m0 + c < p.m) store_chunk<T, 32, 1>(p, &ymap, buffers, count, acc, n - lane, m0 + c, lane, mine[k], sw, bias);
      }
    }
    if (lane == 0) tma_store_wait_all();
  } else if (warp == kPairEpi) {
    if (elect_one()) {
      uint32_t it = 0;
      bool ok = true;
      for (int ti = 0; ti < my_tiles && ok; ++ti) {
        const int t = tile0 + ti * tstep;
        const int n0 = t % n_tiles * 2 * kBP + rank * kBP, m0 = t / n_tiles * kPairN + rank * (kPairN / 2);
        for (int kb = 0; kb < num_kb; ++kb, ++it) {
          const int s = it % STAGES;
          ok = mbar_wait(&empty_bar[s], ((it / STAGES) & 1) ^ 1, &abort_flag, status, 2);
          if (!ok) break;
          uint8_t *st = smem + s * kPairStage;
          const uint32_t bar = map_rank(&full_bar[s], 0);
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[s], 2 * kPairStage);
          tma_load_2d_pair(st, &wmap, kb * kBK, n0, bar);
          tma_load_2d_pair(st + kPBytes, &amap, kb * kBK, m0, bar);
        }
      }
      if (rank == 0) drain_loads(full_bar, STAGES, it);
    }
  } else if (rank == 0 && elect_one()) {
    constexpr uint32_t idesc =
        (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(kPairN >> 3) << 17) | (uint32_t(2 * kBP >> 4) << 24);
    uint32_t it = 0;
    int done = 0;
    bool ok = true;
    for (int ti = 0; ti < my_tiles && ok; ++ti) {
      const int ab = ti & 1;
      ok = mbar_wait_cluster(&acce_bar[ab], ((ti >> 1) & 1) ^ 1, &abort_flag, status, 7);
      if (!ok) break;
      tc_fence_after();
      for (int kb = 0; kb < num_kb; ++kb, ++it) {
        const int s = it % STAGES;
        const uint32_t ph = (it / STAGES) & 1;
        ok = mbar_wait(&full_bar[s], ph, &abort_flag, status, 3);
        if (!ok) break;
        tc_fence_after();
        const uint64_t da = smem_desc(smem + s * kPairStage), db = smem_desc(smem + s * kPairStage + kPBytes);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_i8_pair(tmem + uint32_t(ab * kPairN), da + kk * 2, db + kk * 2, idesc, (kb | kk) ? 1u : 0u);
        mma_commit_pair(&empty_bar[s]);
      }
      if (!ok) break;
      mma_commit_pair(&accf_bar[ab]);
      ++done;
    }
    if (done > 0) {  // every issued MMA has finished before TMEM is freed
      const long long t0 = clock64();
      while (!mbar_try_wait(&accf_bar[(done - 1) & 1], ((done - 1) >> 1) & 1) && clock64() - t0 < kWaitCycles) {
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync();  // the leader's MMAs read the peer's shared memory until here
  if (warp == kPairEpi + 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// ------------------------------------------------------------ choice
// TMA reads rows that start on 16-byte boundaries.
bool tma_rows(const int8_t *base, int64_t rows, int64_t stride, int k) {
  return aligned16(base) && (rows == 1 || (stride % 16 == 0 && stride >= k));
}

bool encode_rows(CUtensorMap *map, const int8_t *base, int64_t rows, int64_t stride, int k, int box) {
  const uint64_t pitch = rows == 1 ? (uint64_t(k) + 15) / 16 * 16 : uint64_t(stride);
  return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, base, uint64_t(k), uint64_t(rows), pitch, uint32_t(box));
}

// Stores of 32 channels x 32 tokens; false where rows of y are not on 16-byte
// boundaries.
template <class T>
bool encode_y(CUtensorMap *map, const LinearArgs &p) {
  if (!aligned16(p.y) || (p.m > 1 && p.y_stride * int64_t(sizeof(T)) % 16 != 0)) return false;
  const uint64_t pitch = p.m > 1 ? uint64_t(p.y_stride) : (uint64_t(p.n) + 7) / 8 * 8;
  return encode_2d_box(map, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, sizeof(T), p.y,
                       uint64_t(p.n), uint64_t(p.m), pitch, 32, 32, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// Shared memory of a CTA: one with fewer K steps than stages asks for what it
// uses, so that clusters find room beside one another.
template <class T>
size_t split_used(int bn, int num_kb, int csize) {
  const size_t stages = size_t(std::min(split_stages(bn), int(ceil_div(num_kb, csize)))) * (kPBytes + bn * kBK);
  return std::max(stages, csize > 1 ? size_t(bn) * kBP * 4 : 4 * 2048 * sizeof(T)) + 1024;
}

template <class T, int BN>
int launch_split(const LinearArgs &p, const CUtensorMap &ymap, int n_tiles, int m_tiles, int num_kb, int csize, cudaStream_t s) {
  if (const int rc = allow_smem<linear_split_kernel<T, BN>>(split_smem(BN))) return rc;
  CUtensorMap wmap, amap;
  if (!encode_rows(&wmap, p.w, p.n, p.w_stride, p.k, kBP) || !encode_rows(&amap, p.a, p.m, p.a_stride, p.k, BN))
    return SPKV2_ERR_CUDA;
  return cuda_status(launch_kernel(linear_split_kernel<T, BN>, unsigned(n_tiles * m_tiles * csize), kSplitThreads,
                                   split_used<T>(BN, num_kb, csize), s, csize,
                                   wmap, amap, ymap, p, n_tiles, num_kb, csize));
}

template <class T>
int launch_pair(const LinearArgs &p, const CUtensorMap &ymap, int n_tiles, int m_tiles, int num_kb, cudaStream_t s) {
  if (const int rc = allow_smem<linear_pair_kernel<T>>(pair_smem(sizeof(T)))) return rc;
  CUtensorMap wmap, amap;
  if (!encode_rows(&wmap, p.w, p.n, p.w_stride, p.k, kBP) || !encode_rows(&amap, p.a, p.m, p.a_stride, p.k, kPairN / 2))
    return SPKV2_ERR_CUDA;
  const int tiles = n_tiles * m_tiles;
  return cuda_status(launch_kernel(linear_pair_kernel<T>, 2u * unsigned(std::min(tiles, sm_count() / 2)), kPairThreads, pair_smem(sizeof(T)),
                                   s, 2, wmap, amap, ymap, p, n_tiles, tiles, num_kb));
}

// The cheapest shape by an estimate of its time in microseconds, fitted to
// measured sweeps over all shapes of some forty sizes (1 .. 16000 tokens, k 93 ..
// 16384, n 64 .. 16384).  Over 40 sizes the choice was within 5 % of the best shape
// for 35, within 20 % for 39, and 36 % behind for 6000 x 8000 x 640, where 120 CTAs of
// 256 columns reach L2's limit, which the estimate sees from the second tile on only:
//   single tile: 2.6 launch, 0.7 first operands (once where a CTA leaves room
//     for a second on its SM), 0.2 a K step (0.28 with 256 columns) while every
//     SM has one tile and 0.0015 a row of operands beyond, when L2 is the limit;
//     epilogue 0.1 + 0.015 a column, twice that where y takes no TMA stores; with
//     a cluster 0.3 + 0.023 a column instead, for the join;
//   pairs: 2.6 launch, 2.4 for the first operands and the last epilogue, 0.31 a
//     K step and 0.4 a tile.
template <class T>
int launch_tc(LinearArgs p, cudaStream_t s) {
  CUtensorMap ymap = {};
  p.y_tma = encode_y<T>(&ymap, p);
  const int num_kb = int(ceil_div(p.k, kBK)), sms = sm_count();
  const int64_t n_tiles = ceil_div(p.n, kBP);
  int best_bn = 0, best_c = 1;
  double best = 1e30;
  for (int bn = 16; bn <= 256; bn *= 2) {
    const int64_t tiles = n_tiles * ceil_div(p.m, bn);
    if (tiles > INT32_MAX / 8) continue;
    for (int c = 1; c <= 8; c *= 2) {
      if (c > 1 && (num_kb < 2 * c || tiles * c > sms)) break;
      const double kb = double(ceil_div(num_kb, c)), rounds = double(ceil_div(tiles * c, sms));
      const double step = rounds > 1.0 ? 0.0015 * (kBP + bn) : bn == 256 ? 0.28 : 0.2;
      const bool roomy = split_used<T>(bn, num_kb, c) <= 110 * 1024;
      const double end = c > 1 ? 0.3 + 0.023 * bn : (0.1 + 0.015 * bn) * (p.y_tma ? 1.0 : 2.0);
      const double cost = 2.6 + 0.7 * (roomy ? 1.0 : rounds) + rounds * (kb * step + end);
      if (cost < best) best = cost, best_bn = bn, best_c = c;
    }
  }
  const int64_t pn = ceil_div(p.n, 2 * kBP), pm = ceil_div(p.m, kPairN);
  const double pair = 5.0 + double(ceil_div(pn * pm, sms / 2)) * (num_kb * 0.31 + 0.4);
  if (pn * pm <= INT32_MAX / 2 && (pair < best || !best_bn)) return launch_pair<T>(p, ymap, int(pn), int(pm), num_kb, s);
  const int nt = int(n_tiles), mt = int(ceil_div(p.m, best_bn));
  switch (best_bn) {
    case 16: return launch_split<T, 16>(p, ymap, nt, mt, num_kb, best_c, s);
    case 32: return launch_split<T, 32>(p, ymap, nt, mt, num_kb, best_c, s);
    case 64: return launch_split<T, 64>(p, ymap, nt, mt, num_kb, best_c, s);
    case 128: return launch_split<T, 128>(p, ymap, nt, mt, num_kb, best_c, s);
    default: return launch_split<T, 256>(p, ymap, nt, mt, num_kb, best_c, s);
  }
}

}  // namespace

int linear_status(int *code) { return take_status(g_linear_status, code); }

}  // namespace spkv2

using namespace spkv2;
using namespace spkv2::xf;

extern "C" int spkv2_cuda_linear_i8(const Spkv2LinearI8 *a, void *stream) {
  if (!a || a->m < 0 || a->n < 0 || a->k < 0) return -1;
  if (a->m == 0 || a->n == 0) return 0;
  if (!a->y || !a->a_scale || !a->w_scale || (a->k > 0 && (!a->a || !a->w))) return -1;
  if (a->a_stride < 0 || a->w_stride < 0 || overlaps(a->y_stride, a->m, a->n)) return -1;
  if (a->activation < SPKV2_CUDA_ACT_NONE || a->activation > SPKV2_CUDA_ACT_SILU) return -1;
  if (!elem_bytes(a->dtype) || a->k > kMaxK || a->m > kMostRows || a->n > kMostRows) return SPKV2_ERR_UNSUPPORTED;
  if (!on_bytes(elem_bytes(a->dtype), a->y) || !on_bytes(4, a->a_scale, a->w_scale, a->bias)) return -1;
  const LinearArgs p = {a->a, a->w, a->a_scale, a->w_scale, a->bias, a->y, a->m, a->n, a->a_stride, a->w_stride,
                        a->y_stride, int(a->k), a->activation};
  const int64_t tiles = ceil_div(a->m, kST) * ceil_div(a->n, kST);
  if (tiles > INT32_MAX) return SPKV2_ERR_UNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p.k > 0 && tma_rows(p.a, p.m, p.a_stride, p.k) && tma_rows(p.w, p.n, p.w_stride, p.k) && encode_fn())
    return by_type(a->dtype, [&](auto t) { return launch_tc<decltype(t)>(p, s); });
  return by_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    return cuda_status(launch_kernel(linear_simt_kernel<T>, unsigned(tiles), 256u, 0, s, 1, p));
  });
}

extern "C" int spkv2_cuda_transformer_status(int *code) {
  if (!code) return -1;
  *code = 0;
  // Copies of the words alone would not wait for streams that do not block the default one.
  if (const int rc = cuda_status(cudaDeviceSynchronize())) return rc;
  int (*const take[])(int *) = {linear_status, cross_tc_status, cross_step_status};
  int first = 0;
  for (auto t : take) {
    int c = 0;
    if (const int rc = t(&c)) return rc;
    if (!first) first = c;
  }
  *code = first;
  return first ? SPKV2_ERR_DEVICE_STATUS : 0;
}
