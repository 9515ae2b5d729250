// Contraction of 8-bit integers on the tcgen05 tensor cores (kind::i8).
//
// acc[t, c] = sum_k left[t, k] right[c, k] in 32-bit integers, which are exact
// in any order; the epilogue scales, adds the bias and applies the activation
// in FP32 and rounds once. The channels (right rows) are the MMA's M side and
// the tokens its N side: an epilogue thread then owns one channel (its scale
// and bias stay in registers), a warp stores 32 neighbouring channels of a
// token at a time, and a single token is an MMA of N = 16 that costs nothing
// beside the weights' bytes. A gated layer stages a tile of gate rows and the
// tile of their value rows and keeps two accumulators, so that no output but the
// activated product is written.
//
// Two kernels:
// * i8_pair_kernel: CTA pairs (cta_group::2) over tiles of 256 channels x 256
//   tokens (gated: 256 + 256 channels x 128 tokens), persistent, accumulators
//   double-buffered in TMEM so that the epilogue runs under the next tile.
// * i8_split_kernel: one tile of 128 channels x NT tokens (NT = 16 .. 128) for
//   problems with too few pair tiles to fill the GPU. A cluster of 1 to 8 CTAs
//   shares the tile's K walk; each holds a partial accumulator, and the
//   cluster adds them through distributed shared memory.
// Both stage 128-byte swizzled K rows with TMA (out-of-range rows and K read
// as zeros) in a ring of mbarrier stages. Every wait is bounded; a wait that
// gives up raises the CTA's (or pair's) abort flag and records a device error.
#include <cuda.h>
#include <algorithm>
#include "eir_launch.h"
#include "i8_common.cuh"

namespace eir {

constexpr int kI8Rows = 128;                      // channels of a CTA
constexpr int kI8BlockK = 128;                    // K of a stage: one swizzle row
constexpr int kI8SubBytes = kI8Rows * kI8BlockK;  // a tile of 128 rows

// ---------------------------------------------------------------- CTA pairs

template <bool GATED>
struct I8Pair {
  static constexpr int kTokens = GATED ? 128 : 256;       // tokens of a tile (N of the MMA)
  static constexpr int kABytes = kI8SubBytes * (GATED ? 2 : 1);
  static constexpr int kBBytes = kTokens / 2 * kI8BlockK;  // each CTA stages half of the tokens
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = (232448 - 1024 - 5120) / kStageBytes;
  static constexpr int kAccCols = kTokens * (GATED ? 2 : 1);
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = 32 * (2 + kEpiWarps);
  static constexpr int kWarpTokens = kTokens / 2;  // columns of one epilogue warp
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + 5120;
  static_assert(kAccCols == 256, "two accumulators fill TMEM");
};

// pair tile -> (channel tile, token tile): bands of 8 token tiles, channels
// outermost within a band, so that the tiles in flight share operands in L2
// and a weight is read from HBM once per 8 token tiles
__device__ __forceinline__ void i8_pair_tile(uint32_t t, uint32_t c_tiles, uint32_t t_tiles, uint32_t &ct,
                                             uint32_t &tt) {
  const uint32_t band = t / (8 * c_tiles), first = band * 8;
  const uint32_t height = min(8u, t_tiles - first), r = t - first * c_tiles;
  tt = first + r % height;
  ct = r / height;
}

template <bool GATED, typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(I8Pair<GATED>::kThreads, 1)
    i8_pair_kernel(const __grid_constant__ CUtensorMap map_c, const __grid_constant__ CUtensorMap map_t,
                   const I8Params p, const I8Ptrs a, uint32_t *err, uint32_t c_tiles, uint32_t t_tiles) {
  using Cfg = I8Pair<GATED>;
  constexpr int S = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sA = smem, *sB = smem + S * Cfg::kABytes;
  float *s_scale = reinterpret_cast<float *>(smem + S * Cfg::kStageBytes);  // token scales, a part per epilogue warp
  uint64_t *bars = reinterpret_cast<uint64_t *>(s_scale + Cfg::kEpiWarps * Cfg::kWarpTokens);
  uint64_t *full = bars, *empty = bars + S, *tfull = bars + 2 * S, *tempty = bars + 2 * S + 2;
  uint64_t *drain = bars + 2 * S + 4;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * S + 5);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank(), peer = rank ^ 1u;
  const uint32_t pair_id = blockIdx.x >> 1, n_pairs = gridDim.x >> 1, tiles = c_tiles * t_tiles;
  const int k_blocks = (int)((p.k + kI8BlockK - 1) / kI8BlockK);
  const int64_t n_out = GATED ? p.n / 2 : p.n;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 2 * Cfg::kEpiWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_map(&map_c);
    tma_prefetch_map(&map_t);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before();
  cluster_sync();  // barriers of both CTAs initialised before any remote arrive
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t peer_abort = mapa_shared(smem_u32((const void *)abort_flag), peer);
  auto raise_abort = [&](uint32_t code) {
    if (!*abort_flag) record_error(err, code);
    *abort_flag = 1;
    st_cluster_u32(peer_abort, 1u);
  };

  if (warp == 0) {
    // ------------------------------------------------------------ producer (both CTAs)
    if (lane == 0) {
      const uint32_t full_leader = mapa_shared(smem_u32(full), 0);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (uint32_t t = pair_id; t < tiles && ok && !*abort_flag; t += n_pairs) {
        uint32_t ct, tt;
        i8_pair_tile(t, c_tiles, t_tiles, ct, tt);
        const int row_c = (int)(ct * 256 + rank * kI8Rows);
        const int row_t = (int)(tt * Cfg::kTokens + rank * (Cfg::kTokens / 2));
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait_bounded(&empty[stage], phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * Cfg::kStageBytes);
          const uint32_t bar = full_leader + 8u * (uint32_t)stage;
          uint8_t *dA = sA + stage * Cfg::kABytes;
          tma_load_2d_pair(dA, &map_c, bar, kb * kI8BlockK, row_c);
          if (GATED) tma_load_2d_pair(dA + kI8SubBytes, &map_c, bar, kb * kI8BlockK, row_c + (int)n_out);
          tma_load_2d_pair(sB + stage * Cfg::kBBytes, &map_t, bar, kb * kI8BlockK, row_t);
          if (++stage == S) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // every stage released: no commit of the leader reaches this CTA's barriers after it exits
      for (int i = 0; i < S && ok && !*abort_flag; ++i) {
        if (!mbar_wait_bounded(&empty[stage], phase ^ 1u, abort_flag)) ok = false;
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) raise_abort(kErrTimeoutProducer);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader)
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = i8_idesc(256, Cfg::kTokens);
      const uint32_t empty_peer = mapa_shared(smem_u32(empty), 1);
      const uint32_t tfull_peer = mapa_shared(smem_u32(tfull), 1);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (uint32_t t = pair_id; t < tiles && ok; t += n_pairs) {
        if (!mbar_wait_bounded(&tempty[acc], acc_phase ^ 1u, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + (uint32_t)(acc * Cfg::kAccCols);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait_bounded(&full[stage], phase, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t ab = smem_u32(sA + stage * Cfg::kABytes), bb = smem_u32(sB + stage * Cfg::kBBytes);
#pragma unroll
          for (int kk = 0; kk < kI8BlockK / 32; ++kk) {
            const uint64_t bd = make_smem_desc(bb + kk * 32, 16, 1024, kLayoutSw128);
            const uint32_t accum = (kb > 0 || kk > 0) ? 1u : 0u;
            umma_i8_pair(d, make_smem_desc(ab + kk * 32, 16, 1024, kLayoutSw128), bd, idesc, accum);
            if (GATED)
              umma_i8_pair(d + Cfg::kTokens, make_smem_desc(ab + kI8SubBytes + kk * 32, 16, 1024, kLayoutSw128),
                           bd, idesc, accum);
          }
          umma_commit_pair(smem_u32(&empty[stage]));
          umma_commit_pair(empty_peer + 8u * (uint32_t)stage);
          if (++stage == S) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit_pair(smem_u32(&tfull[acc]));
        umma_commit_pair(tfull_peer + 8u * (uint32_t)acc);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
      // every MMA of this CTA pair has completed before TMEM is released
      umma_commit_pair(smem_u32(drain));
      if (!mbar_wait_bounded(drain, 0u, abort_flag) && !*abort_flag) ok = false;
      if (!ok) raise_abort(kErrTimeoutMma);
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int q = warp & 3;  // TMEM lane quadrant this warp may access
    const int col0 = ((warp - 2) >> 2) * Cfg::kWarpTokens;
    float *scale = s_scale + (warp - 2) * Cfg::kWarpTokens;
    const uint32_t tempty_leader = mapa_shared(smem_u32(tempty), 0);
    const float low = p.act == EIR_ACT_RELU ? 0.f : -INFINITY;
    // 4-byte stores of two channels need even rows and a 4-byte base
    const bool pairs = sizeof(T) == 2 && p.s_out % 2 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 3) == 0;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (uint32_t t = pair_id; t < tiles; t += n_pairs) {
      uint32_t ct, tt;
      i8_pair_tile(t, c_tiles, t_tiles, ct, tt);
      const int64_t c = (int64_t)ct * 256 + rank * kI8Rows + q * 32 + lane;
      const int64_t t0 = (int64_t)tt * Cfg::kTokens + col0;
      // the tile's scales are fetched under its MMAs
      const I8Channel h = i8_channel(p, a, c, n_out, GATED);
      __syncwarp();
      for (int i = lane; i < Cfg::kWarpTokens; i += 32)
        scale[i] = a.scale_l && t0 + i < p.m ? a.scale_l[t0 + i] : 1.f;
      __syncwarp();
      if (!mbar_wait_warp(&tfull[acc], acc_phase, abort_flag)) {
        if (lane == 0) raise_abort(kErrTimeoutEpilogue);
        break;
      }
      tc_fence_after();
      T *out = static_cast<T *>(a.out) + t0 * p.s_out + c;
      const uint32_t src = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * Cfg::kAccCols + col0);
#pragma unroll 1
      for (int ch = 0; ch < Cfg::kWarpTokens && t0 + ch < p.m; ch += 16, out += 16 * p.s_out) {
        uint32_t v[16], u[16];
        tmem_ld_32x32b_x16(src + ch, v);
        if (GATED) tmem_ld_32x32b_x16(src + Cfg::kTokens + ch, u);
        tmem_ld_wait();
        const int left = (int)min((int64_t)16, p.m - (t0 + ch));
        float z[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          z[i] = i8_value<GATED>((int32_t)v[i], GATED ? (int32_t)u[i] : 0, scale[ch + i], h, low);
        if (pairs && left == 16) {
          // lanes 2j and 2j + 1 swap halves: each then holds two channels of one token
          const bool odd = lane & 1;
          T *o = out - (odd ? 1 : 0) + (odd ? p.s_out : 0);
          const bool two = c - (odd ? 1 : 0) + 1 < n_out, one = c - (odd ? 1 : 0) < n_out;
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(z[i], z[i + 1]);
            const uint32_t mine = *reinterpret_cast<uint32_t const *>(&b);
            const uint32_t theirs = __shfl_xor_sync(0xffffffffu, mine, 1);
            const uint32_t w = odd ? __byte_perm(theirs, mine, 0x7632) : __byte_perm(mine, theirs, 0x5410);
            if (two) *reinterpret_cast<uint32_t *>(o + i * p.s_out) = w;
            else if (one) *reinterpret_cast<uint16_t *>(o + i * p.s_out) = (uint16_t)w;
          }
        } else if (c < n_out) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (i < left) out[i * p.s_out] = from_f32<T>(z[i]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tempty_leader + 8u * (uint32_t)acc);
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
  }

  // After an abort, copies or commits issued before it may still be landing in
  // this CTA's shared memory: give them time before the CTA can exit.
  if (threadIdx.x == 0 && *abort_flag) {
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();  // both CTAs done: no remote arrive or TMEM read is outstanding
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ---------------------------------------------------------------- split K over a cluster

template <int NT, bool GATED>
struct I8Split {
  static constexpr int kABytes = kI8SubBytes * (GATED ? 2 : 1);
  static constexpr int kBBytes = NT * kI8BlockK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kAccBytes = NT * kI8Rows * 4 * (GATED ? 2 : 1);  // the exchanged accumulators
  // about 100 KB a CTA, two CTAs on an SM: enough bytes in flight for HBM
  static constexpr int kFit = 104 * 1024 / kStageBytes;
  static constexpr int kStages = kFit < 2 ? 2 : kFit;
  static constexpr int kRing = kStages * kStageBytes > kAccBytes ? kStages * kStageBytes : kAccBytes;
  static constexpr int kCols0 = NT * (GATED ? 2 : 1);
  static constexpr int kCols = kCols0 < 32 ? 32 : kCols0;
  static constexpr int kThreads = 192;
  static constexpr int kSmemBytes = 1024 + kRing + 512;
  static_assert(kSmemBytes <= 232448 && kCols <= 256, "shared memory and TMEM of two CTAs");
};

__device__ __forceinline__ int32_t ld_cluster_s32(uint32_t addr_cluster) {
  int32_t v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr_cluster) : "memory");
  return v;
}

template <int NT, bool GATED, typename T>
__global__ void __launch_bounds__(192, 1)
    i8_split_kernel(const __grid_constant__ CUtensorMap map_c, const __grid_constant__ CUtensorMap map_t,
                    const I8Params p, const I8Ptrs a, uint32_t *err, uint32_t split, uint32_t t_tiles) {
  using Cfg = I8Split<NT, GATED>;
  constexpr int S = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sA = smem, *sB = smem + S * Cfg::kABytes;
  int32_t *s_acc = reinterpret_cast<int32_t *>(smem);  // [gate, value][token][channel], after the last MMA
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + Cfg::kRing);
  uint64_t *full = bars, *empty = bars + S, *tfull = bars + 2 * S;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * S + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = split > 1 ? cluster_ctarank() : 0u;
  const uint32_t tile = blockIdx.x / split, ct = tile / t_tiles, tt = tile % t_tiles;
  const int k_blocks = (int)((p.k + kI8BlockK - 1) / kI8BlockK);
  const int kb0 = (int)((int64_t)k_blocks * rank / split), kb1 = (int)((int64_t)k_blocks * (rank + 1) / split);
  const int64_t n_out = GATED ? p.n / 2 : p.n;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(tfull, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_map(&map_c);
    tma_prefetch_map(&map_t);
  }
  if (warp == 1) tmem_alloc(tmem_slot, Cfg::kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();
  pdl_wait();

  bool ok = true;  // this thread's view: false once a wait of the CTA has given up
  if (warp == 0) {
    if (lane == 0) {
      const int row_c = (int)(ct * kI8Rows), row_t = (int)(tt * NT);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&empty[stage], phase ^ 1u, abort_flag)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&full[stage], Cfg::kStageBytes);
        uint8_t *dA = sA + stage * Cfg::kABytes;
        tma_load_2d(dA, &map_c, &full[stage], kb * kI8BlockK, row_c);
        if (GATED) tma_load_2d(dA + kI8SubBytes, &map_c, &full[stage], kb * kI8BlockK, row_c + (int)n_out);
        tma_load_2d(sB + stage * Cfg::kBBytes, &map_t, &full[stage], kb * kI8BlockK, row_t);
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok && !*abort_flag) {
        record_error(err, kErrTimeoutProducer);
        *abort_flag = 1;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = i8_idesc(kI8Rows, NT);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&full[stage], phase, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t ab = smem_u32(sA + stage * Cfg::kABytes), bb = smem_u32(sB + stage * Cfg::kBBytes);
#pragma unroll
        for (int kk = 0; kk < kI8BlockK / 32; ++kk) {
          const uint64_t bd = make_smem_desc(bb + kk * 32, 16, 1024, kLayoutSw128);
          const uint32_t accum = (kb > kb0 || kk > 0) ? 1u : 0u;
          umma_i8(tmem_base, make_smem_desc(ab + kk * 32, 16, 1024, kLayoutSw128), bd, idesc, accum);
          if (GATED)
            umma_i8(tmem_base + NT, make_smem_desc(ab + kI8SubBytes + kk * 32, 16, 1024, kLayoutSw128), bd, idesc,
                    accum);
        }
        umma_commit(&empty[stage]);
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
      umma_commit(tfull);
      if (!ok && !*abort_flag) {
        record_error(err, kErrTimeoutMma);
        *abort_flag = 1;
      }
    }
  }
  __syncwarp();
  // every warp waits for the accumulators: the ring is free for the exchange, and nothing is in
  // flight when the CTA ends
  if (!mbar_wait_warp(tfull, 0u, abort_flag) && lane == 0 && !*abort_flag) {
    record_error(err, kErrTimeoutEpilogue);
    *abort_flag = 1;
  }
  __syncwarp();
  if (*abort_flag) {
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);  // copies issued before the abort land first
    ok = false;
  }
  tc_fence_after();
  const int64_t t0 = (int64_t)tt * NT;
  const int tokens = (int)min((int64_t)NT, p.m - t0);
  const float low = p.act == EIR_ACT_RELU ? 0.f : -INFINITY;
  const int q = warp & 3, row = q * 32 + lane;
  const int64_t c = (int64_t)ct * kI8Rows + row;
  const uint32_t src = tmem_base + ((uint32_t)(q * 32) << 16);
  if (split == 1) {
    if (warp >= 2 && ok) {
      const I8Channel h = i8_channel(p, a, c, n_out, GATED);
      T *out = static_cast<T *>(a.out) + t0 * p.s_out + c;
#pragma unroll 1
      for (int ch = 0; ch < tokens; ch += 16) {
        uint32_t v[16], u[16];
        tmem_ld_32x32b_x16(src + ch, v);
        if (GATED) tmem_ld_32x32b_x16(src + NT + ch, u);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (ch + i < tokens && c < n_out) {
            const float sa = a.scale_l ? a.scale_l[t0 + ch + i] : 1.f;
            out[(int64_t)(ch + i) * p.s_out] =
                from_f32<T>(i8_value<GATED>((int32_t)v[i], GATED ? (int32_t)u[i] : 0, sa, h, low));
          }
        }
      }
    }
  } else {
    if (warp >= 2 && ok) {
#pragma unroll 1
      for (int ch = 0; ch < tokens; ch += 16) {
#pragma unroll
        for (int half = 0; half < (GATED ? 2 : 1); ++half) {
          uint32_t v[16];
          tmem_ld_32x32b_x16(src + half * NT + ch, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (ch + i < tokens) s_acc[(half * NT + ch + i) * kI8Rows + row] = (int32_t)v[i];
        }
      }
    }
    __syncwarp();
    cluster_sync();  // every CTA's partial sums are in its shared memory
    if (warp >= 2 && ok) {
      const I8Channel h = i8_channel(p, a, c, n_out, GATED);
      // CTA `rank` adds up and stores every split-th token
      for (int j = (int)rank; j < tokens; j += (int)split) {
        int32_t acc = 0, acc2 = 0;
        const uint32_t at = smem_u32(s_acc + j * kI8Rows + row);
        for (uint32_t r = 0; r < split; ++r) {
          acc += ld_cluster_s32(mapa_shared(at, r));
          if (GATED) acc2 += ld_cluster_s32(mapa_shared(at + NT * kI8Rows * 4, r));
        }
        if (c < n_out) {
          const float sa = a.scale_l ? a.scale_l[t0 + j] : 1.f;
          static_cast<T *>(a.out)[(t0 + j) * p.s_out + c] = from_f32<T>(i8_value<GATED>(acc, acc2, sa, h, low));
        }
      }
    }
    __syncwarp();
    cluster_sync();  // no CTA leaves while its shared memory is read
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::kCols);
  }
}

// ---------------------------------------------------------------- launchers

template <typename Kern>
static cudaError_t i8_allow_smem(Kern kern, int bytes, bool (&done)[32]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 32 && done[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 32) done[dev] = true;
  return e;
}

template <bool GATED, typename T>
static cudaError_t launch_pair(I8TcPlan const &tp, CUtensorMap const &mc, CUtensorMap const &mt, I8Params const &p,
                               I8Ptrs const &a, uint32_t *err, cudaStream_t st) {
  using Cfg = I8Pair<GATED>;
  auto kern = i8_pair_kernel<GATED, T>;
  static bool done[32] = {};
  cudaError_t e = i8_allow_smem(kern, Cfg::kSmemBytes, done);
  if (e != cudaSuccess) return e;
  static int clusters[32] = {};  // per device: pairs that can run at once
  int dev = 0;
  e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  int most = dev < 32 ? clusters[dev] : 0;
  if (most == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2);
    cfg.blockDim = dim3(Cfg::kThreads);
    cfg.dynamicSmemBytes = Cfg::kSmemBytes;
    e = cudaOccupancyMaxActiveClusters(&most, kern, &cfg);
    if (e != cudaSuccess) return e;
    if (most < 1) return cudaErrorInvalidConfiguration;
    if (dev < 32) clusters[dev] = most;
  }
  const int64_t tiles = tp.c_tiles * tp.t_tiles, pairs = std::min<int64_t>(tiles, most);
  return launch_kernel(kern, dim3((unsigned)(2 * pairs)), dim3(Cfg::kThreads), Cfg::kSmemBytes, st, mc, mt, p, a, err,
                       (uint32_t)tp.c_tiles, (uint32_t)tp.t_tiles);
}

template <int NT, bool GATED, typename T>
static cudaError_t launch_split(I8TcPlan const &tp, CUtensorMap const &mc, CUtensorMap const &mt, I8Params const &p,
                                I8Ptrs const &a, uint32_t *err, cudaStream_t st) {
  using Cfg = I8Split<NT, GATED>;
  auto kern = i8_split_kernel<NT, GATED, T>;
  static bool done[32] = {};
  cudaError_t e = i8_allow_smem(kern, Cfg::kSmemBytes, done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tp.c_tiles * tp.t_tiles * tp.split));
  cfg.blockDim = dim3(Cfg::kThreads);
  cfg.dynamicSmemBytes = Cfg::kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (tp.split > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)tp.split;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kern, mc, mt, p, a, err, (uint32_t)tp.split, (uint32_t)tp.t_tiles);
}

template <bool GATED, typename T>
static cudaError_t launch_i8_tc_t(I8TcPlan const &tp, CUtensorMap const &mc, CUtensorMap const &mt,
                                  I8Params const &p, I8Ptrs const &a, uint32_t *err, cudaStream_t st) {
  switch (tp.tokens) {
    case 0: return launch_pair<GATED, T>(tp, mc, mt, p, a, err, st);
    case 16: return launch_split<16, GATED, T>(tp, mc, mt, p, a, err, st);
    case 32: return launch_split<32, GATED, T>(tp, mc, mt, p, a, err, st);
    case 64: return launch_split<64, GATED, T>(tp, mc, mt, p, a, err, st);
    case 128: return launch_split<128, GATED, T>(tp, mc, mt, p, a, err, st);
    default: return cudaErrorInvalidValue;
  }
}

int i8_box_tokens(I8TcPlan const &tp, bool gated) { return tp.tokens ? tp.tokens : (gated ? 64 : 128); }

cudaError_t launch_i8_tc(I8TcPlan const &tp, CUtensorMap const &mc, CUtensorMap const &mt, I8Params const &p,
                         I8Ptrs const &a, uint32_t *err, cudaStream_t st) {
  const bool gated = p.act == EIR_ACT_GATED_SILU;
  if (p.dt_out == EIR_BF16)
    return gated ? launch_i8_tc_t<true, __nv_bfloat16>(tp, mc, mt, p, a, err, st)
                 : launch_i8_tc_t<false, __nv_bfloat16>(tp, mc, mt, p, a, err, st);
  return gated ? launch_i8_tc_t<true, float>(tp, mc, mt, p, a, err, st)
               : launch_i8_tc_t<false, float>(tp, mc, mt, p, a, err, st);
}

}  // namespace eir
