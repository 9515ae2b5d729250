// Contraction of 8-bit integers on the tcgen05 tensor cores (kind::i8).
//
// acc[t, c] = sum_k left[t, k] right[c, k] in 32-bit integers, which are exact
// in any order; the epilogue scales, adds the bias and applies the activation
// in FP32 and rounds once. The channels (right rows) are the MMA's M side and
// the tokens its N side: an epilogue thread then owns one channel (its scale
// and bias stay in registers), a warp stores neighbouring channels of a token
// together, and a single token is an MMA of N = 16 that costs nothing beside
// the weights' bytes. A gated layer interleaves 16 gate rows and their 16 value
// rows in the staged tile (one box of a 3-D tensor map), so that lanes l and
// l + 16 of a warp hold a gate and its value: one shuffle joins them, the MMAs are
// those of a plain layer, and only the activated product is written.
//
// Two kernels:
// * i8_pair_kernel: CTA pairs (cta_group::2) over tiles of 256 rows x 256
//   tokens, persistent, accumulators double-buffered in TMEM so that the
//   epilogue runs under the next tile.
// * i8_split_kernel: one tile of 128 rows x NT tokens (NT = 16 .. 128; 77 tokens x 32768 x 1024
//   take 9.9 us in tiles of 128, 9.1 in tiles of 80) for
//   problems with too few pair tiles to fill the GPU. A cluster of 1 to 8 CTAs
//   shares the tile's K walk; each holds a partial accumulator, and the
//   cluster adds them through distributed shared memory.
// Measured on one B200: pair tiles 8192 x 4096 x 4096 with bias and ReLU 90 us at full clock and 105 us (2.6 P
// operations a second) in a loop, where the 1000 W power cap holds the clock near 1.4 GHz; split tiles
// 77 tokens x 4096 x 10922 gated 13.7 us (45 MB of weights, 3.3 TB/s).
// Both stage 128-byte swizzled K rows with TMA (out-of-range rows and K read
// as zeros) in a ring of mbarrier stages. Every wait is bounded; a wait that
// gives up raises the CTA's (or pair's) abort flag and records a device error.
#include <cuda.h>
#include <algorithm>
#include <atomic>
#include "eir_launch.h"
#include "i8_common.cuh"

namespace eir {

constexpr int kI8Rows = 128;                      // staged right rows of a CTA
constexpr int kI8BlockK = 128;                    // K of a block: one swizzle row
constexpr int kI8SubBytes = kI8Rows * kI8BlockK;  // a block of 128 rows
constexpr int kI8Chunk = 32;                      // tokens the pair kernel drains from TMEM at a time

// output channels of a CTA's 128 rows
template <bool GATED>
__host__ __device__ constexpr int i8_channels() {
  return GATED ? kI8Rows / 2 : kI8Rows;
}
// the output channel of tile row `row` (of a tile whose first channel is c0),
// and whether the row is a value row
template <bool GATED>
__device__ __forceinline__ int64_t i8_row_channel(int64_t c0, int row) {
  return GATED ? c0 + (row >> 5) * 16 + (row & 15) : c0 + row;
}

// one K block of the 128 right rows from channel c0 on into `dst`
template <bool GATED, typename Load2, typename Load3>
__device__ __forceinline__ void i8_load_rows(uint8_t *dst, int k, int c0, Load2 load2, Load3 load3) {
  if (!GATED) {
    load2(dst, k, c0);
  } else {
#pragma unroll
    for (int b = 0; b < 4; ++b) load3(dst + b * 32 * kI8BlockK, k, c0 + 16 * b);
  }
}

// The epilogue's row side, held by the thread that owns the tile row: its
// channel's scale and bias
struct I8Row {
  float sb, bias;
};
template <bool GATED>
__device__ __forceinline__ I8Row i8_row(I8Params const &p, I8Ptrs const &a, int64_t c, int row, int64_t n_out) {
  I8Row h{1.f, 0.f};
  if (c >= n_out) return h;
  const int64_t r = c + (GATED && (row & 16) ? n_out : 0);
  if (a.scale_r) h.sb = a.scale_r[r];
  if (a.bias) h.bias = a.bias[r];
  return h;
}

// accumulators of a thread's row (tokens 0 .. CH - 1), scaled
template <int CH>
__device__ __forceinline__ void i8_scale_row(uint32_t const (&v)[CH], float const *scale, I8Row const &h,
                                             float (&z)[CH]) {
#pragma unroll
  for (int i = 0; i < CH; i += 4) {
    const float4 s = *reinterpret_cast<float4 const *>(scale + i);
    const float2 z0 = scaled2((int32_t)v[i], (int32_t)v[i + 1], make_float2(s.x, s.y), h.sb, h.bias);
    const float2 z1 = scaled2((int32_t)v[i + 2], (int32_t)v[i + 3], make_float2(s.z, s.w), h.sb, h.bias);
    z[i] = z0.x;
    z[i + 1] = z0.y;
    z[i + 2] = z1.x;
    z[i + 3] = z1.y;
  }
}

// how a warp stores its rows: fixed for a kernel's call, or for a tile
struct I8Store {
  bool relu;
  bool words;         // two channels a 4-byte store (BF16, even rows, base on a word)
  uint32_t step[4];   // byte offsets of the tokens 2, 4, 6, 8 (x 2 when gated) after the first, below 2^32
};
template <bool GATED, typename T>
__device__ __forceinline__ I8Store i8_store_mode(I8Params const &p, I8Ptrs const &a) {
  I8Store m;
  constexpr int64_t kStep = (GATED ? 4 : 2) * sizeof(T);
  m.relu = p.act == EIR_ACT_RELU;
  m.words = sizeof(T) == 2 && p.s_out % 2 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 3) == 0 &&
            p.s_out < (1 << 26);
#pragma unroll
  for (int i = 0; i < 4; ++i) m.step[i] = (uint32_t)((i + 1) * kStep * p.s_out);
  return m;
}

// Stores a warp's 32 rows x CH tokens. Gated: lanes l and l + 16 first trade
// halves of their tokens, so that lane l holds gate and value of the even
// tokens and lane l + 16 of the odd ones. BF16 on even rows: lanes 2j and
// 2j + 1 then trade tokens too and store two channels in one word (half the
// store instructions of one channel a lane).
//   out: the first token's row; c: the lane's channel; tokens: how many exist
template <bool GATED, typename T, int CH>
__device__ __forceinline__ void i8_store_chunk(T *out, int64_t stride, float (&z)[CH], int64_t c, int64_t n_out,
                                               int tokens, I8Store const &m) {
  constexpr int N = GATED ? CH / 2 : CH, STEP = GATED ? 2 : 1;  // token of w[j]: STEP j + first
  const int lane = threadIdx.x & 31, first = GATED ? lane >> 4 : 0;
  float w[N];
  if (GATED) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float got = __shfl_xor_sync(0xffffffffu, first ? z[2 * j] : z[2 * j + 1], 16);
      w[j] = first ? silu(got) * z[2 * j + 1] : silu(z[2 * j]) * got;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = z[j];
  }
  const int odd = lane & 1;
  if (sizeof(T) == 2 && m.words && tokens >= CH && __all_sync(0xffffffffu, c - odd + 1 < n_out)) {
    const uint32_t pick = odd ? 0x3276u : 0x5410u;
    // the rounding is monotone, so the ReLU may follow it
    const __nv_bfloat162 low = __float2bfloat162_rn(m.relu ? 0.f : -INFINITY);
    char *o = reinterpret_cast<char *>(out + (first + (odd ? STEP : 0)) * stride + c - odd);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      __nv_bfloat162 b = __floats2bfloat162_rn(w[j], w[j + 1]);
      if (!GATED) b = __hmax2_nan(b, low);
      const uint32_t mine = *reinterpret_cast<uint32_t const *>(&b);
      const uint32_t both = __byte_perm(mine, __shfl_xor_sync(0xffffffffu, mine, 1), pick);
      *reinterpret_cast<uint32_t *>(o + (j % 8 ? m.step[j % 8 / 2 - 1] : 0u)) = both;
      if (j % 8 == 6) o += m.step[3];
    }
  } else if (c < n_out) {
    const float low = m.relu ? 0.f : -INFINITY;
    T *o = out + first * stride + c;
#pragma unroll
    for (int j = 0; j < N; ++j, o += STEP * stride)
      if (STEP * j + first < tokens) *o = from_f32<T>(GATED ? w[j] : relu_from(w[j], low));
  }
}

// ---------------------------------------------------------------- CTA pairs

struct I8Pair {
  static constexpr int kTokens = 256;                    // tokens of a tile (N of the MMA)
  static constexpr int kSub = 2;                         // K blocks of a stage
  static constexpr int kBSub = kTokens / 2 * kI8BlockK;  // each CTA stages half of the tokens
  static constexpr int kABytes = kSub * kI8SubBytes, kBBytes = kSub * kBSub;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = (232448 - 1024 - 5120) / kStageBytes;
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = 32 * (2 + kEpiWarps);
  static constexpr int kWarpTokens = kTokens / 2;  // columns of one epilogue warp
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + 5120;
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
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(I8Pair::kThreads, 1)
    i8_pair_kernel(const __grid_constant__ CUtensorMap map_c, const __grid_constant__ CUtensorMap map_t,
                   const I8Params p, const I8Ptrs a, uint32_t *err, uint32_t c_tiles, uint32_t t_tiles) {
  using Cfg = I8Pair;
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
        const int c0 = (int)((2 * ct + rank) * i8_channels<GATED>());
        const int row_t = (int)(tt * Cfg::kTokens + rank * (Cfg::kTokens / 2));
        for (int kb = 0; kb < k_blocks; kb += Cfg::kSub) {
          if (!mbar_wait_bounded(&empty[stage], phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          const int subs = min(Cfg::kSub, k_blocks - kb);
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * subs * (kI8SubBytes + Cfg::kBSub));
          const uint32_t bar = full_leader + 8u * (uint32_t)stage;
          for (int sub = 0; sub < subs; ++sub) {
            const int k = (kb + sub) * kI8BlockK;
            i8_load_rows<GATED>(
                sA + stage * Cfg::kABytes + sub * kI8SubBytes, k, c0,
                [&](void *dst, int x, int y) { tma_load_2d_pair(dst, &map_c, bar, x, y); },
                [&](void *dst, int x, int y) { tma_load_3d_pair(dst, &map_c, bar, x, y, 0); });
            tma_load_2d_pair(sB + stage * Cfg::kBBytes + sub * Cfg::kBSub, &map_t, bar, k, row_t);
          }
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
      // descriptors: the stage's address moves the low word only
      const uint64_t a_desc = make_smem_desc(smem_u32(sA), 16, 1024, kLayoutSw128);
      const uint64_t b_desc = make_smem_desc(smem_u32(sB), 16, 1024, kLayoutSw128);
      bool ready = false;  // the stage's loads have already been seen to be complete
      for (uint32_t t = pair_id; t < tiles && ok; t += n_pairs) {
        if (!mbar_wait_bounded(&tempty[acc], acc_phase ^ 1u, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + (uint32_t)(acc * Cfg::kTokens);
        for (int kb = 0; kb < k_blocks; kb += Cfg::kSub) {
          if (!ready && !mbar_wait_bounded(&full[stage], phase, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t ad = a_desc + (uint32_t)(stage * (Cfg::kABytes >> 4));
          const uint64_t bd = b_desc + (uint32_t)(stage * (Cfg::kBBytes >> 4));
          const int next = stage + 1 == S ? 0 : stage + 1;
          const uint32_t next_phase = stage + 1 == S ? phase ^ 1u : phase;
          const bool tail = kb + Cfg::kSub > k_blocks;
#pragma unroll
          for (int sub = 0; sub < Cfg::kSub; ++sub) {
            if (sub > 0 && tail && kb + sub >= k_blocks) break;
#pragma unroll
            for (int kk = 0; kk < kI8BlockK / 32; ++kk) {
              const uint32_t off_a = (sub * kI8SubBytes + kk * 32) >> 4, off_b = (sub * Cfg::kBSub + kk * 32) >> 4;
              umma_i8_pair(d, ad + off_a, bd + off_b, idesc, (sub > 0 || kk > 0) ? 1u : (kb > 0 ? 1u : 0u));
              // the next stage's barrier is looked at while the tensor cores have work queued: waiting for it
              // after the commit left them idle (8192 x 4096 x 4096: 154 k cycles against 147 k)
              if (kk == 1 && sub == 0) ready = mbar_test_wait(&full[next], next_phase);
            }
          }
          umma_commit_pair(smem_u32(&empty[stage]));
          umma_commit_pair(empty_peer + 8u * (uint32_t)stage);
          stage = next;
          phase = next_phase;
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
    const I8Store mode = i8_store_mode<GATED, T>(p, a);
    const int row = q * 32 + lane;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (uint32_t t = pair_id; t < tiles; t += n_pairs) {
      uint32_t ct, tt;
      i8_pair_tile(t, c_tiles, t_tiles, ct, tt);
      const int64_t c = i8_row_channel<GATED>((int64_t)(2 * ct + rank) * i8_channels<GATED>(), row);
      const int64_t t0 = (int64_t)tt * Cfg::kTokens + col0;
      // the tile's scales are fetched under its MMAs
      const I8Row h = i8_row<GATED>(p, a, c, row, n_out);
      __syncwarp();
      for (int i = lane; i < Cfg::kWarpTokens; i += 32)
        scale[i] = a.scale_l && t0 + i < p.m ? a.scale_l[t0 + i] : 1.f;
      __syncwarp();
      if (!mbar_wait_warp(&tfull[acc], acc_phase, abort_flag)) {
        if (lane == 0) raise_abort(kErrTimeoutEpilogue);
        break;
      }
      tc_fence_after();
      // the accumulator back to the MMAs once it is in registers. The arrive is relaxed: the
      // tcgen05 fence orders it after the TMEM reads, and a release would wait
      // for the tile's global stores too
      auto release_acc = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(tempty_leader + 8u * (uint32_t)acc);
      };
      T *out = static_cast<T *>(a.out) + t0 * p.s_out;
      const uint32_t src = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * Cfg::kTokens + col0);
      const int tokens = (int)min((int64_t)Cfg::kWarpTokens, p.m - t0);  // <= 0: none of the tile's
      uint32_t v[kI8Chunk];
      if (tokens > 0) tmem_ld_32x32b_x32(src, v);
#pragma unroll 1
      for (int ch = 0; ch < tokens; ch += kI8Chunk, out += kI8Chunk * p.s_out) {
        float z[kI8Chunk];
        tmem_ld_wait();
        i8_scale_row(v, scale + ch, h, z);
        if (ch + kI8Chunk < tokens) tmem_ld_32x32b_x32(src + ch + kI8Chunk, v);  // under this chunk's stores
        else release_acc();
        i8_store_chunk<GATED, T>(out, p.s_out, z, c, n_out, tokens - ch, mode);
      }
      if (tokens <= 0) release_acc();
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
  }

  // After an abort, copies or commits issued before it may still be landing in
  // this CTA's shared memory: give them time before the CTA can exit.
  if (threadIdx.x == 0 && *abort_flag) wait_for_copies();
  __syncwarp();
  tc_fence_before();
  cluster_sync();  // both CTAs done: no remote arrive or TMEM read is outstanding
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ---------------------------------------------------------------- split K over a cluster

template <int NT>
struct I8Split {
  static constexpr int kBBytes = NT * kI8BlockK;
  static constexpr int kStageBytes = kI8SubBytes + kBBytes;
  static constexpr int kAccBytes = NT * kI8Rows * 4;  // the exchanged accumulators
  // about 100 KB a CTA, two CTAs on an SM: enough bytes in flight for HBM
  static constexpr int kStages = 104 * 1024 / kStageBytes;
  static constexpr int kRing = kStages * kStageBytes;
  static constexpr int kCols = NT <= 32 ? 32 : NT <= 64 ? 64 : 128;  // TMEM
  static constexpr int kThreads = 192;
  static constexpr int kSmemBytes = 1024 + kRing + 512 + 512;
  static_assert(kAccBytes <= kRing, "the exchange reuses the ring");
};

__device__ __forceinline__ int4 ld_cluster_v4(uint32_t addr_cluster) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr_cluster)
               : "memory");
  return v;
}

template <int NT, bool GATED, typename T>
__global__ void __launch_bounds__(192, 2)
    i8_split_kernel(const __grid_constant__ CUtensorMap map_c, const __grid_constant__ CUtensorMap map_t,
                    const I8Params p, const I8Ptrs a, uint32_t *err, uint32_t split, uint32_t t_tiles) {
  using Cfg = I8Split<NT>;
  constexpr int S = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sA = smem, *sB = smem + S * kI8SubBytes;
  int32_t *s_acc = reinterpret_cast<int32_t *>(smem);  // [token][row], after the last MMA
  float *s_scale = reinterpret_cast<float *>(smem + Cfg::kRing);  // the tile's token scales
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + Cfg::kRing + 512);
  uint64_t *full = bars, *empty = bars + S, *tfull = bars + 2 * S;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * S + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = split > 1 ? cluster_ctarank() : 0u;
  const uint32_t tile = blockIdx.x / split, ct = tile / t_tiles, tt = tile % t_tiles;
  const int k_blocks = (int)((p.k + kI8BlockK - 1) / kI8BlockK);
  const int kb0 = (int)((int64_t)k_blocks * rank / split), kb1 = (int)((int64_t)k_blocks * (rank + 1) / split);
  const int64_t n_out = GATED ? p.n / 2 : p.n, c0 = (int64_t)ct * i8_channels<GATED>();

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
  if (threadIdx.x == 0) {
    // the channels' rows of the first ring set out for L2 while the kernels before this one end
    // (4 tokens x 32768 x 4096: 23.3 us, 23.9 without; of more K blocks: slower)
    for (int kb = kb0; kb < min(kb1, kb0 + S); ++kb)
      i8_load_rows<GATED>(
          sA, kb * kI8BlockK, (int)c0, [&](void *, int x, int y) { tma_prefetch_2d(&map_c, x, y); },
          [&](void *, int x, int y) { tma_prefetch_3d(&map_c, x, y, 0); });
  }
  pdl_wait();

  const int64_t t0 = (int64_t)tt * NT;
  const int tokens = (int)min((int64_t)NT, p.m - t0);
  const float low = p.act == EIR_ACT_RELU ? 0.f : -INFINITY;
  bool ok = true;  // this thread's view: false once a wait of the CTA has given up
  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&empty[stage], phase ^ 1u, abort_flag)) {
          ok = false;
          break;
        }
        uint64_t *bar = &full[stage];
        mbar_arrive_expect_tx(bar, Cfg::kStageBytes);
        i8_load_rows<GATED>(
            sA + stage * kI8SubBytes, kb * kI8BlockK, (int)c0,
            [&](void *dst, int x, int y) { tma_load_2d(dst, &map_c, bar, x, y); },
            [&](void *dst, int x, int y) { tma_load_3d(dst, &map_c, bar, x, y, 0); });
        tma_load_2d(sB + stage * Cfg::kBBytes, &map_t, bar, kb * kI8BlockK, (int)t0);
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
      const uint64_t a_desc = make_smem_desc(smem_u32(sA), 16, 1024, kLayoutSw128);
      const uint64_t b_desc = make_smem_desc(smem_u32(sB), 16, 1024, kLayoutSw128);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&full[stage], phase, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t ad = a_desc + (uint32_t)(stage * (kI8SubBytes >> 4));
        const uint64_t bd = b_desc + (uint32_t)(stage * (Cfg::kBBytes >> 4));
#pragma unroll
        for (int kk = 0; kk < kI8BlockK / 32; ++kk)
          umma_i8(tmem_base, ad + kk * 2, bd + kk * 2, idesc, kk > 0 ? 1u : (kb > kb0 ? 1u : 0u));
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
  } else {
    for (int i = threadIdx.x - 64; i < NT; i += 128) s_scale[i] = a.scale_l && i < tokens ? a.scale_l[t0 + i] : 1.f;
    asm volatile("bar.sync 1, 128;" ::: "memory");  // the four epilogue warps
  }
  // the row side of this thread's outputs, fetched under the MMAs: of its TMEM
  // row, or of the four rows that it adds up for the cluster
  const int q = warp & 3, row = q * 32 + lane;
  const int64_t c = i8_row_channel<GATED>(c0, row);
  I8Row h[4];
  if (split == 1) {
    if (warp >= 2) h[0] = i8_row<GATED>(p, a, c, row, n_out);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      h[e] = i8_row<GATED>(p, a, i8_row_channel<GATED>(c0, 4 * lane + e), 4 * lane + e, n_out);
  }
  __syncwarp();
  // every warp waits for the accumulators: the ring is free for the exchange, and nothing is in
  // flight when the CTA ends
  int waited = 1;
  if (lane == 0) waited = mbar_wait_bounded(tfull, 0u, abort_flag);
  waited = __shfl_sync(0xffffffffu, waited, 0);
  if (waited) (void)mbar_try_wait(tfull, 0u);  // every lane observes the completed phase itself
  if (!waited && lane == 0 && !*abort_flag) {
    record_error(err, kErrTimeoutEpilogue);
    *abort_flag = 1;
  }
  __syncwarp();
  // (one answer for the warp, whatever another one writes meanwhile: the reads of TMEM below take all lanes)
  if (__any_sync(0xffffffffu, *abort_flag != 0)) {
    wait_for_copies();
    ok = false;
  }
  __syncwarp();
  tc_fence_after();
  const uint32_t src = tmem_base + ((uint32_t)(q * 32) << 16);
  if (split == 1) {
    if (warp >= 2 && ok) {
      const I8Store mode = i8_store_mode<GATED, T>(p, a);
      T *out = static_cast<T *>(a.out) + t0 * p.s_out;
#pragma unroll 1
      for (int ch = 0; ch < tokens; ch += 16, out += 16 * p.s_out) {
        uint32_t v[16];
        float z[16];
        tmem_ld_32x32b_x16(src + ch, v);
        tmem_ld_wait();
        i8_scale_row(v, s_scale + ch, h[0], z);
        i8_store_chunk<GATED, T>(out, p.s_out, z, c, n_out, tokens - ch, mode);
      }
    }
  } else {
    if (warp >= 2 && ok) {
#pragma unroll 1
      for (int ch = 0; ch < tokens; ch += 16) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(src + ch, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) s_acc[(ch + i) * kI8Rows + row] = (int32_t)v[i];
      }
    }
    __syncwarp();
    cluster_sync();  // every CTA's partial sums are in its shared memory
    // CTA `rank` adds up and stores every split-th token, a warp a token, four rows a lane
    if (ok) {
      const bool value = GATED && (lane & 4) != 0;  // lanes l and l + 4: a gate and its value
      const int64_t cq = i8_row_channel<GATED>(c0, 4 * lane);
      const uint32_t at = smem_u32(s_acc) + 16u * (uint32_t)lane;
      T *out = static_cast<T *>(a.out) + t0 * p.s_out + cq;
      const bool wide = p.s_out % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % (4 * sizeof(T)) == 0 && cq + 4 <= n_out;
      auto finish = [&](int j, int4 const &acc) {
        const float sa = s_scale[j];
        float z[4] = {i8_scaled(acc.x, sa, h[0].sb, h[0].bias), i8_scaled(acc.y, sa, h[1].sb, h[1].bias),
                      i8_scaled(acc.z, sa, h[2].sb, h[2].bias), i8_scaled(acc.w, sa, h[3].sb, h[3].bias)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (GATED) z[e] = silu(z[e]) * __shfl_xor_sync(0xffffffffu, z[e], 4);
          else z[e] = relu_from(z[e], low);
        }
        if (value) return;
        T *o = out + j * p.s_out;
        if (wide) {
          if (sizeof(T) == 2) {
            const __nv_bfloat162 lo = __floats2bfloat162_rn(z[0], z[1]), hi = __floats2bfloat162_rn(z[2], z[3]);
            *reinterpret_cast<uint2 *>(o) = make_uint2(*reinterpret_cast<uint32_t const *>(&lo),
                                                       *reinterpret_cast<uint32_t const *>(&hi));
          } else {
            *reinterpret_cast<float4 *>(o) = make_float4(z[0], z[1], z[2], z[3]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (cq + e < n_out) o[e] = from_f32<T>(z[e]);
        }
      };
      // two tokens' reads (of up to four CTAs) are under way before the first is added
      const int step = 6 * (int)split;
      for (int j = (int)rank + warp * (int)split; j < tokens; j += 2 * step) {
        int4 acc[2] = {make_int4(0, 0, 0, 0), make_int4(0, 0, 0, 0)};
        const bool second = j + step < tokens;
        for (uint32_t r0 = 0; r0 < split; r0 += 4) {
          int4 v[2][4];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r)
              v[i][r] = r0 + r < split && (i == 0 || second)
                            ? ld_cluster_v4(mapa_shared(at + (uint32_t)((j + i * step) * kI8Rows * 4), r0 + r))
                            : make_int4(0, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              acc[i].x += v[i][r].x;
              acc[i].y += v[i][r].y;
              acc[i].z += v[i][r].z;
              acc[i].w += v[i][r].w;
            }
        }
        finish(j, acc[0]);
        if (second) finish(j + step, acc[1]);
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

template <bool GATED, typename T>
static cudaError_t launch_pair(I8TcPlan const &tp, CUtensorMap const &mc, CUtensorMap const &mt, I8Params const &p,
                               I8Ptrs const &a, uint32_t *err, cudaStream_t st) {
  using Cfg = I8Pair;
  auto kern = i8_pair_kernel<GATED, T>;
  cudaError_t e = allow_all_smem(reinterpret_cast<void const *>(kern));
  if (e != cudaSuccess) return e;
  static std::atomic<int> clusters[32] = {};  // per device: pairs that can run at once
  int dev = 0;
  e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  int most = dev < 32 ? clusters[dev].load() : 0;
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
  using Cfg = I8Split<NT>;
  auto kern = i8_split_kernel<NT, GATED, T>;
  cudaError_t e = allow_all_smem(reinterpret_cast<void const *>(kern));
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
    case 80: return launch_split<80, GATED, T>(tp, mc, mt, p, a, err, st);
    case 96: return launch_split<96, GATED, T>(tp, mc, mt, p, a, err, st);
    case 128: return launch_split<128, GATED, T>(tp, mc, mt, p, a, err, st);
    default: return cudaErrorInvalidValue;
  }
}

int i8_box_tokens(I8TcPlan const &tp) { return tp.tokens ? tp.tokens : I8Pair::kTokens / 2; }

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
