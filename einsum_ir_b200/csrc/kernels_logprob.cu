// Log probabilities of given tokens, log-sum-exp, entropy and top alternatives
// of rows of logits, and the gradient of the first and third.
//
// One pass over a row, in base 2 (L = log2 e): with the row's maximum m, S = sum 2^d and U = sum d 2^d
// for d = (x - m) L give lse = m + log2 S / L, log p = x - m - log2 S / L and entropy = (log2 S - U / S) / L.
// The pass itself takes d = x L - R, one instruction, with a reference R near m L: any will do, so that R may be
// rounded, and a thread that meets a larger logit raises its own and shrinks its sums by 2^(R - R'). Its sums
// move to its exact maximum at the end. Logits are floored at -2^21, where 2^d is 0 for every m of
// at least -2^20, so that a ruled-out one (-infinity, or a large finite value) adds 0 d = 0 to U. R is off by 2^-4 at
// most for |m| <= 2^20 (from 1.5e9 on its rounding could take 2^d out of FP32's range): the sums of rows
// whose maximum lies beyond are taken once more, as differences to it.
//
// At BF16 no unit is full (4096 x 32768 without alternatives: 53 us, 5.1 TB/s; issue 63 %, exponentials 57 % of
// their rate, HBM 65 % of its peak; with 5 alternatives 61 us, 59, 49 and 57 %: the steps at a row's end keep most of
// a block's warps waiting). FP32 is bound by HBM (4096 x 32768, 5 alternatives: 105 us, 5.1 TB/s). A logit is read once. A piece is 16 bytes of memory on
// the 16-byte grid, so rows of any alignment stream alike; the elements of
// the first and last piece that lie outside the row count as ruled out.
//
// Top alternatives without a second pass: each thread keeps its largest logit, the
// piece it came from, and the largest logit of its other chunks. The k-th largest of the threads'
// logits (ties: the earlier piece) is a lower bound of the row's k-th largest, and only the k threads that
// hold larger ones can hold an alternative: the chunk of their largest logit is read again (4 pieces of
// 16 bytes), their other chunks only where the largest logit of these reaches the bound too (all
// chunks: 65.8 us instead of 61.4 for 4096 x 32768 BF16 and 5 alternatives, 95 instead of 77
// for 20; a looser bound from fewer maxima that each thread compares with its own: 81 and 133).
// The few candidates above the bound are sorted. Order by one 64-bit key,
// logit first and lower index second, so that the result does not depend on the order of work.
//
// Rows that do not fill the GPU by number are split over a cluster of up to 8 blocks, joined
// through distributed shared memory.
//
// Rows with a NaN or +infinity, or with more candidates than their buffer holds, are redone by
// logprob_plain_row: a pass for each value.
//
// Backward: dx = dlogprob (onehot - p) - dentropy p (x - lse + H), bound by HBM (2048 x 50021 BF16 with
// entropy 73 us, 5.6 TB/s).
#include <algorithm>
#include "eir_launch.h"
#include "eir_common.cuh"
#include "op_params.h"
#include "row_vec.cuh"

namespace eir {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -2097152.f;  // -2^21: logits below count as ruled out in the fast pass,
constexpr float kLargest = 1048576.f;  // 2^20: whose sums hold where the row's maximum is no larger than this

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// a logit's rank as an unsigned integer: the order of the floats, both zeros
// alike, NaNs highest; 0 is below every logit's
__device__ __forceinline__ uint32_t rank_bits(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float rank_value(uint32_t r) {
  if (r == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((r & 0x80000000u) ? r ^ 0x80000000u : ~r);
}
// rank and place in one word: larger logits first, then lower indices
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
  return ((uint64_t)rank_bits(x) << 32) | (uint32_t)~index;
}
__device__ __forceinline__ uint64_t warp_max_key(uint64_t k) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return ((uint64_t)hi << 32) | lo;
}

__device__ __forceinline__ float logit_nan() { return __uint_as_float(0x7fc00000u); }

// a thread's reference (0 below kLowest, where S = 0)
__device__ __forceinline__ float log_ref(float m) { return m < kLowest ? 0.f : m * kLog2e; }
// A row's maximum, and its sums as differences to it
struct LogSums {
  float m, S, U;
};
__device__ __forceinline__ float log_prob(float x, LogSums const &v, float log_s) { return (x - v.m) - log_s * kLn2; }
// whether the pass's sums do not hold for a row with this maximum (+infinity: no sums do)
__device__ __forceinline__ bool log_again(float m) { return fabsf(m) > kLargest && fabsf(m) < INFINITY; }
// sums with distances from d on instead of 0 (a NaN stays in them)
__device__ __forceinline__ LogSums log_shifted(float m, float S, float U, float d) {
  const float e = exp2_fast(d);
  return LogSums{m, e * S, e * (U + d * S)};
}
// a thread's sums against R as those of its maximum m (sums of 0 may stand beside any R)
__device__ __forceinline__ LogSums log_of_pass(float R, float S, float U, float m) {
  return S == 0.f ? LogSums{m, 0.f, 0.f} : log_shifted(m, S, U, -fmaf(m, kLog2e, -R));
}
// sums moved to the larger maximum m (2^-300 is 0; -infinity less itself counts as that too)
__device__ __forceinline__ LogSums log_moved(LogSums const &v, float m) {
  return log_shifted(m, v.S, v.U, fmaxf((v.m - m) * kLog2e, -300.f));
}
// the sums of the warp's lanes
__device__ __forceinline__ LogSums log_join_lanes(LogSums v) {
  // (signed integers in the order of the floats; a NaN is no maximum here, but stays in S)
  const int b = __float_as_int(v.m == v.m ? v.m : -INFINITY);
  const int most = __reduce_max_sync(0xffffffffu, b ^ ((b >> 31) & 0x7fffffff));
  v = log_moved(v, __int_as_float(most ^ ((most >> 31) & 0x7fffffff)));
  v.S = warp_sum(v.S);
  v.U = warp_sum(v.U);
  return v;
}

// a row's target: its place (-1: left out; vocab: off the row) and its logit
struct LogTarget {
  int place;
  float x;
};
template <typename T>
__device__ __forceinline__ LogTarget log_target(LogprobParams const &p, LogprobPtrs const &a, int64_t row) {
  const int64_t t = a.targets ? a.targets[row] : -1;
  LogTarget g{t < 0 ? -1 : (int)(t < p.vocab ? t : p.vocab), 0.f};
  if (t >= 0 && t < p.vocab) g.x = to_f32(static_cast<T const *>(a.x)[row * p.s_x + t]);
  return g;
}

// one row's values, written by one thread
__device__ __forceinline__ void logprob_row_values(LogprobParams const &p, LogprobPtrs const &a, int64_t row, bool none,
                                                   float lse, float entropy, int target, float target_logprob) {
  if (a.lse) a.lse[row] = lse;
  if (a.entropy) a.entropy[row] = none ? 0.f : entropy;
  if (a.targets)
    a.logprob[row] = target < 0 ? 0.f : (target >= p.vocab ? logit_nan() : (none ? -INFINITY : target_logprob));
}

// A row by plain passes (all threads of the block): right for every row, a
// pass over it for each value. red: 3 x 32 words; best: 32 keys.
template <typename T>
__device__ __noinline__ void logprob_plain_row(LogprobParams const &p, LogprobPtrs const &a, int64_t row, float *red,
                                               uint64_t *best) {
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  T const *x = static_cast<T const *>(a.x) + row * p.s_x;
  float m = -INFINITY;
  for (int64_t c = threadIdx.x; c < p.vocab; c += blockDim.x) m = fmaxf(m, to_f32(x[c]));
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  __syncthreads();
  if (lane == 0) red[warp] = m;
  __syncthreads();
  for (int w = 0; w < warps; ++w) m = fmaxf(m, red[w]);
  const float ref = m == -INFINITY ? 0.f : m;
  float S = 0.f, U = 0.f;
  for (int64_t c = threadIdx.x; c < p.vocab; c += blockDim.x) {
    const float d = to_f32(x[c]) - ref, e = expf(d);
    S += e;
    U += d == -INFINITY ? 0.f : d * e;
  }
  S = warp_sum(S);
  U = warp_sum(U);
  if (lane == 0) {
    red[32 + warp] = S;
    red[64 + warp] = U;
  }
  __syncthreads();
  S = U = 0.f;
  for (int w = 0; w < warps; ++w) {
    S += red[32 + w];
    U += red[64 + w];
  }
  const bool none = S == 0.f;
  const float log_s = logf(S);
  if (threadIdx.x == 0) {
    const LogTarget t = log_target<T>(p, a, row);
    logprob_row_values(p, a, row, none, none ? -INFINITY : ref + log_s, log_s - U / S, t.place, t.x - ref - log_s);
  }
  uint64_t last = ~0ull;
  for (int i = 0; i < p.top; ++i) {
    uint64_t k = 0;
    for (int64_t c = threadIdx.x; c < p.vocab; c += blockDim.x) {
      const uint64_t key = rank_key(to_f32(x[c]), (uint32_t)c);
      if (key < last || i == 0) k = key > k ? key : k;
    }
    k = warp_max_key(k);
    __syncthreads();
    if (lane == 0) best[warp] = k;
    __syncthreads();
    for (int w = 0; w < warps; ++w) k = best[w] > k ? best[w] : k;
    last = k;
    if (threadIdx.x == 0) {
      const uint32_t at = ~(uint32_t)k;
      if (a.top_index) a.top_index[row * p.top + i] = at;
      if (a.top_logprob) a.top_logprob[row * p.top + i] = none ? -INFINITY : to_f32(x[at]) - ref - log_s;
    }
  }
  __syncthreads();
}

// a row's pieces: 16-byte units of memory that hold some of its elements
template <typename T>
struct LogitRow {
  static constexpr int V = 16 / (int)sizeof(T);
  using Piece = RowPiece<T, V>;
  uint8_t const *base;  // the first unit
  int off;              // elements of it before the row
  int vocab;
  int pieces;
  __device__ __forceinline__ LogitRow(T const *x, int64_t n) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(x);
    base = reinterpret_cast<uint8_t const *>(at & ~(uintptr_t)15);
    off = (int)(at & 15) / (int)sizeof(T);
    vocab = (int)n;
    pieces = (int)((n + off + V - 1) / V);
  }
  __device__ __forceinline__ int first_index(int piece) const { return piece * V - off; }
  // a piece; elements outside the row are -infinity
  __device__ __forceinline__ Piece load(int piece) const {
    Piece v;
    const int i0 = first_index(piece);
    if (i0 >= 0 && i0 <= vocab - V) {
      v.template load<false>(base + (int64_t)piece * 16);
    } else {
#pragma unroll
      for (int i = 0; i < Piece::kWords; ++i) v.w[i] = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
      T const *x = reinterpret_cast<T const *>(base) + off;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (i0 + e < 0 || i0 + e >= vocab) continue;
        if constexpr (sizeof(T) == 4) v.w[e] = *reinterpret_cast<uint32_t const *>(x + i0 + e);
        else {
          const uint32_t b = *reinterpret_cast<unsigned short const *>(x + i0 + e);
          v.w[e / 2] = e % 2 ? (v.w[e / 2] & 0x0000ffffu) | b << 16 : (v.w[e / 2] & 0xffff0000u) | b;
        }
      }
    }
    return v;
  }
  static __device__ __forceinline__ Piece none() {
    Piece v;
#pragma unroll
    for (int i = 0; i < Piece::kWords; ++i) v.w[i] = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
    return v;
  }
  // the piece with its elements not below kLowest (NaNs stay), so that none is infinitely far below the reference
  static __device__ __forceinline__ Piece floored(Piece v) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v.w[i] = __float_as_uint(max_nan(v.get(i), kLowest));
    } else {
      const __nv_bfloat162 low = __float2bfloat162_rn(kLowest);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __hmax2_nan(*reinterpret_cast<__nv_bfloat162 const *>(&v.w[i]), low);
        v.w[i] = *reinterpret_cast<uint32_t const *>(&b);
      }
    }
    return v;
  }
  // the largest element (a NaN counts as absent)
  static __device__ __forceinline__ float largest(Piece const &v) {
    if constexpr (sizeof(T) == 4) {
      return fmaxf(fmaxf(v.get(0), v.get(1)), fmaxf(v.get(2), v.get(3)));
    } else {
      __nv_bfloat162 b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = *reinterpret_cast<__nv_bfloat162 const *>(&v.w[i]);
      const __nv_bfloat162 m = __hmax2(__hmax2(b[0], b[1]), __hmax2(b[2], b[3]));
      return fmaxf(__low2float(m), __high2float(m));
    }
  }
};

// The sums of pieces p0 .. p1 - 1 of a row whose maximum m is large, as differences to it (all threads of the
// block; each gets them): 4096 x 32768 BF16 with 5 alternatives takes 62.3 us where 1 in 100 rows holds nothing but
// -1e30, 112 where all do, 62.0 where none does. red: 2 x 32 words
template <typename T>
__device__ __noinline__ LogSums log_large_row(LogitRow<T> const x, int p0, int p1, float m, float *red) {
  constexpr int V = LogitRow<T>::V, AT_ONCE = 4;
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float2 S = make_float2(0.f, 0.f), U = make_float2(0.f, 0.f);
  for (int q = p0 + (int)threadIdx.x; q < p1; q += AT_ONCE * (int)blockDim.x) {
    typename LogitRow<T>::Piece c[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int at = q + i * (int)blockDim.x;
      c[i] = at < p1 ? x.load(at) : LogitRow<T>::none();
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        float2 d = mul2(add2(c[i].get2(e), make_float2(-m, -m)), make_float2(kLog2e, kLog2e));
        d = make_float2(max_nan(d.x, -200.f), max_nan(d.y, -200.f));  // 2^-200 is 0
        const float2 t = make_float2(exp2_fast(d.x), exp2_fast(d.y));
        S = add2(S, t);
        U = fma2(d, t, U);
      }
  }
  LogSums v{m, warp_sum(S.x + S.y), warp_sum(U.x + U.y)};
  __syncthreads();
  if (lane == 0) {
    red[warp] = v.S;
    red[32 + warp] = v.U;
  }
  __syncthreads();
  v.S = warp_sum(lane < warps ? red[lane] : 0.f);
  v.U = warp_sum(lane < warps ? red[32 + lane] : 0.f);
  return v;
}

// the sums of a cluster's blocks, each lane a block's
__device__ __forceinline__ LogSums log_join_blocks(LogSums const *at, uint32_t blocks) {
  LogSums w{-INFINITY, 0.f, 0.f};
  if ((threadIdx.x & 31) < blocks) {
    const uint32_t sums = mapa_shared(smem_u32(at), threadIdx.x & 31);
    w = LogSums{__uint_as_float(ld_cluster_u32(sums)), __uint_as_float(ld_cluster_u32(sums + 4)),
                __uint_as_float(ld_cluster_u32(sums + 8))};
  }
  return log_join_lanes(w);
}
// the same for a row in parts, by all blocks of the cluster
template <typename T>
__device__ __noinline__ LogSums log_large_blocks(LogitRow<T> const x, int p0, int p1, float m, float *red, LogSums *sums,
                                                 uint32_t blocks) {
  const LogSums part = log_large_row<T>(x, p0, p1, m, red);
  if (threadIdx.x == 0) *sums = part;
  __syncwarp();
  cluster_sync();
  const LogSums v = log_join_blocks(sums, blocks);
  __syncwarp();
  cluster_sync();  // no block ends while its sums are read
  return v;
}

constexpr int kLogStages = 2;  // of a warp, 2 KB each

__device__ __forceinline__ void bulk_copy(void *dst, void const *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <int THREADS>
struct LogShared {
  static constexpr int kCandidates = THREADS < 64 ? 256 : 4 * THREADS;  // (a merge of 8 blocks takes 8 x 32)
  float red[96];           // (m, S, U) of the warps; the plain row's words
  uint64_t keys[THREADS];  // the threads' largest logits
  float second[THREADS];   // and the largest ones of their other chunks
  uint64_t plain[32];      // the plain row's words
  uint64_t top[32];        // the block's alternatives
  uint64_t found[kCandidates];
  int n_found, full_up;    // candidates; more than fit
  volatile int abort;      // a bounded wait has given up
  LogSums sums;            // of the block
  float again;             // the row's maximum, where its sums are taken once more; 0: not so
  alignas(8) uint64_t full[THREADS / 32][kLogStages];
  alignas(128) uint8_t stages[THREADS / 32][kLogStages][2048];
};

// the largest of the warp's keys below `last`, PER of them a lane; 0: none
template <int PER>
__device__ __forceinline__ uint64_t next_largest(uint64_t const (&keys)[PER], uint64_t last) {
  uint64_t best = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (keys[i] < last && keys[i] > best) best = keys[i];
  return warp_max_key(best);
}
// the `k` largest of `n` keys in shared memory by one warp, into lane i's answer (0 where there are fewer)
__device__ __forceinline__ uint64_t pick_largest(uint64_t const *keys, int n, int k) {
  const int lane = threadIdx.x & 31;
  uint64_t last = ~0ull, mine = 0;
  if (n <= 64) {
    const uint64_t two[2] = {lane < n ? keys[lane] : 0, lane + 32 < n ? keys[lane + 32] : 0};
    for (int i = 0; i < k; ++i) {
      last = next_largest<2>(two, last);
      if (lane == i) mine = last;
    }
    return mine;
  }
  for (int i = 0; i < k; ++i) {
    uint64_t best = 0;
    for (int j = lane; j < n; j += 32)
      if (keys[j] < last && keys[j] > best) best = keys[j];
    last = warp_max_key(best);
    if (lane == i) mine = last;
  }
  return mine;
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
    logprob_kernel(const LogprobParams p, const LogprobPtrs a, uint32_t blocks_a_row, uint32_t *err) {
  using Row = LogitRow<T>;
  using Piece = typename Row::Piece;
  constexpr int V = Row::V, AT_ONCE = 4, warps = THREADS / 32, kChunk = 32 * AT_ONCE;
  __shared__ LogShared<THREADS> sh;
  constexpr int kCandidates = LogShared<THREADS>::kCandidates;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) {
    for (int s = 0; s < kLogStages; ++s) mbar_init(&sh.full[warp][s], 1);
    fence_barrier_init();
    if (warp == 0) sh.abort = 0;
  }
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t rank = blocks_a_row > 1 ? cluster_ctarank() : 0u;
  // A warp takes every warps-th chunk of its block's part of a row. Chunks that lie inside the row come through
  // the warp's own stages, copied in bulk ahead of their use; the row's first and last
  // chunk are read piece by piece
  const int64_t row = blockIdx.x / blocks_a_row;
  const Row x(static_cast<T const *>(a.x) + row * p.s_x, p.vocab);
  const int p0 = (int)((int64_t)x.pieces * rank / blocks_a_row);
  const int p1 = (int)((int64_t)x.pieces * (rank + 1) / blocks_a_row);
  const int chunks = (p1 - p0 + kChunk - 1) / kChunk;
  const int inner0 = p0 == 0 ? 1 : 0, inner1 = (p1 == x.pieces ? p1 - 1 - p0 : p1 - p0) / kChunk;
  auto inner = [&](int k) { return k >= inner0 && k < inner1; };
  auto copy = [&](int k, int stage) {
    mbar_arrive_expect_tx(&sh.full[warp][stage], kChunk * 16);
    bulk_copy(sh.stages[warp][stage], x.base + (int64_t)(p0 + k * kChunk) * 16, kChunk * 16, &sh.full[warp][stage]);
  };
  if (lane == 0) {
    const int k0 = inner(warp) ? warp : warp + warps;  // the warp's first inner chunk, if it has any
    for (int s = 0; s < kLogStages; ++s)
      if (inner(k0 + s * warps)) copy(k0 + s * warps, s);
  }
  LogTarget target{-1, 0.f};  // (read now: the end of the row would wait for it twice)
  if (threadIdx.x == 0 && rank == 0) target = log_target<T>(p, a, row);
  uint32_t phases = 0;  // of the warp's stages
  int stage = 0;
  // ---- the pass
  LogSums v{-INFINITY, 0.f, 0.f};
  float2 S2 = make_float2(0.f, 0.f), U2 = make_float2(0.f, 0.f);
  // The reference stays while no logit is more than 5.5 above it (S grows by 2^8 at most, which
  // costs U / S 2^-21 of rounding): a new maximum, which some lane meets in most
  // chunks, then is no branch
  float R = 0.f, limit = -INFINITY;
  int best = p0 + warp * kChunk + lane;  // the piece that holds v.m
  float second = -INFINITY;  // the largest logit of the thread's other chunks
  auto add_pieces = [&](Piece const (&c)[AT_ONCE], int q) {
    float l[AT_ONCE], most = -INFINITY;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      l[i] = Row::largest(c[i]);
      most = fmaxf(most, l[i]);
    }
    int first = AT_ONCE - 1;
#pragma unroll
    for (int i = AT_ONCE - 2; i >= 0; --i) first = l[i] == most ? i : first;
    best = most > v.m ? q + 32 * first : best;
    second = fmaxf(second, fminf(v.m, most));
    v.m = fmaxf(v.m, most);
    if (most > limit) {
      const float to = log_ref(most), d = R - to, e = exp2_fast(d);
      if (S2.x + S2.y != 0.f) {  // (sums of 0 may stand beside any reference)
        U2 = make_float2(e * (U2.x + d * S2.x), e * (U2.y + d * S2.y));
        S2 = make_float2(e * S2.x, e * S2.y);
      }
      R = to;
      limit = most + 5.5f;
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const Piece f = Row::floored(c[i]);
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float2 d = fma2(f.get2(e), make_float2(kLog2e, kLog2e), make_float2(-R, -R));
        const float2 t = make_float2(exp2_fast(d.x), exp2_fast(d.y));
        S2 = add2(S2, t);
        U2 = fma2(d, t, U2);
      }
    }
  };
  bool landed = true;  // every copy that was waited for
  for (int k = warp; k < chunks; k += warps) {
    const int q = p0 + k * kChunk + lane;
    Piece c[AT_ONCE];
    if (inner(k)) {
      if (!mbar_wait_bounded(&sh.full[warp][stage], (phases >> stage) & 1u, &sh.abort)) {
        if (!sh.abort) record_error(err, kErrTimeoutProducer);
        sh.abort = 1;
        landed = false;
      }
      phases ^= 1u << stage;
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) c[i].template load<false>(sh.stages[warp][stage] + (i * 32 + lane) * 16);
      // (without the fence a read that is still queued can meet the next copy's bytes)
      fence_proxy_async_smem();
      __syncwarp();
      // (no copy follows one that did not land)
      if (lane == 0 && landed && inner(k + kLogStages * warps)) copy(k + kLogStages * warps, stage);
      stage = stage + 1 == kLogStages ? 0 : stage + 1;
    } else {
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) c[i] = q + 32 * i < p1 ? x.load(q + 32 * i) : Row::none();
    }
    add_pieces(c, q);
  }
  if (!landed) wait_for_copies();
  const float own = v.m;
  v = log_of_pass(R, S2.x + S2.y, U2.x + U2.y, own);
  // ---- the block's sums, and the threads' largest logits
  v = log_join_lanes(v);
  if (lane == 0) {
    sh.red[warp] = v.m;
    sh.red[32 + warp] = v.S;
    sh.red[64 + warp] = v.U;
  }
  if (p.top > 0) {  // (the end of the piece stands for the logit's place: a lower bound)
    sh.keys[threadIdx.x] = best < p1 ? rank_key(own, (uint32_t)(x.first_index(best) + V - 1)) : 0;
    sh.second[threadIdx.x] = second;
  }
  __syncthreads();
  if (warp == 0) {
    v = log_join_lanes(lane < warps ? LogSums{sh.red[lane], sh.red[32 + lane], sh.red[64 + lane]}
                                    : LogSums{-INFINITY, 0.f, 0.f});
    if (lane == 0) {
      sh.sums = v;
      sh.n_found = 0;
    }
    if (p.top > 0) {  // the k largest of the threads' logits
      uint64_t keys[warps], last = ~0ull, mine = 0;
#pragma unroll
      for (int i = 0; i < warps; ++i) keys[i] = sh.keys[32 * i + lane];
      for (int i = 0; i < p.top; ++i) {
        last = next_largest<warps>(keys, last);
        if (last == 0) break;
        if (lane == i) mine = last;
      }
      sh.top[lane] = mine;
    }
  }
  __syncthreads();
  v = sh.sums;
  // ---- the block's alternatives
  bool full = false;
  if (p.top > 0) {
    const uint64_t bound = sh.top[p.top - 1];  // 0: fewer threads than alternatives, every logit may be one
    const uint32_t bound_bits = (uint32_t)(bound >> 32);
    auto find = [&](int q) {
      const Piece c = x.load(q);
      if (rank_bits(Row::largest(c)) < bound_bits) return;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int at = x.first_index(q) + e;
        const uint64_t key = rank_key(c.get(e), (uint32_t)at);
        if (at < 0 || at >= x.vocab || key < bound) continue;
        const int slot = atomicAdd(&sh.n_found, 1);
        if (slot < kCandidates) sh.found[slot] = key;
      }
    };
    auto piece_of = [&](uint64_t key) { return ((int)~(uint32_t)key - (V - 1) + x.off) / V - p0; };
    // of each thread that holds one of these, the chunk with its largest logit
    for (int u = threadIdx.x; u < AT_ONCE * p.top; u += THREADS) {
      const uint64_t key = sh.top[u / AT_ONCE];
      if (key == 0) break;
      const int piece = piece_of(key), q = p0 + piece / kChunk * kChunk + u % AT_ONCE * 32 + piece % 32;
      if (q < p1) find(q);
    }
    // and its others where the largest of these reaches the bound
    for (int i = warp; i < p.top; i += warps) {
      const uint64_t key = sh.top[i];
      if (key == 0) break;
      const int piece = piece_of(key), its_warp = piece / kChunk % warps;
      if (rank_bits(sh.second[its_warp * 32 + piece % 32]) < bound_bits) continue;
      for (int j = lane;; j += 32) {
        const int chunk = j / AT_ONCE * warps + its_warp, q = p0 + chunk * kChunk + j % AT_ONCE * 32 + piece % 32;
        if (chunk >= chunks) break;
        if (q < p1 && chunk != piece / kChunk) find(q);
      }
    }
    __syncthreads();
    full = sh.n_found > kCandidates;
    if (warp == 0 && !full) {
      const uint64_t t = pick_largest(sh.found, sh.n_found, p.top);
      sh.top[lane] = t;
      __syncwarp();
    }
  }
  bool odd = full;
  if (blocks_a_row == 1) {
    if (log_again(v.m)) v = log_large_row<T>(x, 0, x.pieces, v.m, sh.red);
  } else {
    if (threadIdx.x == 0) {
      sh.full_up = full;
      sh.again = 0.f;
    }
    __syncwarp();
    cluster_sync();  // every block's sums and alternatives are in its shared memory
    if (rank == 0) {
      // the largest of all alternatives
      const int any = lane < (int)blocks_a_row ? (int)ld_cluster_u32(mapa_shared(smem_u32(&sh.full_up), lane)) : 0;
      v = log_join_blocks(&sh.sums, blocks_a_row);
      odd = __any_sync(0xffffffffu, any != 0);
      // (whether the pass's sums hold shows in the whole row's: a part may well have nothing but masked logits)
      if (warp == 0 && log_again(v.m) && lane < (int)blocks_a_row)
        st_cluster_u32(mapa_shared(smem_u32(&sh.again), lane), __float_as_uint(v.m));
      if (p.top > 0 && !odd && warp == 0) {
        for (int i = lane; i < p.top * (int)blocks_a_row; i += 32) {
          const uint32_t key = mapa_shared(smem_u32(&sh.top[i % p.top]), i / p.top);
          sh.found[i] = (uint64_t)ld_cluster_u32(key) | (uint64_t)ld_cluster_u32(key + 4) << 32;
        }
        __syncwarp();
        const uint64_t t = pick_largest(sh.found, p.top * (int)blocks_a_row, p.top);
        __syncwarp();
        sh.found[lane] = t;
      }
    }
    __syncwarp();
    cluster_sync();  // no block ends, or writes its sums again, while they are read
    if (sh.again != 0.f) v = log_large_blocks<T>(x, p0, p1, sh.again, sh.red, &sh.sums, blocks_a_row);
  }
  if (rank != 0) return;
  if (odd || !(v.S == v.S)) {  // (S is NaN where the row has a NaN or +infinity)
    __syncthreads();
    logprob_plain_row<T>(p, a, row, sh.red, sh.plain);
  } else if (warp == 0) {
    const bool none = v.S == 0.f;
    const float log_s = log2f(v.S);
    if (lane == 0) {
      logprob_row_values(p, a, row, none, none ? -INFINITY : v.m + log_s * kLn2, (log_s - v.U / v.S) * kLn2,
                         target.place, log_prob(target.x, v, log_s));
    }
    if (lane < p.top) {
      const uint64_t key = (blocks_a_row > 1 ? sh.found : sh.top)[lane];
      const float xt = rank_value((uint32_t)(key >> 32));
      if (a.top_index) a.top_index[row * p.top + lane] = ~(uint32_t)key;
      if (a.top_logprob)
        a.top_logprob[row * p.top + lane] = none ? -INFINITY : log_prob(xt, v, log_s);
    }
  }
}

// ---------------------------------------------------------------- backward

// 16-byte units of the gradient's row a thread at a time. SAME: the logits lie alike on the grid; else they are
// shifted into place
template <typename T, bool SAME>
__global__ void __launch_bounds__(256) logprob_backward_kernel(const LogprobParams p, const LogprobGradPtrs a,
                                                               int blocks_a_row) {
  using Row = LogitRow<T>;
  using Piece = typename Row::Piece;
  constexpr int V = Row::V, AT_ONCE = 4;
  pdl_launch_dependents();
  pdl_wait();
  const uintptr_t begin = reinterpret_cast<uintptr_t>(a.x);
  const uintptr_t end = begin + (uintptr_t)(((p.rows - 1) * p.s_x + p.vocab) * (int64_t)sizeof(T));
  const int64_t row = blockIdx.x / (uint32_t)blocks_a_row;
  const int part = (int)(blockIdx.x % (uint32_t)blocks_a_row);
  T const *x = static_cast<T const *>(a.x) + row * p.s_x;
  T *dx = static_cast<T *>(a.dx) + row * p.s_dx;
  const Row out(dx, p.vocab), in(x, p.vocab);
  const int q0 = (int)((int64_t)out.pieces * part / blocks_a_row);
  const int q1 = (int)((int64_t)out.pieces * (part + 1) / blocks_a_row);
  const float lse = a.lse[row];
  const int64_t t = a.targets ? a.targets[row] : -1;
  float dlp = t >= 0 ? a.dlogprob[row] : 0.f;
  if (t >= p.vocab) dlp = logit_nan();
  const float dent = a.dentropy ? a.dentropy[row] : 0.f;
  // dx = -p (dlp + dent (x - lse + H)) = p (k0 + k1 d), d = (x - lse) log2 e
  const float k0 = -dlp - dent * (a.dentropy ? a.entropy[row] : 0.f), k1 = -dent * kLn2;
  const bool none = lse == -INFINITY;
  // the gradients of a piece's logits
  auto grads = [&](int q, Piece const &c) {
    const int i0 = out.first_index(q);
    float f[V];
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      float2 d = mul2(add2(c.get2(e), make_float2(-lse, -lse)), make_float2(kLog2e, kLog2e));
      // (2^-200 is 0 in FP32: a ruled-out logit gets 0, not 0 times infinity)
      d = make_float2(max_nan(d.x, -200.f), max_nan(d.y, -200.f));
      const float2 pr = make_float2(exp2_fast(d.x), exp2_fast(d.y));
      const float2 r = mul2(pr, fma2(d, make_float2(k1, k1), make_float2(k0, k0)));
      f[e] = r.x;
      f[e + 1] = r.y;
    }
    if (none) {
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = 0.f;
    } else if (t >= i0 && t < i0 + V) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (t == i0 + e) f[e] += dlp;
    }
    Piece g;
    g.set(f);
    return g;
  };
  const int threads = blockDim.x;
  int q = q0 + (int)threadIdx.x;
  auto ragged = [&]() {  // pieces that may reach outside the row, or the tensor
    const int i0 = out.first_index(q);
    const bool inside = i0 >= 0 && i0 <= p.vocab - V;
    Piece c;
    if (SAME) {
      c = in.load(q);
    } else if (inside) {
      c.load_any(x, i0, p.vocab, begin, end);
    } else {
      float f[V];
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = i0 + e >= 0 && i0 + e < p.vocab ? to_f32(x[i0 + e]) : 0.f;
      c.set(f);
    }
    const Piece g = grads(q, c);
    if (inside) g.store(dx + i0);
    else g.store_some(dx + i0, i0 < 0 ? -i0 : 0, p.vocab - i0 < V ? (int)(p.vocab - i0) : V);
    q += threads;
  };
  if (q < q1) ragged();
  if (SAME) {
    for (; q + (AT_ONCE - 1) * threads < q1 - 1; q += AT_ONCE * threads) {
      Piece c[AT_ONCE];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) c[i].template load<false>(in.base + (int64_t)(q + i * threads) * 16);
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) grads(q + i * threads, c[i]).store(dx + out.first_index(q + i * threads));
    }
  }
  while (q < q1) ragged();
}

// ---------------------------------------------------------------- launchers

cudaError_t launch_logprob(LogprobParams const &p, LogprobPtrs const &a, uint32_t *err, int num_sms,
                           cudaStream_t st) {
  const int64_t pieces = (p.vocab * (p.dt == EIR_FP32 ? 4 : 2) + 15) / 16 + 1;
  // Long rows that leave SMs idle are split over clusters (2048 pieces a block at
  // least; 64 x 131072 BF16: 16.0 us whole, 14.1 over 8 blocks; 4096 pieces are
  // faster whole, 6.6 against 7.5 us).
  uint32_t blocks = 1;
  while (blocks < 8 && p.rows * blocks * 2 <= 6 * num_sms && pieces >= 8192 && pieces >= 4096 * (int64_t)blocks)
    blocks *= 2;
  // Few threads a row make its barriers cheap where many rows wait; as many as fit are on an SM at a time, and
  // the next take the place of the finished ones (persistent blocks that
  // walked rows ran in step with one another: 67 us against 59 without alternatives, 4096 x 32768 BF16).
  // Few rows take more threads instead.
  int threads = pieces <= 512 ? 32 : pieces <= 2048 ? 64 : pieces <= 8192 ? 128 : 256;
  if (p.rows <= 2 * num_sms) threads = pieces <= 256 ? 64 : pieces <= 1024 ? 128 : 256;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.rows * blocks));
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (blocks > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = blocks;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  auto pick = [&](auto zero) {
    using T = decltype(zero);
    switch (threads) {
      case 32: return logprob_kernel<T, 32>;
      case 64: return logprob_kernel<T, 64>;
      case 128: return logprob_kernel<T, 128>;
      default: return logprob_kernel<T, 256>;
    }
  };
  auto kern = p.dt == EIR_FP32 ? pick(float{}) : pick(__nv_bfloat16{});
  return cudaLaunchKernelEx(&cfg, kern, p, a, blocks, err);
}

template <typename T>
static cudaError_t launch_logprob_backward_t(LogprobParams const &p, LogprobGradPtrs const &a, int num_sms,
                                             cudaStream_t st) {
  // blocks of 4096 pieces, smaller where the GPU would not be full. (Blocks that end make room
  // for others out of step: persistent ones took 80 us for 2048 x 50021 BF16, these take 72.)
  const int64_t pieces = (p.vocab * (int64_t)sizeof(T) + 15) / 16 + 1;
  int64_t blocks = (pieces + 4096 - 1) / 4096;
  while (p.rows * blocks < (int64_t)num_sms * 8 && pieces > 1024 * blocks) blocks *= 2;
  blocks = std::max<int64_t>(1, std::min<int64_t>(blocks, INT32_MAX / p.rows));
  const bool same = (reinterpret_cast<uintptr_t>(a.x) - reinterpret_cast<uintptr_t>(a.dx)) % 16 == 0 &&
                    (p.rows == 1 || (p.s_x - p.s_dx) * (int64_t)sizeof(T) % 16 == 0);
  auto kern = same ? logprob_backward_kernel<T, true> : logprob_backward_kernel<T, false>;
  return launch_kernel(kern, dim3((unsigned)(p.rows * blocks)), dim3(pieces <= 256 ? 64 : pieces <= 1024 ? 128 : 256), 0,
                       st, p, a, (int)blocks);
}

cudaError_t launch_logprob_backward(LogprobParams const &p, LogprobGradPtrs const &a, int num_sms,
                                    cudaStream_t st) {
  return p.dt == EIR_FP32 ? launch_logprob_backward_t<float>(p, a, num_sms, st)
                          : launch_logprob_backward_t<__nv_bfloat16>(p, a, num_sms, st);
}

}  // namespace eir
