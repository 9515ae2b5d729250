// Root-mean-square norm with the residual's addition, its backward pass, and
// the quantisation of rows to 8-bit integers.
//
// Forward, a row of C columns: h = x + r, rstd = (sum h^2 / C + eps)^(-1/2),
// y = h rstd w. With 8-bit output v = h w, m = max|v|: y / s = v 127 / m for
// s = m rstd / 127, so the integers need no rstd and the row's two statistics
// (sum of squares, maximum) come from one pass. Backward: g = w dy,
// dx = rstd (g - h rstd^2 mean(g h)) + dsum, dw = sum over rows of dy h rstd
// (computed with dy rstd in place of dy, which saves a product an element).
// Sums are held in FP32.
//
// All three are bound by HBM. A row stays on the SM between the statistics and
// the output, so each input is read once and each output written once. Up to
// kPer elements a thread and 1024 threads it stays in registers: a warp a row for
// narrow rows, a block above, in 16-byte pieces; blocks are persistent, and where
// the rows lie on the pieces' grid they load their next row before they reduce the present
// one. Wider rows stay in shared memory, and rows too wide for that are read twice.
// Measured on one B200 (a copy moves 6.55 TB/s): 8192 x 4096 BF16 with residual to 8 bits 41 us, 5.7 TB/s;
// its backward pass with the weight gradient 46 us, 5.8 TB/s; quantize 4099 x 10920 BF16 26.6 us, 5.0 TB/s.
#include <algorithm>
#include <type_traits>
#include "eir_launch.h"
#include "eir_common.cuh"
#include "op_params.h"
#include "row_vec.cuh"

namespace eir {

// elements of a thread whose row stays in registers: FP32 rows take twice the
// registers an element
template <typename T, bool QUANT>
constexpr int kPer = (sizeof(T) == 4 ? 8 : 16) * (QUANT ? 2 : 1);  // norm; quantize
constexpr int kPerBack = 8;  // backward, of a warp's row

// Sum of v and maximum of m over a row's threads: a warp (`warps` = 1), or the
// block, with one barrier (`red`: 64 words, other ones at the next call).
template <bool SUM, bool MAX>
__device__ __forceinline__ void row_sum_max(float &v, uint32_t &m, uint32_t *red, int warps) {
  if (SUM) v = warp_sum(v);
  if (MAX) m = __reduce_max_sync(0xffffffffu, m);
  if (warps == 1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) {
    if (SUM) red[warp] = __float_as_uint(v);
    if (MAX) red[32 + warp] = m;
  }
  __syncthreads();
  if (SUM) v = warp_sum(lane < warps ? __uint_as_float(red[lane]) : 0.f);
  if (MAX) m = __reduce_max_sync(0xffffffffu, lane < warps ? red[32 + lane] : 0u);
}

// ---------------------------------------------------------------- a ring of rows in shared memory

// Rows of up to three tensors are copied (cp.async.bulk) into a ring of stages, so
// that the bytes in flight do not depend on the registers of the threads that work on a row. A
// copy takes the 16-byte units that cover a row; of the units that reach outside the tensor (its first and
// last row may have one), only the row's own bytes are read, by the thread. In its
// slot a row starts as far off a 16-byte boundary as it does in memory.
constexpr int kMostStages = 8;
struct RingShape {
  int threads;  // that work on rows: whole warps
  int stages;
  int64_t stage_bytes;
  int64_t more;  // bytes behind the stages
};
__host__ __device__ constexpr int64_t ring_slot(int64_t bytes) { return ((bytes + 15) / 16 + 4) * 16; }

__device__ __forceinline__ void bulk_load(void *dst, uintptr_t src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

struct RingTensor {  // in shared memory: only the copying thread needs all of it
  uintptr_t begin, end;  // its bytes; none: absent
  int64_t stride;        // of a row, in bytes
  int64_t bytes;         // of a row
  int64_t slot;          // its place in a stage
  __device__ __forceinline__ void set(void const *p, int64_t rows, int64_t cols, int64_t row_stride, int esize,
                                      int64_t at) {
    begin = reinterpret_cast<uintptr_t>(p);
    stride = row_stride * esize;
    bytes = cols * esize;
    end = p == nullptr ? begin : begin + (uintptr_t)((rows - 1) * stride + bytes);
    slot = at;
  }
  __device__ __forceinline__ int64_t next_slot() const { return slot + (end > begin ? ring_slot(bytes) : 0); }
  // how far into its slot a row lies
  __device__ __forceinline__ uint32_t off(int64_t row) const {
    return ((uint32_t)begin + (uint32_t)row * (uint32_t)stride) & 15u;
  }
  // bytes that arrive by bulk copy; the others are stored here
  __device__ __forceinline__ uint32_t span(int64_t row, uint8_t *stage, uintptr_t &a0, uintptr_t &a1) const {
    const uintptr_t r0 = begin + (uintptr_t)(row * stride), r1 = r0 + (uintptr_t)bytes;
    a0 = r0 & ~(uintptr_t)15;
    a1 = (r1 + 15) & ~(uintptr_t)15;
    uint8_t *to = stage + slot;
    const uintptr_t base = a0;
    if (a0 < begin) a0 += 16;
    if (a1 > end) a1 -= 16;
    for (uintptr_t q = r0; q < a0 && q < r1; ++q) to[q - base] = *reinterpret_cast<uint8_t const *>(q);
    for (uintptr_t q = a1 > r0 ? a1 : r0; q < r1; ++q) to[q - base] = *reinterpret_cast<uint8_t const *>(q);
    return a1 > a0 ? (uint32_t)(a1 - a0) : 0u;
  }
  __device__ __forceinline__ void copy(int64_t row, uint8_t *stage, uintptr_t a0, uint32_t n, uint64_t *bar) const {
    const uintptr_t base = (begin + (uintptr_t)(row * stride)) & ~(uintptr_t)15;
    if (n) bulk_load(stage + slot + (a0 - base), a0, n, bar);
  }
};

template <int TENSORS>
__device__ __forceinline__ void ring_copy(RingTensor (&t)[TENSORS], int64_t row, uint8_t *stage, uint64_t *bar) {
  uintptr_t a0[TENSORS], a1;
  uint32_t n[TENSORS], total = 0;
#pragma unroll
  for (int i = 0; i < TENSORS; ++i) {
    n[i] = 0;
    if (t[i].end > t[i].begin) n[i] = t[i].span(row, stage, a0[i], a1);
    total += n[i];
  }
  mbar_arrive_expect_tx(bar, total);
#pragma unroll
  for (int i = 0; i < TENSORS; ++i)
    if (t[i].end > t[i].begin) t[i].copy(row, stage, a0[i], n[i], bar);
}

// The ring's shared words, and the thread that fills it: a warp of its own beside the
// `warps` that work on rows (in one of those the copies delay every row: 8192 x 4096 BF16
// backward 69 us)
template <int TENSORS>
struct RowRing {
  uint64_t full[kMostStages], empty[kMostStages];
  RingTensor t[TENSORS];
  int abort;

  __device__ __forceinline__ void init(RingShape const &ring) {
    for (int s = 0; s < ring.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], ring.threads >> 5);
    }
    abort = 0;
    fence_barrier_init();
  }
  __device__ __forceinline__ void fill(RingShape const &ring, uint8_t *stages, int64_t rows, uint32_t *err) {
    volatile int *stop = &abort;
    int stage = 0;
    uint32_t phase = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
      // (a stage is freed by threads that gave up waiting for it, too: no copy follows one that did not land)
      if (!mbar_wait_bounded(&empty[stage], phase ^ 1u, stop) || *stop) {
        if (!*stop) record_error(err, kErrTimeoutProducer);
        *stop = 1;
        wait_for_copies();
        return;
      }
      ring_copy(t, row, stages + stage * ring.stage_bytes, &full[stage]);
      if (++stage == ring.stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
  }
  // false: the wait has given up
  __device__ __forceinline__ bool wait(int stage, uint32_t phase, uint32_t *err) {
    volatile int *stop = &abort;
    if (mbar_wait_bounded(&full[stage], phase, stop)) return true;
    if (!*stop) record_error(err, kErrTimeoutEpilogue);
    *stop = 1;
    wait_for_copies();
    return false;
  }
};
// a barrier of the `threads` that work on rows
__device__ __forceinline__ void ring_sync(int threads) { asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); }

// ---------------------------------------------------------------- norm and quantize

// One piece of the forward pass. OUT: int8_t, float or __nv_bfloat16; QUANT:
// quantize (no sum of squares, residual or weight; NormParams' and NormPtrs' fields of the
// same meaning); GRID: every row lies on the pieces' grid and has whole pieces
template <typename T, typename OUT, bool QUANT, bool GRID>
struct NormRow {
  static constexpr int V = 16 / (int)sizeof(T);
  static constexpr bool kInt8 = sizeof(OUT) == 1;
  using Piece = RowPiece<T, V>;
  NormParams const &p;
  NormPtrs const &a;
  RowBounds bx, br;
  bool w_grid;

  __device__ __forceinline__ NormRow(NormParams const &p_, NormPtrs const &a_) : p(p_), a(a_) {
    if (!GRID) {
      bx = row_bounds(a.x, p.rows, p.cols, p.s_x, sizeof(T));
      br = row_bounds(a.res, p.rows, p.cols, p.s_res, sizeof(T));
    }
    w_grid = GRID || row_vec_ok(a.w, 0, 1, p.dt_w == EIR_FP32 ? 4 : 2, V);
  }
  __device__ __forceinline__ bool residual() const { return !QUANT && a.res != nullptr; }
  __device__ __forceinline__ void load(int64_t row, int64_t c, Piece &x, Piece &r) const {
    T const *px = static_cast<T const *>(a.x) + row * p.s_x, *pr = static_cast<T const *>(a.res) + row * p.s_res;
    if (GRID) {
      if (c < p.cols) x.template load<true>(px + c);
      else x.zero();
      if (residual() && c < p.cols) r.template load<true>(pr + c);
    } else {
      x.load_any(px, c, p.cols, bx.begin, bx.end);
      if (residual()) r.load_any(pr, c, p.cols, br.begin, br.end);
    }
  }
  template <typename D>
  __device__ __forceinline__ void put(RowPiece<D, V> const &v, D *row, int64_t c) const {
    if (!GRID) v.store_any(row, c, p.cols);
    else if (c < p.cols) v.store(row + c);
  }
  // h (times the weight for 8-bit output) of a piece and its part of the
  // statistics; stores the sum if `keep`. Every lane of a warp calls it
  __device__ __forceinline__ void take(int64_t row, int64_t c, Piece const &x, Piece const &r, float (&h)[V],
                                       float &ss, uint32_t &mx, bool keep = true) const {
    const bool add = residual() && c < p.cols;
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      float2 v = x.get2(e);
      if (add) v = add2(v, r.get2(e));
      if (!QUANT) sum = fma2(v, v, sum);
      h[e] = v.x;
      h[e + 1] = v.y;
    }
    if (!QUANT) {
      ss += sum.x + sum.y;
      if (a.sum && keep) {
        Piece s;
        s.set(h);
        put<T>(s, static_cast<T *>(a.sum) + row * p.s_sum, c);
      }
      if (kInt8 && a.w && c < p.cols) {
        float w[V];
        load_shared_any<V>(a.w, p.dt_w, c, p.cols, w_grid, w);
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const float2 v = mul2(make_float2(h[e], h[e + 1]), make_float2(w[e], w[e + 1]));
          h[e] = v.x;
          h[e + 1] = v.y;
        }
      }
    }
    if (kInt8) {
      float most = __uint_as_float(mx);
#pragma unroll
      for (int e = 0; e < V; ++e) most = max_nan(most, fabsf(h[e]));
      mx = __float_as_uint(most);
    }
  }
  __device__ __forceinline__ void give(int64_t row, int64_t c, float const (&h)[V], float rstd,
                                       QuantScale const &q) const {
    OUT *out = static_cast<OUT *>(a.out) + row * p.s_out;
    RowPiece<OUT, V> o;
    if constexpr (kInt8) {
      o.zero();
      if (q.finite) {
        // 1.5 * 2^23 + t rounds t to an integer, ties to even, and holds it in its low byte: a
        // quarter of the instructions of conversions and masks
        constexpr float kMagic = 12582912.f;
#pragma unroll
        for (int e = 0; e < V; e += 4) {
          // (__fmul_rn: a packed product and sum would be contracted to one rounding)
          const float2 t = add2(make_float2(__fmul_rn(h[e], q.inv), __fmul_rn(h[e + 1], q.inv)),
                                make_float2(kMagic, kMagic));
          const float2 u = add2(make_float2(__fmul_rn(h[e + 2], q.inv), __fmul_rn(h[e + 3], q.inv)),
                                make_float2(kMagic, kMagic));
          o.w[e / 4] = __byte_perm(__byte_perm(__float_as_uint(t.x), __float_as_uint(t.y), 0x0040),
                                   __byte_perm(__float_as_uint(u.x), __float_as_uint(u.y), 0x0040), 0x5410);
        }
      }
    } else {
      float w[V], y[V];
#pragma unroll
      for (int e = 0; e < V; ++e) w[e] = 1.f;
      if (a.w && c < p.cols) load_shared_any<V>(a.w, p.dt_w, c, p.cols, w_grid, w);
#pragma unroll
      for (int e = 0; e < V; ++e) y[e] = h[e] * rstd * w[e];
      o.set(y);
    }
    put<OUT>(o, out, c);
  }
  __device__ __forceinline__ float rstd_of(float ss) const {
    return QUANT ? 1.f : __frsqrt_rn(ss / (float)p.cols + p.eps);
  }
  __device__ __forceinline__ void row_values(int64_t row, float rstd, QuantScale const &q) const {
    if (kInt8) a.scale[row] = q.scale;
    if (!QUANT && a.rstd) a.rstd[row] = rstd;
  }
};

template <typename T, typename OUT, bool QUANT, bool GRID>
__global__ void __launch_bounds__(1024) norm_kernel(const NormParams p, const NormPtrs a, int row_warps) {
  using Row = NormRow<T, OUT, QUANT, GRID>;
  constexpr int V = Row::V, N = kPer<T, QUANT> / V;
  __shared__ uint32_t red[2][64];
  pdl_launch_dependents();
  pdl_wait();
  const Row op(p, a);
  const int threads = row_warps * 32, tid = row_warps == 1 ? threadIdx.x & 31 : threadIdx.x;
  const int64_t rows_at_once = row_warps == 1 ? (int64_t)gridDim.x * (blockDim.x >> 5) : gridDim.x;
  int64_t row = row_warps == 1 ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  auto column = [&](int j) { return (int64_t)(j * threads + tid) * V; };
  typename Row::Piece x[N], r[N];
  auto fetch = [&](int64_t at) {
#pragma unroll
    for (int j = 0; j < N; ++j) op.load(at, column(j), x[j], r[j]);
  };
  if (GRID && row < p.rows) fetch(row);
  for (int turn = 0; row < p.rows; row += rows_at_once, turn ^= 1) {
    if (!GRID) fetch(row);
    // norm holds the row as h; quantize as it was read, in half the registers or the same
    float h[QUANT ? 1 : N][V];
    typename Row::Piece held[QUANT ? N : 1];
    float ss = 0.f;
    uint32_t mx = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      op.take(row, column(j), x[j], r[j], h[QUANT ? 0 : j], ss, mx);
      if (QUANT) held[j] = x[j];
    }
    if (GRID && row + rows_at_once < p.rows) fetch(row + rows_at_once);
    row_sum_max<!QUANT, Row::kInt8>(ss, mx, red[turn], row_warps);
    const float rstd = op.rstd_of(ss);
    const QuantScale q = quant_scale(mx, rstd);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (QUANT) {
#pragma unroll
        for (int e = 0; e < V; ++e) h[0][e] = held[j].get(e);
      }
      op.give(row, column(j), h[QUANT ? 0 : j], rstd, q);
    }
    if (tid == 0) op.row_values(row, rstd, q);
  }
}

// rows off the pieces' grid, a block a row: they come through the ring, since what is
// shifted into place cannot wait in registers
template <typename T, typename OUT, bool QUANT>
__global__ void __launch_bounds__(1024)
    norm_ring_kernel(const NormParams p, const NormPtrs a, const RingShape ring, uint32_t *err) {
  using Row = NormRow<T, OUT, QUANT, false>;
  constexpr int V = Row::V, N = kPer<T, false> / V;
  extern __shared__ __align__(128) uint8_t stages[];
  __shared__ uint32_t red[2][96];
  __shared__ RowRing<2> rr;
  const int warps = ring.threads >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    rr.t[0].set(a.x, p.rows, p.cols, p.s_x, sizeof(T), 0);
    rr.t[1].set(QUANT ? nullptr : a.res, p.rows, p.cols, p.s_res, sizeof(T), rr.t[0].next_slot());
    rr.init(ring);
  }
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  if (warp == warps) {
    if (lane == 0) rr.fill(ring, stages, p.rows, err);
    return;
  }
  const Row op(p, a);
  const uint32_t slot = (uint32_t)ring_slot(p.cols * sizeof(T));
  auto column = [&](int j) { return (j * ring.threads + (int)threadIdx.x) * V; };
  int stage = 0, turn = 0;
  uint32_t phase = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    const bool late = !rr.wait(stage, phase, err);
    uint8_t const *at = stages + stage * ring.stage_bytes;
    const uint32_t off_x = rr.t[0].off(row), off_r = rr.t[1].off(row);
    float h[N][V];
    float ss = 0.f;
    uint32_t mx = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      typename Row::Piece x, r;
      x.load_slot(at, off_x, column(j), p.cols);
      if (op.residual()) r.load_slot(at + slot, off_r, column(j), p.cols);
      op.take(row, column(j), x, r, h[j], ss, mx);
    }
    fence_proxy_async_smem();  // the row is in registers: its stage may be copied over
    __syncwarp();
    if (lane == 0) mbar_arrive(&rr.empty[stage]);
    if (!QUANT) ss = warp_sum(ss);
    mx = __reduce_max_sync(0xffffffffu, mx);
    const bool warp_late = __any_sync(0xffffffffu, late);
    if (lane == 0) {
      red[turn][warp] = __float_as_uint(ss);
      red[turn][32 + warp] = mx;
      red[turn][64 + warp] = warp_late;
    }
    ring_sync(ring.threads);
    // all threads leave together where a wait has given up
    if (__any_sync(0xffffffffu, lane < warps && red[turn][64 + lane] != 0)) break;
    if (!QUANT) ss = warp_sum(lane < warps ? __uint_as_float(red[turn][lane]) : 0.f);
    mx = __reduce_max_sync(0xffffffffu, lane < warps ? red[turn][32 + lane] : 0u);
    const float rstd = op.rstd_of(ss);
    const QuantScale q = quant_scale(mx, rstd);
#pragma unroll
    for (int j = 0; j < N; ++j) op.give(row, column(j), h[j], rstd, q);
    if (threadIdx.x == 0) op.row_values(row, rstd, q);
    if (++stage == ring.stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
}

// wide rows: h in shared memory (CACHED), or read again
template <typename T, typename OUT, bool QUANT, bool CACHED>
__global__ void __launch_bounds__(1024) norm_wide_kernel(const NormParams p, const NormPtrs a) {
  using Row = NormRow<T, OUT, QUANT, false>;
  constexpr int V = Row::V;
  __shared__ uint32_t red[2][64];
  extern __shared__ float4 held[];  // [piece][V / 4][thread]
  pdl_launch_dependents();
  pdl_wait();
  const Row op(p, a);
  const int threads = blockDim.x, pieces = (int)((p.cols + (int64_t)threads * V - 1) / ((int64_t)threads * V));
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    float ss = 0.f;
    uint32_t mx = 0;
    // (the sum may take x's place: a row that is read twice stores it the second time)
    auto piece = [&](int j, float (&h)[V], bool keep) {
      typename Row::Piece x, r;
      const int64_t c = ((int64_t)j * threads + threadIdx.x) * V;
      op.load(row, c, x, r);
      op.take(row, c, x, r, h, ss, mx, keep);
    };
#pragma unroll 2
    for (int j = 0; j < pieces; ++j) {
      float h[V];
      piece(j, h, CACHED);
      if (CACHED) {
#pragma unroll
        for (int i = 0; i < V / 4; ++i)
          held[(j * (V / 4) + i) * threads + threadIdx.x] = make_float4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
      }
    }
    row_sum_max<!QUANT, Row::kInt8>(ss, mx, red[turn], threads >> 5);
    const float rstd = op.rstd_of(ss);
    const QuantScale q = quant_scale(mx, rstd);
#pragma unroll 2
    for (int j = 0; j < pieces; ++j) {
      float h[V];
      if (CACHED) {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
          const float4 f = held[(j * (V / 4) + i) * threads + threadIdx.x];
          h[4 * i] = f.x;
          h[4 * i + 1] = f.y;
          h[4 * i + 2] = f.z;
          h[4 * i + 3] = f.w;
        }
      } else {
        piece(j, h, true);
      }
      op.give(row, ((int64_t)j * threads + threadIdx.x) * V, h, rstd, q);
    }
    if (threadIdx.x == 0) op.row_values(row, rstd, q);
  }
}

// ---------------------------------------------------------------- backward

// One piece of the backward pass; GRID as above
template <typename T, typename G, bool GRID>
struct NormBackRow {
  static constexpr int V = 16 / (int)(sizeof(T) > sizeof(G) ? sizeof(T) : sizeof(G));
  using PieceH = RowPiece<T, V>;
  using PieceG = RowPiece<G, V>;
  NormParams const &p;
  NormGradPtrs const &a;
  RowBounds bh, bd, bs;
  bool w_grid;

  __device__ __forceinline__ NormBackRow(NormParams const &p_, NormGradPtrs const &a_) : p(p_), a(a_) {
    if (!GRID) {
      bh = row_bounds(a.h, p.rows, p.cols, p.s_h, sizeof(T));
      bd = row_bounds(a.dy, p.rows, p.cols, p.s_dy, sizeof(G));
      bs = row_bounds(a.dsum, p.rows, p.cols, p.s_dsum, sizeof(G));
    }
    w_grid = GRID || row_vec_ok(a.w, 0, 1, p.dt_w == EIR_FP32 ? 4 : 2, V);
  }
  template <typename D>
  __device__ __forceinline__ void get(RowPiece<D, V> &v, void const *base, int64_t stride, RowBounds const &b,
                                      int64_t row, int64_t c) const {
    D const *at = static_cast<D const *>(base) + row * stride;
    if (!GRID) v.load_any(at, c, p.cols, b.begin, b.end);
    else if (c < p.cols) v.template load<true>(at + c);
    else v.zero();
  }
  __device__ __forceinline__ void load(int64_t row, int64_t c, PieceH &h, PieceG &dy) const {
    get<T>(h, a.h, p.s_h, bh, row, c);
    get<G>(dy, a.dy, p.s_dy, bd, row, c);
  }
  __device__ __forceinline__ void load_sum(int64_t row, int64_t c, PieceG &s) const {
    if (a.dsum) get<G>(s, a.dsum, p.s_dsum, bs, row, c);
  }
  // With e = dy rstd and g = w e: held = g + dsum, and the piece's part of sum g h
  // (GH) and of the weight gradients e h (DW)
  __device__ __forceinline__ void weight(int64_t c, float (&w)[V]) const {
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = 1.f;
    if (a.w && c < p.cols) load_shared_any<V>(a.w, p.dt_w, c, p.cols, w_grid, w);
  }
  template <bool GH, bool DW>
  __device__ __forceinline__ void take(float const (&w)[V], PieceH const &h, PieceG const &dy, PieceG const &s,
                                       float rstd, float (&held)[V], float &gh, float (&dw)[V]) const {
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float2 hv = h.get2(e), d = mul2(dy.get2(e), make_float2(rstd, rstd));
      float2 g = mul2(make_float2(w[e], w[e + 1]), d);
      if (GH) sum = fma2(g, hv, sum);
      if (DW) {
        const float2 t = fma2(d, hv, make_float2(dw[e], dw[e + 1]));
        dw[e] = t.x;
        dw[e + 1] = t.y;
      }
      if (a.dsum) g = add2(g, s.get2(e));
      held[e] = g.x;
      held[e + 1] = g.y;
    }
    if (GH) gh += sum.x + sum.y;
  }
  // the factor of h in dx = g - h rstd^2 mean(g h) + dsum
  __device__ __forceinline__ float factor(float rstd, float gh) const { return rstd * rstd * (gh / (float)p.cols); }
  // the elements inside the row of a piece that reaches outside it
  __device__ __forceinline__ void give_some(int64_t row, int64_t c, float const (&held)[V], PieceH const &h, float k) const {
    G *out = static_cast<G *>(a.dx) + row * p.s_dx;
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (c + e >= 0 && c + e < p.cols) out[c + e] = from_f32<G>(fmaf(h.get(e), -k, held[e]));
  }
  // every lane of a warp calls it
  __device__ __forceinline__ void give(int64_t row, int64_t c, float const (&held)[V], PieceH const &h, float k) const {
    float d[V];
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float2 t = fma2(h.get2(e), make_float2(-k, -k), make_float2(held[e], held[e + 1]));
      d[e] = t.x;
      d[e + 1] = t.y;
    }
    PieceG o;
    o.set(d);
    G *out = static_cast<G *>(a.dx) + row * p.s_dx;
    if (!GRID) o.store_any(out, c, p.cols);
    else if (c < p.cols) o.store(out + c);
  }
};

// V columns of a partial row (column a multiple of V; the pitch has room for whole 16-byte pieces)
template <int V>
__device__ __forceinline__ void put_part(float *part, int64_t column, int64_t cols, float const (&v)[V]) {
#pragma unroll
  for (int e = 0; e < V; e += 4)
    if (column + e < cols)
      *reinterpret_cast<float4 *>(part + column + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
}

// Narrow rows: a warp a row, the next one loaded early. The weight gradient of the
// warp's columns stays in registers over all rows that it sees; the block's warps add theirs through
// shared memory into one partial row, summed by norm_dweight_kernel: no atomics, so the order is
// fixed. (So too below, a block a partial row.)
constexpr int kBackWarps = 16;
template <typename T, typename G, bool GRID>
__global__ void __launch_bounds__(kBackWarps * 32) norm_backward_kernel(const NormParams p, const NormGradPtrs a) {
  using Row = NormBackRow<T, G, GRID>;
  constexpr int V = Row::V, N = kPerBack / V;
  pdl_launch_dependents();
  pdl_wait();
  const Row op(p, a);
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int64_t at_once = (int64_t)gridDim.x * kBackWarps, first = (int64_t)blockIdx.x * kBackWarps + warp;
  extern __shared__ float warp_dw[];  // [warp][column]
  auto column = [&](int j) { return (int64_t)(j * 32 + lane) * V; };
  typename Row::PieceH h[N];
  typename Row::PieceG dy[N], ds[N];
  float rstd = 0.f;
  auto fetch = [&](int64_t r) {
    rstd = a.rstd[r];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      op.load(r, column(j), h[j], dy[j]);
      op.load_sum(r, column(j), ds[j]);
    }
  };
  float dw[N][V];
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) dw[j][e] = 0.f;
  if (first < p.rows) fetch(first);
  for (int64_t row = first; row < p.rows; row += at_once) {
    const float unit = rstd;
    float held[N][V];
    typename Row::PieceH hr[N];
    float gh = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float w[V];
      op.weight(column(j), w);
      op.template take<true, true>(w, h[j], dy[j], ds[j], unit, held[j], gh, dw[j]);
      hr[j] = h[j];
    }
    if (row + at_once < p.rows) fetch(row + at_once);
    const float k = op.factor(unit, warp_sum(gh));
#pragma unroll
    for (int j = 0; j < N; ++j) op.give(row, column(j), held[j], hr[j], k);
  }
  if (a.part == nullptr) return;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (column(j) + e < p.cols) warp_dw[warp * p.cols + column(j) + e] = dw[j][e];
  __syncthreads();
  float *part = a.part + (int64_t)blockIdx.x * norm_part_pitch(p.cols);
  for (int c = threadIdx.x; c < p.cols; c += kBackWarps * 32) {
    float sum = warp_dw[c];
#pragma unroll
    for (int w = 1; w < kBackWarps; ++w) sum += warp_dw[w * p.cols + c];
    part[c] = sum;
  }
}

// Blocks a row, over the ring. N: pieces of a thread.
constexpr int kBackThreads = 512;  // of a block, at most
// blocks an SM of that many threads, by a thread's elements
__host__ __device__ constexpr int back_blocks(int per) { return per > 8 ? 1 : 2; }

// How a block's rows lie on the grid of 16-byte pieces: anyhow (pieces are shifted into place), on it, or
// all tensors alike and by the same in every row of the block (the launch's grid is a multiple of the rows after which
// it repeats): then the block's pieces lie on the grid of memory, and only a row's first and last one may be partial.
// There the weight waits in shared memory, laid out like the pieces. (1237 x 2311 FP32: 19.1 us shifted, 14.0
// alike, 12.4 for 2312 columns on the grid; 8192 x 4095 BF16: 103, 49 and 45.)
enum RowsLie { kRowsAnyhow, kRowsOnGrid, kRowsAlike };

template <typename T, typename G, int N, RowsLie LIE>
__global__ void __launch_bounds__(kBackThreads + 32, back_blocks(N * NormBackRow<T, G, false>::V))
    norm_backward_ring_kernel(const NormParams p, const NormGradPtrs a, const RingShape ring, uint32_t *err) {
  using Row = NormBackRow<T, G, LIE != kRowsAnyhow>;
  constexpr int V = Row::V;
  constexpr bool GRID = LIE == kRowsOnGrid, ALIKE = LIE == kRowsAlike;
  extern __shared__ __align__(128) uint8_t stages[];
  __shared__ uint32_t red[2][64];
  __shared__ RowRing<3> rr;
  const int warps = ring.threads >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    rr.t[0].set(a.h, p.rows, p.cols, p.s_h, sizeof(T), 0);
    rr.t[1].set(a.dy, p.rows, p.cols, p.s_dy, sizeof(G), rr.t[0].next_slot());
    rr.t[2].set(a.dsum, p.rows, p.cols, p.s_dsum, sizeof(G), rr.t[1].next_slot());
    rr.init(ring);
  }
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  if (warp == warps) {
    if (lane == 0) rr.fill(ring, stages, p.rows, err);
    return;
  }
  const Row op(p, a);
  const uint32_t slot_h = (uint32_t)ring_slot(p.cols * sizeof(T)), slot_g = (uint32_t)ring_slot(p.cols * sizeof(G));
  const float inv_cols = 1.f / (float)p.cols;
  const int lead = ALIKE ? (int)(rr.t[0].off(blockIdx.x) / sizeof(T)) : 0;
  auto column = [&](int j) { return (j * ring.threads + (int)threadIdx.x) * V - lead; };
  float *held_w = reinterpret_cast<float *>(stages + ring.stages * ring.stage_bytes);  // ALIKE: from column -lead on
  if (ALIKE) {
    const bool w_grid = lead == 0 && row_vec_ok(a.w, 0, 1, p.dt_w == EIR_FP32 ? 4 : 2, V);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = column(j);
      float w[V];
#pragma unroll
      for (int e = 0; e < V; ++e) w[e] = 1.f;
      if (a.w && w_grid && c < p.cols) {
        load_shared_any<V>(a.w, p.dt_w, c, p.cols, true, w);
      } else if (a.w) {
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = c + e >= 0 && c + e < p.cols ? ld_any(a.w, p.dt_w, c + e) : 0.f;
      }
#pragma unroll
      for (int e = 0; e < V; e += 4)
        *reinterpret_cast<float4 *>(held_w + c + lead + e) = make_float4(w[e], w[e + 1], w[e + 2], w[e + 3]);
    }
  }
  float dw[N][V];
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) dw[j][e] = 0.f;
  int stage = 0, turn = 0;
  uint32_t phase = 0;
  float next = a.rstd[blockIdx.x];
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    const float unit = next;
    if (row + gridDim.x < p.rows) next = a.rstd[row + gridDim.x];
    const bool late = !rr.wait(stage, phase, err);
    uint8_t const *at = stages + stage * ring.stage_bytes, *dy_at = at + slot_h, *sum_at = dy_at + slot_g;
    const uint32_t off_h = GRID ? 0 : rr.t[0].off(row), off_d = GRID ? 0 : rr.t[1].off(row);
    const uint32_t off_s = GRID ? 0 : rr.t[2].off(row);
    float held[N][V];
    typename Row::PieceH h[N];
    float gh = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = column(j);
      typename Row::PieceG dy, s;
      if ((GRID || ALIKE) && c >= p.cols) continue;
      float w[V];
      if (ALIKE) {
#pragma unroll
        for (int e = 0; e < V; e += 4) {
          const float4 q = *reinterpret_cast<float4 const *>(held_w + c + lead + e);
          w[e] = q.x, w[e + 1] = q.y, w[e + 2] = q.z, w[e + 3] = q.w;
        }
      } else {
        op.weight(c, w);
      }
      if (GRID || ALIKE) {
        h[j].template load<false>(at + (c + lead) * (int)sizeof(T));
        dy.template load<false>(dy_at + (c + lead) * (int)sizeof(G));
        if (a.dsum) s.template load<false>(sum_at + (c + lead) * (int)sizeof(G));
        if (ALIKE && (c < 0 || c + V > p.cols)) {  // bytes of other rows, or of none
          h[j].clear_outside(c, (int)p.cols);
          dy.clear_outside(c, (int)p.cols);
          if (a.dsum) s.clear_outside(c, (int)p.cols);
        }
      } else {
        h[j].load_slot(at, off_h, c, p.cols);
        dy.load_slot(dy_at, off_d, c, p.cols);
        if (a.dsum) s.load_slot(sum_at, off_s, c, p.cols);
      }
      op.template take<true, true>(w, h[j], dy, s, unit, held[j], gh, dw[j]);
    }
    fence_proxy_async_smem();  // the row is in registers: its stage may be copied over
    __syncwarp();
    if (lane == 0) mbar_arrive(&rr.empty[stage]);
    gh = warp_sum(gh);
    const bool warp_late = __any_sync(0xffffffffu, late);
    if (lane == 0) {
      red[turn][warp] = __float_as_uint(gh);
      red[turn][32 + warp] = warp_late;
    }
    ring_sync(ring.threads);
    // all threads leave together where a wait has given up
    if (__any_sync(0xffffffffu, lane < warps && red[turn][32 + lane] != 0)) break;
    gh = warp_sum(lane < warps ? __uint_as_float(red[turn][lane]) : 0.f);
    const float k = unit * unit * (gh * inv_cols);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = column(j);
      if (ALIKE && (c < 0 || c + V > p.cols)) op.give_some(row, c, held[j], h[j], k);
      else op.give(row, c, held[j], h[j], k);
    }
    if (++stage == ring.stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
  if (a.part != nullptr) {
    float *part = a.part + (int64_t)blockIdx.x * norm_part_pitch(p.cols);
    if (ALIKE && lead != 0) {  // through the weight's place, into whole lines
#pragma unroll
      for (int j = 0; j < N; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) held_w[column(j) + lead + e] = dw[j][e];
      ring_sync(ring.threads);
      for (int c = threadIdx.x; c < p.cols; c += ring.threads) part[c] = held_w[c + lead];
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) put_part<V>(part, column(j), p.cols, dw[j]);
    }
  }
}

// wide rows: h, g + dsum and the block's weight gradient stay in shared memory
// (CACHED); else the row is read again, and the weight gradient is added up in the block's
// partial row (always by the same thread)
template <typename T, typename G, bool CACHED>
__global__ void __launch_bounds__(512) norm_backward_wide_kernel(const NormParams p, const NormGradPtrs a) {
  using Row = NormBackRow<T, G, false>;
  constexpr int V = Row::V, W = Row::PieceH::kWords;
  __shared__ uint32_t red[2][64];
  extern __shared__ uint32_t held_words[];  // h as read, g + dsum, weight gradients: [piece][word][thread]
  pdl_launch_dependents();
  pdl_wait();
  const Row op(p, a);
  const int threads = blockDim.x, pieces = (int)((p.cols + (int64_t)threads * V - 1) / ((int64_t)threads * V));
  uint32_t *held_h = held_words + threadIdx.x;
  float *held_g = reinterpret_cast<float *>(held_h + pieces * W * threads);
  float *held_w = held_g + pieces * V * threads;
  float *part = a.part ? a.part + (int64_t)blockIdx.x * norm_part_pitch(p.cols) : nullptr;
  auto column = [&](int j) { return ((int64_t)j * threads + threadIdx.x) * V; };
  if (CACHED) {
    for (int i = 0; i < pieces * V; ++i) held_w[i * threads] = 0.f;
  }
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    const float rstd = a.rstd[row];
    float gh = 0.f;
#pragma unroll 2
    for (int j = 0; j < pieces; ++j) {
      typename Row::PieceH h;
      typename Row::PieceG dy, s;
      float g[V], dw[V];
      op.load(row, column(j), h, dy);
      if (CACHED) {
        op.load_sum(row, column(j), s);
#pragma unroll
        for (int e = 0; e < V; ++e) dw[e] = held_w[(j * V + e) * threads];
      }
      float w[V];
      op.weight(column(j), w);
      op.template take<true, CACHED>(w, h, dy, s, rstd, g, gh, dw);
      if (CACHED) {
#pragma unroll
        for (int e = 0; e < V; ++e) held_w[(j * V + e) * threads] = dw[e];
#pragma unroll
        for (int i = 0; i < W; ++i) held_h[(j * W + i) * threads] = h.w[i];
#pragma unroll
        for (int e = 0; e < V; ++e) held_g[(j * V + e) * threads] = g[e];
      }
    }
    uint32_t unused = 0;
    row_sum_max<true, false>(gh, unused, red[turn], threads >> 5);
    const float k = op.factor(rstd, gh);
#pragma unroll 2
    for (int j = 0; j < pieces; ++j) {
      const int64_t c = column(j);
      typename Row::PieceH h;
      float g[V];
      if (CACHED) {
#pragma unroll
        for (int i = 0; i < W; ++i) h.w[i] = held_h[(j * W + i) * threads];
#pragma unroll
        for (int e = 0; e < V; ++e) g[e] = held_g[(j * V + e) * threads];
      } else {
        typename Row::PieceG dy, s;
        float dw[V], again = 0.f;
        op.load(row, c, h, dy);
        op.load_sum(row, c, s);
#pragma unroll
        for (int e = 0; e < V; ++e) dw[e] = part && row != blockIdx.x && c + e < p.cols ? part[c + e] : 0.f;
        float w[V];
        op.weight(c, w);
        op.template take<false, true>(w, h, dy, s, rstd, g, again, dw);
        if (part) {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (c + e < p.cols) part[c + e] = dw[e];
        }
      }
      op.give(row, c, g, h, k);
    }
  }
  if (CACHED && part) {
    for (int j = 0; j < pieces; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (column(j) + e < p.cols) part[column(j) + e] = held_w[(j * V + e) * threads];
  }
}

// dw[c] = sum of the partial rows: COLS columns a block in 16-byte pieces (the partial rows' pitch
// is a multiple of 16 bytes), ROWS rows at once, whose sums are added in order
template <int COLS>
__global__ void __launch_bounds__(1024) norm_dweight_kernel(int64_t cols, float const *__restrict__ part,
                                                            int64_t pitch, int64_t n_part, float *__restrict__ dw) {
  constexpr int ROWS = 4096 / COLS;
  __shared__ float sums[ROWS][COLS + 1];
  pdl_launch_dependents();
  pdl_wait();
  const int x = threadIdx.x % (COLS / 4) * 4, y = threadIdx.x / (COLS / 4);
  const int64_t c = (int64_t)blockIdx.x * COLS + x;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < cols) {
    for (int64_t i = y; i < n_part; i += 4 * ROWS) {
      float4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = i + ROWS * j < n_part ? *reinterpret_cast<float4 const *>(part + (i + ROWS * j) * pitch + c)
                                     : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < 4; ++j) s = make_float4(s.x + v[j].x, s.y + v[j].y, s.z + v[j].z, s.w + v[j].w);
    }
  }
  sums[y][x] = s.x;
  sums[y][x + 1] = s.y;
  sums[y][x + 2] = s.z;
  sums[y][x + 3] = s.w;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;  // a warp a column
  if (warp >= COLS) return;
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < ROWS; i += 32) t += sums[i + lane][warp];
  t = warp_sum(t);
  if (lane == 0 && (int64_t)blockIdx.x * COLS + warp < cols) dw[(int64_t)blockIdx.x * COLS + warp] = t;
}

// ---------------------------------------------------------------- launchers

// block and grid: persistent blocks of up to 1024 threads an SM (64 registers a thread)
struct RowGrid {
  int warps;      // of a row
  int threads;    // of a block: four rows of a warp, or a row
  int64_t grid;
};
static RowGrid row_grid(int64_t rows, int64_t cols, int per, int num_sms) {
  RowGrid g;
  g.warps = (int)((cols + 32 * per - 1) / (32 * per));
  g.threads = g.warps == 1 ? 128 : g.warps * 32;
  const int64_t blocks = g.warps == 1 ? (rows + 3) / 4 : rows;
  g.grid = std::min<int64_t>(blocks, (int64_t)num_sms * (1024 / g.threads));
  return g;
}

constexpr int kSmemMost = 227 * 1024 - 1024;  // dynamic, beside the reductions' words

// wide rows: threads of a block, bytes that it holds (0: the row is read twice), and the grid
struct WideGrid {
  int threads;
  int64_t bytes;
  int64_t grid;
};
static WideGrid wide_grid(int64_t rows, int64_t cols, int threads, int v, int per_col, int num_sms) {
  WideGrid g;
  g.threads = threads;
  g.bytes = (cols + (int64_t)threads * v - 1) / ((int64_t)threads * v) * threads * v * per_col;
  if (g.bytes > kSmemMost) g.bytes = 0;
  const int64_t fit = g.bytes ? std::max<int64_t>(1, std::min<int64_t>(1024 / threads, kSmemMost / g.bytes)) : 1024 / threads;
  g.grid = std::min<int64_t>(rows, num_sms * fit);
  return g;
}

template <typename... KArgs, typename... Args>
static cudaError_t launch_wide(void (*kern)(KArgs...), WideGrid const &g, cudaStream_t st, Args const &...args) {
  if (g.bytes > 48 * 1024 - 1024) {
    cudaError_t e = allow_all_smem(reinterpret_cast<void const *>(kern));
    if (e != cudaSuccess) return e;
  }
  return launch_kernel(kern, dim3((unsigned)g.grid), dim3(g.threads), (size_t)g.bytes, st, args...);
}

// stages of a ring for `blocks` blocks an SM at most, `more` bytes behind them (fewer where two stages a block do not
// fit otherwise); 0 stages: too wide
static int64_t ring_fit(int64_t stage_bytes, int64_t blocks, RingShape *r, int64_t more = 0) {
  r->stage_bytes = stage_bytes;
  r->more = more;
  while (blocks > 1 && (2 * stage_bytes + more + 2048) * blocks > kSmemMost) --blocks;
  r->stages = (int)std::min<int64_t>(kMostStages, (kSmemMost / blocks - 2048 - more) / stage_bytes);
  if (r->stages < 2) r->stages = 0;
  return blocks;
}

template <typename... KArgs, typename... Args>
static cudaError_t launch_ring(void (*kern)(KArgs...), RingShape const &r, int64_t grid, cudaStream_t st,
                               Args const &...args) {
  const size_t bytes = (size_t)(r.stages * r.stage_bytes + r.more);
  cudaError_t e = allow_all_smem(reinterpret_cast<void const *>(kern));
  if (e != cudaSuccess) return e;
  return launch_kernel(kern, dim3((unsigned)grid), dim3(r.threads + 32), bytes, st, args...);
}

template <typename T, typename OUT, bool QUANT>
static cudaError_t launch_norm_out(NormParams const &p, NormPtrs const &a, uint32_t *err, int num_sms,
                                   cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  if (p.cols > 1024 * kPer<T, QUANT>) {
    const WideGrid g = wide_grid(p.rows, p.cols, 1024, V, 4, num_sms);
    return launch_wide(g.bytes ? norm_wide_kernel<T, OUT, QUANT, true> : norm_wide_kernel<T, OUT, QUANT, false>, g, st, p, a);
  }
  const bool grid = p.cols % V == 0 && row_vec_ok(a.x, p.s_x, p.rows, sizeof(T), V) &&
                    row_vec_ok(a.res, p.s_res, p.rows, sizeof(T), V) &&
                    row_vec_ok(a.sum, p.s_sum, p.rows, sizeof(T), V) &&
                    row_vec_ok(a.out, p.s_out, p.rows, sizeof(OUT), V) &&
                    row_vec_ok(a.w, 0, 1, p.dt_w == EIR_FP32 ? 4 : 2, V);
  const RowGrid g = row_grid(p.rows, p.cols, kPer<T, QUANT>, num_sms);
  if (!grid && g.warps > 1 && p.cols <= (1024 - 32) * kPer<T, false>) {
    RingShape r;
    r.threads = (int)((p.cols + kPer<T, false> - 1) / kPer<T, false> + 31) / 32 * 32;
    const int64_t blocks = ring_fit(ring_slot(p.cols * sizeof(T)) * (a.res ? 2 : 1), 1024 / (r.threads + 32), &r);
    if (r.stages > 0)
      return launch_ring(norm_ring_kernel<T, OUT, QUANT>, r, std::min<int64_t>(p.rows, num_sms * blocks), st, p, a, r,
                         err);
  }
  auto kern = grid ? norm_kernel<T, OUT, QUANT, true> : norm_kernel<T, OUT, QUANT, false>;
  return launch_kernel(kern, dim3((unsigned)g.grid), dim3(g.threads), 0, st, p, a, g.warps);
}

template <typename T>
static cudaError_t launch_norm_t(NormParams const &p, NormPtrs const &a, uint32_t *err, int num_sms, cudaStream_t st) {
  if (p.dt_out == EIR_FP32) return launch_norm_out<T, float, false>(p, a, err, num_sms, st);
  if (p.dt_out == EIR_BF16) return launch_norm_out<T, __nv_bfloat16, false>(p, a, err, num_sms, st);
  return launch_norm_out<T, int8_t, false>(p, a, err, num_sms, st);
}

cudaError_t launch_norm(NormParams const &p, NormPtrs const &a, uint32_t *err, int num_sms, cudaStream_t st) {
  return p.dt == EIR_FP32 ? launch_norm_t<float>(p, a, err, num_sms, st)
                          : launch_norm_t<__nv_bfloat16>(p, a, err, num_sms, st);
}

cudaError_t launch_quantize(QuantizeParams const &p, void const *x, int8_t *q, float *scale, uint32_t *err,
                            int num_sms, cudaStream_t st) {
  NormParams n;
  n.rows = p.rows;
  n.cols = p.cols;
  n.dt = p.dt;
  n.dt_out = EIR_INT8;
  n.s_x = p.s_x;
  n.s_out = p.s_out;
  const NormPtrs a{x, nullptr, nullptr, nullptr, q, scale, nullptr};
  return p.dt == EIR_FP32 ? launch_norm_out<float, int8_t, true>(n, a, err, num_sms, st)
                          : launch_norm_out<__nv_bfloat16, int8_t, true>(n, a, err, num_sms, st);
}

// Elements of a thread of the backward ring: 8, 16 or 32. Few threads with much to do each make a row's barriers
// cheap where many rows follow one another, more threads make few rows quick (8192 x 4096 BF16: 45.0 us
// with 16 elements, 49.2 with 8; 8192 x 2048: 26.0 and 29.5; 1237 x 2312 FP32: 14.8 and 12.1).
static int back_per(int64_t rows, int64_t cols, int num_sms) {
  const int least = rows >= 32 * (int64_t)num_sms ? 16 : 8;
  return cols <= kBackThreads * least ? least : cols <= kBackThreads * 16 ? 16 : 32;
}
// blocks an SM, if their stages fit, by the registers of a thread; 0: too wide
static int64_t back_ring_blocks(int64_t cols, int per, int *threads) {
  *threads = (int)((cols + per - 1) / per + 31) / 32 * 32;
  const int on_sm = per == 8 ? 2 * (kBackThreads + 32) : per == 16 ? 640 : kBackThreads + 32;
  return *threads > kBackThreads ? 0 : std::min(8, on_sm / (*threads + 32));
}

int64_t norm_backward_parts(NormParams const &p, int num_sms) {
  int threads = 0;
  int64_t an_sm = 2;  // narrow rows and wide ones
  if (p.cols > 32 * kPerBack) {
    for (int per : {8, 16, 32}) an_sm = std::max(an_sm, back_ring_blocks(p.cols, per, &threads));
  }
  return std::min<int64_t>(p.rows, num_sms * an_sm);
}

template <typename T, typename G>
static cudaError_t launch_norm_backward_t(NormParams const &p, NormGradPtrs const &a, uint32_t *err, int num_sms,
                                          cudaStream_t st, int64_t *parts) {
  constexpr int V = NormBackRow<T, G, false>::V;
  const bool grid = p.cols % V == 0 && row_vec_ok(a.h, p.s_h, p.rows, sizeof(T), 16 / sizeof(T)) &&
                    row_vec_ok(a.dy, p.s_dy, p.rows, sizeof(G), 16 / sizeof(G)) &&
                    row_vec_ok(a.dsum, p.s_dsum, p.rows, sizeof(G), 16 / sizeof(G)) &&
                    row_vec_ok(a.dx, p.s_dx, p.rows, sizeof(G), V) &&
                    row_vec_ok(a.w, 0, 1, p.dt_w == EIR_FP32 ? 4 : 2, V);
  if (p.cols <= 32 * kPerBack) {
    *parts = std::min<int64_t>((p.rows + kBackWarps - 1) / kBackWarps, num_sms * 2);
    auto kern = grid ? norm_backward_kernel<T, G, true> : norm_backward_kernel<T, G, false>;
    return launch_kernel(kern, dim3((unsigned)*parts), dim3(kBackWarps * 32), (size_t)(kBackWarps * 4 * p.cols), st, p, a);
  }
  // all rows of a block alike: the same offset of a row's tensors, whose strides step alike
  auto same = [&](void const *q, int64_t stride) {
    return q == nullptr || ((reinterpret_cast<uintptr_t>(q) - reinterpret_cast<uintptr_t>(a.h)) % 16 == 0 &&
                            (p.rows == 1 || (stride - p.s_h) * (int64_t)sizeof(T) % 16 == 0));
  };
  const bool could = std::is_same<T, G>::value && same(a.dy, p.s_dy) && same(a.dsum, p.s_dsum) && same(a.dx, p.s_dx);
  for (bool alike : {true, false}) {  // (with the weight in shared memory a ring may be too wide)
    if (alike && !could) continue;
    const int64_t cols = p.cols + (alike && !grid ? V - 1 : 0);  // that the pieces cover
    const int per = back_per(p.rows, cols, num_sms);
    RingShape r;
    const int64_t most = back_ring_blocks(cols, per, &r.threads);
    if (most == 0) continue;
    const int64_t bytes = ring_slot(p.cols * sizeof(T)) + ring_slot(p.cols * sizeof(G)) * (a.dsum ? 2 : 1);
    const int64_t blocks = ring_fit(bytes, most, &r, alike ? (int64_t)r.threads * per * 4 : 0);
    if (r.stages == 0) continue;
    *parts = std::min<int64_t>(p.rows, num_sms * blocks);
    // rows on the grid read the weight where it is unless a block has several of them (8192 x 4096
    // BF16, 8 elements a thread: 52.2 us so, 49.2 from shared memory; 2048 x 1024: 9.8 and 11.2)
    if (alike && grid && p.rows < 4 * *parts) continue;
    constexpr int kPeriod = 16 / (int)sizeof(T);
    if (alike && !grid && *parts < p.rows) *parts = *parts / kPeriod * kPeriod;
    auto pick = [&](auto lie) {
      constexpr RowsLie L = decltype(lie)::value;
      return per == 8    ? norm_backward_ring_kernel<T, G, 8 / V, L>
             : per == 16 ? norm_backward_ring_kernel<T, G, 16 / V, L>
                         : norm_backward_ring_kernel<T, G, 32 / V, L>;
    };
    auto kern = grid ? pick(std::integral_constant<RowsLie, kRowsOnGrid>{})
                     : pick(std::integral_constant<RowsLie, kRowsAnyhow>{});
    if constexpr (std::is_same<T, G>::value) {
      if (alike) kern = pick(std::integral_constant<RowsLie, kRowsAlike>{});
    }
    return launch_ring(kern, r, *parts, st, p, a, r, err);
  }
  const WideGrid g = wide_grid(p.rows, p.cols, 512, V, sizeof(T) + 8, num_sms);
  *parts = g.grid;
  return launch_wide(g.bytes ? norm_backward_wide_kernel<T, G, true> : norm_backward_wide_kernel<T, G, false>, g, st, p,
                     a);
}

cudaError_t launch_norm_backward(NormParams const &p, NormGradPtrs const &a, uint32_t *err, int num_sms,
                                 cudaStream_t st, int64_t *parts) {
  if (p.dt == EIR_FP32)
    return p.dt_grad == EIR_FP32 ? launch_norm_backward_t<float, float>(p, a, err, num_sms, st, parts)
                                 : launch_norm_backward_t<float, __nv_bfloat16>(p, a, err, num_sms, st, parts);
  return p.dt_grad == EIR_FP32
             ? launch_norm_backward_t<__nv_bfloat16, float>(p, a, err, num_sms, st, parts)
             : launch_norm_backward_t<__nv_bfloat16, __nv_bfloat16>(p, a, err, num_sms, st, parts);
}

cudaError_t launch_norm_dweight(NormParams const &p, float const *part, int64_t n_part, float *dw,
                                cudaStream_t st) {
  // narrower blocks where wide ones leave SMs without work
  const int n = p.cols >= 4096 ? 32 : p.cols >= 2048 ? 16 : 8;
  auto kern = n == 32 ? norm_dweight_kernel<32> : n == 16 ? norm_dweight_kernel<16> : norm_dweight_kernel<8>;
  return launch_kernel(kern, dim3((unsigned)((p.cols + n - 1) / n)), dim3(1024), 0, st, p.cols, part,
                       norm_part_pitch(p.cols), n_part, dw);
}

}  // namespace eir
