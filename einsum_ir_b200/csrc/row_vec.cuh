// Pieces of rows as the row operators move them: V neighbouring elements a
// thread, lane l + 1 the V after those of lane l, held as raw words until they
// are used. Rows that start on the pieces' grid (and have whole pieces) move
// with one vector access a piece. Others are read as the two aligned vectors
// that cover a piece, shifted into place, and written as aligned vectors put
// together from the pieces of two lanes, with single elements at the ends of
// a warp's span: the shift is the same for a whole row.
#pragma once

#include "op_common.cuh"

namespace eir {

// words W of the 2 W words (lo, hi) from byte `shift` on (0 <= shift < 4 W)
template <int W>
__device__ __forceinline__ void shifted_words(uint32_t const (&lo)[W], uint32_t const (&hi)[W], uint32_t shift,
                                              uint32_t (&out)[W]) {
  const uint32_t sh = 8 * (shift & 3), first = shift >> 2;
#pragma unroll
  for (int s = 0; s < W; ++s) {
    if (first == (uint32_t)s) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const uint32_t a = i + s < W ? lo[i + s < W ? i + s : 0] : hi[i + s < W ? 0 : i + s - W];
        const uint32_t b = i + s + 1 < W ? lo[i + s + 1 < W ? i + s + 1 : 0] : hi[i + s + 1 < W ? 0 : i + s + 1 - W];
        out[i] = __funnelshift_r(a, b, sh);
      }
    }
  }
}

template <typename T, int V>
struct RowPiece {
  static constexpr int kBytes = V * (int)sizeof(T);
  static constexpr int kWords = kBytes / 4;
  static_assert(kBytes % 4 == 0 && kBytes <= 32, "whole words");
  uint32_t w[kWords];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  // streaming loads (coherent: an output may share the input's memory), or loads kept in L1
  template <bool STREAM>
  __device__ __forceinline__ void load(void const *p) {
    if constexpr (kBytes == 4) {
      w[0] = STREAM ? __ldcs(static_cast<uint32_t const *>(p)) : *static_cast<uint32_t const *>(p);
    } else if constexpr (kBytes == 8) {
      const uint2 v = STREAM ? __ldcs(static_cast<uint2 const *>(p)) : *static_cast<uint2 const *>(p);
      w[0] = v.x;
      w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) {
        uint4 const *q = static_cast<uint4 const *>(p) + i;
        const uint4 v = STREAM ? __ldcs(q) : *q;
        w[4 * i] = v.x;
        w[4 * i + 1] = v.y;
        w[4 * i + 2] = v.z;
        w[4 * i + 3] = v.w;
      }
    }
  }
  __device__ __forceinline__ void store(void *p) const {
    if constexpr (kBytes == 4) {
      *static_cast<uint32_t *>(p) = w[0];
    } else if constexpr (kBytes == 8) {
      *static_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i)
        static_cast<uint4 *>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  }

  // elements c .. c + V - 1 of a row of any alignment, zeros from column
  // `cols` on; begin, end: the tensor's bytes, outside of which nothing is read
  __device__ __forceinline__ void load_any(T const *row, int64_t c, int64_t cols, uintptr_t begin, uintptr_t end) {
    constexpr uintptr_t kUnit = kBytes < 16 ? kBytes : 16;
    const uintptr_t at = reinterpret_cast<uintptr_t>(row + c), off = at % kUnit;
    if (c + V <= cols) {
      if (off == 0) {
        load<false>(reinterpret_cast<void const *>(at));
        return;
      }
      if constexpr (kBytes <= 16) {
        const uintptr_t base = at - off;
        if (base >= begin && base + 2 * kBytes <= end) {
          RowPiece lo, hi;
          lo.template load<false>(reinterpret_cast<void const *>(base));
          hi.template load<false>(reinterpret_cast<void const *>(base + kBytes));
          shifted_words<kWords>(lo.w, hi.w, (uint32_t)off, w);
          return;
        }
      }
    }
    zero();
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (c + e < cols) {
        if constexpr (sizeof(T) == 4) w[e] = *reinterpret_cast<uint32_t const *>(row + c + e);
        else w[e / 2] |= (uint32_t)*reinterpret_cast<unsigned short const *>(row + c + e) << (16 * (e % 2));
      }
    }
  }

  // the same from a copy of the row in shared memory, which starts `off` bytes
  // after `slot` (16-byte aligned; at least 48 bytes behind the row may be read)
  __device__ __forceinline__ void load_slot(uint8_t const *slot, uint32_t off, int c, int64_t cols) {
    uint8_t const *at = slot + c * (int)sizeof(T);
    if (c >= cols) {
      zero();
      return;
    }
    if (kBytes < 16) {  // (a piece of a narrower type: its own grid within the row's shift)
      at += off / kBytes * kBytes;
      off %= kBytes;
    }
    load<false>(at);
    if (off != 0) {
      RowPiece hi;
      uint32_t lo[kWords];
#pragma unroll
      for (int i = 0; i < kWords; ++i) lo[i] = w[i];
      hi.template load<false>(at + kBytes);
      shifted_words<kWords>(lo, hi.w, off, w);
    }
    if (c + V > cols) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (c + e < cols) continue;
        if constexpr (sizeof(T) == 4) w[e] = 0;
        else w[e / 2] &= e % 2 ? 0x0000ffffu : 0xffff0000u;
      }
    }
  }

  // zeros in place of the elements outside columns 0 .. cols - 1 of a piece at column c
  __device__ __forceinline__ void clear_outside(int c, int cols) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (c + e >= 0 && c + e < cols) continue;
      if constexpr (sizeof(T) == 4) w[e] = 0;
      else w[e / 2] &= e % 2 ? 0x0000ffffu : 0xffff0000u;
    }
  }

  // elements first .. last - 1 of the piece, one by one
  __device__ __forceinline__ void store_some(T *p, int first, int last) const {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (e < first || e >= last) continue;
      if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t *>(p + e) = w[e];
      else if constexpr (sizeof(T) == 2) *reinterpret_cast<unsigned short *>(p + e) = (unsigned short)(w[e / 2] >> (16 * (e % 2)));
      else *reinterpret_cast<uint8_t *>(p + e) = (uint8_t)(w[e / 4] >> (8 * (e % 4)));
    }
  }
  // the counterpart of load_any; all lanes of the warp call it, lane l with
  // the piece after that of lane l - 1 (c may be past the row's end)
  __device__ __forceinline__ void store_any(T *row, int64_t c, int64_t cols) const {
    constexpr int kUnit = kBytes < 16 ? kBytes : 16;
    const int own = (int)(cols - c < 0 ? 0 : cols - c > V ? V : cols - c);  // elements of this piece
    const int off = (int)(reinterpret_cast<uintptr_t>(row + c) % kUnit);
    if (off == 0 || kBytes > 16) {
      if (off == 0 && own == V) store(row + c);
      else store_some(row + c, 0, own);
      return;
    }
    const int lane = threadIdx.x & 31;
    RowPiece before, joined;
#pragma unroll
    for (int i = 0; i < kWords; ++i) before.w[i] = __shfl_up_sync(0xffffffffu, w[i], 1);
    shifted_words<kWords>(before.w, w, (uint32_t)(kBytes - off), joined.w);
    const int head = V - off / (int)sizeof(T);  // own elements in the aligned vector that starts in the piece before
    if (lane > 0 && own >= head) {
      joined.store(reinterpret_cast<char *>(row + c) - off);
    } else {
      if (lane > 0) {
        const int64_t left = cols - (c - V);
        before.store_some(row + c - V, head, (int)(left < 0 ? 0 : left > V ? V : left));
      }
      store_some(row + c, 0, own < head ? own : head);
    }
    if (lane == 31) store_some(row + c, head, own);
  }

  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
  }
  __device__ __forceinline__ float2 get2(int i) const { return make_float2(get(i), get(i + 1)); }
  // all elements from FP32, each rounded once
  __device__ __forceinline__ void set(float const (&f)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(f[i], f[i + 1]);
        w[i >> 1] = *reinterpret_cast<uint32_t const *>(&b);
      }
    }
  }
};

// V elements of a row vector whose type is a run-time choice (and which every
// row shares: loads kept in L1); zeros, or `fill`, from column `cols` on.
// `aligned`: whole pieces on the vectors' grid
template <int V>
__device__ __forceinline__ void load_shared_any(void const *p, int dt, int64_t c, int64_t cols, bool aligned,
                                                float (&f)[V]) {
  if (aligned && c + V <= cols) {
    if (dt == EIR_FP32) {
      RowPiece<float, V> r;
      r.template load<false>(static_cast<float const *>(p) + c);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = r.get(e);
    } else {
      RowPiece<__nv_bfloat16, V> r;
      r.template load<false>(static_cast<__nv_bfloat16 const *>(p) + c);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = r.get(e);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = c + e < cols ? ld_any(p, dt, c + e) : 0.f;
  }
}

// whether rows of `bytes`-byte elements, `stride` apart, lie on the grid of V-element vectors
__host__ __device__ inline bool row_vec_ok(void const *p, int64_t stride, int64_t rows, int bytes, int v) {
  const uintptr_t unit = (uintptr_t)(v * bytes < 16 ? v * bytes : 16);
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % unit == 0 &&
                          (rows <= 1 || (uintptr_t)(stride * bytes) % unit == 0));
}

// the bytes of a tensor of rows
struct RowBounds {
  uintptr_t begin, end;
};
__device__ __forceinline__ RowBounds row_bounds(void const *p, int64_t rows, int64_t cols, int64_t stride, int bytes) {
  const uintptr_t b = reinterpret_cast<uintptr_t>(p);
  return RowBounds{b, b + (uintptr_t)(((rows - 1) * stride + cols) * bytes)};
}

}  // namespace eir
