// Tiles of the attention kernels: 32 x 32 products on the matrix cores over 16
// of the contraction, fed from row-major tiles in LDS.
//
// A wave's 32 x 32 result holds column lane & 31 in each lane and, in register
// r, row (r & 3) + 8 (r >> 2) + 4 (lane >> 5).  As the second operand of a
// product that contracts over those rows, registers 8 s .. 8 s + 7 are the
// fragment of rows 16 s .. 16 s + 15 as they stand, provided the first operand
// takes its rows in the same order: 4 h .. 4 h + 3 and 8 + 4 h .. 8 + 4 h + 3 for
// the lanes' half h.  load_turned reads it so.  Probabilities therefore go from
// one product into the next without leaving their registers.
#pragma once

#include "sequence.h"

namespace gs {
namespace att {

using namespace seq;

using Acc = FloatVec<16>;

template <typename T>
using Frag = Vec<T, 8>;

__device__ __forceinline__ int acc_row(int r) {
  return (r & 3) + 8 * (r >> 2) + 4 * (int(threadIdx.x & 63) >> 5);
}

__device__ __forceinline__ void mma(const Frag<bf16>& a, const Frag<bf16>& b, Acc& c) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void mma(const Frag<f16>& a, const Frag<f16>& b, Acc& c) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// float32 has products over 2 of the contraction: element i of both halves.
__device__ __forceinline__ void mma(const Frag<float>& a, const Frag<float>& b, Acc& c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
}

// Row pitch of an LDS tile in elements: 16 bytes more than the row, so that the
// 16-byte reads of neighbouring rows fall into different banks.
template <typename T, int kDim>
constexpr int kPitch = kDim + 16 / int(sizeof(T));

// Rows row0 + (lane & 31), contraction k0 + 8 (lane >> 5) .. + 7.
template <typename T>
__device__ __forceinline__ Frag<T> load_rows(const T* tile, int pitch, int row0, int k0) {
  const int lane = threadIdx.x & 63;
  const T* p = tile + (row0 + (lane & 31)) * pitch + k0 + 8 * (lane >> 5);
  if constexpr (sizeof(T) == 2) {
    return *reinterpret_cast<const Frag<T>*>(__builtin_assume_aligned(p, 16));
  } else {
    const Vec<T, 4> lo = *reinterpret_cast<const Vec<T, 4>*>(p);
    const Vec<T, 4> hi = *reinterpret_cast<const Vec<T, 4>*>(p + 4);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// Columns col0 + (lane & 31); the contraction runs over the tile's rows row0 ..
// row0 + 15 in the order of a result's registers.  16-bit types use the
// transposing read: 16 lanes fetch 4 rows of 16 columns and each gets a column.
template <typename T>
__device__ __forceinline__ Frag<T> load_turned(const T* tile, int pitch, int row0, int col0) {
  const int lane = threadIdx.x & 63;
  if constexpr (sizeof(T) == 2) {
    using Short4 = Vec<short, 4>;
    using Lds = __attribute__((address_space(3))) Short4*;
    const T* p = tile + (row0 + 4 * (lane >> 5) + ((lane & 15) >> 2)) * pitch + col0 +
                 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const Short4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(p));
    const Short4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(p + 8 * pitch));
    return __builtin_bit_cast(Frag<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    const T* p = tile + (row0 + 4 * (lane >> 5)) * pitch + col0 + (lane & 31);
    Frag<T> f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = p[i * pitch];
      f[4 + i] = p[(8 + i) * pitch];
    }
    return f;
  }
}

// Eight elements of global memory, 16-byte aligned; zeros where !ok.
template <typename T>
__device__ __forceinline__ Frag<T> load_global(const T* p, bool ok) {
  Frag<T> f(T(0.0f));
  if (ok) {
    if constexpr (sizeof(T) == 2) {
      f = *reinterpret_cast<const Frag<T>*>(__builtin_assume_aligned(p, 16));
    } else {
      const Vec<T, 4> lo = *reinterpret_cast<const Vec<T, 4>*>(p);
      const Vec<T, 4> hi = *reinterpret_cast<const Vec<T, 4>*>(p + 4);
      f = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  return f;
}

// The fragment of rows 16 s .. 16 s + 15 of a result, rounded to the type.
template <typename T>
__device__ __forceinline__ Frag<T> acc_frag(const Acc& c, int s) {
  FloatVec<8> v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = c[8 * s + i];
  return from_float<T, 8>(v);
}

// A [kRows, kDim] tile on its way from global memory through a workgroup's
// registers into LDS.  Rows outside [0, end) and columns from dim on are zeros.
template <typename T, int kRows, int kDim, int kThreads>
struct Stage {
  static constexpr int kV = 16 / int(sizeof(T));
  static constexpr int kPerRow = kDim / kV;
  static constexpr int kCount = kRows * kPerRow / kThreads;
  static_assert(kRows * kPerRow % kThreads == 0, "whole chunks per thread");
  Vec<T, kV> r[kCount];

  __device__ __forceinline__ void load(const T* base, int64_t stride, int row0, int end, int dim) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int chunk = i * kThreads + int(threadIdx.x);
      const int row = row0 + chunk / kPerRow, col = chunk % kPerRow * kV;
      r[i] = Vec<T, kV>(T(0.0f));
      if (row >= 0 && row < end && col < dim)
        r[i] = *reinterpret_cast<const Vec<T, kV>*>(base + row * stride + col);
    }
  }
  __device__ __forceinline__ void store(T* tile) const {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int chunk = i * kThreads + int(threadIdx.x);
      *reinterpret_cast<Vec<T, kV>*>(tile + chunk / kPerRow * kPitch<T, kDim> +
                                     chunk % kPerRow * kV) = r[i];
    }
  }
};

__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.4028235e38f; }

// acc[n] += a[n] b over 16 of the contraction, where `seen(k)` says whether the
// lane's column takes element k of it at all.  b is zero where it does not, but
// zero times an infinity or a NaN of a, which the column must not see, is a NaN:
// where a holds one, the product is formed without it, and what it gives is
// added, one element of the contraction at a time, to the columns that see it.
// The others keep the bits that they would have had.
template <typename T, int kCount, typename F>
__device__ __forceinline__ void mma_seen(Frag<T> (&a)[kCount], const Frag<T>& b,
                                         Acc (&acc)[kCount], F&& seen) {
  const int half = int(threadIdx.x & 63) >> 5;
#pragma unroll
  for (int n = 0; n < kCount; ++n) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) bad |= !finite(float(a[n][i]));
    if (__any(bad)) {
#pragma unroll 1
      for (int k = 0; k < 16; ++k) {
        const int at = ((k >> 2) & 1) == half ? (k & 3) + 4 * (k >> 3) : -1;
        Frag<T> a1(T(0.0f)), b1(T(0.0f));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (i != at) continue;
          b1[i] = b[i];
          if (!finite(float(a[n][i]))) a1[i] = a[n][i];
        }
        Acc one(0.0f);
        mma(a1, b1, one);
        const bool see = seen(k);
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[n][r] += see ? one[r] : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!finite(float(a[n][i]))) a[n][i] = T(0.0f);
    }
    mma(a[n], b, acc[n]);
  }
}

// Problem of one call; strides in elements, rows contiguous.
struct Strides {
  int64_t batch, token, head;
};

struct Problem {
  int batch, heads, kv_heads, dim;
  int queries, keys;
  int window, sinks;
  float scale;
  const int32_t* lengths;  // keys of each sequence that exist, or null: all

  __device__ __forceinline__ int offset() const { return keys - queries; }
  __device__ __forceinline__ int length(int b) const {
    return lengths ? min(max(lengths[b], 0), keys) : keys;
  }
  // Key j (below the length) is seen from position p.
  __device__ __forceinline__ bool sees(int p, int j, int length) const {
    return j <= p && (j > p - window || j < sinks) && j < length;
  }
};

// Workgroups in order of their index go to the 8 XCDs in turn: gives each XCD a
// contiguous run of the work, so that neighbours share its L2.
__device__ __forceinline__ int64_t xcd_order(int64_t id, int64_t count) {
  const int64_t per = (count + 7) / 8;
  return (id & 7) * per + (id >> 3);
}
inline int64_t xcd_grid(int64_t count) { return (count + 7) / 8 * 8; }

constexpr float kLog2e = 1.4426950408889634f;

// 2^v.  The instruction flushes results below 2^-126 to zero, which no 16-bit
// type tells from what it would hold; float32 keeps them.
template <typename T>
__device__ __forceinline__ float power(float v) {
  if constexpr (sizeof(T) == 4)
    return exp2f(v);
  else
    return __builtin_amdgcn_exp2f(v);
}

}  // namespace att

// Argument checks of the attention entry points (window_attention.hip).
int check_attention(const gs_attention& d);
int check_rows(const void* p, const int64_t* strides, int32_t type, const char* name);
att::Problem make_problem(const gs_attention& d, const int32_t* lengths);

}  // namespace gs
