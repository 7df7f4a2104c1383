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

#include <type_traits>

#include "sequence.h"

namespace gs {
namespace att {

using namespace seq;

using Acc = FloatVec<16>;

template <typename T>
using Frag = Vec<T, 8>;

__device__ __forceinline__ constexpr int acc_row_of_half(int r) { return (r & 3) + 8 * (r >> 2); }
__device__ __forceinline__ int acc_row(int r) {
  return acc_row_of_half(r) + 4 * (int(threadIdx.x & 63) >> 5);
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

// sum + the fragment's elements: two at a time where the type has a product of
// pairs, which takes half the instructions of plain additions.
__device__ __forceinline__ float add_all(const Frag<bf16>& f, float sum) {
  const Vec<bf16, 2> one(bf16(1.0f));
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    sum = __builtin_amdgcn_fdot2_f32_bf16(Vec<bf16, 2>{f[i], f[i + 1]}, one, sum, false);
  return sum;
}
__device__ __forceinline__ float add_all(const Frag<f16>& f, float sum) {
  const Vec<f16, 2> one(f16(1.0f));
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    sum = __builtin_amdgcn_fdot2(Vec<f16, 2>{f[i], f[i + 1]}, one, sum, false);
  return sum;
}
__device__ __forceinline__ float add_all(const Frag<float>& f, float sum) {
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += f[i];
  return sum;
}

// A [kRows, kDim] tile on its way from global memory through the registers of
// kThreads threads into LDS.  Rows outside [0, end) and columns from dim on are zeros.
// A thread's places are the same in every tile, so a tile inside the tensor
// takes no address arithmetic but the wave's.
template <typename T, int kRows, int kDim, int kThreads>
struct Stage {
  static constexpr int kV = 16 / int(sizeof(T));
  static constexpr int kPerRow = kDim / kV;
  static constexpr int kStep = kThreads / kPerRow;  // rows between a thread's chunks
  static constexpr int kCount = kRows / kStep;
  static_assert(kThreads % kPerRow == 0 && kRows % kStep == 0, "whole rows per step");
  Vec<T, kV> r[kCount];
  int row, col;
  bool in;          // the thread's columns exist
  uint32_t offset;  // of the thread's first chunk, in bytes
  int64_t stride;   // of a row, in bytes

  __device__ __forceinline__ Stage(int64_t row_stride, int dim, int thread)
      : row(thread / kPerRow), col(thread % kPerRow * kV), in(col < dim),
        stride(row_stride * int64_t(sizeof(T))) {
    offset = uint32_t(row * stride) + uint32_t(col * sizeof(T));
#pragma unroll
    for (int i = 0; i < kCount; ++i) r[i] = Vec<T, kV>(T(0.0f));
  }
  __device__ __forceinline__ void load(const T* base, int row0, int end) {
    const char* first = reinterpret_cast<const char*>(base) + row0 * stride;
    if (row0 + kRows <= end) {
      if (in) {
#pragma unroll
        for (int i = 0; i < kCount; ++i)
          r[i] = *reinterpret_cast<const Vec<T, kV>*>(first + i * kStep * stride + offset);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kCount; ++i) {
        r[i] = Vec<T, kV>(T(0.0f));
        if (in && row0 + row + i * kStep < end)
          r[i] = *reinterpret_cast<const Vec<T, kV>*>(first + i * kStep * stride + offset);
      }
    }
  }
  __device__ __forceinline__ void store(T* tile) const {
#pragma unroll
    for (int i = 0; i < kCount; ++i)
      *reinterpret_cast<Vec<T, kV>*>(tile + (row + i * kStep) * kPitch<T, kDim> + col) = r[i];
  }
};

__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.4028235e38f; }

// Whether any lane's fragments hold an infinity or a NaN.
template <typename T, int kCount>
__device__ __forceinline__ bool any_not_finite(const Frag<T> (&a)[kCount]) {
  int none = 0;
  asm volatile("" : "+v"(none));  // or the compiler looks before the caller's branch
  bool bad = none != 0;
#pragma unroll
  for (int n = 0; n < kCount; ++n)
#pragma unroll
    for (int i = 0; i < 8; ++i) bad |= !finite(float(a[n][i]));
  return __any(bad);
}
template <typename T, int kCount>
__device__ __forceinline__ void drop_not_finite(Frag<T> (&a)[kCount]) {
#pragma unroll
  for (int n = 0; n < kCount; ++n)
#pragma unroll
    for (int i = 0; i < 8; ++i) a[n][i] = finite(float(a[n][i])) ? a[n][i] : T(0.0f);
}

// Infinities and NaN at places that some columns of a tile do not see.  In a
// product those columns hold a zero there, but zero times such a value is a NaN.
// So they are dropped from the first operand, and mark() notes by two bits for
// each element of the result what they add to the columns that do see them;
// apply() adds that at the end.  The other columns keep the bits that they would
// have.
template <typename T, int kCount>
struct Poison {
  uint32_t marks[kCount] = {};  // +inf: bit r, -inf: bit 16 + r, NaN: both

  // For rows row0 .. row0 + 15 and columns 32 n .. of the tile, which are
  // multiplied with b; seen(k): whether the lane's column takes row row0 + k.
  // Marks are made element by element: the code is small and needs few
  // registers beside the caller's.
  template <typename F>
  __device__ __forceinline__ void mark(const T* tile, int pitch, int row0, const Frag<T>& b,
                                       F&& seen) {
    const int lane = threadIdx.x & 63;
#pragma unroll 1
    for (int k = 0; k < 16; ++k) {
      float w = float(b[0]);
#pragma unroll
      for (int i = 1; i < 8; ++i) w = (k & 3) + 4 * (k >> 3) == i ? float(b[i]) : w;
      w = __shfl(w, (lane & 31) + 32 * ((k >> 2) & 1), 64);
      const bool see = seen(k);
#pragma unroll 1
      for (int r = 0; r < 16; ++r) {
        const T* at = tile + (row0 + k) * pitch + acc_row(r);
#pragma unroll
        for (int n = 0; n < kCount; ++n) {
          const float v = float(at[32 * n]), t = w * v;
          const uint32_t up = !(t <= 3.4028235e38f), down = !(t >= -3.4028235e38f);
          if (see && !finite(v)) marks[n] |= (up << r) | (down << (16 + r));
        }
      }
    }
  }
  // mark() and the dropping for a single second operand.
  template <typename F>
  __device__ __forceinline__ void guard(const T* tile, int pitch, int row0, Frag<T> (&a)[kCount],
                                        const Frag<T>& b, F&& seen) {
    if (__builtin_expect(!any_not_finite<T>(a), 1)) return;
    mark(tile, pitch, row0, b, seen);
    drop_not_finite<T>(a);
  }
  __device__ __forceinline__ void apply(Acc (&acc)[kCount]) const {
    uint32_t any = 0;
#pragma unroll
    for (int n = 0; n < kCount; ++n) any |= marks[n];
    if (!__any(any != 0)) return;
#pragma unroll
    for (int n = 0; n < kCount; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if (marks[n] >> r & 1) acc[n][r] += INFINITY;
        if (marks[n] >> (16 + r) & 1) acc[n][r] -= INFINITY;
      }
  }
};

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
};

// The tiles of kKeys keys that queries from `query` on, `queries` of them, walk:
// those that hold first tokens, then those of the window.
template <int kKeys>
struct KeyTiles {
  int count, head, tail;
  __device__ __forceinline__ KeyTiles(const Problem& p, int query, int queries, int length) {
    const int first = p.offset() + query;
    const int last = min(p.offset() + min(query + queries, p.queries), length) - 1;
    tail = max(0, first - p.window + 1) / kKeys;
    head = min((min(p.sinks, last + 1) + kKeys - 1) / kKeys, tail);
    count = last < 0 ? 0 : head + max(0, last / kKeys - tail + 1);
    tail -= head;
  }
  __device__ __forceinline__ int first_key(int it) const {
    return (it < head ? it : tail + it) * kKeys;
  }
};

// Fewer workgroups of 128 queries than this, and 32 queries a workgroup with the
// keys shared out over its waves take over.  Forward, 128 a workgroup against 32,
// us: heads of 64, 80 workgroups 19 and 15, 256 between 20 and 21 and 42 and 37,
// 512 24 and 31; heads of 128, 64 workgroups 34 and 23, 128 between 27 and 29 and
// 60 and 52, 256 43 and 82.
inline int64_t split_below(int dim) { return dim <= 64 ? 256 : 160; }

// What a wave's lanes wrote to LDS of their own is there for all of them: LDS
// serves a wave in order, so only the compiler has to be held.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Which of the keys base + k a query at position p sees: comparisons of k,
// known at compile time, with a few registers.
struct KeySight {
  int top, low, sinks;
  __device__ __forceinline__ KeySight(const Problem& p, int pos, int base, int length)
      : top(min(pos, length - 1) - base), low(pos - p.window - base), sinks(p.sinks - base) {}
  __device__ __forceinline__ bool sees(int k) const {
    return bool(int(k <= top) & (int(k > low) | int(k < sinks)));
  }
};

// Which of the queries base + k, of those in [from, to), see key j.
struct QuerySight {
  int low, end;
  __device__ __forceinline__ QuerySight(const Problem& p, int j, int base, int from, int to,
                                        int length) {
    const int at = p.offset() + base;  // position of k = 0
    low = max(j - at, from - base);
    end = j >= length ? low : j < p.sinks ? to - base : min(to - base, j - at + p.window);
  }
  __device__ __forceinline__ bool sees(int k) const {
    return bool(int(k >= low) & int(k < end));
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
