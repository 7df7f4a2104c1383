// Shared pieces of the sequence operators (norm, scan, attention): the element
// types gs_raster.h names, their vectors, and conversions to and from float.
#pragma once

#include "common.h"

namespace gs {
namespace seq {

using bf16 = __bf16;
using f16 = _Float16;

template <typename T, int N>
using Vec = T __attribute__((ext_vector_type(N)));

template <int N>
using FloatVec = Vec<float, N>;

template <typename T>
struct TypeId;
template <>
struct TypeId<float> {
  static constexpr int value = GS_F32;
};
template <>
struct TypeId<f16> {
  static constexpr int value = GS_F16;
};
template <>
struct TypeId<bf16> {
  static constexpr int value = GS_BF16;
};

inline bool float_type(int32_t t) { return t == GS_F32 || t == GS_F16 || t == GS_BF16; }
inline int type_bytes(int32_t t) { return t == GS_F32 ? 4 : 2; }

// Calls f with a value of the C++ type that `type` names.
template <typename F>
int with_type(int32_t type, F&& f) {
  switch (type) {
    case GS_F32:
      return f(float{});
    case GS_F16:
      return f(f16{});
    default:
      return f(bf16{});
  }
}

template <typename T, int N>
__device__ __forceinline__ FloatVec<N> to_float(const Vec<T, N>& v) {
  return __builtin_convertvector(v, FloatVec<N>);
}

// Round to nearest even.
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> from_float(const FloatVec<N>& v) {
  return __builtin_convertvector(v, Vec<T, N>);
}

// One element of a type known at run time (a uniform branch).
__device__ __forceinline__ float load_as_float(const void* p, int64_t i, int type) {
  if (type == GS_F32) return static_cast<const float*>(p)[i];
  if (type == GS_F16) return float(static_cast<const f16*>(p)[i]);
  return float(static_cast<const bf16*>(p)[i]);
}
__device__ __forceinline__ void store_from_float(void* p, int64_t i, int type, float v) {
  if (type == GS_F32)
    static_cast<float*>(p)[i] = v;
  else if (type == GS_F16)
    static_cast<f16*>(p)[i] = f16(v);
  else
    static_cast<bf16*>(p)[i] = bf16(v);
}

// The larger one; NaN if either is NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  return a != a ? a : (b != b ? b : fmaxf(a, b));
}

// `blocks` workgroups of up to 1024 threads.  One dimension holds less than 2^32
// threads: beyond, a launch is refused or, worse, does the remainder alone.  So
// many workgroups go over two dimensions, and block_index() counts them; up to a
// few more than `blocks` are launched.
inline dim3 grid_of(int64_t blocks) {
  constexpr int64_t kMost = 1 << 21;
  if (blocks <= kMost) return dim3(unsigned(blocks));
  const int64_t y = (blocks + kMost - 1) / kMost;
  return dim3(unsigned((blocks + y - 1) / y), unsigned(y));
}
__device__ __forceinline__ int64_t block_index() {
  return int64_t(blockIdx.y) * gridDim.x + blockIdx.x;
}

inline bool aligned_to(const void* p, size_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

}  // namespace seq
}  // namespace gs
