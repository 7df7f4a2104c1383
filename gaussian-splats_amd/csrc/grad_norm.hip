// The 2-norm of many tensors together, and their scaling to a limit.
//
//   norm = sqrt(sum of all squares),   factor = min(1, max_norm / (norm + 1e-6))
//
// as torch.nn.utils.clip_grad_norm_ has it.  Bound by the tensors' bytes: read
// once for the norm, read and written once more only where the factor is not one.
//
// A launch takes up to 128 tensors, whose addresses travel in its arguments, cut
// into chunks of 16 KB; a workgroup has a contiguous run of chunks, so it looks
// its first tensor up once.  Squares are added in float64 from the first one on:
// values whose squares float32 does not hold count, and the conversions and
// additions take a quarter of the time that the loads leave them.  Each workgroup
// writes one partial sum; whoever needs the norm adds them in their order, so the
// result does not depend on the schedule.  The scaling's workgroups do that
// themselves (8 KB each from L2, 1.5 us) instead of waiting for a launch that does.
//
// Measured, 55 tensors of 74 M bfloat16 values (147 MB): within the limit 75 us a call,
// most of it the host's walk of the list (kernels 31 us, 4.8 TB/s, and 4); above it, scaled, 108.
// Adam with the limit on 59 M parameters: 360 us a call for 1.9 GB, 5.2 TB/s.
#include "sequence.h"

namespace gs {
namespace {

using namespace seq;

constexpr int kThreads = 256;
constexpr int kUnroll = 4;
constexpr int kChunkBytes = kThreads * 16 * kUnroll;
constexpr int kMostBlocks = 1024;  // of a launch: four workgroups a CU
constexpr int kMostTensors = 128;  // of a launch

struct TensorArg {
  void* data;
  int64_t numel;
  int64_t first;  // chunk
};

struct NormArgs {
  TensorArg t[kMostTensors];
  uint8_t type[kMostTensors];
  uint8_t aligned[kMostTensors];
  int count;
  int64_t chunks, each;  // of the launch, of a workgroup
};

struct ScaleArgs {
  const double* partials;
  int parts;
  double limit;
  float* norm;
  float* factor;
};

__device__ __forceinline__ double square(float v, double sum) {
  const double d = double(v);
  return fma(d, d, sum);
}

// Calls f with the tensor, the first element and the end of each of the
// workgroup's chunks.
template <typename F>
__device__ __forceinline__ void for_chunks(const NormArgs& a, F&& f) {
  int64_t c = int64_t(blockIdx.x) * a.each;
  const int64_t end = min(c + a.each, a.chunks);
  int k = 0;
  for (int step = kMostTensors / 2; step; step >>= 1)
    if (k + step < a.count && a.t[k + step].first <= c) k += step;
  for (; c < end; ++c) {
    while (k + 1 < a.count && a.t[k + 1].first <= c) ++k;
    const int size = a.type[k] == GS_F32 ? 4 : 2;
    const int64_t lo = (c - a.t[k].first) * (kChunkBytes / size);
    f(k, lo, min(lo + kChunkBytes / size, a.t[k].numel));
  }
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* p, int64_t lo, int64_t hi, bool aligned,
                                                double sum) {
  constexpr int kV = 16 / int(sizeof(T));
  const int64_t mine = lo + int64_t(threadIdx.x) * kV;
  if (aligned && hi - lo == kChunkBytes / int(sizeof(T))) {
    Vec<T, kV> v[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      v[i] = *reinterpret_cast<const Vec<T, kV>*>(p + mine + i * kThreads * kV);
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
#pragma unroll
      for (int j = 0; j < kV; ++j) sum = square(float(v[i][j]), sum);
  } else {
    for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads) sum = square(float(p[i]), sum);
  }
  return sum;
}

template <typename T>
__device__ __forceinline__ void chunk_scale(T* p, int64_t lo, int64_t hi, bool aligned, float by) {
  constexpr int kV = 16 / int(sizeof(T));
  const int64_t mine = lo + int64_t(threadIdx.x) * kV;
  if (aligned && hi - lo == kChunkBytes / int(sizeof(T))) {
    Vec<T, kV> v[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      v[i] = *reinterpret_cast<const Vec<T, kV>*>(p + mine + i * kThreads * kV);
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      *reinterpret_cast<Vec<T, kV>*>(p + mine + i * kThreads * kV) =
          from_float<T, kV>(to_float<T, kV>(v[i]) * by);
  } else {
    for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads) p[i] = T(float(p[i]) * by);
  }
}

// The workgroup's sum, in every thread.
__device__ __forceinline__ double block_sum(double v, double (&shared)[kThreads / kWave]) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) v += __shfl_xor(v, d, kWave);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x / kWave] = v;
  __syncthreads();
  return (shared[0] + shared[1]) + (shared[2] + shared[3]);
}

__global__ __launch_bounds__(kThreads) void norm_kernel(NormArgs a, double* partials) {
  __shared__ double shared[kThreads / kWave];
  double sum = 0.0;
  for_chunks(a, [&](int k, int64_t lo, int64_t hi) {
    const void* p = a.t[k].data;
    const bool aligned = a.aligned[k];
    if (a.type[k] == GS_F32)
      sum = chunk_squares(static_cast<const float*>(p), lo, hi, aligned, sum);
    else if (a.type[k] == GS_F16)
      sum = chunk_squares(static_cast<const f16*>(p), lo, hi, aligned, sum);
    else
      sum = chunk_squares(static_cast<const bf16*>(p), lo, hi, aligned, sum);
  });
  sum = block_sum(sum, shared);
  if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

// The norm and its factor from the partial sums; the workgroup that `writes`
// stores them.
__device__ __forceinline__ float factor_of(const ScaleArgs& s, bool writes) {
  __shared__ double shared[kThreads / kWave];
  double sum = 0.0;
  for (int i = threadIdx.x; i < s.parts; i += kThreads) sum += s.partials[i];
  const double norm = sqrt(block_sum(sum, shared));
  const double ratio = s.limit / (norm + 1e-6);
  // A NaN stays one, as clamping leaves it.
  const float factor = ratio > 1.0 ? 1.0f : float(ratio);
  if (writes && threadIdx.x == 0) {
    *s.norm = float(norm);
    if (s.factor) *s.factor = factor;
  }
  return factor;
}

__global__ __launch_bounds__(kThreads) void norm_finish_kernel(ScaleArgs s) { factor_of(s, true); }

__global__ __launch_bounds__(kThreads) void norm_scale_kernel(NormArgs a, ScaleArgs s, bool writes) {
  const float by = factor_of(s, writes && blockIdx.x == 0);
  if (by == 1.0f) return;
  for_chunks(a, [&](int k, int64_t lo, int64_t hi) {
    void* p = a.t[k].data;
    const bool aligned = a.aligned[k];
    if (a.type[k] == GS_F32)
      chunk_scale(static_cast<float*>(p), lo, hi, aligned, by);
    else if (a.type[k] == GS_F16)
      chunk_scale(static_cast<f16*>(p), lo, hi, aligned, by);
    else
      chunk_scale(static_cast<bf16*>(p), lo, hi, aligned, by);
  });
}

// Fills `a` with the tensors from `next` on that fit a launch; returns its workgroups.
int64_t fill_args(const gs_tensor* tensors, int64_t count, int64_t& next, NormArgs& a) {
  a.count = 0;
  a.chunks = 0;
  for (; next < count && a.count < kMostTensors; ++next) {
    const gs_tensor& t = tensors[next];
    if (t.numel == 0) continue;
    const int64_t per = kChunkBytes / type_bytes(int32_t(t.type));
    a.t[a.count] = {t.data, t.numel, a.chunks};
    a.type[a.count] = uint8_t(t.type);
    a.aligned[a.count] = aligned_to(t.data, 16);
    a.chunks += (t.numel + per - 1) / per;
    ++a.count;
  }
  if (a.count == 0) return 0;
  const int64_t blocks = std::min<int64_t>(a.chunks, kMostBlocks);
  a.each = (a.chunks + blocks - 1) / blocks;
  return (a.chunks + a.each - 1) / a.each;
}

int64_t launches(int64_t count) { return (count + kMostTensors - 1) / kMostTensors; }

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" GS_API size_t gs_grad_norm_workspace_bytes(int64_t count) {
  return count <= 0 ? 0 : size_t(launches(count)) * kMostBlocks * sizeof(double);
}

extern "C" GS_API int gs_grad_norm(const gs_tensor* tensors, int64_t count, double max_norm,
                                   int32_t scale, float* norm, float* factor, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  clear_error();
  GS_REQUIRE(count >= 0 && count < (int64_t(1) << 20), GS_ERR_INVALID_ARGUMENT,
             "between 0 and 2^20 - 1 tensors (got %lld)", (long long)count);
  GS_REQUIRE(count == 0 || tensors, GS_ERR_INVALID_ARGUMENT, "null tensor list");
  GS_REQUIRE(norm, GS_ERR_INVALID_ARGUMENT, "null pointer: norm");
  GS_REQUIRE(max_norm >= 0.0, GS_ERR_INVALID_ARGUMENT, "max_norm must be non-negative");
  for (int64_t i = 0; i < count; ++i) {
    const gs_tensor& t = tensors[i];
    GS_REQUIRE(t.numel >= 0 && t.numel < (int64_t(1) << 48), GS_ERR_INVALID_ARGUMENT,
               "tensor %lld: %lld elements", (long long)i, (long long)t.numel);
    GS_REQUIRE(t.numel == 0 || t.data, GS_ERR_INVALID_ARGUMENT, "tensor %lld: null pointer",
               (long long)i);
    GS_REQUIRE(t.type >= 0 && t.type <= GS_BF16, GS_ERR_INVALID_ARGUMENT,
               "tensor %lld: unknown type %lld", (long long)i, (long long)t.type);
  }
  const size_t need = gs_grad_norm_workspace_bytes(count);
  GS_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), GS_ERR_WORKSPACE,
             "workspace too small: %zu bytes, %zu needed", workspace_bytes, need);
  const hipStream_t s = as_stream(stream);
  double* partials = static_cast<double*>(workspace);
  ScaleArgs end{partials, 0, max_norm, norm, factor};
  NormArgs a;
  for (int64_t next = 0; next < count;) {
    const int64_t blocks = fill_args(tensors, count, next, a);
    if (blocks == 0) continue;
    norm_kernel<<<unsigned(blocks), kThreads, 0, s>>>(a, partials + end.parts);
    GS_TRY(check_launch("grad_norm"));
    end.parts += int(blocks);
  }
  if (!scale || end.parts == 0) {
    norm_finish_kernel<<<1, kThreads, 0, s>>>(end);
    return check_launch("grad_norm finish");
  }
  bool writes = true;
  for (int64_t next = 0; next < count;) {
    const int64_t blocks = fill_args(tensors, count, next, a);
    if (blocks == 0) continue;
    norm_scale_kernel<<<unsigned(blocks), kThreads, 0, s>>>(a, end, writes);
    GS_TRY(check_launch("grad_norm scale"));
    writes = false;
  }
  return GS_OK;
}
