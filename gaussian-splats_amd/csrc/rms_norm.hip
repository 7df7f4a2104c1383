// Root-mean-square norm with the residual's addition:
//   s = x + residual,  r = 1 / sqrt(mean(s^2) + eps),  y = s r w
// over the rows of [rows, width], in float32 whatever the types; y is rounded
// once to x's type and s once to the residual's, and y is computed from the s
// that has not been rounded.  The 8-bit form writes y / scale with one scale
// per row, max|y| / 127 or / 448.
//
// Backward, with t = grad_y w and the rounded s of the forward:
//   grad_s = r (t - s r mean(t s r)) + grad_sum,   grad_w = sum_rows grad_y s r.
// Each workgroup adds grad_w of its rows in registers and writes one partial
// row; a second kernel adds the partial rows in a fixed order, so the result
// does not depend on the schedule.
//
// Bound by memory: every element is read once and written once, a row stays in
// registers between its reduction and its use.  A wave holds a row of up to
// 1024 elements, a workgroup one of up to 8192; longer rows are read twice.
// Measured, 40000 x 768, bfloat16 beside a float32 residual: forward 64 us for 368
// MB (5.8 TB/s, where a large copy moves 5.2), backward 96 us for 491 MB (5.1) and 4
// for the weight's sum; 32 rows of 4096 as int8: 8.1 us, one chain of loads, two
// reductions and divisions.
#include "sequence.h"

namespace gs {
namespace {

using namespace seq;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
// Partial rows of grad_w, and the most workgroups of the backward, two for each
// CU.  Backward with 256, 512 and 1024, us, bfloat16 beside float32: 40000 x 768 121,
// 95 and 100; 20000 x 2048 172, 121 and 130; 5000 x 8192 141, 130 and 136.
constexpr int kMaxPartials = 512;

enum class Out { kValues, kInt8, kE4M3 };

// How a row is spread over threads: kVecs vectors of 8 elements for each of
// kRowThreads threads.  kAligned: 16-byte accesses to 8 neighbouring elements;
// otherwise single elements, neighbours in neighbouring threads.
template <int kRowThreads, int kVecs, bool kAligned>
struct Row {
  static constexpr int kThreadsPerRow = kRowThreads;
  static constexpr int kCount = kVecs;
  static constexpr bool kVector = kAligned;
  static constexpr int kRows = kThreads / kRowThreads;  // rows of a workgroup
  __device__ static int column(int v, int u, int t) {
    return kAligned ? (v * kRowThreads + t) * 8 + u : (v * 8 + u) * kRowThreads + t;
  }
};

template <typename R, typename T>
__device__ __forceinline__ void load_row(const T* p, int width, int t, FloatVec<8> (&out)[R::kCount]) {
#pragma unroll
  for (int v = 0; v < R::kCount; ++v) {
    if constexpr (R::kVector) {
      const int c = R::column(v, 0, t);
      if (c < width)
        out[v] = to_float<T, 8>(*reinterpret_cast<const Vec<T, 8>*>(p + c));
      else
        out[v] = FloatVec<8>(0.0f);
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int c = R::column(v, u, t);
        out[v][u] = c < width ? float(p[c]) : 0.0f;
      }
    }
  }
}

template <typename R, typename T>
__device__ __forceinline__ void store_row(T* p, int width, int t, const FloatVec<8> (&in)[R::kCount]) {
#pragma unroll
  for (int v = 0; v < R::kCount; ++v) {
    if constexpr (R::kVector) {
      const int c = R::column(v, 0, t);
      if (c < width) *reinterpret_cast<Vec<T, 8>*>(p + c) = from_float<T, 8>(in[v]);
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int c = R::column(v, u, t);
        if (c < width) p[c] = T(in[v][u]);
      }
    }
  }
}

template <typename R>
__device__ __forceinline__ void load_weight(const void* w, int type, int width, int t,
                                            FloatVec<8> (&out)[R::kCount]) {
  if (type == GS_F32)
    load_row<R>(static_cast<const float*>(w), width, t, out);
  else if (type == GS_F16)
    load_row<R>(static_cast<const f16*>(w), width, t, out);
  else
    load_row<R>(static_cast<const bf16*>(w), width, t, out);
}

// Reduction over the threads of a row; every thread gets the result.
// `scratch` is used by rows wider than a wave, one slot per wave and call.
template <int kRowThreads, typename F>
__device__ __forceinline__ float row_reduce(float v, float* scratch, F&& op) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
  if constexpr (kRowThreads > kWave) {
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    v = scratch[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) v = op(v, scratch[i]);
  }
  return v;
}

__device__ __forceinline__ float add(float a, float b) { return a + b; }

__device__ __forceinline__ int8_t to_int8(float v) {
  return v == v ? int8_t(fminf(fmaxf(rintf(v), -127.0f), 127.0f)) : int8_t(0);
}

// Four values as e4m3 bytes (the conversion rounds to nearest even).
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}
__device__ __forceinline__ float clamp_e4m3(float v) {
  return v == v ? fminf(fmaxf(v, -448.0f), 448.0f) : v;
}

struct NormArgs {
  const void* x;
  const void* residual;  // null: s = x, which is not written
  const void* weight;
  int64_t rows;
  int width;
  int64_t x_stride;
  int64_t residual_stride;
  int weight_type;
  float eps;
  void* y;  // values or codes
  float* scales;
  void* sum;
  float* inverse;  // r of each row, or null
  Out out;
};

template <typename R>
__device__ __forceinline__ void store_codes(const NormArgs& a, int64_t row, int t,
                                            const FloatVec<8> (&y)[R::kCount], float scale) {
  uint8_t* p = static_cast<uint8_t*>(a.y) + row * a.width;
  const float safe = scale > 0.0f ? scale : 1.0f;
  const bool int8 = a.out == Out::kInt8;
#pragma unroll
  for (int v = 0; v < R::kCount; ++v) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float q[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) q[u] = y[v][i * 4 + u] / safe;
      if (int8) {
        w[i] = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) w[i] |= uint32_t(uint8_t(to_int8(q[u]))) << (8 * u);
      } else {
        w[i] = to_e4m3(clamp_e4m3(q[0]), clamp_e4m3(q[1]), clamp_e4m3(q[2]), clamp_e4m3(q[3]));
      }
    }
    if constexpr (R::kVector) {
      const int c = R::column(v, 0, t);
      if (c < a.width) *reinterpret_cast<uint2*>(p + c) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int c = R::column(v, u, t);
        if (c < a.width) p[c] = uint8_t(w[u >> 2] >> (8 * (u & 3)));
      }
    }
  }
}

template <typename TX, typename TR, typename R>
__global__ __launch_bounds__(kThreads) void norm_kernel(NormArgs a) {
  __shared__ float scratch[2][kWaves];
  const int t = threadIdx.x % R::kThreadsPerRow;
  const int64_t row = block_index() * R::kRows + threadIdx.x / R::kThreadsPerRow;
  if (row >= a.rows) return;  // whole waves; workgroups of one row have no such row
  FloatVec<8> s[R::kCount], w[R::kCount];
  load_row<R>(static_cast<const TX*>(a.x) + row * a.x_stride, a.width, t, s);
  if (a.residual) {
    FloatVec<8> res[R::kCount];
    load_row<R>(static_cast<const TR*>(a.residual) + row * a.residual_stride, a.width, t, res);
#pragma unroll
    for (int v = 0; v < R::kCount; ++v) s[v] += res[v];
    store_row<R>(static_cast<TR*>(a.sum) + row * a.width, a.width, t, s);
  }
  load_weight<R>(a.weight, a.weight_type, a.width, t, w);
  float sq = 0.0f;
#pragma unroll
  for (int v = 0; v < R::kCount; ++v)
#pragma unroll
    for (int u = 0; u < 8; ++u) sq += s[v][u] * s[v][u];
  sq = row_reduce<R::kThreadsPerRow>(sq, scratch[0], add);
  const float r = 1.0f / sqrtf(sq / float(a.width) + a.eps);
  if (a.inverse && t == 0) a.inverse[row] = r;
#pragma unroll
  for (int v = 0; v < R::kCount; ++v) s[v] = s[v] * r * w[v];
  if (a.out == Out::kValues) {
    store_row<R>(static_cast<TX*>(a.y) + row * a.width, a.width, t, s);
    return;
  }
  float top = 0.0f;
#pragma unroll
  for (int v = 0; v < R::kCount; ++v)
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (R::column(v, u, t) < a.width) top = max_nan(top, fabsf(s[v][u]));
  top = row_reduce<R::kThreadsPerRow>(top, scratch[1], max_nan);
  const float scale = top / (a.out == Out::kInt8 ? 127.0f : 448.0f);
  if (t == 0) a.scales[row] = scale;
  store_codes<R>(a, row, t, s, scale);
}

// Rows of any width, read twice (three times for 8-bit output): one workgroup a row.
template <typename TX, typename TR>
__global__ __launch_bounds__(kThreads) void norm_long_kernel(NormArgs a) {
  __shared__ float scratch[2][kWaves];
  const int64_t row = block_index();
  if (row >= a.rows) return;
  const TX* x = static_cast<const TX*>(a.x) + row * a.x_stride;
  const TR* res = static_cast<const TR*>(a.residual);
  if (res) res += row * a.residual_stride;
  TR* sum = static_cast<TR*>(a.sum) + row * a.width;
  const auto value = [&](int c) { return res ? float(x[c]) + float(res[c]) : float(x[c]); };
  float sq = 0.0f;
  for (int c = threadIdx.x; c < a.width; c += kThreads) {
    const float s = value(c);
    sq += s * s;
    if (res) sum[c] = TR(s);
  }
  sq = row_reduce<kThreads>(sq, scratch[0], add);
  const float r = 1.0f / sqrtf(sq / float(a.width) + a.eps);
  if (a.inverse && threadIdx.x == 0) a.inverse[row] = r;
  const auto normed = [&](int c) { return value(c) * r * load_as_float(a.weight, c, a.weight_type); };
  if (a.out == Out::kValues) {
    TX* y = static_cast<TX*>(a.y) + row * a.width;
    for (int c = threadIdx.x; c < a.width; c += kThreads) y[c] = TX(normed(c));
    return;
  }
  float top = 0.0f;
  for (int c = threadIdx.x; c < a.width; c += kThreads) top = max_nan(top, fabsf(normed(c)));
  top = row_reduce<kThreads>(top, scratch[1], max_nan);
  const float scale = top / (a.out == Out::kInt8 ? 127.0f : 448.0f);
  const float safe = scale > 0.0f ? scale : 1.0f;
  if (threadIdx.x == 0) a.scales[row] = scale;
  uint8_t* p = static_cast<uint8_t*>(a.y) + row * a.width;
  for (int c = threadIdx.x; c < a.width; c += kThreads) {
    const float q = normed(c) / safe;
    p[c] = a.out == Out::kInt8 ? uint8_t(to_int8(q))
                               : uint8_t(to_e4m3(clamp_e4m3(q), 0.0f, 0.0f, 0.0f));
  }
}

struct NormBwdArgs {
  const void* sum;
  const void* weight;
  const float* inverse;
  const void* grad_y;    // null: zeros
  const void* grad_sum;  // null: zeros
  int64_t rows;
  int width;
  int64_t sum_stride;
  int weight_type;
  void* grad_x;         // null: not wanted
  void* grad_residual;  // null: not wanted, or the same tensor as grad_x
  float* partials;      // [gridDim.x, width], or null
};

template <typename TX, typename TR, typename R>
__global__ __launch_bounds__(kThreads) void norm_bwd_kernel(NormBwdArgs a) {
  __shared__ float scratch[2][kWaves];
  __shared__ float joined[R::kRows > 1 ? R::kCount * 8 * kWave : 1];
  const int t = threadIdx.x % R::kThreadsPerRow;
  const int group = threadIdx.x / R::kThreadsPerRow;
  FloatVec<8> w[R::kCount], dw[R::kCount];
  load_weight<R>(a.weight, a.weight_type, a.width, t, w);
#pragma unroll
  for (int v = 0; v < R::kCount; ++v) dw[v] = FloatVec<8>(0.0f);
  int turn = 0;
  for (int64_t row = int64_t(blockIdx.x) * R::kRows + group; row < a.rows;
       row += int64_t(gridDim.x) * R::kRows, turn ^= 1) {
    FloatVec<8> s[R::kCount], dy[R::kCount], ds[R::kCount];
    load_row<R>(static_cast<const TR*>(a.sum) + row * a.sum_stride, a.width, t, s);
    if (a.grad_y) {
      load_row<R>(static_cast<const TX*>(a.grad_y) + row * a.width, a.width, t, dy);
    } else {
#pragma unroll
      for (int v = 0; v < R::kCount; ++v) dy[v] = FloatVec<8>(0.0f);
    }
    if (a.grad_sum) {
      load_row<R>(static_cast<const TR*>(a.grad_sum) + row * a.width, a.width, t, ds);
    } else {
#pragma unroll
      for (int v = 0; v < R::kCount; ++v) ds[v] = FloatVec<8>(0.0f);
    }
    const float r = a.inverse[row];
    float dot = 0.0f;
#pragma unroll
    for (int v = 0; v < R::kCount; ++v) {
      s[v] = s[v] * r;
      dw[v] += dy[v] * s[v];
      dy[v] = dy[v] * w[v];
#pragma unroll
      for (int u = 0; u < 8; ++u) dot += dy[v][u] * s[v][u];
    }
    // Two turns' slots alternate, so one barrier a row is enough.
    const float c = row_reduce<R::kThreadsPerRow>(dot, scratch[turn], add) / float(a.width);
#pragma unroll
    for (int v = 0; v < R::kCount; ++v) ds[v] += r * (dy[v] - s[v] * c);
    if (a.grad_x) store_row<R>(static_cast<TX*>(a.grad_x) + row * a.width, a.width, t, ds);
    if (a.grad_residual)
      store_row<R>(static_cast<TR*>(a.grad_residual) + row * a.width, a.width, t, ds);
  }
  if (!a.partials) return;
  float* p = a.partials + int64_t(blockIdx.x) * a.width;
  if constexpr (R::kRows > 1) {
    // The waves' sums one after the other.
    for (int g = 0; g < R::kRows; ++g) {
      if (group == g) {
#pragma unroll
        for (int v = 0; v < R::kCount; ++v)
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            float& j = joined[(v * 8 + u) * kWave + t];
            j = g ? j + dw[v][u] : dw[v][u];
            dw[v][u] = j;
          }
      }
      __syncthreads();
    }
    if (group != R::kRows - 1) return;
  }
  store_row<R>(p, a.width, t, dw);
}

template <typename TX, typename TR>
__global__ __launch_bounds__(kThreads) void norm_bwd_long_kernel(NormBwdArgs a) {
  __shared__ float scratch[2][kWaves];
  int turn = 0;
  float* p = a.partials ? a.partials + int64_t(blockIdx.x) * a.width : nullptr;
  if (p)
    for (int c = threadIdx.x; c < a.width; c += kThreads) p[c] = 0.0f;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const TR* s = static_cast<const TR*>(a.sum) + row * a.sum_stride;
    const TX* dy = static_cast<const TX*>(a.grad_y);
    const TR* dsum = static_cast<const TR*>(a.grad_sum);
    if (dy) dy += row * a.width;
    if (dsum) dsum += row * a.width;
    const float r = a.inverse[row];
    float dot = 0.0f;
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
      const float unit = float(s[c]) * r, g = dy ? float(dy[c]) : 0.0f;
      dot += g * load_as_float(a.weight, c, a.weight_type) * unit;
      if (p) p[c] += g * unit;  // this thread's own columns
    }
    const float m = row_reduce<kThreads>(dot, scratch[turn], add) / float(a.width);
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
      const float unit = float(s[c]) * r;
      const float g = dy ? float(dy[c]) * load_as_float(a.weight, c, a.weight_type) : 0.0f;
      const float ds = r * (g - unit * m) + (dsum ? float(dsum[c]) : 0.0f);
      if (a.grad_x) static_cast<TX*>(a.grad_x)[row * a.width + c] = TX(ds);
      if (a.grad_residual) static_cast<TR*>(a.grad_residual)[row * a.width + c] = TR(ds);
    }
  }
}

// grad_w from the partial rows: a workgroup adds 64 columns, its sixteen waves
// every sixteenth row each.
constexpr int kSumWaves = 16;
__global__ __launch_bounds__(kSumWaves* kWave) void norm_weight_kernel(
    const float* __restrict__ partials, int count, int width, void* grad_w, int type) {
  __shared__ float parts[kSumWaves][kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = block_index() * kWave + lane;
  float sum = 0.0f;
  if (c < width) {
#pragma unroll 8
    for (int i = wave; i < count; i += kSumWaves) sum += partials[int64_t(i) * width + c];
  }
  parts[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && c < width) {
#pragma unroll
    for (int i = 1; i < kSumWaves; ++i) sum += parts[i][lane];
    store_from_float(grad_w, c, type, sum);
  }
}

// Calls f with the row layout for a width; `long_f` where none holds the row.
// Both sides of each border, us forward and backward, bfloat16 beside float32:
// 40000 x 768, a row to a wave 67 and 95, to a workgroup 81 and 161 (x 1024: 90 and
// 123, 91 and 166); 20000 x 2048, a vector to a thread 87 and 121, four 98 and 127;
// 5000 x 8192, rows in registers 96 and 130, read twice 225 and 784.
template <typename F, typename G>
void with_row(int width, bool vec, F&& f, G&& long_f) {
  if (width <= 1024)
    vec ? f(Row<64, 2, true>{}) : f(Row<64, 2, false>{});
  else if (width <= 2048)
    vec ? f(Row<256, 1, true>{}) : f(Row<256, 1, false>{});
  else if (width <= 8192)
    vec ? f(Row<256, 4, true>{}) : f(Row<256, 4, false>{});
  else
    long_f();
}

int partial_rows(int64_t rows, int width) {
  const int per_block = width <= 1024 ? kThreads / kWave : 1;
  return int(std::min<int64_t>(kMaxPartials, (rows + per_block - 1) / per_block));
}

// Calls f(x type, residual type) for the pairs that are supported: the same
// type, or float32 beside a 16-bit x.
template <typename F>
int with_types(int32_t x_type, int32_t r_type, F&& f) {
  return with_type(x_type, [&](auto x) {
    using TX = decltype(x);
    if (r_type == GS_F32) return f(TX{}, float{});
    return f(TX{}, TX{});
  });
}

int check_norm(int64_t rows, int64_t width, int32_t x_type, int32_t r_type, int32_t w_type) {
  GS_REQUIRE(rows >= 0 && width > 0, GS_ERR_INVALID_ARGUMENT,
             "rows must be non-negative and width positive, got %lld x %lld", (long long)rows,
             (long long)width);
  GS_REQUIRE(rows < (int64_t(1) << 31) && width < (int64_t(1) << 30), GS_ERR_OVERFLOW,
             "too many rows or columns (%lld x %lld)", (long long)rows, (long long)width);
  GS_REQUIRE(seq::float_type(x_type) && seq::float_type(r_type) && seq::float_type(w_type),
             GS_ERR_INVALID_ARGUMENT, "types must be GS_F32, GS_F16 or GS_BF16");
  GS_REQUIRE(r_type == x_type || r_type == GS_F32, GS_ERR_UNSUPPORTED,
             "the residual must have x's type or float32");
  GS_REQUIRE(w_type == x_type || w_type == GS_F32, GS_ERR_UNSUPPORTED,
             "the weight must have x's type or float32");
  return GS_OK;
}

// Whether rows `stride` apart allow accesses to eight elements at once.
bool fits(const void* p, int32_t type, int64_t stride) {
  const size_t bytes = 8 * size_t(type_bytes(type));
  return !p || (aligned_to(p, bytes) && (stride * type_bytes(type)) % int64_t(bytes) == 0);
}

int run_norm(NormArgs a, int32_t x_type, int32_t r_type, void* stream) {
  if (a.rows == 0) return GS_OK;
  const bool vec = a.width % 8 == 0 && fits(a.x, x_type, a.x_stride) &&
                   fits(a.residual, r_type, a.residual_stride) && fits(a.sum, r_type, 8) &&
                   fits(a.weight, a.weight_type, 8) && fits(a.y, x_type, 8);
  return with_types(x_type, r_type, [&](auto x, auto r) {
    using TX = decltype(x);
    using TR = decltype(r);
    with_row(
        a.width, vec,
        [&](auto row) {
          using R = decltype(row);
          const dim3 blocks = grid_of((a.rows + R::kRows - 1) / R::kRows);
          norm_kernel<TX, TR, R><<<blocks, kThreads, 0, as_stream(stream)>>>(a);
        },
        [&] {
          norm_long_kernel<TX, TR><<<grid_of(a.rows), kThreads, 0, as_stream(stream)>>>(a);
        });
    return check_launch("add_rms_norm");
  });
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" GS_API int gs_add_rms_norm_fwd(const void* x, const void* residual, const void* weight,
                                          int64_t rows, int64_t width, int64_t x_stride,
                                          int64_t residual_stride, int32_t x_type,
                                          int32_t residual_type, int32_t weight_type, float eps,
                                          void* y, void* sum, float* inverse_rms, void* stream) {
  clear_error();
  GS_TRY(check_norm(rows, width, x_type, residual_type, weight_type));
  GS_REQUIRE(rows == 0 || (x && weight && y && (!residual || sum)), GS_ERR_INVALID_ARGUMENT,
             "null pointer");
  return run_norm({x, residual, weight, rows, int(width), x_stride, residual_stride, weight_type,
                   eps, y, nullptr, residual ? sum : nullptr, inverse_rms, Out::kValues},
                  x_type, residual_type, stream);
}

extern "C" GS_API int gs_add_rms_norm_quant(const void* x, const void* residual, const void* weight,
                                            int64_t rows, int64_t width, int64_t x_stride,
                                            int64_t residual_stride, int32_t x_type,
                                            int32_t residual_type, int32_t weight_type, float eps,
                                            int32_t code_type, void* codes, float* scales,
                                            void* sum, void* stream) {
  clear_error();
  GS_TRY(check_norm(rows, width, x_type, residual_type, weight_type));
  GS_REQUIRE(code_type == GS_I8 || code_type == GS_E4M3, GS_ERR_INVALID_ARGUMENT,
             "codes must be GS_I8 or GS_E4M3");
  GS_REQUIRE(rows == 0 || (x && weight && codes && scales && (!residual || sum)),
             GS_ERR_INVALID_ARGUMENT, "null pointer");
  return run_norm({x, residual, weight, rows, int(width), x_stride, residual_stride, weight_type,
                   eps, codes, scales, residual ? sum : nullptr, nullptr,
                   code_type == GS_I8 ? Out::kInt8 : Out::kE4M3},
                  x_type, residual_type, stream);
}

extern "C" GS_API size_t gs_add_rms_norm_bwd_workspace_bytes(int64_t rows, int64_t width) {
  if (rows <= 0 || width <= 0 || rows >= (int64_t(1) << 31) || width >= (int64_t(1) << 30)) return 0;
  return size_t(partial_rows(rows, int(width))) * size_t(width) * sizeof(float);
}

extern "C" GS_API int gs_add_rms_norm_bwd(const void* sum, const void* weight,
                                          const float* inverse_rms, const void* grad_y,
                                          const void* grad_sum, int64_t rows, int64_t width,
                                          int64_t sum_stride, int32_t x_type,
                                          int32_t residual_type, int32_t weight_type, void* grad_x,
                                          void* grad_residual, void* grad_weight, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  clear_error();
  GS_TRY(check_norm(rows, width, x_type, residual_type, weight_type));
  GS_REQUIRE(rows == 0 || (sum && weight && inverse_rms), GS_ERR_INVALID_ARGUMENT, "null pointer");
  GS_REQUIRE(!grad_weight || workspace_bytes >= gs_add_rms_norm_bwd_workspace_bytes(rows, width),
             GS_ERR_WORKSPACE, "workspace too small: %zu bytes", workspace_bytes);
  GS_REQUIRE(!grad_weight || rows == 0 || workspace, GS_ERR_INVALID_ARGUMENT, "null workspace");
  NormBwdArgs a{sum,  weight,        inverse_rms, grad_y,     grad_sum,
                rows, int(width),    sum_stride,  weight_type, grad_x,
                grad_residual, grad_weight ? static_cast<float*>(workspace) : nullptr};
  const int blocks = rows ? partial_rows(rows, int(width)) : 0;
  if (rows) {
    const bool vec = width % 8 == 0 && fits(sum, residual_type, sum_stride) &&
                     fits(weight, weight_type, 8) && fits(grad_y, x_type, 8) &&
                     fits(grad_sum, residual_type, 8) && fits(grad_x, x_type, 8) &&
                     fits(grad_residual, residual_type, 8) && fits(workspace, GS_F32, 8);
    GS_TRY(with_types(x_type, residual_type, [&](auto x, auto r) {
      using TX = decltype(x);
      using TR = decltype(r);
      with_row(
          a.width, vec,
          [&](auto row) {
            norm_bwd_kernel<TX, TR, decltype(row)>
                <<<unsigned(blocks), kThreads, 0, as_stream(stream)>>>(a);
          },
          [&] {
            norm_bwd_long_kernel<TX, TR>
                <<<unsigned(blocks), kThreads, 0, as_stream(stream)>>>(a);
          });
      return check_launch("add_rms_norm backward");
    }));
  }
  if (grad_weight) {
    norm_weight_kernel<<<grid_of((width + kWave - 1) / kWave), kSumWaves * kWave, 0,
                         as_stream(stream)>>>(a.partials, blocks, a.width, grad_weight, weight_type);
    return check_launch("add_rms_norm weight gradient");
  }
  return GS_OK;
}
