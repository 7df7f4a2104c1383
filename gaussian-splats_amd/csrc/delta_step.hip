// One token of the gated delta rule (delta_scan.h) for each head of several streams.
//
// Bound by the states, read and written once.  Columns of a state do not mix: a
// workgroup takes 32 of them, its threads four columns and every 32nd row, so the
// state stays in registers between the one sum over its rows and its update.  That
// sum gives S^T k and S^T q at once; the new state's product with q follows from
// o = scale (a S^T q + (k . q) u).
//
// Measured, 32 streams of 32 heads of 128 x 128, bfloat16: 27.8 us a
// call, 135 MB at 4.9 TB/s.
#include "delta_scan.h"

namespace gs {

int check_delta(const gs_delta& d);

namespace delta {
namespace {

constexpr int kWide = 32;   // columns of a workgroup
constexpr int kLanes = kWide / 4;
constexpr int kRowStep = kThreads / kLanes;

template <typename T>
struct StepArgs {
  Problem p;
  const T* q;
  const T* k;
  const T* v;
  const T* gate;
  const T* beta;
  const float* state;
  float* state_out;
  T* out;
};

template <typename T, int kKey>
__global__ __launch_bounds__(kThreads) void delta_step_kernel(StepArgs<T> a) {
  constexpr int kRows = kKey / kRowStep, kWaves = kThreads / kWave;
  __shared__ FloatVec<4> sums[kWaves][2][kLanes];
  __shared__ float products[kWaves];
  const int blocks = (a.p.dim + kWide - 1) / kWide;
  const int64_t index = seq::block_index(), head = index / blocks;
  if (head >= int64_t(a.p.batch) * a.p.heads) return;
  const int b = int(head / a.p.heads), h = int(head % a.p.heads);
  const int64_t key = int64_t(b) * a.p.key_heads + int64_t(h) * a.p.key_heads / a.p.heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int place = threadIdx.x % kLanes, first = threadIdx.x / kLanes;
  const int col = int(index % blocks) * kWide + 4 * place;
  const bool live = col < a.p.dim;
  const int64_t at = head * a.p.key_dim * a.p.dim + col;
  FloatVec<4> s[kRows], reads(0.0f), answers(0.0f);
  float k[kRows], q[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int row = first + i * kRowStep;
    const bool in = row < a.p.key_dim;
    s[i] = in && live ? *reinterpret_cast<const FloatVec<4>*>(a.state + at + int64_t(row) * a.p.dim)
                      : FloatVec<4>(0.0f);
    k[i] = in ? float(a.k[key * a.p.key_dim + row]) : 0.0f;
    q[i] = in ? float(a.q[key * a.p.key_dim + row]) : 0.0f;
  }
  float product = 0.0f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    reads += s[i] * k[i];
    answers += s[i] * q[i];
    product += k[i] * q[i];
  }
#pragma unroll
  for (int d = kLanes; d < kWave; d <<= 1) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      reads[c] += __shfl_xor(reads[c], d, kWave);
      answers[c] += __shfl_xor(answers[c], d, kWave);
    }
    product += __shfl_xor(product, d, kWave);
  }
  if (lane < kLanes) {
    sums[wave][0][lane] = reads;
    sums[wave][1][lane] = answers;
    if (lane == 0) products[wave] = product;
  }
  __syncthreads();
  reads = (sums[0][0][place] + sums[1][0][place]) + (sums[2][0][place] + sums[3][0][place]);
  answers = (sums[0][1][place] + sums[1][1][place]) + (sums[2][1][place] + sums[3][1][place]);
  product = (products[0] + products[1]) + (products[2] + products[3]);
  if (!live) return;
  const float keep = sigmoid(float(a.gate[head])), write = sigmoid(float(a.beta[head]));
  const FloatVec<4> v = to_float<T, 4>(*reinterpret_cast<const Vec<T, 4>*>(a.v + head * a.p.dim + col));
  const FloatVec<4> u = write * (v - keep * reads);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int row = first + i * kRowStep;
    if (row < a.p.key_dim)
      *reinterpret_cast<FloatVec<4>*>(a.state_out + at + int64_t(row) * a.p.dim) = keep * s[i] + k[i] * u;
  }
  if (first == 0)
    *reinterpret_cast<Vec<T, 4>*>(a.out + head * a.p.dim + col) =
        from_float<T, 4>(a.p.scale * (keep * answers + product * u));
}

}  // namespace
}  // namespace delta
}  // namespace gs

using namespace gs;

extern "C" GS_API int gs_delta_scan_step(const gs_delta* desc, const void* q, const void* k,
                                         const void* v, const void* gate, const void* beta,
                                         const float* state, void* out, float* state_out,
                                         void* stream) {
  clear_error();
  GS_REQUIRE(desc, GS_ERR_INVALID_ARGUMENT, "null description");
  GS_TRY(check_delta(*desc));
  if (desc->batch == 0) return GS_OK;
  const void* const all[] = {q, k, v, gate, beta, state, out, state_out};
  for (const void* p : all) GS_REQUIRE(p, GS_ERR_INVALID_ARGUMENT, "null pointer");
  for (const void* p : {v, static_cast<const void*>(state), static_cast<const void*>(state_out),
                        static_cast<const void*>(out)})
    GS_REQUIRE(seq::aligned_to(p, 16), GS_ERR_INVALID_ARGUMENT,
               "v, out and the states must start on a 16-byte boundary");
  const int64_t blocks = desc->batch * desc->heads * ((desc->dim + delta::kWide - 1) / delta::kWide);
  return seq::with_type(desc->type, [&](auto t) {
    using T = decltype(t);
    delta::StepArgs<T> a{{int(desc->batch), 1, desc->heads, desc->key_heads, desc->key_dim, desc->dim, 1,
                          desc->scale, nullptr},
                         static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v),
                         static_cast<const T*>(gate), static_cast<const T*>(beta), state, state_out,
                         static_cast<T*>(out)};
    const hipStream_t s = as_stream(stream);
    const dim3 grid = seq::grid_of(blocks);
    if (a.p.key_dim <= 32)
      delta::delta_step_kernel<T, 32><<<grid, delta::kThreads, 0, s>>>(a);
    else if (a.p.key_dim <= 64)
      delta::delta_step_kernel<T, 64><<<grid, delta::kThreads, 0, s>>>(a);
    else
      delta::delta_step_kernel<T, 128><<<grid, delta::kThreads, 0, s>>>(a);
    return check_launch("delta_scan_step");
  });
}
