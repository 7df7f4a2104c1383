// One token of each of several streams: attention over a cache of the first
// tokens and a ring of the last `window` ones.  Every filled slot is seen, so a
// stream's keys are the first min(p + 1, sinks + window) slots, in any order.
//
// Bound by the cache's bytes, which are read once.  A workgroup takes a share of
// one stream's slots for one key head and the (up to 32) query heads that read
// it, its four waves tiles of 32 keys in turn, each with a running maximum and
// sum; the waves join in LDS, and where the slots are shared out over several
// workgroups a second kernel joins those, both in a fixed order.  The new token's
// key and value come from the call's own inputs, not from the cache: the one
// workgroup whose share holds their slot writes them there, and no other reads it.
// Probabilities are rounded to the inputs' type for the product with the values,
// an operand of the matrix cores, and for the sum alike, so that weights add up
// to one.
//
// Measured, bfloat16, 32 streams of up to 8176 slots, 32 heads of 128 on 8: 189 us
// for 975 MB, 5.1 TB/s, where a large copy moves 5.2; the join 5.5 us.
#include "attention_tile.h"

namespace gs {
namespace {

using namespace att;

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kKeys = 32;  // of a wave's tile

struct StepArgs {
  int batch, heads, kv_heads, dim, window, sinks, splits;
  float scale;
  const void* q;
  const void* k;
  const void* v;
  void* k_cache;
  void* v_cache;
  Strides sk, sv;
  const int32_t* positions;
  void* out;
  float* parts;  // [batch, heads, splits, dim]
  float* stats;  // [batch, heads, splits, 2]: maximum (in powers of two) and sum
};

template <typename T, int kDim>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) void attention_step_kernel(StepArgs a) {
  constexpr int kPitchT = kPitch<T, kDim>;
  constexpr int kSteps = kDim / 16, kBlocks = kDim / 32;
  constexpr int kV = 16 / int(sizeof(T)), kPerRow = kDim / kV, kCount = kKeys * kPerRow / kWave;
  __shared__ __align__(16) T tiles[kWaves][kKeys * kPitchT];
  __shared__ float joined[32][kDim + 1];
  __shared__ float tops[kWaves][32], sums[kWaves][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
  const int group = a.heads / a.kv_heads, group_tiles = (group + 31) / 32;
  const int kv = blockIdx.y / group_tiles, group_tile = blockIdx.y % group_tiles;
  const int b = blockIdx.z, split = blockIdx.x;
  const int member = group_tile * 32 + col;
  const bool live = member < group;
  const int head = kv * group + member;
  const int pos = a.positions[b];
  const int capacity = a.sinks + a.window;
  const int filled = pos < 0 ? 0 : int(min(int64_t(pos) + 1, int64_t(capacity)));
  const int slot = pos < a.sinks ? pos : a.sinks + (pos - a.sinks) % a.window;
  const int share = ((filled + a.splits - 1) / a.splits + kKeys - 1) / kKeys * kKeys;
  const int lo = int(min(int64_t(split) * share, int64_t(filled))), hi = min(lo + share, filled);

  T* kc = static_cast<T*>(a.k_cache) + b * a.sk.batch + kv * a.sk.head;
  T* vc = static_cast<T*>(a.v_cache) + b * a.sv.batch + kv * a.sv.head;
  const T* kn = static_cast<const T*>(a.k) + (int64_t(b) * a.kv_heads + kv) * a.dim;
  const T* vn = static_cast<const T*>(a.v) + (int64_t(b) * a.kv_heads + kv) * a.dim;
  if (group_tile == 0 && slot >= lo && slot < hi) {
    for (int d = threadIdx.x; d < a.dim; d += kThreads) {
      kc[slot * a.sk.token + d] = kn[d];
      vc[slot * a.sv.token + d] = vn[d];
    }
  }
  Frag<T> q[kSteps];
  {
    const T* row = static_cast<const T*>(a.q) + (int64_t(b) * a.heads + head) * a.dim;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = 16 * s + 8 * half;
      q[s] = load_global<T>(row + d, live && d < a.dim);
    }
  }
  const float c = a.scale * kLog2e;
  float top = -INFINITY, sum = 0.0f;
  Acc o[kBlocks];
#pragma unroll
  for (int n = 0; n < kBlocks; ++n) o[n] = Acc(0.0f);
  Frag<T> kf[kSteps];
  Vec<T, kV> vr[kCount];
  const auto fetch = [&](int j0) {
    const int j = j0 + col;
    const T* row = j == slot ? kn : kc + j * a.sk.token;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = 16 * s + 8 * half;
      kf[s] = load_global<T>(row + d, j < hi && d < a.dim);
    }
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int chunk = i * kWave + lane;
      const int r = j0 + chunk / kPerRow, d = chunk % kPerRow * kV;
      vr[i] = Vec<T, kV>(T(0.0f));
      if (r < hi && d < a.dim)
        vr[i] = *reinterpret_cast<const Vec<T, kV>*>((r == slot ? vn : vc + r * a.sv.token) + d);
    }
  };
  T* tile = tiles[wave];
  int j0 = lo + wave * kKeys;
  if (j0 < hi) fetch(j0);
  for (; j0 < hi; j0 += kWaves * kKeys) {
    Acc s(0.0f);
#pragma unroll
    for (int st = 0; st < kSteps; ++st) mma(kf[st], q[st], s);
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int chunk = i * kWave + lane;
      *reinterpret_cast<Vec<T, kV>*>(tile + chunk / kPerRow * kPitchT + chunk % kPerRow * kV) = vr[i];
    }
    wave_sync();
    if (j0 + kWaves * kKeys < hi) fetch(j0 + kWaves * kKeys);
    if (j0 + kKeys > hi) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (j0 + acc_row(r) >= hi) s[r] = -INFINITY;
    }
    float m = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) m = fmaxf(m, s[r]);
    m = fmaxf(m, __shfl_xor(m, 32, 64)) * c;
    if (__any(m > top)) {
      const float up = fmaxf(top, m);
      const float shrink = up == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - up);
      sum *= shrink;
#pragma unroll
      for (int n = 0; n < kBlocks; ++n) o[n] *= shrink;
      top = up;
    }
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] * c - base);
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const Frag<T> pf = acc_frag<T>(s, st);
      sum = add_all(pf, sum);
#pragma unroll
      for (int n = 0; n < kBlocks; ++n) mma(load_turned<T>(tile, kPitchT, 16 * st, 32 * n), pf, o[n]);
    }
    wave_sync();
  }
  // The waves join: the largest maximum, then the sums one wave after the other.
  sum += __shfl_xor(sum, 32, 64);
  if (half == 0) {
    tops[wave][col] = top;
    sums[wave][col] = sum;
  }
  __syncthreads();
  float all = tops[0][col];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) all = fmaxf(all, tops[w][col]);
  const float base = all == -INFINITY ? 0.0f : all;
  float whole = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float t = tops[w][col];
    whole += sums[w][col] * __builtin_amdgcn_exp2f(t - base);
  }
  const float shrink = __builtin_amdgcn_exp2f(top - base);
  for (int w = 0; w < kWaves; ++w) {
    if (wave == w) {
#pragma unroll
      for (int n = 0; n < kBlocks; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float& at = joined[col][32 * n + acc_row(r)];
          at = w ? at + o[n][r] * shrink : o[n][r] * shrink;
        }
    }
    __syncthreads();
  }
  // Rows of the result; thread t holds element t % kDim of every (256 / kDim)th.
  if (wave == 0 && half == 0) {
    tops[0][col] = all;
    sums[0][col] = whole;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 32 * kDim; e += kThreads) {
    const int m = e / kDim, d = e % kDim;
    if (group_tile * 32 + m >= group || d >= a.dim) continue;
    const int64_t row = int64_t(b) * a.heads + kv * group + group_tile * 32 + m;
    if (a.splits == 1) {
      const float l = sums[0][m];
      const bool none = tops[0][m] == -INFINITY && l == 0.0f;
      static_cast<T*>(a.out)[row * a.dim + d] = T(none ? 0.0f : joined[m][d] / l);
    } else {
      a.parts[(row * a.splits + split) * a.dim + d] = joined[m][d];
      if (d == 0) {
        a.stats[(row * a.splits + split) * 2] = tops[0][m];
        a.stats[(row * a.splits + split) * 2 + 1] = sums[0][m];
      }
    }
  }
}

// The shares of each row, in order.
template <typename T>
__global__ __launch_bounds__(128) void attention_step_join_kernel(StepArgs a) {
  const int64_t row = blockIdx.x;
  const int d = threadIdx.x;
  const float* stats = a.stats + row * a.splits * 2;
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, stats[2 * s]);
  const float base = top == -INFINITY ? 0.0f : top;
  if (d >= a.dim) return;
  float sum = 0.0f, o = 0.0f;
  for (int s = 0; s < a.splits; ++s) {
    const float w = __builtin_amdgcn_exp2f(stats[2 * s] - base);
    sum += stats[2 * s + 1] * w;
    o += a.parts[(row * a.splits + s) * a.dim + d] * w;
  }
  const bool none = top == -INFINITY && sum == 0.0f;
  static_cast<T*>(a.out)[row * a.dim + d] = T(none ? 0.0f : o / sum);
}

// Workgroups of one stream and key head: as many as fill the GPU three times over
// (512 at a time; streams of different lengths even out), with a tile for each of
// their waves.  The case above with 1024 workgroups: 202 us, 1536: 189, 2048: 196,
// twice 1536: 272.
int plan_splits(const gs_attention& d) {
  const int64_t capacity = d.sinks + d.window;
  const int64_t rows = d.batch * d.kv_heads * ((d.heads / d.kv_heads + 31) / 32);
  const int64_t most = (capacity + kWaves * kKeys - 1) / (kWaves * kKeys);
  return int(std::max<int64_t>(1, std::min<int64_t>({most, 1536 / std::max<int64_t>(rows, 1), 256})));
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" GS_API size_t gs_window_attention_step_workspace_bytes(const gs_attention* desc) {
  if (!desc || check_attention(*desc) != GS_OK) return 0;
  const int splits = plan_splits(*desc);
  if (splits == 1) return 0;
  return size_t(desc->batch) * size_t(desc->heads) * size_t(splits) *
         (size_t(desc->head_dim) + 2) * sizeof(float);
}

extern "C" GS_API int gs_window_attention_step(const gs_attention* desc, const void* q,
                                               const void* k, const void* v, void* k_cache,
                                               void* v_cache, const int64_t* strides,
                                               const int32_t* positions, void* out,
                                               void* workspace, size_t workspace_bytes,
                                               void* stream) {
  clear_error();
  GS_REQUIRE(desc, GS_ERR_INVALID_ARGUMENT, "null description");
  GS_TRY(check_attention(*desc));
  // The kernel counts slots in 32 bits, up to a round of tiles beyond the last.
  GS_REQUIRE(desc->window < (int64_t(1) << 30) && desc->sinks < (int64_t(1) << 30) - desc->window,
             GS_ERR_OVERFLOW, "cache too large: %lld first tokens and a window of %lld",
             (long long)desc->sinks, (long long)desc->window);
  if (desc->batch == 0) return GS_OK;
  const int64_t none[3] = {0, 0, 0};
  GS_REQUIRE(strides && positions, GS_ERR_INVALID_ARGUMENT, "null pointer");
  GS_TRY(check_rows(q, none, desc->type, "q"));
  GS_TRY(check_rows(k, none, desc->type, "k"));
  GS_TRY(check_rows(v, none, desc->type, "v"));
  GS_TRY(check_rows(out, none, desc->type, "out"));
  GS_TRY(check_rows(k_cache, strides, desc->type, "k_cache"));
  GS_TRY(check_rows(v_cache, strides + 3, desc->type, "v_cache"));
  const size_t need = gs_window_attention_step_workspace_bytes(desc);
  GS_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), GS_ERR_WORKSPACE,
             "workspace too small: %zu bytes, %zu needed", workspace_bytes, need);
  StepArgs a{};
  a.batch = int(desc->batch);
  a.heads = desc->heads;
  a.kv_heads = desc->kv_heads;
  a.dim = desc->head_dim;
  a.window = int(desc->window);
  a.sinks = int(desc->sinks);
  a.splits = plan_splits(*desc);
  a.scale = desc->scale;
  a.q = q;
  a.k = k;
  a.v = v;
  a.k_cache = k_cache;
  a.v_cache = v_cache;
  a.sk = {strides[0], strides[1], strides[2]};
  a.sv = {strides[3], strides[4], strides[5]};
  a.positions = positions;
  a.out = out;
  a.stats = static_cast<float*>(workspace);
  a.parts = a.stats + int64_t(a.batch) * a.heads * a.splits * 2;
  const int64_t rows = int64_t(a.kv_heads) * ((a.heads / a.kv_heads + 31) / 32);
  const dim3 grid(unsigned(a.splits), unsigned(rows), unsigned(a.batch));
  const hipStream_t s = as_stream(stream);
  return seq::with_type(desc->type, [&](auto t) {
    using T = decltype(t);
    if (a.dim <= 64)
      attention_step_kernel<T, 64><<<grid, kThreads, 0, s>>>(a);
    else
      attention_step_kernel<T, 128><<<grid, kThreads, 0, s>>>(a);
    GS_TRY(check_launch("window_attention_step"));
    if (a.splits == 1) return int(GS_OK);
    attention_step_join_kernel<T><<<unsigned(a.batch * a.heads), 128, 0, s>>>(a);
    return check_launch("window_attention_step join");
  });
}
