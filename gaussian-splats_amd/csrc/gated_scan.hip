// Gated linear recurrence over the tokens of [batch, tokens, channels], per channel:
//   a_t = sigmoid(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  h_0 = state,
// and its backward,
//   G_t = grad_y_t + R_t,  R_{t-1} = a_t G_t,  R_T = grad_last,
//   grad_x = (1 - a) G,  grad_gate = G (h_{t-1} - x) a (1 - a),  grad_state = R_0.
// A step of either is the affine map h -> A h + B, and a run of steps composes
// to one such map, so the tokens are cut into chunks of 256: the chunks' maps
// are computed side by side, a walk over the maps gives the state at each
// chunk's start, and each chunk is then run from it.  States, maps and sums are
// float32; y is rounded once.  The forward keeps the chunks' start states, from
// which the backward runs h again: that reads x and gate, which it needs in any
// case, and no h, and h does not carry y's rounding.
//
// A workgroup holds one chunk of 64 lanes' channels in registers, its waves a
// run of tokens each; the waves' maps meet in LDS.  A lane holds two
// neighbouring channels of a 16-bit type where rows allow 4-byte accesses.
#include "sequence.h"

namespace gs {
namespace {

using namespace seq;

constexpr int kChunk = 256;  // tokens

struct Gate {
  float a;     // sigmoid(g)
  float keep;  // sigmoid(-g)
};

template <typename T>
__device__ __forceinline__ Gate gate_of(float g) {
  // exp(-|g|) does not overflow, and neither a nor 1 - a loses bits near 0 or 1.
  // float32 inputs get the library's exp; for 16-bit ones the instruction's
  // error is far below their rounding.
  float e;
  if constexpr (sizeof(T) == 4)
    e = expf(-fabsf(g));
  else
    e = __builtin_amdgcn_exp2f(-fabsf(g) * 1.44269504f);
  const float r = __builtin_amdgcn_rcpf(1.0f + e);
  return g >= 0.0f ? Gate{r, e * r} : Gate{e * r, r};
}

// N channels of one lane.
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_channels(const T* p) {
  if constexpr (N == 1)
    return Vec<T, 1>{*p};
  else
    return *reinterpret_cast<const Vec<T, N>*>(p);
}
template <typename T, int N>
__device__ __forceinline__ void store_channels(T* p, const FloatVec<N>& v) {
  if constexpr (N == 1)
    *p = T(v[0]);
  else
    *reinterpret_cast<Vec<T, N>*>(p) = from_float<T, N>(v);
}

struct ScanArgs {
  const void* x;
  const void* gate;
  const void* grad_y;      // backward; null: zeros
  int64_t x_batch, x_token, gate_batch, gate_token, grad_batch, grad_token;  // strides
  int64_t batch, tokens, channels, chunks;
  float* maps;        // [batch, chunks, 2, channels]: A and B of each chunk
  float* starts;      // [batch, chunks, channels]: h before each chunk
  const float* state;      // h_0, or null
  void* y;
  float* last;
  const float* grad_last;  // or null
  float* carries;     // backward: R after each chunk
  void* grad_x;
  void* grad_gate;
  float* grad_state;  // or null
};

template <typename T, int kChannels>
struct Tile {
  int64_t b, chunk, c;  // batch, chunk, first channel of the lane
  int64_t t0;           // first token of the wave
  int count;            // tokens of the wave
  bool live;            // the lane has channels
  __device__ Tile(const ScanArgs& a, int run) {
    b = blockIdx.z;
    chunk = blockIdx.y;
    c = (int64_t(blockIdx.x) * kWave + (threadIdx.x & 63)) * kChannels;
    live = c < a.channels;
    t0 = chunk * kChunk + int64_t(threadIdx.x >> 6) * run;
    const int64_t left = a.tokens - t0;
    count = int(left < 0 ? 0 : (left < run ? left : run));
  }
};

// Forward.  kMaps: write the chunk's map; otherwise run it from its start
// state.  Eight waves, 32 tokens each.
template <typename T, int kChannels, bool kMaps>
__global__ __launch_bounds__(512) void scan_fwd_kernel(ScanArgs a) {
  constexpr int kRun = 32, kWaves = 8;
  __shared__ FloatVec<kChannels> mapA[kWaves][kWave], mapB[kWaves][kWave];
  const Tile<T, kChannels> w(a, kRun);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Vec<T, kChannels> x[kRun], g[kRun];
  if (w.live) {
    const T* px = static_cast<const T*>(a.x) + w.b * a.x_batch + w.t0 * a.x_token + w.c;
    const T* pg = static_cast<const T*>(a.gate) + w.b * a.gate_batch + w.t0 * a.gate_token + w.c;
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      if (i < w.count) {
        x[i] = load_channels<T, kChannels>(px + i * a.x_token);
        g[i] = load_channels<T, kChannels>(pg + i * a.gate_token);
      }
  }
  FloatVec<kChannels> A(1.0f), B(0.0f);
  if (w.live) {
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      if (i < w.count) {
#pragma unroll
        for (int n = 0; n < kChannels; ++n) {
          const Gate gt = gate_of<T>(float(g[i][n]));
          B[n] = gt.a * B[n] + gt.keep * float(x[i][n]);
          A[n] *= gt.a;
        }
      }
  }
  mapA[wave][lane] = A;
  mapB[wave][lane] = B;
  __syncthreads();
  if (!w.live) return;
  const int64_t at = (w.b * a.chunks + w.chunk) * a.channels + w.c;
  if constexpr (kMaps) {
    if (wave != 0) return;
    for (int i = 1; i < kWaves; ++i) {
      B = mapA[i][lane] * B + mapB[i][lane];
      A = A * mapA[i][lane];
    }
    float* m = a.maps + 2 * (w.b * a.chunks + w.chunk) * a.channels + w.c;
#pragma unroll
    for (int n = 0; n < kChannels; ++n) {
      m[n] = A[n];
      m[a.channels + n] = B[n];
    }
  } else {
    FloatVec<kChannels> h;
#pragma unroll
    for (int n = 0; n < kChannels; ++n) h[n] = a.starts[at + n];
    for (int i = 0; i < wave; ++i) h = mapA[i][lane] * h + mapB[i][lane];
    T* py = static_cast<T*>(a.y) + (w.b * a.tokens + w.t0) * a.channels + w.c;
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      if (i < w.count) {
#pragma unroll
        for (int n = 0; n < kChannels; ++n) {
          const Gate gt = gate_of<T>(float(g[i][n]));
          h[n] = gt.a * h[n] + gt.keep * float(x[i][n]);
        }
        store_channels<T, kChannels>(py + i * a.channels, h);
      }
    if (w.count > 0 && w.t0 + w.count == a.tokens) {
#pragma unroll
      for (int n = 0; n < kChannels; ++n) a.last[w.b * a.channels + w.c + n] = h[n];
    }
  }
}

// Backward, the tokens last to first.  Sixteen waves, 16 tokens each: a lane
// also holds the run's states.
template <typename T, int kChannels, bool kMaps>
__global__ __launch_bounds__(1024) void scan_bwd_kernel(ScanArgs a) {
  constexpr int kRun = 16, kWaves = 16;
  __shared__ FloatVec<kChannels> mapA[kWaves][kWave], mapB[kWaves][kWave], mapR[kWaves][kWave];
  const Tile<T, kChannels> w(a, kRun);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Vec<T, kChannels> x[kRun], g[kRun], dy[kRun];
  if (w.live) {
    const T* px = static_cast<const T*>(a.x) + w.b * a.x_batch + w.t0 * a.x_token + w.c;
    const T* pg = static_cast<const T*>(a.gate) + w.b * a.gate_batch + w.t0 * a.gate_token + w.c;
    const T* pd = static_cast<const T*>(a.grad_y) + w.b * a.grad_batch + w.t0 * a.grad_token + w.c;
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      if (i < w.count) {
        if constexpr (!kMaps) x[i] = load_channels<T, kChannels>(px + i * a.x_token);
        g[i] = load_channels<T, kChannels>(pg + i * a.gate_token);
        dy[i] = a.grad_y ? load_channels<T, kChannels>(pd + i * a.grad_token)
                         : Vec<T, kChannels>(T(0.0f));
      }
  }
  // A: the run's gates' product, in both directions; B: forward map of h;
  // R: backward map of the carried gradient.
  FloatVec<kChannels> A(1.0f), B(0.0f), R(0.0f);
  if (w.live) {
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      if (i < w.count) {
#pragma unroll
        for (int n = 0; n < kChannels; ++n) {
          const Gate gt = gate_of<T>(float(g[i][n]));
          // Terms of R in the order of the tokens: token i reaches the run's
          // start through a_0 .. a_i.
          A[n] *= gt.a;
          R[n] += A[n] * float(dy[i][n]);
          if constexpr (!kMaps) B[n] = gt.a * B[n] + gt.keep * float(x[i][n]);
        }
      }
  }
  mapA[wave][lane] = A;
  mapR[wave][lane] = R;
  if constexpr (!kMaps) mapB[wave][lane] = B;
  __syncthreads();
  if (!w.live) return;
  const int64_t at = (w.b * a.chunks + w.chunk) * a.channels + w.c;
  if constexpr (kMaps) {
    if (wave != kWaves - 1) return;
    for (int i = kWaves - 2; i >= 0; --i) {
      R = mapA[i][lane] * R + mapR[i][lane];
      A = A * mapA[i][lane];
    }
    float* m = a.maps + 2 * (w.b * a.chunks + w.chunk) * a.channels + w.c;
#pragma unroll
    for (int n = 0; n < kChannels; ++n) {
      m[n] = A[n];
      m[a.channels + n] = R[n];
    }
  } else {
    FloatVec<kChannels> h, r, before[kRun];
#pragma unroll
    for (int n = 0; n < kChannels; ++n) {
      h[n] = a.starts[at + n];
      r[n] = a.carries[at + n];
    }
    for (int i = 0; i < wave; ++i) h = mapA[i][lane] * h + mapB[i][lane];
    for (int i = kWaves - 1; i > wave; --i) r = mapA[i][lane] * r + mapR[i][lane];
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      if (i < w.count) {
        before[i] = h;
#pragma unroll
        for (int n = 0; n < kChannels; ++n) {
          const Gate gt = gate_of<T>(float(g[i][n]));
          h[n] = gt.a * h[n] + gt.keep * float(x[i][n]);
        }
      }
    const int64_t row = (w.b * a.tokens + w.t0) * a.channels + w.c;
    T* pdx = static_cast<T*>(a.grad_x) + row;
    T* pdg = static_cast<T*>(a.grad_gate) + row;
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i)
      if (i < w.count) {
        FloatVec<kChannels> dx, dg;
#pragma unroll
        for (int n = 0; n < kChannels; ++n) {
          const Gate gt = gate_of<T>(float(g[i][n]));
          const float G = float(dy[i][n]) + r[n];
          dx[n] = gt.keep * G;
          dg[n] = G * (before[i][n] - float(x[i][n])) * (gt.a * gt.keep);
          r[n] = gt.a * G;
        }
        store_channels<T, kChannels>(pdx + i * a.channels, dx);
        store_channels<T, kChannels>(pdg + i * a.channels, dg);
      }
    if (a.grad_state && w.t0 == 0) {
#pragma unroll
      for (int n = 0; n < kChannels; ++n) a.grad_state[w.b * a.channels + w.c + n] = r[n];
    }
  }
}

// The walk over a channel's chunks: forward, h before each chunk; backward,
// the carried gradient after each chunk, last chunk first.  A lane has a
// channel, the sixteen waves a run of chunks each: they compose their run's map,
// get the state before it from the runs in front, and walk the run from it.
template <bool kBackward>
__global__ __launch_bounds__(1024) void scan_walk_kernel(ScanArgs a) {
  constexpr int kWaves = 16, kAhead = 8;
  __shared__ float mapA[kWaves][kWave], mapB[kWaves][kWave];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t c = int64_t(blockIdx.x) * kWave + lane, b = blockIdx.y;
  const bool live = c < a.channels;
  const int64_t run = (a.chunks + kWaves - 1) / kWaves;
  const int64_t lo = std::min<int64_t>(a.chunks, wave * run), hi = std::min<int64_t>(a.chunks, lo + run);
  const auto chunk = [&](int64_t i) { return b * a.chunks + (kBackward ? a.chunks - 1 - i : i); };
  // Calls f(i, A, B) for the run's chunks; kAhead maps are loaded together.
  const auto each = [&](auto&& f) {
    for (int64_t i = lo; i < hi; i += kAhead) {
      float A[kAhead], B[kAhead];
#pragma unroll
      for (int n = 0; n < kAhead; ++n)
        if (i + n < hi) {
          const float* m = a.maps + 2 * chunk(i + n) * a.channels + c;
          A[n] = m[0];
          B[n] = m[a.channels];
        }
#pragma unroll
      for (int n = 0; n < kAhead; ++n)
        if (i + n < hi) f(i + n, A[n], B[n]);
    }
  };
  float A = 1.0f, B = 0.0f;
  if (live && a.maps && wave + 1 < kWaves)
    each([&](int64_t, float x, float y) {
      B = x * B + y;
      A *= x;
    });
  mapA[wave][lane] = A;
  mapB[wave][lane] = B;
  __syncthreads();
  if (!live) return;
  const float* init = kBackward ? a.grad_last : a.state;
  float h = init ? init[b * a.channels + c] : 0.0f;
  for (int i = 0; i < wave; ++i) h = mapA[i][lane] * h + mapB[i][lane];
  float* out = kBackward ? a.carries : a.starts;
  if (a.maps)
    each([&](int64_t i, float x, float y) {
      out[chunk(i) * a.channels + c] = h;
      h = x * h + y;
    });
  else if (wave == 0)
    out[chunk(0) * a.channels + c] = h;
}

template <typename T, int kChannels>
__global__ __launch_bounds__(256) void scan_step_kernel(const T* x, const T* gate,
                                                        const float* state, int64_t groups,
                                                        T* y, float* state_out) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= groups) return;
  const FloatVec<kChannels> xs = to_float<T, kChannels>(load_channels<T, kChannels>(x + i * kChannels));
  const FloatVec<kChannels> gs = to_float<T, kChannels>(load_channels<T, kChannels>(gate + i * kChannels));
  FloatVec<kChannels> h = load_channels<float, kChannels>(state + i * kChannels);
#pragma unroll
  for (int n = 0; n < kChannels; ++n) {
    const Gate gt = gate_of<T>(gs[n]);
    h[n] = gt.a * h[n] + gt.keep * xs[n];
  }
  store_channels<float, kChannels>(state_out + i * kChannels, h);
  store_channels<T, kChannels>(y + i * kChannels, h);
}

int check_scan(int64_t batch, int64_t tokens, int64_t channels, int32_t type) {
  GS_REQUIRE(batch >= 0 && tokens >= 0 && channels >= 0, GS_ERR_INVALID_ARGUMENT,
             "sizes must be non-negative, got [%lld, %lld, %lld]", (long long)batch,
             (long long)tokens, (long long)channels);
  GS_REQUIRE(seq::float_type(type), GS_ERR_INVALID_ARGUMENT,
             "type must be GS_F32, GS_F16 or GS_BF16");
  GS_REQUIRE(batch < 65536 && tokens <= int64_t(65535) * kChunk && channels < (int64_t(1) << 31),
             GS_ERR_OVERFLOW, "too large: [%lld, %lld, %lld]", (long long)batch,
             (long long)tokens, (long long)channels);
  return GS_OK;
}

int64_t chunks_of(int64_t tokens) { return (tokens + kChunk - 1) / kChunk; }

// Two channels a lane where every row of every tensor allows 4-byte accesses.
bool pairs(const ScanArgs& a, int32_t type) {
  if (type == GS_F32 || a.channels % 2) return false;
  const int64_t strides = a.x_batch | a.x_token | a.gate_batch | a.gate_token | a.grad_batch |
                          a.grad_token;
  if (strides & 1) return false;
  for (const void* p : {a.x, a.gate, a.grad_y, static_cast<const void*>(a.y),
                        static_cast<const void*>(a.grad_x), static_cast<const void*>(a.grad_gate)})
    if (!aligned_to(p, 4)) return false;
  return true;
}

template <typename F>
int with_lane(int32_t type, bool two, F&& f) {
  return with_type(type, [&](auto v) {
    using T = decltype(v);
    if constexpr (sizeof(T) == 2) {
      if (two) return f(v, std::integral_constant<int, 2>{});
    }
    return f(v, std::integral_constant<int, 1>{});
  });
}

template <bool kBackward>
int run_scan(const ScanArgs& a, int32_t type, hipStream_t s) {
  const bool two = pairs(a, type);
  const int64_t lanes = two ? 2 * kWave : kWave;
  const dim3 grid(unsigned((a.channels + lanes - 1) / lanes), unsigned(a.chunks),
                  unsigned(a.batch));
  return with_lane(type, two, [&](auto v, auto n) {
    using T = decltype(v);
    constexpr int kN = decltype(n)::value;
    if (a.maps) {
      if constexpr (kBackward)
        scan_bwd_kernel<T, kN, true><<<grid, 1024, 0, s>>>(a);
      else
        scan_fwd_kernel<T, kN, true><<<grid, 512, 0, s>>>(a);
      GS_TRY(check_launch("gated_scan maps"));
    }
    scan_walk_kernel<kBackward>
        <<<dim3(unsigned((a.channels + 63) / 64), unsigned(a.batch)), 1024, 0, s>>>(a);
    GS_TRY(check_launch("gated_scan walk"));
    if constexpr (kBackward)
      scan_bwd_kernel<T, kN, false><<<grid, 1024, 0, s>>>(a);
    else
      scan_fwd_kernel<T, kN, false><<<grid, 512, 0, s>>>(a);
    return check_launch("gated_scan");
  });
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" GS_API int64_t gs_gated_scan_chunks(int64_t tokens) {
  return tokens < 0 ? 0 : chunks_of(tokens);
}

extern "C" GS_API size_t gs_gated_scan_workspace_bytes(int64_t batch, int64_t tokens,
                                                       int64_t channels, int32_t backward) {
  if (batch <= 0 || tokens <= 0 || channels <= 0) return 0;
  const size_t states = size_t(batch) * size_t(chunks_of(tokens)) * size_t(channels);
  return states * sizeof(float) * (backward ? 3 : 2);
}

extern "C" GS_API int gs_gated_scan_fwd(const void* x, const void* gate, const float* state,
                                        int64_t batch, int64_t tokens, int64_t channels,
                                        const int64_t* strides, int32_t type, void* y, float* last,
                                        float* starts, void* workspace, size_t workspace_bytes,
                                        void* stream) {
  clear_error();
  GS_TRY(check_scan(batch, tokens, channels, type));
  if (batch == 0 || tokens == 0 || channels == 0) return GS_OK;
  GS_REQUIRE(x && gate && strides && y && last && starts, GS_ERR_INVALID_ARGUMENT, "null pointer");
  GS_REQUIRE(workspace && workspace_bytes >=
                 gs_gated_scan_workspace_bytes(batch, tokens, channels, 0),
             GS_ERR_WORKSPACE, "workspace too small: %zu bytes", workspace_bytes);
  ScanArgs a{};
  a.x = x;
  a.gate = gate;
  a.x_batch = strides[0];
  a.x_token = strides[1];
  a.gate_batch = strides[2];
  a.gate_token = strides[3];
  a.batch = batch;
  a.tokens = tokens;
  a.channels = channels;
  a.chunks = chunks_of(tokens);
  a.maps = a.chunks > 1 ? static_cast<float*>(workspace) : nullptr;
  a.starts = starts;
  a.state = state;
  a.y = y;
  a.last = last;
  return run_scan<false>(a, type, as_stream(stream));
}

extern "C" GS_API int gs_gated_scan_bwd(const void* x, const void* gate, const float* starts,
                                        const void* grad_y, const float* grad_last, int64_t batch,
                                        int64_t tokens, int64_t channels, const int64_t* strides,
                                        int32_t type, void* grad_x, void* grad_gate,
                                        float* grad_state, void* workspace, size_t workspace_bytes,
                                        void* stream) {
  clear_error();
  GS_TRY(check_scan(batch, tokens, channels, type));
  if (batch == 0 || tokens == 0 || channels == 0) return GS_OK;
  GS_REQUIRE(x && gate && strides && starts && grad_x && grad_gate, GS_ERR_INVALID_ARGUMENT,
             "null pointer");
  GS_REQUIRE(workspace && workspace_bytes >=
                 gs_gated_scan_workspace_bytes(batch, tokens, channels, 1),
             GS_ERR_WORKSPACE, "workspace too small: %zu bytes", workspace_bytes);
  ScanArgs a{};
  a.x = x;
  a.gate = gate;
  a.grad_y = grad_y;
  a.x_batch = strides[0];
  a.x_token = strides[1];
  a.gate_batch = strides[2];
  a.gate_token = strides[3];
  a.grad_batch = strides[4];
  a.grad_token = strides[5];
  a.batch = batch;
  a.tokens = tokens;
  a.channels = channels;
  a.chunks = chunks_of(tokens);
  a.carries = static_cast<float*>(workspace);
  a.maps = a.chunks > 1 ? a.carries + batch * a.chunks * channels : nullptr;
  a.starts = const_cast<float*>(starts);
  a.grad_last = grad_last;
  a.grad_x = grad_x;
  a.grad_gate = grad_gate;
  a.grad_state = grad_state;
  return run_scan<true>(a, type, as_stream(stream));
}

extern "C" GS_API int gs_gated_scan_step(const void* x, const void* gate, const float* state,
                                         int64_t batch, int64_t channels, int32_t type, void* y,
                                         float* state_out, void* stream) {
  clear_error();
  GS_TRY(check_scan(batch, 1, channels, type));
  const int64_t n = batch * channels;
  if (n == 0) return GS_OK;
  GS_REQUIRE(x && gate && state && y && state_out, GS_ERR_INVALID_ARGUMENT, "null pointer");
  GS_REQUIRE(n < (int64_t(1) << 38), GS_ERR_OVERFLOW, "too many channels");
  return with_lane(type, n % 2 == 0 && type != GS_F32 && aligned_to(x, 4) && aligned_to(gate, 4) &&
                             aligned_to(y, 4) && aligned_to(state, 8) && aligned_to(state_out, 8),
                   [&](auto v, auto k) {
                     using T = decltype(v);
                     constexpr int kN = decltype(k)::value;
                     const int64_t groups = n / kN;
                     scan_step_kernel<T, kN>
                         <<<unsigned((groups + 255) / 256), 256, 0, as_stream(stream)>>>(
                             static_cast<const T*>(x), static_cast<const T*>(gate), state, groups,
                             static_cast<T*>(y), state_out);
                     return check_launch("gated_scan_step");
                   });
}
