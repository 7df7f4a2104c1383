// Gated linear recurrence over the tokens of [batch, tokens, channels], per channel:
//   a_t = sigmoid(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  h_0 = state,
// and its backward,
//   G_t = grad_y_t + R_t,  R_{t-1} = a_t G_t,  R_T = grad_last,
//   grad_x = (1 - a) G,  grad_gate = G (h_{t-1} - x) a (1 - a),  grad_state = R_0.
// A step of either is the affine map h -> A h + B, and a run of steps composes
// to one such map, so the tokens are cut into chunks of 128 that workgroups hold
// in registers, a wave a run of tokens.  Each workgroup publishes its chunk's
// map, looks back for the nearest chunk whose end state is known, takes the maps
// in between from there in order, publishes its own end state and runs its
// tokens: every tensor is read and written once.  A chunk's state comes from the
// same products and sums whichever end state was found first, so the results do
// not depend on the schedule.  States, maps and sums are float32; y is rounded
// once.  The forward keeps the chunks' start states, from which the backward
// runs h again: that reads x and gate, which it needs in any case, and no h, and
// h does not carry y's rounding.
//
// A lane holds two neighbouring channels of a 16-bit type where rows allow
// 4-byte accesses.
#include "sequence.h"

namespace gs {
namespace {

using namespace seq;

constexpr int kChunk = 128;  // tokens of a workgroup

// Waves of a workgroup and each one's run of tokens.  The backward holds more
// for a token, so it gets by with shorter runs: both stay within the registers
// that let 16 waves share a CU.
template <bool kBackward>
struct Shape {
  static constexpr int kWaves = kBackward ? 16 : 8;
  static constexpr int kRun = kChunk / kWaves;
  static constexpr int kThreads = kWaves * kWave;
};

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
  // Published words; all bits set: not yet.  maps [batch, chunks, channels]: A
  // and B of a chunk in one word.  ends [batch, chunks, channels]: forward, h
  // before each chunk (the starts that the backward reads); backward, the
  // carried gradient after each chunk.  The entry of the chunk that comes next
  // is a chunk's end state.
  uint64_t* maps;
  float* ends;
  uint32_t* ticket;        // null: a single chunk
  uint32_t* flags;         // the device's check-failure word
  const float* state;      // h_0, or null
  const float* starts;     // backward: the forward's ends
  void* y;
  float* last;
  const float* grad_last;  // or null
  void* grad_x;
  void* grad_gate;
  float* grad_state;       // or null
};

constexpr uint32_t kUnset = 0xffffffffu;
constexpr int kSpinLimit = 1 << 20;
constexpr int kAhead = 8;  // published words that are requested together

// A float as a word that is not kUnset (a NaN of that pattern becomes another).
__device__ __forceinline__ uint32_t word_of(float v) {
  return v == v ? __float_as_uint(v) : 0x7fc00000u;
}
__device__ __forceinline__ uint64_t load_word(const uint64_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint32_t load_word(const uint32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename W>
__device__ __forceinline__ void store_word(W* p, W v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The lane's channels of one published row.
template <int kChannels>
struct Words {
  uint32_t w[kChannels];
  __device__ __forceinline__ void load(const float* p) {
    if constexpr (kChannels == 2) {
      const uint64_t v = load_word(reinterpret_cast<const uint64_t*>(p));
      w[0] = uint32_t(v);
      w[1] = uint32_t(v >> 32);
    } else {
      w[0] = load_word(reinterpret_cast<const uint32_t*>(p));
    }
  }
  __device__ __forceinline__ void store(float* p) const {
    if constexpr (kChannels == 2)
      store_word(reinterpret_cast<uint64_t*>(p), w[0] | uint64_t(w[1]) << 32);
    else
      store_word(reinterpret_cast<uint32_t*>(p), w[0]);
  }
  __device__ __forceinline__ bool set() const {
    bool ok = true;
#pragma unroll
    for (int n = 0; n < kChannels; ++n) ok &= w[n] != kUnset;
    return ok;
  }
};

// State before the chunk whose place in the walk is `place` (forward: the chunk,
// backward: counted from the last), for the channels of one wave's lanes: the
// nearest published end state and the maps after it.  A place's words are
// published by a workgroup with an earlier ticket, so every wait ends; the spin
// limit turns a broken invariant into an error flag.  `init` is the state before
// place 0.
template <bool kBackward, int kChannels>
__device__ FloatVec<kChannels> look_back(const ScanArgs& a, int64_t b, int64_t place, int64_t c,
                                         bool live, FloatVec<kChannels> init) {
  if (place == 0) return init;
  const auto row = [&](int64_t i) {
    return (b * a.chunks + (kBackward ? a.chunks - 1 - i : i)) * a.channels + c;
  };
  int spins = 0;
  // The nearest place whose start is known; that of place 0 always is.
  FloatVec<kChannels> h = init;
  int64_t from = place;
  for (bool found = false; !found && from > 0;) {
    Words<kChannels> w[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (live && from - i > 0) w[i].load(a.ends + row(from - i));
    int step = kAhead;
#pragma unroll
    for (int i = kAhead - 1; i >= 0; --i) {
      const bool known = from - i > 0 && __all(!live || w[i].set());
      if (known) {
        step = i;
#pragma unroll
        for (int n = 0; n < kChannels; ++n) h[n] = __uint_as_float(w[i].w[n]);
        found = true;
      }
    }
    from -= step;
  }
  if (from <= 0) {
    from = 0;
    h = init;
  }
  // The maps of places from .. place - 1, in order.
  while (from < place) {
    uint64_t m[kAhead][kChannels];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int n = 0; n < kChannels; ++n)
        m[i][n] = live && from + i < place ? load_word(a.maps + row(from + i) + n) : 0;
    int taken = 0;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      bool ready = from + i < place && taken == i;
#pragma unroll
      for (int n = 0; n < kChannels; ++n) ready &= bool(__all(m[i][n] != ~uint64_t(0)));
      if (ready) {
#pragma unroll
        for (int n = 0; n < kChannels; ++n)
          h[n] = __builtin_fmaf(__uint_as_float(uint32_t(m[i][n])), h[n],
                                __uint_as_float(uint32_t(m[i][n] >> 32)));
        taken = i + 1;
      }
    }
    from += taken;
    if (taken == 0) {
      if (++spins > kSpinLimit) {
        if ((threadIdx.x & 63) == 0) atomicOr(a.flags, kDeviceFlagSpinLimit);
        return h;
      }
      __builtin_amdgcn_s_sleep(1);
    }
  }
  return h;
}

// A workgroup's place: tickets in the order of the places, so that what a
// workgroup waits for is held by others that already run.
template <bool kBackward, int kChannels>
struct Place {
  static constexpr int kRun = Shape<kBackward>::kRun;
  int64_t b, place, chunk, c, t0;
  int count, lane, wave;
  bool live;
  __device__ Place(const ScanArgs& a, uint32_t* shared) {
    uint32_t item = blockIdx.x;
    if (a.ticket) {
      if (threadIdx.x == 0) *shared = atomicAdd(a.ticket, 1u);
      __syncthreads();
      item = *shared;
    }
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tiles = uint32_t((a.channels + kWave * kChannels - 1) / (kWave * kChannels));
    c = (int64_t(item % tiles) * kWave + lane) * kChannels;
    b = item / tiles % uint32_t(a.batch);
    place = item / tiles / uint32_t(a.batch);
    chunk = kBackward ? a.chunks - 1 - place : place;
    live = c < a.channels;
    t0 = chunk * kChunk + wave * kRun;
    const int64_t left = a.tokens - t0;
    count = int(left < 0 ? 0 : (left < kRun ? left : kRun));
  }
};

template <int kChannels>
__device__ __forceinline__ FloatVec<kChannels> load_state(const float* p, int64_t at, bool live) {
  FloatVec<kChannels> v(0.0f);
  if (p && live) {
#pragma unroll
    for (int n = 0; n < kChannels; ++n) v[n] = p[at + n];
  }
  return v;
}

template <int kChannels>
__device__ __forceinline__ FloatVec<kChannels> fma(FloatVec<kChannels> a, FloatVec<kChannels> x,
                                                   FloatVec<kChannels> y) {
#pragma unroll
  for (int n = 0; n < kChannels; ++n) y[n] = __builtin_fmaf(a[n], x[n], y[n]);
  return y;
}

template <typename T, int kChannels>
__global__ __launch_bounds__(Shape<false>::kThreads, 4) void scan_fwd_kernel(ScanArgs a) {
  constexpr int kRun = Shape<false>::kRun, kWaves = Shape<false>::kWaves;
  using Channels = FloatVec<kChannels>;
  __shared__ Channels mapA[kWaves][kWave], mapB[kWaves][kWave], before[kWave];
  __shared__ uint32_t ticket;
  const Place<false, kChannels> w(a, &ticket);
  Channels ga[kRun], gb[kRun];  // a and (1 - a) x
  {
    Vec<T, kChannels> x[kRun], g[kRun];
    const T* px = static_cast<const T*>(a.x) + w.b * a.x_batch + w.t0 * a.x_token + w.c;
    const T* pg = static_cast<const T*>(a.gate) + w.b * a.gate_batch + w.t0 * a.gate_token + w.c;
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      if (w.live && i < w.count) {
        x[i] = load_channels<T, kChannels>(px + i * a.x_token);
        g[i] = load_channels<T, kChannels>(pg + i * a.gate_token);
      }
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      ga[i] = Channels(1.0f);
      gb[i] = Channels(0.0f);
      if (w.live && i < w.count) {
#pragma unroll
        for (int n = 0; n < kChannels; ++n) {
          const Gate gt = gate_of<T>(float(g[i][n]));
          ga[i][n] = gt.a;
          gb[i][n] = gt.keep * float(x[i][n]);
        }
      }
    }
  }
  Channels A(1.0f), B(0.0f);
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    B = fma<kChannels>(ga[i], B, gb[i]);
    A *= ga[i];
  }
  mapA[w.wave][w.lane] = A;
  mapB[w.wave][w.lane] = B;
  __syncthreads();
  if (w.wave == 0) {
    const int64_t at = (w.b * a.chunks + w.chunk) * a.channels + w.c;
    for (int i = 1; i < kWaves; ++i) {
      B = fma<kChannels>(mapA[i][w.lane], B, mapB[i][w.lane]);
      A *= mapA[i][w.lane];
    }
    const bool more = w.chunk + 1 < a.chunks;
    if (w.live && more) {
#pragma unroll
      for (int n = 0; n < kChannels; ++n)
        store_word(a.maps + at + n, word_of(A[n]) | uint64_t(word_of(B[n])) << 32);
    }
    const Channels init = load_state<kChannels>(a.state, w.b * a.channels + w.c, w.live);
    const Channels h = look_back<false, kChannels>(a, w.b, w.place, w.c, w.live, init);
    const Channels end = fma<kChannels>(A, h, B);
    if (w.live) {
      Words<kChannels> v;
      if (more) {
#pragma unroll
        for (int n = 0; n < kChannels; ++n) v.w[n] = word_of(end[n]);
        v.store(a.ends + at + a.channels);
      }
      if (w.chunk == 0) {
#pragma unroll
        for (int n = 0; n < kChannels; ++n) a.ends[at + n] = h[n];
      }
    }
    before[w.lane] = h;
  }
  __syncthreads();
  if (!w.live) return;
  Channels h = before[w.lane];
  for (int i = 0; i < w.wave; ++i) h = fma<kChannels>(mapA[i][w.lane], h, mapB[i][w.lane]);
  T* py = static_cast<T*>(a.y) + (w.b * a.tokens + w.t0) * a.channels + w.c;
#pragma unroll
  for (int i = 0; i < kRun; ++i)
    if (i < w.count) {
      h = fma<kChannels>(ga[i], h, gb[i]);
      store_channels<T, kChannels>(py + i * a.channels, h);
    }
  if (w.count > 0 && w.t0 + w.count == a.tokens) {
#pragma unroll
    for (int n = 0; n < kChannels; ++n) a.last[w.b * a.channels + w.c + n] = h[n];
  }
}

// Backward, the tokens last to first.
template <typename T, int kChannels>
__global__ __launch_bounds__(Shape<true>::kThreads, 4) void scan_bwd_kernel(ScanArgs a) {
  constexpr int kRun = Shape<true>::kRun, kWaves = Shape<true>::kWaves;
  using Channels = FloatVec<kChannels>;
  // A: the run's gates' product, in both directions; B: forward map of h; R:
  // backward map of the carried gradient.
  __shared__ Channels mapA[kWaves][kWave], mapB[kWaves][kWave], mapR[kWaves][kWave], after[kWave];
  __shared__ uint32_t ticket;
  const Place<true, kChannels> w(a, &ticket);
  const int64_t at = (w.b * a.chunks + w.chunk) * a.channels + w.c;
  Channels ga[kRun], keep[kRun], gap[kRun];  // gap: x, later h_{t-1} - x
  Vec<T, kChannels> dy[kRun];
  {
    Vec<T, kChannels> x[kRun], g[kRun];
    const T* px = static_cast<const T*>(a.x) + w.b * a.x_batch + w.t0 * a.x_token + w.c;
    const T* pg = static_cast<const T*>(a.gate) + w.b * a.gate_batch + w.t0 * a.gate_token + w.c;
    const T* pd = static_cast<const T*>(a.grad_y) + w.b * a.grad_batch + w.t0 * a.grad_token + w.c;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      dy[i] = Vec<T, kChannels>(T(0.0f));
      if (w.live && i < w.count) {
        x[i] = load_channels<T, kChannels>(px + i * a.x_token);
        g[i] = load_channels<T, kChannels>(pg + i * a.gate_token);
        if (a.grad_y) dy[i] = load_channels<T, kChannels>(pd + i * a.grad_token);
      }
    }
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      ga[i] = Channels(1.0f);
      keep[i] = gap[i] = Channels(0.0f);
      if (w.live && i < w.count) {
#pragma unroll
        for (int n = 0; n < kChannels; ++n) {
          const Gate gt = gate_of<T>(float(g[i][n]));
          ga[i][n] = gt.a;
          keep[i][n] = gt.keep;
          gap[i][n] = float(x[i][n]);
        }
      }
    }
  }
  Channels A(1.0f), B(0.0f), R(0.0f);
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    A *= ga[i];
#pragma unroll
    for (int n = 0; n < kChannels; ++n) {
      // Token i's gradient reaches the run's start through a_0 .. a_i.
      R[n] = __builtin_fmaf(A[n], float(dy[i][n]), R[n]);
      B[n] = __builtin_fmaf(ga[i][n], B[n], keep[i][n] * gap[i][n]);
    }
  }
  mapA[w.wave][w.lane] = A;
  mapB[w.wave][w.lane] = B;
  mapR[w.wave][w.lane] = R;
  __syncthreads();
  if (w.wave == kWaves - 1) {
    for (int i = kWaves - 2; i >= 0; --i) {
      R = fma<kChannels>(mapA[i][w.lane], R, mapR[i][w.lane]);
      A *= mapA[i][w.lane];
    }
    const bool more = w.place + 1 < a.chunks;
    if (w.live && more) {
#pragma unroll
      for (int n = 0; n < kChannels; ++n)
        store_word(a.maps + at + n, word_of(A[n]) | uint64_t(word_of(R[n])) << 32);
    }
    const Channels init = load_state<kChannels>(a.grad_last, w.b * a.channels + w.c, w.live);
    const Channels r = look_back<true, kChannels>(a, w.b, w.place, w.c, w.live, init);
    const Channels end = fma<kChannels>(A, r, R);
    if (w.live && more) {
      Words<kChannels> v;
#pragma unroll
      for (int n = 0; n < kChannels; ++n) v.w[n] = word_of(end[n]);
      v.store(a.ends + at - a.channels);
    }
    after[w.lane] = r;
  }
  // Meanwhile the states: gap becomes h_{t-1} - x.
  Channels h = load_state<kChannels>(a.starts, at, w.live);
  for (int i = 0; i < w.wave; ++i) h = fma<kChannels>(mapA[i][w.lane], h, mapB[i][w.lane]);
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    const Channels next = fma<kChannels>(ga[i], h, keep[i] * gap[i]);
    gap[i] = h - gap[i];
    h = next;
  }
  __syncthreads();
  if (!w.live) return;
  Channels r = after[w.lane];
  for (int i = kWaves - 1; i > w.wave; --i) r = fma<kChannels>(mapA[i][w.lane], r, mapR[i][w.lane]);
  const int64_t row = (w.b * a.tokens + w.t0) * a.channels + w.c;
  T* pdx = static_cast<T*>(a.grad_x) + row;
  T* pdg = static_cast<T*>(a.grad_gate) + row;
#pragma unroll
  for (int i = kRun - 1; i >= 0; --i)
    if (i < w.count) {
      const Channels G = to_float<T, kChannels>(dy[i]) + r;
      store_channels<T, kChannels>(pdx + i * a.channels, keep[i] * G);
      store_channels<T, kChannels>(pdg + i * a.channels, G * gap[i] * (ga[i] * keep[i]));
      r = ga[i] * G;
    }
  if (a.grad_state && w.t0 == 0) {
#pragma unroll
    for (int n = 0; n < kChannels; ++n) a.grad_state[w.b * a.channels + w.c + n] = r[n];
  }
}

// Nothing published yet: `words` 32-bit words at p and `more` at q; the ticket at 0.
__global__ __launch_bounds__(256) void scan_clear_kernel(uint32_t* p, int64_t words, uint32_t* q,
                                                         int64_t more, uint32_t* ticket) {
  const int64_t step = int64_t(gridDim.x) * 256;
  const int64_t first = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (first == 0) *ticket = 0;
  for (int64_t i = first; i < words; i += step) p[i] = kUnset;
  for (int64_t i = first; i < more; i += step) q[i] = kUnset;
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
  GS_REQUIRE(batch < 65536 && tokens < (int64_t(1) << 40) && channels < (int64_t(1) << 31),
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
  return aligned_to(a.ends, 8) && aligned_to(a.starts, 8);
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

// Published words of one call (when there is more than one chunk): the maps,
// the ticket and, for the backward, the carried gradients.
struct ScanSpace {
  size_t maps, ticket, carries, bytes;
};
ScanSpace scan_space(int64_t batch, int64_t chunks, int64_t channels, bool backward) {
  const size_t states = size_t(batch) * size_t(chunks) * size_t(channels);
  ScanSpace s{};
  if (chunks <= 1) return s;
  s.ticket = 0;
  s.maps = 16;
  s.carries = s.maps + states * 8;
  s.bytes = s.carries + (backward ? states * 4 : 0);
  return s;
}

template <bool kBackward>
int run_scan(ScanArgs& a, int32_t type, char* workspace, hipStream_t s) {
  const bool two = pairs(a, type);
  const int64_t lanes = two ? 2 * kWave : kWave;
  const int64_t blocks = (a.channels + lanes - 1) / lanes * a.chunks * a.batch;
  GS_REQUIRE(blocks < (int64_t(1) << 31), GS_ERR_OVERFLOW, "scan too large");
  if (a.chunks > 1) {
    const ScanSpace space = scan_space(a.batch, a.chunks, a.channels, kBackward);
    a.ticket = reinterpret_cast<uint32_t*>(workspace + space.ticket);
    a.maps = reinterpret_cast<uint64_t*>(workspace + space.maps);
    if (kBackward) a.ends = reinterpret_cast<float*>(workspace + space.carries);
    GS_TRY(device_flags(s, &a.flags));
    const int64_t states = a.batch * a.chunks * a.channels;
    const int64_t words = (states * 3 + 255) / 256;
    scan_clear_kernel<<<unsigned(std::min<int64_t>(words, 2048)), 256, 0, s>>>(
        reinterpret_cast<uint32_t*>(a.maps), states * 2, reinterpret_cast<uint32_t*>(a.ends), states,
        a.ticket);
    GS_TRY(check_launch("gated_scan"));
  }
  return with_lane(type, two, [&](auto v, auto n) {
    using T = decltype(v);
    constexpr int kN = decltype(n)::value;
    if constexpr (kBackward)
      scan_bwd_kernel<T, kN><<<unsigned(blocks), Shape<true>::kThreads, 0, s>>>(a);
    else
      scan_fwd_kernel<T, kN><<<unsigned(blocks), Shape<false>::kThreads, 0, s>>>(a);
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
  return scan_space(batch, chunks_of(tokens), channels, backward != 0).bytes;
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
  const size_t need = gs_gated_scan_workspace_bytes(batch, tokens, channels, 0);
  GS_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), GS_ERR_WORKSPACE,
             "workspace too small: %zu bytes", workspace_bytes);
  GS_REQUIRE(aligned_to(workspace, 8), GS_ERR_INVALID_ARGUMENT, "workspace must be 8-byte aligned");
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
  a.ends = starts;
  a.state = state;
  a.y = y;
  a.last = last;
  return run_scan<false>(a, type, static_cast<char*>(workspace), as_stream(stream));
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
  const size_t need = gs_gated_scan_workspace_bytes(batch, tokens, channels, 1);
  GS_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), GS_ERR_WORKSPACE,
             "workspace too small: %zu bytes", workspace_bytes);
  GS_REQUIRE(aligned_to(workspace, 8), GS_ERR_INVALID_ARGUMENT, "workspace must be 8-byte aligned");
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
  a.starts = starts;
  a.grad_last = grad_last;
  a.grad_x = grad_x;
  a.grad_gate = grad_gate;
  a.grad_state = grad_state;
  return run_scan<true>(a, type, static_cast<char*>(workspace), as_stream(stream));
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
