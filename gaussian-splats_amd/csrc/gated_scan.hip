// Gated linear recurrence over the tokens of [batch, tokens, channels], per channel:
//   a_t = sigmoid(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  h_0 = state,
// and its backward,
//   G_t = grad_y_t + R_t,  R_{t-1} = a_t G_t,  R_T = grad_last,
//   grad_x = (1 - a) G,  grad_gate = G (h_{t-1} - x) a (1 - a),  grad_state = R_0.
// A step of either is the affine map h -> A h + B, and a run of steps composes
// to one such map, so the tokens are cut into chunks (240 forward, 120 backward)
// that workgroups hold in registers, a wave a run of tokens.  Each workgroup publishes its chunk's
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
//
// Bound by memory in principle.  Measured, bfloat16, [1, 160000, 768]: forward 193
// us for 0.74 GB (3.8 TB/s, where a large copy moves 5.2), backward 304-317 us for
// 1.23 GB (3.9-4.0 TB/s): a workgroup fills a CU, and its items' loads run ahead by one item,
// but what a look back waits for is not all hidden.  Three kernels that read the
// inputs twice (maps, walk, run) took 375 and 500 us.  [2, 8160, 1024]: 37 and 46 us
// for 19 and 32 of bytes: 544 items forward on 256 workgroups, of which 32 take a
// third one while the others wait.
#include "sequence.h"

namespace gs {
namespace {

using namespace seq;

// A workgroup has 15 waves that hold a run of tokens each, and one that only
// looks back: it starts at once, while the others wait for their loads, and its
// registers and theirs are the same ones.  The backward holds more for a token,
// so its runs and chunks are half as long; the forward keeps a state at each
// start of the backward's chunks.
constexpr int kWaves = 15;
constexpr int kThreads = (kWaves + 1) * kWave;

template <bool kBackward>
struct Shape {
  static constexpr int kRun = kBackward ? 8 : 16;
  static constexpr int kChunk = kWaves * kRun;
};
constexpr int kStartTokens = Shape<true>::kChunk;  // tokens from one kept state to the next
constexpr int kStarts = Shape<false>::kChunk / kStartTokens;  // kept states of a forward chunk

struct Gate {
  float a;     // sigmoid(g)
  float keep;  // sigmoid(-g)
};

template <typename T>
__device__ __forceinline__ Gate gate_of(float g) {
  // With e = exp(-g), a = 1 / (1 + e) and 1 - a = e a lose no bits near 0 or 1.
  // Where e is huge a may be 0 (the reciprocal instruction's results have no
  // subnormals) and e a anything: 1 - a is 1 there.  A NaN of g stays in both.
  // float32 inputs get the library's exp; for 16-bit ones the instruction's error
  // is far below their rounding.
  float e;
  if constexpr (sizeof(T) == 4)
    e = expf(-g);
  else
    e = __builtin_amdgcn_exp2f(g * -1.44269504f);
  const float a = __builtin_amdgcn_rcpf(1.0f + e);
  return {a, e > 1e30f ? 1.0f : e * a};
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
  int64_t batch, tokens, channels, chunks, starts_count;
  uint32_t items;          // chunks of all channels' tiles and sequences
  // Published words; all bits set: not yet.  maps [batch, chunks, channels]: A
  // and B of a chunk in one word.  ends: the state that a chunk starts from,
  // forward h [batch, starts_count, channels], of which a chunk has kStarts,
  // backward the carried gradient [batch, chunks, channels].
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
constexpr int kComputeUnits = 256;
// Published words that are requested together: starts, and maps.
constexpr int kSeek = 4, kAhead = 8;

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

// One item of the work: a chunk of a tile of channels of a sequence.  Items are
// numbered in the order of the chunks' places in the walk (forward the chunk,
// backward counted from the last one).
template <bool kBackward, int kChannels>
struct Item {
  static constexpr int kRun = Shape<kBackward>::kRun;
  int64_t b, place, chunk, c, t0;
  int count;  // tokens of the wave's run that exist
  bool live;  // the lane has channels; others repeat the last ones
  __device__ __forceinline__ Item(const ScanArgs& a, uint32_t item, int wave, int lane) {
    const uint32_t tiles = uint32_t((a.channels + kWave * kChannels - 1) / (kWave * kChannels));
    c = (int64_t(item % tiles) * kWave + lane) * kChannels;
    live = c < a.channels;
    c = live ? c : a.channels - kChannels;
    b = item / tiles % uint32_t(a.batch);
    place = item / tiles / uint32_t(a.batch);
    chunk = kBackward ? a.chunks - 1 - place : place;
    t0 = chunk * Shape<kBackward>::kChunk + wave * kRun;
    const int64_t left = a.tokens - t0;
    count = int(left < 0 ? 0 : (left < kRun ? left : kRun));
  }
  __device__ __forceinline__ bool last(const ScanArgs& a) const { return place + 1 >= a.chunks; }
};

template <bool kBackward>
__device__ __forceinline__ int64_t map_row(const ScanArgs& a, int64_t b, int64_t place) {
  return (b * a.chunks + (kBackward ? a.chunks - 1 - place : place)) * a.channels;
}
template <bool kBackward>
__device__ __forceinline__ int64_t end_row(const ScanArgs& a, int64_t b, int64_t place) {
  return kBackward ? map_row<true>(a, b, place)
                   : (b * a.starts_count + place * kStarts) * a.channels;
}

// State before an item's chunk for the channels of one wave's lanes: the nearest
// published one and the maps after it.  These are published by workgroups that
// hold earlier tickets, so every wait ends; the spin limit turns a broken
// invariant into an error flag and a state of NaN, as no call waits for the flag:
// an output that misses what was waited for is NaN, never a wrong number (seen with
// a limit of 0).  `init` is the state before place 0.
template <bool kBackward, int kChannels>
__device__ FloatVec<kChannels> look_back(const ScanArgs& a, int64_t b, int64_t place, int64_t c,
                                         FloatVec<kChannels> init) {
  FloatVec<kChannels> h = init;
  int64_t from = place;  // down to the nearest place whose start is known
  for (bool found = false; !found && from > 0;) {
    Words<kChannels> w[kSeek];
#pragma unroll
    for (int i = 0; i < kSeek; ++i)
      if (from - i > 0) w[i].load(a.ends + end_row<kBackward>(a, b, from - i) + c);
    int step = kSeek;
#pragma unroll
    for (int i = kSeek - 1; i >= 0; --i)
      if (from - i > 0 && __all(w[i].set())) {
        step = i;
        found = true;
#pragma unroll
        for (int n = 0; n < kChannels; ++n) h[n] = __uint_as_float(w[i].w[n]);
      }
    from -= step;
    if (!found) h = init;
  }
  from = from > 0 ? from : 0;
  int spins = 0;
  while (from < place) {  // the maps of places from .. place - 1, in order
    uint64_t m[kAhead][kChannels];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int n = 0; n < kChannels; ++n)
        m[i][n] = from + i < place
                      ? load_word(a.maps + map_row<kBackward>(a, b, from + i) + c + n)
                      : ~uint64_t(0);
    int taken = 0;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      bool ready = taken == i;
#pragma unroll
      for (int n = 0; n < kChannels; ++n) ready = ready && __all(m[i][n] != ~uint64_t(0));
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
        if ((threadIdx.x & 63) == 0) atomicOr(a.flags, kDeviceFlagScan);
        return FloatVec<kChannels>(NAN);
      }
      __builtin_amdgcn_s_sleep(1);
    }
  }
  return h;
}

template <int kChannels>
__device__ __forceinline__ FloatVec<kChannels> load_state(const float* p, int64_t at) {
  FloatVec<kChannels> v(0.0f);
  if (p) {
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

// What a workgroup's waves share.  A workgroup takes items until none is left;
// of what one item's waves still read, the next item uses the other half.
// Counters only grow: the n-th item's signals have been given when `runs` is
// (n + 1) kWaves and `whole` n + 1.  Waves that wait for a counter wait for waves
// of their own workgroup, which wait for nothing.
template <int kChannels>
struct Shared {
  FloatVec<kChannels> mapA[2][kWaves][kWave], mapB[2][kWaves][kWave];
  FloatVec<kChannels> wholeA[2][kWave], wholeB[2][kWave], before[2][kWave];
  uint32_t ticket[4], runs, whole;
};

__device__ __forceinline__ void signal(uint32_t* counter) {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  if ((threadIdx.x & 63) == 0)
    __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}
__device__ __forceinline__ void await(uint32_t* counter, uint32_t count) {
  while (__hip_atomic_load(counter, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) < count)
    __builtin_amdgcn_s_sleep(1);
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Tickets in the order of the items, two ahead of the work: an item is only
// waited for by later ones, and whoever holds the earliest unfinished one works
// on it.
__device__ __forceinline__ uint32_t next_ticket(const ScanArgs& a, uint32_t turn) {
  return a.ticket ? atomicAdd(a.ticket, 1u) : turn ? a.items : uint32_t(block_index());
}

// The looking wave: finds the state before each item's chunk, publishes the one
// after it once the chunk's map is there, and leaves the former to the others.
template <bool kBackward, int kChannels>
__device__ __forceinline__ void look_wave(const ScanArgs& a, Shared<kChannels>& sh,
                                          const float* first) {
  using Channels = FloatVec<kChannels>;
  const int lane = threadIdx.x & 63;
  for (uint32_t n = 0;; ++n) {
    const uint32_t item = sh.ticket[n & 3];
    if (item >= a.items) return;
    if (lane == 0) sh.ticket[(n + 2) & 3] = next_ticket(a, 1);
    const Item<kBackward, kChannels> w(a, item, 0, lane);
    const Channels init = load_state<kChannels>(first, w.b * a.channels + w.c);
    const Channels h = look_back<kBackward, kChannels>(a, w.b, w.place, w.c, init);
    sh.before[n & 1][lane] = h;
    if (!w.last(a)) {
      await(&sh.whole, n + 1);
      const Channels end = fma<kChannels>(sh.wholeA[n & 1][lane], h, sh.wholeB[n & 1][lane]);
      Words<kChannels> v;
#pragma unroll
      for (int k = 0; k < kChannels; ++k) v.w[k] = word_of(end[k]);
      if (w.live) v.store(a.ends + end_row<kBackward>(a, w.b, w.place + 1) + w.c);
    }
    __syncthreads();
  }
}

// The first wave in the walk's order: composes and publishes the chunk's map.
template <bool kBackward, int kChannels>
__device__ __forceinline__ void publish_map(const ScanArgs& a, const Item<kBackward, kChannels>& w,
                                            Shared<kChannels>& sh, uint32_t n) {
  using Channels = FloatVec<kChannels>;
  const int lane = threadIdx.x & 63;
  await(&sh.runs, (n + 1) * kWaves);
  Channels A(1.0f), B(0.0f);
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const int k = kBackward ? kWaves - 1 - i : i;
    B = fma<kChannels>(sh.mapA[n & 1][k][lane], B, sh.mapB[n & 1][k][lane]);
    A *= sh.mapA[n & 1][k][lane];
  }
  if (w.live && !w.last(a)) {
#pragma unroll
    for (int k = 0; k < kChannels; ++k)
      store_word(a.maps + map_row<kBackward>(a, w.b, w.place) + w.c + k,
                 word_of(A[k]) | uint64_t(word_of(B[k])) << 32);
  }
  sh.wholeA[n & 1][lane] = A;
  sh.wholeB[n & 1][lane] = B;
  signal(&sh.whole);
}

// A run's rows of one tensor.  Tokens beyond the sequence repeat its last one;
// what is made of them is neutral or not stored.
template <typename T, int kChannels, int kRun>
struct Rows {
  Vec<T, kChannels> v[kRun];
  __device__ __forceinline__ void load(const void* base, int64_t batch, int64_t token, int64_t b,
                                       int64_t t0, int64_t c, int count, int64_t tokens) {
    const T* p = static_cast<const T*>(base) + b * batch + c;
    if (count == kRun) {
      p += t0 * token;
#pragma unroll
      for (int i = 0; i < kRun; ++i) v[i] = load_channels<T, kChannels>(p + i * token);
    } else {
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        const int64_t t = t0 + i < tokens ? t0 + i : tokens - 1;
        v[i] = load_channels<T, kChannels>(p + t * token);
      }
    }
  }
};

template <typename T, int kChannels>
__global__ __launch_bounds__(kThreads, 4) void scan_fwd_kernel(ScanArgs a) {
  using Channels = FloatVec<kChannels>;
  constexpr int kRun = Shape<false>::kRun;
  __shared__ Shared<kChannels> sh;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (threadIdx.x == 0) {
    sh.ticket[0] = next_ticket(a, 0);
    sh.ticket[1] = sh.ticket[0] < a.items ? next_ticket(a, 1) : a.items;
    sh.runs = sh.whole = 0;
  }
  __syncthreads();
  if (wave == kWaves) {
    look_wave<false, kChannels>(a, sh, a.state);
    return;
  }
  Rows<T, kChannels, kRun> x, g;
  const auto fetch = [&](uint32_t item) {
    if (item >= a.items) return;
    const Item<false, kChannels> w(a, item, wave, lane);
    x.load(a.x, a.x_batch, a.x_token, w.b, w.t0, w.c, w.count, a.tokens);
    g.load(a.gate, a.gate_batch, a.gate_token, w.b, w.t0, w.c, w.count, a.tokens);
  };
  fetch(sh.ticket[0]);
  for (uint32_t n = 0;; ++n) {
    const uint32_t item = sh.ticket[n & 3];
    if (item >= a.items) return;
    const Item<false, kChannels> w(a, item, wave, lane);
    Channels ga[kRun], gb[kRun];  // a and (1 - a) x
#pragma unroll
    for (int i = 0; i < kRun; ++i)
#pragma unroll
      for (int k = 0; k < kChannels; ++k) {
        const Gate gt = gate_of<T>(float(g.v[i][k]));
        ga[i][k] = gt.a;
        gb[i][k] = gt.keep * float(x.v[i][k]);
      }
    fetch(sh.ticket[(n + 1) & 3]);
    if (w.count < kRun) {
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        if (i >= w.count) {
          ga[i] = Channels(1.0f);
          gb[i] = Channels(0.0f);
        }
    }
    Channels A(1.0f), B(0.0f);
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      B = fma<kChannels>(ga[i], B, gb[i]);
      A *= ga[i];
    }
    sh.mapA[n & 1][wave][lane] = A;
    sh.mapB[n & 1][wave][lane] = B;
    signal(&sh.runs);
    if (wave == 0) publish_map<false, kChannels>(a, w, sh, n);
    __syncthreads();
    Channels h = sh.before[n & 1][lane];
    for (int i = 0; i < wave; ++i)
      h = fma<kChannels>(sh.mapA[n & 1][i][lane], h, sh.mapB[n & 1][i][lane]);
    T* py = static_cast<T*>(a.y) + (w.b * a.tokens + w.t0) * a.channels + w.c;
    float* kept = a.ends + end_row<false>(a, w.b, w.place) + w.c;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      // States at the starts of the backward's chunks; the one at this chunk's
      // own start, after place 0, is published by the looking wave.
      const int t = wave * kRun + i;
      static_assert(kStarts == 2);
      if ((t == kStartTokens || (t == 0 && w.place == 0)) && i < w.count && w.live) {
#pragma unroll
        for (int k = 0; k < kChannels; ++k) kept[t / kStartTokens * a.channels + k] = h[k];
      }
      h = fma<kChannels>(ga[i], h, gb[i]);
      if (i < w.count && w.live) store_channels<T, kChannels>(py + i * a.channels, h);
    }
    if (w.count > 0 && w.t0 + w.count == a.tokens && w.live) {
#pragma unroll
      for (int k = 0; k < kChannels; ++k) a.last[w.b * a.channels + w.c + k] = h[k];
    }
  }
}

// Backward, the tokens last to first.  sh.mapA: the runs' gates' products, in both
// directions; sh.mapB: backward maps of the carried gradient; mapH: forward maps of h.
template <typename T, int kChannels>
__global__ __launch_bounds__(kThreads, 4) void scan_bwd_kernel(ScanArgs a) {
  using Channels = FloatVec<kChannels>;
  constexpr int kRun = Shape<true>::kRun;
  __shared__ Shared<kChannels> sh;
  __shared__ Channels mapH[2][kWaves][kWave];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (threadIdx.x == 0) {
    sh.ticket[0] = next_ticket(a, 0);
    sh.ticket[1] = sh.ticket[0] < a.items ? next_ticket(a, 1) : a.items;
    sh.runs = sh.whole = 0;
  }
  __syncthreads();
  if (wave == kWaves) {
    look_wave<true, kChannels>(a, sh, a.grad_last);
    return;
  }
  Rows<T, kChannels, kRun> x, g, d;
  const auto fetch = [&](uint32_t item) {
    if (item >= a.items) return;
    const Item<true, kChannels> w(a, item, wave, lane);
    x.load(a.x, a.x_batch, a.x_token, w.b, w.t0, w.c, w.count, a.tokens);
    g.load(a.gate, a.gate_batch, a.gate_token, w.b, w.t0, w.c, w.count, a.tokens);
    if (a.grad_y)
      d.load(a.grad_y, a.grad_batch, a.grad_token, w.b, w.t0, w.c, w.count, a.tokens);
  };
  if (!a.grad_y) {
#pragma unroll
    for (int i = 0; i < kRun; ++i) d.v[i] = Vec<T, kChannels>(T(0.0f));
  }
  fetch(sh.ticket[0]);
  for (uint32_t n = 0;; ++n) {
    const uint32_t item = sh.ticket[n & 3];
    if (item >= a.items) return;
    const Item<true, kChannels> w(a, item, wave, lane);
    Channels h = load_state<kChannels>(a.starts, map_row<true>(a, w.b, w.place) + w.c);
    Channels ga[kRun], keep[kRun], gap[kRun];  // gap: x, later h_{t-1} - x
    Vec<T, kChannels> dy[kRun];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      dy[i] = d.v[i];
#pragma unroll
      for (int k = 0; k < kChannels; ++k) {
        const Gate gt = gate_of<T>(float(g.v[i][k]));
        ga[i][k] = gt.a;
        keep[i][k] = gt.keep;
        gap[i][k] = float(x.v[i][k]);
      }
    }
    fetch(sh.ticket[(n + 1) & 3]);
    if (w.count < kRun) {
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        if (i >= w.count) {
          ga[i] = Channels(1.0f);
          keep[i] = gap[i] = Channels(0.0f);
          dy[i] = Vec<T, kChannels>(T(0.0f));
        }
    }
    Channels A(1.0f), B(0.0f), R(0.0f);
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      A *= ga[i];
#pragma unroll
      for (int k = 0; k < kChannels; ++k) {
        // Token i's gradient reaches the run's start through a_0 .. a_i.
        R[k] = __builtin_fmaf(A[k], float(dy[i][k]), R[k]);
        B[k] = __builtin_fmaf(ga[i][k], B[k], keep[i][k] * gap[i][k]);
      }
    }
    sh.mapA[n & 1][wave][lane] = A;
    sh.mapB[n & 1][wave][lane] = R;
    mapH[n & 1][wave][lane] = B;
    signal(&sh.runs);
    if (wave == kWaves - 1) publish_map<true, kChannels>(a, w, sh, n);
    // While the looking wave is at work, the states: gap becomes h_{t-1} - x.
    await(&sh.runs, (n + 1) * kWaves);
    for (int i = 0; i < wave; ++i)
      h = fma<kChannels>(sh.mapA[n & 1][i][lane], h, mapH[n & 1][i][lane]);
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const Channels next = fma<kChannels>(ga[i], h, keep[i] * gap[i]);
      gap[i] = h - gap[i];
      h = next;
    }
    __syncthreads();
    Channels r = sh.before[n & 1][lane];
    for (int i = kWaves - 1; i > wave; --i)
      r = fma<kChannels>(sh.mapA[n & 1][i][lane], r, sh.mapB[n & 1][i][lane]);
    const int64_t row = (w.b * a.tokens + w.t0) * a.channels + w.c;
    T* pdx = static_cast<T*>(a.grad_x) + row;
    T* pdg = static_cast<T*>(a.grad_gate) + row;
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i) {
      const Channels G = to_float<T, kChannels>(dy[i]) + r;
      if (i < w.count && w.live) {
        store_channels<T, kChannels>(pdx + i * a.channels, keep[i] * G);
        store_channels<T, kChannels>(pdg + i * a.channels, G * gap[i] * (ga[i] * keep[i]));
      }
      r = ga[i] * G;
    }
    if (a.grad_state && w.t0 == 0 && w.live) {
#pragma unroll
      for (int k = 0; k < kChannels; ++k) a.grad_state[w.b * a.channels + w.c + k] = r[k];
    }
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
  const int64_t i = block_index() * 256 + threadIdx.x;
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

template <bool kBackward>
int64_t chunks_of(int64_t tokens) {
  return (tokens + Shape<kBackward>::kChunk - 1) / Shape<kBackward>::kChunk;
}
int64_t starts_of(int64_t tokens) { return (tokens + kStartTokens - 1) / kStartTokens; }

// Two channels a lane where every row of every tensor allows 4-byte accesses.  us
// forward and backward with two and with one, bfloat16: [1, 160000, 768] 193 and 304,
// 223 and 420; [2, 8160, 1024] 37 and 46, 39 and 57; [1, 2000, 256], of few workgroups,
// 15.5 and 16.4, 14.4 and 14.8.
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
  a.chunks = chunks_of<kBackward>(a.tokens);
  a.starts_count = starts_of(a.tokens);
  const int64_t items = (a.channels + lanes - 1) / lanes * a.chunks * a.batch;
  GS_REQUIRE(items < (int64_t(1) << 31), GS_ERR_OVERFLOW, "scan too large");
  a.items = uint32_t(items);
  int64_t blocks = items;
  if (a.chunks > 1) {
    // One workgroup's waves fill a CU.
    blocks = std::min<int64_t>(items, kComputeUnits);
    const ScanSpace space = scan_space(a.batch, a.chunks, a.channels, kBackward);
    a.ticket = reinterpret_cast<uint32_t*>(workspace + space.ticket);
    a.maps = reinterpret_cast<uint64_t*>(workspace + space.maps);
    if (kBackward) a.ends = reinterpret_cast<float*>(workspace + space.carries);
    GS_TRY(device_flags(s, &a.flags));
    const int64_t maps = a.batch * a.chunks * a.channels * 2;
    const int64_t ends = a.batch * (kBackward ? a.chunks : a.starts_count) * a.channels;
    scan_clear_kernel<<<unsigned(std::min<int64_t>((maps + ends + 255) / 256, 2048)), 256, 0, s>>>(
        reinterpret_cast<uint32_t*>(a.maps), maps, reinterpret_cast<uint32_t*>(a.ends), ends,
        a.ticket);
    GS_TRY(check_launch("gated_scan"));
  }
  return with_lane(type, two, [&](auto v, auto n) {
    using T = decltype(v);
    constexpr int kN = decltype(n)::value;
    if constexpr (kBackward)
      scan_bwd_kernel<T, kN><<<grid_of(blocks), kThreads, 0, s>>>(a);
    else
      scan_fwd_kernel<T, kN><<<grid_of(blocks), kThreads, 0, s>>>(a);
    return check_launch("gated_scan");
  });
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" GS_API int64_t gs_gated_scan_chunks(int64_t tokens) {
  return tokens < 0 ? 0 : starts_of(tokens);
}

extern "C" GS_API size_t gs_gated_scan_workspace_bytes(int64_t batch, int64_t tokens,
                                                       int64_t channels, int32_t backward) {
  if (batch <= 0 || tokens <= 0 || channels <= 0) return 0;
  return scan_space(batch, backward ? chunks_of<true>(tokens) : chunks_of<false>(tokens), channels,
                    backward != 0)
      .bytes;
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
                         <<<grid_of((groups + 255) / 256), 256, 0, as_stream(stream)>>>(
                             static_cast<const T*>(x), static_cast<const T*>(gate), state, groups,
                             static_cast<T*>(y), state_out);
                     return check_launch("gated_scan_step");
                   });
}
