// Attention with a sliding window and visible first tokens, backward.  With
// P_ij = exp(scale q_i . k_j - lse_i) where query i sees key j and 0 elsewhere,
//   delta_i = sum_d grad_out_i out_i,   dP = grad_out V^T,   dS = P (dP - delta),
//   grad_v = P^T grad_out,   grad_q = scale dS K,   grad_k = scale dS^T Q.
// P is computed again from q, k and lse instead of being kept.
//
// Two kernels: one holds a workgroup's keys and walks the queries that see them
// (grad_k, grad_v), one holds queries and walks the keys that they see
// (grad_q).  P and dP are computed twice, 7 products for 5, and in return every
// gradient is added up in registers in a fixed order: no atomics.  Heads that
// share keys are walked one after the other by their keys' workgroup.
//
// The first tokens are seen by every later query.  Their keys' walk, far longer
// than a window, is cut into segments, each a workgroup of its own that leaves
// float32 sums, which a last kernel adds in the order of the segments.  Where there are few keys the other walks are cut too.
// Measured, bfloat16, 40000 tokens, 12 heads of 64 on 4, window 5000: keys 1.51 ms
// (760 TFLOP/s, two waves a SIMD, 232 registers), queries 0.98 ms (880 TFLOP/s,
// three waves); bound as the forward is.  64 keys a wave: 2.57 ms, one wave a SIMD.
//
// P and dS are operands of products in the inputs' type, delta reads the rounded
// out, and outputs are rounded once: relative to 64 bits the gradients are off by
// 0.0025 in bfloat16 and 0.0003 in float16, where a single rounding leaves 0.0017 and
// 0.0002.  Products with each rounding's rest would cost twice.
//
// float16 would lose small values of dS below its normal range and large ones
// above it, as gradients and values come in any size (and P is about one over the
// window): there dS carries a power of two, taken out of the sums in float32.
// |dP - delta| is at most B = 2 max|grad_out_i| max|v_j| over the rows of a sequence
// that share a key head; the power brings B to between 2^13 and 2^15, half of what
// the type holds, so nothing overflows, and what is lost is below 2^-38 of B.  Each
// sequence and key head has its own, so none takes bits of another.  P, grad_v's
// operand and about one at most, carries 2^14 there: a window of a million keys
// leaves probabilities of 2^-20, of which float16 itself keeps four bits.
#include "attention_tile.h"

namespace gs {
namespace {

using namespace att;

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kBlockKeys = 32 * kWaves;     // keys of a workgroup of the first kernel
constexpr int kBlockQueries = 32 * kWaves;  // queries of one of the second

// Rows of the tiles that are walked: halved for float32 to leave registers.
template <typename T, int kDim>
constexpr int kTileRows = sizeof(T) == 2 ? 64 : 32;

struct BackwardArgs {
  Problem p;
  const void* q;
  const void* k;
  const void* v;
  const void* out;
  const void* grad;
  Strides sq, sk, sv, sg;
  const float* lse;
  float* delta;  // [batch, heads, queries]
  // float16, [batch, kv_heads, 2]: the bits of the largest |grad_out_i|^2 and
  // |v_j|^2, of rows that count, without elements that are not finite.
  uint32_t* sizes;
  void* dq;
  void* dk;
  void* dv;
  // The walks of the blocks of keys that hold first tokens are cut into
  // sink_segments, those of the others into segments; more than one leave parts,
  // each [2, kBlockKeys, dim].
  float* parts;
  int sink_blocks, sink_segments, segments;
};

__host__ __device__ inline int key_blocks(const Problem& p) {
  return (p.keys + kBlockKeys - 1) / kBlockKeys;
}
// Parts of one key head, and the place of one among all.
__host__ __device__ inline int64_t parts_per_head(const BackwardArgs& a) {
  return (a.sink_segments > 1 ? int64_t(a.sink_blocks) * a.sink_segments : 0) +
         (a.segments > 1 ? int64_t(key_blocks(a.p) - a.sink_blocks) * a.segments : 0);
}
__device__ __forceinline__ int64_t part_index(const BackwardArgs& a, int b, int kv, int block,
                                              int segment) {
  const int64_t head = (int64_t(b) * a.p.kv_heads + kv) * parts_per_head(a);
  if (block < a.sink_blocks) return head + int64_t(block) * a.sink_segments + segment;
  const int64_t before = a.sink_segments > 1 ? int64_t(a.sink_blocks) * a.sink_segments : 0;
  return head + before + int64_t(block - a.sink_blocks) * a.segments + segment;
}

// The power of two that P carries as an operand.
template <typename T>
constexpr int kProbabilityShift = std::is_same_v<T, f16> ? 14 : 0;

// The power of two that dS carries.
template <typename T>
__device__ __forceinline__ int gradient_shift(const BackwardArgs& a, int b, int kv) {
  if constexpr (std::is_same_v<T, f16>) {
    const uint32_t* sizes = a.sizes + (int64_t(b) * a.p.kv_heads + kv) * 2;
    const uint32_t grad = sizes[0], value = sizes[1];
    // A square below 2^e: B = 2 sqrt(their product) is below 2^(1 + half the sum of
    // the exponents, rounded up).
    if (grad != 0 && value != 0) return 14 - ((int(grad >> 23) + int(value >> 23) - 252 + 1) >> 1);
  }
  return 0;
}

__global__ __launch_bounds__(256) void attention_clear_kernel(uint32_t* words, int64_t count) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i < count) words[i] = 0;
}

// Sum of the finite elements' squares.
__device__ __forceinline__ float square(const Frag<f16>& f) {
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = float(f[e]);
    sum = finite(x) ? sum + x * x : sum;
  }
  return sum;
}
// The rows' squares of a workgroup, of which 16 lanes hold a part each, into the
// largest one.  A maximum does not depend on the order.
__device__ __forceinline__ void note_size(uint32_t* largest, float part, bool counts) {
  __shared__ float tops[4];
#pragma unroll
  for (int s = 8; s > 0; s >>= 1) part += __shfl_xor(part, s, 64);
  part = counts ? part : 0.0f;
#pragma unroll
  for (int s = 32; s > 8; s >>= 1) part = fmaxf(part, __shfl_xor(part, s, 64));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = part;
  __syncthreads();
  if (threadIdx.x != 0) return;
  const uint32_t bits = __float_as_uint(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
  // Most workgroups find a larger one there.
  if (bits > __hip_atomic_load(largest, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT))
    atomicMax(largest, bits);
}

// delta, a workgroup for 16 queries of a head, 16 lanes each; float16: the sizes
// of grad_out's rows and, in the workgroups from row_blocks on, those of v's.
template <typename T>
__global__ __launch_bounds__(256) void attention_delta_kernel(BackwardArgs a, unsigned row_blocks) {
  const Problem& p = a.p;
  const int d = (threadIdx.x & 15) * 8, row = threadIdx.x >> 4;
  const unsigned index = unsigned(block_index());
  if constexpr (std::is_same_v<T, f16>) {
    if (index >= row_blocks) {
      const unsigned at = index - row_blocks, blocks = unsigned(p.keys + 15) / 16;
      if (at >= unsigned(p.batch) * p.kv_heads * blocks) return;
      const int kv = int(at % p.kv_heads), b = int(at / p.kv_heads / blocks);
      const int j = int(at / p.kv_heads % blocks) * 16 + row;
      // Keys that some query sees.
      const bool counts = j < p.length(b) && (j > p.offset() - p.window || j < p.sinks);
      const Frag<T> v = load_global<T>(static_cast<const T*>(a.v) + b * a.sv.batch +
                                           j * a.sv.token + kv * a.sv.head + d,
                                       counts && d < p.dim);
      note_size(a.sizes + (int64_t(b) * p.kv_heads + kv) * 2 + 1, square(v), counts);
      return;
    }
  }
  if (index >= row_blocks) return;
  const unsigned blocks = unsigned(p.queries + 15) / 16;
  const int head = int(index % p.heads), b = int(index / p.heads / blocks);
  const int i = int(index / p.heads % blocks) * 16 + row;
  const int64_t at = (int64_t(b) * p.heads + head) * p.queries + i;
  float sum = 0.0f, size = 0.0f;
  if (i < p.queries && d < p.dim) {
    const Frag<T> o = load_global<T>(static_cast<const T*>(a.out) +
                                         ((int64_t(b) * p.queries + i) * p.heads + head) * p.dim + d,
                                     true);
    const Frag<T> g = load_global<T>(static_cast<const T*>(a.grad) + b * a.sg.batch +
                                         i * a.sg.token + head * a.sg.head + d, true);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += float(o[e]) * float(g[e]);
    if constexpr (std::is_same_v<T, f16>) size = square(g);
  }
  if constexpr (std::is_same_v<T, f16>) {
    // A query that sees nothing has no dS.
    const bool counts = i < p.queries && a.lse[at] != -INFINITY;
    const int kv = head / (p.heads / p.kv_heads);
    note_size(a.sizes + (int64_t(b) * p.kv_heads + kv) * 2, size, counts);
  }
#pragma unroll
  for (int s = 8; s > 0; s >>= 1) sum += __shfl_xor(sum, s, 64);
  if (i < p.queries && (threadIdx.x & 15) == 0) a.delta[at] = sum;
}

// grad_k and grad_v of a workgroup's keys: a wave holds 32, queries walk by.
template <typename T, int kDim>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 && kDim <= 64 ? 2 : 1) void attention_bwd_keys_kernel(
    BackwardArgs a) {
  constexpr int kRows = kTileRows<T, kDim>;
  constexpr int kPitchT = kPitch<T, kDim>;
  constexpr int kSteps = kDim / 16, kBlocks = kDim / 32;
  __shared__ __align__(16) T tiles[2][2][kRows * kPitchT];
  __shared__ float rows[2][2][kRows];  // lse (in powers of two) and delta
  const Problem& p = a.p;
  const int blocks = key_blocks(p);
  // Items of a key head: the segments of the first tokens' blocks, then those of
  // the other blocks.
  const int split = a.sink_blocks * a.sink_segments;
  const int per = split + (blocks - a.sink_blocks) * a.segments;
  const int64_t total = int64_t(per) * p.kv_heads * p.batch;
  const int64_t id = xcd_order(blockIdx.x, total);
  if (id >= total) return;
  const int item = int(id % per);
  const int kv = int(id / per % p.kv_heads), b = int(id / per / p.kv_heads);
  const int pieces = item < split ? a.sink_segments : a.segments;
  const int block = (item < split ? 0 : a.sink_blocks) + (item < split ? item : item - split) / pieces;
  const int segment = (item < split ? item : item - split) % pieces;
  const bool part = pieces > 1;
  const int group = p.heads / p.kv_heads;
  const int length = p.length(b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int k0 = block * kBlockKeys;  // first key of the workgroup
  const int w0 = k0 + wave * 32;      // of the wave
  const int j = w0 + (lane & 31);     // the lane's

  Frag<T> kf[kSteps], vf[kSteps];
  {
    const T* kr = static_cast<const T*>(a.k) + b * a.sk.batch + j * a.sk.token + kv * a.sk.head;
    const T* vr = static_cast<const T*>(a.v) + b * a.sv.batch + j * a.sv.token + kv * a.sv.head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = 16 * s + 8 * (lane >> 5);
      kf[s] = load_global<T>(kr + d, j < length && d < p.dim);
      vf[s] = load_global<T>(vr + d, j < length && d < p.dim);
    }
  }

  // Queries that see any of the keys, and the walk over their tiles, head after
  // head, of which the workgroup takes its segment.
  const int off = p.offset();
  const int from = max(0, k0 - off);
  const int to = k0 >= length ? from
                 : k0 < p.sinks
                     ? p.queries
                     : int(min(int64_t(p.queries), int64_t(k0) + kBlockKeys - 1 + p.window - off));
  const int first_tile = from / kRows;
  const int tiles_per_head = to > from ? (to - 1) / kRows - first_tile + 1 : 0;
  const int64_t walk = int64_t(tiles_per_head) * group;
  const int begin = int(walk * segment / pieces), count = int(walk * (segment + 1) / pieces);

  const int shift = gradient_shift<T>(a, b, kv);
  // P comes out of the exponential with its power of two, and dS with P's.
  const float up = ldexpf(1.0f, shift - kProbabilityShift<T>), down = ldexpf(1.0f, -shift);
  Acc dk[kBlocks], dv[kBlocks];
  Poison<T, kBlocks> pk, pv;
#pragma unroll
  for (int n = 0; n < kBlocks; ++n) dk[n] = dv[n] = Acc(0.0f);
  const float c = p.scale * kLog2e;

  Stage<T, kRows, kDim, kThreads> sq(a.sq.token, p.dim, threadIdx.x),
      sg(a.sg.token, p.dim, threadIdx.x);
  float row_lse = 0.0f, row_delta = 0.0f;
  const auto fetch = [&](int it) {
    const int head = kv * group + it / tiles_per_head;
    const int i0 = (first_tile + it % tiles_per_head) * kRows;
    sq.load(static_cast<const T*>(a.q) + b * a.sq.batch + head * a.sq.head, i0, p.queries);
    sg.load(static_cast<const T*>(a.grad) + b * a.sg.batch + head * a.sg.head, i0, p.queries);
    if (threadIdx.x < kRows) {
      const int i = i0 + threadIdx.x;
      const int64_t at = (int64_t(b) * p.heads + head) * p.queries + i;
      row_lse = i < p.queries ? a.lse[at] * kLog2e - float(kProbabilityShift<T>) : 0.0f;
      row_delta = i < p.queries ? a.delta[at] : 0.0f;
    }
  };
  const auto keep = [&](int buffer) {
    sq.store(tiles[buffer][0]);
    sg.store(tiles[buffer][1]);
    if (threadIdx.x < kRows) {
      rows[buffer][0][threadIdx.x] = row_lse;
      rows[buffer][1][threadIdx.x] = row_delta;
    }
  };
  if (begin < count) {
    fetch(begin);
    keep(begin & 1);
  }
  __syncthreads();
  // One tile of queries.  `full` (known at compile time): every query of it sees
  // all of the wave's keys; otherwise each half looks for itself.
  const auto turn = [&](int it, auto full) {
    if (it + 1 < count) fetch(it + 1);
    const T* qt = tiles[it & 1][0];
    const T* gt = tiles[it & 1][1];
    const int i0 = (first_tile + it % tiles_per_head) * kRows;
    const auto half = [&](int h) {
      const int p0 = off + i0 + 32 * h, p1 = p0 + 31;  // positions
      const bool inside = i0 + 32 * h >= from && i0 + 32 * h + 31 < to;
      const int w1 = w0 + 31;
      const bool any = full || (w0 <= p1 && w0 < length && i0 + 32 * h < to &&
                                (w1 > p0 - p.window || w0 < p.sinks));
      const bool all = full || (inside && w1 <= p0 && w1 < length &&
                                (w0 > p1 - p.window || w1 < p.sinks));
      if (!any) return;
      Acc s(0.0f), dp(0.0f);
#pragma unroll
      for (int st = 0; st < kSteps; ++st)
        mma(load_rows<T>(qt, kPitchT, 32 * h, 16 * st), kf[st], s);
#pragma unroll
      for (int st = 0; st < kSteps; ++st)
        mma(load_rows<T>(gt, kPitchT, 32 * h, 16 * st), vf[st], dp);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = 32 * h + acc_row(r);
        const float lse = rows[it & 1][0][row], delta = rows[it & 1][1][row];
        s[r] = power<T>(s[r] * c - lse);
        dp[r] = s[r] * (dp[r] - delta);
        if constexpr (std::is_same_v<T, f16>) dp[r] *= up;
      }
      if (!all) {
        const QuerySight sight(p, j, i0 + 32 * h + 4 * (lane >> 5), from, to, length);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool see = sight.sees(acc_row_of_half(r));
          s[r] = see ? s[r] : 0.0f;
          dp[r] = see ? dp[r] : 0.0f;
        }
      }
      // Two products that contract over the queries: of a tile's turned rows and
      // the probabilities or their gradients.
      const auto add = [&](const T* tile, const Acc& x, Poison<T, kBlocks>& poison,
                           Acc (&acc)[kBlocks], int st) {
        const Frag<T> xf = acc_frag<T>(x, st);
        Frag<T> f[kBlocks];
#pragma unroll
        for (int n = 0; n < kBlocks; ++n)
          f[n] = load_turned<T>(tile, kPitchT, 32 * h + 16 * st, 32 * n);
        if (!all) {
          const QuerySight sight(p, j, i0 + 32 * h + 16 * st, from, to, length);
          poison.guard(tile, kPitchT, 32 * h + 16 * st, f, xf, [&](int e) { return sight.sees(e); });
        }
#pragma unroll
        for (int n = 0; n < kBlocks; ++n) mma(f[n], xf, acc[n]);
      };
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        add(gt, s, pv, dv, st);
        add(qt, dp, pk, dk, st);
      }
    };
    if constexpr (full) {
#pragma unroll
      for (int h = 0; h < kRows / 32; ++h) half(h);
    } else {
#pragma unroll 1
      for (int h = 0; h < kRows / 32; ++h) half(h);
    }
    if (it + 1 < count) keep((it + 1) & 1);
    __syncthreads();
  };
  const auto full_tile = [&](int it) {
    const int i0 = (first_tile + it % tiles_per_head) * kRows;
    return i0 >= from && i0 + kRows <= to && w0 + 31 <= off + i0 && w0 + 31 < length &&
           (w0 > off + i0 + kRows - 1 - p.window || w0 + 31 < p.sinks);
  };
  // Runs of full tiles in a loop of their own: without branches the compiler
  // lays the products of one half over the exponentials of the other.
  for (int it = begin; it < count;) {
    while (it < count && !full_tile(it)) turn(it++, std::false_type{});
    while (it < count && full_tile(it)) turn(it++, std::true_type{});
  }
  pk.apply(dk);
  pv.apply(dv);
  float* part_at = part ? a.parts + (part_index(a, b, kv, block, segment) * 2 * kBlockKeys +
                                     wave * 32 + (lane & 31)) * p.dim
                        : nullptr;
  if (!part && j >= p.keys) return;
  const int64_t row = ((int64_t(b) * p.keys + j) * p.kv_heads + kv) * p.dim;
#pragma unroll
  for (int n = 0; n < kBlocks; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * n + 8 * g + 4 * (lane >> 5);
      if (d >= p.dim) continue;
      FloatVec<4> x, y;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[r] = dk[n][4 * g + r] * down;
        y[r] = dv[n][4 * g + r] * (1.0f / float(1 << kProbabilityShift<T>));
      }
      if (part) {
        *reinterpret_cast<FloatVec<4>*>(part_at + d) = x;
        *reinterpret_cast<FloatVec<4>*>(part_at + kBlockKeys * p.dim + d) = y;
      } else {
        *reinterpret_cast<Vec<T, 4>*>(static_cast<T*>(a.dk) + row + d) = from_float<T, 4>(x * p.scale);
        *reinterpret_cast<Vec<T, 4>*>(static_cast<T*>(a.dv) + row + d) = from_float<T, 4>(y);
      }
    }
}

// The blocks that left parts: their segments' sums in order.  One thread for
// four elements of [batch, kv_heads, blocks, kBlockKeys, dim], of the blocks from
// `first` on.
template <typename T>
__global__ __launch_bounds__(256) void attention_bwd_join_kernel(BackwardArgs a, int first,
                                                                 int blocks) {
  const Problem& p = a.p;
  const int64_t plane = int64_t(kBlockKeys) * p.dim;
  const int64_t e = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (e >= int64_t(p.batch) * p.kv_heads * blocks * plane) return;
  const int64_t in = e % plane, at = e / plane;
  const int block = first + int(at % blocks);
  const int kv = int(at / blocks % p.kv_heads), b = int(at / blocks / p.kv_heads);
  const int j = block * kBlockKeys + int(in / p.dim);
  if (j >= p.keys) return;
  const float* part = a.parts + part_index(a, b, kv, block, 0) * 2 * plane + in;
  const int pieces = block < a.sink_blocks ? a.sink_segments : a.segments;
  FloatVec<4> dk(0.0f), dv(0.0f);
#pragma unroll 4
  for (int s = 0; s < pieces; ++s) {
    dk += *reinterpret_cast<const FloatVec<4>*>(part + 2 * s * plane);
    dv += *reinterpret_cast<const FloatVec<4>*>(part + (2 * s + 1) * plane);
  }
  const int64_t row = ((int64_t(b) * p.keys + j) * p.kv_heads + kv) * p.dim + in % p.dim;
  *reinterpret_cast<Vec<T, 4>*>(static_cast<T*>(a.dk) + row) = from_float<T, 4>(dk * p.scale);
  *reinterpret_cast<Vec<T, 4>*>(static_cast<T*>(a.dv) + row) = from_float<T, 4>(dv);
}

// grad_q of a wave's 32 queries: what their walk over the keys carries.
template <typename T, int kDim>
struct GradQueries {
  static constexpr int kSteps = kDim / 16, kBlocks = kDim / 32;
  static constexpr int kPitchT = kPitch<T, kDim>;
  Frag<T> q[kSteps], g[kSteps];
  float lse, delta;  // lse in powers of two; P carries dS's power of two
  float factor;      // of the result
  Acc dq[kBlocks];
  Poison<T, kBlocks> poison;
  int first, pos, length;  // position of the wave's first query and of the lane's

  __device__ __forceinline__ GradQueries(const BackwardArgs& a, int b, int head, int query,
                                         int length_)
      : first(a.p.offset() + query), length(length_) {
    const Problem& p = a.p;
    const int lane = threadIdx.x & 63, i = query + (lane & 31);
    pos = p.offset() + i;
    const bool live = i < p.queries;
    const T* qr = static_cast<const T*>(a.q) + b * a.sq.batch + i * a.sq.token + head * a.sq.head;
    const T* gr = static_cast<const T*>(a.grad) + b * a.sg.batch + i * a.sg.token + head * a.sg.head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = 16 * s + 8 * (lane >> 5);
      q[s] = load_global<T>(qr + d, live && d < p.dim);
      g[s] = load_global<T>(gr + d, live && d < p.dim);
    }
    const int64_t at = (int64_t(b) * p.heads + head) * p.queries + i;
    const int shift = gradient_shift<T>(a, b, head / (p.heads / p.kv_heads));
    lse = live ? a.lse[at] * kLog2e - float(shift) : 0.0f;
    delta = live ? a.delta[at] : 0.0f;
    factor = ldexpf(p.scale, -shift);
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) dq[n] = Acc(0.0f);
  }

  // Whether every query sees each of `keys` keys from j0 on.
  __device__ __forceinline__ bool sees_all(const Problem& p, int j0, int keys) const {
    const int last = first + 31, j1 = j0 + keys - 1;
    return j1 <= first && j1 < length && (j0 > last - p.window || j1 < p.sinks);
  }

  // 32 keys from j0 on, rows row0 .. of the LDS tiles kt and vt.  kFull: every
  // query sees all of them.
  template <bool kFull>
  __device__ __forceinline__ void take(const Problem& p, const T* kt, const T* vt, int row0, int j0,
                                       float c) {
    const int lane = threadIdx.x & 63;
    const bool all = kFull || sees_all(p, j0, 32);
    if constexpr (!kFull) {
      if (j0 > first + 31 || j0 >= length || (j0 + 31 <= first - p.window && j0 >= p.sinks)) return;
    }
    Acc s(0.0f), dp(0.0f);
#pragma unroll
    for (int st = 0; st < kSteps; ++st) mma(load_rows<T>(kt, kPitchT, row0, 16 * st), q[st], s);
#pragma unroll
    for (int st = 0; st < kSteps; ++st) mma(load_rows<T>(vt, kPitchT, row0, 16 * st), g[st], dp);
#pragma unroll
    for (int r = 0; r < 16; ++r) dp[r] = power<T>(s[r] * c - lse) * (dp[r] - delta);
    if (!all) {
      const KeySight sight(p, pos, j0 + 4 * (lane >> 5), length);
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] = sight.sees(acc_row_of_half(r)) ? dp[r] : 0.0f;
    }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const Frag<T> df = acc_frag<T>(dp, st);
      Frag<T> f[kBlocks];
#pragma unroll
      for (int n = 0; n < kBlocks; ++n) f[n] = load_turned<T>(kt, kPitchT, row0 + 16 * st, 32 * n);
      if (!all) {
        const KeySight sight(p, pos, j0 + 16 * st, length);
        poison.guard(kt, kPitchT, row0 + 16 * st, f, df, [&](int e) { return sight.sees(e); });
      }
#pragma unroll
      for (int n = 0; n < kBlocks; ++n) mma(f[n], df, dq[n]);
    }
  }
};

// The heads that share keys side by side.
struct QueryPlace {
  int b, kv, head, block;
  __device__ __forceinline__ QueryPlace(const Problem& p, int64_t id, int blocks) {
    const int group = p.heads / p.kv_heads;
    block = int(id / group % blocks);
    kv = int(id / group / blocks % p.kv_heads);
    b = int(id / group / blocks / p.kv_heads);
    head = kv * group + int(id % group);
  }
};

// 128 queries a workgroup, whose waves share tiles of keys in LDS.
template <typename T, int kDim>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 && kDim <= 64 ? 2 : 1) void
attention_bwd_queries_kernel(BackwardArgs a) {
  constexpr int kRows = kTileRows<T, kDim>, kBlocks = kDim / 32;
  __shared__ __align__(16) T tiles[2][2][kRows * kPitch<T, kDim>];
  const Problem& p = a.p;
  const int blocks = (p.queries + kBlockQueries - 1) / kBlockQueries;
  const int64_t id = xcd_order(blockIdx.x, int64_t(blocks) * p.heads * p.batch);
  if (id >= int64_t(blocks) * p.heads * p.batch) return;
  const QueryPlace at(p, id, blocks);
  const int length = p.length(at.b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int query = at.block * kBlockQueries + wave * 32;
  GradQueries<T, kDim> w(a, at.b, at.head, query, length);
  const KeyTiles<kRows> walk(p, at.block * kBlockQueries, kBlockQueries, length);
  const float c = p.scale * kLog2e;
  const T* kbase = static_cast<const T*>(a.k) + at.b * a.sk.batch + at.kv * a.sk.head;
  const T* vbase = static_cast<const T*>(a.v) + at.b * a.sv.batch + at.kv * a.sv.head;
  Stage<T, kRows, kDim, kThreads> sk(a.sk.token, p.dim, threadIdx.x), sv(a.sv.token, p.dim, threadIdx.x);
  const auto fetch = [&](int it) {
    sk.load(kbase, walk.first_key(it), length);
    sv.load(vbase, walk.first_key(it), length);
  };
  if (walk.count > 0) {
    fetch(0);
    sk.store(tiles[0][0]);
    sv.store(tiles[0][1]);
  }
  __syncthreads();
  const auto turn = [&](int it, auto full) {
    if (it + 1 < walk.count) fetch(it + 1);
    const T* kt = tiles[it & 1][0];
    const T* vt = tiles[it & 1][1];
    if constexpr (full) {
#pragma unroll
      for (int h = 0; h < kRows / 32; ++h)
        w.template take<true>(p, kt, vt, 32 * h, walk.first_key(it) + 32 * h, c);
    } else {
#pragma unroll 1
      for (int h = 0; h < kRows / 32; ++h)
        w.template take<false>(p, kt, vt, 32 * h, walk.first_key(it) + 32 * h, c);
    }
    if (it + 1 < walk.count) {
      sk.store(tiles[(it + 1) & 1][0]);
      sv.store(tiles[(it + 1) & 1][1]);
    }
    __syncthreads();
  };
  // Runs of tiles that the wave's queries see whole in a loop of their own.
  for (int it = 0; it < walk.count;) {
    while (it < walk.count && !w.sees_all(p, walk.first_key(it), kRows)) turn(it++, std::false_type{});
    while (it < walk.count && w.sees_all(p, walk.first_key(it), kRows)) turn(it++, std::true_type{});
  }
  w.poison.apply(w.dq);
  const int i = query + (lane & 31);
  if (i >= p.queries) return;
  T* out = static_cast<T*>(a.dq) + ((int64_t(at.b) * p.queries + i) * p.heads + at.head) * p.dim;
#pragma unroll
  for (int n = 0; n < kBlocks; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 32 * n + 8 * e + 4 * (lane >> 5);
      FloatVec<4> x;
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = w.dq[n][4 * e + r] * w.factor;
      if (d < p.dim) *reinterpret_cast<Vec<T, 4>*>(out + d) = from_float<T, 4>(x);
    }
}

// 32 queries a workgroup: every wave has all of them and every fourth tile of 32
// keys, which it loads by itself; the waves' sums are added one after the other.
template <typename T, int kDim>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) void
attention_bwd_queries_split_kernel(BackwardArgs a) {
  constexpr int kKeys = 32, kQueries = 32, kBlocks = kDim / 32;
  __shared__ __align__(16) T tiles[kWaves][2][kKeys * kPitch<T, kDim>];
  __shared__ float joined[32][kDim + 1];
  const Problem& p = a.p;
  const int blocks = (p.queries + kQueries - 1) / kQueries;
  const int64_t id = xcd_order(blockIdx.x, int64_t(blocks) * p.heads * p.batch);
  if (id >= int64_t(blocks) * p.heads * p.batch) return;
  const QueryPlace at(p, id, blocks);
  const int length = p.length(at.b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  GradQueries<T, kDim> w(a, at.b, at.head, at.block * kQueries, length);
  const KeyTiles<kKeys> walk(p, at.block * kQueries, kQueries, length);
  const float c = p.scale * kLog2e;
  const T* kbase = static_cast<const T*>(a.k) + at.b * a.sk.batch + at.kv * a.sk.head;
  const T* vbase = static_cast<const T*>(a.v) + at.b * a.sv.batch + at.kv * a.sv.head;
  Stage<T, kKeys, kDim, kWave> sk(a.sk.token, p.dim, lane), sv(a.sv.token, p.dim, lane);
  const auto fetch = [&](int it) {
    sk.load(kbase, walk.first_key(it), length);
    sv.load(vbase, walk.first_key(it), length);
  };
  if (wave < walk.count) fetch(wave);
  for (int it = wave; it < walk.count; it += kWaves) {
    sk.store(tiles[wave][0]);
    sv.store(tiles[wave][1]);
    if (it + kWaves < walk.count) fetch(it + kWaves);
    wave_sync();
    w.template take<false>(p, tiles[wave][0], tiles[wave][1], 0, walk.first_key(it), c);
    wave_sync();
  }
  w.poison.apply(w.dq);
  for (int k = 0; k < kWaves; ++k) {
    if (wave == k) {
#pragma unroll
      for (int n = 0; n < kBlocks; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float& sum = joined[lane & 31][32 * n + acc_row(r)];
          sum = k ? sum + w.dq[n][r] : w.dq[n][r];
        }
    }
    __syncthreads();
  }
  const int i0 = at.block * kQueries;
  T* out = static_cast<T*>(a.dq) + ((int64_t(at.b) * p.queries + i0) * p.heads + at.head) * p.dim;
  for (int e = threadIdx.x; e < 32 * kDim; e += kThreads) {
    const int row = e / kDim, d = e % kDim;
    if (i0 + row < p.queries && d < p.dim)
      out[int64_t(row) * p.heads * p.dim + d] = T(joined[row][d] * w.factor);
  }
}

template <typename T, int kDim>
void launch_queries(const BackwardArgs& a, hipStream_t s) {
  const auto items = [&](int queries) {
    return (int64_t(a.p.queries) + queries - 1) / queries * a.p.heads * a.p.batch;
  };
  if (items(kBlockQueries) < split_below(a.p.dim))
    attention_bwd_queries_split_kernel<T, kDim>
        <<<unsigned(xcd_grid(items(32))), kThreads, 0, s>>>(a);
  else
    attention_bwd_queries_kernel<T, kDim>
        <<<unsigned(xcd_grid(items(kBlockQueries))), kThreads, 0, s>>>(a);
}

// How the walks are cut.  Where the blocks of keys are fewer than two for each
// CU, into segments of at least two tiles that make up for it, and the first
// tokens' walks into as long ones.  Backward in us, uncut and cut for 256, 512 and
// 1024 workgroups: 4096 tokens, 8 heads of 64 on 2, window 1024 187, 138, 101 and 111;
// 2 x 777, 6 heads of 40 on 2, float32 189, 80, 77 and 77; 1200, 8 heads of 64, window
// 300 47, 42, 42 and 42; 2 x 2500, 8 heads of 128, window 1250 (320 blocks) 212, 212,
// 212 and 231.  Else the first tokens' alone, into segments a
// quarter as long as the others' walks: most of their tiles are masked, and at the
// others' length they end last (40000 tokens: 2.41 ms, 1.81 with a quarter).  The
// first tokens' segments are about 1024 at most over all their blocks, four for
// each CU, which bounds the parts to 128 MiB for heads of 128.  Backward in ms
// with at most 512, 1024, 2048 and without a bound: 40000 tokens, 12 heads of 64 on
// 4, window 64, 2500 first ones 2.51, 2.16, 1.63 and 3.36 (4.6 GiB of parts); 16
// heads of 128, window 300, 1200 first ones 3.94, 3.73, 3.64 and 9.51 (12 GiB); 9600,
// 8 heads of 64, window 1200, 1200 first ones 0.22, 0.25, 0.26 and 0.27.
constexpr int64_t kSinkParts = 1024;

void plan_segments(const Problem& p, int32_t type, BackwardArgs& a) {
  const int64_t blocks = key_blocks(p), rows = type == GS_F32 ? 32 : 64;
  const int64_t group = p.heads / p.kv_heads;
  const int64_t reach = std::min<int64_t>(p.queries, int64_t(p.window) + kBlockKeys);
  const int64_t walk = std::max<int64_t>(1, (reach + rows - 1) / rows * group);
  const int64_t items = std::max<int64_t>(1, blocks * p.kv_heads * p.batch);
  a.segments = int(std::max<int64_t>(1, std::min<int64_t>(512 / items, walk / 2)));
  a.sink_blocks = int(std::min<int64_t>(blocks, (p.sinks + kBlockKeys - 1) / kBlockKeys));
  const int64_t long_walk = (int64_t(p.queries) + rows - 1) / rows * group;
  const int64_t piece = a.segments > 1 ? walk / a.segments : std::max<int64_t>(1, walk / 4);
  const int64_t sink_items = std::max<int64_t>(1, int64_t(a.sink_blocks) * p.kv_heads * p.batch);
  a.sink_segments =
      int(std::max<int64_t>(1, std::min<int64_t>(long_walk / piece, kSinkParts / sink_items)));
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// delta and, behind it, float16's sizes.
size_t delta_bytes(const Problem& p) {
  return align256(size_t(p.batch) * (size_t(p.heads) * size_t(p.queries) + 2 * size_t(p.kv_heads)) *
                  sizeof(float));
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" GS_API size_t gs_window_attention_bwd_workspace_bytes(const gs_attention* desc) {
  if (!desc || check_attention(*desc) != GS_OK) return 0;
  BackwardArgs a{};
  a.p = make_problem(*desc, nullptr);
  const Problem& p = a.p;
  plan_segments(p, desc->type, a);
  return delta_bytes(p) + size_t(p.batch) * size_t(p.kv_heads) * size_t(parts_per_head(a)) * 2 *
                              kBlockKeys * size_t(p.dim) * sizeof(float);
}

extern "C" GS_API int gs_window_attention_bwd(const gs_attention* desc, const void* q,
                                              const void* k, const void* v, const void* out,
                                              const float* lse, const void* grad_out,
                                              const int64_t* strides, const int32_t* lengths,
                                              void* grad_q, void* grad_k, void* grad_v,
                                              void* workspace, size_t workspace_bytes,
                                              void* stream) {
  clear_error();
  GS_REQUIRE(desc, GS_ERR_INVALID_ARGUMENT, "null description");
  GS_TRY(check_attention(*desc));
  if (desc->batch == 0 || (desc->queries == 0 && desc->keys == 0)) return GS_OK;
  GS_REQUIRE(strides, GS_ERR_INVALID_ARGUMENT, "null strides");
  const int64_t none[3] = {0, 0, 0};
  if (desc->queries > 0) {
    GS_TRY(check_rows(q, strides, desc->type, "q"));
    GS_TRY(check_rows(grad_out, strides + 9, desc->type, "grad_out"));
    GS_TRY(check_rows(out, none, desc->type, "out"));
    GS_TRY(check_rows(grad_q, none, desc->type, "grad_q"));
    GS_REQUIRE(lse, GS_ERR_INVALID_ARGUMENT, "null lse");
  }
  if (desc->keys > 0) {
    GS_TRY(check_rows(k, strides + 3, desc->type, "k"));
    GS_TRY(check_rows(v, strides + 6, desc->type, "v"));
    GS_TRY(check_rows(grad_k, none, desc->type, "grad_k"));
    GS_TRY(check_rows(grad_v, none, desc->type, "grad_v"));
  }
  const size_t need = gs_window_attention_bwd_workspace_bytes(desc);
  GS_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), GS_ERR_WORKSPACE,
             "workspace too small: %zu bytes, %zu needed", workspace_bytes, need);
  GS_REQUIRE(seq::aligned_to(workspace, 16), GS_ERR_INVALID_ARGUMENT,
             "workspace must be 16-byte aligned");
  BackwardArgs a{};
  a.p = make_problem(*desc, lengths);
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.grad = grad_out;
  a.sq = {strides[0], strides[1], strides[2]};
  a.sk = {strides[3], strides[4], strides[5]};
  a.sv = {strides[6], strides[7], strides[8]};
  a.sg = {strides[9], strides[10], strides[11]};
  a.lse = lse;
  a.delta = static_cast<float*>(workspace);
  a.dq = grad_q;
  a.dk = grad_k;
  a.dv = grad_v;
  plan_segments(a.p, desc->type, a);
  a.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + delta_bytes(a.p));
  const Problem& p = a.p;
  const int64_t rows = int64_t(p.batch) * p.queries * p.heads;
  a.sizes = reinterpret_cast<uint32_t*>(a.delta + rows);
  const int64_t row_blocks = int64_t(p.batch) * p.heads * ((int64_t(p.queries) + 15) / 16);
  const int64_t value_blocks =
      desc->type == GS_F16 ? int64_t(p.batch) * p.kv_heads * ((int64_t(p.keys) + 15) / 16) : 0;
  const int64_t blocks = key_blocks(p), others = blocks - a.sink_blocks;
  const int64_t key_items = (int64_t(a.sink_blocks) * a.sink_segments + others * a.segments) *
                            p.kv_heads * p.batch;
  // Blocks that leave parts: all, the first tokens' or the others.
  const int join_first = a.sink_segments > 1 ? 0 : a.sink_blocks;
  const int join_blocks = int((a.sink_segments > 1 ? a.sink_blocks : 0) + (a.segments > 1 ? others : 0));
  const int64_t joined = int64_t(p.batch) * p.kv_heads * join_blocks * kBlockKeys * p.dim / 4;
  const hipStream_t s = as_stream(stream);
  return seq::with_type(desc->type, [&](auto t) {
    using T = decltype(t);
    // Without queries the keys' kernel reads them all the same.
    if (std::is_same_v<T, f16>) {
      const int64_t words = int64_t(p.batch) * p.kv_heads * 2;
      attention_clear_kernel<<<unsigned((words + 255) / 256), 256, 0, s>>>(a.sizes, words);
    }
    if (rows) {
      attention_delta_kernel<T>
          <<<grid_of(row_blocks + value_blocks), 256, 0, s>>>(a, unsigned(row_blocks));
      GS_TRY(check_launch("window_attention backward"));
    }
    if (key_items) {
      const unsigned grid = unsigned(xcd_grid(key_items));
      if (p.dim <= 64)
        attention_bwd_keys_kernel<T, 64><<<grid, kThreads, 0, s>>>(a);
      else
        attention_bwd_keys_kernel<T, 128><<<grid, kThreads, 0, s>>>(a);
      GS_TRY(check_launch("window_attention backward, keys"));
    }
    if (joined) {
      attention_bwd_join_kernel<T><<<unsigned((joined + 255) / 256), 256, 0, s>>>(a, join_first,
                                                                                  join_blocks);
      GS_TRY(check_launch("window_attention backward, first tokens"));
    }
    if (rows) {
      if (p.dim <= 64)
        launch_queries<T, 64>(a, s);
      else
        launch_queries<T, 128>(a, s);
    }
    return check_launch("window_attention backward, queries");
  });
}
