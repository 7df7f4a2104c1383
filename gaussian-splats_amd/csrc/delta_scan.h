// Shared pieces of the gated delta rule's kernels.
//
// A head's state is a matrix S [key_dim, dim].  With a = sigmoid(gate) and b =
// sigmoid(beta), a token reads what its key finds, and writes the difference:
//   u_t = b_t (v_t - a_t S_{t-1}^T k_t),  S_t = a_t S_{t-1} + k_t u_t^T,
//   o_t = scale S_t^T q_t.
// In chunks of 64 tokens, with S the state before one, G_i the logarithm of a_1 ..
// a_i and D_ij = e^(G_i - G_j) for j <= i, the updates of a chunk solve a triangular
// system:
//   (I + A) U = b V - (b e^G) K S,   A_ij = b_i D_ij (k_i . k_j) for j < i,
// so with T = (I + A)^-1, W = T (b e^G) K and F = T b V,
//   U = F - W S,   O = scale (e^G Q S + (Q K^T * D) U),
//   S' = e^(G_C) S + K^T (e^(G_C - G) U).
// W and F need no state, O needs no later one: only the second line's U and the
// third line go from chunk to chunk (delta_chain.hip), two products each, and the
// rest runs over all chunks at once.  The backward has the same shape: with P =
// scale Q K^T * D,
//   dU = P^T dO + e^(G_C - G) K dS',   dS = e^(G_C) dS' + scale Q^T e^G dO - W^T dU.
//
// Products run on the matrix cores, whose sums are float32, as are the states that go
// from chunk to chunk.  bfloat16 inputs go in as they are, float16 as a sum of two
// bfloat16 numbers, exactly; any other factor of what states depend on is two as well,
// 16 bits of mantissa and float32's range, with products of two second parts left out:
// the last state is within some 5e-6 (2-norm) where sums in float32 alone leave 1e-7.
// float32 inputs stay in float32, and become three parts in the chain.
//
// bfloat16's outputs and gradients take such factors (states, U, P, dR, ..) in one part,
// and what is kept for their products is kept so, which gives the bits that rounding it
// there would.  They are 0.0026-0.0033 off (2-norm), a rounding of their own alone is
// 0.0017.  With two parts there too they had that: the view stream of 40000 tokens, 12 heads
// of 64 on 4, took 1033 us for 893; 16 sequences of 1024 tokens, 16 heads on 4, forwards and
// backwards, 494 for 414 at 64 x 64 and 1457 for 1101 at 128 x 128.
#pragma once

#include "attention_tile.h"

namespace gs {
namespace delta {

using namespace att;

constexpr int kChunk = 64;
constexpr int kThreads = 256;

// All of the workgroup's writes to LDS are there; loads and stores of global memory
// go on.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Parts of an input, of another factor of what states depend on, and of an output.
template <typename T>
struct Form {
  using Elem = bf16;
  using Store = bf16;
  static constexpr int in = 1, mid = 2, out = 1;
  static constexpr int chain_in = 1, chain = 2;
};
template <>
struct Form<f16> {
  using Elem = bf16;
  using Store = float;
  static constexpr int in = 2, mid = 2, out = 2;
  static constexpr int chain_in = 2, chain = 2;
};
template <>
struct Form<float> {
  using Elem = float;
  using Store = float;
  static constexpr int in = 1, mid = 1, out = 1;
  static constexpr int chain_in = 3, chain = 3;
};

// The parts of N numbers, largest first.
template <typename E, int P, int N>
struct Parts {
  Vec<E, N> v[P];
  __device__ __forceinline__ Parts() {}
  __device__ __forceinline__ explicit Parts(FloatVec<N> x) {
    v[0] = from_float<E, N>(x);
    if constexpr (P > 1) {
#pragma unroll
      for (int i = 1; i < P; ++i) {
        // The number that a bfloat16 is has its bits above sixteen zeros.
        using Words = Vec<uint32_t, N / 2>;
        const Words w = __builtin_bit_cast(Words, v[i - 1]);
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {
          x[2 * k] -= __uint_as_float(w[k] << 16);
          x[2 * k + 1] -= __uint_as_float(w[k] & 0xffff0000u);
        }
        v[i] = from_float<E, N>(x);
      }
    }
  }
};

template <typename E, int PA, int PB>
__device__ __forceinline__ void mma_parts(const Parts<E, PA, 8>& a, const Parts<E, PB, 8>& b, Acc& c) {
#pragma unroll
  for (int i = 0; i < PA; ++i)
#pragma unroll
    for (int j = 0; j < PB; ++j)
      if (i + j < (PA > PB ? PA : PB)) mma(a.v[i], b.v[j], c);
}

// Columns n0 + (lane & 31) of a tile, its rows k0 + 8 (lane >> 5) .. + 7: what
// load_rows gives of the turned tile.
template <typename T>
__device__ __forceinline__ Frag<T> load_cols(const T* tile, int pitch, int k0, int n0) {
  const int lane = threadIdx.x & 63;
  if constexpr (sizeof(T) == 2) {
    using Short4 = Vec<short, 4>;
    using Lds = __attribute__((address_space(3))) Short4*;
    const T* p = tile + (k0 + 8 * (lane >> 5) + ((lane & 15) >> 2)) * pitch + n0 +
                 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const Short4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(p));
    const Short4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(p + 4 * pitch));
    return __builtin_bit_cast(Frag<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    const T* p = tile + (k0 + 8 * (lane >> 5)) * pitch + n0 + (lane & 31);
    Frag<T> f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = p[i * pitch];
    return f;
  }
}

// A [kRows, kWide] matrix in LDS, a tile for each part.
template <typename E, int P, int kRows, int kWide>
struct Tile {
  static constexpr int pitch = kWide + 16 / int(sizeof(E));
  static constexpr int part = kRows * pitch;
  static constexpr int bytes = P * part * int(sizeof(E));
  E* p;

  __device__ __forceinline__ explicit Tile(char* at) : p(reinterpret_cast<E*>(at)) {}
  __device__ __forceinline__ Parts<E, P, 8> rows(int row0, int k0) const {
    Parts<E, P, 8> f;
#pragma unroll
    for (int i = 0; i < P; ++i) f.v[i] = load_rows<E>(p + i * part, pitch, row0, k0);
    return f;
  }
  __device__ __forceinline__ Parts<E, P, 8> cols(int k0, int n0) const {
    Parts<E, P, 8> f;
#pragma unroll
    for (int i = 0; i < P; ++i) f.v[i] = load_cols<E>(p + i * part, pitch, k0, n0);
    return f;
  }
  template <int N>
  __device__ __forceinline__ void put(int row, int col, const Parts<E, P, N>& v) const {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      E* at = p + i * part + row * pitch + col;
      if constexpr (N * sizeof(E) > 16) {
        *reinterpret_cast<Vec<E, 4>*>(at) = __builtin_shufflevector(v.v[i], v.v[i], 0, 1, 2, 3);
        *reinterpret_cast<Vec<E, 4>*>(at + 4) = __builtin_shufflevector(v.v[i], v.v[i], 4, 5, 6, 7);
      } else {
        *reinterpret_cast<Vec<E, N>*>(at) = v.v[i];
      }
    }
  }
  __device__ __forceinline__ float get(int row, int col) const {
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < P; ++i) x += float(p[i * part + row * pitch + col]);
    return x;
  }
  // Four numbers of a row.
  __device__ __forceinline__ FloatVec<4> get4(int row, int col) const {
    FloatVec<4> x(0.0f);
#pragma unroll
    for (int i = 0; i < P; ++i)
      x += to_float<E, 4>(*reinterpret_cast<const Vec<E, 4>*>(p + i * part + row * pitch + col));
    return x;
  }
};

// Calls f(s) for N steps of a contraction, unrolled: all reads of LDS can be ahead of
// the products.
template <int N, typename F>
__device__ __forceinline__ void steps(F&& f) {
#pragma unroll
  for (int s = 0; s < N; ++s) f(s);
}
// Rows 0 .. 31 of a lower triangle of 64 have 32 columns, rows 32 .. 63 all of them.
template <typename F>
__device__ __forceinline__ void steps_to(int row0, F&& f) {
  if (row0)
    steps<4>(f);
  else
    steps<2>(f);
}
// Columns 0 .. 31 have all rows, columns 32 .. 63 the rows from 32 on.
template <typename F>
__device__ __forceinline__ void steps_from(int col0, F&& f) {
  if (col0)
    steps<2>([&](int s) { f(s + 2); });
  else
    steps<4>(f);
}

// Four consecutive numbers of a 32 x 32 result's column, the s-th of four.
__device__ __forceinline__ FloatVec<4> four(const Acc& c, int s) {
  return FloatVec<4>{c[4 * s], c[4 * s + 1], c[4 * s + 2], c[4 * s + 3]};
}
__device__ __forceinline__ int four_row(int s) { return 8 * s + 4 * (int(threadIdx.x & 63) >> 5); }

// Rows 0 .. kRows - 1 of a matrix on their way through the workgroup's registers into
// a tile, zeros from row `rows` and column `wide` on.  Loading and storing are apart, so
// that all matrices of a phase, and those of the next, are on their way at once: a
// kernel of short phases waits for memory once instead of once a matrix (gradients of
// 40000 tokens, 12 heads of 64: 523 us one matrix after the other, 421 so).
template <typename T, int kRows, int kWide>
struct Fetch {
  static constexpr int kPerRow = kWide / 8, kCount = kRows * kPerRow / kThreads;
  static_assert(kRows * kPerRow % kThreads == 0, "whole chunks");
  Frag<T> x[kCount];

  static __device__ __forceinline__ int row(int i) { return (i * kThreads + int(threadIdx.x)) / kPerRow; }
  static __device__ __forceinline__ int col(int i) { return (i * kThreads + int(threadIdx.x)) % kPerRow * 8; }
  // T of a chunk: its upper right quarter is zeros.
  __device__ __forceinline__ void load_triangle(const T* from) {
#pragma unroll
    for (int i = 0; i < kCount; ++i)
      x[i] = load_global<T>(from + row(i) * kWide + col(i), row(i) >= kRows / 2 || col(i) < kWide / 2);
  }
  __device__ __forceinline__ void load(const T* from, int64_t stride, int rows, int wide) {
#pragma unroll
    for (int i = 0; i < kCount; ++i)
      x[i] = load_global<T>(from + row(i) * stride + col(i), row(i) < rows && col(i) < wide);
  }
  // Calls f(row, col, numbers) for what is kept of eight.
  template <typename E, int P, typename F>
  __device__ __forceinline__ void put(const Tile<E, P, kRows, kWide>& tile, F&& f) const {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      if constexpr (std::is_same_v<T, E> && P == 1) {
        Parts<E, 1, 8> one;
        one.v[0] = x[i];
        f(row(i), col(i), one.v[0]);
        tile.put(row(i), col(i), one);
      } else {
        FloatVec<8> y = to_float<T, 8>(x[i]);
        f(row(i), col(i), y);
        tile.put(row(i), col(i), Parts<E, P, 8>(y));
      }
    }
  }
  template <typename E, int P>
  __device__ __forceinline__ void put(const Tile<E, P, kRows, kWide>& tile) const {
    put(tile, [](int, int, auto&) {});
  }
};

// Numbers of a chunk's tokens that all products take.
struct alignas(16) Gates {
  float beta[kChunk];             // b
  float hi[kChunk], lo[kChunk];   // G in powers of two, as a sum
  float up[kChunk], down[kChunk]; // e^G, e^(G_C - G)
  float fade[kChunk], rest[kChunk];  // 1 - a, 1 - b
  float whole;                    // e^(G_C)
  int bad;  // the first token with a number that is not finite; kChunk: none
  // D_ij of j .. j + 3, a multiple of four.
  __device__ __forceinline__ FloatVec<4> decay(int i, int j) const {
    const FloatVec<4> h = *reinterpret_cast<const FloatVec<4>*>(hi + j);
    const FloatVec<4> l = *reinterpret_cast<const FloatVec<4>*>(lo + j);
    const float high = hi[i], low = lo[i];
    FloatVec<4> d;
#pragma unroll
    for (int r = 0; r < 4; ++r) d[r] = __builtin_amdgcn_exp2f((high - h[r]) + (low - l[r]));
    return d;
  }
};

// log2 of sigmoid(x); below -300 it is no longer told from a state that is gone.
__device__ __forceinline__ float log2_sigmoid(float x) {
  return fmaxf(kLog2e * (fminf(x, 0.0f) - log1pf(expf(-fabsf(x)))), -300.0f);
}
__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }

struct Problem {
  int batch, tokens, heads, key_heads, key_dim, dim, chunks;
  float scale;
  const int32_t* lengths;

  __device__ __forceinline__ int length(int b) const {
    return lengths ? min(max(lengths[b], 0), tokens) : tokens;
  }
};

// A workgroup's chunk of one head.
struct Place {
  int b, h, c, key_head, t0, rows, valid;  // rows that exist, rows of the sequence
  int64_t id;
  __device__ __forceinline__ Place(const Problem& p, int64_t index) : id(index) {
    c = int(index % p.chunks);
    const int64_t head = index / p.chunks;
    h = int(head % p.heads);
    b = int(head / p.heads);
    key_head = int(int64_t(h) * p.key_heads / p.heads);
    t0 = c * kChunk;
    rows = min(p.tokens - t0, kChunk);
    valid = max(0, min(p.length(b) - t0, kChunk));
  }
};

template <typename T>
struct Rows {
  const T* p;
  Strides s;
  __device__ __forceinline__ const T* at(int b, int t, int h) const {
    return p + b * s.batch + t * s.token + h * s.head;
  }
};

// The gates on their way: a kernel loads them before its tiles, which they would else
// wait behind.
struct GatePair {
  float gate, beta;
  template <typename T>
  __device__ __forceinline__ GatePair(const Rows<T>& g, const Rows<T>& b, const Place& at)
      : gate(INFINITY), beta(-INFINITY) {
    const int lane = threadIdx.x & 63;
    if (lane < at.valid) {
      gate = float(*g.at(at.b, at.t0 + lane, at.h));
      beta = float(*b.at(at.b, at.t0 + lane, at.h));
    }
  }
  // By one wave, a lane a token.  The sums are float64: differences of far tokens'
  // logarithms keep their bits.
  __device__ __forceinline__ void put(Gates& g) const {
    const int lane = threadIdx.x & 63;
    const bool bad = gate != gate || beta != beta;
    double total = bad ? 0.0 : double(log2_sigmoid(gate));
#pragma unroll
    for (int d = 1; d < kChunk; d <<= 1) {
      const double before = __shfl_up(total, d, kChunk);
      if (lane >= d) total += before;
    }
    const double last = __shfl(total, kChunk - 1, kChunk);
    g.beta[lane] = bad ? 0.0f : sigmoid(beta);
    g.hi[lane] = float(total);
    g.lo[lane] = float(total - double(float(total)));
    g.up[lane] = __builtin_amdgcn_exp2f(float(total));
    g.down[lane] = __builtin_amdgcn_exp2f(float(last - total));
    g.fade[lane] = sigmoid(-gate);
    g.rest[lane] = sigmoid(-beta);
    const uint64_t marks = __ballot(bad);
    if (lane == 0) {
      g.whole = __builtin_amdgcn_exp2f(float(last));
      g.bad = marks ? __builtin_ctzll(marks) : kChunk;
    }
  }
};

// What is kept between the kernels, one after the other for each chunk of each
// head; widths padded to kKey and kDim.  A column lies together: the chain's lanes
// have one, with consecutive rows in their registers.
// What products take in one bfloat16 part is kept so (Form's Store).
struct Kept {
  float* solve;   // [64, 64]: T, or null; its upper right quarter is not written
  void* starts;   // [kDim, kKey]: the state before the chunk, turned
  void* updates;  // [kDim, 64]: U, turned
};

// Where four elements of a row, from column `col` on, lie in a first operand of 16 x 16
// results: fragments of 16 rows and 32 columns, `steps` of them beside each other,
// each in the order of the lanes, whose group g has columns 4 g .. + 3 and 16 + 4 g ..
// + 3 of it.
__device__ __forceinline__ int fragment_at(int row, int col, int steps) {
  return ((row >> 4) * steps + (col >> 5)) * 512 + ((row & 15) + 16 * ((col & 15) >> 2)) * 8 +
         ((col & 16) >> 2);
}

// Factors of the chain, a chunk of a head each.
struct Chain {
  bf16* left;      // parts of [64, kKey], in fragments
  bf16* right;     // parts of [kKey, 64], in fragments
  float* factors;  // 64 of e^(G_C - G), then e^(G_C) and the first token that is not finite
};
constexpr int kFactors = kChunk + 4;

int64_t padded(int dim);

// The chain over the chunks of every head (delta_chain.hip).
struct ChainArgs {
  int64_t heads;  // of all sequences
  int chunks, key_dim, dim;
  Chain chain;
  const float* first;  // the state before the first chunk [heads, key_dim, dim], or null
  int group;                 // heads that share keys
  const float* rows_from;    // [kDim, 64] a chunk: what the rows start with
  void* rows;                // the rows, float32 or (forward) Form's Store; may be rows_from
  const float* states_from;  // [kDim, kKey] a chunk: what the next state starts with (backward)
  void* states;              // the state before the chunk, Form's Store; may be states_from
  float* last;         // the state behind the last chunk, or null
  // Cut sequences: what each segment maps a state to, in fragments, and what it adds
  // [kDim, kKey].
  int segments;
  bf16* maps;
  float* adds;
  int each, blocks;  // chunks of a segment, blocks of columns (the launch's)
};
int chain_segments(int64_t heads, int64_t chunks, int dim);
int launch_chain(const ChainArgs& a, int key_wide, int wide, int parts_in, bool backward,
                 hipStream_t s);

}  // namespace delta
}  // namespace gs
