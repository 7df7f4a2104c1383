// The gated delta rule over a sequence, forward (delta_scan.h has the formulas):
// a workgroup a chunk of a head prepares T, W and F, the chain runs over the
// chunks, a workgroup a chunk gives the outputs.
//
// T, the inverse of a unit lower triangle of 64, is built of blocks of 16: those on
// the diagonal by substitution, a lane a column, the others from T_ij = -T_ii sum_k
// A_ik T_kj, one diagonal after the other, with float32 products.  A token that is
// not finite is taken out of its chunk and leaves its mark instead: from it on, and
// in all later chunks, outputs and states are NaN; products with zeros of a triangle
// would carry it to tokens before it.
//
// Measured, 40000 tokens, 12 heads of 64 on 4, bfloat16: 132 us to prepare (with three
// workgroups a CU, LDS used twice; 186 with two), 73 the outputs, and the chain.  The
// inverse's short dependent steps bound the first, the reads of states the second.
#include "delta_scan.h"

namespace gs {
namespace delta {
namespace {

template <typename T>
struct ForwardArgs {
  Problem p;
  Rows<T> q, k, v, gate, beta;
  Kept kept;
  float* free;  // [kDim, 64] a chunk: F turned
  Chain chain;
  T* out;
  int64_t count;  // chunks of all heads
  int segments;   // of the chain, with its scratch
  bf16* maps;
  float* adds;
};

constexpr int kPitchA = kChunk + 4;

// T_ij of the block (i, j), i > j, 16 x 16 each: a lane has column lane & 15 and rows
// 4 (lane >> 4) .. + 3 of a result, and the products contract over those rows in the
// order of the registers, so the sum is the second product's operand as it stands.
__device__ __forceinline__ void solve_block(const float* a, float* t, int i, int j) {
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  FloatVec<4> sum(0.0f);
  for (int k = j; k < i; ++k) {
    const FloatVec<4> left = *reinterpret_cast<const FloatVec<4>*>(a + (16 * i + m) * kPitchA + 16 * k + 4 * g);
#pragma unroll
    for (int s = 0; s < 4; ++s)
      sum = __builtin_amdgcn_mfma_f32_16x16x4f32(left[s], t[(16 * k + 4 * g + s) * kPitchA + 16 * j + m],
                                                 sum, 0, 0, 0);
  }
  const FloatVec<4> left = *reinterpret_cast<const FloatVec<4>*>(t + (16 * i + m) * kPitchA + 16 * i + 4 * g);
  FloatVec<4> out(0.0f);
#pragma unroll
  for (int s = 0; s < 4; ++s) out = __builtin_amdgcn_mfma_f32_16x16x4f32(left[s], sum[s], out, 0, 0, 0);
#pragma unroll
  for (int s = 0; s < 4; ++s) t[(16 * i + 4 * g + s) * kPitchA + 16 * j + m] = -out[s];
}

// T of A's strictly lower part; its upper blocks beside the diagonal become zeros.
__device__ __forceinline__ void solve_triangle(const float* a, float* t) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (wave == 0) {
    const int block = 16 * (lane >> 4), c = lane & 15;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float y = i == c ? 1.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < i; ++j) y -= a[(block + i) * kPitchA + block + j] * x[j];
      x[i] = y;
      t[(block + i) * kPitchA + block + c] = y;
    }
  } else if (wave == 1) {
    // The blocks (0, 1) and (2, 3), which products over 32 columns read.
    const int block = 32 * (lane >> 5), c = lane & 31;
#pragma unroll
    for (int i = 0; i < 8; ++i) t[(block + 2 * i + (c >> 4)) * kPitchA + block + 16 + (c & 15)] = 0.0f;
  }
  lds_barrier();
  for (int d = 1; d < 4; ++d) {
    if (wave < 4 - d) solve_block(a, t, d + wave, wave);
    lds_barrier();
  }
}

// Rows m0 + (lane & 31), columns k0 + 8 (lane >> 5) .. + 7 of T, times by[column].
template <typename E, int P>
__device__ __forceinline__ Parts<E, P, 8> solve_rows(const float* t, int m0, int k0, const float* by) {
  const int lane = threadIdx.x & 63, k = k0 + 8 * (lane >> 5);
  const float* row = t + (m0 + (lane & 31)) * kPitchA + k;
  const FloatVec<4> lo = *reinterpret_cast<const FloatVec<4>*>(row);
  const FloatVec<4> hi = *reinterpret_cast<const FloatVec<4>*>(row + 4);
  FloatVec<8> x = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= by[k + i];
  return Parts<E, P, 8>(x);
}

template <typename T, int kKey, int kDim>
__global__ __launch_bounds__(kThreads) void delta_prepare_kernel(ForwardArgs<T> a) {
  using M = Form<T>;
  using E = typename M::Elem;
  using KTile = Tile<E, M::in, kChunk, kKey>;
  // The values take the place of A, once T is there, 64 columns at a time: three
  // workgroups of 64 x 64 share a CU in bfloat16, two of 128 x 128 in every type
  // (float16, 4096 chunks: 176 us, 235 with all columns at once and one).
  using VTile = Tile<E, M::in, kChunk, 64>;
  constexpr int kSystem = kChunk * kPitchA * int(sizeof(float));
  __shared__ __align__(16) char k_space[KTile::bytes];
  __shared__ __align__(16) char v_space[kSystem > VTile::bytes ? kSystem : VTile::bytes];
  __shared__ __align__(16) float solve[kChunk * kPitchA];
  __shared__ float by_key[kChunk], by_value[kChunk];
  __shared__ Gates g;
  const int64_t index = seq::block_index();
  if (index >= a.count) return;
  const Place at(a.p, index);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const KTile k(k_space);
  const VTile v(v_space);
  float* system = reinterpret_cast<float*>(v_space);
  const GatePair gates(a.gate, a.beta, at);
  Fetch<T, kChunk, kKey> k_in;
  Fetch<T, kChunk, 64> v_in[kDim / 64];
  k_in.load(a.k.at(at.b, at.t0, at.key_head), a.k.s.token, at.valid, a.p.key_dim);
#pragma unroll
  for (int t = 0; t < kDim / 64; ++t)
    v_in[t].load(a.v.at(at.b, at.t0, at.h) + 64 * t, a.v.s.token, at.valid, a.p.dim - 64 * t);
  if (wave == 0) gates.put(g);
  lds_barrier();
  const auto mark = [&](int row, int, auto& x) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) bad |= !finite(float(x[i]));
    if (__builtin_expect(bad, 0)) {
      x = {};
      atomicMin(&g.bad, row);
    }
  };
  k_in.put(k, mark);
#pragma unroll
  for (int t = 0; t < kDim / 64; ++t)
#pragma unroll
    for (int i = 0; i < v_in[t].kCount; ++i) mark(v_in[t].row(i), 0, v_in[t].x[i]);
  if (threadIdx.x < kChunk) {
    by_value[threadIdx.x] = g.beta[threadIdx.x];
    by_key[threadIdx.x] = -g.beta[threadIdx.x] * g.up[threadIdx.x];
  }
  lds_barrier();
  // A: a wave each for the blocks of 32 on and below the diagonal; a lane has a row
  // i and the columns of its registers.
  if (wave < 3) {
    const int i0 = wave ? 32 : 0, j0 = wave == 2 ? 32 : 0;
    Acc c(0.0f);
#pragma unroll
    for (int s = 0; s < kKey / 16; ++s) mma_parts(k.rows(j0, 16 * s), k.rows(i0, 16 * s), c);
    const int i = i0 + (lane & 31);
    const float b = g.beta[i];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int j = j0 + four_row(s);
      FloatVec<4> x = four(c, s) * g.decay(i, j);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = j + r < i ? b * x[r] : 0.0f;
      *reinterpret_cast<FloatVec<4>*>(system + i * kPitchA + j) = x;
    }
  }
  lds_barrier();
  solve_triangle(system, solve);
  v_in[0].put(v);
  lds_barrier();
  if (a.kept.solve) {
    float* to = a.kept.solve + index * kChunk * kChunk;
#pragma unroll
    for (int s = 0; s < kChunk * kChunk / 4 / kThreads; ++s) {
      const int e = (s * kThreads + int(threadIdx.x)) * 4, row = e / kChunk, col = e % kChunk;
      if (row >= 32 || col < 32)
        *reinterpret_cast<FloatVec<4>*>(to + e) = *reinterpret_cast<const FloatVec<4>*>(solve + row * kPitchA + col);
    }
  }
  // -W: a lane has a token and consecutive columns in its registers.
  const int m0 = 32 * (wave & 1), token = m0 + (lane & 31);
  bf16* left = a.chain.left + index * M::chain * kChunk * kKey;
#pragma unroll
  for (int t = 0; t < kKey / 64; ++t) {
    const int n0 = 32 * ((wave >> 1) + 2 * t);
    Acc c(0.0f);
    steps_to(m0, [&](int s) {
      mma_parts(k.cols(16 * s, n0), solve_rows<E, M::mid>(solve, m0, 16 * s, by_key), c);
    });
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const Parts<bf16, M::chain, 4> x(four(c, s));
#pragma unroll
      for (int i = 0; i < M::chain; ++i)
        *reinterpret_cast<Vec<bf16, 4>*>(left + i * kChunk * kKey +
                                         fragment_at(token, n0 + four_row(s), kKey / 32)) = x.v[i];
    }
  }
  // F turned: a lane has a column and consecutive tokens.
  float* rows = a.free + index * kChunk * kDim;
#pragma unroll
  for (int t = 0; t < kDim / 64; ++t) {
    const int n0 = 32 * (wave >> 1);
    if (t) {
      lds_barrier();
      v_in[t].put(v);
      lds_barrier();
    }
    Acc c(0.0f);
    steps_to(m0, [&](int s) {
      mma_parts(solve_rows<E, M::mid>(solve, m0, 16 * s, by_value), v.cols(16 * s, n0), c);
    });
#pragma unroll
    for (int s = 0; s < 4; ++s)
      *reinterpret_cast<FloatVec<4>*>(rows + (64 * t + n0 + (lane & 31)) * kChunk + m0 + four_row(s)) = four(c, s);
  }
  // K turned, once for the heads that share it.
  const int group = a.p.heads / a.p.key_heads;
  bf16* right = a.chain.right + ((int64_t(at.b) * a.p.key_heads + at.key_head) * a.p.chunks + at.c) *
                                    M::chain_in * kKey * kChunk;
  for (int e = at.h % group ? kKey : wave; e < kKey / 32 * 4; e += 4) {
    const int n0 = 32 * (e / 4), t0 = 16 * (e % 4);
    FloatVec<8> x(0.0f);
    const Parts<E, M::in, 8> f = k.cols(t0, n0);
#pragma unroll
    for (int i = 0; i < M::in; ++i) x += to_float<E, 8>(f.v[i]);
    const Parts<bf16, M::chain_in, 8> y(x);
    const int row = n0 + (lane & 31), col = t0 + 8 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < M::chain_in; ++i) {
      bf16* to = right + i * kKey * kChunk;
      *reinterpret_cast<Vec<bf16, 4>*>(to + fragment_at(row, col, 2)) =
          __builtin_shufflevector(y.v[i], y.v[i], 0, 1, 2, 3);
      *reinterpret_cast<Vec<bf16, 4>*>(to + fragment_at(row, col + 4, 2)) =
          __builtin_shufflevector(y.v[i], y.v[i], 4, 5, 6, 7);
    }
  }
  float* factors = a.chain.factors + index * kFactors;
  if (threadIdx.x < kChunk) factors[threadIdx.x] = g.down[threadIdx.x];
  if (threadIdx.x == 0) {
    // A state that has met a token that is not finite.
    factors[kChunk] = g.bad < kChunk ? __builtin_nanf("") : g.whole;
    factors[kChunk + 1] = float(g.bad);
  }
}

// Q and K are in LDS for P = Q K^T alone; then Q's rows are in registers, and the
// state's columns, U and P take the place, so that two workgroups share a CU in every
// type and size (float16 heads of 128: 177 us for 4096 chunks, 268 with one).
template <typename T, int kKey, int kDim>
__global__ __launch_bounds__(kThreads, 2) void delta_output_kernel(ForwardArgs<T> a) {
  using M = Form<T>;
  using E = typename M::Elem;
  using KTile = Tile<E, M::in, kChunk, kKey>;
  using STile = Tile<E, M::out, 64, kKey>;  // 64 columns of the state, turned
  using UTile = Tile<E, M::out, 64, kChunk>;
  using PTile = Tile<E, M::out, kChunk, kChunk>;
  constexpr int kFirst = 2 * KTile::bytes, kThen = STile::bytes + UTile::bytes + PTile::bytes;
  __shared__ __align__(16) char space[kFirst > kThen ? kFirst : kThen];
  __shared__ Gates g;
  const int64_t index = seq::block_index();
  if (index >= a.count) return;
  const Place at(a.p, index);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const KTile q(space), k(space + KTile::bytes);
  const STile state(space);
  const UTile u(space + STile::bytes);
  const PTile p(space + STile::bytes + UTile::bytes);
  const GatePair gates(a.gate, a.beta, at);
  using Store = typename M::Store;
  const Store* starts = static_cast<const Store*>(a.kept.starts) + index * kKey * kDim;
  const Store* updates = static_cast<const Store*>(a.kept.updates) + index * kChunk * kDim;
  Fetch<T, kChunk, kKey> q_in, k_in;
  Fetch<Store, 64, kKey> state_in;
  Fetch<Store, 64, kChunk> u_in;
  const auto fetch = [&](int d0) {
    state_in.load(starts + d0 * kKey, kKey, a.p.dim - d0, a.p.key_dim);
    u_in.load(updates + d0 * kChunk, kChunk, a.p.dim - d0, kChunk);
  };
  q_in.load(a.q.at(at.b, at.t0, at.key_head), a.q.s.token, at.valid, a.p.key_dim);
  k_in.load(a.k.at(at.b, at.t0, at.key_head), a.k.s.token, at.valid, a.p.key_dim);
  fetch(0);
  if (wave == 0) gates.put(g);
  q_in.put(q);
  k_in.put(k, [](int, int, auto& x) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = finite(float(x[i])) ? x[i] : decltype(x[i] + x[i])(0.0f);
  });
  lds_barrier();
  const int m0 = 32 * (wave & 1), token = m0 + (lane & 31), n0 = 32 * (wave >> 1);
  Parts<E, M::in, 8> own[kKey / 16];
#pragma unroll
  for (int s = 0; s < kKey / 16; ++s) own[s] = q.rows(m0, 16 * s);
  // P = scale Q K^T * D.
  {
    const int i0 = wave ? 32 : 0, j0 = wave == 2 ? 32 : 0;
    Acc c(0.0f);
    if (wave < 3) {
#pragma unroll
      for (int s = 0; s < kKey / 16; ++s) mma_parts(k.rows(j0, 16 * s), q.rows(i0, 16 * s), c);
    }
    lds_barrier();
    const int i = i0 + (lane & 31);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int j = j0 + four_row(s);
      FloatVec<4> x = four(c, s) * g.decay(i, j);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = j + r <= i ? a.p.scale * x[r] : 0.0f;
      if (wave < 3) p.put(i, j, Parts<E, M::out, 4>(x));
    }
  }
  const float up = a.p.scale * g.up[token];
  const bool bad = token >= int(a.chain.factors[index * kFactors + kChunk + 1]);
  T* out = a.out + ((int64_t(at.b) * a.p.tokens + at.t0 + token) * a.p.heads + at.h) * a.p.dim;
#pragma unroll
  for (int d0 = 0; d0 < kDim; d0 += 64) {
    if (d0 >= a.p.dim) break;
    if (d0) lds_barrier();
    state_in.put(state);
    u_in.put(u);
    if (d0 + 64 < a.p.dim) fetch(d0 + 64);
    lds_barrier();
    Acc c(0.0f);
#pragma unroll
    for (int s = 0; s < kKey / 16; ++s) mma_parts(state.rows(n0, 16 * s), own[s], c);
    c *= up;
    steps_to(m0, [&](int s) { mma_parts(u.rows(n0, 16 * s), p.rows(m0, 16 * s), c); });
    if (token < at.rows) {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int n = d0 + n0 + four_row(s);
        FloatVec<4> x = four(c, s);
        if (bad) x = FloatVec<4>(__builtin_nanf(""));
        if (token >= at.valid) x = FloatVec<4>(0.0f);
        if (n < a.p.dim) *reinterpret_cast<Vec<T, 4>*>(out + n) = from_float<T, 4>(x);
      }
    }
  }
}

template <typename T, int kKey, int kDim>
int forward(const ForwardArgs<T>& a, const float* state, float* last, hipStream_t s) {
  const dim3 grid = seq::grid_of(a.count);
  delta_prepare_kernel<T, kKey, kDim><<<grid, kThreads, 0, s>>>(a);
  GS_TRY(check_launch("delta_scan prepare"));
  ChainArgs chain{int64_t(a.p.batch) * a.p.heads, a.p.chunks, a.p.key_dim, a.p.dim, a.chain, state,
                  a.p.heads / a.p.key_heads, a.free, a.kept.updates, nullptr, a.kept.starts, last,
                  a.segments, a.maps, a.adds, 0, 0};
  GS_TRY(launch_chain(chain, kKey, kDim, Form<T>::chain_in, false, s));
  delta_output_kernel<T, kKey, kDim><<<grid, kThreads, 0, s>>>(a);
  return check_launch("delta_scan output");
}

}  // namespace

int64_t padded(int dim) { return dim <= 64 ? 64 : 128; }

}  // namespace delta

int check_delta(const gs_delta& d) {
  GS_REQUIRE(d.batch >= 0 && d.tokens >= 0 && d.heads > 0 && d.key_heads > 0, GS_ERR_INVALID_ARGUMENT,
             "delta rule: sizes must be positive");
  GS_REQUIRE(d.heads % d.key_heads == 0, GS_ERR_INVALID_ARGUMENT, "%d heads cannot share %d keys",
             d.heads, d.key_heads);
  GS_REQUIRE(d.key_dim > 0 && d.dim > 0, GS_ERR_INVALID_ARGUMENT, "dimensions must be positive");
  GS_REQUIRE(d.key_dim % 8 == 0 && d.key_dim <= 128 && d.dim % 8 == 0 && d.dim <= 128,
             GS_ERR_UNSUPPORTED, "heads of %d x %d not supported (multiples of 8 up to 128)", d.key_dim,
             d.dim);
  GS_REQUIRE(seq::float_type(d.type), GS_ERR_INVALID_ARGUMENT, "type must be GS_F32, GS_F16 or GS_BF16");
  GS_REQUIRE(d.scale > 0.0f && d.scale <= 3.4e38f, GS_ERR_INVALID_ARGUMENT,
             "scale must be positive, got %g", double(d.scale));
  GS_REQUIRE(d.tokens < (int64_t(1) << 30) && d.batch < (int64_t(1) << 30) && d.heads < 65536 &&
                 d.batch * d.heads < (int64_t(1) << 30),
             GS_ERR_OVERFLOW, "delta rule problem too large");
  // Chunks of all heads: workgroups over two dimensions.
  GS_REQUIRE((d.tokens + delta::kChunk - 1) / delta::kChunk * d.batch * d.heads < (int64_t(1) << 36),
             GS_ERR_OVERFLOW, "delta rule problem too large");
  return GS_OK;
}

int64_t delta_chunks(const gs_delta& d) {
  return d.batch * d.heads * ((d.tokens + delta::kChunk - 1) / delta::kChunk);
}

// Bytes of the chain's factors of one chunk, and the workspace they are cut from.
size_t delta_left_bytes(const gs_delta& d, int parts) {
  return size_t(parts) * delta::kChunk * delta::padded(d.key_dim) * sizeof(uint16_t);
}

delta::Problem delta_problem(const gs_delta& d, const int32_t* lengths) {
  return {int(d.batch), int(d.tokens), d.heads, d.key_heads, d.key_dim, d.dim,
          int((d.tokens + delta::kChunk - 1) / delta::kChunk), d.scale, lengths};
}

// Bytes of an element of what is kept for one product (Form's Store).
size_t delta_store_bytes(const gs_delta& d) { return d.type == GS_BF16 ? 2 : 4; }

delta::Kept delta_kept(const gs_delta& d, void* kept, bool solve) {
  const int64_t n = delta_chunks(d), wide = delta::padded(d.dim);
  char* at = static_cast<char*>(kept);
  delta::Kept k;
  k.solve = solve ? reinterpret_cast<float*>(at) : nullptr;
  if (solve) at += n * delta::kChunk * delta::kChunk * sizeof(float);
  k.starts = at;
  k.updates = at + n * delta::padded(d.key_dim) * wide * delta_store_bytes(d);
  return k;
}

// Scratch of a chain in segments.
size_t delta_segment_bytes(const gs_delta& d) {
  const int64_t chunks = (d.tokens + delta::kChunk - 1) / delta::kChunk;
  const int n = delta::chain_segments(d.batch * d.heads, chunks, d.dim);
  const size_t key = delta::padded(d.key_dim), parts = d.type == GS_F32 ? 3 : 2;
  return n == 1 ? 0
                : size_t(n) * d.batch * d.heads *
                      (key * delta::padded(d.dim) * sizeof(float) + parts * key * key * sizeof(uint16_t));
}

// Parts in the chain of an input and of another factor.
int delta_parts_in(const gs_delta& d) { return d.type == GS_F32 ? 3 : d.type == GS_F16 ? 2 : 1; }
int delta_parts_mid(const gs_delta& d) { return d.type == GS_F32 ? 3 : 2; }

// A tensor whose rows the kernels read by 16 bytes; elements of gates one by one.
int check_delta_rows(const void* p, const int64_t* strides, int32_t type, const char* name) {
  GS_REQUIRE(p, GS_ERR_INVALID_ARGUMENT, "null %s", name);
  const int64_t unit = 16 / seq::type_bytes(type);
  GS_REQUIRE(seq::aligned_to(p, 16) && strides[0] % unit == 0 && strides[1] % unit == 0 &&
                 strides[2] % unit == 0,
             GS_ERR_INVALID_ARGUMENT, "%s must have rows on 16-byte boundaries", name);
  return GS_OK;
}

}  // namespace gs

using namespace gs;

extern "C" GS_API size_t gs_delta_scan_kept_bytes(const gs_delta* desc, int32_t backward) {
  if (!desc || check_delta(*desc) != GS_OK) return 0;
  const size_t wide = delta::padded(desc->dim);
  const size_t a_chunk = (delta::padded(desc->key_dim) + delta::kChunk) * wide * delta_store_bytes(*desc) +
                         (backward ? delta::kChunk * delta::kChunk * sizeof(float) : 0);
  return size_t(delta_chunks(*desc)) * a_chunk;
}

extern "C" GS_API size_t gs_delta_scan_workspace_bytes(const gs_delta* desc) {
  if (!desc || check_delta(*desc) != GS_OK) return 0;
  return delta_segment_bytes(*desc) +
         size_t(delta_chunks(*desc)) *
             (delta_left_bytes(*desc, delta_parts_in(*desc) + delta_parts_mid(*desc)) +
              (delta::kFactors + delta::kChunk * delta::padded(desc->dim)) * sizeof(float));
}

extern "C" GS_API int gs_delta_scan_fwd(const gs_delta* desc, const void* q, const void* k,
                                        const void* v, const void* gate, const void* beta,
                                        const int64_t* strides, const int32_t* lengths,
                                        const float* state, int32_t backward, void* out, float* last,
                                        void* kept, void* workspace, size_t workspace_bytes,
                                        void* stream) {
  clear_error();
  GS_REQUIRE(desc, GS_ERR_INVALID_ARGUMENT, "null description");
  GS_TRY(check_delta(*desc));
  if (desc->batch == 0 || desc->tokens == 0) return GS_OK;
  GS_REQUIRE(strides && gate && beta && out && last, GS_ERR_INVALID_ARGUMENT, "null pointer");
  GS_TRY(check_delta_rows(q, strides, desc->type, "q"));
  GS_TRY(check_delta_rows(k, strides + 3, desc->type, "k"));
  GS_TRY(check_delta_rows(v, strides + 6, desc->type, "v"));
  GS_REQUIRE(kept && seq::aligned_to(kept, 16), GS_ERR_INVALID_ARGUMENT, "kept must be on a 16-byte boundary");
  const size_t need = gs_delta_scan_workspace_bytes(desc);
  GS_REQUIRE(workspace && workspace_bytes >= need && seq::aligned_to(workspace, 16), GS_ERR_WORKSPACE,
             "workspace too small or off a 16-byte boundary: %zu bytes, %zu needed", workspace_bytes, need);
  const int64_t n = delta_chunks(*desc);
  return seq::with_type(desc->type, [&](auto t) {
    using T = decltype(t);
    delta::ForwardArgs<T> a;
    a.p = delta_problem(*desc, lengths);
    const auto rows = [&](const void* p, int i) {
      return delta::Rows<T>{static_cast<const T*>(p), {strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]}};
    };
    a.q = rows(q, 0);
    a.k = rows(k, 1);
    a.v = rows(v, 2);
    a.gate = rows(gate, 3);
    a.beta = rows(beta, 4);
    a.kept = delta_kept(*desc, kept, backward);
    a.chain.factors = static_cast<float*>(workspace);
    a.free = a.chain.factors + n * delta::kFactors;
    a.chain.left = reinterpret_cast<delta::bf16*>(a.free + n * delta::kChunk * delta::padded(desc->dim));
    a.chain.right = a.chain.left + n * delta_left_bytes(*desc, delta_parts_mid(*desc)) / 2;
    a.out = static_cast<T*>(out);
    a.count = n;
    a.segments = delta::chain_segments(desc->batch * desc->heads, a.p.chunks, desc->dim);
    a.adds = reinterpret_cast<float*>(a.chain.right + n * delta_left_bytes(*desc, delta_parts_in(*desc)) / 2);
    a.maps = reinterpret_cast<delta::bf16*>(a.adds + int64_t(a.segments) * desc->batch * desc->heads *
                                                         delta::padded(desc->key_dim) * delta::padded(desc->dim));
    const hipStream_t s = as_stream(stream);
    // Heads of up to 64 have tiles of their own.
    if (desc->key_dim <= 64)
      return desc->dim <= 64 ? delta::forward<T, 64, 64>(a, state, last, s)
                             : delta::forward<T, 64, 128>(a, state, last, s);
    return desc->dim <= 64 ? delta::forward<T, 128, 64>(a, state, last, s)
                           : delta::forward<T, 128, 128>(a, state, last, s);
  });
}
