// Gradients of the gated delta rule (delta_scan.h has the formulas): a workgroup a
// chunk of a head prepares what the chain needs, the chain runs backwards, and a
// workgroup a chunk of a key, with the heads that share it in order, gives the
// gradients:
//   dR = T^T dU, dV = b dR, N = scale (dO U^T) * D, M = -(dR U^T) * D below the
//   diagonal,
//   dQ = scale e^G dO S^T + N K,
//   Z  = -e^G dR S^T + M K              what a key reads with, before b,
//   Y  = e^(G_C - G) U dS'^T + N^T Q + (b M)^T K   what it writes with,
//   dK = b Z + Y,   db_i = dR_i . v_i + Z_i . k_i.
// The gate of token t decays what tokens before it wrote on its way to those from t
// on, so the logarithm of a_t has the gradient of all that crosses t:
//   dlog a_t = sum over i >= t > j of E_ij + sum over i >= t of r_i
//              + sum over j < t of w_j + e^(G_C) <S, dS'>,
//   E = N * Q K^T + b M * K K^T,  r_i = scale e^G q_i . S dO_i - b e^G k_i . S dR_i,
//   w_j = e^(G_C - G) k_j . dS' u_j.
// That is a sum over i >= t of r_i - w_i + sum_j E_ij - sum_j E_ji, and a constant, and
// with the same numbers E, r and w in rows and columns nothing but what crosses is left
// of it, whatever their rounding (taken from q . dQ, k . dK and <S', dS'>, which round
// apart, the gates' gradient in bfloat16 is off by 0.0065 to 0.015).  db goes by
// b_i db_i = u_i . dR_i, which A's lines make of dR_i . v_i + Z_i . k_i.
//
// All results are taken turned: a lane has one token, with the dimensions in its
// registers, so that the factors of a token are one number, its scalar products need
// no exchange but of four lanes, and stores are of consecutive elements.
//
// Measured, 40000 tokens, 12 heads of 64 on 4, bfloat16: 134 us to prepare (227 with two
// workgroups a CU), 213 the gradients (421 before sums stayed in registers and gates
// were read as vectors), and the chain.  LDS traffic and latency bound both.
#include "delta_scan.h"

namespace gs {

int check_delta(const gs_delta& d);
int check_delta_rows(const void* p, const int64_t* strides, int32_t type, const char* name);
int64_t delta_chunks(const gs_delta& d);
size_t delta_left_bytes(const gs_delta& d, int parts);
delta::Problem delta_problem(const gs_delta& d, const int32_t* lengths);
size_t delta_store_bytes(const gs_delta& d);
delta::Kept delta_kept(const gs_delta& d, void* kept, bool solve);
int delta_parts_in(const gs_delta& d);
int delta_parts_mid(const gs_delta& d);
size_t delta_segment_bytes(const gs_delta& d);

namespace delta {
namespace {

template <typename T>
struct BackwardArgs {
  Problem p;
  Rows<T> q, k, v, gate, beta, grad;  // grad.p may be null
  Kept kept;
  Chain chain;
  float* du;      // [kDim, 64] a chunk
  float* begins;  // [kDim, kKey] a chunk: scale Q^T e^G dO
  void* ends;     // [kDim, kKey] a chunk, Form's Store: dS behind it; may be begins
  T* dq;
  T* dk;
  T* dv;
  T* dgate;
  T* dbeta;
  int64_t count;
  int segments;
  bf16* maps;
  float* adds;
};

constexpr int kPitchA = kChunk + 4;

template <typename T, int kKey, int kDim>
__global__ __launch_bounds__(kThreads) void delta_back_prepare_kernel(BackwardArgs<T> a) {
  using F = Form<T>;
  using E = typename F::Elem;
  using KTile = Tile<E, F::in, kChunk, kKey>;
  using QTile = Tile<E, F::mid, kChunk, kKey>;
  using OTile = Tile<E, F::in, kChunk, kDim>;
  using PTile = Tile<E, F::mid, kChunk, kChunk>;
  static_assert(QTile::bytes <= 2 * KTile::bytes, "the scaled q takes the place of k and q");
  // P takes T's place, once W is there: three workgroups share a CU.
  constexpr int kSolve = kChunk * kPitchA * int(sizeof(float));
  __shared__ __align__(16) char kq_space[2 * KTile::bytes], o_space[OTile::bytes];
  __shared__ __align__(16) char p_space[kSolve > PTile::bytes ? kSolve : PTile::bytes];
  __shared__ float by_key[kChunk];
  __shared__ Gates g;
  const int64_t index = seq::block_index();
  if (index >= a.count) return;
  const Place at(a.p, index);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const KTile k(kq_space), q(kq_space + KTile::bytes);
  const QTile q_up(kq_space);
  const OTile grad(o_space);
  const PTile p(p_space);
  float* solve = reinterpret_cast<float*>(p_space);
  const T* q_rows = a.q.at(at.b, at.t0, at.key_head);
  const GatePair gates(a.gate, a.beta, at);
  Fetch<T, kChunk, kKey> k_in, q_in;
  Fetch<T, kChunk, kDim> grad_in;
  Fetch<float, kChunk, kChunk> solve_in;
  k_in.load(a.k.at(at.b, at.t0, at.key_head), a.k.s.token, at.valid, a.p.key_dim);
  q_in.load(q_rows, a.q.s.token, at.valid, a.p.key_dim);
  grad_in.load(a.grad.at(at.b, at.t0, at.h), a.grad.s.token, a.grad.p ? at.valid : 0, a.p.dim);
  solve_in.load_triangle(a.kept.solve + index * kChunk * kChunk);
  if (wave == 0) gates.put(g);
  k_in.put(k);
  q_in.put(q);
  grad_in.put(grad);
  solve_in.put(Tile<float, 1, kChunk, kChunk>(reinterpret_cast<char*>(solve)));
  lds_barrier();
  if (threadIdx.x < kChunk) by_key[threadIdx.x] = -g.beta[threadIdx.x] * g.up[threadIdx.x];
  lds_barrier();
  const int m0 = 32 * (wave & 1), token = m0 + (lane & 31);
  // -W turned: a lane has a dimension and consecutive tokens.
  bf16* right = a.chain.right + index * F::chain * kKey * kChunk;
#pragma unroll
  for (int t = 0; t < kKey / 64; ++t) {
    const int n0 = 32 * ((wave >> 1) + 2 * t);
    Acc c(0.0f);
    steps_to(m0, [&](int s) {
      const int kk = 16 * s + 8 * (lane >> 5);
      const float* row = solve + token * kPitchA + kk;
      FloatVec<8> x;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = row[i] * by_key[kk + i];
      mma_parts(Parts<E, F::mid, 8>(x), k.cols(16 * s, n0), c);
    });
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const Parts<bf16, F::chain, 4> x(four(c, s));
#pragma unroll
      for (int i = 0; i < F::chain; ++i)
        *reinterpret_cast<Vec<bf16, 4>*>(right + i * kKey * kChunk +
                                         fragment_at(n0 + (lane & 31), m0 + four_row(s), 2)) = x.v[i];
    }
  }
  // K, once for the heads that share it.
  const int group = a.p.heads / a.p.key_heads;
  bf16* left = a.chain.left + ((int64_t(at.b) * a.p.key_heads + at.key_head) * a.p.chunks + at.c) *
                                  F::chain_in * kChunk * kKey;
  for (int e = at.h % group ? kKey : wave; e < 2 * (kKey / 16); e += 4) {
    const int row0 = 32 * (e & 1), k0 = 16 * (e >> 1);
    FloatVec<8> x(0.0f);
    const Parts<E, F::in, 8> f = k.rows(row0, k0);
#pragma unroll
    for (int i = 0; i < F::in; ++i) x += to_float<E, 8>(f.v[i]);
    const Parts<bf16, F::chain_in, 8> y(x);
    const int row = row0 + (lane & 31), col = k0 + 8 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < F::chain_in; ++i) {
      bf16* to = left + i * kChunk * kKey;
      *reinterpret_cast<Vec<bf16, 4>*>(to + fragment_at(row, col, kKey / 32)) =
          __builtin_shufflevector(y.v[i], y.v[i], 0, 1, 2, 3);
      *reinterpret_cast<Vec<bf16, 4>*>(to + fragment_at(row, col + 4, kKey / 32)) =
          __builtin_shufflevector(y.v[i], y.v[i], 4, 5, 6, 7);
    }
  }
  lds_barrier();
  if (wave < 3) {
    const int i0 = wave ? 32 : 0, j0 = wave == 2 ? 32 : 0, i = i0 + (lane & 31);
    Acc c(0.0f);
#pragma unroll
    for (int s = 0; s < kKey / 16; ++s) mma_parts(k.rows(j0, 16 * s), q.rows(i0, 16 * s), c);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int j = j0 + four_row(s);
      FloatVec<4> x = four(c, s) * g.decay(i, j);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = j + r <= i ? a.p.scale * x[r] : 0.0f;
      p.put(i, j, Parts<E, F::mid, 4>(x));
    }
  }
  lds_barrier();
  // P^T dO.
  float* du = a.du + index * kChunk * kDim;
#pragma unroll
  for (int t = 0; t < kDim / 64; ++t) {
    const int n0 = 32 * ((wave >> 1) + 2 * t);
    Acc c(0.0f);
    steps_from(m0, [&](int s) { mma_parts(p.cols(16 * s, m0), grad.cols(16 * s, n0), c); });
#pragma unroll
    for (int s = 0; s < 4; ++s)
      *reinterpret_cast<FloatVec<4>*>(du + (n0 + (lane & 31)) * kChunk + m0 + four_row(s)) = four(c, s);
  }
  lds_barrier();
  q_in.put(q_up, [&](int row, int, auto& x) { x = x * (a.p.scale * g.up[row]); });
  lds_barrier();
  // scale Q^T e^G dO.
  float* begins = a.begins + index * kKey * kDim;
  for (int e = wave; e < kKey / 32 * (kDim / 32); e += 4) {
    const int k0 = 32 * (e / (kDim / 32)), n0 = 32 * (e % (kDim / 32));
    Acc c(0.0f);
#pragma unroll
    for (int s = 0; s < 4; ++s) mma_parts(q_up.cols(16 * s, k0), grad.cols(16 * s, n0), c);
#pragma unroll
    for (int s = 0; s < 4; ++s)
      *reinterpret_cast<FloatVec<4>*>(begins + (n0 + (lane & 31)) * kKey + k0 + four_row(s)) = four(c, s);
  }
  float* factors = a.chain.factors + index * kFactors;
  if (threadIdx.x < kChunk) factors[threadIdx.x] = g.down[threadIdx.x];
  if (threadIdx.x == 0) factors[kChunk] = g.whole;
}

// Sums of a result's columns, over the 32 lanes of a half: each lane with bit 4 clear
// gets that of one register, sums_register().  A step adds what the lane's neighbour
// gives of its half of the registers, and halves them.
template <int N>
__device__ __forceinline__ float column_sums(const FloatVec<2 * N>& c) {
  constexpr int kFar = 8 / N;
  const bool high = (threadIdx.x & 63) & kFar;
  FloatVec<N> sums;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float low = c[i], up = c[i + N];
    asm volatile("" : "+v"(low), "+v"(up));  // or the choice becomes a search by index
    sums[i] = (high ? up : low) + __shfl_xor(high ? low : up, kFar, kWave);
  }
  if constexpr (N == 1)
    return sums[0] + __shfl_xor(sums[0], 16, kWave);
  else
    return column_sums<N / 2>(sums);
}
__device__ __forceinline__ int sums_register() {
  const int lane = threadIdx.x;
  return (lane & 1) << 3 | (lane & 2) << 1 | (lane & 4) >> 1 | (lane & 8) >> 3;
}

template <typename T, int kKey, int kDim>
__global__ __launch_bounds__(kThreads, (kKey == 64 && std::is_same_v<T, bf16> ? 2 : 1)) void delta_grads_kernel(
    BackwardArgs<T> a) {
  using F = Form<T>;
  using E = typename F::Elem;
  constexpr int P = F::out;
  static_assert(P == F::in, "inputs and results have the same parts here");
  using Half = Tile<E, P, kChunk, 64>;   // half of a value's dimensions
  using STile = Tile<E, P, 64, kKey>;  // 64 columns of a state, turned
  using KTile = Tile<E, P, kChunk, kKey>;
  using Fine = Tile<E, F::mid, kChunk, 64>;
  constexpr int kFirst = 2 * Half::bytes + 2 * Fine::bytes + STile::bytes;
  constexpr int kSecond = 2 * Half::bytes + 2 * KTile::bytes;
  __shared__ __align__(16) char space[kFirst > kSecond ? kFirst : kSecond];
  __shared__ Gates g;
  __shared__ float dots[3][2][kChunk], crossing[2][3][32], inner[4];
  const Half grad(space), u(space + Half::bytes), x(space + 2 * Half::bytes);
  const Fine du(space + 2 * Half::bytes), solve(space + 2 * Half::bytes + Fine::bytes);
  const STile state(space + 2 * Half::bytes + 2 * Fine::bytes);
  const Half n_tile(space), m_tile(space + Half::bytes);
  const KTile q(space + 2 * Half::bytes), k(space + 2 * Half::bytes + KTile::bytes);
  constexpr int kTiles = kKey / 64;
  const int64_t work = seq::block_index();
  const int group = a.p.heads / a.p.key_heads;
  if (work >= a.count / group) return;
  // The heads of a key are chunks apart.
  const int64_t first = work % a.p.chunks + work / a.p.chunks * a.p.chunks * group;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m0 = 32 * (wave & 1), side = wave >> 1, token = m0 + (lane & 31);
  const int i0 = wave ? 32 : 0, j0 = wave == 2 ? 32 : 0;  // of the triangles, waves 0 .. 2
  Fetch<T, kChunk, 64> grad_in;
  using Store = typename F::Store;
  Fetch<Store, 64, kChunk> u_in;
  Fetch<float, 64, kChunk> du_in;
  Fetch<float, kChunk, kChunk> solve_in;
  Fetch<Store, 64, kKey> state_in, end_in;
  Fetch<T, kChunk, kKey> q_in, k_in;
  const auto fetch_half = [&](const Place& at, int d0) {
    const int64_t base = at.id * kDim + d0;
    const int wide = a.p.dim - d0;
    grad_in.load(a.grad.at(at.b, at.t0, at.h) + d0, a.grad.s.token, a.grad.p ? at.valid : 0, wide);
    u_in.load(static_cast<const Store*>(a.kept.updates) + base * kChunk, kChunk, wide, kChunk);
    du_in.load(a.du + base * kChunk, kChunk, wide, kChunk);
    state_in.load(static_cast<const Store*>(a.kept.starts) + base * kKey, kKey, wide, a.p.key_dim);
    end_in.load(static_cast<const Store*>(a.ends) + base * kKey, kKey, wide, a.p.key_dim);
  };
  Acc dq_all[kTiles], dk_all[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) dq_all[t] = dk_all[t] = Acc(0.0f);
  for (int member = 0; member < group; ++member) {
    const int64_t index = first + int64_t(member) * a.p.chunks;
    const Place at(a.p, index);
    const GatePair gates(a.gate, a.beta, at);
    solve_in.load_triangle(a.kept.solve + index * kChunk * kChunk);
    fetch_half(at, 0);
    q_in.load(a.q.at(at.b, at.t0, at.key_head), a.q.s.token, at.valid, a.p.key_dim);
    k_in.load(a.k.at(at.b, at.t0, at.key_head), a.k.s.token, at.valid, a.p.key_dim);
    lds_barrier();
    if (wave == 0) gates.put(g);
    Acc dq[kTiles], z[kTiles], y[kTiles], n(0.0f), m(0.0f);
#pragma unroll
    for (int t = 0; t < kTiles; ++t) dq[t] = z[t] = y[t] = Acc(0.0f);
    float found = 0.0f, both = 0.0f;
    solve_in.put(solve);
    const int64_t row = ((int64_t(at.b) * a.p.tokens + at.t0 + token) * a.p.heads + at.h) * a.p.dim;
#pragma unroll
    for (int d0 = 0; d0 < kDim; d0 += 64) {
      if (d0 >= a.p.dim) break;
      const int wide = a.p.dim - d0;
      if (d0) lds_barrier();
      grad_in.put(grad);
      u_in.put(u);
      du_in.put(du);
      state_in.put(state);
#pragma unroll
      for (int i = 0; i < end_in.kCount; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) both += float(end_in.x[i][e]) * float(state_in.x[i][e]);
      lds_barrier();
      // dR of the wave's tokens and 32 dimensions.
      Acc r(0.0f);
      steps_from(m0, [&](int s) { mma_parts(du.rows(32 * side, 16 * s), solve.cols(16 * s, m0), r); });
      lds_barrier();
      const float b = g.beta[token];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int col = 32 * side + four_row(s);
        const FloatVec<4> dr = four(r, s);
        x.put(token, col, Parts<E, P, 4>(dr));
        if (token < at.rows && col < wide) {
          FloatVec<4> out = b * dr;
          if (token < at.valid) {
#pragma unroll
            for (int i = 0; i < 4; ++i) found += u.get(col + i, token) * dr[i];
          } else {
            out = FloatVec<4>(0.0f);
          }
          *reinterpret_cast<Vec<T, 4>*>(a.dv + row + d0 + col) = from_float<T, 4>(out);
        }
      }
      lds_barrier();
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (wave < 3) {
          const auto left = u.cols(16 * s, j0);
          mma_parts(left, grad.rows(i0, 16 * s), n);
          mma_parts(left, x.rows(i0, 16 * s), m);
        }
        const auto go = grad.rows(m0, 16 * s), dr = x.rows(m0, 16 * s);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const auto left = state.cols(16 * s, 32 * (side + 2 * t));
          mma_parts(left, go, dq[t]);
          mma_parts(left, dr, z[t]);
        }
      }
      lds_barrier();
      end_in.put(state);
      if (d0 + 64 < a.p.dim) fetch_half(at, d0 + 64);
      lds_barrier();
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const auto right = u.cols(16 * s, m0);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) mma_parts(state.cols(16 * s, 32 * (side + 2 * t)), right, y[t]);
      }
    }
    const float up = g.up[token], down = g.down[token], beta = g.beta[token];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      dq[t] *= a.p.scale * up;
      z[t] *= -up;
      y[t] *= down;
    }
    lds_barrier();
    if (wave < 3) {
      const int i = i0 + (lane & 31);
      const float b = g.beta[i];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int j = j0 + four_row(s);
        const FloatVec<4> d = g.decay(i, j);
        FloatVec<4> nn = four(n, s) * d, mm = four(m, s) * d;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          nn[e] = j + e <= i ? a.p.scale * nn[e] : 0.0f;
          mm[e] = j + e < i ? -mm[e] : 0.0f;
        }
        n_tile.put(i, j, Parts<E, P, 4>(nn));
        m_tile.put(i, j, Parts<E, P, 4>(b * mm));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          n[4 * s + e] = nn[e];
          m[4 * s + e] = b * mm[e];
        }
      }
    }
    q_in.put(q);
    k_in.put(k);
    lds_barrier();
    if (wave < 3) {
      Acc qk(0.0f), kk(0.0f);
#pragma unroll
      for (int s = 0; s < kKey / 16; ++s) {
        const auto left = k.rows(j0, 16 * s);
        mma_parts(left, q.rows(i0, 16 * s), qk);
        mma_parts(left, k.rows(i0, 16 * s), kk);
      }
      n = n * qk + m * kk;
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += n[r];
      sum += __shfl_xor(sum, 32, kWave);
      if (lane < 32) crossing[0][wave][lane] = sum;
      const float column = column_sums<8>(n);
      if ((lane & 16) == 0) crossing[1][wave][acc_row_of_half(sums_register()) + 4 * (lane >> 5)] = column;
    }
    float reads = 0.0f, writes = 0.0f;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int col = 32 * (side + 2 * t) + four_row(s);
        const FloatVec<4> qq = q.get4(token, col), kk = k.get4(token, col);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          reads += qq[i] * dq[t][4 * s + i] + beta * kk[i] * z[t][4 * s + i];
          writes += kk[i] * y[t][4 * s + i];
        }
      }
    // The rest goes to the sums over the heads: b M has b of the key that reads in its
    // rows.
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      dq_all[t] += dq[t];
      dk_all[t] += beta * z[t] + y[t];
    }
    steps_to(m0, [&](int s) {
      const auto nn = n_tile.rows(m0, 16 * s), mm = m_tile.rows(m0, 16 * s);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const auto left = k.cols(16 * s, 32 * (side + 2 * t));
        mma_parts(left, nn, dq_all[t]);
        mma_parts(left, mm, dk_all[t]);
      }
    });
    steps_from(m0, [&](int s) {
      const auto nn = n_tile.cols(16 * s, m0), mm = m_tile.cols(16 * s, m0);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        mma_parts(q.cols(16 * s, 32 * (side + 2 * t)), nn, dk_all[t]);
        mma_parts(k.cols(16 * s, 32 * (side + 2 * t)), mm, dk_all[t]);
      }
    });
    const float all[3] = {reads, writes, found};
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const float sum = all[i] + __shfl_xor(all[i], 32, kWave);
      if (lane < 32) dots[i][side][token] = sum;
    }
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) both += __shfl_xor(both, d, kWave);
    if (lane == 0) inner[wave] = both;
    lds_barrier();
    if (wave == 0) {
      const int row = lane & 31;
      const float wrote = dots[1][0][lane] + dots[1][1][lane];
      float total = dots[0][0][lane] + dots[0][1][lane] - wrote;
      if (lane < 32)
        total += crossing[0][0][row] - (crossing[1][0][row] + crossing[1][1][row]);
      else
        total += (crossing[0][1][row] + crossing[0][2][row]) - crossing[1][2][row];
      float rest = wrote;
#pragma unroll
      for (int d = 1; d < kWave; d <<= 1) rest += __shfl_xor(rest, d, kWave);
      rest += g.whole * ((inner[0] + inner[1]) + (inner[2] + inner[3]));
#pragma unroll
      for (int d = 1; d < kChunk; d <<= 1) {
        const float later = __shfl_down(total, d, kChunk);
        if (lane + d < kChunk) total += later;
      }
      if (lane < at.rows) {
        float dgate = 0.0f, dbeta = 0.0f;
        if (lane < at.valid) {
          dgate = (total + rest) * g.fade[lane];
          dbeta = (dots[2][0][lane] + dots[2][1][lane]) * g.rest[lane];
        }
        const int64_t to = (int64_t(at.b) * a.p.tokens + at.t0 + lane) * a.p.heads + at.h;
        a.dgate[to] = T(dgate);
        a.dbeta[to] = T(dbeta);
      }
    }
  }
  const Place at(a.p, first);
  if (token < at.rows) {
    const int64_t to = ((int64_t(at.b) * a.p.tokens + at.t0 + token) * a.p.key_heads + at.key_head) * a.p.key_dim;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int col = 32 * (side + 2 * t) + four_row(s);
        if (col < a.p.key_dim) {
          const bool none = token >= at.valid;
          *reinterpret_cast<Vec<T, 4>*>(a.dq + to + col) =
              from_float<T, 4>(none ? FloatVec<4>(0.0f) : four(dq_all[t], s));
          *reinterpret_cast<Vec<T, 4>*>(a.dk + to + col) =
              from_float<T, 4>(none ? FloatVec<4>(0.0f) : four(dk_all[t], s));
        }
      }
  }
}

template <typename T, int kKey, int kDim>
int backward(const BackwardArgs<T>& a, const float* grad_last, float* grad_state, hipStream_t s) {
  delta_back_prepare_kernel<T, kKey, kDim><<<seq::grid_of(a.count), kThreads, 0, s>>>(a);
  GS_TRY(check_launch("delta_scan backward prepare"));
  ChainArgs chain{int64_t(a.p.batch) * a.p.heads, a.p.chunks, a.p.key_dim, a.p.dim, a.chain, grad_last,
                  a.p.heads / a.p.key_heads, a.du, a.du, a.begins, a.ends, grad_state, a.segments, a.maps,
                  a.adds, 0, 0};
  GS_TRY(launch_chain(chain, kKey, kDim, Form<T>::chain_in, true, s));
  const int64_t groups = a.count / (a.p.heads / a.p.key_heads);
  delta_grads_kernel<T, kKey, kDim><<<seq::grid_of(groups), kThreads, 0, s>>>(a);
  return check_launch("delta_scan gradients");
}

}  // namespace
}  // namespace delta
}  // namespace gs

using namespace gs;

extern "C" GS_API size_t gs_delta_scan_bwd_workspace_bytes(const gs_delta* desc) {
  if (!desc || check_delta(*desc) != GS_OK) return 0;
  const size_t wide = delta::padded(desc->dim);
  return delta_segment_bytes(*desc) +
         size_t(delta_chunks(*desc)) *
         (delta_left_bytes(*desc, delta_parts_in(*desc) + delta_parts_mid(*desc)) +
          (delta::kFactors + (delta::kChunk + delta::padded(desc->key_dim)) * wide) * sizeof(float) +
          (delta_store_bytes(*desc) == 2 ? delta::padded(desc->key_dim) * wide * 2 : 0));
}

extern "C" GS_API int gs_delta_scan_bwd(
    const gs_delta* desc, const void* q, const void* k, const void* v, const void* gate,
    const void* beta, const void* grad_out, const int64_t* strides, const int32_t* lengths,
    const float* grad_last, const void* kept, void* grad_q, void* grad_k,
    void* grad_v, void* grad_gate, void* grad_beta, float* grad_state, void* workspace,
    size_t workspace_bytes, void* stream) {
  clear_error();
  GS_REQUIRE(desc, GS_ERR_INVALID_ARGUMENT, "null description");
  GS_TRY(check_delta(*desc));
  if (desc->batch == 0 || desc->tokens == 0) return GS_OK;
  GS_REQUIRE(strides && gate && beta, GS_ERR_INVALID_ARGUMENT, "null pointer");
  for (const void* p : {grad_q, grad_k, grad_v, grad_gate, grad_beta})
    GS_REQUIRE(p, GS_ERR_INVALID_ARGUMENT, "null pointer: a gradient");
  GS_TRY(check_delta_rows(q, strides, desc->type, "q"));
  GS_TRY(check_delta_rows(k, strides + 3, desc->type, "k"));
  GS_TRY(check_delta_rows(v, strides + 6, desc->type, "v"));
  if (grad_out) GS_TRY(check_delta_rows(grad_out, strides + 15, desc->type, "grad_out"));
  for (const void* p : {grad_q, grad_k, grad_v})
    GS_REQUIRE(seq::aligned_to(p, 16), GS_ERR_INVALID_ARGUMENT, "gradients must be on 16-byte boundaries");
  GS_REQUIRE(kept && seq::aligned_to(kept, 16), GS_ERR_INVALID_ARGUMENT, "kept must be on a 16-byte boundary");
  const size_t need = gs_delta_scan_bwd_workspace_bytes(desc);
  GS_REQUIRE(workspace && workspace_bytes >= need && seq::aligned_to(workspace, 16), GS_ERR_WORKSPACE,
             "workspace too small or off a 16-byte boundary: %zu bytes, %zu needed", workspace_bytes, need);
  const int64_t n = delta_chunks(*desc);
  return seq::with_type(desc->type, [&](auto t) {
    using T = decltype(t);
    delta::BackwardArgs<T> a;
    a.p = delta_problem(*desc, lengths);
    const auto rows = [&](const void* p, int i) {
      return delta::Rows<T>{static_cast<const T*>(p), {strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]}};
    };
    a.q = rows(q, 0);
    a.k = rows(k, 1);
    a.v = rows(v, 2);
    a.gate = rows(gate, 3);
    a.beta = rows(beta, 4);
    a.grad = grad_out ? rows(grad_out, 5) : delta::Rows<T>{nullptr, {0, 0, 0}};
    a.kept = delta_kept(*desc, const_cast<void*>(kept), true);
    const int64_t wide = delta::padded(desc->dim);
    a.chain.factors = static_cast<float*>(workspace);
    a.du = a.chain.factors + n * delta::kFactors;
    a.begins = a.du + n * delta::kChunk * wide;
    a.ends = a.begins;
    a.chain.left = reinterpret_cast<delta::bf16*>(a.begins + n * delta::padded(desc->key_dim) * wide);
    if (delta_store_bytes(*desc) == 2) {
      a.ends = a.chain.left;
      a.chain.left += n * delta::padded(desc->key_dim) * wide;
    }
    a.chain.right = a.chain.left + n * delta_left_bytes(*desc, delta_parts_in(*desc)) / 2;
    a.dq = static_cast<T*>(grad_q);
    a.dk = static_cast<T*>(grad_k);
    a.dv = static_cast<T*>(grad_v);
    a.dgate = static_cast<T*>(grad_gate);
    a.dbeta = static_cast<T*>(grad_beta);
    a.count = n;
    a.segments = delta::chain_segments(desc->batch * desc->heads, a.p.chunks, desc->dim);
    a.adds = reinterpret_cast<float*>(a.chain.right + n * delta_left_bytes(*desc, delta_parts_mid(*desc)) / 2);
    a.maps = reinterpret_cast<delta::bf16*>(a.adds + int64_t(a.segments) * desc->batch * desc->heads *
                                                         delta::padded(desc->key_dim) * wide);
    const hipStream_t s = as_stream(stream);
    if (desc->key_dim <= 64)
      return desc->dim <= 64 ? delta::backward<T, 64, 64>(a, grad_last, grad_state, s)
                             : delta::backward<T, 64, 128>(a, grad_last, grad_state, s);
    return desc->dim <= 64 ? delta::backward<T, 128, 64>(a, grad_last, grad_state, s)
                           : delta::backward<T, 128, 128>(a, grad_last, grad_state, s);
  });
}
