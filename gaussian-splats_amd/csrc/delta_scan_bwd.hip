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
// Measured, 40000 tokens, 12 heads of 64 on 4, bfloat16: 227 us to
// prepare, 421 the gradients, and the chain.
#include "delta_scan.h"

namespace gs {

int check_delta(const gs_delta& d);
int check_delta_rows(const void* p, const int64_t* strides, int32_t type, const char* name);
int64_t delta_chunks(const gs_delta& d);
size_t delta_left_bytes(const gs_delta& d, int parts);
delta::Problem delta_problem(const gs_delta& d, const int32_t* lengths);
delta::Kept delta_kept(const gs_delta& d, float* kept, bool solve);
int delta_parts_in(const gs_delta& d);
int delta_parts_mid(const gs_delta& d);

namespace delta {
namespace {

template <typename T>
struct BackwardArgs {
  Problem p;
  Rows<T> q, k, v, gate, beta, grad;  // grad.p may be null
  Kept kept;
  Chain chain;
  float* du;    // [64, kDim] a chunk
  float* ends;  // [kKey, kDim] a chunk: dS behind it
  T* dq;
  T* dk;
  T* dv;
  T* dgate;
  T* dbeta;
  int64_t count;
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
  __shared__ __align__(16) char kq_space[2 * KTile::bytes], o_space[OTile::bytes], p_space[PTile::bytes];
  __shared__ __align__(16) float solve[kChunk * kPitchA];
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
  const T* q_rows = a.q.at(at.b, at.t0, at.key_head);
  if (wave == 0) load_gates(g, a.gate, a.beta, at);
  load_tile<T>(k, a.k.at(at.b, at.t0, at.key_head), a.k.s.token, at.valid, a.p.key_dim, Keep{});
  load_tile<T>(q, q_rows, a.q.s.token, at.valid, a.p.key_dim, Keep{});
  load_tile<T>(grad, a.grad.at(at.b, at.t0, at.h), a.grad.s.token, a.grad.p ? at.valid : 0, a.p.dim, Keep{});
  {
    const float* from = a.kept.solve + index * kChunk * kChunk;
#pragma unroll
    for (int s = 0; s < kChunk * kChunk / 4 / kThreads; ++s) {
      const int e = (s * kThreads + int(threadIdx.x)) * 4;
      *reinterpret_cast<FloatVec<4>*>(solve + e / kChunk * kPitchA + e % kChunk) =
          *reinterpret_cast<const FloatVec<4>*>(from + e);
    }
  }
  __syncthreads();
  if (threadIdx.x < kChunk) by_key[threadIdx.x] = -g.beta[threadIdx.x] * g.up[threadIdx.x];
  if (wave < 3) {
    const int i0 = wave ? 32 : 0, j0 = wave == 2 ? 32 : 0, i = i0 + (lane & 31);
    Acc c(0.0f);
#pragma unroll
    for (int s = 0; s < kKey / 16; ++s) mma_parts(k.rows(j0, 16 * s), q.rows(i0, 16 * s), c);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int j = j0 + four_row(s);
      FloatVec<4> x = four(c, s);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = j + r <= i ? a.p.scale * g.decay(i, j + r) * x[r] : 0.0f;
      p.put(i, j, Parts<E, F::mid, 4>(x));
    }
  }
  __syncthreads();
  const int m0 = 32 * (wave & 1), token = m0 + (lane & 31);
  // -W turned: a lane has a dimension and consecutive tokens.
  bf16* right = a.chain.right + index * F::chain * kKey * kChunk;
#pragma unroll
  for (int t = 0; t < kKey / 64; ++t) {
    const int n0 = 32 * ((wave >> 1) + 2 * t);
    Acc c(0.0f);
    for (int s = 0; s < (m0 ? 4 : 2); ++s) {
      const int kk = 16 * s + 8 * (lane >> 5);
      const float* row = solve + token * kPitchA + kk;
      FloatVec<8> x;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = row[i] * by_key[kk + i];
      mma_parts(Parts<E, F::mid, 8>(x), k.cols(16 * s, n0), c);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const Parts<bf16, F::chain, 4> x(four(c, s));
#pragma unroll
      for (int i = 0; i < F::chain; ++i)
        *reinterpret_cast<Vec<bf16, 4>*>(right + (i * kKey + n0 + (lane & 31)) * kChunk + m0 + four_row(s)) = x.v[i];
    }
  }
  bf16* left = a.chain.left + index * F::chain_in * kChunk * kKey;
  for (int e = wave; e < 2 * (kKey / 16); e += 4) {
    const int row0 = 32 * (e & 1), k0 = 16 * (e >> 1);
    FloatVec<8> x(0.0f);
    const Parts<E, F::in, 8> f = k.rows(row0, k0);
#pragma unroll
    for (int i = 0; i < F::in; ++i) x += to_float<E, 8>(f.v[i]);
    const Parts<bf16, F::chain_in, 8> y(x);
#pragma unroll
    for (int i = 0; i < F::chain_in; ++i)
      *reinterpret_cast<Frag<bf16>*>(left + (i * kChunk + row0 + (lane & 31)) * kKey + k0 + 8 * (lane >> 5)) = y.v[i];
  }
  // P^T dO.
  float* du = a.du + index * kChunk * kDim;
#pragma unroll
  for (int t = 0; t < kDim / 64; ++t) {
    const int n0 = 32 * ((wave >> 1) + 2 * t);
    Acc c(0.0f);
    for (int s = m0 / 16; s < 4; ++s) mma_parts(grad.cols(16 * s, n0), p.cols(16 * s, m0), c);
#pragma unroll
    for (int s = 0; s < 4; ++s)
      *reinterpret_cast<FloatVec<4>*>(du + token * kDim + n0 + four_row(s)) = four(c, s);
  }
  __syncthreads();
  load_tile<T>(q_up, q_rows, a.q.s.token, at.valid, a.p.key_dim,
               [&](int row, int, auto& x) { x = x * (a.p.scale * g.up[row]); });
  __syncthreads();
  // scale Q^T e^G dO.
  float* ends = a.ends + index * kKey * kDim;
  for (int e = wave; e < kKey / 32 * (kDim / 32); e += 4) {
    const int k0 = 32 * (e / (kDim / 32)), n0 = 32 * (e % (kDim / 32));
    Acc c(0.0f);
#pragma unroll
    for (int s = 0; s < 4; ++s) mma_parts(grad.cols(16 * s, n0), q_up.cols(16 * s, k0), c);
#pragma unroll
    for (int s = 0; s < 4; ++s)
      *reinterpret_cast<FloatVec<4>*>(ends + (k0 + (lane & 31)) * kDim + n0 + four_row(s)) = four(c, s);
  }
  float* factors = a.chain.factors + index * kFactors;
  if (threadIdx.x < kChunk) factors[threadIdx.x] = g.down[threadIdx.x];
  if (threadIdx.x == 0) factors[kChunk] = g.whole;
}

// Sums of a result's columns, over the 32 lanes of a half: each lane with bit 4 clear
// gets that of one register, sums_register().
__device__ __forceinline__ float column_sums(const Acc& c) {
  const int lane = threadIdx.x & 63;
  float e[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) e[i] = c[i];
#pragma unroll
  for (int d = 1, n = 8; n; d <<= 1, n >>= 1) {
    const bool high = lane & d;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float send = high ? e[i] : e[i + n], keep = high ? e[i + n] : e[i];
      e[i] = keep + __shfl_xor(send, d, kWave);
    }
  }
  return e[0] + __shfl_xor(e[0], 16, kWave);
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
  using STile = Tile<E, P, kKey, 64>;
  using KTile = Tile<E, P, kChunk, kKey>;
  using Fine = Tile<E, F::mid, kChunk, 64>;
  constexpr int kFirst = 2 * Half::bytes + 2 * Fine::bytes + STile::bytes;
  constexpr int kSecond = 3 * Half::bytes + 2 * KTile::bytes;
  __shared__ __align__(16) char space[kFirst > kSecond ? kFirst : kSecond];
  __shared__ Gates g;
  __shared__ float dots[3][2][kChunk], crossing[2][3][32], inner[4];
  const Half grad(space), u(space + Half::bytes), x(space + 2 * Half::bytes);
  const Fine du(space + 2 * Half::bytes), solve(space + 2 * Half::bytes + Fine::bytes);
  const STile state(space + 2 * Half::bytes + 2 * Fine::bytes);
  const Half n_tile(space), m_tile(space + Half::bytes), mb_tile(space + 2 * Half::bytes);
  const KTile q(space + 3 * Half::bytes), k(space + 3 * Half::bytes + KTile::bytes);
  constexpr int kTiles = kKey / 64;
  const int64_t work = seq::block_index();
  const int group = a.p.heads / a.p.key_heads;
  if (work >= a.count / group) return;
  // The heads of a key are chunks apart.
  const int64_t first = work % a.p.chunks + work / a.p.chunks * a.p.chunks * group;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m0 = 32 * (wave & 1), side = wave >> 1, token = m0 + (lane & 31);
  const int i0 = wave ? 32 : 0, j0 = wave == 2 ? 32 : 0;  // of the triangles, waves 0 .. 2
  Acc dq_all[kTiles], dk_all[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) dq_all[t] = dk_all[t] = Acc(0.0f);
  for (int member = 0; member < group; ++member) {
    const int64_t index = first + int64_t(member) * a.p.chunks;
    const Place at(a.p, index);
    __syncthreads();
    if (wave == 0) load_gates(g, a.gate, a.beta, at);
    Acc dq[kTiles], z[kTiles], y[kTiles], n(0.0f), m(0.0f);
#pragma unroll
    for (int t = 0; t < kTiles; ++t) dq[t] = z[t] = y[t] = Acc(0.0f);
    float found = 0.0f, both = 0.0f;
    const float* from = a.kept.solve + index * kChunk * kChunk;
    load_tile<float>(solve, from, kChunk, kChunk, kChunk, Keep{});
    const float* u_row = a.kept.updates + (index * kChunk + token) * kDim;
    const int64_t row = ((int64_t(at.b) * a.p.tokens + at.t0 + token) * a.p.heads + at.h) * a.p.dim;
#pragma unroll
    for (int d0 = 0; d0 < kDim; d0 += 64) {
      if (d0 >= a.p.dim) break;
      const int wide = a.p.dim - d0;
      if (d0) __syncthreads();
      load_tile<T>(grad, a.grad.at(at.b, at.t0, at.h) + d0, a.grad.s.token, a.grad.p ? at.valid : 0, wide, Keep{});
      load_tile<float>(u, a.kept.updates + index * kChunk * kDim + d0, kDim, kChunk, wide, Keep{});
      load_tile<float>(du, a.du + index * kChunk * kDim + d0, kDim, kChunk, wide, Keep{});
      load_tile<float>(state, a.kept.starts + index * kKey * kDim + d0, kDim, a.p.key_dim, wide, Keep{});
      __syncthreads();
      // dR of the wave's tokens and 32 dimensions.
      Acc r(0.0f);
      for (int s = m0 / 16; s < 4; ++s) mma_parts(du.cols(16 * s, 32 * side), solve.cols(16 * s, m0), r);
      __syncthreads();
      const float b = g.beta[token];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int col = 32 * side + four_row(s);
        const FloatVec<4> dr = four(r, s);
        x.put(token, col, Parts<E, P, 4>(dr));
        if (token < at.rows && col < wide) {
          FloatVec<4> out = b * dr;
          if (token < at.valid) {
            const FloatVec<4> uu = *reinterpret_cast<const FloatVec<4>*>(u_row + d0 + col);
#pragma unroll
            for (int i = 0; i < 4; ++i) found += uu[i] * dr[i];
          } else {
            out = FloatVec<4>(0.0f);
          }
          *reinterpret_cast<Vec<T, 4>*>(a.dv + row + d0 + col) = from_float<T, 4>(out);
        }
      }
      __syncthreads();
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (wave < 3) {
          const auto left = u.rows(j0, 16 * s);
          mma_parts(left, grad.rows(i0, 16 * s), n);
          mma_parts(left, x.rows(i0, 16 * s), m);
        }
        const auto go = grad.rows(m0, 16 * s), dr = x.rows(m0, 16 * s);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const auto left = state.rows(32 * (side + 2 * t), 16 * s);
          mma_parts(left, go, dq[t]);
          mma_parts(left, dr, z[t]);
        }
      }
      __syncthreads();
      // dS', and its product with S.
      const float* start = a.kept.starts + index * kKey * kDim + d0;
      load_tile<float>(state, a.ends + index * kKey * kDim + d0, kDim, a.p.key_dim, wide,
                       [&](int row, int col, auto& ds) {
                         if (row < a.p.key_dim && col < wide) {
                           const FloatVec<8> s = to_float<float, 8>(load_global<float>(start + row * kDim + col, true));
#pragma unroll
                           for (int i = 0; i < 8; ++i) both += ds[i] * s[i];
                         }
                       });
      __syncthreads();
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const auto right = u.rows(m0, 16 * s);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) mma_parts(state.rows(32 * (side + 2 * t), 16 * s), right, y[t]);
      }
    }
    const float up = g.up[token], down = g.down[token], beta = g.beta[token];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      dq[t] *= a.p.scale * up;
      z[t] *= -up;
      y[t] *= down;
    }
    __syncthreads();
    if (wave < 3) {
      const int i = i0 + (lane & 31);
      const float b = g.beta[i];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int j = j0 + four_row(s);
        FloatVec<4> nn = four(n, s), mm = four(m, s);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float d = g.decay(i, j + e);
          nn[e] = j + e <= i ? a.p.scale * d * nn[e] : 0.0f;
          mm[e] = j + e < i ? -d * mm[e] : 0.0f;
        }
        n_tile.put(i, j, Parts<E, P, 4>(nn));
        m_tile.put(i, j, Parts<E, P, 4>(mm));
        mb_tile.put(i, j, Parts<E, P, 4>(b * mm));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          n[4 * s + e] = nn[e];
          m[4 * s + e] = b * mm[e];
        }
      }
    }
    load_tile<T>(q, a.q.at(at.b, at.t0, at.key_head), a.q.s.token, at.valid, a.p.key_dim, Keep{});
    load_tile<T>(k, a.k.at(at.b, at.t0, at.key_head), a.k.s.token, at.valid, a.p.key_dim, Keep{});
    __syncthreads();
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
      const float column = column_sums(n);
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
    for (int s = 0; s < (m0 ? 4 : 2); ++s) {
      const auto nn = n_tile.rows(m0, 16 * s), mm = m_tile.rows(m0, 16 * s);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const auto left = k.cols(16 * s, 32 * (side + 2 * t));
        mma_parts(left, nn, dq[t]);
        mma_parts(left, mm, z[t]);
      }
    }
    for (int s = m0 / 16; s < 4; ++s) {
      const auto nn = n_tile.cols(16 * s, m0), mm = mb_tile.cols(16 * s, m0);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        mma_parts(q.cols(16 * s, 32 * (side + 2 * t)), nn, y[t]);
        mma_parts(k.cols(16 * s, 32 * (side + 2 * t)), mm, y[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      dq_all[t] += dq[t];
      dk_all[t] += beta * z[t] + y[t];
    }
    const float all[3] = {reads, writes, found};
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const float sum = all[i] + __shfl_xor(all[i], 32, kWave);
      if (lane < 32) dots[i][side][token] = sum;
    }
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) both += __shfl_xor(both, d, kWave);
    if (lane == 0) inner[wave] = both;
    __syncthreads();
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
          const float gate = float(*a.gate.at(at.b, at.t0 + lane, at.h));
          const float raw = float(*a.beta.at(at.b, at.t0 + lane, at.h));
          dgate = (total + rest) * sigmoid(-gate);
          dbeta = (dots[2][0][lane] + dots[2][1][lane]) * sigmoid(-raw);
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
                  a.du, a.ends, grad_state};
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
  return size_t(delta_chunks(*desc)) *
         (delta_left_bytes(*desc, delta_parts_in(*desc) + delta_parts_mid(*desc)) +
          (delta::kFactors + (delta::kChunk + delta::padded(desc->key_dim)) * wide) * sizeof(float));
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
    a.kept = delta_kept(*desc, static_cast<float*>(const_cast<void*>(kept)), true);
    const int64_t wide = delta::padded(desc->dim);
    a.chain.factors = static_cast<float*>(workspace);
    a.du = a.chain.factors + n * delta::kFactors;
    a.ends = a.du + n * delta::kChunk * wide;
    a.chain.left = reinterpret_cast<delta::bf16*>(a.ends + n * delta::padded(desc->key_dim) * wide);
    a.chain.right = a.chain.left + n * delta_left_bytes(*desc, delta_parts_in(*desc)) / 2;
    a.dq = static_cast<T*>(grad_q);
    a.dk = static_cast<T*>(grad_k);
    a.dv = static_cast<T*>(grad_v);
    a.dgate = static_cast<T*>(grad_gate);
    a.dbeta = static_cast<T*>(grad_beta);
    a.count = n;
    const hipStream_t s = as_stream(stream);
    if (desc->key_dim <= 64)
      return desc->dim <= 64 ? delta::backward<T, 64, 64>(a, grad_last, grad_state, s)
                             : delta::backward<T, 64, 128>(a, grad_last, grad_state, s);
    return desc->dim <= 64 ? delta::backward<T, 128, 64>(a, grad_last, grad_state, s)
                           : delta::backward<T, 128, 128>(a, grad_last, grad_state, s);
  });
}
