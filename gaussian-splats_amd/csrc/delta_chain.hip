// The gated delta rule's states from chunk to chunk, the one part of it that
// cannot run over all chunks at once (delta_scan.h):
//   forward, in order:   U = F + L S,          S' = e^(G_C) S + R (e^(G_C - G) U)
//   backward, reversed:  dU = F + e^(G_C - G) L dS,  dS' = e^(G_C) dS + Y + R dU
// with L = -W, R = K^T forwards and L = K, R = -W^T backwards.
//
// Columns of a state do not mix, so a workgroup takes sixteen of them; its four
// waves share the 64 rows of U and the rows of S.  A chunk is two small products
// with an exchange through LDS behind each, so the time is that of the exchanges:
// factors are loaded some chunks ahead straight into the registers in which the
// matrix cores take them, the state and the rows lie in LDS turned, in which the
// other operand is read by 16 bytes, and a barrier waits for LDS alone.
//
// Measured, 12 heads of 64 x 64, 625 chunks, bfloat16: 823 us, 1.3 a
// chunk.
#include "delta_scan.h"

namespace gs {
namespace delta {
namespace {

constexpr int kCols = 16;

using Acc4 = FloatVec<4>;

// All of the workgroup's writes to LDS are there; loads and stores of global memory
// go on.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <int kKey, int kDim, int PL, int PR, int PS, bool kBack>
struct Stage {
  static constexpr int kSteps = kKey / 32, kTiles = kKey / 64;
  Frag<bf16> left[PL][kSteps], right[PR][kTiles][2];
  Acc4 rows, down;
  float whole;
  Acc4 next[kTiles];  // backward

  __device__ __forceinline__ void load(const ChainArgs& a, int64_t id, int col) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, group = lane >> 4;
    const bf16* l = a.chain.left + (id * PL * kChunk + 16 * wave + row) * kKey + 8 * group;
#pragma unroll
    for (int i = 0; i < PL; ++i)
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        left[i][s] = *reinterpret_cast<const Frag<bf16>*>(l + i * kChunk * kKey + 32 * s);
    const bf16* r = a.chain.right + (id * PR * kKey + 16 * wave * kTiles + row) * kChunk + 8 * group;
#pragma unroll
    for (int i = 0; i < PR; ++i)
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int s = 0; s < 2; ++s)
          right[i][t][s] =
              *reinterpret_cast<const Frag<bf16>*>(r + (i * kKey + 16 * t) * kChunk + 32 * s);
    const float* x = a.rows + (id * kChunk + 16 * wave + 4 * group) * kDim + col;
#pragma unroll
    for (int i = 0; i < 4; ++i) rows[i] = x[i * kDim];
    const float* f = a.chain.factors + id * kFactors;
    down = *reinterpret_cast<const Acc4*>(f + 16 * wave + 4 * group);
    whole = f[kChunk];
    if constexpr (kBack) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const float* y = a.states + (id * kKey + 16 * (wave * kTiles + t) + 4 * group) * kDim + col;
#pragma unroll
        for (int i = 0; i < 4; ++i) next[t][i] = y[i * kDim];
      }
    }
  }
};

template <int P>
__device__ __forceinline__ void put_turned(bf16* to, int part, const Acc4& x) {
  const Parts<bf16, P, 4> v(x);
#pragma unroll
  for (int i = 0; i < P; ++i) *reinterpret_cast<Vec<bf16, 4>*>(to + i * part) = v.v[i];
}

template <int kKey, int kDim, int PL, int PR, int PS, bool kBack, int kAhead>
__global__ __launch_bounds__(kThreads, 1) void chain_kernel(ChainArgs a) {
  using S = Stage<kKey, kDim, PL, PR, PS, kBack>;
  constexpr int kPitchS = kKey + 8, kPitchX = kChunk + 8;
  __shared__ __align__(16) bf16 states[PS][kCols][kPitchS], rows[PS][kCols][kPitchX];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, group = lane >> 4;
  const int col = blockIdx.x * kCols + n;
  const int64_t head = blockIdx.y + int64_t(blockIdx.z) * gridDim.y;
  if (head >= a.heads) return;
  const int64_t id0 = head * a.chunks;
  const auto chunk_of = [&](int i) { return id0 + (kBack ? a.chunks - 1 - i : i); };
  Acc4 s[S::kTiles];
#pragma unroll
  for (int t = 0; t < S::kTiles; ++t) {
    const int row = 16 * (wave * S::kTiles + t) + 4 * group;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      s[t][i] = a.first && row + i < a.key_dim && col < a.dim
                    ? a.first[(head * a.key_dim + row + i) * a.dim + col]
                    : 0.0f;
    put_turned<PS>(&states[0][n][row], kCols * kPitchS, s[t]);
  }
  S stage[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (i < a.chunks) stage[i].load(a, chunk_of(i), col);
  lds_barrier();
  for (int i0 = 0; i0 < a.chunks; i0 += kAhead) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k;
      if (i >= a.chunks) break;
      const S& f = stage[k];
      const int64_t id = chunk_of(i);
      Acc4 x(0.0f), x2(0.0f);
#pragma unroll
      for (int st = 0; st < S::kSteps; ++st) {
        Frag<bf16> b[PS];
#pragma unroll
        for (int j = 0; j < PS; ++j)
          b[j] = *reinterpret_cast<const Frag<bf16>*>(&states[j][n][32 * st + 8 * group]);
#pragma unroll
        for (int p = 0; p < PL; ++p)
#pragma unroll
          for (int j = 0; j < PS; ++j)
            if (p + j < (PL > PS ? PL : PS)) {
              Acc4& to = (p + j) & 1 ? x2 : x;
              to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.left[p][st], b[j], to, 0, 0, 0);
            }
      }
      x += x2;
      x = kBack ? f.rows + f.down * x : f.rows + x;
      put_turned<PS>(&rows[0][n][16 * wave + 4 * group], kCols * kPitchX, kBack ? x : f.down * x);
      {
        float* to = a.rows + (id * kChunk + 16 * wave + 4 * group) * kDim + col;
#pragma unroll
        for (int r = 0; r < 4; ++r) to[r * kDim] = x[r];
      }
#pragma unroll
      for (int t = 0; t < S::kTiles; ++t) {
        float* to = a.states + (id * kKey + 16 * (wave * S::kTiles + t) + 4 * group) * kDim + col;
#pragma unroll
        for (int r = 0; r < 4; ++r) to[r * kDim] = s[t][r];
        s[t] *= f.whole;
        if constexpr (kBack) s[t] += f.next[t];
      }
      lds_barrier();
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        Frag<bf16> b[PS];
#pragma unroll
        for (int j = 0; j < PS; ++j)
          b[j] = *reinterpret_cast<const Frag<bf16>*>(&rows[j][n][32 * st + 8 * group]);
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t)
#pragma unroll
          for (int p = 0; p < PR; ++p)
#pragma unroll
            for (int j = 0; j < PS; ++j)
              if (p + j < (PR > PS ? PR : PS))
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.right[p][t][st], b[j], s[t], 0, 0, 0);
      }
#pragma unroll
      for (int t = 0; t < S::kTiles; ++t)
        put_turned<PS>(&states[0][n][16 * (wave * S::kTiles + t) + 4 * group], kCols * kPitchS, s[t]);
      if (i + kAhead < a.chunks) stage[k].load(a, chunk_of(i + kAhead), col);
      lds_barrier();
    }
  }
  if (a.last && col < a.dim) {
#pragma unroll
    for (int t = 0; t < S::kTiles; ++t) {
      const int row = 16 * (wave * S::kTiles + t) + 4 * group;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (row + r < a.key_dim) a.last[(head * a.key_dim + row + r) * a.dim + col] = s[t][r];
    }
  }
}

template <int kKey, int kDim, int PI, int PM, bool kBack>
int launch(const ChainArgs& a, hipStream_t s) {
  // Registers for the chunks ahead: a stage takes 33 to 120 of them.
  constexpr int kAhead = kKey == 64 && PM == 2 ? 4 : PM == 2 ? 3 : 2;
  constexpr int kMost = 32768;
  const unsigned y = unsigned(std::min<int64_t>(a.heads, kMost));
  const dim3 grid(unsigned((a.dim + kCols - 1) / kCols), y, unsigned((a.heads + y - 1) / y));
  constexpr int PL = kBack ? PI : PM, PR = kBack ? PM : PI;
  chain_kernel<kKey, kDim, PL, PR, PM, kBack, kAhead><<<grid, kThreads, 0, s>>>(a);
  return check_launch("delta_scan chain");
}

template <int kKey, int kDim, bool kBack>
int launch_parts(const ChainArgs& a, int parts_in, hipStream_t s) {
  if (parts_in == 1) return launch<kKey, kDim, 1, 2, kBack>(a, s);
  if (parts_in == 2) return launch<kKey, kDim, 2, 2, kBack>(a, s);
  return launch<kKey, kDim, 3, 3, kBack>(a, s);
}

template <bool kBack>
int launch_sizes(const ChainArgs& a, int key_wide, int wide, int parts_in, hipStream_t s) {
  if (key_wide == 64)
    return wide == 64 ? launch_parts<64, 64, kBack>(a, parts_in, s)
                      : launch_parts<64, 128, kBack>(a, parts_in, s);
  return wide == 64 ? launch_parts<128, 64, kBack>(a, parts_in, s)
                    : launch_parts<128, 128, kBack>(a, parts_in, s);
}

}  // namespace

int launch_chain(const ChainArgs& a, int key_wide, int wide, int parts_in, bool backward,
                 hipStream_t s) {
  return backward ? launch_sizes<true>(a, key_wide, wide, parts_in, s)
                  : launch_sizes<false>(a, key_wide, wide, parts_in, s);
}

}  // namespace delta
}  // namespace gs
