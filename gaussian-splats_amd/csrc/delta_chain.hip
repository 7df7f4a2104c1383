// The gated delta rule's states from chunk to chunk, the one part of it that
// cannot run over all chunks at once (delta_scan.h):
//   forward, in order:   U = F + L S,                  S' = e^(G_C) S + R (e^(G_C - G) U)
//   backward, reversed:  dU = F + e^(G_C - G) L dS,    dS' = e^(G_C) dS + Y + R dU
// with L = -W, R = K^T forwards and L = K, R = -W^T backwards.
//
// Columns of a state do not mix: a wave takes sixteen and keeps them in registers.  A
// 16 x 16 result holds rows 4 g .. 4 g + 3 of a column in the lanes' group g, and a
// product over 32 may take them in any order, so two results are the next product's
// second operand as they stand, if L and R have their columns in that order
// (fragment_at): nothing is exchanged between lanes or waves.  What the four waves of a
// workgroup share is L and R, which come through registers into LDS some chunks ahead,
// in the order in which lanes read them, with one barrier a chunk.
//
// A chunk is two products of a few hundred cycles behind each other, and a long
// sequence of few heads has hundreds of chunks while most of the GPU is idle.  So it
// is cut into segments, which all run at once, from a state of zeros and, without F and
// Y, from the unit matrix: that is what a segment adds and what it maps a state to.
// Each workgroup of the second pass starts from the product of the maps before it and
// walks its segment once more.
//
// Measured, 12 heads of 64 x 64, 625 chunks, bfloat16: 823 us forwards and 827 backwards
// in one pass, 169 (68 and 101) and 240 (111 and 129) in 21 segments.  Many segments are
// bound by what they move, counted: forwards 163 and 286 MB, backwards 241 and 410, which is
// 2.2 to 3.2 TB/s of a copy's 5.1; a walk of few by a chunk's two products behind each
// other and their barrier, some 1.5 us.
#include "delta_scan.h"

namespace gs {
namespace delta {
namespace {

constexpr int kCols = 16;  // of a wave
constexpr int kPiece = kWave * 8;  // elements of a fragment

using Acc4 = FloatVec<4>;

// Two results, split, as a second operand.
template <int P>
__device__ __forceinline__ void operand(const Acc4& a, const Acc4& b, Frag<bf16> (&to)[P]) {
  const Parts<bf16, P, 8> v(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
  for (int i = 0; i < P; ++i) to[i] = v.v[i];
}

__device__ __forceinline__ Acc4 mma16(const Frag<bf16>& a, const Frag<bf16>& b, const Acc4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

enum Pass { kWhole, kMaps, kAgain };

// kWaves: of a workgroup.
template <int kKey, int kDim, int PL, int PR, int PS, bool kBack, int kPass, int kWaves>
struct Walk {
  static constexpr int kSteps = kKey / 32, kTiles = kKey / 16;
  static constexpr int kLeft = PL * 4 * kSteps, kRight = PR * kTiles * 2, kPieces = kLeft + kRight;
  static constexpr int kLoads = (kPieces + kWaves - 1) / kWaves;  // of a thread
  // Two chunks in LDS where they fit, and one or two more on their way, where the
  // registers hold them: two ahead, the maps of 625 chunks forwards take 71 us, one
  // ahead 98; at keys of 128 two spill (32 chunks, 8 heads, again: 137 us, 52 with one).
  // Backwards, with states on their way too, two spill earlier (the same maps in bfloat16:
  // 20 registers, 129 us, 111 with one; the passes of float32 as well).
  static constexpr int kRing = kPieces <= 64 ? 2 : 1;
  static constexpr int kAhead = kKey == 64 && (kWaves == 8 ? kPieces <= 24 && !kBack
                                                           : kWaves == 4 && kPieces > 24 && kPieces <= (kBack ? 32 : 48))
                                    ? 2 : 1;
  static constexpr int kPerSimd = kWaves == 8 ? 2 : 1;
  static constexpr int kFactorsAt = kRing * kPieces * kPiece * 2;  // bytes
  static constexpr int kShared = kFactorsAt + kRing * kFactors * 4;
  // What later kernels take in one bfloat16 part is stored so.
  using State = std::conditional_t<(kBack ? PL : PR) == 1, bf16, float>;
  using Row = std::conditional_t<kBack, float, State>;

  // A chunk on its way: the workgroup's share of L and R, and the wave's own rows.
  struct Stage {
    Frag<bf16> piece[kLoads];
    Acc4 factors, rows[4], next[kBack ? kTiles : 1];

    // id: the chunk of the head; key: that of the keys that its group shares.
    // col < 0: the unit matrix's, all lanes of which load one place that they do not take.
    __device__ __forceinline__ void load(const ChainArgs& a, int64_t id, int64_t key, int col) {
      const int thread = threadIdx.x, wave = thread >> 6, lane = thread & 63;
      const bf16* l = a.chain.left + (kBack ? key : id) * kLeft * kPiece + lane * 8;
      const bf16* r = a.chain.right + (kBack ? id : key) * kRight * kPiece + lane * 8;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int at = min(i * kWaves + wave, kPieces - 1);
        piece[i] = *reinterpret_cast<const Frag<bf16>*>(at < kLeft ? l + at * kPiece : r + (at - kLeft) * kPiece);
      }
      factors = *reinterpret_cast<const Acc4*>(a.chain.factors + id * kFactors + 4 * min(thread, kFactors / 4 - 1));
      const int group = lane >> 4;
      const float* x = a.rows_from + id * kDim * kChunk + (col < 0 ? 0 : col * kChunk + 4 * group);
#pragma unroll
      for (int m = 0; m < 4; ++m) rows[m] = *reinterpret_cast<const Acc4*>(x + 16 * m);
      if constexpr (kBack) {
        const float* y = a.states_from + id * kDim * kKey + (col < 0 ? 0 : col * kKey + 4 * group);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) next[t] = *reinterpret_cast<const Acc4*>(y + 16 * t);
      }
    }
    __device__ __forceinline__ void put(char* space, int slot) const {
      const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
      bf16* to = reinterpret_cast<bf16*>(space) + slot * kPieces * kPiece + lane * 8;
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        *reinterpret_cast<Frag<bf16>*>(to + min(i * kWaves + wave, kPieces - 1) * kPiece) = piece[i];
      *reinterpret_cast<Acc4*>(space + kFactorsAt + slot * kFactors * 4 +
                               16 * min(int(threadIdx.x), kFactors / 4 - 1)) = factors;
    }
  };

  // One chunk: s goes on by it; its rows and the state before it are stored.
  static __device__ __forceinline__ void step(const ChainArgs& a, const char* space, int slot, int64_t id,
                                              int col, Acc4 (&s)[kTiles], const Acc4 (&rows)[4],
                                              const Acc4 (&next)[kBack ? kTiles : 1]) {
    const int lane = threadIdx.x & 63, group = lane >> 4;
    const bf16* pieces = reinterpret_cast<const bf16*>(space) + slot * kPieces * kPiece + lane * 8;
    const float* factors = reinterpret_cast<const float*>(space + kFactorsAt) + slot * kFactors;
    // Fragments in the order in which they are taken, eight of them ahead; the
    // scheduler would read each where it is needed.
    constexpr int kGroup = 8, kGroups = kPieces / kGroup;
    static_assert(kLeft % kGroup == 0 && kRight % kGroup == 0, "whole groups");
    Frag<bf16> f[2][kGroup], b[PS];
    const auto read = [&](int g) {
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        const int at = g * kGroup + i, r = at - kLeft;
        const int place = at < kLeft ? (at % (4 * PL)) * kSteps + at / (4 * PL)
                                     : kLeft + (r % (kTiles * PR)) * 2 + r / (kTiles * PR);
        f[g & 1][i] = *reinterpret_cast<const Frag<bf16>*>(pieces + place * kPiece);
      }
    };
    Acc4 x[4], down[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) x[m] = kBack ? Acc4(0.0f) : rows[m];
    read(0);
#pragma unroll
    for (int m = 0; m < 4; ++m) down[m] = *reinterpret_cast<const Acc4*>(factors + 16 * m + 4 * group);
    const float whole = factors[kChunk];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      if (g + 1 < kGroups) read(g + 1);
      __builtin_amdgcn_sched_barrier(0x76);  // no product and no read of LDS across
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        const int at = g * kGroup + i, r = at - kLeft;
        const Frag<bf16>& part = f[g & 1][i];
        if (at < kLeft) {
          const int st = at / (4 * PL), p = at / 4 % PL, m = at % 4;
          if (at % (4 * PL) == 0) operand<PS>(s[2 * st], s[2 * st + 1], b);
#pragma unroll
          for (int j = 0; j < PS; ++j)
            if (p + j < (PL > PS ? PL : PS)) x[m] = mma16(part, b[j], x[m]);
          continue;
        }
        if (r == 0) {
          if constexpr (kPass != kMaps) {
            State* to = static_cast<State*>(a.states) + (id * kDim + col) * kKey + 4 * group;
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
              *reinterpret_cast<Vec<State, 4>*>(to + 16 * t) = from_float<State, 4>(s[t]);
          }
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            s[t] *= whole;
            if constexpr (kBack) s[t] += next[t];
          }
          Row* out = static_cast<Row*>(a.rows) + (id * kDim + col) * kChunk + 4 * group;
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            if constexpr (kBack) x[m] = rows[m] + down[m] * x[m];
            if constexpr (kPass != kMaps)
              *reinterpret_cast<Vec<Row, 4>*>(out + 16 * m) = from_float<Row, 4>(x[m]);
            if constexpr (!kBack) x[m] = down[m] * x[m];
          }
        }
        const int st = r / (kTiles * PR), p = r / kTiles % PR, t = r % kTiles;
        if (r % (kTiles * PR) == 0) operand<PS>(x[2 * st], x[2 * st + 1], b);
#pragma unroll
        for (int j = 0; j < PS; ++j)
          if (p + j < (PR > PS ? PR : PS)) s[t] = mma16(part, b[j], s[t]);
      }
    }
  }
};

template <int kKey, int kDim, int PL, int PR, int PS, bool kBack, int kPass, int kWaves>
__global__ __launch_bounds__(kWaves * kWave)
__attribute__((amdgpu_waves_per_eu(Walk<kKey, kDim, PL, PR, PS, kBack, kPass, kWaves>::kPerSimd,
                                   Walk<kKey, kDim, PL, PR, PS, kBack, kPass, kWaves>::kPerSimd)))
void chain_kernel(ChainArgs a) {
  using W = Walk<kKey, kDim, PL, PR, PS, kBack, kPass, kWaves>;
  __shared__ __align__(16) char space[W::kShared];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, group = lane >> 4;
  const int64_t head = block_index();
  if (head >= a.heads) return;
  // Waves of columns; behind them, in the maps' pass, the unit matrix's.  The last
  // workgroup's spare waves take their share of L and R to LDS too, and no two waves store
  // to one place: rows and states may be walked in place (backwards), with nothing between
  // one wave's loads of them and another's stores.  In the passes that store, spare waves
  // have the padding's columns, which are zeros and exist up to kDim; in the maps' pass
  // they repeat the last wave's walk and store nothing.
  static_assert(kPass == kMaps || kDim / kCols % kWaves == 0, "spare waves' columns exist");
  const int own = (a.dim + kCols - 1) / kCols, all = own + W::kTiles;
  const int segment = blockIdx.z / a.blocks, ticket = int(blockIdx.z % a.blocks) * kWaves + wave;
  const int place = kPass == kMaps ? min(ticket, all - 1) : ticket;
  const bool unit = kPass == kMaps && place >= own;
  const int col = (unit ? place - own : place) * kCols + n;
  const int from = unit ? -1 : col;
  const int first = segment * a.each, count = min(a.each, a.chunks - first);
  const auto chunk_of = [&](int i) {
    const int c = first + min(i, count - 1);
    return kBack ? a.chunks - 1 - c : c;
  };
  const int64_t id0 = head * a.chunks, key0 = head / a.group * a.chunks;
  const auto load = [&](typename W::Stage& stage, int i) {
    const int c = chunk_of(i);
    stage.load(a, id0 + c, key0 + c, from);
  };
  Acc4 s[W::kTiles];
#pragma unroll
  for (int t = 0; t < W::kTiles; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * t + 4 * group + i;
      if constexpr (kPass == kMaps)
        s[t][i] = unit && row == col ? 1.0f : 0.0f;
      else
        s[t][i] = a.first && row < a.key_dim && col < a.dim
                      ? a.first[(head * a.key_dim + row) * a.dim + col]
                      : 0.0f;
    }
  typename W::Stage stage[W::kAhead];
#pragma unroll
  for (int i = 0; i < W::kAhead; ++i) load(stage[i], i);
  if constexpr (kPass == kAgain) {
    // What the segments before this one make of the state, of maps that the workgroup
    // reads once and puts in LDS, each while the one before is taken.  The state goes
    // in with all its bits, in three parts: a segment behind a sequence's end, whose map
    // is the unit matrix, leaves it as it is.
    constexpr int kMap = PS * W::kTiles * W::kSteps, kEach = kMap / kWaves;
    static_assert(kMap % kWaves == 0 && kMap <= W::kRing * W::kPieces, "a map has its place");
    Frag<bf16> piece[kEach];
    Acc4 y[W::kTiles];
    const int known = min(place, own - 1) * kCols + n;  // the maps' pass adds to no padding
    const auto fetch = [&](int g) {
      const int64_t at = head * a.segments + min(g, segment - 1);
      const bf16* map = a.maps + at * kMap * kPiece + lane * 8;
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        piece[i] = *reinterpret_cast<const Frag<bf16>*>(map + (i * kWaves + wave) * kPiece);
    };
    if (segment) fetch(0);
    bf16* held = reinterpret_cast<bf16*>(space) + lane * 8;
    for (int g = 0; g < segment; ++g) {
      const float* add = a.adds + ((head * a.segments + g) * kDim + known) * kKey + 4 * group;
#pragma unroll
      for (int t = 0; t < W::kTiles; ++t) y[t] = *reinterpret_cast<const Acc4*>(add + 16 * t);
      lds_barrier();
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        *reinterpret_cast<Frag<bf16>*>(held + (i * kWaves + wave) * kPiece) = piece[i];
      fetch(g + 1);
      lds_barrier();
#pragma unroll
      for (int st = 0; st < W::kSteps; ++st) {
        Frag<bf16> b[3];
        operand<3>(s[2 * st], s[2 * st + 1], b);
#pragma unroll
        for (int p = 0; p < PS; ++p)
#pragma unroll
          for (int t = 0; t < W::kTiles; ++t) {
            const Frag<bf16> f =
                *reinterpret_cast<const Frag<bf16>*>(held + ((p * W::kTiles + t) * W::kSteps + st) * kPiece);
#pragma unroll
            for (int j = 0; j < 3; ++j)
              if (p == 0 || p + j < PS) y[t] = mma16(f, b[j], y[t]);
          }
      }
#pragma unroll
      for (int t = 0; t < W::kTiles; ++t) s[t] = y[t];
    }
    if (segment) lds_barrier();
  }
  // No branch in the loop: at one the loads that are on their way would have to be
  // waited for.  Behind the last chunk it is loaded again.
  constexpr int kNext = kBack ? W::kTiles : 1;
  Acc4 rows[4], next[kNext], rows_then[4], next_then[kNext];
  const auto put = [&](int i, typename W::Stage& stage) {  // chunk i, on its way in the stage
    stage.put(space, i % W::kRing);
#pragma unroll
    for (int m = 0; m < 4; ++m) rows_then[m] = unit ? Acc4(0.0f) : stage.rows[m];
    if constexpr (kBack) {
#pragma unroll
      for (int t = 0; t < kNext; ++t) next_then[t] = unit ? Acc4(0.0f) : stage.next[t];
    }
    load(stage, i + W::kAhead);
  };
  const auto turn = [&] {
#pragma unroll
    for (int m = 0; m < 4; ++m) rows[m] = rows_then[m];
    if constexpr (kBack) {
#pragma unroll
      for (int t = 0; t < kNext; ++t) next[t] = next_then[t];
    }
  };
  // With two chunks in LDS the next one is put there while this one is taken, and the
  // one barrier keeps it from the chunk before; with one, it waits for that to end.
  const auto run = [&](int i, typename W::Stage& stage) {
    if constexpr (W::kRing == 2) {
      lds_barrier();
      put(i + 1, stage);
      W::step(a, space, i % 2, id0 + chunk_of(i), col, s, rows, next);
      turn();
    } else {
      lds_barrier();
      put(i, stage);
      turn();
      lds_barrier();
      W::step(a, space, 0, id0 + chunk_of(i), col, s, rows, next);
    }
  };
  constexpr int kLead = W::kRing - 1;
  if constexpr (kLead) {
    put(0, stage[0]);
    turn();
  }
  // The first ones before the loop: its waits then count the stores of the chunk before,
  // instead of waiting for all that is on its way as the loop's entry would have it.
  int i0 = 0;
  if (count >= W::kAhead) {
#pragma unroll
    for (int k = 0; k < W::kAhead; ++k) run(k, stage[(k + kLead) % W::kAhead]);
    for (i0 = W::kAhead; i0 + W::kAhead <= count; i0 += W::kAhead) {
#pragma unroll
      for (int k = 0; k < W::kAhead; ++k) run(i0 + k, stage[(k + kLead) % W::kAhead]);
    }
  }
#pragma unroll
  for (int k = 0; k < W::kAhead - 1; ++k)
    if (i0 + k < count) run(i0 + k, stage[(k + kLead) % W::kAhead]);
  if constexpr (kPass == kMaps) {
    if (ticket >= all) return;
    const int64_t at = head * a.segments + segment;
    if (unit) {
      // As a first operand: row 16 t + 4 g + i of column col, in the order of fragments.
      bf16* to = a.maps + at * PS * W::kTiles * W::kSteps * kPiece;
#pragma unroll
      for (int t = 0; t < W::kTiles; ++t) {
        const Parts<bf16, PS, 4> v(s[t]);
#pragma unroll
        for (int p = 0; p < PS; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            to[p * W::kTiles * W::kSteps * kPiece +
               fragment_at(16 * t + 4 * group + i, col & ~3, W::kSteps) + (col & 3)] = v.v[p][i];
      }
    } else {
      float* to = a.adds + (at * kDim + col) * kKey + 4 * group;
#pragma unroll
      for (int t = 0; t < W::kTiles; ++t) *reinterpret_cast<Acc4*>(to + 16 * t) = s[t];
    }
  } else if (a.last && col < a.dim && segment + 1 == a.segments) {
#pragma unroll
    for (int t = 0; t < W::kTiles; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * t + 4 * group + i;
        if (row < a.key_dim) a.last[(head * a.key_dim + row) * a.dim + col] = s[t][i];
      }
  }
}

template <int kKey, int kDim, int PI, int PM, bool kBack, int kPass, int kWaves>
int launch_pass(ChainArgs a, hipStream_t s) {
  constexpr int PL = kBack ? PI : PM, PR = kBack ? PM : PI;
  const int waves = (a.dim + kCols - 1) / kCols + (kPass == kMaps ? kKey / kCols : 0);
  a.blocks = (waves + kWaves - 1) / kWaves;
  dim3 grid = seq::grid_of(a.heads);
  grid.z = unsigned(a.blocks * a.segments);
  chain_kernel<kKey, kDim, PL, PR, PM, kBack, kPass, kWaves><<<grid, kWaves * kWave, 0, s>>>(a);
  return check_launch("delta_scan chain");
}

template <int kKey, int kDim, int PI, int PM, bool kBack>
int launch(ChainArgs a, hipStream_t s) {
  // A map's waves are its columns' and the unit matrix's: eight of them share L and R
  // where 256 registers hold a wave's part (float16 of 128, 16 heads, 8 segments of 16:
  // 63 us, 102 with four).  Again they do not: there they spill (113 us, 156 with eight).
  constexpr int kMapWaves = PI <= 2 ? 8 : 4, kColWaves = 4;
  a.each = (a.chunks + a.segments - 1) / a.segments;
  a.segments = (a.chunks + a.each - 1) / a.each;
  if (a.segments > 1) {
    GS_TRY((launch_pass<kKey, kDim, PI, PM, kBack, kMaps, kMapWaves>(a, s)));
    return launch_pass<kKey, kDim, PI, PM, kBack, kAgain, kColWaves>(a, s);
  }
  // A CU alone gets some 40 GB/s from behind its L2, and a barrier waits for the slowest
  // of its waves: with CUs to spare, workgroups are smaller.  A wave alone, where 512
  // registers hold its part and a chunk on its way (8 heads of 64, 19 chunks, bfloat16:
  // 29 us, 37 with four waves), else two (12 heads of 40 x 72, 13 chunks, float32: 31 us,
  // 40 with four, and one spills; 8 heads of 128, 32 chunks: 136, 156 with four).  With
  // keys of 64 that holds up to two such waves a CU (128 heads of 64, 19 chunks,
  // backwards: bfloat16 61 us, 72 with four; float32 72 and 99; 192 heads: 77 and 75),
  // with wider ones for one (64 heads of 128, float32, backwards: 186 us with two waves,
  // 144 with four).
  const int64_t waves = a.heads * ((a.dim + kCols - 1) / kCols);
  constexpr int64_t kSpare = kKey == 64 ? 512 : 256;
  if constexpr ((PI + PM) * kKey <= 192) {
    if (waves <= kSpare) return launch_pass<kKey, kDim, PI, PM, kBack, kWhole, 1>(a, s);
  } else if (waves <= kSpare) {
    return launch_pass<kKey, kDim, PI, PM, kBack, kWhole, 2>(a, s);
  }
  return launch_pass<kKey, kDim, PI, PM, kBack, kWhole, kColWaves>(a, s);
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

// Segments of a sequence: as many as give every CU a workgroup of the second pass, of
// eight chunks and more, from four on.  Four take between a fifth less and a tenth more
// than one pass (12 heads of 64, 32 chunks: 37 us for 45 in bfloat16, 53 for 68 in
// float32; 8 heads of 128: 61 for 69, 32 heads: 78 for 70), three gain nothing at 32
// chunks (35 for 36), twenty-one are five times as quick.  So 65 heads of 64 and more
// (33 above 64) walk in one pass, however long: a forward call of 625 chunks in bfloat16 takes
// 1.90 ms for 64 heads in four segments and 2.18 for 65 in none.
int chain_segments(int64_t heads, int64_t chunks, int dim) {
  const int64_t blocks = (dim + 63) / 64;
  const int64_t most = std::min<int64_t>({chunks / 8, 256 / std::max<int64_t>(heads * blocks, 1), 32});
  return most < 4 ? 1 : int(most);
}

int launch_chain(const ChainArgs& a, int key_wide, int wide, int parts_in, bool backward,
                 hipStream_t s) {
  return backward ? launch_sizes<true>(a, key_wide, wide, parts_in, s)
                  : launch_sizes<false>(a, key_wide, wide, parts_in, s);
}

}  // namespace delta
}  // namespace gs
