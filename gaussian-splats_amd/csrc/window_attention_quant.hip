// The window cache held in 4 bits: a step of each of several streams over it, and
// its filling from a prefill.
//
// A row of keys or values is cut into blocks of 32 elements.  A block has one
// power of two, 2^(floor(log2 max|x|) - 2), kept as a byte (the exponent + 127), and
// a 4-bit code an element: a sign, and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times the
// power, the nearest to x (of two as near the one with the even code, 6 beyond 6).
// That is the microscaling format MXFP4 of the Open Compute Project, 4.25 bits an
// element, which gfx950 converts in one instruction for two elements with their
// power applied: exactly, since a code and a power of two are a value of any of the
// inputs' types.  A block with an infinity or a NaN has the byte 255 and is NaN.
//
// The step is that of a cache in the inputs' type (one pass, running maximum and
// sum, slots shared out over workgroups and joined in order), bound by the cache's
// bytes.  The first product may take the elements of a row in any order, if the
// query has the same: a lane's half takes the first or the second half of a row, 16
// or 32 bytes in a piece.  Values are converted on their way into LDS, from which
// the second product reads them turned.  A wave has a quarter of the bytes in
// flight that it has with 16-bit elements, so more waves share a CU: LDS is used
// twice, for the values' tiles and for the join of the waves.
//
// Codes are exact in 16 bits, so all that an output loses before its own rounding is
// what its probabilities lose on their way into the second product.  They go in as two
// numbers of the type: the result's 32 columns are 16 heads twice, and the upper ones take
// the second part, in products that would else multiply columns without a head.  Once
// rounded probabilities left 0.0021 (2-norm, bfloat16) where one rounding leaves 0.0017,
// in 65 us a call instead of 66; from 17 heads a key on there are two tiles for one
// (32 heads a key: 118 us for 81, and 158 with both parts in 32 columns).
//
// Measured, bfloat16, 32 streams of up to 8176 slots, 32 heads of 128 on 8: 66 us a call
// for 259 MB; the step's kernel 58 us, 4.5 TB/s, the join 5; the cache in 16 bits takes
// 189.  Three workgroups a CU leave 168 registers, and rows of 128 spill 17 that every
// tile reads again.  In float32 (328 us) one workgroup a CU, for its registers and LDS,
// and float32's products at a seventh of the rate bound it.
#include "attention_tile.h"

namespace gs {
namespace {

using namespace att;

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kKeys = 32;  // of a wave's tile
constexpr int kBlock = 32;  // elements that share a power of two

struct Cache {
  uint8_t* codes;      // [batch, kv_heads, slots, dim / 2], the even element in the low half
  uint8_t* exponents;  // [batch, kv_heads, slots, dim / 32]
};

struct StepArgs {
  int batch, heads, kv_heads, dim, window, sinks, splits;
  float scale;
  const void* q;
  const void* k;
  const void* v;
  Cache kc, vc;
  const int32_t* positions;
  void* out;
  float* parts;  // [batch, heads, splits, dim]
  float* stats;  // [batch, heads, splits, 2]: maximum (in powers of two) and sum
};

// The byte of a block whose largest magnitude has the float32 bits `top`.
__device__ __forceinline__ uint32_t block_exponent(uint32_t top) {
  const uint32_t field = top >> 23;
  return field == 255 ? 255 : max(field, 2u) - 2;
}

__device__ __forceinline__ uint32_t encode(float x, uint32_t exponent) {
  const float y = ldexpf(fabsf(x), 127 - int(exponent));
  const uint32_t code = uint32_t(y > 0.25f) + uint32_t(y >= 0.75f) + uint32_t(y > 1.25f) +
                        uint32_t(y >= 1.75f) + uint32_t(y > 2.5f) + uint32_t(y >= 3.5f) +
                        uint32_t(y > 5.0f);
  return exponent == 255 ? 0 : code | (__float_as_uint(x) >> 31) << 3;
}

// A block's power of two; its smallest one, 2^-127, is not a normal number.
__device__ __forceinline__ float power_of(uint32_t exponent) {
  return __uint_as_float(exponent ? exponent << 23 : 1u << 22);
}

// The eight elements of a word of codes.
template <typename T>
__device__ __forceinline__ Frag<T> decode(uint32_t w, float power) {
  Frag<T> f;
  if constexpr (std::is_same_v<T, bf16>) {
    const Vec<T, 2> a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, 0);
    const Vec<T, 2> b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, 1);
    const Vec<T, 2> c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, 2);
    const Vec<T, 2> d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, 3);
    f = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  } else if constexpr (std::is_same_v<T, f16>) {
    const Vec<T, 2> a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, power, 0);
    const Vec<T, 2> b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, power, 1);
    const Vec<T, 2> c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, power, 2);
    const Vec<T, 2> d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, power, 3);
    f = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  } else {
    const Vec<T, 2> a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, power, 0);
    const Vec<T, 2> b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, power, 1);
    const Vec<T, 2> c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, power, 2);
    const Vec<T, 2> d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, power, 3);
    f = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
  return f;
}

template <typename T>
__device__ __forceinline__ void store_frag(T* p, const Frag<T>& f) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<Frag<T>*>(__builtin_assume_aligned(p, 16)) = f;
  } else {
    *reinterpret_cast<Vec<T, 4>*>(p) = __builtin_shufflevector(f, f, 0, 1, 2, 3);
    *reinterpret_cast<Vec<T, 4>*>(p + 4) = __builtin_shufflevector(f, f, 4, 5, 6, 7);
  }
}

using Word4 = Vec<uint32_t, 4>;

// Of a float32, those that a 16-bit type has (float16 from its smallest normal number on).
template <typename T>
constexpr uint32_t kTakenBits = std::is_same_v<T, bf16> ? 0xffff0000u : 0xffffe000u;

// acc_frag, cut off to these bits.
template <typename T>
__device__ __forceinline__ Frag<T> cut_frag(const Acc& c, int s) {
  if constexpr (sizeof(T) == 4) {
    return acc_frag<T>(c, s);
  } else {
    Word4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = c[8 * s + 2 * i], b = c[8 * s + 2 * i + 1];
      if constexpr (std::is_same_v<T, bf16>)
        w[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
      else
        w[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
    }
    return __builtin_bit_cast(Frag<T>, w);
  }
}

// Heads of a tile, the columns of its products.  With 16-bit types its upper 16 columns
// are the lower ones' heads once more, for the second part of their probabilities.
template <typename T>
constexpr int kHeads = sizeof(T) == 2 ? 16 : 32;

template <typename T, int kDim>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 3 : 1) void step_quant_kernel(StepArgs a) {
  constexpr int kPitchT = kPitch<T, kDim>;
  constexpr bool kBeside = sizeof(T) == 2;
  constexpr int kSteps = kDim / 16, kBlocks = kDim / 32;
  constexpr int kHalf = kDim / 64;                     // blocks of half a row
  constexpr int kCount = kKeys * kBlocks / kWave;      // blocks of values a lane converts
  static_assert(kCount * kWave == kKeys * kBlocks && kHalf * 64 == kDim, "whole blocks");
  union Shared {
    T tiles[kWaves][kKeys * kPitchT];
    float joined[32][kDim + 1];
  };
  __shared__ __align__(16) Shared shared;
  __shared__ __align__(16) uint32_t fresh_codes[2][kDim / 8];  // the new token's key and value
  __shared__ uint32_t fresh_exponents[2][kBlocks];
  __shared__ float tops[kWaves][32], sums[kWaves][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int group = a.heads / a.kv_heads, group_tiles = (group + kHeads<T> - 1) / kHeads<T>;
  const int kv = blockIdx.y / group_tiles, group_tile = blockIdx.y % group_tiles;
  const int b = blockIdx.z, split = blockIdx.x;
  const int member = group_tile * kHeads<T> + col % kHeads<T>;
  const bool live = member < group;
  const int pos = a.positions[b];
  const int capacity = a.sinks + a.window;
  const int filled = pos < 0 ? 0 : int(min(int64_t(pos) + 1, int64_t(capacity)));
  const int slot = pos < a.sinks ? pos : a.sinks + (pos - a.sinks) % a.window;
  const int share = ((filled + a.splits - 1) / a.splits + kKeys - 1) / kKeys * kKeys;
  const int lo = int(min(int64_t(split) * share, int64_t(filled))), hi = min(lo + share, filled);
  const int row_bytes = a.dim / 2, row_blocks = a.dim / kBlock;
  const int64_t row0 = (int64_t(b) * a.kv_heads + kv) * capacity;
  const bool mine = slot >= lo && slot < hi;
  if (mine) {
    // A group of 32 lanes a block: first the key's, then the value's.
    const int block = threadIdx.x / kBlock;
    const bool value = block >= kBlocks;
    const int at = block % kBlocks, d = at * kBlock + col;
    if (block < 2 * kBlocks && at < row_blocks) {
      const T* row = static_cast<const T*>(value ? a.v : a.k) + (int64_t(b) * a.kv_heads + kv) * a.dim;
      const float x = float(row[d]);
      uint32_t top = __float_as_uint(fabsf(x));
#pragma unroll
      for (int i = 1; i < kBlock; i <<= 1) top = max(top, uint32_t(__shfl_xor(int(top), i, 64)));
      const uint32_t exponent = block_exponent(top);
      uint32_t word = encode(x, exponent) << 4 * (col & 7);
#pragma unroll
      for (int i = 1; i < 8; i <<= 1) word |= uint32_t(__shfl_xor(int(word), i, 64));
      if ((col & 7) == 0) fresh_codes[value][d / 8] = word;
      if (col == 0) fresh_exponents[value][at] = exponent;
      if (group_tile == 0) {
        const Cache& c = value ? a.vc : a.kc;
        if ((col & 7) == 0)
          *reinterpret_cast<uint32_t*>(c.codes + (row0 + slot) * row_bytes + d / 2) = word;
        if (col == 0) c.exponents[(row0 + slot) * row_blocks + at] = uint8_t(exponent);
      }
    }
    __syncthreads();  // the slot is the workgroup's: all of its threads are here
  }
  Frag<T> q[kSteps];
  {
    const T* row = static_cast<const T*>(a.q) + (int64_t(b) * a.heads + kv * group + member) * a.dim;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = half * (kDim / 2) + 8 * s;
      q[s] = load_global<T>(row + d, live && d < a.dim);
    }
  }
  const float c = a.scale * kLog2e;
  // The bits of a probability that the lower columns take.
  const uint32_t upper = col < 16 ? 0u : kTakenBits<T>;
  float top = -INFINITY, sum = 0.0f;
  Acc o[kBlocks];
#pragma unroll
  for (int n = 0; n < kBlocks; ++n) o[n] = Acc(0.0f);
  Word4 kw[kHalf], vw[kCount];
  uint32_t ke[kHalf], ve[kCount];
  const uint8_t* k_codes = a.kc.codes + row0 * row_bytes;
  const uint8_t* v_codes = a.vc.codes + row0 * row_bytes;
  const uint8_t* k_exponents = a.kc.exponents + row0 * row_blocks;
  const uint8_t* v_exponents = a.vc.exponents + row0 * row_blocks;
  // Places beyond the share or the row are zeros.
  const auto fetch = [&](int j0) {
    const int j = j0 + col;
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
      const int block = half * kHalf + i;
      kw[i] = Word4(0);
      ke[i] = 0;
      if (j < hi && block < row_blocks) {
        kw[i] = *reinterpret_cast<const Word4*>(k_codes + int64_t(j) * row_bytes + block * 16);
        ke[i] = k_exponents[int64_t(j) * row_blocks + block];
      }
    }
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int chunk = i * kWave + lane;
      const int r = j0 + chunk / kBlocks, block = chunk % kBlocks;
      vw[i] = Word4(0);
      ve[i] = 0;
      if (r < hi && block < row_blocks) {
        vw[i] = *reinterpret_cast<const Word4*>(v_codes + int64_t(r) * row_bytes + block * 16);
        ve[i] = v_exponents[int64_t(r) * row_blocks + block];
      }
    }
    // The new token's row is being written: its codes are here already.
    if (mine && slot >= j0 && slot < j0 + kKeys) {
      if (j == slot) {
#pragma unroll
        for (int i = 0; i < kHalf; ++i) {
          const int block = half * kHalf + i;
          if (block < row_blocks) {
            kw[i] = *reinterpret_cast<const Word4*>(&fresh_codes[0][block * 4]);
            ke[i] = fresh_exponents[0][block];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kCount; ++i) {
        const int chunk = i * kWave + lane, block = chunk % kBlocks;
        if (j0 + chunk / kBlocks == slot && block < row_blocks) {
          vw[i] = *reinterpret_cast<const Word4*>(&fresh_codes[1][block * 4]);
          ve[i] = fresh_exponents[1][block];
        }
      }
    }
  };
  T* tile = shared.tiles[wave];
  int j0 = lo + wave * kKeys;
  if (j0 < hi) fetch(j0);
  for (; j0 < hi; j0 += kWaves * kKeys) {
    Acc s(0.0f);
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
      const float power = power_of(ke[i]);
      bad |= ke[i] == 255;
#pragma unroll
      for (int w = 0; w < 4; ++w) mma(decode<T>(kw[i][w], power), q[4 * i + w], s);
    }
    const uint64_t marked = __ballot(bad);
    if (__builtin_expect(marked != 0, 0)) {
      const uint32_t rows = uint32_t(marked) | uint32_t(marked >> 32);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (rows >> acc_row(r) & 1) s[r] = __builtin_nanf("");
    }
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int chunk = i * kWave + lane;
      const float power = power_of(ve[i]);
      T* at = tile + chunk / kBlocks * kPitchT + chunk % kBlocks * kBlock;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        Frag<T> f = decode<T>(vw[i][w], power);
        if (__builtin_expect(ve[i] == 255, 0)) f = Frag<T>(T(__builtin_nanf("")));
        store_frag(at + 8 * w, f);
      }
    }
    wave_sync();
    if (j0 + kWaves * kKeys < hi) fetch(j0 + kWaves * kKeys);
    if (j0 + kKeys > hi) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (j0 + acc_row(r) >= hi) s[r] = -INFINITY;
    }
    float m = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) m = fmaxf(m, s[r]);
    m = fmaxf(m, __shfl_xor(m, 32, 64)) * c;
    if (__any(m > top)) {
      const float up = fmaxf(top, m);
      const float shrink = up == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - up);
      sum *= shrink;
#pragma unroll
      for (int n = 0; n < kBlocks; ++n) o[n] *= shrink;
      top = up;
    }
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] * c - base);
    // Probabilities go into the second product, and so into the sum, as two numbers of a
    // 16-bit type that add up to them but for 2^-16: the values are exact in it, which
    // leaves the output its own rounding.  Beside each other the parts cost no product.
    if constexpr (kBeside) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] -= __uint_as_float(__float_as_uint(s[r]) & upper);
    }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const Frag<T> pf = cut_frag<T>(s, st);
      sum = add_all(pf, sum);
#pragma unroll
      for (int n = 0; n < kBlocks; ++n) mma(load_turned<T>(tile, kPitchT, 16 * st, 32 * n), pf, o[n]);
    }
    wave_sync();
  }
  // The waves join: the largest maximum, then the sums one wave after the other.
  sum += __shfl_xor(sum, 32, 64);
  if constexpr (kBeside) sum += __shfl_xor(sum, 16, 64);
  if (half == 0) {
    tops[wave][col] = top;
    sums[wave][col] = sum;
  }
  __syncthreads();
  float all = tops[0][col];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) all = fmaxf(all, tops[w][col]);
  const float base = all == -INFINITY ? 0.0f : all;
  float whole = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) whole += sums[w][col] * __builtin_amdgcn_exp2f(tops[w][col] - base);
  const float shrink = __builtin_amdgcn_exp2f(top - base);
  for (int w = 0; w < kWaves; ++w) {
    if (wave == w) {
#pragma unroll
      for (int n = 0; n < kBlocks; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float& at = shared.joined[col][32 * n + acc_row(r)];
          at = w ? at + o[n][r] * shrink : o[n][r] * shrink;
        }
    }
    __syncthreads();
  }
  if (wave == 0 && half == 0) {
    tops[0][col] = all;
    sums[0][col] = whole;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < kHeads<T> * kDim; e += kThreads) {
    const int m = e / kDim, d = e % kDim;
    if (group_tile * kHeads<T> + m >= group || d >= a.dim) continue;
    const int64_t row = int64_t(b) * a.heads + kv * group + group_tile * kHeads<T> + m;
    float value = shared.joined[m][d];
    if constexpr (kBeside) value += shared.joined[m + 16][d];
    if (a.splits == 1) {
      const float l = sums[0][m];
      const bool none = tops[0][m] == -INFINITY && l == 0.0f;
      static_cast<T*>(a.out)[row * a.dim + d] = T(none ? 0.0f : value / l);
    } else {
      a.parts[(row * a.splits + split) * a.dim + d] = value;
      if (d == 0) {
        a.stats[(row * a.splits + split) * 2] = tops[0][m];
        a.stats[(row * a.splits + split) * 2 + 1] = sums[0][m];
      }
    }
  }
}

// The shares of a row: their weights first, a thread each, then two halves of the
// shares side by side, eight loads in flight.
constexpr int kMostSplits = 256;

template <typename T>
__global__ __launch_bounds__(kThreads) void step_quant_join_kernel(StepArgs a) {
  __shared__ float weights[kMostSplits], reduced[kWaves], other[128];
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const bool live = t < a.splits;
  const float* stats = a.stats + row * a.splits * 2;
  const float top = live ? stats[2 * t] : -INFINITY, sum = live ? stats[2 * t + 1] : 0.0f;
  float m = top;
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) m = fmaxf(m, __shfl_xor(m, i, 64));
  if (lane == 0) reduced[wave] = m;
  __syncthreads();
  const float all = fmaxf(fmaxf(reduced[0], reduced[1]), fmaxf(reduced[2], reduced[3]));
  const float w = live ? __builtin_amdgcn_exp2f(top - (all == -INFINITY ? 0.0f : all)) : 0.0f;
  weights[t] = w;
  float whole = sum * w;
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) whole += __shfl_xor(whole, i, 64);
  __syncthreads();
  if (lane == 0) reduced[wave] = whole;
  __syncthreads();
  whole = (reduced[0] + reduced[1]) + (reduced[2] + reduced[3]);
  const int d = t & 127, part = t >> 7, count = (a.splits + 1) / 2;
  float o = 0.0f;
  if (d < a.dim) {
    const float* parts = a.parts + row * a.splits * a.dim + d;
    const int end = min(a.splits, (part + 1) * count);
#pragma unroll 8
    for (int s = part * count; s < end; ++s) o += parts[int64_t(s) * a.dim] * weights[s];
  }
  if (part) other[d] = o;
  __syncthreads();
  if (part || d >= a.dim) return;
  const bool none = all == -INFINITY && whole == 0.0f;
  static_cast<T*>(a.out)[row * a.dim + d] = T(none ? 0.0f : (o + other[d]) / whole);
}

// Tiles of heads of a stream.
int64_t key_tiles(const gs_attention& d) {
  const int heads = d.type == GS_F32 ? kHeads<float> : kHeads<f16>;
  return int64_t(d.kv_heads) * ((d.heads / d.kv_heads + heads - 1) / heads);
}

// Workgroups of one stream and key head: as many as the GPU holds at once (three a CU,
// in float32 one), with a tile for each of their waves.  More wait for a place and
// spend more on starts and ends (calls, 32 streams of 32 heads of 128 on 8 over 8176
// slots: bfloat16 74-76 us with 768, 81-83 with 2048; 6 streams: 22 and 34; float32 326 with
// 256, 368 with 2048; 6 streams: 79 and 127).
int plan_splits(const gs_attention& d) {
  const int64_t capacity = d.sinks + d.window;
  const int64_t rows = d.batch * key_tiles(d);
  const int64_t most = (capacity + kWaves * kKeys - 1) / (kWaves * kKeys);
  const int64_t held = d.type == GS_F32 ? 256 : 768;
  return int(std::max<int64_t>(1, std::min<int64_t>({most, held / std::max<int64_t>(rows, 1), kMostSplits})));
}

// Filling: a slot takes the last of its tokens.  Four lanes a block, eight elements
// each; keys and values in one launch.  Bound by the issue of instructions: 367 vector
// ones a wave (counted), 16 waves a SIMD for 2 x 8160 tokens of 4 heads of 128 into 4096
// slots, 10 of its 12 us; its 21 MB are 4 us.
struct FillArgs {
  int batch, kv_heads, dim, window, sinks, tokens;
  const void* from[2];
  Strides strides[2];
  const int32_t* lengths;
  Cache to[2];
};

template <typename T>
__global__ __launch_bounds__(kThreads) void fill_quant_kernel(FillArgs a) {
  const int capacity = a.sinks + a.window, lanes = a.dim / 8;
  const int64_t rows = int64_t(a.batch) * a.kv_heads * capacity;
  const int64_t id = seq::block_index() * kThreads + threadIdx.x;
  const int64_t both = id / lanes;
  const int at = int(id % lanes), value = both >= rows;
  const int64_t row = both - (value ? rows : 0);
  const int slot = int(row % capacity);
  const int64_t head = row / capacity;
  const int kv = int(head % a.kv_heads), b = int(head / a.kv_heads);
  bool live = both < 2 * rows;
  int token = slot;
  if (live) {
    const int length = a.lengths ? min(max(a.lengths[b], 0), a.tokens) : a.tokens;
    live = slot < length;
    if (slot >= a.sinks) token = slot + (length - 1 - slot) / a.window * a.window;
  }
  FloatVec<8> x(0.0f);
  if (live) {
    const Strides& s = a.strides[value];
    const T* from = static_cast<const T*>(a.from[value]) + b * s.batch + token * s.token + kv * s.head;
    x = to_float<T, 8>(load_global<T>(from + at * 8, true));
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(fabsf(x[i])));
  // The lanes of a block are neighbours in a wave: a row has a multiple of four.
  top = max(top, uint32_t(__shfl_xor(int(top), 1, 64)));
  top = max(top, uint32_t(__shfl_xor(int(top), 2, 64)));
  if (!live) return;
  const uint32_t exponent = block_exponent(top);
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) word |= encode(x[i], exponent) << 4 * i;
  *reinterpret_cast<uint32_t*>(a.to[value].codes + row * (a.dim / 2) + at * 4) = word;
  if ((at & 3) == 0) a.to[value].exponents[row * (a.dim / kBlock) + at / 4] = uint8_t(exponent);
}

int check_cache(const gs_attention& d, const void* k_codes, const void* k_exponents,
                const void* v_codes, const void* v_exponents) {
  GS_REQUIRE(d.head_dim % kBlock == 0, GS_ERR_UNSUPPORTED,
             "head_dim %d not supported in 4 bits (a multiple of %d up to 128)", d.head_dim, kBlock);
  GS_REQUIRE(d.window < (int64_t(1) << 30) && d.sinks < (int64_t(1) << 30) - d.window,
             GS_ERR_OVERFLOW, "cache too large: %lld first tokens and a window of %lld",
             (long long)d.sinks, (long long)d.window);
  if (d.batch == 0) return GS_OK;
  GS_REQUIRE(k_codes && k_exponents && v_codes && v_exponents, GS_ERR_INVALID_ARGUMENT,
             "null cache");
  GS_REQUIRE(aligned_to(k_codes, 16) && aligned_to(v_codes, 16), GS_ERR_INVALID_ARGUMENT,
             "codes must start on a 16-byte boundary");
  return GS_OK;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" GS_API size_t gs_window_attention_step_quant_workspace_bytes(const gs_attention* desc) {
  if (!desc || check_attention(*desc) != GS_OK) return 0;
  const int splits = plan_splits(*desc);
  if (splits == 1) return 0;
  return size_t(desc->batch) * size_t(desc->heads) * size_t(splits) *
         (size_t(desc->head_dim) + 2) * sizeof(float);
}

extern "C" GS_API int gs_window_attention_step_quant(
    const gs_attention* desc, const void* q, const void* k, const void* v, void* k_codes,
    void* k_exponents, void* v_codes, void* v_exponents, const int32_t* positions, void* out,
    void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  GS_REQUIRE(desc, GS_ERR_INVALID_ARGUMENT, "null description");
  GS_TRY(check_attention(*desc));
  GS_TRY(check_cache(*desc, k_codes, k_exponents, v_codes, v_exponents));
  if (desc->batch == 0) return GS_OK;
  const int64_t none[3] = {0, 0, 0};
  GS_REQUIRE(positions, GS_ERR_INVALID_ARGUMENT, "null pointer: positions");
  GS_TRY(check_rows(q, none, desc->type, "q"));
  GS_TRY(check_rows(k, none, desc->type, "k"));
  GS_TRY(check_rows(v, none, desc->type, "v"));
  GS_TRY(check_rows(out, none, desc->type, "out"));
  const size_t need = gs_window_attention_step_quant_workspace_bytes(desc);
  GS_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), GS_ERR_WORKSPACE,
             "workspace too small: %zu bytes, %zu needed", workspace_bytes, need);
  StepArgs a{};
  a.batch = int(desc->batch);
  a.heads = desc->heads;
  a.kv_heads = desc->kv_heads;
  a.dim = desc->head_dim;
  a.window = int(desc->window);
  a.sinks = int(desc->sinks);
  a.splits = plan_splits(*desc);
  a.scale = desc->scale;
  a.q = q;
  a.k = k;
  a.v = v;
  a.kc = {static_cast<uint8_t*>(k_codes), static_cast<uint8_t*>(k_exponents)};
  a.vc = {static_cast<uint8_t*>(v_codes), static_cast<uint8_t*>(v_exponents)};
  a.positions = positions;
  a.out = out;
  a.stats = static_cast<float*>(workspace);
  a.parts = a.stats + int64_t(a.batch) * a.heads * a.splits * 2;
  const dim3 grid(unsigned(a.splits), unsigned(key_tiles(*desc)), unsigned(a.batch));
  const hipStream_t s = as_stream(stream);
  return seq::with_type(desc->type, [&](auto t) {
    using T = decltype(t);
    if (a.dim <= 64)
      step_quant_kernel<T, 64><<<grid, kThreads, 0, s>>>(a);
    else
      step_quant_kernel<T, 128><<<grid, kThreads, 0, s>>>(a);
    GS_TRY(check_launch("window_attention_step_quant"));
    if (a.splits == 1) return int(GS_OK);
    step_quant_join_kernel<T><<<unsigned(a.batch * a.heads), kThreads, 0, s>>>(a);
    return check_launch("window_attention_step_quant join");
  });
}

extern "C" GS_API int gs_window_cache_fill_quant(const gs_attention* desc, const void* k,
                                                 const void* v, const int64_t* strides,
                                                 const int32_t* lengths, void* k_codes,
                                                 void* k_exponents, void* v_codes,
                                                 void* v_exponents, void* stream) {
  clear_error();
  GS_REQUIRE(desc, GS_ERR_INVALID_ARGUMENT, "null description");
  GS_TRY(check_attention(*desc));
  GS_TRY(check_cache(*desc, k_codes, k_exponents, v_codes, v_exponents));
  if (desc->batch == 0 || desc->keys == 0) return GS_OK;
  GS_REQUIRE(strides, GS_ERR_INVALID_ARGUMENT, "null pointer: strides");
  GS_TRY(check_rows(k, strides, desc->type, "k"));
  GS_TRY(check_rows(v, strides + 3, desc->type, "v"));
  FillArgs a{};
  a.batch = int(desc->batch);
  a.kv_heads = desc->kv_heads;
  a.dim = desc->head_dim;
  a.window = int(desc->window);
  a.sinks = int(desc->sinks);
  a.tokens = int(desc->keys);
  a.from[0] = k;
  a.from[1] = v;
  a.strides[0] = {strides[0], strides[1], strides[2]};
  a.strides[1] = {strides[3], strides[4], strides[5]};
  a.lengths = lengths;
  a.to[0] = {static_cast<uint8_t*>(k_codes), static_cast<uint8_t*>(k_exponents)};
  a.to[1] = {static_cast<uint8_t*>(v_codes), static_cast<uint8_t*>(v_exponents)};
  const int64_t lanes = 2 * desc->batch * a.kv_heads * (desc->sinks + desc->window) * (a.dim / 8);
  const int64_t blocks = (lanes + kThreads - 1) / kThreads;
  GS_REQUIRE(blocks < (int64_t(1) << 31), GS_ERR_OVERFLOW, "cache too large");
  return seq::with_type(desc->type, [&](auto t) {
    fill_quant_kernel<decltype(t)><<<seq::grid_of(blocks), kThreads, 0, as_stream(stream)>>>(a);
    return check_launch("window_cache_fill_quant");
  });
}
