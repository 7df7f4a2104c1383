// Attention with a sliding window and visible first tokens, forward.  Query i
// stands at position p = keys - queries + i and sees key j when
//   j <= p  and  (j > p - window or j < sinks)  and  j < length:
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j,  lse_i = log sum_j exp(scale q_i . k_j).
// A query that sees nothing gets zeros and lse = -inf.
//
// One pass over the keys that a workgroup's queries reach, in tiles of 64, with
// the running maximum and sum in float32.  A wave holds 32 queries.  Scores are
// computed transposed (keys in rows, queries in columns), so a lane holds 16 of
// 32 scores of one query: maximum, sum and rescaling are the lane's own up to
// one exchange with the other half, and the exponentials are the next product's
// operand in place.  Probabilities are rounded to the inputs' type for that
// product and for the sum alike, so that a row's weights add up to one.
//
// Measured, bfloat16, 40000 tokens, 12 heads of 64 on 4, window 5000: 0.76 ms, 760
// TFLOP/s, where a large square matrix product reaches 1126.  Matrix cores are
// busy 40 % of the time, a SIMD issues vector instructions (half of them the
// exponentials' path) for about 45 %, LDS serves for 40 %: what is left is the
// latency from one to the other, which four waves a SIMD hide in part.  64
// queries a wave would halve the LDS reads but leave two waves a SIMD: 0.90 ms.
// float16, 2 x 8160 tokens, 16 heads of 128: 0.33 ms, 700 TFLOP/s at two waves.
#include "attention_tile.h"

namespace gs {
namespace {

using namespace att;

struct ForwardArgs {
  Problem p;
  const void* q;
  const void* k;
  const void* v;
  Strides sq, sk, sv;
  void* out;   // [batch, queries, heads, dim]
  float* lse;  // [batch, heads, queries]
};

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;

// 32 queries of a wave, a query for each pair of lanes: what their walk over the
// keys carries.
template <typename T, int kDim>
struct Queries {
  static constexpr int kSteps = kDim / 16, kBlocks = kDim / 32;
  static constexpr int kPitchT = kPitch<T, kDim>;
  Frag<T> q[kSteps];
  float top = -INFINITY, sum = 0.0f;
  Acc o[kBlocks];
  Poison<T, kBlocks> poison;
  int first, pos, length;  // position of the wave's first query and of the lane's

  __device__ __forceinline__ Queries(const ForwardArgs& a, int b, int head, int query, int length_)
      : first(a.p.offset() + query), length(length_) {
    const int lane = threadIdx.x & 63, i = query + (lane & 31);
    pos = a.p.offset() + i;
    const T* row = static_cast<const T*>(a.q) + b * a.sq.batch + i * a.sq.token + head * a.sq.head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = 16 * s + 8 * (lane >> 5);
      q[s] = load_global<T>(row + d, i < a.p.queries && d < a.p.dim);
    }
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) o[n] = Acc(0.0f);
  }

  // Whether every query sees each of `keys` keys from j0 on.
  __device__ __forceinline__ bool sees_all(const Problem& p, int j0, int keys) const {
    const int last = first + 31, j1 = j0 + keys - 1;
    return j1 <= first && j1 < length && (j0 > last - p.window || j1 < p.sinks);
  }

  // 32 kHalves keys from j0 on, rows row0 .. of the LDS tiles kt and vt; c: the
  // scale in powers of two.  kFull: every query sees all of them.
  template <bool kFull, int kHalves>
  __device__ __forceinline__ void take(const Problem& p, const T* kt, const T* vt, int row0, int j0,
                                       float c) {
    const int lane = threadIdx.x & 63;
    const bool all = kFull || sees_all(p, j0, 32 * kHalves);
    if constexpr (!kFull) {
      if (j0 > first + 31 || j0 >= length ||
          (j0 + 32 * kHalves - 1 <= first - p.window && j0 >= p.sinks))
        return;
    }
    Acc s[kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      s[h] = Acc(0.0f);
#pragma unroll
      for (int st = 0; st < kSteps; ++st)
        mma(load_rows<T>(kt, kPitchT, row0 + 32 * h, 16 * st), q[st], s[h]);
    }
    if (!all) {
      const KeySight sight(p, pos, j0 + 4 * (lane >> 5), length);
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!sight.sees(32 * h + acc_row_of_half(r))) s[h][r] = -INFINITY;
    }
    float m = s[0][0];
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
      for (int r = 0; r < 16; ++r) m = fmaxf(m, s[h][r]);
    m *= c;
    // The maximum that exponents are taken against follows the true one at a
    // distance of up to 2^8, so that most tiles rescale nothing, and need nothing
    // of the scores that the lane's other half holds.
    if (__builtin_expect(__any(m > top + 8.0f), 0)) {
      const float whole = fmaxf(m, __shfl_xor(m, 32, 64));
      const float up = whole > top + 8.0f ? whole : top;
      float shrink = up == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - up);
      asm volatile("" : "+v"(shrink));  // or the compiler rescales without the branch
      sum *= shrink;
#pragma unroll
      for (int n = 0; n < kBlocks; ++n) o[n] *= shrink;
      top = up;
    }
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        Frag<T> vf[kBlocks];
#pragma unroll
        for (int n = 0; n < kBlocks; ++n)
          vf[n] = load_turned<T>(vt, kPitchT, row0 + 32 * h + 16 * st, 32 * n);
#pragma unroll
        for (int r = 8 * st; r < 8 * st + 8; ++r) s[h][r] = power<T>(s[h][r] * c - base);
        const Frag<T> pf = acc_frag<T>(s[h], st);
        sum = add_all(pf, sum);
        if (!all) {
          const KeySight sight(p, pos, j0 + 32 * h + 16 * st, length);
          poison.guard(vt, kPitchT, row0 + 32 * h + 16 * st, vf, pf,
                       [&](int e) { return sight.sees(e); });
        }
#pragma unroll
        for (int n = 0; n < kBlocks; ++n) mma(vf[n], pf, o[n]);
      }
  }
};

// Which heads and queries a workgroup has: the heads that share keys side by side.
struct Place {
  int b, kv, head, block;
  __device__ __forceinline__ Place(const Problem& p, int64_t id, int blocks) {
    const int group = p.heads / p.kv_heads;
    block = int(id / group % blocks);
    kv = int(id / group / blocks % p.kv_heads);
    b = int(id / group / blocks / p.kv_heads);
    head = kv * group + int(id % group);
  }
};

// 128 queries a workgroup, whose waves share tiles of 64 keys in LDS.
template <typename T, int kDim>
__global__ __launch_bounds__(kThreads, sizeof(T) == 4 ? 1 : kDim <= 64 ? 4 : 2) void attention_fwd_kernel(
    ForwardArgs a) {
  constexpr int kKeys = 64, kQueries = 32 * kWaves;
  constexpr int kBlocks = kDim / 32;
  __shared__ __align__(16) T tiles[2][2][kKeys * kPitch<T, kDim>];
  const Problem& p = a.p;
  const int blocks = (p.queries + kQueries - 1) / kQueries;
  const int64_t id = xcd_order(blockIdx.x, int64_t(blocks) * p.heads * p.batch);
  if (id >= int64_t(blocks) * p.heads * p.batch) return;
  const Place at(p, id, blocks);
  const int length = p.length(at.b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T* kbase = static_cast<const T*>(a.k) + at.b * a.sk.batch + at.kv * a.sk.head;
  const T* vbase = static_cast<const T*>(a.v) + at.b * a.sv.batch + at.kv * a.sv.head;
  Queries<T, kDim> w(a, at.b, at.head, at.block * kQueries + wave * 32, length);
  const KeyTiles<kKeys> walk(p, at.block * kQueries, kQueries, length);
  const float c = p.scale * kLog2e;

  Stage<T, kKeys, kDim, kThreads> sk(a.sk.token, p.dim, threadIdx.x), sv(a.sv.token, p.dim, threadIdx.x);
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
      w.template take<true, kKeys / 32>(p, kt, vt, 0, walk.first_key(it), c);
    } else {
#pragma unroll 1
      for (int h = 0; h < kKeys / 32; ++h)
        w.template take<false, 1>(p, kt, vt, 32 * h, walk.first_key(it) + 32 * h, c);
    }
    if (it + 1 < walk.count) {
      sk.store(tiles[(it + 1) & 1][0]);
      sv.store(tiles[(it + 1) & 1][1]);
    }
    __syncthreads();
  };
  // Runs of tiles that the wave's queries see whole in a loop of their own:
  // without branches the compiler lays products over exponentials.
  for (int it = 0; it < walk.count;) {
    while (it < walk.count && !w.sees_all(p, walk.first_key(it), kKeys)) turn(it++, std::false_type{});
    while (it < walk.count && w.sees_all(p, walk.first_key(it), kKeys)) turn(it++, std::true_type{});
  }
  w.poison.apply(w.o);
  const int i = at.block * kQueries + wave * 32 + (lane & 31);
  const float l = w.sum + __shfl_xor(w.sum, 32, 64);
  if (i >= p.queries) return;
  const float inverse = w.top == -INFINITY && l == 0.0f ? 0.0f : 1.0f / l;
  T* out = static_cast<T*>(a.out) + ((int64_t(at.b) * p.queries + i) * p.heads + at.head) * p.dim;
#pragma unroll
  for (int n = 0; n < kBlocks; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * n + 8 * g + 4 * (lane >> 5);
      FloatVec<4> f;
#pragma unroll
      for (int r = 0; r < 4; ++r) f[r] = w.o[n][4 * g + r] * inverse;
      if (d < p.dim) *reinterpret_cast<Vec<T, 4>*>(out + d) = from_float<T, 4>(f);
    }
  if (lane < 32)
    a.lse[(int64_t(at.b) * p.heads + at.head) * p.queries + i] =
        w.top == -INFINITY && l == 0.0f ? -INFINITY : (w.top + __builtin_amdgcn_logf(l)) / kLog2e;
}

// 32 queries a workgroup: every wave has all of them and every fourth tile of 32
// keys, which it loads by itself, and the waves join at the end.  For calls that
// would leave most of the GPU idle with 128 queries a workgroup.
template <typename T, int kDim>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) void attention_fwd_split_kernel(
    ForwardArgs a) {
  constexpr int kKeys = 32, kQueries = 32;
  constexpr int kBlocks = kDim / 32;
  __shared__ __align__(16) T tiles[kWaves][2][kKeys * kPitch<T, kDim>];
  __shared__ float joined[32][kDim + 1];
  __shared__ float tops[kWaves][32], sums[kWaves][32];
  const Problem& p = a.p;
  const int blocks = (p.queries + kQueries - 1) / kQueries;
  const int64_t id = xcd_order(blockIdx.x, int64_t(blocks) * p.heads * p.batch);
  if (id >= int64_t(blocks) * p.heads * p.batch) return;
  const Place at(p, id, blocks);
  const int length = p.length(at.b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T* kbase = static_cast<const T*>(a.k) + at.b * a.sk.batch + at.kv * a.sk.head;
  const T* vbase = static_cast<const T*>(a.v) + at.b * a.sv.batch + at.kv * a.sv.head;
  Queries<T, kDim> w(a, at.b, at.head, at.block * kQueries, length);
  const KeyTiles<kKeys> walk(p, at.block * kQueries, kQueries, length);
  const float c = p.scale * kLog2e;
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
    w.template take<false, 1>(p, tiles[wave][0], tiles[wave][1], 0, walk.first_key(it), c);
    wave_sync();
  }
  w.poison.apply(w.o);
  // The waves join: the largest maximum, then the sums one wave after the other.
  // No maximum and no sum: the query sees nothing.  NaN scores leave no maximum
  // either, but a sum of NaN, which reaches the result.
  const float l = w.sum + __shfl_xor(w.sum, 32, 64);
  if (lane < 32) {
    tops[wave][lane] = w.top;
    sums[wave][lane] = l;
  }
  __syncthreads();
  const int col = lane & 31;
  float top = tops[0][col], whole = 0.0f;
#pragma unroll
  for (int k = 1; k < kWaves; ++k) top = fmaxf(top, tops[k][col]);
  const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
  for (int k = 0; k < kWaves; ++k)
    whole += sums[k][col] * __builtin_amdgcn_exp2f(tops[k][col] - base);
  const float inverse = top == -INFINITY && whole == 0.0f ? 0.0f : 1.0f / whole;
  const float shrink = __builtin_amdgcn_exp2f(w.top - base) * inverse;
  for (int k = 0; k < kWaves; ++k) {
    if (wave == k) {
#pragma unroll
      for (int n = 0; n < kBlocks; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float& sum = joined[col][32 * n + acc_row(r)];
          const float v = w.o[n][r] * shrink;  // zero of a wave that saw nothing
          sum = k ? sum + v : v;
        }
    }
    __syncthreads();
  }
  const int i0 = at.block * kQueries;
  T* out = static_cast<T*>(a.out) + ((int64_t(at.b) * p.queries + i0) * p.heads + at.head) * p.dim;
  for (int e = threadIdx.x; e < 32 * kDim; e += kThreads) {
    const int row = e / kDim, d = e % kDim;
    if (i0 + row < p.queries && d < p.dim)
      out[int64_t(row) * p.heads * p.dim + d] = T(joined[row][d]);
  }
  if (threadIdx.x < 32 && i0 + col < p.queries)
    a.lse[(int64_t(at.b) * p.heads + at.head) * p.queries + i0 + col] =
        top == -INFINITY && whole == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(whole)) / kLog2e;
}

template <typename T, int kDim>
int launch_forward(const ForwardArgs& a, hipStream_t s) {
  const auto items = [&](int queries) {
    return (int64_t(a.p.queries) + queries - 1) / queries * a.p.heads * a.p.batch;
  };
  if (items(32 * kWaves) < split_below(a.p.dim))
    attention_fwd_split_kernel<T, kDim><<<unsigned(xcd_grid(items(32))), kThreads, 0, s>>>(a);
  else
    attention_fwd_kernel<T, kDim><<<unsigned(xcd_grid(items(32 * kWaves))), kThreads, 0, s>>>(a);
  return check_launch("window_attention");
}

}  // namespace

int check_attention(const gs_attention& d) {
  GS_REQUIRE(d.batch >= 0 && d.queries >= 0 && d.keys >= 0 && d.heads > 0 && d.kv_heads > 0,
             GS_ERR_INVALID_ARGUMENT, "attention sizes must be positive");
  GS_REQUIRE(d.heads % d.kv_heads == 0, GS_ERR_INVALID_ARGUMENT,
             "%d heads cannot share %d key heads", d.heads, d.kv_heads);
  GS_REQUIRE(d.head_dim > 0, GS_ERR_INVALID_ARGUMENT, "head_dim must be positive");
  GS_REQUIRE(d.head_dim % 8 == 0 && d.head_dim <= 128, GS_ERR_UNSUPPORTED,
             "head_dim %d not supported (a multiple of 8 up to 128)", d.head_dim);
  GS_REQUIRE(d.window > 0 && d.sinks >= 0, GS_ERR_INVALID_ARGUMENT,
             "window must be positive and sinks non-negative, got %lld and %lld",
             (long long)d.window, (long long)d.sinks);
  GS_REQUIRE(d.scale > 0.0f && d.scale <= 3.4e38f, GS_ERR_INVALID_ARGUMENT,
             "scale must be positive, got %g", double(d.scale));
  GS_REQUIRE(seq::float_type(d.type), GS_ERR_INVALID_ARGUMENT,
             "type must be GS_F32, GS_F16 or GS_BF16");
  GS_REQUIRE(d.keys < (int64_t(1) << 30) && d.queries < (int64_t(1) << 30) && d.batch < 65536 &&
                 d.heads < 65536,
             GS_ERR_OVERFLOW, "attention problem too large");
  // Workgroups of 256 threads: a launch holds less than 2^32.
  const int64_t most = (int64_t(1) << 24) - 8;
  GS_REQUIRE((d.queries + 127) / 128 * d.heads * d.batch < most &&
                 (d.keys + 127) / 128 * d.kv_heads * d.batch < most,
             GS_ERR_OVERFLOW, "attention problem too large");
  return GS_OK;
}

att::Problem make_problem(const gs_attention& d, const int32_t* lengths) {
  att::Problem p{};
  p.batch = int(d.batch);
  p.heads = d.heads;
  p.kv_heads = d.kv_heads;
  p.dim = d.head_dim;
  p.queries = int(d.queries);
  p.keys = int(d.keys);
  p.window = int(std::min(d.window, std::max<int64_t>(d.keys, 1)));
  p.sinks = int(std::min(d.sinks, d.keys));
  p.scale = d.scale;
  p.lengths = lengths;
  return p;
}

// Rows of 16-byte pieces: pointer and strides.
int check_rows(const void* p, const int64_t* strides, int32_t type, const char* name) {
  GS_REQUIRE(p, GS_ERR_INVALID_ARGUMENT, "null %s", name);
  const int64_t unit = 16 / seq::type_bytes(type);
  GS_REQUIRE(seq::aligned_to(p, 16) && strides[0] % unit == 0 && strides[1] % unit == 0 &&
                 strides[2] % unit == 0,
             GS_ERR_INVALID_ARGUMENT, "%s must have rows on 16-byte boundaries", name);
  // A tile's rows lie within 32 bits of its first one.
  GS_REQUIRE(strides[1] >= 0 && strides[1] < (int64_t(1) << 24), GS_ERR_OVERFLOW,
             "the tokens of %s lie too far apart (%lld elements)", name, (long long)strides[1]);
  return GS_OK;
}

}  // namespace gs

using namespace gs;

extern "C" GS_API int gs_window_attention_fwd(const gs_attention* desc, const void* q,
                                              const void* k, const void* v, const int64_t* strides,
                                              const int32_t* lengths, void* out, float* lse,
                                              void* stream) {
  clear_error();
  GS_REQUIRE(desc, GS_ERR_INVALID_ARGUMENT, "null description");
  GS_TRY(check_attention(*desc));
  if (desc->batch == 0 || desc->queries == 0) return GS_OK;
  GS_REQUIRE(strides && out && lse, GS_ERR_INVALID_ARGUMENT, "null pointer");
  GS_TRY(check_rows(q, strides, desc->type, "q"));
  if (desc->keys > 0) {
    GS_TRY(check_rows(k, strides + 3, desc->type, "k"));
    GS_TRY(check_rows(v, strides + 6, desc->type, "v"));
  }
  ForwardArgs a{make_problem(*desc, lengths), q, k, v,
                {strides[0], strides[1], strides[2]},
                {strides[3], strides[4], strides[5]},
                {strides[6], strides[7], strides[8]},
                out, lse};
  // Heads of up to 64 have tiles of their own, here, in the backward and in the
  // step.  In tiles of 64 and of 128, us forward and backward: 40000 tokens, 12 heads
  // of 64 on 4, window 5000, bfloat16 763 and 2435, 1281 and 6479; 1200, 8 heads of 64
  // 10 and 42, 23 and 61; 2 x 8160, 16 heads of 40 on 4, float16 174 and 656, 306 and
  // 1579; a step of 8 heads of 64 14, 16.
  return seq::with_type(desc->type, [&](auto t) {
    using T = decltype(t);
    if (desc->head_dim <= 64) return launch_forward<T, 64>(a, as_stream(stream));
    return launch_forward<T, 128>(a, as_stream(stream));
  });
}
