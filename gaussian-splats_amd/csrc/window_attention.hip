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
constexpr int kKeys = 64;  // of a tile

// kTiles: tiles of 32 queries that a wave holds.
template <typename T, int kDim, int kTiles>
constexpr int kWavesPerSimd = sizeof(T) == 2 && sizeof(T) == 2 && kDim * kTiles <= 64 ? 4 : sizeof(T) == 2 && kDim * kTiles <= 128 ? 2 : 1;

template <typename T, int kDim, int kTiles>
__global__ __launch_bounds__(kThreads, (kWavesPerSimd<T, kDim, kTiles>)) void attention_fwd_kernel(
    ForwardArgs a) {
  constexpr int kPitchT = kPitch<T, kDim>;
  constexpr int kSteps = kDim / 16, kBlocks = kDim / 32;
  constexpr int kQueries = 32 * kTiles * kWaves;  // of a workgroup
  __shared__ __align__(16) T tiles[2][2][kKeys * kPitchT];
  const Problem& p = a.p;
  const int blocks = (p.queries + kQueries - 1) / kQueries;
  const int64_t id = xcd_order(blockIdx.x, int64_t(blocks) * p.heads * p.batch);
  if (id >= int64_t(blocks) * p.heads * p.batch) return;
  // The heads that share keys side by side.
  const int group = p.heads / p.kv_heads;
  const int of = int(id % group);
  const int block = int(id / group % blocks);
  const int kv = int(id / group / blocks % p.kv_heads);
  const int b = int(id / group / blocks / p.kv_heads);
  const int head = kv * group + of;
  const int length = p.length(b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  const int i0 = block * kQueries + wave * 32 * kTiles + (lane & 31);  // the lane's first query
  const int pos = p.offset() + i0;
  Frag<T> q[kTiles][kSteps];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    const int i = i0 + 32 * t;
    const T* row = static_cast<const T*>(a.q) + b * a.sq.batch + i * a.sq.token + head * a.sq.head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = 16 * s + 8 * (lane >> 5);
      q[t][s] = load_global<T>(row + d, i < p.queries && d < p.dim);
    }
  }
  const T* kbase = static_cast<const T*>(a.k) + b * a.sk.batch + kv * a.sk.head;
  const T* vbase = static_cast<const T*>(a.v) + b * a.sv.batch + kv * a.sv.head;

  // Tiles of the first tokens, then those of the window.
  const int first = p.offset() + block * kQueries;
  const int last = min(p.offset() + min((block + 1) * kQueries, p.queries), length) - 1;
  int tail = max(0, first - p.window + 1) / kKeys;
  const int head_tiles = min((min(p.sinks, last + 1) + kKeys - 1) / kKeys, tail);
  const int count = last < 0 ? 0 : head_tiles + max(0, last / kKeys - tail + 1);
  tail -= head_tiles;

  const float c = p.scale * kLog2e;
  const int wave_first = first + wave * 32 * kTiles, wave_last = wave_first + 32 * kTiles - 1;
  float top[kTiles], sum[kTiles];
  Acc o[kTiles][kBlocks];
  Poison<T, kBlocks> poison[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    top[t] = -INFINITY;
    sum[t] = 0.0f;
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) o[t][n] = Acc(0.0f);
  }

  Stage<T, kKeys, kDim, kThreads> sk(a.sk.token, p.dim), sv(a.sv.token, p.dim);
  const auto fetch = [&](int it) {
    const int j0 = (it < head_tiles ? it : tail + it) * kKeys;
    sk.load(kbase, j0, length);
    sv.load(vbase, j0, length);
  };
  if (count > 0) {
    fetch(0);
    sk.store(tiles[0][0]);
    sv.store(tiles[0][1]);
  }
  __syncthreads();
  for (int it = 0; it < count; ++it) {
    if (it + 1 < count) fetch(it + 1);
    const T* kt = tiles[it & 1][0];
    const T* vt = tiles[it & 1][1];
#pragma unroll
    for (int h = 0; h < kKeys / 32; ++h) {
      const int j0 = (it < head_tiles ? it : tail + it) * kKeys + 32 * h, j1 = j0 + 31;
      const bool any = j0 <= wave_last && j0 < length && (j1 > wave_first - p.window || j0 < p.sinks);
      const bool all = j1 <= wave_first && j1 < length && (j0 > wave_last - p.window || j1 < p.sinks);
      if (__builtin_expect(any, 1)) {
        Acc s[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) s[t] = Acc(0.0f);
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          const Frag<T> kf = load_rows<T>(kt, kPitchT, 32 * h, 16 * st);
#pragma unroll
          for (int t = 0; t < kTiles; ++t) mma(kf, q[t][st], s[t]);
        }
        if (__builtin_expect(!all, 0)) {
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            const KeySight sight(p, pos + 32 * t, j0 + 4 * (lane >> 5), length);
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (!sight.sees(acc_row_of_half(r))) s[t][r] = -INFINITY;
          }
        }
        float m[kTiles];
        bool grows = false;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          m[t] = s[t][0];
#pragma unroll
          for (int r = 1; r < 16; ++r) m[t] = fmaxf(m[t], s[t][r]);
          m[t] *= c;
          grows |= m[t] > top[t] + 8.0f;
        }
        // The maximum that exponents are taken against follows the true one at a
        // distance of up to 2^8, so that most tiles rescale nothing, and need
        // nothing of the half of the scores that the lane's other half holds.
        if (__builtin_expect(__any(grows), 0)) {
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            const float whole = fmaxf(m[t], __shfl_xor(m[t], 32, 64));
            const float up = whole > top[t] + 8.0f ? whole : top[t];
            float shrink = up == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top[t] - up);
            asm volatile("" : "+v"(shrink));  // or the compiler rescales without the branch
            sum[t] *= shrink;
#pragma unroll
            for (int n = 0; n < kBlocks; ++n) o[t][n] *= shrink;
            top[t] = up;
          }
        }
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          Frag<T> pf[kTiles], vf[kBlocks];
#pragma unroll
          for (int n = 0; n < kBlocks; ++n)
            vf[n] = load_turned<T>(vt, kPitchT, 32 * h + 16 * st, 32 * n);
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            const float base = top[t] == -INFINITY ? 0.0f : top[t];
#pragma unroll
            for (int r = 8 * st; r < 8 * st + 8; ++r) s[t][r] = power<T>(s[t][r] * c - base);
            pf[t] = acc_frag<T>(s[t], st);
            sum[t] = add_all(pf[t], sum[t]);
          }
          if (__builtin_expect(!all, 0)) {
            if (__builtin_expect(any_not_finite<T>(vf), 0)) {
#pragma unroll
              for (int t = 0; t < kTiles; ++t) {
                const KeySight sight(p, pos + 32 * t, j0 + 16 * st, length);
                poison[t].mark(vt, kPitchT, 32 * h + 16 * st, pf[t],
                               [&](int e) { return sight.sees(e); });
              }
              drop_not_finite<T>(vf);
            }
          }
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int n = 0; n < kBlocks; ++n) mma(vf[n], pf[t], o[t][n]);
        }
      }
    }
    if (it + 1 < count) {
      sk.store(tiles[(it + 1) & 1][0]);
      sv.store(tiles[(it + 1) & 1][1]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    const int i = i0 + 32 * t;
    poison[t].apply(o[t]);
    const float l = sum[t] + __shfl_xor(sum[t], 32, 64);
    if (i >= p.queries) continue;
    const float inverse = top[t] == -INFINITY && l == 0.0f ? 0.0f : 1.0f / l;
    T* out = static_cast<T*>(a.out) + ((int64_t(b) * p.queries + i) * p.heads + head) * p.dim;
#pragma unroll
    for (int n = 0; n < kBlocks; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * n + 8 * g + 4 * (lane >> 5);
        FloatVec<4> f;
#pragma unroll
        for (int r = 0; r < 4; ++r) f[r] = o[t][n][4 * g + r] * inverse;
        if (d < p.dim) *reinterpret_cast<Vec<T, 4>*>(out + d) = from_float<T, 4>(f);
      }
    if (lane < 32)
      a.lse[(int64_t(b) * p.heads + head) * p.queries + i] =
          top[t] == -INFINITY ? -INFINITY : (top[t] + __builtin_amdgcn_logf(l)) / kLog2e;
  }
}

template <typename T, int kDim, int kTiles>
int launch_forward(const ForwardArgs& a, hipStream_t s) {
  constexpr int kQueries = 32 * kTiles * kWaves;
  const int64_t items =
      (int64_t(a.p.queries) + kQueries - 1) / kQueries * a.p.heads * a.p.batch;
  GS_REQUIRE(items < (int64_t(1) << 30), GS_ERR_OVERFLOW, "attention problem too large");
  attention_fwd_kernel<T, kDim, kTiles><<<unsigned(xcd_grid(items)), kThreads, 0, s>>>(a);
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
  return seq::with_type(desc->type, [&](auto t) {
    using T = decltype(t);
    if (desc->head_dim <= 64) return launch_forward<T, 64, 1>(a, as_stream(stream));
    return launch_forward<T, 128, 1>(a, as_stream(stream));
  });
}
