// Rotary positions: pairs of a head's elements turned by an angle that grows
// with the token's position, alone or on the way into a 4-bit cache.
//
//   x' = f (x cos a - y sin a),  y' = f (x sin a + y cos a),  a = position * freq
//
// Angles, their sines and the turn itself are in 64 bits and the result is
// rounded once (to fp32 and on to the type, as a double is converted).  In 32
// bits a position of 131072 has its angle off by 2^-8 already, and a key that
// falls to the other side of a border of its type can fall to the other side
// of one of the cache's 4-bit levels, so that the cache would depend on which
// of two roundings made it.  fp64 runs at fp32's rate here, and the bytes are
// the bound all the same.
#include <type_traits>

#include "vqx_kv4_values.h"
#include "vqx_rotary.h"

namespace vqx {
namespace {

struct Angle {
  double cos, sin;
};

// cos and sin of a, to a few 2^-53: a less the nearest multiple of pi / 2 (in
// two terms; the first difference is exact but for one rounding while the
// multiple is below 2^53), and Taylor's series, whose first term left out is
// below 2^-53 of the result up to pi / 4.
__device__ __forceinline__ Angle angle_of(double a) {
  const double k = __builtin_rint(a * 0.63661977236758134308);  // 2 / pi
  double r = __builtin_fma(-k, 1.57079632679489655800, a);
  r = __builtin_fma(-k, 6.12323399573676603587e-17, r);
  const double z = r * r;
  double s = -1.0 / 1307674368000.0;
  s = __builtin_fma(s, z, 1.0 / 6227020800.0);
  s = __builtin_fma(s, z, -1.0 / 39916800.0);
  s = __builtin_fma(s, z, 1.0 / 362880.0);
  s = __builtin_fma(s, z, -1.0 / 5040.0);
  s = __builtin_fma(s, z, 1.0 / 120.0);
  s = __builtin_fma(s, z, -1.0 / 6.0);
  s = __builtin_fma(r * z, s, r);
  double c = 1.0 / 20922789888000.0;
  c = __builtin_fma(c, z, -1.0 / 87178291200.0);
  c = __builtin_fma(c, z, 1.0 / 479001600.0);
  c = __builtin_fma(c, z, -1.0 / 3628800.0);
  c = __builtin_fma(c, z, 1.0 / 40320.0);
  c = __builtin_fma(c, z, -1.0 / 720.0);
  c = __builtin_fma(c, z, 1.0 / 24.0);
  c = __builtin_fma(c, z, -0.5);
  c = __builtin_fma(c, z, 1.0);
  const int quarter = (int)(k - 4.0 * __builtin_floor(0.25 * k));
  const double u = quarter & 1 ? s : c, v = quarter & 1 ? c : s;
  return Angle{(quarter + 1) & 2 ? -u : u, quarter & 2 ? -v : v};
}

// A pair's turn at a position, the factor and the direction in it.
__device__ __forceinline__ Angle turn_of(const Turn& t, int position, int pair) {
  Angle a = angle_of((double)position * (double)t.freqs[pair]);
  a.cos *= (double)t.factor;
  a.sin *= t.back ? -(double)t.factor : (double)t.factor;
  return a;
}

// fp16 by the conversion instructions (subnormals included, which is these
// kernels' mode): the integer ones of values8 and store8 are 8 and 12
// instructions an element (10377 tokens of 48 heads, half of each turned: 106 and
// 65 us).
template <typename T>
__device__ __forceinline__ void values_of(const Raw8F& r, T, float (&x)[8]) {
  values8(r, T(), x);
}
__device__ __forceinline__ void values_of(const Raw8F& r, F16, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    x[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? r[0][i / 2] >> 16 : r[0][i / 2] & 0xFFFFu));
}
template <typename T>
__device__ __forceinline__ void store_of(void* p, int64_t at, T, const float (&x)[8]) {
  store8(p, at, T(), x);
}
__device__ __forceinline__ uint32_t half_of(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
__device__ __forceinline__ void store_of(void* p, int64_t at, F16, const float (&x)[8]) {
  u32x4 a;
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = half_of(x[2 * i]) | half_of(x[2 * i + 1]) << 16;
  st_nt(reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + at), a);
}
// 8 elements as they are
template <typename T>
__device__ __forceinline__ void copy_of(void* p, int64_t at, T, const Raw8F& r) {
  constexpr int kSize = std::is_same<T, float>::value ? 4 : 2;
  u32x4* to = reinterpret_cast<u32x4*>(static_cast<uint8_t*>(p) + at * kSize);
  st_nt(to, r[0]);
  if constexpr (kSize == 4) st_nt(to + 1, r[1]);
}

// Which elements are pairs: neighbours; those half a turn's elements apart, 8 by
// 8; or those one by one, where that is no multiple of 8.
enum Layout { kNeighbours, kHalves, kSingles };

// What a thread has of a row: its own 8 values from element 8 part on and, for
// kHalves, the 8 that they are paired with.
template <typename T, Layout kLayout>
struct Pairs {
  Raw8F own;
};
template <typename T>
struct Pairs<T, kHalves> {
  Raw8F own, other;
};

__device__ __forceinline__ float load1(const void* p, int64_t at, float) { return static_cast<const float*>(p)[at]; }
__device__ __forceinline__ float load1(const void* p, int64_t at, Bf16) {
  return u2f((uint32_t)static_cast<const uint16_t*>(p)[at] << 16);
}
__device__ __forceinline__ float load1(const void* p, int64_t at, F16) {
  return h2f_exact(static_cast<const uint16_t*>(p)[at]);
}

template <typename T, Layout kLayout>
__device__ __forceinline__ void load_pairs(const Turn& t, const void* x, int64_t row, int part, Pairs<T, kLayout>& p) {
  const int e = 8 * part;
  load8(x, row + e, T(), p.own);
  if constexpr (kLayout == kHalves)
    if (e < 2 * t.half) load8(x, row + (e < t.half ? e + t.half : e - t.half), T(), p.other);
}

// The thread's 8 values turned; angles: those of the row's token, a pair each.
template <typename T, Layout kLayout>
__device__ __forceinline__ void turn_pairs(const Turn& t, const Angle* angles, const void* x, int64_t row, int part,
                                           const Pairs<T, kLayout>& p, float (&y)[8]) {
  const int e = 8 * part;
  values_of(p.own, T(), y);
  if (e >= 2 * t.half) return;
  if constexpr (kLayout == kNeighbours) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      if (e + j >= 2 * t.half) break;
      const Angle a = angles[(e + j) / 2];
      const double u = (double)y[j], v = (double)y[j + 1];
      y[j] = (float)__builtin_fma(u, a.cos, -(v * a.sin));
      y[j + 1] = (float)__builtin_fma(u, a.sin, v * a.cos);
    }
  } else if constexpr (kLayout == kHalves) {
    float z[8];
    values_of(p.other, T(), z);
    const bool first = e < t.half;
    const Angle* at = angles + (first ? e : e - t.half);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const Angle a = at[j];
      const double w = (double)z[j] * (first ? -a.sin : a.sin);
      y[j] = (float)__builtin_fma((double)y[j], a.cos, w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (e + j >= 2 * t.half) break;
      const bool first = e + j < t.half;
      const int pair = first ? e + j : e + j - t.half;
      const double other = (double)load1(x, row + (first ? e + j + t.half : pair), T());
      const Angle a = angles[pair];
      y[j] = (float)__builtin_fma((double)y[j], a.cos, other * (first ? -a.sin : a.sin));
    }
  }
}

// A row's rounding to its type, as values.
__device__ __forceinline__ void round8(float (&)[8], float) {}
__device__ __forceinline__ void round8(float (&x)[8], Bf16) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const uint32_t w = pack_bf16x2(x[j], x[j + 1]);
    x[j] = u2f(w << 16), x[j + 1] = u2f(w & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void round8(float (&x)[8], F16) {
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = (float)(_Float16)x[j];
}

// Angles of `count` tokens into LDS, [token][pair]; position(i) of the i-th.
template <typename Position>
__device__ __forceinline__ void fill_angles(const Turn& t, Angle* angles, int count, Position position) {
  for (int i = threadIdx.x; i < count * t.half; i += 256) {
    const int token = i / t.half;
    angles[i] = turn_of(t, position(token), i - token * t.half);
  }
}

// One thread's 8 elements: the part-th of a row of head h of token `token` of the
// workgroup's.
struct Place {
  uint32_t token, h, part;
  int64_t row;  // where the row begins in x
};

// put(place, values) for every 8 elements of the rows of tokens first .. first +
// count; begin() comes before, while the first loads are on their way.  The
// four threads of 32 elements stay together: one without elements of its own
// takes those that it had and puts them with own false.
template <typename T, Layout kLayout, typename Begin, typename Put>
__device__ __forceinline__ void for_rows(const Turn& t, const Rows& x, int first, int count, Begin begin, Put put) {
  const uint32_t parts = (uint32_t)x.dim / 8, heads = (uint32_t)x.heads, items = (uint32_t)count * heads * parts;
  // the place of an item, kept up by steps of 256 (a division is some 20
  // instructions)
  uint32_t part = threadIdx.x % parts, h = threadIdx.x / parts % heads, token = threadIdx.x / parts / heads;
  const uint32_t step_part = 256 % parts, step_h = 256 / parts % heads, step_token = 256 / parts / heads;
  constexpr int kAhead = 2;
  Pairs<T, kLayout> raw[2][kAhead];
  Place place[2][kAhead];
  auto load = [&](uint32_t w, Pairs<T, kLayout> (&r)[kAhead], Place (&at)[kAhead]) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const bool own = w + a * 256 < items;
      // past the last: some row of the last token
      at[a] = Place{own ? token : (uint32_t)count - 1, own ? h : 0, own ? part : threadIdx.x % parts, 0};
      at[a].row = (first + (int64_t)at[a].token) * x.sn + (int64_t)at[a].h * x.sh;
      load_pairs<T, kLayout>(t, x.p, at[a].row, (int)at[a].part, r[a]);
      part += step_part, h += step_h, token += step_token;
      if (part >= parts) part -= parts, ++h;
      if (h >= heads) h -= heads, ++token;
    }
  };
  auto work = [&](uint32_t w, const Pairs<T, kLayout> (&r)[kAhead], const Place (&at)[kAhead]) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a) put(at[a], r[a], w + a * 256 < items);
  };
  uint32_t w = threadIdx.x;
  load(w, raw[0], place[0]);
  begin();
  __syncthreads();
  const uint32_t first_item = w & ~255u;
  for (uint32_t s = first_item; s < items; s += 4 * 256) {
    load(w + kAhead * 256, raw[1], place[1]);
    work(w, raw[0], place[0]);
    w += kAhead * 256;
    if (s + kAhead * 256 >= items) break;
    load(w + kAhead * 256, raw[0], place[0]);
    work(w, raw[1], place[1]);
    w += kAhead * 256;
  }
}

// Rows turned into out, which is dense.
template <typename T, Layout kLayout>
__device__ __forceinline__ void put_turned(const Turn& t, const Angle* angles, const Rows& x, void* out, int first,
                                           const Place& at, const Pairs<T, kLayout>& raw, bool own) {
  if (!own) return;
  const int64_t to = ((first + (int64_t)at.token) * x.heads + at.h) * x.dim + 8 * at.part;
  if (8 * (int)at.part >= 2 * t.half) {
    copy_of(out, to, T(), raw.own);
    return;
  }
  float y[8];
  turn_pairs<T, kLayout>(t, angles + at.token * (uint32_t)t.half, x.p, at.row, (int)at.part, raw, y);
  store_of(out, to, T(), y);
}

// Bound by the bytes: every element read and written once (8192 tokens of 32
// heads of 128, bf16: 134 MB in 31 us, 4.3 TB/s).
template <typename T, Layout kLayout>
__global__ __launch_bounds__(256) void rotary_kernel(Turn t, Rows x, void* out, int n, int tokens) {
  extern __shared__ __align__(16) uint8_t shared[];
  Angle* angles = reinterpret_cast<Angle*>(shared);
  const int first = (int)blockIdx.x * tokens, count = n - first < tokens ? n - first : tokens;
  for_rows<T, kLayout>(
      t, x, first, count, [&] { fill_angles(t, angles, count, [&](int i) { return t.positions[first + i]; }); },
      [&](const Place& at, const Pairs<T, kLayout>& raw, bool own) { put_turned<T, kLayout>(t, angles, x, out, first, at, raw, own); });
}

// The new tokens' queries turned, their keys turned and quantized into the
// cache, their values quantized, each kind by workgroups of its own.  Bound by
// the bytes (8 ragged prompts, 10377 tokens of 32 + 8 + 8 heads of 128, fp16: 224
// MB in 56 us, 4.0 TB/s); a decode step by its launch and two chains of loads
// (16 tokens: 5 us).
template <int kDim, typename T, Layout kLayout>
__global__ __launch_bounds__(256) void kv4_append_rotary_kernel(Kv4View c, Kv4Tokens q, Turn t, Rows query, Rows key,
                                                               Rows value, void* out, int kv_tokens, int kv_groups,
                                                               int tokens) {
  extern __shared__ __align__(16) uint8_t shared[];
  __shared__ int32_t places[kMostTokens];
  __shared__ uint32_t rows[kMostTokens];
  Angle* angles = reinterpret_cast<Angle*>(shared);
  // one of each kind in turn while there are all three: those of keys and values
  // are short and begin with a chain of loads, which the others' work covers
  const int groups = (q.n + tokens - 1) / tokens, mixed = kv_groups < groups ? kv_groups : groups;
  const int id = (int)blockIdx.x, rest = id - 3 * mixed;
  const int which = rest < 0 ? id % 3 : (mixed == kv_groups ? 2 : rest & 1);
  const int group = rest < 0 ? id / 3 : mixed + (mixed == kv_groups ? rest : rest / 2);
  const int each = which < 2 ? kv_tokens : tokens;
  const int first = group * each, count = q.n - first < each ? q.n - first : each;
  // The tokens' places and rows in the cache.  A thread has a sequence and the
  // tokens of it that are the workgroup's (one search a token is a chain of
  // loads); a token of no sequence is at place 0 and has no row.
  auto find = [&] {
    if ((int)threadIdx.x < count) places[threadIdx.x] = 0, rows[threadIdx.x] = kNoRow;
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < c.seqs; b += 256) {
      int begin, n;
      kv4_span(q, b, begin, n);
      const int lo = begin > first ? begin : first, end = begin + n < first + count ? begin + n : first + count;
      for (int i = lo; i < end; ++i) {
        const int64_t place = (int64_t)c.lengths[b] - n + (i - begin);
        places[i - first] = (int)place;
        if (which == 2 || place < 0 || place >= (int64_t)c.cap) continue;
        const uint32_t page = kv4_page(c, b, (uint32_t)place);
        if (page < c.pages) rows[i - first] = kv4_row(c, page, 0, (uint32_t)place);
      }
    }
    __syncthreads();
  };
  auto turns = [&] {
    fill_angles(t, angles, count, [&](int i) { return t.positions ? t.positions[first + i] : places[i]; });
  };
  auto to_cache = [&](const Place& at, float (&y)[8], bool own) {
    const uint32_t row = rows[at.token];
    put_codes<kDim>(c, Item{(uint32_t)which, at.h, at.part, row == kNoRow ? kNoRow : row + at.h * c.size, 0}, y, T(), own);
  };
  if (which == 0)
    for_rows<T, kLayout>(
        t, key, first, count, [&] { find(), turns(); },
        [&](const Place& at, const Pairs<T, kLayout>& raw, bool own) {
          float y[8];
          turn_pairs<T, kLayout>(t, angles + at.token * (uint32_t)t.half, key.p, at.row, (int)at.part, raw, y);
          round8(y, T());  // a key has its type's values before it has the cache's
          to_cache(at, y, own);
        });
  else if (which == 1)
    for_rows<T, kNeighbours>(
        t, value, first, count, [&] { find(); },
        [&](const Place& at, const Pairs<T, kNeighbours>& raw, bool own) {
          float y[8];
          values_of(raw.own, T(), y);
          to_cache(at, y, own);
        });
  else
    for_rows<T, kLayout>(
        t, query, first, count,
        [&] {
          if (!t.positions) find();
          turns();
        },
        [&](const Place& at, const Pairs<T, kLayout>& raw, bool own) { put_turned<T, kLayout>(t, angles, query, out, first, at, raw, own); });
}

// Tokens of a workgroup: a round of its threads at least, as many more as leave
// four workgroups for every compute unit, and angles within 32 KB of LDS.
int tokens_of(const Turn& t, int64_t items, int64_t n) {
  int64_t tokens = n / (4ll * num_cus());
  const int64_t least = (256 + items - 1) / items, most = 2048 / t.half < kMostTokens ? 2048 / t.half : kMostTokens;
  if (tokens < least) tokens = least;
  return (int)(tokens > most ? most : tokens);
}

size_t angle_bytes(const Turn& t, int tokens) { return (size_t)tokens * t.half * sizeof(Angle); }

}  // namespace

#define VQX_TYPED(CALL, ...)    \
  do {                          \
    if (dtype == kF32)          \
      CALL(float, __VA_ARGS__); \
    else if (dtype == kBF16)    \
      CALL(Bf16, __VA_ARGS__);  \
    else                        \
      CALL(F16, __VA_ARGS__);   \
  } while (0)
#define VQX_LAYOUTS(CALL)         \
  do {                            \
    if (t.interleaved)            \
      VQX_TYPED(CALL, kNeighbours); \
    else if (t.half % 8 == 0)     \
      VQX_TYPED(CALL, kHalves);   \
    else                          \
      VQX_TYPED(CALL, kSingles);  \
  } while (0)

int rotary(const Turn& t, const Rows& x, int dtype, int64_t n, void* out, hipStream_t st) {
  if (n == 0) return kOk;
  const int tokens = tokens_of(t, (int64_t)x.heads * (x.dim / 8), n);
  const dim3 grid((unsigned)((n + tokens - 1) / tokens));
  const size_t lds = angle_bytes(t, tokens);
#define VQX_ROTARY(T, LAYOUT) hipLaunchKernelGGL((rotary_kernel<T, LAYOUT>), grid, dim3(256), lds, st, t, x, out, (int)n, tokens)
  VQX_LAYOUTS(VQX_ROTARY);
#undef VQX_ROTARY
  return check_launch("rotary");
}

int kv4_append_rotary(const Kv4View& c, int dim, const Kv4Tokens& q, const Turn& t, const Rows& query, const Rows& key,
                      const Rows& value, int dtype, void* out, hipStream_t st) {
  if (q.n == 0) return kOk;
  const int kv_tokens = tokens_of(t, (int64_t)c.kv * (dim / 8), q.n), kv_groups = (q.n + kv_tokens - 1) / kv_tokens;
  const int tokens = tokens_of(t, (int64_t)query.heads * (dim / 8), q.n);
  const dim3 grid(2u * (unsigned)kv_groups + (unsigned)((q.n + tokens - 1) / tokens));
  const size_t lds = angle_bytes(t, tokens > kv_tokens ? tokens : kv_tokens);
#define VQX_APPEND(T, LAYOUT)                                                                                           \
  do {                                                                                                                  \
    auto kernel = dim == 64 ? kv4_append_rotary_kernel<64, T, LAYOUT>                                                   \
                            : (dim == 128 ? kv4_append_rotary_kernel<128, T, LAYOUT> : kv4_append_rotary_kernel<256, T, LAYOUT>); \
    hipLaunchKernelGGL(kernel, grid, dim3(256), lds, st, c, q, t, query, key, value, out, kv_tokens, kv_groups, tokens); \
  } while (0)
  VQX_LAYOUTS(VQX_APPEND);
#undef VQX_APPEND
  return check_launch("kv4_append_rotary");
}
#undef VQX_LAYOUTS
#undef VQX_TYPED

}  // namespace vqx
