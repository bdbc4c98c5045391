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

// What a thread has of a row: its own 8 values from element 8 part on and, for
// the half layout, the 8 that they are paired with.
template <typename T>
struct Pairs {
  Raw8F own, other;
};

__device__ __forceinline__ float load1(const void* p, int64_t at, float) { return static_cast<const float*>(p)[at]; }
__device__ __forceinline__ float load1(const void* p, int64_t at, Bf16) {
  return u2f((uint32_t)static_cast<const uint16_t*>(p)[at] << 16);
}
__device__ __forceinline__ float load1(const void* p, int64_t at, F16) {
  return h2f_exact(static_cast<const uint16_t*>(p)[at]);
}

// Halves of a multiple of 8 are paired 8 by 8.
__device__ __forceinline__ bool paired_whole(const Turn& t) { return (t.half & 7) == 0; }

template <typename T>
__device__ __forceinline__ void load_pairs(const Turn& t, const void* x, int64_t row, int part, Pairs<T>& p) {
  const int e = 8 * part;
  load8(x, row + e, T(), p.own);
  if (!t.interleaved && paired_whole(t) && e < 2 * t.half) load8(x, row + (e < t.half ? e + t.half : e - t.half), T(), p.other);
}

// The thread's 8 values turned; angles: those of the row's token, a pair each.
template <typename T>
__device__ __forceinline__ void turn_pairs(const Turn& t, const Angle* angles, const void* x, int64_t row, int part,
                                           const Pairs<T>& p, float (&y)[8]) {
  const int e = 8 * part;
  values8(p.own, T(), y);
  if (e >= 2 * t.half) return;
  if (t.interleaved) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      if (e + j >= 2 * t.half) break;
      const Angle a = angles[(e + j) / 2];
      const double u = (double)y[j], v = (double)y[j + 1];
      y[j] = (float)__builtin_fma(u, a.cos, -(v * a.sin));
      y[j + 1] = (float)__builtin_fma(u, a.sin, v * a.cos);
    }
  } else if (paired_whole(t)) {
    float z[8];
    values8(p.other, T(), z);
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
  for (int j = 0; j < 8; ++j) x[j] = h2f_exact(f2h_exact(x[j]));
}

// Angles of `count` tokens into LDS, [token][pair]; position(i) of the i-th.
template <typename Position>
__device__ __forceinline__ void fill_angles(const Turn& t, Angle* angles, int count, Position position) {
  for (int i = threadIdx.x; i < count * t.half; i += 256) {
    const int token = i / t.half;
    angles[i] = turn_of(t, position(token), i - token * t.half);
  }
}

// Rows of `heads` heads of tokens first .. first + count turned into out, which
// is dense.  A thread has 8 elements at a time, two loads of them ahead.
template <typename T>
__device__ __forceinline__ void turn_rows(const Turn& t, const Angle* angles, const Rows& x, void* out, int first,
                                          int count) {
  const uint32_t parts = (uint32_t)x.dim / 8, per = (uint32_t)x.heads * parts, items = (uint32_t)count * per;
  constexpr int kAhead = 2;
  for (uint32_t w = threadIdx.x; w < items; w += kAhead * 256) {
    Pairs<T> p[kAhead];
    uint32_t token[kAhead], part[kAhead];
    int64_t row[kAhead], to[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const uint32_t i = w + a * 256 < items ? w + a * 256 : items - 1;
      token[a] = i / per;
      const uint32_t rest = i - token[a] * per, head = rest / parts;
      part[a] = rest - head * parts;
      const int64_t n = first + (int64_t)token[a];
      row[a] = n * x.sn + (int64_t)head * x.sh;
      to[a] = (n * x.heads + head) * x.dim + 8 * part[a];
      load_pairs(t, x.p, row[a], (int)part[a], p[a]);
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (w + a * 256 >= items) break;
      float y[8];
      turn_pairs(t, angles + token[a] * (uint32_t)t.half, x.p, row[a], (int)part[a], p[a], y);
      store8(out, to[a], T(), y);
    }
  }
}

// Bound by the bytes: every element read and written once.
template <typename T>
__global__ __launch_bounds__(256) void rotary_kernel(Turn t, Rows x, void* out, int n, int tokens) {
  extern __shared__ __align__(16) uint8_t shared[];
  Angle* angles = reinterpret_cast<Angle*>(shared);
  const int first = (int)blockIdx.x * tokens, count = n - first < tokens ? n - first : tokens;
  fill_angles(t, angles, count, [&](int i) { return t.positions[first + i]; });
  __syncthreads();
  turn_rows<T>(t, angles, x, out, first, count);
}

// The new tokens' queries turned, their keys turned and quantized into the
// cache, their values quantized: workgroups of keys, then of values, then of
// queries.
template <int kDim, typename T>
__global__ __launch_bounds__(256) void kv4_append_rotary_kernel(Kv4View c, Kv4Tokens q, Kv4Share share, Turn t, Rows query,
                                                               Rows key, Rows value, void* out, int tokens) {
  extern __shared__ __align__(16) uint8_t shared[];
  Angle* angles = reinterpret_cast<Angle*>(shared);
  // a token's place in its sequence, where the caller gives no positions
  auto position = [&](int i) {
    if (t.positions) return t.positions[i];
    const uint32_t b = sequence_of(c, q, i);
    int first, count;
    kv4_span(q, b, first, count);
    return c.lengths[b] - count + (i - first);
  };
  if (blockIdx.x >= 2u * (uint32_t)share.groups) {
    const int first = (int)(blockIdx.x - 2u * (uint32_t)share.groups) * tokens;
    const int count = q.n - first < tokens ? q.n - first : tokens;
    fill_angles(t, angles, count, [&](int i) { return position(first + i); });
    __syncthreads();
    turn_rows<T>(t, angles, query, out, first, count);
    return;
  }
  int begin = 0;
  for_new_values<kDim, Pairs<T>>(
      c, q, share,
      [&](uint32_t plane, int i0, int count) {
        begin = i0;
        if (plane == 0) fill_angles(t, angles, count, [&](int i) { return position(i0 + i); });
      },
      [&](const Item& i, Pairs<T>& p) {
        if (i.plane)
          load8(value.p, i.i * value.sn + (int64_t)i.h * value.sh + i.part * 8, T(), p.own);
        else
          load_pairs(t, key.p, i.i * key.sn + (int64_t)i.h * key.sh, (int)i.part, p);
      },
      [&](const Item& i, const Pairs<T>& p, bool own) {
        float y[8];
        if (i.plane) {
          values8(p.own, T(), y);
        } else {
          turn_pairs(t, angles + (i.i - begin) * t.half, key.p, i.i * key.sn + (int64_t)i.h * key.sh, (int)i.part, p, y);
          round8(y, T());  // a key has its type's values before it has the cache's
        }
        put_codes<kDim>(c, i, y, T(), own);
      });
}

// Tokens of a workgroup: a round of its threads at least, as many more as leave
// four workgroups for every compute unit, and angles within 32 KB of LDS.
int tokens_of(const Turn& t, int64_t items, int64_t n) {
  int64_t tokens = n / (4ll * num_cus());
  const int64_t least = (256 + items - 1) / items, most = t.half > 0 && 2048 / t.half < 32 ? 2048 / t.half : 32;
  if (tokens < least) tokens = least;
  return (int)(tokens > most ? most : tokens);
}

size_t angle_bytes(const Turn& t, int tokens) { return (size_t)tokens * t.half * sizeof(Angle); }

}  // namespace

int rotary(const Turn& t, const Rows& x, int dtype, int64_t n, void* out, hipStream_t st) {
  if (n == 0) return kOk;
  const int tokens = tokens_of(t, (int64_t)x.heads * (x.dim / 8), n);
  const dim3 grid((unsigned)((n + tokens - 1) / tokens));
  const size_t lds = angle_bytes(t, tokens);
  if (dtype == kF32)
    hipLaunchKernelGGL((rotary_kernel<float>), grid, dim3(256), lds, st, t, x, out, (int)n, tokens);
  else if (dtype == kBF16)
    hipLaunchKernelGGL((rotary_kernel<Bf16>), grid, dim3(256), lds, st, t, x, out, (int)n, tokens);
  else
    hipLaunchKernelGGL((rotary_kernel<F16>), grid, dim3(256), lds, st, t, x, out, (int)n, tokens);
  return check_launch("rotary");
}

int kv4_append_rotary(const Kv4View& c, int dim, const Kv4Tokens& q, const Turn& t, const Rows& query, const Rows& key,
                      const Rows& value, int dtype, void* out, hipStream_t st) {
  if (q.n == 0) return kOk;
  Kv4Share share = share_of(c, dim, q.n);
  const int keys = tokens_of(t, (int64_t)c.kv * (dim / 8), q.n);
  if (share.tokens > keys) share = Kv4Share{keys, (int32_t)((q.n + keys - 1) / keys)};
  const int tokens = tokens_of(t, (int64_t)query.heads * (dim / 8), q.n);
  const dim3 grid(2u * (unsigned)share.groups + (unsigned)((q.n + tokens - 1) / tokens));
  const size_t lds = angle_bytes(t, tokens > share.tokens ? tokens : share.tokens);
#define VQX_APPEND(D, T)                                                                                              \
  hipLaunchKernelGGL((kv4_append_rotary_kernel<D, T>), grid, dim3(256), lds, st, c, q, share, t, query, key, value, out, \
                     tokens)
#define VQX_TYPES(D)       \
  if (dtype == kF32)       \
    VQX_APPEND(D, float);  \
  else if (dtype == kBF16) \
    VQX_APPEND(D, Bf16);   \
  else                     \
    VQX_APPEND(D, F16)
  if (dim == 64) {
    VQX_TYPES(64);
  } else if (dim == 128) {
    VQX_TYPES(128);
  } else {
    VQX_TYPES(256);
  }
#undef VQX_TYPES
#undef VQX_APPEND
  return check_launch("kv4_append_rotary");
}

}  // namespace vqx
