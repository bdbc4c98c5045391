// Values on their way into a 4-bit cache and out of it: loads and stores of 8, the
// rounding to fp4, and how the new tokens' values are shared out.
#pragma once

#include "vqx_kv4.h"

namespace vqx {
namespace {

// floor(log2) of a block's largest magnitude, as quantize_mx_packed has it: the
// log is rounded to the input's type first (bf16: log2floor_bf16).  In fp32 the
// log reaches the integer above for the last few mantissas of a binade: the
// top floor(2^24 (1 - 2^(-u / 2))) of them, u the spacing of fp32 next to that
// integer.  A fp16 magnitude is never as near to the next power of two.
__device__ __forceinline__ int log2_floor(float amax, float) {
  const uint32_t b = f2u(amax), m = b & 0x7FFFFFu;
  const int p = (int)(b >> 23) - 127;
  if (p < -126 || p == -1) return p;  // below fp32's normal range every scale is the smallest
  const uint32_t n = p >= 0 ? (uint32_t)p + 1u : (uint32_t)(-p - 1);
  int band = 31 - clz32(n);
  if (p >= 0 && (n & (n - 1u)) == 0) band -= 1;
  const uint64_t kTop = 0x2C160B0502010000ull;  // 0, 0, 1, 2, 5, 11, 22, 44 for bands -1 .. 6
  const uint32_t top = (uint32_t)(kTop >> (8 * (band + 1))) & 0xFFu;
  return p + (m + top >= 0x800000u ? 1 : 0);
}
struct Bf16 {};
struct F16 {};
__device__ __forceinline__ int log2_floor(float amax, F16) { return (int)(f2u(amax) >> 23) - 127; }
__device__ __forceinline__ int log2_floor(float amax, Bf16) { return log2floor_bf16(f2u(amax) >> 16); }

// 8 consecutive values as they are, and as fp32 (exact).
typedef u32x4 Raw8F[2];
__device__ __forceinline__ void load8(const void* p, int64_t at, float, Raw8F& r) {
  const u32x4* q = reinterpret_cast<const u32x4*>(static_cast<const float*>(p) + at);
  r[0] = ld_nt(q), r[1] = ld_nt(q + 1);
}
template <typename T>
__device__ __forceinline__ void load8(const void* p, int64_t at, T, Raw8F& r) {
  r[0] = ld_nt(reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + at));
}
__device__ __forceinline__ void values8(const Raw8F& r, float, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = u2f(r[0][i]), x[i + 4] = u2f(r[1][i]);
}
__device__ __forceinline__ void values8(const Raw8F& r, Bf16, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = u2f(r[0][i] << 16), x[2 * i + 1] = u2f(r[0][i] & 0xFFFF0000u);
}
__device__ __forceinline__ void values8(const Raw8F& r, F16, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = h2f_exact(r[0][i] & 0xFFFFu), x[2 * i + 1] = h2f_exact(r[0][i] >> 16);
}
__device__ __forceinline__ void store8(void* p, int64_t at, float, const float (&x)[8]) {
  f32x4* q = reinterpret_cast<f32x4*>(static_cast<float*>(p) + at);
  const f32x4 a = {x[0], x[1], x[2], x[3]}, b = {x[4], x[5], x[6], x[7]};
  st_nt(q, a);
  st_nt(q + 1, b);
}
__device__ __forceinline__ void store8(void* p, int64_t at, Bf16, const float (&x)[8]) {
  u32x4 a;
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
  st_nt(reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + at), a);
}
__device__ __forceinline__ void store8(void* p, int64_t at, F16, const float (&x)[8]) {
  u32x4 a;
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = f2h_exact(x[2 * i]) | f2h_exact(x[2 * i + 1]) << 16;
  st_nt(reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + at), a);
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// The codes of 8 quotients that are bf16 values, two a word: the nearest of 0,
// 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even code, signs kept (the instruction's
// own rounding).
__device__ __forceinline__ uint32_t fp4_codes(const uint32_t (&v)[4]) {
  uint32_t code = 0;
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2, v[0]), 1.0f, 0);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2, v[1]), 1.0f, 1);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2, v[2]), 1.0f, 2);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2, v[3]), 1.0f, 3);
  return code;
}
__device__ __forceinline__ void fp4_values(uint32_t code, float (&x)[8]) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 0),
              b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 1),
              c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 2),
              d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 3);
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y, x[4] = c.x, x[5] = c.y, x[6] = d.x, x[7] = d.y;
}

// The sequence of new token i: the last b with cu[b] <= i.
__device__ __forceinline__ uint32_t sequence_of(const Kv4View& c, const Kv4Tokens& q, int i) {
  if (!q.cu) return (uint32_t)(i / q.each);
  uint32_t lo = 0, hi = c.seqs;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (q.cu[mid] <= i)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// The row of new token i of head 0 (head h is h * size further), kNoRow where
// it has none: a place before the sequence's first token or past its room, or a
// page that is none.
constexpr uint32_t kNoRow = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t new_token_row(const Kv4View& c, const Kv4Tokens& q, int i) {
  const uint32_t b = sequence_of(c, q, i);
  int first, count;
  kv4_span(q, b, first, count);
  const int64_t pos = (int64_t)c.lengths[b] - count + (i - first);
  if (i < first || i >= first + count || pos < 0 || pos >= (int64_t)c.cap) return kNoRow;
  const uint32_t page = kv4_page(c, b, (uint32_t)pos);
  return page < c.pages ? kv4_row(c, page, 0, (uint32_t)pos) : kNoRow;
}

constexpr int kMostTokens = 32;  // of a workgroup

// How new tokens are shared out: a workgroup has `tokens` of them in one plane;
// its threads go over their values, 8 each, four threads a block, D / 8 a row.
struct Kv4Share {
  int32_t tokens, groups;  // workgroups of a plane
};
Kv4Share share_of(const Kv4View& c, int dim, int n) {
  // a few rounds of the 256 threads each, but enough workgroups to fill the card
  const int64_t items = (int64_t)c.kv * (dim / 8);
  int64_t tokens = n / (4ll * num_cus());
  const int64_t least = (256 + items - 1) / items;
  if (tokens < least) tokens = least;
  if (tokens > kMostTokens) tokens = kMostTokens;
  return Kv4Share{(int32_t)tokens, (int32_t)((n + tokens - 1) / tokens)};
}

// One thread's 8 values: the part-th of a row of head h of new token i.
struct Item {
  uint32_t plane, h, part, row;
  int i;
};

// take(item, what) and then put(item, what) for every 8 values of this
// workgroup's tokens, kAhead of them taken before the first is put; the rows are
// found once a token, for all of them at a time.  A thread without an item of
// its own takes the last one and does not put it, so that the four threads of a
// block stay together.
template <int kDim, typename What, typename Take, typename Put>
__device__ __forceinline__ void for_new_values(const Kv4View& c, const Kv4Tokens& q, const Kv4Share& share, Take take,
                                               Put put) {
  constexpr uint32_t kPerRow = kDim / 8;
  constexpr int kAhead = 2;
  __shared__ uint32_t rows[kMostTokens];
  const uint32_t plane = blockIdx.x >= (uint32_t)share.groups;
  const int i0 = (int)(blockIdx.x - plane * (uint32_t)share.groups) * share.tokens;
  const int count = q.n - i0 < share.tokens ? q.n - i0 : share.tokens;
  if ((int)threadIdx.x < count) rows[threadIdx.x] = new_token_row(c, q, i0 + (int)threadIdx.x);
  __syncthreads();
  const uint32_t per = c.kv * kPerRow, items = (uint32_t)count * per;
  uint32_t token = threadIdx.x / per, rest = threadIdx.x % per;
  const uint32_t step_token = 256 / per, step_rest = 256 % per;
  for (uint32_t w = threadIdx.x; w < items; w += kAhead * 256) {
    Item item[kAhead];
    What what[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const bool own = w + a * 256 < items;
      const uint32_t t = own ? token : (uint32_t)count - 1, r = own ? rest : per - kPerRow + threadIdx.x % kPerRow;
      const uint32_t h = r / kPerRow, row = rows[t];
      item[a] = Item{plane, h, r % kPerRow, row == kNoRow ? kNoRow : row + h * c.size, i0 + (int)t};
      take(item[a], what[a]);
      token += step_token, rest += step_rest;
      if (rest >= per) rest -= per, ++token;
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) put(item[a], what[a], w + a * 256 < items);
  }
}

// A thread's 8 values of a new token, quantized into its place; the four threads
// of a block call together.
template <int kDim, typename T>
__device__ __forceinline__ void put_codes(const Kv4View& c, const Item& t, const float (&x)[8], T, bool own) {
  constexpr uint32_t kPerRow = kDim / 8;
  // the largest magnitude as a bit pattern, so that a NaN is the largest
  uint32_t amax = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) amax = umax32(amax, f2u(x[j]) & 0x7FFFFFFFu);
  amax = umax32(amax, (uint32_t)__shfl_xor((int)amax, 1));
  amax = umax32(amax, (uint32_t)__shfl_xor((int)amax, 2));
  int e = (amax == 0 ? -126 : log2_floor(u2f(amax), T())) - 2;
  e = e < -127 ? -127 : (e > 127 ? 127 : e);
  const bool finite = amax < 0x7F800000u;
  const float r = exp2i(-e);
  uint32_t v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)  // + 0: both zeros have code 0
    v[j] = pack_bf16x2(__builtin_fmaf(x[2 * j], r, 0.0f), __builtin_fmaf(x[2 * j + 1], r, 0.0f));
  const uint32_t code = fp4_codes(v);
  if (t.row == kNoRow || !own) return;
  const uint64_t at = t.plane * c.plane_rows + t.row;
  reinterpret_cast<uint32_t*>(c.codes)[at * kPerRow + t.part] = finite ? code : 0u;
  // a block with an infinity or a NaN is NaN as a whole
  if ((t.part & 3) == 0) c.scales[at * (kPerRow / 4) + t.part / 4] = (uint8_t)(finite ? e + 127 : 255);
}

}  // namespace
}  // namespace vqx
