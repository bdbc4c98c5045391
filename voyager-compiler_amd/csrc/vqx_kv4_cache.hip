// Writing, reading and thinning out a 4-bit cache of keys and values.
//
// All of it moves bytes: a value is read once, quantized in registers and
// written as 4.25 bits, and back.
#include "vqx_kv4.h"

namespace vqx {
namespace {

// ---------------------------------------------------------------------------
// append: x -> codes and scales
// ---------------------------------------------------------------------------
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

// work(plane, token, head, part, row) for every 8 values of this workgroup's
// tokens; the rows are found once a token, for all of them at a time.
template <int kDim, typename F>
__device__ __forceinline__ void for_new_values(const Kv4View& c, const Kv4Tokens& q, const Kv4Share& share, F work) {
  constexpr uint32_t kPerRow = kDim / 8;
  __shared__ uint32_t rows[kMostTokens];
  const uint32_t plane = blockIdx.x >= (uint32_t)share.groups;
  const int i0 = (int)(blockIdx.x - plane * (uint32_t)share.groups) * share.tokens;
  const int count = q.n - i0 < share.tokens ? q.n - i0 : share.tokens;
  if ((int)threadIdx.x < count) rows[threadIdx.x] = new_token_row(c, q, i0 + (int)threadIdx.x);
  __syncthreads();
  // the four threads of a block stay together: items are a multiple of 8
  const uint32_t per = c.kv * kPerRow, items = (uint32_t)count * per;
  uint32_t token = threadIdx.x / per, rest = threadIdx.x % per;
  const uint32_t step_token = 256 / per, step_rest = 256 % per;
  for (uint32_t w = threadIdx.x; w < items; w += 256) {
    const uint32_t h = rest / kPerRow, part = rest % kPerRow, row = rows[token];
    work(plane, i0 + (int)token, h, part, row == kNoRow ? kNoRow : row + h * c.size);
    token += step_token, rest += step_rest;
    if (rest >= per) rest -= per, ++token;
  }
}

// Bound by the values' bytes; a call of a decode step by its launch.
template <int kDim, typename T>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4View c, Kv4Tokens q, Kv4Share share, const void* key,
                                                         const void* value, int64_t key_sn, int64_t key_sh,
                                                         int64_t value_sn, int64_t value_sh) {
  constexpr uint32_t kPerRow = kDim / 8;
  for_new_values<kDim>(c, q, share, [&](uint32_t plane, int i, uint32_t h, uint32_t part, uint32_t row) {
    Raw8F raw;
    load8(plane ? value : key, (int64_t)i * (plane ? value_sn : key_sn) + (int64_t)h * (plane ? value_sh : key_sh) + part * 8,
          T(), raw);
    float x[8];
    values8(raw, T(), x);
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
    if (row == kNoRow) return;
    const uint64_t at = plane * c.plane_rows + row;
    reinterpret_cast<uint32_t*>(c.codes)[at * kPerRow + part] = finite ? code : 0u;
    // a block with an infinity or a NaN is NaN as a whole
    if ((part & 3) == 0) c.scales[at * (kPerRow / 4) + part / 4] = (uint8_t)(finite ? e + 127 : 255);
  });
}

template <int kDim, typename T>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4View c, Kv4Tokens q, Kv4Share share, void* key, void* value) {
  constexpr uint32_t kPerRow = kDim / 8;
  for_new_values<kDim>(c, q, share, [&](uint32_t plane, int i, uint32_t h, uint32_t part, uint32_t row) {
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (row != kNoRow) {
      const uint64_t at = plane * c.plane_rows + row;
      const uint32_t code = reinterpret_cast<const uint32_t*>(c.codes)[at * kPerRow + part];
      const float s = kv4_scale(c.scales[at * (kPerRow / 4) + part / 4]);
      fp4_values(code, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= s;
    }
    store8(plane ? value : key, (((int64_t)i * c.kv + h) * kPerRow + part) * 8, T(), x);
  });
}

// ---------------------------------------------------------------------------
// evict: the heaviest and the latest tokens of each head
// ---------------------------------------------------------------------------
// The order of weights as one of unsigned numbers; both zeros are one weight,
// a NaN is above all.  No weight has a key below that of -infinity, 0x7FFFFF;
// key 0 stands for no token.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xFFFFFFFFu;
  const uint32_t b = w == 0.0f ? 0u : f2u(w);
  return b >> 31 ? ~b : b | 0x80000000u;
}
// The weight of a key.
__device__ __forceinline__ float key_weight(uint32_t k) { return u2f(k >> 31 ? k & 0x7FFFFFFFu : ~k); }

constexpr int kSelectThreads = 1024;
constexpr int kBins = 2048;
constexpr int kCopies = 4;  // of a histogram, by lane: many weights share a bin

// One workgroup picks the tokens of one head of one sequence: of the `old`
// tokens before the latest `recent` it finds the weight of the room-th heaviest
// by histograms of 11, 11 and 10 bits of the key, fewer where one settles it,
// then each wave counts and writes the tokens of its own run, lowest first, so
// that equal weights go by their place.  A wave's run is steps of 64 tokens;
// kHeld of them stay in registers, so that up to 1024 kHeld tokens are read
// once: bound by the latency of that and by the histogram's LDS atomics (read
// anew for each pass, 50001 tokens took 48 us).  Longer runs are read again.
template <int kHeld, bool kAll>
__global__ __launch_bounds__(kSelectThreads) void kv4_select_kernel(Kv4View c, const float* weights,
                                                                    int64_t weights_len, int budget, int recent,
                                                                    int32_t* index, int32_t* kept,
                                                                    float* out_weights) {
  __shared__ uint32_t hist[kBins][kCopies];
  __shared__ uint32_t wave_sum[kSelectThreads / 64], wave_tie[kSelectThreads / 64];
  __shared__ uint32_t found[3];
  const uint32_t b = blockIdx.x / c.kv;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  constexpr int kWaves = kSelectThreads / 64;
  int n = kv4_length(c, b);
  if (n > weights_len) n = (int)weights_len;
  const float* w = weights + (int64_t)blockIdx.x * weights_len;
  int32_t* idx = index + (int64_t)blockIdx.x * budget;
  float* ow = out_weights + (int64_t)blockIdx.x * budget;
  const int keep = n < budget ? n : budget;
  if (tid == 0 && blockIdx.x % c.kv == 0) kept[b] = keep;
  for (int j = keep + tid; j < budget; j += kSelectThreads) idx[j] = -1, ow[j] = 0.0f;
  const int old = n > recent ? n - recent : 0;
  const int room = keep - (n - old);  // of the old tokens; recent <= budget, so it is not negative
  // the latest
  for (int j = old + tid; j < n; j += kSelectThreads) idx[room + j - old] = j, ow[room + j - old] = w[j];
  if (room == 0) return;
  if (room == old) {
    for (int j = tid; j < old; j += kSelectThreads) idx[j] = j, ow[j] = w[j];
    return;
  }
  const int steps = (old + 63) / 64, per = (steps + kWaves - 1) / kWaves;
  // the wave's run of tokens; work(token, key) is for all of it, and for tokens
  // past its limit with key 0
  const int begin = wave * per * 64, end = begin + per * 64, limit = end < old ? end : old;
  uint32_t held[kHeld];
  auto read = [&](int at) {
#pragma unroll
    for (int a = 0; a < kHeld; ++a) {
      const int j = at + a * 64 + lane;
      const float x = w[j < limit ? j : old - 1];
      held[a] = j < limit ? weight_key(x) : 0u;
    }
  };
  if (kAll) read(begin);
  auto each = [&](auto work) {
    for (int at = begin; at < limit; at += kHeld * 64) {
      if (!kAll) read(at);
#pragma unroll
      for (int a = 0; a < kHeld; ++a) work(at + a * 64 + lane, held[a]);
    }
  };
  uint32_t prefix = 0, need = (uint32_t)room;
  int low = 32;  // bits of the key below those that prefix settles
#pragma clang loop unroll(disable)
  while (low > 0) {
    const int bits = low == 10 ? 10 : 11;
    const uint32_t known = low == 32 ? 0u : ~0u << low;
    low -= bits;
    for (int j = tid; j < kBins * kCopies; j += kSelectThreads) (&hist[0][0])[j] = 0;
    __syncthreads();
    each([&](int, uint32_t k) {
      // counts: no order in them; no token's key comes into bin 0
      if ((k & known) == prefix)
        atomicAdd(&hist[k >> low & ((1u << bits) - 1)][lane & (kCopies - 1)], 1u);
    });
    __syncthreads();
    // bin 2047 - 2 tid and the one below it: how many keys are above
    const int hi = kBins - 1 - 2 * tid;
    uint32_t h0 = 0, h1 = 0;
#pragma unroll
    for (int a = 0; a < kCopies; ++a) h0 += hist[hi][a], h1 += hist[hi - 1][a];
    uint32_t sum = h0 + h1;
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t o = __shfl_up(sum, d);
      if (lane >= d) sum += o;
    }
    if (lane == 63) wave_sum[wave] = sum;
    __syncthreads();
    uint32_t above = sum - h0 - h1;
    for (int k = 0; k < wave; ++k) above += wave_sum[k];
    if (above < need && need <= above + h0) found[0] = (uint32_t)hi, found[1] = need - above, found[2] = h0;
    if (above + h0 < need && need <= above + h0 + h1)
      found[0] = (uint32_t)hi - 1, found[1] = need - above - h0, found[2] = h1;
    __syncthreads();
    prefix |= found[0] << low;
    need = found[1];
    const bool whole = need == found[2] && prefix != 0;  // every key of the bin is kept: all from its lowest on
    __syncthreads();
    if (whole) {
      prefix -= 1;
      need = 0;
      break;
    }
  }
  // keys above prefix are kept, and the first `need` of those that equal it
  uint32_t more = 0, tie = 0;
  each([&](int, uint32_t k) {
    more += (uint32_t)__popcll(__ballot(k > prefix));
    tie += (uint32_t)__popcll(__ballot(k == prefix));
  });
  if (lane == 0) wave_sum[wave] = more, wave_tie[wave] = tie;
  __syncthreads();
  uint32_t at = 0, ties = 0;  // kept and equal tokens before this wave's run
  for (int k = 0; k < wave; ++k) at += wave_sum[k], ties += wave_tie[k];
  at += ties < need ? ties : need;
  const uint64_t below = (1ull << lane) - 1;
  // the masks of the count are made again: kept, they spill
  prefix = (uint32_t)__builtin_amdgcn_readfirstlane((int)prefix);
  asm volatile("" : "+s"(prefix));
  each([&](int j, uint32_t k) {
    const uint64_t eq = __ballot(k == prefix);
    const bool take = k > prefix || (k == prefix && ties + (uint32_t)__popcll(eq & below) < need);
    const uint64_t all = __ballot(take);
    if (take) {
      const uint32_t p = at + (uint32_t)__popcll(all & below);
      idx[p] = j;
      ow[p] = key_weight(k);
    }
    at += (uint32_t)__popcll(all);
    ties += (uint32_t)__popcll(eq);
  });
}

// The kept tokens' rows into the other cache: D / 32 lanes a row of 16 bytes
// each, the first of them with the row's scales as well.
template <int D>
__global__ __launch_bounds__(256) void kv4_move_kernel(Kv4View c, Kv4View out, const int32_t* index, int budget,
                                                       uint64_t items) {
  constexpr int kLanes = D / 32;
  for (uint64_t w = (uint64_t)blockIdx.x * 256 + threadIdx.x; w < items; w += (uint64_t)gridDim.x * 256) {
    const uint64_t slot = w / kLanes;
    const uint32_t part = (uint32_t)(w % kLanes);
    const int t = index[slot];
    if (t < 0) continue;
    const uint64_t head = slot / (uint32_t)budget;
    const uint32_t j = (uint32_t)(slot - head * (uint32_t)budget);
    const uint32_t b = (uint32_t)(head / c.kv), h = (uint32_t)(head - (uint64_t)b * c.kv);
    const uint32_t from = kv4_page(c, b, (uint32_t)t), to = kv4_page(out, b, j);
    if (to >= out.pages) continue;
    const uint64_t src = kv4_row(c, from, h, (uint32_t)t), dst = kv4_row(out, to, h, j);
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
      const uint64_t s = plane * c.plane_rows + src, d = plane * out.plane_rows + dst;
      u32x4 v = {0u, 0u, 0u, 0u};  // a token without a page is kept as zeros
      if (from < c.pages) v = ld_nt(reinterpret_cast<const u32x4*>(c.codes) + s * kLanes + part);
      reinterpret_cast<u32x4*>(out.codes)[d * kLanes + part] = v;
      out.scales[d * kLanes + part] = from < c.pages ? c.scales[s * kLanes + part] : (uint8_t)0;
    }
  }
}

}  // namespace

#define VQX_KV4_EACH(CALL)                                             \
  do {                                                                 \
    if (dim == 64) {                                                   \
      VQX_KV4_TYPES(CALL, 64);                                         \
    } else if (dim == 128) {                                           \
      VQX_KV4_TYPES(CALL, 128);                                        \
    } else {                                                           \
      VQX_KV4_TYPES(CALL, 256);                                        \
    }                                                                  \
  } while (0)
#define VQX_KV4_TYPES(CALL, D) \
  if (dtype == kF32)           \
    CALL(D, float);            \
  else if (dtype == kBF16)     \
    CALL(D, Bf16);             \
  else                         \
    CALL(D, F16)

int kv4_append(const Kv4View& c, int dim, const Kv4Tokens& t, const void* key, const void* value, int dtype,
               int64_t key_sn, int64_t key_sh, int64_t value_sn, int64_t value_sh, hipStream_t st) {
  if (t.n == 0) return kOk;
  const Kv4Share share = share_of(c, dim, t.n);
#define VQX_KV4_APPEND(D, T)                                                                                       \
  hipLaunchKernelGGL((kv4_append_kernel<D, T>), dim3(2u * (unsigned)share.groups), dim3(256), 0, st, c, t, share, \
                     key, value, key_sn, key_sh, value_sn, value_sh)
  VQX_KV4_EACH(VQX_KV4_APPEND);
#undef VQX_KV4_APPEND
  return check_launch("kv4_append");
}

int kv4_read(const Kv4View& c, int dim, const Kv4Tokens& t, void* key, void* value, int dtype, hipStream_t st) {
  if (t.n == 0) return kOk;
  const Kv4Share share = share_of(c, dim, t.n);
#define VQX_KV4_READ(D, T)                                                                                       \
  hipLaunchKernelGGL((kv4_read_kernel<D, T>), dim3(2u * (unsigned)share.groups), dim3(256), 0, st, c, t, share, \
                     key, value)
  VQX_KV4_EACH(VQX_KV4_READ);
#undef VQX_KV4_READ
  return check_launch("kv4_read");
}

int kv4_evict(const Kv4View& c, int dim, const float* weights, int64_t weights_len, int budget, int recent,
              const Kv4View& out, int32_t* index, int32_t* kept, float* out_weights, hipStream_t st) {
  if (c.seqs == 0) return kOk;
  // the weights of a head in registers where they fit
#define VQX_KV4_SELECT(HELD, ALL)                                                                                  \
  hipLaunchKernelGGL((kv4_select_kernel<HELD, ALL>), dim3(c.seqs * c.kv), dim3(kSelectThreads), 0, st, c, weights, \
                     weights_len, budget, recent, index, kept, out_weights)
  const int64_t most = weights_len < (int64_t)c.cap ? weights_len : (int64_t)c.cap;
  if (most <= 8 * kSelectThreads)
    VQX_KV4_SELECT(8, true);
  else if (most <= 56 * kSelectThreads)
    VQX_KV4_SELECT(56, true);
  else
    VQX_KV4_SELECT(16, false);
#undef VQX_KV4_SELECT
  int rc = check_launch("kv4_evict (selection)");
  if (rc != kOk) return rc;
  const uint64_t items = (uint64_t)c.seqs * c.kv * (uint64_t)budget * (uint64_t)(dim / 32);
  const unsigned grid = grid_for((int64_t)items, 256, 16);
#define VQX_KV4_MOVE(D) \
  hipLaunchKernelGGL((kv4_move_kernel<D>), dim3(grid), dim3(256), 0, st, c, out, index, budget, items)
  if (dim == 64)
    VQX_KV4_MOVE(64);
  else if (dim == 128)
    VQX_KV4_MOVE(128);
  else
    VQX_KV4_MOVE(256);
#undef VQX_KV4_MOVE
  return check_launch("kv4_evict (move)");
}

}  // namespace vqx
