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

// Bound by the values' bytes (10377 tokens of 32 heads of 128, bf16, keys and
// values: 215 MB in 56 us, 3.9 TB/s; reading them back 38 us); a call of a decode
// step by its launch (3.4 us).
template <int kDim, typename T>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4View c, Kv4Tokens q, Kv4Share share, const void* key,
                                                         const void* value, int64_t key_sn, int64_t key_sh,
                                                         int64_t value_sn, int64_t value_sh) {
  constexpr uint32_t kPerRow = kDim / 8;
  struct Raw {
    Raw8F v;
  };
  for_new_values<kDim, Raw>(
      c, q, share,
      [&](const Item& t, Raw& raw) {
        load8(t.plane ? value : key,
              (int64_t)t.i * (t.plane ? value_sn : key_sn) + (int64_t)t.h * (t.plane ? value_sh : key_sh) + t.part * 8, T(),
              raw.v);
      },
      [&](const Item& t, const Raw& raw, bool own) {
        float x[8];
        values8(raw.v, T(), x);
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
      });
}

template <int kDim, typename T>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4View c, Kv4Tokens q, Kv4Share share, void* key, void* value) {
  constexpr uint32_t kPerRow = kDim / 8;
  struct Raw {
    uint32_t code, scale;
  };
  for_new_values<kDim, Raw>(
      c, q, share,
      [&](const Item& t, Raw& raw) {
        raw = Raw{0u, 127u};
        if (t.row != kNoRow) {
          const uint64_t at = t.plane * c.plane_rows + t.row;
          raw.code = reinterpret_cast<const uint32_t*>(c.codes)[at * kPerRow + t.part];
          raw.scale = c.scales[at * (kPerRow / 4) + t.part / 4];
        }
      },
      [&](const Item& t, const Raw& raw, bool own) {
        float x[8];
        fp4_values(raw.code, x);
        const float s = kv4_scale(raw.scale);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= s;
        if (own) store8(t.plane ? value : key, (((int64_t)t.i * c.kv + t.h) * kPerRow + t.part) * 8, T(), x);
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

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;
constexpr int kBins = 2048;  // two a thread
constexpr int kCopies = 4;   // of a histogram, by lane: many weights share a bin
constexpr int kHeld = 8;     // weights of a thread
constexpr int kSlice = kHeld * kSelectThreads;  // tokens of a workgroup that holds them
constexpr int kMostSlices = 16;
constexpr int kState = 4;  // words that a slice hands to its next launch

// What is kept of one head of one sequence: all but the room-th heaviest of its
// `old` tokens before the latest `recent` ones.
struct Selection {
  int n, keep, old, room;
  const float* w;
  int32_t* idx;
  float* ow;
};
__device__ __forceinline__ Selection selection_of(const Kv4View& c, uint32_t head, const float* weights,
                                                  int64_t weights_len, int budget, int recent, int32_t* index,
                                                  float* out_weights) {
  Selection s;
  s.n = kv4_length(c, head / c.kv);
  if (s.n > weights_len) s.n = (int)weights_len;
  s.keep = s.n < budget ? s.n : budget;
  s.old = s.n > recent ? s.n - recent : 0;
  s.room = s.keep - (s.n - s.old);  // recent <= budget, so it is not negative
  s.w = weights + (int64_t)head * weights_len;
  s.idx = index + (int64_t)head * budget;
  s.ow = out_weights + (int64_t)head * budget;
  return s;
}
// What needs no weight to decide: the latest tokens, the end, and all old ones
// where there is room for all.  Thread t of `threads`.
__device__ __forceinline__ void keep_latest(const Selection& s, int budget, int t, int threads) {
  for (int j = s.keep + t; j < budget; j += threads) s.idx[j] = -1, s.ow[j] = 0.0f;
  for (int j = s.old + t; j < s.n; j += threads) s.idx[s.room + j - s.old] = j, s.ow[s.room + j - s.old] = s.w[j];
  if (s.room == s.old)
    for (int j = t; j < s.old; j += threads) s.idx[j] = j, s.ow[j] = s.w[j];
}

struct SelectShared {
  uint32_t hist[kBins][kCopies];
  uint32_t wave_sum[kSelectWaves], wave_tie[kSelectWaves];
  uint32_t found[3];
};

// How far the key of the room-th heaviest is known: its bits from `low` up, and
// that the `need`-th heaviest of the keys with those bits is meant.  Where all
// of them are kept (`settled`) prefix is the key below the lowest of them, and
// none that equals it is kept.
struct Threshold {
  uint32_t prefix, need;
  int low;
  bool settled;
  __device__ __forceinline__ int bits() const { return low == 10 ? 10 : 11; }
};

// From the counts of the two bins of this thread, 2047 - 2 tid and the one
// below it, over all tokens: the bin of the need-th heaviest, which is returned.
__device__ __forceinline__ uint32_t refine(SelectShared& sh, uint32_t h0, uint32_t h1, Threshold& t) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = kBins - 1 - 2 * tid;
  uint32_t sum = h0 + h1;
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t o = __shfl_up(sum, d);
    if (lane >= d) sum += o;
  }
  if (lane == 63) sh.wave_sum[wave] = sum;
  __syncthreads();
  uint32_t above = sum - h0 - h1;
  for (int k = 0; k < wave; ++k) above += sh.wave_sum[k];
  if (above < t.need && t.need <= above + h0) sh.found[0] = (uint32_t)hi, sh.found[1] = t.need - above, sh.found[2] = h0;
  if (above + h0 < t.need && t.need <= above + h0 + h1)
    sh.found[0] = (uint32_t)hi - 1, sh.found[1] = t.need - above - h0, sh.found[2] = h1;
  __syncthreads();
  const uint32_t bin = sh.found[0];
  t.low -= t.bits();
  t.prefix |= bin << t.low;
  t.need = sh.found[1];
  if (t.need == sh.found[2] && t.low > 0) t.settled = true, t.prefix -= 1, t.need = 0;
  __syncthreads();
  return bin;
}

// The histogram of the keys that have the threshold's known bits, in LDS.
template <typename F>
__device__ __forceinline__ void histogram(SelectShared& sh, const Threshold& t, F each) {
  const uint32_t known = t.low == 32 ? 0u : ~0u << t.low;
  const int shift = t.low - t.bits();
  const uint32_t mask = (1u << t.bits()) - 1u;
  for (int j = threadIdx.x; j < kBins * kCopies; j += kSelectThreads) (&sh.hist[0][0])[j] = 0;
  __syncthreads();
  each([&](int, uint32_t k) {
    // counts: no order in them
    if ((k & known) == t.prefix && k != 0) atomicAdd(&sh.hist[k >> shift & mask][threadIdx.x & (kCopies - 1)], 1u);
  });
  __syncthreads();
}
__device__ __forceinline__ uint32_t bin_count(const SelectShared& sh, int bin) {
  uint32_t h = 0;
#pragma unroll
  for (int a = 0; a < kCopies; ++a) h += sh.hist[bin][a];
  return h;
}

// Keys above the threshold and the first of those that equal it, written in
// their order from place `at`; `ties` of the equal ones come before.
template <typename F>
__device__ __forceinline__ void write_kept(SelectShared& sh, const Selection& s, const Threshold& t, uint32_t at,
                                           uint32_t ties, F each) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t more = 0, tie = 0;
  each([&](int, uint32_t k) {
    more += (uint32_t)__popcll(__ballot(k > t.prefix));
    tie += (uint32_t)__popcll(__ballot(k == t.prefix));
  });
  if (lane == 0) sh.wave_sum[wave] = more, sh.wave_tie[wave] = tie;
  __syncthreads();
  for (int k = 0; k < wave; ++k) at += sh.wave_sum[k], ties += sh.wave_tie[k];
  at += ties < t.need ? ties : t.need;
  const uint64_t below = (1ull << lane) - 1;
  each([&](int j, uint32_t k) {
    const uint64_t eq = __ballot(k == t.prefix);
    const bool take = k > t.prefix || (k == t.prefix && ties + (uint32_t)__popcll(eq & below) < t.need);
    const uint64_t all = __ballot(take);
    if (take) {
      const uint32_t p = at + (uint32_t)__popcll(all & below);
      s.idx[p] = j;
      s.ow[p] = key_weight(k);
    }
    at += (uint32_t)__popcll(all);
    ties += (uint32_t)__popcll(eq);
  });
}

// A run of tokens, cut into one of steps of 64 for each wave; work(token, key)
// is called for all of a wave's, and with key 0 for tokens past its limit.
struct WaveRun {
  int begin, limit;
};
__device__ __forceinline__ WaveRun wave_run(int begin, int end, int waves) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = ((end - begin + 63) / 64 + waves - 1) / waves * 64, first = begin + wave * per;
  return WaveRun{first, first + per < end ? first + per : end};
}
__device__ __forceinline__ void read_keys(const Selection& s, const WaveRun& r, int at, uint32_t (&k)[kHeld]) {
#pragma unroll
  for (int a = 0; a < kHeld; ++a) {
    const int j = at + a * 64 + (threadIdx.x & 63);
    const float x = s.w[j < r.limit ? j : s.old - 1];
    k[a] = j < r.limit ? weight_key(x) : 0u;
  }
}

// Up to 8192 tokens: one workgroup picks the tokens of one head.  It finds the
// weight of the room-th heaviest by histograms of 11, 11 and 10 bits of the
// key, fewer where one settles it, then each wave counts and writes the tokens
// of its own run, lowest first, so that equal weights go by their place.  The
// weights are read once: bound by a few latencies and barriers (640 tokens: 11
// us).
__global__ __launch_bounds__(kSelectThreads) void kv4_select_kernel(Kv4View c, const float* weights,
                                                                    int64_t weights_len, int budget, int recent,
                                                                    int32_t* index, int32_t* kept,
                                                                    float* out_weights) {
  __shared__ SelectShared sh;
  const Selection s = selection_of(c, blockIdx.x, weights, weights_len, budget, recent, index, out_weights);
  if (threadIdx.x == 0 && blockIdx.x % c.kv == 0) kept[blockIdx.x / c.kv] = s.keep;
  keep_latest(s, budget, threadIdx.x, kSelectThreads);
  if (s.room == 0 || s.room == s.old) return;
  const WaveRun run = wave_run(0, s.old, kSelectWaves);
  uint32_t held[kHeld];
  read_keys(s, run, run.begin, held);
  auto each = [&](auto work) {
#pragma unroll
    for (int a = 0; a < kHeld; ++a)
      if (run.begin + a * 64 < run.limit) work(run.begin + a * 64 + (int)(threadIdx.x & 63), held[a]);
  };
  Threshold t{0u, (uint32_t)s.room, 32, false};
#pragma clang loop unroll(disable)
  while (t.low > 0 && !t.settled) {
    histogram(sh, t, each);
    const int hi = kBins - 1 - 2 * (int)threadIdx.x;
    refine(sh, bin_count(sh, hi), bin_count(sh, hi - 1), t);
  }
  write_kept(sh, s, t, 0, 0, each);
}

// More tokens: the same by slices, a workgroup each, in four launches.  Launch
// kPass < 3 leaves the histogram of its slice's keys for the bits that the
// launches before settled, counts[pass][head][slice][bin]; the last one has
// from them how many tokens the slices before it keep, and writes.  Bound by the
// latency of four launches (50001 tokens of 32 heads: 8, 10, 10 and 11 us); one
// workgroup for a head took 52 us, instructions of 16 waves on one compute unit.
template <int kPass>
__global__ __launch_bounds__(kSelectThreads) void kv4_slice_kernel(Kv4View c, const float* weights,
                                                                   int64_t weights_len, int budget, int recent,
                                                                   int32_t* index, int32_t* kept, float* out_weights,
                                                                   uint32_t* counts, int slices) {
  __shared__ SelectShared sh;
  __shared__ uint32_t before[2];
  const uint32_t heads = c.seqs * c.kv, head = blockIdx.x / (uint32_t)slices, slice = blockIdx.x % (uint32_t)slices;
  const int tid = threadIdx.x;
  const Selection s = selection_of(c, head, weights, weights_len, budget, recent, index, out_weights);
  if (kPass == 0) {
    if (tid == 0 && slice == 0 && head % c.kv == 0) kept[head / c.kv] = s.keep;
    keep_latest(s, budget, (int)slice * kSelectThreads + tid, slices * kSelectThreads);
  }
  if (s.room == 0 || s.room == s.old) return;
  const int size = ((s.old + 63) / 64 + slices - 1) / slices * 64, begin = (int)slice * size;
  const WaveRun run = wave_run(begin, begin + size < s.old ? begin + size : (begin < s.old ? s.old : begin), kSelectWaves);
  auto each = [&](auto work) {
    for (int at = run.begin; at < run.limit; at += kHeld * 64) {
      uint32_t k[kHeld];
      read_keys(s, run, at, k);
#pragma unroll
      for (int a = 0; a < kHeld; ++a)
        if (at + a * 64 < run.limit) work(at + a * 64 + (tid & 63), k[a]);
    }
  };
  auto counts_of = [&](int pass, uint32_t sl) {
    return counts + (((int64_t)pass * heads + head) * slices + sl) * kBins;
  };
  const int hi = kBins - 1 - 2 * tid;
  // what the launch before knew, and from its histograms what this one does
  uint32_t* known = counts + (int64_t)3 * heads * slices * kBins + ((int64_t)head * slices + slice) * kState;
  Threshold t{0u, (uint32_t)s.room, 32, false};
  uint32_t kept_before = 0, ties_before = 0;  // by the slices before this one
  if constexpr (kPass > 0) {
    if constexpr (kPass > 1) t.prefix = known[0], t.need = known[1], t.low = (int)known[2], kept_before = known[3];
    t.settled = t.low < 0;
    if (!t.settled) {
      uint32_t h0 = 0, h1 = 0, b0 = 0, b1 = 0;
#pragma unroll 8
      for (uint32_t sl = 0; sl < (uint32_t)slices; ++sl) {
        const u32x2 two = *reinterpret_cast<const u32x2*>(counts_of(kPass - 1, sl) + hi - 1);
        h0 += two[1], h1 += two[0];
        if (sl < slice) b0 += two[1], b1 += two[0];
      }
      const int bin = (int)refine(sh, h0, h1, t);
      const int from = t.settled ? bin : bin + 1;  // bins that are kept whole
      uint32_t more = (hi >= from ? b0 : 0) + (hi - 1 >= from ? b1 : 0);
      uint32_t ties = kPass < 3 ? 0u : (hi == bin ? b0 : 0) + (hi - 1 == bin ? b1 : 0);
      if (tid < 2) before[tid] = 0;
      __syncthreads();
      for (int d = 1; d < 64; d *= 2) more += __shfl_xor(more, d), ties += __shfl_xor(ties, d);
      if ((tid & 63) == 0) atomicAdd(&before[0], more), atomicAdd(&before[1], ties);  // whole numbers: no order in them
      __syncthreads();
      kept_before += before[0], ties_before = before[1];
    }
    if (kPass < 3 && tid == 0)
      known[0] = t.prefix, known[1] = t.need, known[2] = t.settled ? (uint32_t)-1 : (uint32_t)t.low, known[3] = kept_before;
  }
  if constexpr (kPass < 3) {
    if (t.settled) return;
    histogram(sh, t, each);
    *reinterpret_cast<u32x2*>(counts_of(kPass, slice) + hi - 1) = u32x2{bin_count(sh, hi - 1), bin_count(sh, hi)};
  } else {
    write_kept(sh, s, t, kept_before, ties_before, each);
  }
}

// The kept tokens' rows into the other cache: D / 32 lanes a row of 16 bytes and
// a scale each, in both planes, kAhead rows of a thread on their way at a time.
// Bound by the memory's lines: kept rows are mostly single ones, 64 bytes of
// codes and 4 of scales (8192 of 50001 tokens of 32 heads: 71 MB in 20 us, with
// one row on its way as with four).
template <int D>
__global__ __launch_bounds__(256) void kv4_move_kernel(Kv4View c, Kv4View out, const int32_t* index, uint32_t budget,
                                                       uint32_t groups) {
  constexpr uint32_t kLanes = D / 32, kEach = 256 / kLanes;
  constexpr int kAhead = 4;
  const uint32_t head = blockIdx.x / groups, b = head / c.kv, h = head % c.kv, part = threadIdx.x % kLanes;
  const uint32_t first = blockIdx.x % groups * (kEach * kAhead) + threadIdx.x / kLanes;
  int t[kAhead];
  uint32_t from[kAhead], to[kAhead];
#pragma unroll
  for (int a = 0; a < kAhead; ++a) {
    const uint32_t j = first + a * kEach;
    t[a] = j < budget ? index[(uint64_t)head * budget + j] : -1;
    to[a] = j < budget ? kv4_page(out, b, j) : 0xFFFFFFFFu;
  }
#pragma unroll
  for (int a = 0; a < kAhead; ++a) from[a] = t[a] >= 0 ? kv4_page(c, b, (uint32_t)t[a]) : 0xFFFFFFFFu;
  u32x4 code[kAhead][2];
  uint8_t scale[kAhead][2];
#pragma unroll
  for (int a = 0; a < kAhead; ++a) {
    const uint64_t row = kv4_row(c, from[a], h, (uint32_t)t[a]);
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
      // a token without a page is kept as zeros
      const uint64_t s = (plane * c.plane_rows + row) * kLanes + part;
      code[a][plane] = ld_nt(reinterpret_cast<const u32x4*>(c.codes) + s);
      scale[a][plane] = c.scales[s];
      if (from[a] >= c.pages) code[a][plane] = u32x4{0u, 0u, 0u, 0u}, scale[a][plane] = 0;
    }
  }
#pragma unroll
  for (int a = 0; a < kAhead; ++a) {
    if (t[a] < 0 || to[a] >= out.pages) continue;
    const uint64_t row = kv4_row(out, to[a], h, first + a * kEach);
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
      const uint64_t d = (plane * out.plane_rows + row) * kLanes + part;
      reinterpret_cast<u32x4*>(out.codes)[d] = code[a][plane];
      out.scales[d] = scale[a][plane];
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

// Slices of a head's selection, 1 for one workgroup.
static int select_slices(const Kv4View& c, int64_t weights_len) {
  const int64_t most = weights_len < (int64_t)c.cap ? weights_len : (int64_t)c.cap;
  const int64_t slices = (most + kSlice - 1) / kSlice;
  return slices < 1 ? 1 : (slices > kMostSlices ? kMostSlices : (int)slices);
}

int64_t kv4_evict_workspace(const Kv4View& c, int64_t weights_len) {
  const int slices = select_slices(c, weights_len);
  return slices > 1 ? (int64_t)c.seqs * c.kv * slices * (3 * kBins + kState) * 4 : 0;
}

int kv4_evict(const Kv4View& c, int dim, const float* weights, int64_t weights_len, int budget, int recent,
              const Kv4View& out, int32_t* index, int32_t* kept, float* out_weights, void* ws, hipStream_t st) {
  if (c.seqs == 0) return kOk;
  const int slices = select_slices(c, weights_len);
  if (slices == 1) {
    hipLaunchKernelGGL(kv4_select_kernel, dim3(c.seqs * c.kv), dim3(kSelectThreads), 0, st, c, weights, weights_len,
                       budget, recent, index, kept, out_weights);
  } else {
    const dim3 grid(c.seqs * c.kv * (unsigned)slices);
#define VQX_KV4_SLICE(PASS)                                                                                          \
  hipLaunchKernelGGL((kv4_slice_kernel<PASS>), grid, dim3(kSelectThreads), 0, st, c, weights, weights_len, budget, \
                     recent, index, kept, out_weights, (uint32_t*)ws, slices)
    VQX_KV4_SLICE(0);
    VQX_KV4_SLICE(1);
    VQX_KV4_SLICE(2);
    VQX_KV4_SLICE(3);
#undef VQX_KV4_SLICE
  }
  int rc = check_launch("kv4_evict (selection)");
  if (rc != kOk) return rc;
  const uint32_t each = 4u * 256u / (uint32_t)(dim / 32), groups = ((uint32_t)budget + each - 1) / each;
  if ((uint64_t)c.seqs * c.kv * groups >= 1ull << 31)
    return set_error(kErrUnsupported, "kv4_evict: a budget of %d tokens for %u heads does not fit a launch", budget,
                     c.seqs * c.kv);
#define VQX_KV4_MOVE(D)                                                                                        \
  hipLaunchKernelGGL((kv4_move_kernel<D>), dim3(c.seqs * c.kv * groups), dim3(256), 0, st, c, out, index, \
                     (uint32_t)budget, groups)
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
