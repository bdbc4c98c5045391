// A token for each row of logits from a given random number.
//
// A token's weight is a whole number, w = 2^40 exp((x - largest) / temperature)
// rounded, so that sums of weights have no order: what a cut keeps and which
// token the random number falls on do not depend on how a row is shared out.
// (2^40 is 2^-41 off in the largest weight's units, and 2^22 of the largest
// weights sum to 2^62.)  Weights are computed in 64 bits, to some 2^-48.
//
// Order: a row's tokens from the largest logit down, equal ones by index, as
// whole numbers too: the logit's bits, turned so that smaller is larger, above
// the index.  A cut (k tokens, a share p of the weights) is the last of these
// numbers that is kept.
#include <type_traits>

#include "vqx_sampling.h"

namespace vqx {
namespace {

struct Bf16 {};
struct F16 {};

constexpr int kThreads = 1024, kWaves = kThreads / 64;
// Bins of a histogram of logits: kFine for each halving of the weight; tokens
// kHalvings and more below the largest have weight 0.
constexpr int kBins = 2048, kFine = 48, kHalvings = 42;
constexpr int kMostListed = 4096;  // tokens that are sorted in LDS
constexpr double kUnit = 0x1p40;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNone = -__builtin_huge_valf();

typedef unsigned long long u64;

// ---------------------------------------------------------------------------
// a row's logits, 8 at a time from aligned addresses
// ---------------------------------------------------------------------------
template <typename T>
struct Raw {
  u32x4 a;
};
template <>
struct Raw<float> {
  u32x4 a, b;
};
__device__ __forceinline__ float sound(float x) { return x == x ? x + 0.0f : kNone; }  // one zero, no NaN
__device__ __forceinline__ float value(uint32_t h, Bf16) { return u2f(h << 16); }
__device__ __forceinline__ float value(uint32_t h, F16) { return h2f_exact(h); }
__device__ __forceinline__ float element(const void* p, int64_t i, float) { return static_cast<const float*>(p)[i]; }
template <typename T>
__device__ __forceinline__ float element(const void* p, int64_t i, T) {
  return value(static_cast<const uint16_t*>(p)[i], T());
}
// 8 logits as they are; NaN and both zeros too
template <typename T>
__device__ __forceinline__ void values(const Raw<T>& r, float (&x)[8]) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = u2f(r.a[j]), x[j + 4] = u2f(r.b[j]);
  } else if constexpr (std::is_same<T, Bf16>::value) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[2 * j] = u2f(r.a[j] << 16), x[2 * j + 1] = u2f(r.a[j] & 0xFFFF0000u);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[2 * j] = value(r.a[j] & 0xFFFFu, T()), x[2 * j + 1] = value(r.a[j] >> 16, T());
  }
}

template <typename T>
struct Row {
  static constexpr int kSize = std::is_same<T, float>::value ? 4 : 2;
  const uint8_t* base;  // of vector 0, aligned
  int before;           // elements of vector 0 that are not the row's
  int size, vectors;
  int whole, past;  // vectors [whole, past) have 8 of the row's

  __device__ __forceinline__ Row(const void* p, int64_t offset, int n) {
    const uintptr_t at = (uintptr_t)p + (uintptr_t)offset * kSize;
    before = (int)(at & 15) / kSize;
    base = reinterpret_cast<const uint8_t*>(at) - before * kSize;
    size = n;
    vectors = (n + before + 7) / 8;
    whole = before > 0;
    past = (n + before) / 8;
  }
  __device__ __forceinline__ int first(int v) const { return 8 * v - before; }
  __device__ __forceinline__ Raw<T> raw(int v) const {
    const uint8_t* p = base + (int64_t)v * 8 * kSize;
    if constexpr (kSize == 4)
      return Raw<T>{reinterpret_cast<const u32x4*>(p)[0], reinterpret_cast<const u32x4*>(p)[1]};
    else
      return Raw<T>{reinterpret_cast<const u32x4*>(p)[0]};
  }
  // any vector: -inf where the row has no element
  __device__ __forceinline__ void load(int v, float (&x)[8]) const {
    const int e = first(v);
    if (e >= 0 && e + 8 <= size) {
      values(raw(v), x);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = e + j >= 0 && e + j < size ? element(base, 8 * (int64_t)v + j, T()) : kNone;
    }
  }
};

// ---------------------------------------------------------------------------
// weights and order
// ---------------------------------------------------------------------------
struct Scale {
  float top;      // the row's largest logit
  double inner;   // log2(e) / temperature
  float coarse;   // that, in bins
  const double* powers;  // 2^(j / 64) in LDS
};

__device__ __forceinline__ u64 weight(const Scale& s, float x) {
  if (x == s.top) return (u64)kUnit;
  const double q = ((double)x - (double)s.top) * s.inner;
  if (!(q > -41.5)) return 0;
  const double n = __builtin_rint(64.0 * q);
  const double r = __builtin_fma(n, -1.0 / 64.0, q);
  // 2^r to 2^-54: Taylor's series in r ln 2, up to 0.0054
  double p = 0x1.5d87fe78a6731p-10;                     // ln2^5 / 120
  p = __builtin_fma(p, r, 0x1.3b2ab6fba4e77p-7);        // ln2^4 / 24
  p = __builtin_fma(p, r, 0x1.c6b08d704a0c0p-5);        // ln2^3 / 6
  p = __builtin_fma(p, r, 0x1.ebfbdff82c58fp-3);        // ln2^2 / 2
  p = __builtin_fma(p, r, 0x1.62e42fefa39efp-1);        // ln2
  p = __builtin_fma(p, r, 1.0);
  const int i = (int)n;
  const double unit = __builtin_bit_cast(double, (u64)(1023 + 40 + (i >> 6)) << 52);
  // a number below 2^52 is rounded to a whole one by the addition
  return __builtin_bit_cast(u64, __builtin_fma(s.powers[i & 63] * p, unit, 0x1p52)) - __builtin_bit_cast(u64, 0x1p52);
}

// The bin of a logit, or kBins of one whose weight is 0; larger logits have no
// larger bins.
__device__ __forceinline__ int bin_of(const Scale& s, float x) {
  const float y = x == s.top ? 0.0f : (s.top - x) * s.coarse;
  return y < (float)(kHalvings * kFine) ? (int)y : kBins;
}

__device__ __forceinline__ u64 order(float x, int index) {
  const uint32_t b = f2u(x), up = b >> 31 ? ~b : b | 0x80000000u;
  return (u64)~up << 32 | (uint32_t)index;
}
__device__ __forceinline__ float logit_of(u64 o) {
  const uint32_t up = ~(uint32_t)(o >> 32);
  return u2f(up >> 31 ? up & 0x7FFFFFFFu : ~up);
}

// Which of `total` units of weight a random number falls on.
__device__ __forceinline__ u64 target_of(float u, u64 total) {
  const double at = __builtin_floor((double)u * (double)total);
  const u64 target = at > 0.0 ? (u64)at : 0;
  return target < total ? target : total - 1;
}

// ---------------------------------------------------------------------------
// a workgroup's sums
// ---------------------------------------------------------------------------
__device__ __forceinline__ u64 wave_scan(u64 x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const u64 y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}

struct Shared {
  u64 list[kMostListed];
  u64 mass[kBins];
  uint32_t count[kBins];
  double powers[64];
  float tops[kWaves];
  u64 sums[kWaves];
  u64 found[4];
  int at, listed;
};

// The sum of what the threads before this one have, and of all.
__device__ __forceinline__ u64 scan_before(Shared& s, u64 x, u64& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 upto = wave_scan(x);
  __syncthreads();
  if (lane == 63) s.sums[wave] = upto;
  __syncthreads();
  u64 before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? s.sums[w] : 0;
    all += s.sums[w];
  }
  return before + upto - x;
}
__device__ __forceinline__ u64 sum_of(Shared& s, u64 x) {
  u64 all;
  scan_before(s, x, all);
  return all;
}

// Where a cut falls: everything before the bin is kept, `count` tokens with
// `mass`, and the cut is in the bin.
struct Cut {
  int bin;  // kBins: there is none, everything is kept
  u64 count, mass;
};

// The bin in which the first `most` tokens end, or (kShare) the first with which
// the masses come to `share`; base: what is before the first bin.  Of the other
// of the two sums a caller that counts may want to know too (kBoth).
template <bool kShare, bool kBoth = false>
__device__ __forceinline__ Cut find_bin(Shared& s, const Cut& base, u64 most, double share) {
  const int b = 2 * (int)threadIdx.x;
  static_assert(2 * kThreads == kBins, "");
  u64 all, count[2] = {0, 0}, mass[2] = {0, 0}, before = base.count, sum = base.mass;
  if (threadIdx.x == 0) s.at = kBins;
  if (!kShare || kBoth) {
    count[0] = s.count[b], count[1] = s.count[b + 1];
    before += scan_before(s, count[0] + count[1], all);
  }
  if (kShare || kBoth) {
    mass[0] = s.mass[b], mass[1] = s.mass[b + 1];
    sum += scan_before(s, mass[0] + mass[1], all);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool here = kShare ? (double)sum < share && (double)(sum + mass[i]) >= share
                             : before < most && before + count[i] >= most;
    if (here) s.at = b + i, s.found[0] = before, s.found[1] = sum;
    before += count[i], sum += mass[i];
  }
  __syncthreads();
  const Cut c = {s.at, s.found[0], s.found[1]};
  __syncthreads();
  return c;
}

__device__ __forceinline__ void clear_bins(Shared& s) {
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kThreads) s.count[i] = 0, s.mass[i] = 0;
  __syncthreads();
}

// A row's logits, 8 to a call: what(logits, the first one's index).  Four loads
// are on their way before the first is used.
template <typename T, typename What>
__device__ __forceinline__ void each_vector(const Row<T>& row, What what) {
  constexpr int kAhead = 4;
  for (int v = row.whole + (int)threadIdx.x; v < row.past; v += kAhead * kThreads) {
    Raw<T> r[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) r[a] = row.raw(v + a * kThreads < row.past ? v + a * kThreads : v);
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (v + a * kThreads >= row.past) break;
      float x[8];
      values(r[a], x);
      what(x, row.first(v + a * kThreads));
    }
  }
  // the first and the last, where they are parts of one
  const int part = threadIdx.x == 0 && row.whole > 0 ? 0 : (threadIdx.x == 64 && row.past >= row.whole ? row.past : -1);
  if (part >= 0 && part < row.vectors) {
    float x[8];
    row.load(part, x);
    what(x, row.first(part));
  }
}
template <typename T, typename What>
__device__ __forceinline__ void each_token(const Row<T>& row, What what) {
  each_vector(row, [&](const float(&x)[8], int e) {
#pragma unroll
    for (int j = 0; j < 8; ++j) what(sound(x[j]), e + j);
  });
}

// The listed orders sorted, padded to a power of two with the largest.
__device__ __forceinline__ int sort_list(Shared& s, int n) {
  int size = 64;
  while (size < n) size *= 2;
  for (int i = n + (int)threadIdx.x; i < size; i += kThreads) s.list[i] = ~0ull;
  __syncthreads();
  for (int k = 2; k <= size; k *= 2)
    for (int d = k / 2; d > 0; d /= 2) {
      for (int i = threadIdx.x; i < size / 2; i += kThreads) {
        const int a = 2 * i - (i & (d - 1)), b = a + d;
        const u64 x = s.list[a], y = s.list[b];
        if ((x > y) == ((a & k) == 0)) s.list[a] = y, s.list[b] = x;
      }
      __syncthreads();
    }
  return size;
}

// The last token that a cut in a bin keeps: the `most`-th of all, or the first
// with which the masses come to `share`; the mass up to it.  Where the bin has
// too many tokens to sort it is cut into finer ones by their order, again and
// again: an order's 64 bits end after six times.
template <bool kShare, typename T>
__device__ u64 resolve(Shared& s, const Row<T>& row, const Scale& scale, Cut cut, u64 most, double share, u64& upto) {
  u64 lo = 0, hi = ~0ull;
  uint32_t n = s.count[cut.bin];
  for (int level = 0; level < 6 && n > (uint32_t)kMostListed; ++level) {
    // the range that the tokens have
    u64 least = ~0ull, greatest = 0;
    each_token(row, [&](float x, int i) {
      const u64 o = order(x, i);
      if (bin_of(scale, x) == cut.bin && o >= lo && o <= hi) {
        least = o < least ? o : least;
        greatest = o > greatest ? o : greatest;
      }
    });
    __syncthreads();
    if (threadIdx.x == 0) s.found[2] = ~0ull, s.found[3] = 0;
    __syncthreads();
    atomicMin(&s.found[2], least);
    atomicMax(&s.found[3], greatest);
    __syncthreads();
    lo = s.found[2], hi = s.found[3];
    const int bits = 64 - __builtin_clzll(hi - lo), shift = bits > 11 ? bits - 11 : 0;
    clear_bins(s);
    each_token(row, [&](float x, int i) {
      const u64 o = order(x, i);
      if (bin_of(scale, x) == cut.bin && o >= lo && o <= hi) {
        const int b = (int)((o - lo) >> shift);
        atomicAdd(&s.count[b], 1u);
        atomicAdd(&s.mass[b], weight(scale, x));
      }
    });
    __syncthreads();
    const Cut finer = find_bin<kShare, true>(s, cut, most, share);
    n = s.count[finer.bin & (kBins - 1)];
    lo += (u64)finer.bin << shift;
    const u64 last = lo + ((1ull << shift) - 1);
    hi = last < hi ? last : hi;
    cut.count = finer.count, cut.mass = finer.mass;
  }
  __syncthreads();
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
  each_token(row, [&](float x, int i) {
    const u64 o = order(x, i);
    if (bin_of(scale, x) == cut.bin && o >= lo && o <= hi) {
      const int at = atomicAdd(&s.listed, 1);
      if (at < kMostListed) s.list[at] = o;
    }
  });
  __syncthreads();
  n = s.listed < kMostListed ? s.listed : kMostListed;
  sort_list(s, (int)n);
  // masses before each of the sorted: four to a thread
  u64 w[4], mine = 0, all;
  const int first = 4 * (int)threadIdx.x;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    w[j] = first + j < (int)n ? weight(scale, logit_of(s.list[first + j])) : 0;
    mine += w[j];
  }
  u64 before = cut.mass + scan_before(s, mine, all);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const u64 rank = cut.count + (u64)(first + j);
    const bool last = kShare ? (double)before < share && !((double)(before + w[j]) < share) : rank + 1 == most;
    if (first + j < (int)n && last) s.found[0] = s.list[first + j], s.found[1] = before + w[j];
    before += w[j];
  }
  __syncthreads();
  const u64 o = s.found[0];
  upto = s.found[1];
  __syncthreads();
  return o;
}

// The tokens of a bin that the listed ones are in, of those up to `cut`, gathered
// behind each other: order and weight.  Their number, or more than kMostNear.
constexpr int kEach = kMostListed / kThreads;
constexpr int kMostNear = 512;

template <typename In>
__device__ __forceinline__ int gather_near(Shared& s, const u64 (&o)[kEach], const u64 (&w)[kEach], In in) {
  __syncthreads();
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (in(j)) {
      const int at = atomicAdd(&s.listed, 1);
      if (at < kMostNear) s.list[2 * at] = o[j], s.list[2 * at + 1] = w[j];
    }
  __syncthreads();
  return s.listed;
}

// The token drawn where all that can be kept lies in bins up to `last` and those
// have few tokens: they are listed, and what is left is about the list.  most:
// tokens kept by count, which end in bin `at`, 0 for all; mass: what a share is of,
// where it is not of the first `most`.
enum Few { kDrawn, kTooMany, kTooNear };  // kTooNear: and the masses of the bins are gone
template <typename T>
__device__ Few few(Shared& s, const Row<T>& row, const Scale& scale, const Sampling& p, int64_t r, int last, u64 most,
                   const Cut& at, bool by_share, float share, u64 mass, double bar) {
  uint32_t n = 0;
  for (int b = threadIdx.x; b <= last; b += kThreads) n += s.count[b];
  const u64 all = sum_of(s, n);
  if (all > (u64)kMostListed) return kTooMany;
  __syncthreads();
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
  each_vector(row, [&](const float(&x)[8], int e) {
    bool any = false;
    int b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = bin_of(scale, x[j]), any |= b[j] <= last;
    if (!any) return;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (b[j] <= last) {
        const int at = atomicAdd(&s.listed, 1);
        if (at < kMostListed) s.list[at] = order(sound(x[j]), e + j);
      }
  });
  __syncthreads();
  const int listed = s.listed < kMostListed ? s.listed : kMostListed;
  u64 o[kEach], w[kEach];
  int bin[kEach];
  bool keeps[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = j * kThreads + (int)threadIdx.x;
    keeps[j] = i < listed;
    o[j] = keeps[j] ? s.list[i] : ~0ull;
    const float x = logit_of(o[j]);
    w[j] = keeps[j] ? weight(scale, x) : 0;
    bin[j] = keeps[j] ? bin_of(scale, x) : kBins;
  }
  const Cut none = {kBins, 0, 0};
  if (most > 0 && at.bin < kBins) {
    const int near = gather_near(s, o, w, [&](int j) { return bin[j] == at.bin; });
    if (near > kMostNear) return kTooNear;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      if (bin[j] != at.bin) {
        keeps[j] = keeps[j] && bin[j] < at.bin;
        continue;
      }
      u64 rank = at.count;
      for (int i = 0; i < near; ++i) rank += s.list[2 * i] < o[j];
      keeps[j] = rank < most;
    }
  }
  if (by_share) {
    // the masses of the bins, and of all where it is of the first `most`
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.mass[i] = 0;
    __syncthreads();
    u64 mine = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (keeps[j]) atomicAdd(&s.mass[bin[j]], w[j]), mine += w[j];
    if (most > 0) mass = sum_of(s, mine);
    __syncthreads();
    const double wanted = share > 0.0f ? (double)share * (double)mass : 0.5;
    const Cut c = find_bin<true>(s, none, 0, wanted);
    if (c.bin < kBins) {
      const int near = gather_near(s, o, w, [&](int j) { return keeps[j] && bin[j] == c.bin; });
      if (near > kMostNear) return kTooNear;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        if (!keeps[j] || bin[j] != c.bin) {
          keeps[j] = keeps[j] && bin[j] < c.bin;
          continue;
        }
        u64 before = c.mass;
        for (int i = 0; i < near; ++i) before += s.list[2 * i] < o[j] ? s.list[2 * i + 1] : 0;
        keeps[j] = (double)before < wanted;
      }
    }
  }
  // the kept ones by their index: bins of as many indexes, and in the bin where
  // the random number falls one by one
  const int shift = 32 - __builtin_clz((unsigned)(p.vocab - 1) | (kBins - 1)) - 11;
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kThreads) s.mass[i] = 0;
  __syncthreads();
  u64 mine = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    keeps[j] = keeps[j] && w[j] > 0 && (double)w[j] >= bar;
    if (keeps[j]) atomicAdd(&s.mass[(uint32_t)o[j] >> shift], w[j]), mine += w[j];
  }
  const u64 total = sum_of(s, mine), target = target_of(p.random[r], total);
  const int b0 = 2 * (int)threadIdx.x;
  u64 sum;
  const u64 m0 = s.mass[b0], m1 = s.mass[b0 + 1], before = scan_before(s, m0 + m1, sum);
  if (target >= before && target < before + m0 + m1) {
    const bool second = target >= before + m0;
    s.at = b0 + second, s.found[0] = second ? before + m0 : before;
  }
  __syncthreads();
  const int run = s.at;
  const u64 rest = target - s.found[0];
  const int near = gather_near(s, o, w, [&](int j) { return keeps[j] && (int)((uint32_t)o[j] >> shift) == run; });
  if (near > kMostNear) return kTooNear;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    if (!keeps[j] || (int)((uint32_t)o[j] >> shift) != run) continue;
    u64 upto = 0;
    for (int i = 0; i < near; ++i) upto += (uint32_t)s.list[2 * i] < (uint32_t)o[j] ? s.list[2 * i + 1] : 0;
    if (rest >= upto && rest < upto + w[j]) {
      p.tokens[r] = (int64_t)(uint32_t)o[j];
      p.chances[r] = (float)log((double)w[j] / (double)total);
    }
  }
  return kDrawn;
}

// ---------------------------------------------------------------------------
// a row
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(Sampling p) {
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r = blockIdx.x;
  const Row<T> row(p.logits, r * p.stride, p.vocab);
  if (tid < 64) s.powers[tid] = exp2((double)tid / 64.0);

  float top = kNone;
  each_vector(row, [&](const float(&x)[8], int) {
#pragma unroll
    for (int j = 0; j < 8; ++j) top = __builtin_fmaxf(top, x[j]);  // a NaN is no maximum
  });
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = __builtin_fmaxf(top, __shfl_xor(top, d));
  if (lane == 0) s.tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = __builtin_fmaxf(top, s.tops[w]);
  top += 0.0f;
  const float t = p.temperature ? p.temperature[r] : 1.0f;
  if (top == kNone || !(t > 0.0f)) {
    // the first that is the largest
    int at = p.vocab;
    if (top != kNone)
      each_vector(row, [&](const float(&x)[8], int e) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (x[j] == top && e + j < at) at = e + j;
      });
    if (tid == 0) s.at = p.vocab;
    __syncthreads();
    if (at < p.vocab) atomicMin(&s.at, at);
    __syncthreads();
    if (tid == 0) {
      p.tokens[r] = top == kNone ? -1 : s.at;
      p.chances[r] = top == kNone ? kNone : 0.0f;
    }
    return;
  }
  Scale scale;
  scale.top = top;
  scale.inner = 1.44269504088896340736 / (double)t;
  const double coarse = scale.inner * kFine;
  scale.coarse = coarse < 1e30 ? (float)coarse : 1e30f;
  scale.powers = s.powers;

  const int k = p.top_k ? p.top_k[r] : 0;
  const float share = p.top_p ? p.top_p[r] : 1.0f, least = p.min_p ? p.min_p[r] : 0.0f;
  const bool by_count = k > 0 && k < p.vocab, by_share = share < 1.0f;
  const double bar = least > 0.0f ? (least < 1.0f ? (double)least * kUnit : kUnit) : 0.0;
  u64 cut = ~0ull;
  if (by_count || by_share || bar > 0.0) {
    const Cut none = {kBins, 0, 0};
    Cut at = none;
    u64 mass = 0;
    // of the bins' masses none is needed where the first k tokens, or those above
    // a share of the largest, are few
    auto count_bins = [&](auto with_masses) {
      clear_bins(s);
      each_vector(row, [&](const float(&x)[8], int) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int b = bin_of(scale, x[j]);
          if (b < kBins) {
            atomicAdd(&s.count[b], 1u);
            if (decltype(with_masses)::value) atomicAdd(&s.mass[b], weight(scale, sound(x[j])));
          }
        }
      });
      __syncthreads();
    };
    bool masses = by_share && !by_count;
    if (masses) {
      count_bins(std::true_type());
      for (int i = tid; i < kBins; i += kThreads) mass += s.mass[i];
      mass = sum_of(s, mass);
    } else {
      count_bins(std::false_type());
    }
    if (by_count) at = find_bin<false>(s, none, (u64)k, 0.0);
    // no share at all is the first token's
    auto wanted = [&] { return share > 0.0f ? (double)share * (double)mass : 0.5; };
    // the last bin that a kept token can be in
    int last = kBins - 1;
    if (by_count && at.bin < last) last = at.bin;
    if (masses) {
      const Cut by = find_bin<true>(s, none, 0, wanted());
      if (by.bin < last) last = by.bin;
    }
    if (bar > 0.0 && (!by_share || masses)) {
      const double y = (40.0 - log2(bar)) * kFine + 1.0;  // one more for the rounding of a bin
      if (y < (double)last) last = (int)y;
    }
    const Few done = few(s, row, scale, p, r, last, by_count ? (u64)k : 0, at, by_share, share, mass, bar);
    if (done == kDrawn) return;
    if (by_count) {
      if (by_share) {
        count_bins(std::true_type());
        for (int i = tid; i < kBins; i += kThreads) mass += s.mass[i];
        mass = sum_of(s, mass);
        at = find_bin<false, true>(s, none, (u64)k, 0.0);
      }
      if (at.bin < kBins) {
        // the histogram is made again by a bin that is cut finer
        const bool keeps = s.count[at.bin] <= (uint32_t)kMostListed;
        cut = resolve<false>(s, row, scale, at, (u64)k, 0.0, mass);
        if (by_share && !keeps) count_bins(std::true_type());
      }
    } else if (masses && done == kTooNear) {
      count_bins(std::true_type());
    }
    if (by_share) {
      const Cut by = find_bin<true>(s, none, 0, wanted());
      if (by.bin < kBins) {
        u64 upto;
        const u64 o = resolve<true>(s, row, scale, by, 0, wanted(), upto);
        cut = o < cut ? o : cut;
      }
    }
  }
  auto kept = [&](float x, int i) -> u64 {
    if (order(x, i) > cut) return 0;
    const u64 w = weight(scale, x);
    return (double)w >= bar ? w : 0;
  };
  // which run of vectors, then which of a wave's, then which token: the runs of
  // the waves, then one of them shared out again
  int from = 0, to = row.vectors;
  u64 total = 0, target = 0;
  while (true) {
    const int each = (to - from + kWaves - 1) / kWaves, begin = from + wave * each;
    const int end = begin + each < to ? begin + each : to;
    u64 mine = 0, upto = 0;
    for (int v = begin + lane; v < end; v += 64) {
      float x[8];
      row.load(v, x);
      const int e = row.first(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) mine += kept(sound(x[j]), e + j);
    }
    upto = wave_scan(mine);
    __syncthreads();
    if (lane == 63) s.sums[wave] = upto;
    __syncthreads();
    u64 before = 0, all = 0;
    int run = 0;
    if (total == 0) {
      for (int w = 0; w < kWaves; ++w) total += s.sums[w];
      target = target_of(p.random[r], total);
    }
    for (int w = 0; w < kWaves; ++w) {
      if (all + s.sums[w] > target) break;
      all += s.sums[w];
      run = w + 1;
    }
    target -= all;
    from += run * each;
    to = from + each < to ? from + each : to;
    if (each > 64) continue;
    // one vector a lane: the lane, then the token
    if (wave != run) return;
    before = upto - mine;
    if (target >= before && target < upto) {
      const int v = begin + lane;
      float x[8];
      row.load(v, x);
      const int e = row.first(v);
      u64 left = target - before, weighs = 0;
      int token = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const u64 w = kept(sound(x[j]), e + j);
        if (weighs == 0) {
          if (left < w) weighs = w, token = e + j;
          left -= w;
        }
      }
      p.tokens[r] = token;
      p.chances[r] = (float)log((double)weighs / (double)total);
    }
    return;
  }
}

}  // namespace

int sample(const Sampling& p, int dtype, hipStream_t st) {
  if (p.rows == 0) return kOk;
  const dim3 grid((unsigned)p.rows);
  if (dtype == kF32)
    hipLaunchKernelGGL((sample_kernel<float>), grid, dim3(kThreads), 0, st, p);
  else if (dtype == kBF16)
    hipLaunchKernelGGL((sample_kernel<Bf16>), grid, dim3(kThreads), 0, st, p);
  else
    hipLaunchKernelGGL((sample_kernel<F16>), grid, dim3(kThreads), 0, st, p);
  return check_launch("sample_tokens");
}

}  // namespace vqx
