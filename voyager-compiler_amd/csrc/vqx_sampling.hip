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
//
// A row is one workgroup's, of 256 to 1024 threads: they hold it in registers, so
// that it is read once, and everything after its largest logit is about the tokens
// that a cut can keep.  Which those are is known from the threads' own largest
// logits (the k-th of them bounds the k-th of all), from min_p, or from a
// histogram of the logits; up to four a thread are listed in LDS, and the cuts and
// the drawing are about the list.  More than that, or no cut, is a pass of
// weights in 64 bits over the row.  256 rows of 131072 bf16 logits (67 MB, which a
// copy's rate would read in 13 us), from a graph: top 50 25 us, top 1000 31, top
// 1000 with top_p and min_p 37; 50 us with min_p alone, 56 without cuts (weights:
// some 15 fp64 instructions a logit), 106 with the top 20000, 149 with a top_p
// that keeps thousands (histograms of masses, and cuts resolved one by one).  One
// row of 32000, top 50: 10.4 us, a chain of some 20 barriers; of 1000 7.5.
#include <type_traits>

#include "vqx_sampling.h"

namespace vqx {
namespace {

struct Bf16 {};
struct F16 {};

// Bins for each 42 halvings of the weight: tokens so far below the largest have
// weight 0.
constexpr int kHalvings = 42;
constexpr double kUnit = 0x1p40;
constexpr float kNone = -__builtin_huge_valf();

typedef unsigned long long u64;

// of a lambda: what it takes stays in registers
#define VQX_INLINE __attribute__((always_inline))

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
  bool head;        // vector 0 has fewer, and so has
  int tail;         // this one, -1: none
  bool infinite;    // where some are +inf those count as 0 and all others as -inf

  __device__ __forceinline__ Row(const void* p, int64_t offset, int n) {
    const uint8_t* at = static_cast<const uint8_t*>(p) + offset * kSize;
    before = (int)((uintptr_t)at & 15) / kSize;
    base = at - before * kSize;
    size = n;
    vectors = (n + before + 7) / 8;
    whole = before > 0;
    past = (n + before) / 8;
    head = before > 0;
    tail = past >= whole && past < vectors ? past : -1;
    infinite = false;
  }
  __device__ __forceinline__ int runs() const { return past > whole ? (past - whole + 63) / 64 : 0; }
  // The g-th of `parts` of the row: as many runs of 64 vectors each.
  __device__ __forceinline__ Row part(int g, int parts) const {
    Row r = *this;
    const int each = (runs() + parts - 1) / parts * 64, begin = whole + g * each;
    r.whole = begin < past ? begin : past;
    r.past = begin + each < past ? begin + each : past;
    if (r.past < r.whole) r.past = r.whole;
    if (g > 0) r.head = false;
    if (g + 1 < parts) r.tail = -1;
    return r;
  }

  __device__ __forceinline__ int first(int v) const { return 8 * v - before; }
  __device__ __forceinline__ Raw<T> raw(int v) const {
    const uint8_t* p = base + (int64_t)v * 8 * kSize;
    if constexpr (kSize == 4)
      return Raw<T>{reinterpret_cast<const u32x4*>(p)[0], reinterpret_cast<const u32x4*>(p)[1]};
    else
      return Raw<T>{reinterpret_cast<const u32x4*>(p)[0]};
  }
  // NaN and both zeros as they are
  __device__ __forceinline__ void logits(const Raw<T>& r, float (&x)[8]) const {
    values(r, x);
    if (infinite) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = x[j] == -kNone ? 0.0f : kNone;
    }
  }
  __device__ __forceinline__ float logit(int i) const {
    const float x = element(base, (int64_t)i + before, T());
    return !infinite ? x : (x == -kNone ? 0.0f : kNone);
  }
  // any vector: -inf where the row has no element
  __device__ __forceinline__ void load(int v, float (&x)[8]) const {
    const int e = first(v);
    if (e >= 0 && e + 8 <= size) {
      logits(raw(v), x);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = e + j >= 0 && e + j < size ? logit(e + j) : kNone;
    }
  }
};

// What a workgroup of kThreads does.
template <int kThreads>
struct Sampler {
  static constexpr int kWaves = kThreads / 64;
  // Bins of a histogram of logits: kFine for each halving of the weight.
  static constexpr int kBins = 2 * kThreads, kBinBits = kThreads == 1024 ? 11 : (kThreads == 512 ? 10 : 9);
  static constexpr int kFine = 12 * kThreads / 256;
  static constexpr int kMostListed = 4 * kThreads;  // tokens that are sorted in LDS
  static_assert(kBins == 1 << kBinBits && kHalvings * kFine <= kBins, "");

  // ---------------------------------------------------------------------------
  // weights and order
  // ---------------------------------------------------------------------------
  struct Shared {
    u64 list[kMostListed];
    u64 mass[kBins];
    uint32_t count[kBins];
    double powers[64];
    float tops[kWaves];
    u64 sums[4][kWaves];
    u64 found[4];
    int at, listed, spot[3], near[3];
  };

  struct Scale {
    float top;     // the row's largest logit
    double inner;  // 64 log2(e) / temperature
    // log2(e) / temperature, in bins, as three factors: halves of logits where the
    // temperature is 1 and more, whose difference is no infinity, and two of the
    // rest, which is past 32 bits for the smallest temperatures
    float half, half_top, bins[2];
    __device__ __forceinline__ float bin(float x) const { return __builtin_fmaf(-half, x, half_top) * bins[0] * bins[1]; }
    __device__ __forceinline__ float span(int count) const { return (float)count / bins[0] / bins[1] / half; }  // of so many bins
  };

  // A whole number up to 2^40, as a double: sums of them are exact up to 2^53.
  static __device__ __forceinline__ double weight(const Shared& s, const Scale& scale, float x) {
    // 64ths of a halving; 42 of these are 0 already, a NaN or -inf is one of those
    const double q = __builtin_fmax(((double)x - (double)scale.top) * scale.inner, -64.0 * kHalvings);
    // a number below 2^51 is rounded to a whole one by the addition, which stands
    // in the sum's low bits
    const double n = q + 0x1.8p52;
    const int i = (int)(uint32_t)__builtin_bit_cast(u64, n);
    const double r = q - (n - 0x1.8p52);
    // 2^(r / 64) to 2^-54: Taylor's series in r ln2 / 64, up to 0.0054
    double p = __builtin_fma(0x1.5d87fe78a6731p-40, r, 0x1.3b2ab6fba4e77p-31);  // (ln2 / 64)^5 / 120, (ln2 / 64)^4 / 24
    p = __builtin_fma(p, r, 0x1.c6b08d704a0c0p-23);                             // (ln2 / 64)^3 / 6
    p = __builtin_fma(p, r, 0x1.ebfbdff82c58fp-15);                             // (ln2 / 64)^2 / 2
    p = __builtin_fma(p, r, 0x1.62e42fefa39efp-7);                              // ln2 / 64
    p = __builtin_fma(p, r, 1.0);
    // times 2^((i % 64) / 64) 2^(i / 64) 2^40, rounded to a whole number
    const u64 power = __builtin_bit_cast(u64, s.powers[i & 63]) + ((u64)(uint32_t)(((i >> 6) + 40) << 20) << 32);
    return __builtin_fma(__builtin_bit_cast(double, power), p, 0x1p52) - 0x1p52;
  }
  static __device__ __forceinline__ u64 whole_weight(const Shared& s, const Scale& scale, float x) {
    return (u64)weight(s, scale, x);
  }

  // The bin of a logit, or kBins of one whose weight is 0; larger logits have no
  // larger bins.
  static __device__ __forceinline__ int bin_of(const Scale& s, float x) {
    const float y = s.bin(x);
    return y < (float)(kHalvings * kFine) ? (int)y : kBins;
  }

  static __device__ __forceinline__ u64 order(float x, int index) {
    const uint32_t b = f2u(x), up = b >> 31 ? ~b : b | 0x80000000u;
    return (u64)~up << 32 | (uint32_t)index;
  }
  static __device__ __forceinline__ float logit_of(u64 o) {
    const uint32_t up = ~(uint32_t)(o >> 32);
    return u2f(up >> 31 ? up & 0x7FFFFFFFu : ~up);
  }

  // Which of `total` units of weight a random number falls on.
  static __device__ __forceinline__ u64 target_of(float u, u64 total) {
    const double at = __builtin_floor((double)u * (double)total);
    const u64 target = at > 0.0 ? (u64)at : 0;
    return target < total ? target : total - 1;
  }

  // ---------------------------------------------------------------------------
  // a workgroup's sums
  // ---------------------------------------------------------------------------
  // The sum of what the threads before this one have, and of all.  Callers that
  // follow each other without a barrier have slots of their own and no fence.
  template <int kSlot = 0, bool kFence = true>
  static __device__ __forceinline__ u64 scan_before(Shared& s, u64 x, u64& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u64 upto = wave_scan(x);
    if (kFence) __syncthreads();
    if (lane == 63) s.sums[kSlot][wave] = upto;
    __syncthreads();
    // every row of 16 lanes has the waves' sums, summed up to each
    u64 sum = (lane & 15) < kWaves ? s.sums[kSlot][lane & 15] : 0;
    sum += from_lane<0x111, 0xF>(sum);
    sum += from_lane<0x112, 0xF>(sum);
    sum += from_lane<0x114, 0xF>(sum);
    sum += from_lane<0x118, 0xF>(sum);
    const int w = __builtin_amdgcn_readfirstlane(wave);
    const u64 before = w > 0 ? lane_of(sum, w - 1) : 0;
    all = lane_of(sum, kWaves - 1);
    return before + upto - x;
  }
  static __device__ __forceinline__ u64 sum_of(Shared& s, u64 x) {
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
  static __device__ __forceinline__ Cut find_bin(Shared& s, const Cut& base, u64 most, double share) {
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

  // What a share is of all: the weight that kept tokens have before them is below
  // it (no share at all is the first token's).
  static __device__ __forceinline__ double share_of(float share, u64 all) {
    return share > 0.0f ? (double)share * (double)all : 0.5;
  }

  // The first bin that is certainly not before the one in which the masses come to
  // `share` of `mass`, from counts: what lies behind it, each token of bin b with no
  // more than the weight of the bin's beginning, is not more than the rest.
  static __device__ __forceinline__ Cut find_least(Shared& s, double share, u64 mass) {
    const int b = 2 * (int)threadIdx.x;
    const uint32_t c0 = s.count[b], c1 = s.count[b + 1];
    // and what a bin's border, a weight's rounding and this power may be off by
    auto at_most = [](int bin) {
      return (u64)(0x1p40f * __builtin_amdgcn_exp2f(-(float)bin / kFine) * (1.0f + 0x1p-16f)) + 2;
    };
    const u64 m0 = c0 * at_most(b), m1 = c1 * at_most(b + 1);
    const double rest = (double)mass - share;
    u64 all, bound;
    u64 before = scan_before(s, c0 + c1, all);
    u64 behind = scan_before(s, m0 + m1, bound);
    behind = bound - behind;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const u64 m = i ? m1 : m0;
      if ((double)(behind - m) <= rest && (double)behind > rest) s.at = b + i, s.found[0] = before;
      before += i ? c1 : c0, behind -= m;
    }
    __syncthreads();
    const Cut c = {s.at, s.found[0], 0};
    __syncthreads();
    return c;
  }

  static __device__ __forceinline__ void clear_bins(Shared& s) {
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.count[i] = 0, s.mass[i] = 0;
    __syncthreads();
  }

  // A row's first vectors, held in 64 registers of each thread, so that a row of
  // 131072 two-byte logits is read once (256 such rows read a second time, from
  // beyond the L2s, take 13 us).
  template <typename T>
  struct Held {
    static constexpr int kVectors = std::is_same<T, float>::value ? 8 : 16;
    Raw<T> r[kVectors];

    __device__ __forceinline__ void load(const Row<T>& row) {
      const int v0 = row.whole + (int)threadIdx.x;
#pragma unroll
      for (int a = 0; a < kVectors; ++a) {
        if (row.whole + a * kThreads >= row.past) break;
        r[a] = row.raw(v0 + a * kThreads < row.past ? v0 + a * kThreads : row.past - 1);
      }
    }
  };

  // A row's whole vectors from the begin-th of each thread on, what(raw, the first
  // element's index); four loads are on their way before the first is used.
  template <typename T, typename What>
  static __device__ __forceinline__ void each_raw(const Row<T>& row, What what, int begin = 0) {
    constexpr int kAhead = 4;
    for (int v = row.whole + begin * kThreads + (int)threadIdx.x; v < row.past; v += kAhead * kThreads) {
      Raw<T> r[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) r[a] = row.raw(v + a * kThreads < row.past ? v + a * kThreads : v);
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        if (v + a * kThreads >= row.past) break;
        what(r[a], row.first(v + a * kThreads));
      }
    }
  }
  struct NotHeld {};  // four loads ahead
  struct OneAhead {};  // one: for much work on each, whose code is there once (unrolled it is fetched for one pass only)
  template <typename T, typename What>
  static __device__ __forceinline__ void each_raw(const Row<T>& row, OneAhead, What what) {
    int v = row.whole + (int)threadIdx.x;
    if (v >= row.past) return;
    Raw<T> next = row.raw(v);
#pragma clang loop unroll(disable)
    for (; v < row.past; v += kThreads) {
      const Raw<T> r = next;
      next = row.raw(v + kThreads < row.past ? v + kThreads : v);
      what(r, row.first(v));
    }
  }
  template <typename H>
  static constexpr int held_vectors() {
    if constexpr (std::is_same<H, NotHeld>::value || std::is_same<H, OneAhead>::value)
      return 0;
    else
      return H::kVectors;
  }
  template <typename T, typename What>
  static __device__ __forceinline__ void each_raw(const Row<T>& row, NotHeld, What what) {
    each_raw(row, what);
  }
  template <typename T, typename What>
  static __device__ __forceinline__ void each_raw(const Row<T>& row, const Held<T>& held, What what) {
    const int v0 = row.whole + (int)threadIdx.x;
#pragma unroll
    for (int a = 0; a < Held<T>::kVectors; ++a) {
      if (row.whole + a * kThreads >= row.past) break;
      if (v0 + a * kThreads < row.past) what(held.r[a], row.first(v0 + a * kThreads));
    }
    each_raw(row, what, Held<T>::kVectors);
  }
  // A row's logits, 8 to a call: what(logits, the first one's index).
  template <typename T, typename What, typename H = NotHeld>
  static __device__ __forceinline__ void each_vector(const Row<T>& row, What what, const H& held = H()) {
    auto one = [&](const Raw<T>& r, int e) VQX_INLINE {
      float x[8];
      row.logits(r, x);
      what(x, e);
    };
    each_raw(row, held, one);
    // the first and the last, where they are parts of one
    const int part = threadIdx.x == 0 && row.head ? 0 : (threadIdx.x == 64 ? row.tail : -1);
    if (part >= 0) {
      float x[8];
      row.load(part, x);
      what(x, row.first(part));
    }
  }
  template <typename T, typename What>
  static __device__ __forceinline__ void each_token(const Row<T>& row, What what) {
    each_vector(row, [&](const float(&x)[8], int e) VQX_INLINE {
#pragma unroll
      for (int j = 0; j < 8; ++j) what(sound(x[j]), e + j);
    }, OneAhead());
  }

  // The listed orders sorted, padded to a power of two with the largest.
  static __device__ __forceinline__ int sort_list(Shared& s, int n) {
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
  // again, until an order's 64 bits end.
  template <bool kShare, typename T>
  static __device__ __forceinline__ u64 resolve(Shared& s, const Row<T>& row, const Scale& scale, Cut cut, u64 most, double share, u64& upto) {
    u64 lo = 0, hi = ~0ull;
    uint32_t n = s.count[cut.bin];
    for (int level = 0; level * kBinBits < 64 && n > (uint32_t)kMostListed; ++level) {
      // the range that the tokens have
      u64 least = ~0ull, greatest = 0;
      each_token(row, [&](float x, int i) VQX_INLINE {
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
      const int bits = 64 - __builtin_clzll(hi - lo), shift = bits > kBinBits ? bits - kBinBits : 0;
      clear_bins(s);
      each_token(row, [&](float x, int i) VQX_INLINE {
        const u64 o = order(x, i);
        if (bin_of(scale, x) == cut.bin && o >= lo && o <= hi) {
          const int b = (int)((o - lo) >> shift);
          atomicAdd(&s.count[b], 1u);
          if (kShare) atomicAdd(&s.mass[b], whole_weight(s, scale, x));
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
    each_token(row, [&](float x, int i) VQX_INLINE {
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
      w[j] = first + j < (int)n ? whole_weight(s, scale, logit_of(s.list[first + j])) : 0;
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

  static constexpr int kEach = kMostListed / kThreads;  // listed tokens of a thread
  static constexpr int kMostNear = kThreads / 2;        // tokens of a bin that are compared with each other

  // The indexes of a row's tokens whose bins are up to `last`, and perhaps of some
  // in the next, into the list; s.listed: their number.
  template <typename T, typename H>
  static __device__ __forceinline__ void list_tokens(Shared& s, const Row<T>& row, const H& held, const Scale& scale, int last) {
    uint32_t* list = reinterpret_cast<uint32_t*>(s.list);
    // Logits are compared as they are, bf16 in the upper half of a word with the
    // lower half behind it: that moves them by less than their last place, 2^-7 of
    // them (an infinity would become a NaN; rows with one have their own way).  The
    // border is lower by that and by the roundings here.
    const float span = scale.span(last + 1);
    float least = scale.top - span;
    least -= __builtin_fabsf(least) * 0x1p-6f + (__builtin_fabsf(scale.top) + span) * 0x1p-20f + 0x1p-100f;
    if (!(least > -3.4028235e38f)) least = -3.4028235e38f;  // every finite one
    // a bit for each element, from the highest down
    auto marks = [&](const Raw<T>& r, bool there, uint32_t bits) VQX_INLINE -> uint32_t {
      if (std::is_same<T, Bf16>::value && !row.infinite) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          bits = 2 * bits + (u2f(r.a[j] << 16) >= least);
          bits = 2 * bits + (u2f(r.a[j]) >= least);
        }
      } else {
        float x[8];
        row.logits(r, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) bits = 2 * bits + (x[j] >= least);
      }
      return there ? bits : bits & ~0xFFu;
    };
    // one addition to the list's length for a wave, then a marked element of each
    // lane at a time
    auto put = [&](auto& bits, int v0) VQX_INLINE {
      constexpr int kWords = sizeof(bits) / 4;
      int n = 0;
#pragma unroll
      for (int g = 0; g < kWords; ++g) n += __popc(bits[g]);
      const u64 upto = wave_scan((u64)n);
      const int all = (int)lane_of(upto, 63);
      if (all == 0) return;
      int at = 0;
      if ((threadIdx.x & 63) == 0) at = atomicAdd(&s.listed, all);
      at = __builtin_amdgcn_readfirstlane(at) + (int)upto - n;
#pragma unroll
      for (int g = 0; g < kWords; ++g) {
        while (bits[g]) {
          const int i = __builtin_clz(bits[g]);
          bits[g] &= ~(0x80000000u >> i);
          if (at < kMostListed) list[at] = (uint32_t)(row.first(v0 + (4 * g + i / 8) * kThreads) + i % 8);
          ++at;
        }
      }
    };
    const int v0 = row.whole + (int)threadIdx.x;
    constexpr int kHeld = held_vectors<H>();
    if constexpr (kHeld > 0) {
      uint32_t bits[kHeld / 4];
#pragma unroll
      for (int g = 0; g < kHeld / 4; ++g) {
        bits[g] = 0;
        if (row.whole + 4 * g * kThreads >= row.past) continue;
#pragma unroll
        for (int a = 0; a < 4; ++a) bits[g] = marks(held.r[4 * g + a], v0 + (4 * g + a) * kThreads < row.past, bits[g]);
      }
      put(bits, v0);
    }
    for (int v = kHeld; row.whole + v * kThreads < row.past; v += 4) {
      Raw<T> r[4];
      const int first = v0 + v * kThreads;
#pragma unroll
      for (int a = 0; a < 4; ++a) r[a] = row.raw(first + a * kThreads < row.past ? first + a * kThreads : row.past - 1);
      uint32_t bits[1] = {0};
#pragma unroll
      for (int a = 0; a < 4; ++a) bits[0] = marks(r[a], first + a * kThreads < row.past, bits[0]);
      put(bits, first);
    }
    // what is not in whole vectors, a thread each
    const int head = row.whole ? (8 - row.before < row.size ? 8 - row.before : row.size) : 0, tail = row.first(row.past);
    const int i = threadIdx.x < 8 ? (int)threadIdx.x : tail + (int)threadIdx.x - 8;
    if (threadIdx.x < 8 ? i < head : (threadIdx.x < 16 && i >= head && i < row.size)) {
      if (row.logit(i) >= least) {
        const int at = atomicAdd(&s.listed, 1);
        if (at < kMostListed) list[at] = (uint32_t)i;
      }
    }
  }

  // The token drawn where all that can be kept lies in bins up to `last` and those
  // have few tokens: they are listed, and what is left is about the list.  most:
  // tokens kept by count, 0 for all; mass: what a share is of, where it is not of
  // the first `most`.  A cut is found by finer bins and, in the one where it falls,
  // by comparing that one's tokens with each other.  The histogram is gone
  // afterwards.
  enum Few { kDrawn, kTooMany, kTooNear };
  static __device__ __forceinline__ u64* index_bins(Shared& s) {
    static_assert(kMostListed / 2 >= kBins && kMostListed / 2 >= 2 * 2 * kMostNear, "");
    return s.list + kMostListed / 2;  // behind the list of tokens and those of near ones
  }
  // What few() finds: needs a barrier on either side.
  static __device__ __forceinline__ void clear_few(Shared& s) {
    const int b0 = 2 * (int)threadIdx.x;
    u64* drawn = index_bins(s);
    s.count[b0] = 0, s.count[b0 + 1] = 0, s.mass[b0] = 0, s.mass[b0 + 1] = 0, drawn[b0] = 0, drawn[b0 + 1] = 0;
    if (threadIdx.x < 3) s.spot[threadIdx.x] = kBins, s.near[threadIdx.x] = 0;
    if (threadIdx.x == 0) s.listed = 0;
  }
  template <typename T, typename H>
  static __device__ __forceinline__ Few few(Shared& s, const Row<T>& row, const H& held, const Scale& scale, const Sampling& p, int64_t r,
                     int last, u64 most, bool by_share, float share, u64 mass, double bar) {
    const int b0 = 2 * (int)threadIdx.x;
    u64* drawn = index_bins(s);
    list_tokens(s, row, held, scale, last);
    __syncthreads();
    const int listed = s.listed;
    if (listed > kMostListed) return kTooMany;
    const uint32_t* list = reinterpret_cast<const uint32_t*>(s.list);
    u64 o[kEach], w[kEach];
    int bin[kEach];
    bool keeps[kEach];
    float x[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = j * kThreads + (int)threadIdx.x;
      keeps[j] = i < listed;
      const uint32_t at = list[keeps[j] ? i : 0];
      x[j] = keeps[j] ? sound(row.logit((int)at)) : kNone;
      o[j] = order(x[j], (int)at);
    }
    const float fine = (float)kBins / (float)(last + 1);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      w[j] = 0, bin[j] = kBins;
      if (j * kThreads >= listed) continue;
      const float y = scale.bin(x[j]);
      keeps[j] = keeps[j] && y < (float)(last + 1);
      if (!keeps[j]) continue;
      w[j] = whole_weight(s, scale, x[j]);
      bin[j] = (int)(y * fine);
      if (bin[j] >= kBins) bin[j] = kBins - 1;
    }
    // the tokens of one bin, order and weight, each cut's in one half of the list
    auto gather_near = [&](int which, int half, auto in) {
      u64* near = s.list + half * 2 * kMostNear;
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (keeps[j] && in(j)) {
          const int at = atomicAdd(&s.near[which], 1);
          if (at < kMostNear) near[2 * at] = o[j], near[2 * at + 1] = w[j];
        }
      __syncthreads();
      return near;
    };
    if (most > 0) {
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (keeps[j]) atomicAdd(&s.count[bin[j]], 1u);
      __syncthreads();
      const u64 c0 = s.count[b0], c1 = s.count[b0 + 1];
      u64 all;
      const u64 before = scan_before<1, false>(s, c0 + c1, all);
      if (before < most && before + c0 + c1 >= most) {
        const bool second = before + c0 < most;
        s.spot[0] = b0 + second, s.found[0] = second ? before + c0 : before;
      }
      __syncthreads();
      const int spot = s.spot[0];
      if (spot < kBins) {
        const u64 first = s.found[0];
        const u64* near = gather_near(0, 0, [&](int j) { return bin[j] == spot; });
        const int n = s.near[0];
        if (n > kMostNear) return kTooNear;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          if (bin[j] == spot) {
            u64 rank = first;
#pragma unroll 4
            for (int i = 0; i < n; ++i) rank += near[2 * i] < o[j];
            keeps[j] = keeps[j] && rank < most;
          } else {
            keeps[j] = keeps[j] && bin[j] < spot;
          }
        }
      }
    }
    if (by_share) {
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (keeps[j]) atomicAdd(&s.mass[bin[j]], w[j]);
      __syncthreads();
      const u64 m0 = s.mass[b0], m1 = s.mass[b0 + 1];
      u64 all;
      const u64 before = scan_before<2, false>(s, m0 + m1, all);
      const double wanted = share_of(share, most > 0 ? all : mass);
      if ((double)before < wanted && (double)(before + m0 + m1) >= wanted) {
        const bool second = (double)(before + m0) < wanted;
        s.spot[1] = b0 + second, s.found[1] = second ? before + m0 : before;
      }
      __syncthreads();
      const int spot = s.spot[1];
      if (spot < kBins) {
        const u64 first = s.found[1];
        const u64* near = gather_near(1, 1, [&](int j) { return bin[j] == spot; });
        const int n = s.near[1];
        if (n > kMostNear) return kTooNear;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          if (!keeps[j]) continue;
          if (bin[j] == spot) {
            u64 sum = first;
#pragma unroll 4
            for (int i = 0; i < n; ++i) sum += near[2 * i] < o[j] ? near[2 * i + 1] : 0;
            keeps[j] = (double)sum < wanted;
          } else {
            keeps[j] = bin[j] < spot;
          }
        }
      }
    }
    // the kept ones by their index: bins of as many indexes, and in the bin where
    // the random number falls one by one
    const int shift = 32 - __builtin_clz((unsigned)(p.vocab - 1) | (kBins - 1)) - kBinBits;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      keeps[j] = keeps[j] && w[j] > 0 && (double)w[j] >= bar;
      if (keeps[j]) atomicAdd(&drawn[(uint32_t)o[j] >> shift], w[j]);
    }
    __syncthreads();
    u64 total;
    const u64 m0 = drawn[b0], m1 = drawn[b0 + 1], before = scan_before<3, false>(s, m0 + m1, total);
    const u64 target = target_of(p.random[r], total);
    if (target >= before && target < before + m0 + m1) {
      const bool second = target >= before + m0;
      s.spot[2] = b0 + second, s.found[2] = second ? before + m0 : before;
    }
    __syncthreads();
    const int spot = s.spot[2];
    const u64 rest = target - s.found[2];
    auto here = [&](int j) { return (int)((uint32_t)o[j] >> shift) == spot; };
    const u64* near = gather_near(2, 0, here);
    const int n = s.near[2];
    if (n > kMostNear) return kTooNear;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      if (!keeps[j] || !here(j)) continue;
      u64 upto = 0;
      for (int i = 0; i < n; ++i) upto += (uint32_t)near[2 * i] < (uint32_t)o[j] ? near[2 * i + 1] : 0;
      if (rest >= upto && rest < upto + w[j]) {
        p.tokens[r] = (int64_t)(uint32_t)o[j];
        p.chances[r] = (float)log((double)w[j] / (double)total);
      }
    }
    return kDrawn;
  }

  // The weight of a token that is kept, 0 of another: those up to `cut` with
  // weights from `bar` on.
  struct Kept {
    float low;      // the last kept logit,
    int low_index;  // and the last index that is kept of it
    double bar;

    __device__ __forceinline__ Kept(u64 cut, double least) {
      const bool every = cut == ~0ull;
      low = every ? kNone : logit_of(cut);
      low_index = every ? 0x7FFFFFFF : (int)(uint32_t)cut;
      bar = least;
    }
    __device__ __forceinline__ double operator()(const Shared& s, const Scale& scale, float x, int i) const {
      const double w = weight(s, scale, x);
      // no branches: eight of these side by side
      const bool in = ((x > low) | ((x == low) & (i <= low_index))) & (w >= bar);
      return in ? w : 0.0;
    }
  };

  // The masses of a row's runs of 64 vectors: put(run, mass) by one lane each.
  template <typename T, typename Put>
  static __device__ __forceinline__ void sum_runs(const Shared& s, const Row<T>& row, const Scale& scale, const Kept& kept, Put put) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row.whole >= row.past) return;
    int v = row.whole + (int)threadIdx.x, run = wave;
    Raw<T> next = row.raw(v < row.past ? v : row.past - 1);
#pragma clang loop unroll(disable)
    for (; row.whole + run * 64 < row.past; run += kWaves, v += kThreads) {
      const Raw<T> raw = next;
      next = row.raw(v + kThreads < row.past ? v + kThreads : row.past - 1);
      float x[8];
      row.logits(raw, x);
      const int e = row.first(v);
      double a = 0.0, b = 0.0;
#pragma unroll
      for (int j = 0; j < 4; ++j) a += kept(s, scale, x[2 * j], e + 2 * j), b += kept(s, scale, x[2 * j + 1], e + 2 * j + 1);
      const u64 upto = wave_scan(v < row.past ? (u64)(a + b) : 0);
      if (lane == 63) put(run, upto);
    }
  }
  // Of a vector that the row has a part of.
  template <typename T>
  static __device__ __forceinline__ u64 sum_part(const Shared& s, const Row<T>& row, const Scale& scale, const Kept& kept, int v) {
    float x[8];
    row.load(v, x);
    double a = 0.0;
#pragma unroll
    for (int j = 0; j < 8; ++j) a += kept(s, scale, x[j], row.first(v) + j);
    return (u64)a;
  }

  // The token drawn, given the masses in s.mass: bin 0 is the part of a vector that
  // a row begins with, then come 2^shift runs each, then the part that it ends with.
  template <typename T>
  static __device__ __forceinline__ void pick(Shared& s, const Row<T>& row, const Scale& scale, const Sampling& p, int64_t r,
                                       const Kept& kept, int shift) {
    const int lane = threadIdx.x & 63, tail = 2 + (row.runs() >> shift);
    __syncthreads();
    const int b0 = 2 * (int)threadIdx.x;
    u64 total;
    const u64 m0 = s.mass[b0], m1 = s.mass[b0 + 1], before = scan_before(s, m0 + m1, total);
    const u64 target = target_of(p.random[r], total);
    if (target >= before && target < before + m0 + m1) {
      const bool second = target >= before + m0;
      s.at = b0 + second, s.found[0] = second ? before + m0 : before;
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    const int bin = __builtin_amdgcn_readfirstlane(s.at);
    u64 rest = target - s.found[0];
    // the vectors of the bin, 64 at a time
    const int first = bin == 0 ? 0 : (bin == tail ? row.tail : row.whole + ((bin - 1) << shift) * 64);
    const int end = bin == 0 ? 1 : (bin == tail ? row.tail + 1 : first + (64 << shift) < row.past ? first + (64 << shift) : row.past);
    for (int v = first + lane; v - lane < end; v += 64) {
      float x[8];
      double w[8], sum = 0.0;
      row.load(v < end ? v : end - 1, x);
      const int e = row.first(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = v < end ? kept(s, scale, x[j], e + j) : 0.0, sum += w[j];
      const u64 upto = wave_scan((u64)sum), all = lane_of(upto, 63);
      if (rest >= all) {
        rest -= all;
        continue;
      }
      u64 left = upto - (u64)sum;
      if (rest >= left && rest < upto) {
        int token = 0;
        double weighs = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (weighs == 0.0 && rest < left + (u64)w[j]) weighs = w[j], token = e + j;
          left += (u64)w[j];
        }
        p.tokens[r] = token;
        p.chances[r] = (float)log(weighs / (double)total);
      }
      return;
    }
  }

  // Runs of 64 vectors that have a bin of their own, with two for the row's ends.
  static constexpr int kMostRuns = kBins - 3;

  // The token drawn of those that are kept, however many they are: the masses of
  // runs, and in the one where the random number falls a wave by itself.
  template <typename T>
  static __device__ __forceinline__ void draw(Shared& s, const Row<T>& row, const Scale& scale, const Sampling& p, int64_t r,
                                       const Kept& kept) {
    int shift = 0;
    while ((row.runs() >> shift) > kMostRuns) ++shift;
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.mass[i] = 0;
    __syncthreads();
    sum_runs(s, row, scale, kept, [&](int run, u64 mass) { if (mass) atomicAdd(&s.mass[1 + (run >> shift)], mass); });
    if (threadIdx.x == 0 && row.head) s.mass[0] = sum_part(s, row, scale, kept, 0);
    if (threadIdx.x == 64 && row.tail >= 0) s.mass[2 + (row.runs() >> shift)] = sum_part(s, row, scale, kept, row.tail);
    pick(s, row, scale, p, r, kept, shift);
  }

  // ---------------------------------------------------------------------------
  // a row
  // ---------------------------------------------------------------------------
  // What the workgroups of a row leave each other.
  static constexpr int kMostParts = 256;
  struct Parts {
    u64 runs[kBins];  // the masses of runs, as pick() takes them,
    u64 mass[kBins];  // or the histogram
    uint32_t count[kBins];
    float tops[kMostParts];
  };

  static __device__ __forceinline__ Scale scale_of(float top, float t) {
    Scale scale;
    scale.top = top;
    scale.inner = 64.0 * 1.44269504088896340736 / (double)t;
    scale.half = t < 1.0f ? 1.0f : 0.5f;
    scale.half_top = scale.half * top;
    const double bins = scale.inner * (kFine / 64.0) / (double)scale.half;
    scale.bins[0] = (float)(bins > 0x1p100 ? 0x1p100 : bins);
    scale.bins[1] = bins > 0x1p100 ? (float)(bins * 0x1p-100) : 1.0f;
    return scale;
  }
  // The least weight that is kept.
  static __device__ __forceinline__ double bar_of(float least) {
    return least > 0.0f ? (least < 1.0f ? (double)least * kUnit : kUnit) : 0.0;
  }
  // The largest of the lanes' and the waves'.
  static __device__ __forceinline__ float top_of(Shared& s, float top) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) top = __builtin_fmaxf(top, __shfl_xor(top, d));
    if ((threadIdx.x & 63) == 0) s.tops[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = __builtin_fmaxf(top, s.tops[w]);
    return top + 0.0f;
  }
  template <typename T, typename H>
  static __device__ __forceinline__ float largest(const Row<T>& row, const H& held) {
    float top = kNone;
    each_vector(row, [&](const float(&x)[8], int) VQX_INLINE {
#pragma unroll
      for (int j = 0; j < 8; ++j) top = __builtin_fmaxf(top, x[j]);  // a NaN is no maximum
    }, held);
    return top;
  }

  // Few rows: a row's largest logit by many workgroups; what the next launch adds
  // to is cleared.
  template <typename T>
  static __device__ __forceinline__ void top(Shared& s, const Sampling& p, Parts* parts, int each) {
    const int64_t r = blockIdx.x / (unsigned)each;
    const int g = (int)(blockIdx.x % (unsigned)each);
    const Row<T> row = Row<T>(p.logits, r * p.stride, p.vocab).part(g, each);
    const float top = top_of(s, largest(row, NotHeld()));
    Parts& to = parts[r];
    if (threadIdx.x == 0) to.tops[g] = top;
    for (int i = g * kThreads + (int)threadIdx.x; i < kBins; i += each * kThreads) to.runs[i] = 0, to.mass[i] = 0, to.count[i] = 0;
  }

  // Few rows: the masses of its runs, or (top-p) its histogram.
  template <typename T>
  static __device__ __forceinline__ void sums(Shared& s, const Sampling& p, Parts* parts, int each) {
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x / (unsigned)each;
    const int g = (int)(blockIdx.x % (unsigned)each);
    Parts& to = parts[r];
    const Row<T> whole(p.logits, r * p.stride, p.vocab);
    Row<T> row = whole.part(g, each);
    const float t = p.temperature ? p.temperature[r] : 1.0f, share = p.top_p ? p.top_p[r] : 1.0f;
    const double bar = bar_of(p.min_p ? p.min_p[r] : 0.0f);
    if (tid < 64) s.powers[tid] = exp2((double)tid / 64.0);
    float top = top_of(s, tid < each ? to.tops[tid] : kNone);
    if (top == kNone || !(t > 0.0f)) return;
    if (top == -kNone) row.infinite = true, top = 0.0f;
    const Scale scale = scale_of(top, t);
    if (!(share < 1.0f)) {
      const Kept kept(~0ull, bar);
      const int before = 1 + (row.whole - whole.whole) / 64;
      sum_runs(s, row, scale, kept, [&](int run, u64 mass) { to.runs[before + run] = mass; });
      if (tid == 0 && row.head) to.runs[0] = sum_part(s, row, scale, kept, 0);
      if (tid == 64 && row.tail >= 0) to.runs[2 + whole.runs()] = sum_part(s, row, scale, kept, row.tail);
      return;
    }
    clear_bins(s);
    each_vector(row, [&](const float(&x)[8], int) VQX_INLINE {
      double w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = weight(s, scale, x[j]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int b = bin_of(scale, x[j]);
        if (b < kBins) atomicAdd(&s.count[b], 1u), atomicAdd(&s.mass[b], (u64)w[j]);
      }
    }, OneAhead());
    __syncthreads();
    for (int i = tid; i < kBins; i += kThreads)
      if (s.count[i]) atomicAdd(&to.count[i], s.count[i]), atomicAdd(&to.mass[i], s.mass[i]);
  }

  // kParts: the launches above have been there.
  template <typename T, bool kParts>
  static __device__ __forceinline__ void sample(Shared& s, const Sampling& p, const Parts* parts, int each) {
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    Row<T> row(p.logits, r * p.stride, p.vocab);
    std::conditional_t<kParts, NotHeld, Held<T>> held;
    if constexpr (!kParts) held.load(row);
    const float t = p.temperature ? p.temperature[r] : 1.0f;
    const int k = !kParts && p.top_k ? p.top_k[r] : 0;
    const float share = p.top_p ? p.top_p[r] : 1.0f, least = p.min_p ? p.min_p[r] : 0.0f;
    if (tid < 64) s.powers[tid] = exp2((double)tid / 64.0);
    clear_few(s);
    float mine = kNone;
    if constexpr (!kParts)
      mine = largest(row, held);
    else if (tid < each)
      mine = parts[r].tops[tid];
    float top = top_of(s, mine);
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
    if (top == -kNone) row.infinite = true, top = 0.0f;
    const Scale scale = scale_of(top, t);
    const bool by_count = k > 0 && k < p.vocab, by_share = share < 1.0f;
    const double bar = bar_of(least);
    u64 cut = ~0ull;
    const Cut none = {kBins, 0, 0};
    if constexpr (kParts) {
      if (!by_share) {
        for (int i = tid; i < kBins; i += kThreads) s.mass[i] = parts[r].runs[i];
        pick(s, row, scale, p, r, Kept(cut, bar), 0);
        return;
      }
    }
    // the last bin that a kept token can be in, as far as it is known without a
    // histogram: by the share of the largest weight (half a unit less, which is
    // rounded up to it, and one bin more for a bin's rounding), and by the k-th of
    // the threads' largest logits
    int last = kBins;
    if (bar > 0.0 && !(by_share && by_count)) {
      const float y = -__builtin_amdgcn_logf(least - 0x1p-41f) * kFine + 1.0f;  // NaN: none
      if (y < (float)kBins) last = y > 0.0f ? (int)y : 0;
    }
    const int tight = last;
    if (by_count && k <= kThreads) {
      uint32_t* count = reinterpret_cast<uint32_t*>(index_bins(s));
      const int b = bin_of(scale, row.infinite && mine != -kNone ? kNone : __builtin_fminf(mine, top)), b0 = 2 * tid;
      if (b < kBins) atomicAdd(&count[b], 1u);
      __syncthreads();
      const u64 c0 = count[b0], c1 = count[b0 + 1];
      u64 all;
      const u64 before = scan_before<0, false>(s, c0 + c1, all);
      index_bins(s)[b0] = 0, index_bins(s)[b0 + 1] = 0;
      if (before < (u64)k && before + c0 + c1 >= (u64)k) s.at = before + c0 < (u64)k ? b0 + 1 : b0;
      __syncthreads();
      if (all >= (u64)k && s.at < last) last = s.at;
    }
    // a histogram: how many; and all weights' sum; and each bin's
    u64 mass = 0;
    enum Sums { kCounts, kTotal, kMasses };
    auto count_bins = [&](auto what) VQX_INLINE {
      constexpr Sums kWhat = decltype(what)::value;
      if constexpr (kParts) {
        u64 sum = 0;
        __syncthreads();
        for (int i = tid; i < kBins; i += kThreads) {
          s.count[i] = parts[r].count[i];
          s.mass[i] = parts[r].mass[i], sum += s.mass[i];
        }
        mass = sum_of(s, sum);
        __syncthreads();
        return;
      }
      clear_bins(s);
      double sum = 0.0;
      each_vector(row, [&](const float(&x)[8], int) VQX_INLINE {
        double w[8];
        if (kWhat != kCounts) {
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = weight(s, scale, x[j]), sum += w[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int b = bin_of(scale, x[j]);
          if (b < kBins) {
            atomicAdd(&s.count[b], 1u);
            if (kWhat == kMasses) atomicAdd(&s.mass[b], (u64)w[j]);
          }
        }
      }, std::conditional_t<kWhat == kCounts, NotHeld, OneAhead>());
      __syncthreads();
      if (kWhat != kCounts) mass = sum_of(s, (u64)sum);
    };
    auto counts = std::integral_constant<Sums, kCounts>();
    auto with_total = std::integral_constant<Sums, kTotal>();
    auto with_masses = std::integral_constant<Sums, kMasses>();
    // few tokens, by what is known so far, or by a histogram of the row
    const u64 most = by_count ? (u64)k : 0;
    Few done = kTooMany;
    if (last < kBins && !(by_share && !by_count)) done = few(s, row, held, scale, p, r, last, most, by_share, share, mass, bar);
    if (done == kDrawn) return;
    if (done == kTooMany && (by_count || by_share)) {
      last = tight;
      Cut c;
      if (by_count) {
        count_bins(counts);
        c = find_bin<false>(s, none, most, 0.0);
      } else {
        count_bins(with_total);
        c = kParts ? find_bin<true, true>(s, none, 0, share_of(share, mass)) : find_least(s, share_of(share, mass), mass);
      }
      const bool listable = c.bin < last ? c.count + s.count[c.bin] <= (u64)kMostListed : last < kBins;
      if (c.bin < last) last = c.bin;
      if (listable) {
        __syncthreads();
        clear_few(s);
        __syncthreads();
        if (few(s, row, NotHeld(), scale, p, r, last, most, by_share, share, mass, bar) == kDrawn) return;
      }
    }
    if (by_count || by_share) {
      // cut by cut
      if (by_share)
        count_bins(with_masses);
      else
        count_bins(counts);
      if (by_count) {
        const Cut c = by_share ? find_bin<false, true>(s, none, most, 0.0) : find_bin<false>(s, none, most, 0.0);
        if (c.bin < kBins) {
          // the histogram is made again by a bin that is cut finer
          const bool keeps = s.count[c.bin] <= (uint32_t)kMostListed;
          u64 upto;
          cut = resolve<false>(s, row, scale, c, most, 0.0, upto);
          if (by_share && !keeps) {
            // up to the cut, which is in the bin
            double sum = 0.0;
            each_token(row, [&](float x, int i) VQX_INLINE {
              if (order(x, i) <= cut) sum += weight(s, scale, x);
            });
            upto = sum_of(s, (u64)sum);
            count_bins(with_masses);
          }
          mass = upto;
        }
      }
      if (by_share) {
        const double wanted = share_of(share, mass);
        const Cut c = find_bin<true>(s, none, 0, wanted);
        if (c.bin < kBins) {
          u64 upto;
          const u64 o = resolve<true>(s, row, scale, c, 0, wanted, upto);
          cut = o < cut ? o : cut;
        }
      }
    }
    draw(s, row, scale, p, r, Kept(cut, bar));
  }
};

template <int kThreads, typename T>
__global__ __launch_bounds__(kThreads) void sample_top_kernel(Sampling p, typename Sampler<kThreads>::Parts* parts, int each) {
  __shared__ typename Sampler<kThreads>::Shared s;
  Sampler<kThreads>::template top<T>(s, p, parts, each);
}
template <int kThreads, typename T>
__global__ __launch_bounds__(kThreads) void sample_sums_kernel(Sampling p, typename Sampler<kThreads>::Parts* parts, int each) {
  __shared__ typename Sampler<kThreads>::Shared s;
  Sampler<kThreads>::template sums<T>(s, p, parts, each);
}
template <int kThreads, typename T, bool kParts>
__global__ __launch_bounds__(kThreads) void sample_kernel(Sampling p, const typename Sampler<kThreads>::Parts* parts, int each) {
  __shared__ typename Sampler<kThreads>::Shared s;
  Sampler<kThreads>::template sample<T, kParts>(s, p, parts, each);
}

using Large = Sampler<1024>;

}  // namespace

// Workgroups of a row of their own launches before the row's, 0 for none: where
// rows are fewer than half the compute units, no number of tokens bounds what
// is looked at and a part has 4096 logits or more.  bf16, without cuts: one row of
// 131072 12 us, 42 by one workgroup; 16 rows 17; with a top_p that keeps thousands
// 79 and 185.
static int parts_of(const Sampling& p) {
  if (p.top_k || p.rows == 0 || p.vocab > Large::kMostRuns * 64 * 8) return 0;
  int64_t each = num_cus() / p.rows;
  if (each > p.vocab / 4096) each = p.vocab / 4096;
  if (each > Large::kMostParts) each = Large::kMostParts;
  return each < 2 ? 0 : (int)each;
}

int64_t sample_workspace(const Sampling& p) { return parts_of(p) ? p.rows * (int64_t)sizeof(Large::Parts) : 0; }

// Threads of a row's workgroup: barriers and scans of few waves are short, and
// workgroups of few share a compute unit, but each has as many more of the logits
// and lists fewer tokens.  1024, 512 and 256, us: 13 rows of 2000 fp32 logits, top
// 40, 9.9, 7.9 and 7.5; 1000 of 4096 35, 27 and 14; 13 of 8000 bf16 10.3, 8.3 and 8.0,
// top_p alone 17, 15 and 27; 512 of 32000 22, 14 and 14, top 1000 29, 24 and 61; 256
// of 131072, top 50, 25, 27 and 44, top 1000 30, 50 and 191.
static int threads_of(const Sampling& p) {
  return p.vocab <= 4096 ? 256 : (p.vocab <= 8192 || p.rows > num_cus() ? 512 : 1024);
}

int sample(const Sampling& p, int dtype, void* ws, hipStream_t st) {
  if (p.rows == 0) return kOk;
  const int each = parts_of(p), threads = each ? 1024 : threads_of(p);
  Large::Parts* parts = static_cast<Large::Parts*>(ws);
  const dim3 grid((unsigned)p.rows), all((unsigned)(p.rows * each)), block(threads);
#define VQX_SAMPLE(T)                                                                                      \
  do {                                                                                                     \
    if (each) {                                                                                            \
      hipLaunchKernelGGL((sample_top_kernel<1024, T>), all, block, 0, st, p, parts, each);                 \
      hipLaunchKernelGGL((sample_sums_kernel<1024, T>), all, block, 0, st, p, parts, each);                \
      hipLaunchKernelGGL((sample_kernel<1024, T, true>), grid, block, 0, st, p, parts, each);              \
    } else if (threads == 1024) {                                                                          \
      hipLaunchKernelGGL((sample_kernel<1024, T, false>), grid, block, 0, st, p, nullptr, 0);              \
    } else if (threads == 512) {                                                                           \
      hipLaunchKernelGGL((sample_kernel<512, T, false>), grid, block, 0, st, p, nullptr, 0);               \
    } else {                                                                                               \
      hipLaunchKernelGGL((sample_kernel<256, T, false>), grid, block, 0, st, p, nullptr, 0);               \
    }                                                                                                      \
  } while (0)
  if (dtype == kF32)
    VQX_SAMPLE(float);
  else if (dtype == kBF16)
    VQX_SAMPLE(Bf16);
  else
    VQX_SAMPLE(F16);
#undef VQX_SAMPLE
  return check_launch("sample_tokens");
}

}  // namespace vqx
