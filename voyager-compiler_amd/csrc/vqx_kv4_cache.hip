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

// 8 consecutive values as fp32 (exact).
__device__ __forceinline__ void load8(const void* p, int64_t at, float, float (&x)[8]) {
  const f32x4* q = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
  const f32x4 a = ld_nt(q), b = ld_nt(q + 1);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = a[i], x[i + 4] = b[i];
}
__device__ __forceinline__ void load8(const void* p, int64_t at, Bf16, float (&x)[8]) {
  const u32x4 a = ld_nt(reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + at));
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = u2f(a[i] << 16), x[2 * i + 1] = u2f(a[i] & 0xFFFF0000u);
}
__device__ __forceinline__ void load8(const void* p, int64_t at, F16, float (&x)[8]) {
  const u32x4 a = ld_nt(reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + at));
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = h2f_exact(a[i] & 0xFFFFu), x[2 * i + 1] = h2f_exact(a[i] >> 16);
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

// The code of v (a bf16 value): the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties
// to the even code, both zeros 0.  A small value that rounds to 0 keeps its sign.
__device__ __forceinline__ uint32_t fp4_code(float v) {
  const float a = __builtin_fabsf(v);
  const uint32_t m = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
  return a == 0.0f ? 0u : m | (f2u(v) >> 31) << 3;
}
__device__ __forceinline__ float fp4_value(uint32_t code) {
  const uint32_t m = code & 7u;
  // exponent field 0: 0 or 0.5; else (1 + fraction / 2) 2^(field - 1)
  const uint32_t b = m < 2 ? m * 0x3F000000u : ((m >> 1) + 126u) << 23 | (m & 1u) << 22;
  return u2f(b | (code & 8u) << 28);
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

// The row of new token i of head h, false where it has none: a place before
// the sequence's first token or past its room, or a page that is none.
__device__ __forceinline__ bool new_token_row(const Kv4View& c, const Kv4Tokens& q, int i, uint32_t h, uint32_t& row) {
  const uint32_t b = sequence_of(c, q, i);
  int first, count;
  kv4_span(q, b, first, count);
  const int64_t pos = (int64_t)c.lengths[b] - count + (i - first);
  if (i < first || i >= first + count || pos < 0 || pos >= (int64_t)c.cap) return false;
  const uint32_t page = kv4_page(c, b, (uint32_t)pos);
  row = kv4_row(c, page, h, (uint32_t)pos);
  return page < c.pages;
}

// One lane has 8 values, four lanes a block, D / 8 lanes a row; both planes in
// one launch.  Bound by the values' bytes; a call of a decode step by its launch.
template <typename T>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4View c, Kv4Tokens q, int dim, const void* key,
                                                         const void* value, int64_t key_sn, int64_t key_sh,
                                                         int64_t value_sn, int64_t value_sh, uint64_t items) {
  const uint32_t per_row = (uint32_t)dim / 8;
  const uint64_t half = items / 2;
  for (uint64_t w = (uint64_t)blockIdx.x * 256 + threadIdx.x; w < items; w += (uint64_t)gridDim.x * 256) {
    const uint32_t plane = w >= half;
    const uint64_t v = w - (plane ? half : 0);
    const uint64_t pair = v / per_row;
    const uint32_t part = (uint32_t)(v - pair * per_row);
    const int i = (int)(pair / c.kv);
    const uint32_t h = (uint32_t)(pair - (uint64_t)i * c.kv);
    float x[8];
    load8(plane ? value : key, (int64_t)i * (plane ? value_sn : key_sn) + (int64_t)h * (plane ? value_sh : key_sh) + part * 8,
          T(), x);
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
    uint32_t code = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) code |= fp4_code(bf2f(f2bf(x[j] * r))) << (4 * j);
    uint32_t row;
    if (!new_token_row(c, q, i, h, row)) continue;
    const uint64_t at = plane * c.plane_rows + row;
    reinterpret_cast<uint32_t*>(c.codes)[at * per_row + part] = finite ? code : 0u;
    // a block with an infinity or a NaN is NaN as a whole
    if ((part & 3) == 0) c.scales[at * (per_row / 4) + part / 4] = (uint8_t)(finite ? e + 127 : 255);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4View c, Kv4Tokens q, int dim, void* key, void* value,
                                                       uint64_t items) {
  const uint32_t per_row = (uint32_t)dim / 8;
  const uint64_t half = items / 2;
  for (uint64_t w = (uint64_t)blockIdx.x * 256 + threadIdx.x; w < items; w += (uint64_t)gridDim.x * 256) {
    const uint32_t plane = w >= half;
    const uint64_t v = w - (plane ? half : 0);
    const uint64_t pair = v / per_row;
    const uint32_t part = (uint32_t)(v - pair * per_row);
    const int i = (int)(pair / c.kv);
    const uint32_t h = (uint32_t)(pair - (uint64_t)i * c.kv);
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    uint32_t row;
    if (new_token_row(c, q, i, h, row)) {
      const uint64_t at = plane * c.plane_rows + row;
      const uint32_t code = reinterpret_cast<const uint32_t*>(c.codes)[at * per_row + part];
      const float s = kv4_scale(c.scales[at * (per_row / 4) + part / 4]);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = fp4_value(code >> (4 * j) & 15u) * s;
    }
    store8(plane ? value : key, (int64_t)v * 8, T(), x);
  }
}

// ---------------------------------------------------------------------------
// evict: the heaviest and the latest tokens of each head
// ---------------------------------------------------------------------------
// The order of weights as one of unsigned numbers; both zeros are one weight,
// a NaN is above all.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xFFFFFFFFu;
  const uint32_t b = w == 0.0f ? 0u : f2u(w);
  return b >> 31 ? ~b : b | 0x80000000u;
}

constexpr int kSelectThreads = 1024;
constexpr int kBins = 2048;

// One workgroup picks the tokens of one head of one sequence: of the `old`
// tokens before the latest `recent` it finds the weight of the room-th heaviest
// by three histograms of 11, 11 and 10 bits of the key, then each wave counts
// and writes the tokens of its own run, lowest first, so that equal weights go
// by their place.  Five passes over weights that stay in L2.
__global__ __launch_bounds__(kSelectThreads) void kv4_select_kernel(Kv4View c, const float* weights,
                                                                    int64_t weights_len, int budget, int recent,
                                                                    int32_t* index, int32_t* kept,
                                                                    float* out_weights) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t wave_sum[kSelectThreads / 64], wave_tie[kSelectThreads / 64];
  __shared__ uint32_t found[2];
  const uint32_t b = blockIdx.x / c.kv;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
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
  uint32_t prefix = 0, need = (uint32_t)room;
  int low = 32;  // bits of the key below those that prefix settles
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass == 2 ? 10 : 11;
    const uint32_t known = low == 32 ? 0u : ~0u << low;
    low -= bits;
    for (int j = tid; j < kBins; j += kSelectThreads) hist[j] = 0;
    __syncthreads();
    for (int j = tid; j < old; j += kSelectThreads) {
      const uint32_t k = weight_key(w[j]);
      if ((k & known) == prefix) atomicAdd(&hist[k >> low & (kBins - 1)], 1u);  // counts: no order in them
    }
    __syncthreads();
    // bin 2047 - 2 tid and the one below it: how many keys are above
    const int hi = kBins - 1 - 2 * tid;
    const uint32_t h0 = hist[hi], h1 = hist[hi - 1];
    uint32_t sum = h0 + h1;
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t o = __shfl_up(sum, d);
      if (lane >= d) sum += o;
    }
    if (lane == 63) wave_sum[wave] = sum;
    __syncthreads();
    uint32_t above = sum - h0 - h1;
    for (int k = 0; k < wave; ++k) above += wave_sum[k];
    if (above < need && need <= above + h0) found[0] = (uint32_t)hi, found[1] = need - above;
    if (above + h0 < need && need <= above + h0 + h1) found[0] = (uint32_t)hi - 1, found[1] = need - above - h0;
    __syncthreads();
    prefix |= found[0] << low;
    need = found[1];
    __syncthreads();
  }
  // prefix is the key of the room-th heaviest, `need` of the tokens with that
  // very key are kept.  Each wave has a run of 64-token steps.
  const int steps = (old + 63) / 64, per = (steps + kWaves - 1) / kWaves;
  const int s0 = wave * per, s1 = s0 + per < steps ? s0 + per : steps;
  uint32_t more = 0, tie = 0;
  for (int s = s0; s < s1; ++s) {
    const int j = s * 64 + lane;
    const uint32_t k = j < old ? weight_key(w[j]) : 0u;
    more += (uint32_t)__popcll(__ballot(j < old && k > prefix));
    tie += (uint32_t)__popcll(__ballot(j < old && k == prefix));
  }
  if (lane == 0) wave_sum[wave] = more, wave_tie[wave] = tie;
  __syncthreads();
  uint32_t at = 0, ties = 0;  // kept and equal tokens before this wave's run
  for (int k = 0; k < wave; ++k) at += wave_sum[k], ties += wave_tie[k];
  at += ties < need ? ties : need;
  const uint64_t below = (1ull << lane) - 1;
  for (int s = s0; s < s1; ++s) {
    const int j = s * 64 + lane;
    const float x = j < old ? w[j] : 0.0f;
    const uint32_t k = weight_key(x);
    const uint64_t eq = __ballot(j < old && k == prefix);
    const bool take = j < old && (k > prefix || (k == prefix && ties + (uint32_t)__popcll(eq & below) < need));
    const uint64_t all = __ballot(take);
    if (take) {
      const uint32_t p = at + (uint32_t)__popcll(all & below);
      idx[p] = j;
      ow[p] = x;
    }
    at += (uint32_t)__popcll(all);
    ties += (uint32_t)__popcll(eq);
  }
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

int kv4_append(const Kv4View& c, int dim, const Kv4Tokens& t, const void* key, const void* value, int dtype,
               int64_t key_sn, int64_t key_sh, int64_t value_sn, int64_t value_sh, hipStream_t st) {
  const uint64_t items = 2ull * (uint64_t)t.n * c.kv * (uint64_t)(dim / 8);
  if (items == 0) return kOk;
  const unsigned grid = grid_for((int64_t)items, 256, 16);
#define VQX_KV4_APPEND(T)                                                                                          \
  hipLaunchKernelGGL((kv4_append_kernel<T>), dim3(grid), dim3(256), 0, st, c, t, dim, key, value, key_sn, key_sh, \
                     value_sn, value_sh, items)
  if (dtype == kF32)
    VQX_KV4_APPEND(float);
  else if (dtype == kBF16)
    VQX_KV4_APPEND(Bf16);
  else
    VQX_KV4_APPEND(F16);
#undef VQX_KV4_APPEND
  return check_launch("kv4_append");
}

int kv4_read(const Kv4View& c, int dim, const Kv4Tokens& t, void* key, void* value, int dtype, hipStream_t st) {
  const uint64_t items = 2ull * (uint64_t)t.n * c.kv * (uint64_t)(dim / 8);
  if (items == 0) return kOk;
  const unsigned grid = grid_for((int64_t)items, 256, 16);
#define VQX_KV4_READ(T) \
  hipLaunchKernelGGL((kv4_read_kernel<T>), dim3(grid), dim3(256), 0, st, c, t, dim, key, value, items)
  if (dtype == kF32)
    VQX_KV4_READ(float);
  else if (dtype == kBF16)
    VQX_KV4_READ(Bf16);
  else
    VQX_KV4_READ(F16);
#undef VQX_KV4_READ
  return check_launch("kv4_read");
}

int kv4_evict(const Kv4View& c, int dim, const float* weights, int64_t weights_len, int budget, int recent,
              const Kv4View& out, int32_t* index, int32_t* kept, float* out_weights, hipStream_t st) {
  if (c.seqs == 0) return kOk;
  hipLaunchKernelGGL(kv4_select_kernel, dim3(c.seqs * c.kv), dim3(kSelectThreads), 0, st, c, weights, weights_len,
                     budget, recent, index, kept, out_weights);
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
