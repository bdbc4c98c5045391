// A cache of keys and values in the fp4_e2m1 microscaling format, as the
// kernels of vqx_kv4_cache.hip and vqx_kv4_attention.hip see it.
//
// A row is one token of one head in one plane (keys or values): D / 2 bytes of
// codes, element 2 i in the low nibble, and D / 32 E8M0 scale bytes.  Rows are
// counted in 32 bits (the host checks that a plane has fewer than 2^32), byte
// offsets in 64.
#pragma once

#include "vqx_common.h"

namespace vqx {

struct Kv4View {
  uint8_t* codes;          // [2, pages, kv, size, D / 2]
  uint8_t* scales;         // [2, pages, kv, size, D / 32]
  const int32_t* table;    // [seqs, per_seq], or NULL: page b is sequence b
  const int32_t* lengths;  // [seqs]
  uint64_t plane_rows;     // pages * kv * size
  uint32_t pages, per_seq, kv, size;
  uint32_t cap;   // tokens a sequence can have
  int32_t shift;  // log2(size), or -1 where size is no power of two
  uint32_t seqs;
};

// New tokens [n] of the sequences: those of sequence b are cu[b] .. cu[b + 1],
// or n / seqs each, and stand at the end of what lengths counts.
struct Kv4Tokens {
  const int32_t* cu;
  int32_t n, each;
};

__device__ __forceinline__ void kv4_span(const Kv4Tokens& q, uint32_t b, int& first, int& count) {
  if (q.cu) {
    // a table of offsets is the caller's data: no access follows it out of [0, n]
    const int lo = q.cu[b], hi = q.cu[b + 1];
    first = lo < 0 ? 0 : (lo > q.n ? q.n : lo);
    const int end = hi > q.n ? q.n : hi;
    count = end > first ? end - first : 0;
  } else {
    first = (int)b * q.each;
    count = q.each;
  }
}

__device__ __forceinline__ int kv4_length(const Kv4View& c, uint32_t b) {
  const int n = c.lengths[b];
  return n < 0 ? 0 : ((uint32_t)n > c.cap ? (int)c.cap : n);
}

__device__ __forceinline__ uint32_t kv4_div(const Kv4View& c, uint32_t t) {
  return c.shift >= 0 ? t >> c.shift : t / c.size;
}

// The page of token t < cap of sequence b; one outside [0, pages) is no page.
__device__ __forceinline__ uint32_t kv4_page(const Kv4View& c, uint32_t b, uint32_t t) {
  return c.table ? (uint32_t)c.table[(uint64_t)b * c.per_seq + kv4_div(c, t)] : b;
}

// The row of token t of head h on that page, 0 where the page is none.
__device__ __forceinline__ uint32_t kv4_row(const Kv4View& c, uint32_t page, uint32_t h, uint32_t t) {
  return page < c.pages ? (page * c.kv + h) * c.size + (t - kv4_div(c, t) * c.size) : 0u;
}

// A scale byte's value: 2^(byte - 127), NaN for 255 (2^-127 is subnormal).
__device__ __forceinline__ float kv4_scale(uint32_t byte) {
  return byte == 0 ? u2f(0x00400000u) : (byte == 255 ? u2f(0x7FC00000u) : u2f(byte << 23));
}

int kv4_append(const Kv4View& c, int dim, const Kv4Tokens& t, const void* key, const void* value, int dtype,
               int64_t key_sn, int64_t key_sh, int64_t value_sn, int64_t value_sh, hipStream_t st);
int kv4_read(const Kv4View& c, int dim, const Kv4Tokens& t, void* key, void* value, int dtype, hipStream_t st);
int kv4_evict(const Kv4View& c, int dim, const float* weights, int64_t weights_len, int budget, int recent,
              const Kv4View& out, int32_t* index, int32_t* kept, float* out_weights, void* ws, hipStream_t st);
int64_t kv4_evict_workspace(const Kv4View& c, int64_t weights_len);  // bytes

// Queries [n, heads, D] of the new tokens and what becomes of their scores.
struct Kv4Query {
  const void* q;
  int64_t sn, sh;  // elements between tokens, between heads
  Kv4Tokens tokens;
  int32_t heads, group;  // query heads, query heads of one kv head
  int32_t most;          // no sequence has more new tokens
  int32_t window;        // 0: none
  float scale, softcap;  // softcap 0: none
  const float* slopes;   // [heads], or NULL
};

// Bytes of workspace a call needs (0: none).
int64_t kv4_workspace(const Kv4View& c, int dim, const Kv4Query& q, int dtype);
int kv4_attention(const Kv4View& c, int dim, const Kv4Query& q, int dtype, void* out, float* lse, float* ws,
                  hipStream_t st);
int kv4_accumulate(const Kv4View& c, int dim, const Kv4Query& q, int dtype, const float* lse, float* weights,
                   int64_t weights_len, hipStream_t st);

}  // namespace vqx
