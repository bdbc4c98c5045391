// Rotary positions, as the kernels of vqx_rotary.hip see them.
#pragma once

#include "vqx_kv4.h"

namespace vqx {

// How pairs are turned: the first 2 half elements of a head, i with i + half or
// (interleaved) 2 i with 2 i + 1.
struct Turn {
  const float* freqs;        // [half], radians from one position to the next
  const int32_t* positions;  // [tokens]; NULL with a cache: places in it
  int32_t half;
  bool interleaved, back;  // back: by the negative angles
  float factor;
};

// [tokens, heads, dim] with rows that start on 16 bytes; dim a multiple of 8.
struct Rows {
  const void* p;
  int64_t sn, sh;  // elements between tokens, between heads
  int32_t heads, dim;
};

int rotary(const Turn& t, const Rows& x, int dtype, int64_t n, void* out, hipStream_t st);
int kv4_append_rotary(const Kv4View& c, int dim, const Kv4Tokens& q, const Turn& t, const Rows& query, const Rows& key,
                      const Rows& value, int dtype, void* out, hipStream_t st);

}  // namespace vqx
