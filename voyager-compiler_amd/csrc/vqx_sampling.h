// Sampling, as the kernel of vqx_sampling.hip sees it.
#pragma once

#include "vqx_common.h"

namespace vqx {

// What may be NULL is not asked for.
struct Sampling {
  const void* logits;  // [rows, vocab]
  int64_t stride;      // elements between rows
  int64_t rows;
  int32_t vocab;
  const float* random;       // [rows]
  const float* temperature;  // [rows], or NULL
  const int32_t* top_k;      // [rows], or NULL
  const float* top_p;        // [rows], or NULL
  const float* min_p;        // [rows], or NULL
  int64_t* tokens;           // [rows]
  float* chances;            // [rows]
};

int64_t sample_workspace(const Sampling& p);  // bytes, 0: none
int sample(const Sampling& p, int dtype, void* ws, hipStream_t st);

}  // namespace vqx
