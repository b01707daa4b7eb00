// Interface of the sampling translation unit.
#pragma once
#include "ugb_internal.h"

struct ugb_sample_args {
  const void *logits;          // T [rows], ld apart: [vocab]
  bool bf16;
  const float *temperature;    // [rows] each; null = 1, off, off, off
  const int *top_k;
  const float *top_p, *min_p;
  const float *u;              // [rows], 0 <= u < 1
  int *tokens;                 // [rows]
  float *prob;                 // [rows] or null
  int rows, vocab;
  long long ld;
};
constexpr int UGB_SAMPLE_VOCAB_MAX = 1 << 18;
int32_t ugb_sample_rows(ugb_device *dev, const ugb_sample_args &a);
