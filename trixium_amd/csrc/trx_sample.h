// Sampling from the whole vocabulary (trx_sample.hip): parameter block and launcher, for the public
// entry point and the decoder's step.
#pragma once

#include "trx_internal.h"

namespace trx {

struct SampleRowsParams {
  const void* logits;          // [n][ld], fp32 or fp16
  bool half;
  int n, vocab;
  long long ld;
  const trx_sampling* rows;    // [n], or one for every row
  bool per_row;
  const float* u;              // [n]
  int32_t* tokens;             // [n]
  float* logp;                 // [n] or null
  void* work;                  // sample_rows_work_bytes
  // Set by the launcher.
  int chunk, chunks, frac;     // logits a block; blocks a row; fractional bits of a mass
};

const char* sample_rows_refuses(int n, int vocab);
size_t sample_rows_work_bytes(int n, int vocab);
int launch_sample_rows(const SampleRowsParams& p, hipStream_t s);

}  // namespace trx
