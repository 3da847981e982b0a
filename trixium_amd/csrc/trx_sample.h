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
  // A decode position's call (one row; null otherwise): nothing while *gate_pos < *gate_from; u is the next
  // number of the xorshift32 stream at rng, as the firmware's sampler draws it (firmware/infer.c:456-466),
  // but on a row that takes the largest logit; the token replaces the argmax in *slot.
  const int* gate_pos;
  const int* gate_from;
  uint32_t* rng;
  unsigned long long* slot;
  // Set by the launcher.
  int chunk, chunks, frac;     // logits a block; blocks a row; fractional bits of a mass
  int part, parts;             // logits a part of a chunk; parts a chunk
};

const char* sample_rows_refuses(int n, int vocab);
size_t sample_rows_work_bytes(int n, int vocab);
int launch_sample_rows(const SampleRowsParams& p, hipStream_t s);

// The logits with the repetition penalty (firmware/infer.c:395-412: above zero divided, else multiplied)
// on the tokens of the last `window` positions, into out. Nothing while *pos < *head_from.
struct PenaltyParams {
  const float* logits;
  float* out;
  int vocab, window;
  const int* pos;
  const int* head_from;
  const int* tokens;           // the positions' tokens: position p at p % ring
  int ring;
  const float* repetition;
};
int launch_penalty(const PenaltyParams& p, hipStream_t s);

}  // namespace trx
