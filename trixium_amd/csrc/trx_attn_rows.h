// Attention over caches whose rows stand one behind the other (trx_attn_rows.hip): a batch of drafts
// behind a prefix that they share, and one sequence whose rows add up the probabilities they get.
#pragma once

#include "trx_internal.h"

namespace trx {

// New row i of draft b (row b n + i of q, k, v, gate and out) sees the prefix, the rows of the draft's
// tail and the draft's new rows 0 .. i, which take the tail's next slots. A draft with a length or a
// count out of range takes no part.
struct AttnRowsParams {
  bool half_io;                // q, gate and out in fp16 (else fp32)
  const void* q;               // [batch * n][q_stride], head h at h * hd
  const void* gate;            // [batch * n][gate_stride], head h at h * gate_head_stride (or null)
  void* out;                   // [batch * n][out_stride], head h at h * hd
  const __half* k;             // [batch * n][kv_stride], kv head g at g * hd
  const __half* v;
  const __half* kprefix;       // [n_kv][prefix_slots][hd], the first `prefix` rows
  const __half* vprefix;
  __half* ktail;               // [batch][n_kv][tail_slots][hd]
  __half* vtail;
  const int* lengths;          // rows of each tail, on the device, or null: length
  const int* counts;           // new rows of each draft, on the device, or null: n
  int batch, n, prefix, length;
  int n_head, n_kv, hd, prefix_slots, tail_slots;
  int q_stride, kv_stride, out_stride, gate_stride, gate_head_stride;
  float scale;
  // One sequence with masses (mass not null): its rows are the one tail.
  float* mass;                 // [n_kv][tail_slots]
  int* positions;              // [n_kv][tail_slots]
  const int* state;            // {length, pos} on the device, or null
  int pos;                     // of the first new row
  void* work;                  // attn_rows_work_bytes, with masses attn_mass_work_bytes behind them
  // Set by the launcher.
  int rep, nsplit, cols;       // heads a kv head; parts of a column's keys; batch * n * rep
  unsigned long long rep_m;    // for the division by rep: a product with rep_m, shifted by rep_s
  int rep_s;
  int prefix_splits, tail_splits;
  int prefix_blocks;           // of this launch, before the tails' blocks
  int prefix_cb, tail_cb;      // column blocks of the batch and of a draft
  float* scores;               // [n_kv][cols][score_ld], powers of two, of calls with masses that keep them
  long long score_ld;
  float4* norms;               // [n_kv][cols]: a probability is 2^(z raw score - x) y
  float* partial;              // [parts][kv head and block of keys][128], sums of a part of the columns
  void* planes;                // the queries as operands, of calls of many columns with masses
};

// Why a geometry is not taken (null: it is), and why not for a sequence with masses.
const char* attn_rows_refuses(const AttnRowsParams& p);
const char* attn_mass_refuses(const AttnRowsParams& p);
// Bytes that any call of up to p.batch drafts, p.n new rows and p.prefix prefix rows needs.
size_t attn_rows_work_bytes(const AttnRowsParams& p);
// And what a sequence with masses needs besides.
size_t attn_mass_work_bytes(const AttnRowsParams& p);
int launch_attn_rows(const AttnRowsParams& p, hipStream_t s);

}  // namespace trx
