// Attention of the next n positions with a sliding window and sinks over a KV ring
// (trx_attn_window.hip): parameter block and launcher, for the public entry point and the prefill
// past the window.
#pragma once

#include "trx_internal.h"

namespace trx {

// Position p of the ring takes slot p where p < pin, else pin + (p - pin) % (slots - pin). A query at
// position t sees u <= t with u < sinks or u > t - window (sinks <= pin, window <= slots - pin). The
// rows of positions below pos come from the ring, those of pos .. pos + n - 1 from k and v, which
// take their slots after every query has read the old ones.
struct AttnWindowParams {
  bool half_io;                // q, gate and out in fp16 (else fp32)
  const void* q;               // [n][q_stride], head h at h * hd
  const void* gate;            // [n][gate_stride], head h at h * gate_head_stride (or null)
  void* out;                   // [n][out_stride], head h at h * hd
  const __half* k;             // [n][kv_stride], kv head g at g * hd
  const __half* v;
  __half* kcache;              // [n_kv][slots][hd]
  __half* vcache;
  const int* pos_dev;          // the first position on the device, or null: pos
  int pos, n;
  int n_head, n_kv, hd, slots, pin, window, sinks;
  int q_stride, kv_stride, out_stride, gate_stride, gate_head_stride;
  float scale;
  void* work;                  // attn_window_work_bytes (null where the call splits no keys)
  // Set by the launcher.
  int rep, nsplit, cols;       // heads a kv head; splits of the keys; n * rep
  unsigned long long rep_m;    // for the division by rep: a product with rep_m, shifted by rep_s
  int rep_s;
};

// Why a geometry is not taken (null: it is).
const char* attn_window_refuses(const AttnWindowParams& p);
// Bytes that any call of up to p.n positions needs; and whether the one of p.n needs any.
size_t attn_window_work_bytes(const AttnWindowParams& p);
bool attn_window_splits(const AttnWindowParams& p);
int launch_attn_window(const AttnWindowParams& p, hipStream_t s);

}  // namespace trx
