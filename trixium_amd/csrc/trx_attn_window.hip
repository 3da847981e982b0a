// Attention of the next n positions over a KV ring, with a sliding window and a few first positions
// that stay visible (sinks). A query at position t sees V(t) = {u <= t : u < sinks or u > t - window}:
//   o_t = sum_{u in V(t)} e^{scale q_t.k_u - m} v_u / sum_{u in V(t)} e^{scale q_t.k_u - m},
// m the largest score, one pass over the keys with a running maximum and sum.
//
// Columns: a (position, head of the kv head) pair each, 32 a wave, so the heads that share K and V
// read them once. Many columns (attn_window_kernel): a block takes WQ waves of columns times WK waves of
// keys; every stage of WK * 32 keys goes into LDS once, the WK waves of a column take 32 of them each, and
// are joined at the end. Few columns (attn_window_few_kernel): the keys are the long axis, split over the
// four waves of a block. Either way the keys may be split over blocks, joined by attn_window_finish.
// The keys any query of the block sees are numbered in order (the sinks, then the window from the
// first query's on): tiles of that numbering never hold rows outside it, whatever the ring's seam.
//
// Products on the matrix cores (v_mfma_f32_32x32x16_f16), K and V as the ring holds them:
//   S^T = K Q^T: fp32 queries enter as two fp16 planes of q * 2^e (e per query: the largest element
//   below 2^14), so a score is the fp32 dot product to 2^-22; fp16 queries as they are.
//   O^T += V^T P^T: P^T stands in the score registers in the operand's layout but for the order of
//   the keys, which V^T, read transposed from LDS, follows. P in two fp16 planes (2^-22), but in one for
//   fp16 outputs of many columns: 2^-11 a probability at most, as the output's own rounding, independent
//   from key to key (against 64 bits 2.9e-4 of the result's norm, 2.1e-4 with two planes). The second plane
//   is a third of the products: 1021 positions x 32 heads of 128 over 6000 keys 130 us with one, 164 with two;
//   one position over 32768 keys 35.1 and 35.6.
// Probabilities are 2^(s - r + 7) against a reference r that follows the running maximum only where
// that exceeds it by 2^8: at most 2^15 (finite in fp16), and those that vanish in fp16 are below 2^-32
// of the largest.

#include "trx_attn_window.h"
#include "trx_attn_tile.h"

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <limits.h>

namespace trx {
// The first position, and whether the call has positions that the ring's arithmetic holds.
__device__ __forceinline__ bool aw_pos(const AttnWindowParams& p, int& pos) {
  pos = p.pos_dev ? *p.pos_dev : p.pos;
  return pos >= 0 && pos <= INT_MAX - p.n;
}

// What the waves of a block know of their work: the call's first position and the block's keys, numbered
// x in [0, N): position x below ns (the sinks), else x - ns + lo.
struct AwBlock {
  int pos, g, sp, c0, end;     // first position; kv head; split; first column and that behind the last
  int split, splits;           // of the keys
  int t_first, t_last, ns, lo, N;
  int ub, roff, R;             // ring: position u >= ub stands at offset roff + u - ub, modulo R
};

__device__ __forceinline__ AwBlock aw_block(const AttnWindowParams& p, int pos, int columns) {
  AwBlock b;
  b.pos = pos;
  // A kv head's blocks stay on the XCDs of its number (blocks go round-robin over them): its K and V
  // are read into few L2s.
  const unsigned cb = blockIdx.x / (unsigned)p.n_kv;
  b.g = (int)(blockIdx.x - cb * p.n_kv);
  b.sp = b.split = blockIdx.y;
  b.splits = p.nsplit;
  b.c0 = (int)cb * columns;
  b.end = p.cols;
  b.t_first = pos + aw_row(p, b.c0);
  b.t_last = pos + aw_row(p, min(b.c0 + columns - 1, p.cols - 1));
  b.ns = min(p.sinks, b.t_last + 1);
  b.lo = max(b.ns, b.t_first - p.window + 1);
  b.N = b.ns + (b.t_last + 1 - b.lo);
  b.R = p.slots - p.pin;
  b.ub = max(b.lo, p.pin);
  b.roff = (int)((unsigned)(b.ub - p.pin) % (unsigned)b.R);
  return b;
}

// Where K and V rows of a block's keys lie: in the ring, or among the call's own rows.
template <int HD>
struct AwRows {
  const char *kc, *vc;         // the ring's rows of the kv head
  long long kd, vd;            // from there to the call's own rows
  int kv_stride, pin;

  __device__ __forceinline__ AwRows(const AttnWindowParams& p, const AwBlock& b) : kv_stride(p.kv_stride), pin(p.pin) {
    const int g = b.g;
    kc = (const char*)(p.kcache + (size_t)g * p.slots * HD);
    vc = (const char*)(p.vcache + (size_t)g * p.slots * HD);
    kd = (const char*)(p.k + g * HD) - kc;
    vd = (const char*)(p.v + g * HD) - vc;
  }
  // Byte distance of key x's row from the ring's rows (past the last key: that key again, masked), and
  // all ones if it is one of the call's own.
  __device__ __forceinline__ long long row(const AwBlock& b, int x, long long& fresh) const {
    x = min(x, b.N - 1);
    const int u = x < b.ns ? x : x - b.ns + b.lo;
    const int ro = b.roff + (u - b.ub);               // u - ub < window <= R
    const int slot = u < pin ? u : pin + (ro >= b.R ? ro - b.R : ro);
    const bool own = u >= b.pos;
    fresh = own ? -1 : 0;
    return 2ll * (own ? u - b.pos : slot) * (own ? kv_stride : HD);
  }
  // How many runs of `count` keys from key x0 on lie evenly spaced (uniform); with one at least, the first
  // one's distance and the step in bytes.
  __device__ __forceinline__ int flat(const AwBlock& b, int x0, int count, long long& at, bool& own, uint32_t& step) const {
    if (x0 < b.ns || x0 >= b.N) return 0;
    const int u0 = x0 - b.ns + b.lo;
    if (u0 < pin) return 0;
    int ro = b.roff + (u0 - b.ub);
    ro = ro >= b.R ? ro - b.R : ro;
    own = u0 >= b.pos;
    step = 2u * (uint32_t)(own ? kv_stride : HD);
    at = own ? 2ll * (u0 - b.pos) * kv_stride : 2ll * (pin + ro) * HD;
    return (own ? b.t_last + 1 - u0 : min(b.pos - u0, b.R - ro)) / count;
  }
};

// The column of a lane (32 a wave, lanes j and j + 32 the same): a position and a head of kv head g.
struct AwColumn {
  int row, head, t;            // row: the position's index in the call; t: the position
  int w_first, w_last;         // positions of the wave's columns

  __device__ __forceinline__ AwColumn(const AttnWindowParams& p, const AwBlock& b, int first, int j) {
    const int last = p.cols - 1, col = min(first + j, last);
    row = aw_row(p, col);
    head = b.g * p.rep + (col - row * p.rep);
    t = b.pos + row;
    w_first = b.pos + aw_row(p, min(first, last));
    w_last = b.pos + aw_row(p, min(first + 31, last));
  }
};
// The ring as a layout of the keys (trx_attn_tile.h).
template <int HD>
struct AwRing {
  using Params = AttnWindowParams;
  using Block = AwBlock;
  using Rows = AwRows<HD>;
  using Column = AwColumn;
  static constexpr bool TWO = false;

  __device__ __forceinline__ static bool block(const Params& p, int columns, Block& b) {
    int pos;
    if (!aw_pos(p, pos)) return false;
    b = aw_block(p, pos, columns);
    return true;
  }
  // Whether the column sees key x.
  __device__ __forceinline__ static auto sight(const Params& p, const Block& b, const Column& c) {
    // last: the number of the column's own position; key x is last - x before it.
    return [ns = b.ns, t = c.t, last = c.t - b.lo + b.ns, window = p.window](int x) AW_INLINE {
      return x < ns ? x <= t : (unsigned)(last - x) < (unsigned)window;
    };
  }
  // Whole stages are [a0, a1) of those whose wave takes keys SR st + own .. + 31; the others are at the sinks and
  // at both ends of the window.
  __device__ __forceinline__ static void whole(const Params& p, const Block& b, const Column& c, int own, int SR, int& a0, int& a1) {
    const int first = own - b.ns + b.lo;           // position of stage st's first key of the wave: first + SR st
    a0 = (max(b.lo, c.w_last - p.window + 1) - first + SR - 1) / SR;
    a1 = c.w_first + 1 - kAwKeys < first ? 0 : (c.w_first + 1 - kAwKeys - first) / SR + 1;
  }
  __device__ __forceinline__ static bool all_see(const Params& p, const Block& b, const Column& c, int x0) {
    const int u0 = x0 - b.ns + b.lo;
    return x0 >= b.ns && u0 > c.w_last - p.window && u0 <= c.w_first - (kAwKeys - 1);
  }
  __device__ __forceinline__ static size_t sum_at(const Params&, const Block&, int, size_t at) { return at; }
  __device__ __forceinline__ static void query(const Params&, const Block&, int, int, int, const half8_t&, const half8_t&, float) {}
  __device__ __forceinline__ static void scored(const Params&, const Block&, int, int, const f32x16_t&, float) {}
  __device__ __forceinline__ static void total(const Params&, const Block&, int, const float2&) {}
};

template <int HD, bool HALF, int WQ, int WK, int D>
__global__ __launch_bounds__(64 * WQ * WK, WQ * WK / 4) void attn_window_kernel(AttnWindowParams p) {
  aw_many<AwRing<HD>, HD, HALF, WQ, WK, D>(p);
}

template <int HD, bool HALF>
__global__ __launch_bounds__(256, 1) void attn_window_few_kernel(AttnWindowParams p) {
  aw_few<AwRing<HD>, HD, HALF>(p);
}

// The splits of a (position, head) joined by one wave.
template <int HD, bool HALF>
__device__ __forceinline__ void aw_join(const AttnWindowParams& p, int row, int head, int lane) {
  constexpr int E = HD / 64;                       // dims a lane: E lane .. + E - 1
  const int g = aw_row(p, head), col = row * p.rep + head - g * p.rep;
  const size_t all = (size_t)p.nsplit * p.n_kv * p.cols, step = (size_t)p.n_kv * p.cols;
  const size_t at = (size_t)g * p.cols + col;
  const float2* ml = (const float2*)((const float*)p.work + all * HD) + at;
  const float* po = (const float*)p.work + at * HD + E * lane;
  const size_t gi = (size_t)row * p.gate_stride + (size_t)head * p.gate_head_stride + E * lane;
  const size_t oi = (size_t)row * p.out_stride + (size_t)head * HD + E * lane;
  typedef typename std::conditional<HALF, _Float16, float>::type io_t;
  io_t gate[E], out[E];
  if (p.gate) __builtin_memcpy(gate, (const io_t*)p.gate + gi, sizeof gate);
  float M = -INFINITY, l = 0.f, o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = 0.f;
  // Eight splits' loads at a time in flight (the gate's with them), a running reference over the eights.
  for (int s0 = 0; s0 < p.nsplit; s0 += 8) {
    float2 a[8];
    float x[8][E];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      a[k] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int i = 0; i < E; ++i) x[k][i] = 0.f;
      if (s0 + k < p.nsplit) {
        a[k] = ml[(s0 + k) * step];
        __builtin_memcpy(x[k], po + (s0 + k) * step * HD, 4 * E);
      }
    }
    float top = M;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, a[k].x);
    const float keep = aw_rescale(M, top);
    M = top;
    l *= keep;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] *= keep;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float f = aw_rescale(a[k].x, M);
      l += a[k].y * f;
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] += x[k][i] * f;
    }
  }
  const float inv = 1.0f / l;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float v = o[i] * inv;
    out[i] = (io_t)(p.gate ? v * sigmoidf_((float)gate[i]) : v);
  }
  __builtin_memcpy((io_t*)p.out + oi, out, sizeof out);
}

// After the attention: the splits of each (position, head) joined (a wave each, blocks of four), and
// the call's last rows of K and V into their slots.
template <int HD, bool HALF>
__global__ __launch_bounds__(256) void attn_window_finish(AttnWindowParams p, int join_blocks) {
  int pos;
  if (!aw_pos(p, pos)) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if ((int)blockIdx.x < join_blocks) {
    const unsigned id = blockIdx.x * 4 + w;         // below 2^25 + 4
    if (id >= (unsigned)(p.n * p.n_head)) return;
    const int row = (int)(id / (unsigned)p.n_head);
    aw_join<HD, HALF>(p, row, (int)id - row * p.n_head, lane);
    return;
  }
  // Rows pos .. pos + n - 1, 16 bytes of K and V a thread. A ring row that a later row of the call
  // replaces is left out.
  constexpr int SEG = HD / 8;
  const int R = p.slots - p.pin;
  const long long id = (long long)(blockIdx.x - join_blocks) * 256 + threadIdx.x;
  const long long pieces = (long long)p.n * p.n_kv * SEG;
  if (id >= pieces) return;
  const unsigned at = (unsigned)(id / SEG);        // below 2^25
  const int sd = (int)(id % SEG) * 8, r = (int)(at / (unsigned)p.n_kv), g = (int)at - r * p.n_kv, u = pos + r;
  if (u >= p.pin && p.n - r > R) return;
  const int slot = u < p.pin ? u : p.pin + (int)((unsigned)(u - p.pin) % (unsigned)R);
  const size_t to = ((size_t)g * p.slots + slot) * HD + sd, from = (size_t)r * p.kv_stride + (size_t)g * HD + sd;
  *(uint4*)(p.kcache + to) = *(const uint4*)(p.k + from);
  *(uint4*)(p.vcache + to) = *(const uint4*)(p.v + from);
}
// Launch ------------------------------------------------------------------------------------------

constexpr int kAwCus = 256;
constexpr int kAwMaxSplits = 64;

// How a call is cut: columns a block (in waves of 32; 1: the kernel for few columns) and splits of the keys.
struct AwPlan {
  int wq, nsplit;
};

// The cut that takes the least time by this estimate in microseconds. A block takes a fixed part (its queries, the
// first rows' latency, the join of its waves, the outputs) and a step for each wk tiles of keys; a full chip
// makes a step 1.4 times as long; splits write and read their sums once at 3 TB/s. Measured (us, by wq and
// splits), the choice first:
//   27 positions over 4061 keys, 32 heads of 128, 8 kv heads: (1, 8) 20; (1, 6) 23, (2, 16) 23, (4, 32) 25, (1, 1) 68
//   200 of them: (4, 4) 51; (2, 2) 53, (2, 4) 61, (1, 1) 71
//   1024 over windows of 2048: (4, 1) 85; (4, 2) 105, (2, 1) 115, (1, 1) 155
//   509 over up to 1209 keys, 24 heads of 256, 4 kv heads: (4, 2) 70; (4, 4) 78, (2, 1) 88, (1, 1) 93, (4, 1) 103
//   1 over 32768 keys, fp16 queries: (1, 32) 32; (1, 24) 34, (2, 32) 36, (1, 1) 437
//   1 over 1024 keys, 16 heads: (1, 8) 12; (1, 16) 13, (1, 4) 14, (1, 1) 24
static AwPlan aw_plan(const AttnWindowParams& p, long long pos, int most) {
  const int rep = p.n_head / p.n_kv, cols = p.n * rep;
  AwPlan best = {1, 1};
  double least = 1e300;
  for (int wq : {1, 2, 4}) {
    const int wk = wq == 1 ? 4 : (p.hd == 256 ? 4 : 8) / wq;
    const double fixed = wq == 1 ? 2 : 11;
    // A few-columns step waits for its own rows. Of the others' the matrix products are the larger part (two
    // planes of queries and probabilities with fp32); wq = 2 has one stage less on the way.
    const double unit = wq == 1 ? p.hd / 64.0 : 1.35 * (p.half_io ? 0.56 : 1.0) * (p.hd == 64 ? 0.6 : 1.0);
    const double step = wq == 2 ? unit * (p.half_io ? 1.75 : p.hd == 256 ? 1.7 : 1.3) : unit;
    const long long span = std::min<long long>(p.n, (32 * wq + rep - 1) / rep + 1);
    const long long keys = std::min<long long>((long long)p.sinks + p.window + span - 1, pos + p.n);
    const int tiles = (int)((keys + kAwKeys - 1) / kAwKeys), blocks = cdiv(cols, 32 * wq) * p.n_kv;
    for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
      if (s > most || s > tiles) break;
      const int steps = cdiv(cdiv(tiles, s), wk);
      const double full = (double)blocks * s / kAwCus;
      // (Between whole rounds of blocks and none wasted: blocks at a chunk's ends are shorter.)
      const double rounds = full <= 1 ? 1 : 0.5 * (full + std::ceil(full));
      const double t = rounds * (fixed + steps * step * (1 + 0.4 * std::min(full, 1.0))) +
                       (s > 1 ? 2 + 8.0 * s * p.n * p.n_head * p.hd / 3e6 : 0);
      if (t < least) least = t, best = {wq, s};
    }
  }
  return best;
}

const char* attn_window_refuses(const AttnWindowParams& p) {
  if (p.hd != 64 && p.hd != 128 && p.hd != 256) return "head_dim is not 64, 128 or 256";
  if (p.n_kv < 1 || p.n_head < 1 || p.n_head % p.n_kv) return "n_head is not a multiple of n_kv_head";
  if (p.n_head > 1024) return "more than 1024 heads";
  if (p.slots > 1 << 30) return "more than 2^30 slots";
  if (p.pin < 0 || p.slots <= p.pin) return "pin outside [0, slots)";
  if (p.sinks < 0 || p.sinks > p.pin) return "sinks outside [0, pin]";
  if (p.window < 1 || p.window > p.slots - p.pin) return "window outside [1, slots - pin]";
  // (The second kernel's threads, up to 64 a position and head, stay below a grid's 2^32.)
  if (p.n < 0 || (long long)p.n * p.n_head > (1 << 25)) return "too many positions";
  if (!(p.scale > 0.f && p.scale < INFINITY)) return "scale is not positive and finite";
  const int q4 = p.half_io ? 8 : 4, o4 = 4;
  if (p.q_stride < p.n_head * p.hd || p.q_stride % q4) return "q_stride";
  if (p.kv_stride < p.n_kv * p.hd || p.kv_stride % 8 || p.kv_stride > 1 << 22) return "kv_stride";
  if (p.out_stride < p.n_head * p.hd || p.out_stride % o4) return "out_stride";
  if (p.gate && (p.gate_head_stride < p.hd || p.gate_head_stride % o4 || p.gate_stride % o4 ||
                 p.gate_stride < (long long)(p.n_head - 1) * p.gate_head_stride + p.hd))
    return "gate strides";
  return nullptr;
}

// Lengths in steps of 1/64 to 1/32 of them (of one below 64). A call takes at most as many split positions, n times
// the splits, as the calls at both ends of its step would at the step's last length: so the workspace of a length
// holds that of every shorter one (the splits fall as n grows, and with them, here and there, the bytes). Of 1.3
// million calls (1 to 9000 positions, windows of 30 to 131068, 1 to 128 heads) that takes splits from 424, by the
// estimate at most 1% slower for it.
static int aw_step(int n) {
  int step = 1;
  while (64ll * step <= n) step *= 2;
  return step;
}
static long long aw_split_positions(AttnWindowParams p, int first, int step) {
  int s = 1;
  for (int n : {first, first + step - 1}) {
    p.n = n;
    s = std::max(s, aw_plan(p, LLONG_MAX / 2, kAwMaxSplits).nsplit);
  }
  return s > 1 ? (long long)s * (first + step - 1) : 0;
}
// The cut of a call whose windows are full.
static AwPlan aw_full_plan(const AttnWindowParams& p) {
  const AwPlan plan = aw_plan(p, LLONG_MAX / 2, kAwMaxSplits);
  const int step = aw_step(p.n);
  if (step == 1 || plan.nsplit == 1) return plan;
  const long long most = aw_split_positions(p, p.n / step * step, step) / p.n;
  return plan.nsplit <= most ? plan : aw_plan(p, LLONG_MAX / 2, (int)std::max(most, 1ll));
}

// Of any call of up to n positions.
size_t attn_window_work_bytes(const AttnWindowParams& p) {
  long long most = 0;
  for (int n = 1; n <= p.n; n += aw_step(n)) most = std::max(most, aw_split_positions(p, n, aw_step(n)));
  return (size_t)most * p.n_head * (p.hd + 2) * 4;
}
bool attn_window_splits(const AttnWindowParams& p) { return p.n > 0 && aw_full_plan(p).nsplit > 1; }

template <int HD, bool HALF>
static int aw_launch(const AttnWindowParams& p, int wq, hipStream_t s) {
  constexpr int WT = HD == 256 ? 4 : 8;              // waves of the kernel for many columns
  const dim3 grid(cdiv(p.cols, 32 * wq) * p.n_kv, p.nsplit);
  if (wq == 1) hipLaunchKernelGGL((attn_window_few_kernel<HD, HALF>), grid, dim3(256), 0, s, p);
  else if (wq == 2) hipLaunchKernelGGL((attn_window_kernel<HD, HALF, 2, WT / 2, HD == 64 ? 2 : 1>), grid, dim3(64 * WT), 0, s, p);
  else hipLaunchKernelGGL((attn_window_kernel<HD, HALF, 4, WT / 4, 2>), grid, dim3(64 * WT), 0, s, p);
  TRX_LAUNCHED();
  const int join = p.nsplit > 1 ? (int)(((long long)p.n * p.n_head + 3) / 4) : 0;
  const int append = (int)(((long long)p.n * p.n_kv * (HD / 8) + 255) / 256);
  hipLaunchKernelGGL((attn_window_finish<HD, HALF>), dim3(join + append), dim3(256), 0, s, p, join);
  TRX_LAUNCHED();
  return TRX_OK;
}

int launch_attn_window(const AttnWindowParams& params, hipStream_t s) {
  AttnWindowParams p = params;
  const char* why = attn_window_refuses(p);
  TRX_CHECK(!why, TRX_E_INVALID, "window attention: %s", why);
  if (p.n == 0) return TRX_OK;
  p.rep = p.n_head / p.n_kv;
  p.cols = p.n * p.rep;
  p.rep_s = 32;
  while (1 << (p.rep_s - 32) < p.rep) ++p.rep_s;
  p.rep_m = ((1ull << p.rep_s) + p.rep - 1) / p.rep;
  // The workspace holds the splits of a full window; a ring that is still filling takes no more.
  AwPlan plan = aw_full_plan(p);
  if (!p.pos_dev && p.pos < (long long)p.sinks + p.window) plan = aw_plan(p, p.pos, plan.nsplit);
  p.nsplit = plan.nsplit;
  if (p.half_io) {
    if (p.hd == 64) return aw_launch<64, true>(p, plan.wq, s);
    if (p.hd == 128) return aw_launch<128, true>(p, plan.wq, s);
    return aw_launch<256, true>(p, plan.wq, s);
  }
  if (p.hd == 64) return aw_launch<64, false>(p, plan.wq, s);
  if (p.hd == 128) return aw_launch<128, false>(p, plan.wq, s);
  return aw_launch<256, false>(p, plan.wq, s);
}

}  // namespace trx

using namespace trx;

#define TRX_API extern "C" __attribute__((visibility("default")))

static AttnWindowParams window_params(const trx_attn_window_shape* a, int n) {
  AttnWindowParams p = {};
  p.half_io = a->kind == TRX_KIND_F16;
  p.n = n;
  p.n_head = a->n_head;
  p.n_kv = a->n_kv_head;
  p.hd = a->head_dim;
  p.slots = a->slots;
  p.pin = a->pin;
  p.window = a->window;
  p.sinks = a->sinks;
  p.q_stride = a->q_stride;
  p.kv_stride = a->kv_stride;
  p.out_stride = a->out_stride;
  p.gate_stride = a->gate_stride;
  p.gate_head_stride = a->gate_head_stride;
  p.scale = a->scale;
  return p;
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

TRX_API int trx_attn_window_geometry(const trx_attn_window_shape* shape, int n, size_t* workspace_bytes) {
  TRX_CHECK(shape && workspace_bytes, TRX_E_INVALID, "trx_attn_window_geometry: null argument");
  TRX_CHECK(shape->kind == TRX_KIND_F32 || shape->kind == TRX_KIND_F16, TRX_E_INVALID,
            "trx_attn_window_geometry: kind %d is not F32 or F16", shape->kind);
  const AttnWindowParams p = window_params(shape, n);
  const char* why = attn_window_refuses(p);
  TRX_CHECK(!why, TRX_E_INVALID, "trx_attn_window_geometry: %s", why);
  *workspace_bytes = attn_window_work_bytes(p);
  return TRX_OK;
}

TRX_API int trx_attn_window(const trx_attn_window_shape* shape, int n, int pos, const int32_t* pos_dev, const void* q,
                            const uint16_t* k, const uint16_t* v, uint16_t* kcache, uint16_t* vcache,
                            const void* gate, void* out, void* workspace, trx_stream_t s) {
  TRX_CHECK(shape, TRX_E_INVALID, "trx_attn_window: null shape");
  TRX_CHECK(shape->kind == TRX_KIND_F32 || shape->kind == TRX_KIND_F16, TRX_E_INVALID,
            "trx_attn_window: kind %d is not F32 or F16", shape->kind);
  AttnWindowParams p = window_params(shape, n);
  p.gate = gate;
  const char* why = attn_window_refuses(p);
  TRX_CHECK(!why, TRX_E_INVALID, "trx_attn_window: %s", why);
  TRX_CHECK(pos_dev || (pos >= 0 && pos <= INT_MAX - n), TRX_E_INVALID, "trx_attn_window: position %d", pos);
  if (n == 0) return TRX_OK;
  TRX_CHECK(q && k && v && kcache && vcache && out, TRX_E_INVALID, "trx_attn_window: null argument");
  TRX_CHECK(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(kcache) && aligned16(vcache) && aligned16(gate) &&
            aligned16(out) && aligned16(workspace), TRX_E_INVALID, "trx_attn_window: a pointer is not 16-byte aligned");
  TRX_CHECK(workspace || !attn_window_splits(p), TRX_E_INVALID, "trx_attn_window: null workspace");
  p.q = q;
  p.out = out;
  p.k = (const __half*)k;
  p.v = (const __half*)v;
  p.kcache = (__half*)kcache;
  p.vcache = (__half*)vcache;
  p.pos_dev = pos_dev;
  p.pos = pos;
  p.work = workspace;
  return launch_attn_window(p, (hipStream_t)s);
}
