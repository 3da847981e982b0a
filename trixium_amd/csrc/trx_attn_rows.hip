// Attention over caches whose rows stand one behind the other, on the tiles of trx_attn_tile.h:
// - drafts behind a shared prefix: o = sum_u e^{scale q.k_u - m} v_u / sum_u e^{scale q.k_u - m} over the prefix's
//   rows, the draft's tail and its new rows up to the query's own. The sum splits at the prefix's end: the
//   prefix takes the columns of all drafts together, so that its rows are read once for all of them, a tail those
//   of its draft; the parts (m, the sum behind m, the outputs) are joined by the second launch.
// - one sequence with masses: mass_u += sum of e^{scale q.k_u - m} / sum_u' e^{scale q.k_u' - m} over the positions
//   and heads of the kv head. The final sums have to be there: calls of few columns keep their scores (a column's
//   4 bytes a key, beside the key's 4 hd bytes of K and V) and the second launch adds their probabilities up; of
//   many columns the scores are taken again, keys staying where the columns pass.
// No sum depends on the order of blocks.

#include "trx_attn_plan.h"
#include "trx_attn_rows.h"
#include "trx_attn_tile.h"

#include <algorithm>
#include <type_traits>
#include <limits.h>

namespace trx {

// The rows that sequence seq has and gets; whether it takes part.
__device__ __forceinline__ bool ar_sequence(const AttnRowsParams& p, int seq, int& have, int& fresh) {
  // (Read first: a choice between addresses would put the arguments into memory of the lane's own.)
  have = __builtin_amdgcn_readfirstlane(p.length);
  fresh = __builtin_amdgcn_readfirstlane(p.n);
  if (p.state) have = p.state[0];
  else if (p.lengths) have = p.lengths[seq];
  if (p.counts) fresh = p.counts[seq];
  return have >= 0 && fresh > 0 && fresh <= p.n && have <= p.tail_slots - fresh;
}
__device__ __forceinline__ bool ar_position(const AttnRowsParams& p, int& pos) {
  pos = __builtin_amdgcn_readfirstlane(p.pos);
  if (p.state) pos = p.state[1];
  return pos >= 0 && pos <= INT_MAX - p.n;
}

// A probability is 2^(score - norm.x) norm.y: of a column's reference and the sum behind it.
__device__ __forceinline__ float2 ar_norm(float M, float l) { return make_float2(M - kAwBias, 1.f / l); }

// What the waves of a block know of their work. Keys x below `cached` stand in the cache, the others are new rows.
struct ArBlock {
  int g, sp, c0, end;          // kv head; part; first column and that behind the last
  int split, splits;           // of the keys
  int N, cached, row0, seq;    // keys; the draft's first row
  bool tail;
};

// The column of a lane (32 a wave, lanes j and j + 32 the same): it sees the keys below lim.
struct ArColumn {
  int row, head, lim, w_first; // w_first: the smallest limit of the wave's columns

  __device__ __forceinline__ ArColumn(const AttnRowsParams& p, const ArBlock& b, int first, int j) {
    const int last = b.end - 1, col = min(first + j, last);
    row = aw_row(p, col);
    head = b.g * p.rep + (col - row * p.rep);
    lim = b.tail ? b.cached + row - b.row0 + 1 : b.N;
    w_first = b.tail ? b.cached + aw_row(p, min(first, last)) - b.row0 + 1 : b.N;
  }
};

template <int HD>
struct ArRows {
  const char *kc, *vc;         // the cache's rows of the kv head
  long long kd, vd;            // from there to the call's own rows
  int kv_stride;

  __device__ __forceinline__ ArRows(const AttnRowsParams& p, const ArBlock& b) : kv_stride(p.kv_stride) {
    const size_t at = b.tail ? ((size_t)b.seq * p.n_kv + b.g) * p.tail_slots * HD : (size_t)b.g * p.prefix_slots * HD;
    kc = (const char*)((b.tail ? (const __half*)p.ktail : p.kprefix) + at);
    vc = (const char*)((b.tail ? (const __half*)p.vtail : p.vprefix) + at);
    const size_t own = (size_t)b.row0 * p.kv_stride + (size_t)b.g * HD;
    kd = (const char*)(p.k + own) - kc;
    vd = (const char*)(p.v + own) - vc;
  }
  // Byte distance of key x's row from the cache's rows (past the last key: that key again, masked), and all ones
  // if it is one of the call's own.
  __device__ __forceinline__ long long row(const ArBlock& b, int x, long long& fresh) const {
    x = min(x, b.N - 1);
    const bool own = x >= b.cached;
    fresh = own ? -1 : 0;
    return 2ll * (own ? x - b.cached : x) * (own ? kv_stride : HD);
  }
  // How many runs of `count` keys from key x0 on lie evenly spaced (uniform); with one at least, the first
  // one's distance and the step in bytes.
  __device__ __forceinline__ int flat(const ArBlock& b, int x0, int count, long long& at, bool& own, uint32_t& step) const {
    if (x0 >= b.N) return 0;
    own = x0 >= b.cached;
    step = 2u * (uint32_t)(own ? kv_stride : HD);
    at = own ? 2ll * (x0 - b.cached) * kv_stride : 2ll * x0 * HD;
    return ((own ? b.N : b.cached) - x0) / count;
  }
};

// Rows in a line as a layout of the keys (trx_attn_tile.h).
template <int HD, bool HALF, bool MASS>
struct ArLine {
  using Params = AttnRowsParams;
  using Block = ArBlock;
  using Rows = ArRows<HD>;
  using Column = ArColumn;
  // fp16 calls of many columns take both planes of the probabilities, as those of few: fp16 outputs are the fp32 result
  // rounded, however many drafts share the call (2.1e-4 of the result's norm against 64 bits; 2.9e-4 with one plane). The
  // second one is a third of the products: 64 drafts over 32768 rows 107 us, 95 with one; 1021 positions over 7001 rows 280
  // and 237.
  static constexpr bool TWO = true;

  // A kv head's blocks stay on the XCDs of its number (blocks go round-robin over them), so that the prefix and a
  // sequence's rows are read into few L2s.
  __device__ __forceinline__ static bool block(const Params& p, int columns, Block& b) {
    unsigned i = blockIdx.x, t;
    b.tail = i >= (unsigned)p.prefix_blocks;
    if (!b.tail) {
      t = i / (unsigned)p.n_kv;
      b.g = (int)(i - t * p.n_kv);
      b.splits = p.prefix_splits;
      b.split = b.sp = (int)(t / (unsigned)p.prefix_cb);
      b.c0 = (int)(t - (unsigned)b.split * p.prefix_cb) * columns;
      b.end = p.cols;
      b.seq = b.row0 = 0;
      b.N = b.cached = p.prefix;
      return true;
    }
    i -= p.prefix_blocks;
    t = i / (unsigned)p.n_kv;
    b.g = (int)(i - t * p.n_kv);
    i = t / (unsigned)p.tail_splits;
    b.splits = p.tail_splits;
    b.split = (int)(t - i * p.tail_splits);
    b.sp = p.prefix_splits + b.split;
    b.seq = (int)(i / (unsigned)p.tail_cb);
    const int cb = (int)(i - (unsigned)b.seq * p.tail_cb);
    int fresh, pos;
    if (!ar_sequence(p, b.seq, b.cached, fresh) || (MASS && !ar_position(p, pos))) return false;
    b.cached = __builtin_amdgcn_readfirstlane(b.cached);   // (loaded, so not known to be uniform)
    fresh = __builtin_amdgcn_readfirstlane(fresh);
    b.row0 = b.seq * p.n;
    b.c0 = b.row0 * p.rep + cb * columns;
    b.end = (b.row0 + fresh) * p.rep;
    if (b.c0 >= b.end) return false;
    b.N = b.cached + aw_row(p, min(b.c0 + columns, b.end) - 1) - b.row0 + 1;
    return true;
  }
  // Whether the column sees key x.
  __device__ __forceinline__ static auto sight(const Params&, const Block&, const Column& c) {
    return [lim = c.lim](int x) AW_INLINE { return x < lim; };
  }
  // Whole stages are [a0, a1) of those whose wave takes keys SR st + own .. + 31.
  __device__ __forceinline__ static void whole(const Params&, const Block&, const Column& c, int own, int SR, int& a0, int& a1) {
    a0 = 0;
    a1 = c.w_first - kAwKeys < own ? 0 : (c.w_first - kAwKeys - own) / SR + 1;
  }
  __device__ __forceinline__ static bool all_see(const Params&, const Block&, const Column& c, int x0) {
    return x0 + kAwKeys <= c.w_first;
  }
  // A column's parts beside each other, as the join reads them.
  __device__ __forceinline__ static size_t sum_at(const Params& p, const Block& b, int col, size_t) {
    return ((size_t)b.g * p.cols + col) * p.nsplit + b.sp;
  }
  // Chunk k of a wave's 32 queries as the mass kernel takes them: column block by column block, plane by plane, 16 bytes
  // a lane.
  __device__ __forceinline__ static void query(const Params& p, const Block& b, int first, int lane, int k, const half8_t& hi,
                                               const half8_t& lo, float cs) {
    if (!MASS || !p.planes || b.split || first >= p.cols) return;
    constexpr int NC = HD / 16, ALL = HALF ? NC : 2 * NC;
    half8_t* to = (half8_t*)p.planes + ((size_t)b.g * ((p.cols + 31) / 32) + first / 32) * ALL * 64 + lane;
    to[k * 64] = hi;
    if constexpr (!HALF) to[(NC + k) * 64] = lo;
    if (k == 0 && lane < 32 && first + lane < p.cols) p.norms[(size_t)b.g * p.cols + first + lane].z = cs;
  }
  // A lane's scores of keys x, x + 8, x + 16 and x + 24, four each, in powers of two.
  __device__ __forceinline__ static void scored(const Params& p, const Block& b, int col, int x, const f32x16_t& s, float cs) {
    if (MASS && p.scores) {
      float* to = p.scores + ((size_t)b.g * p.cols + col) * p.score_ld + x;
#pragma unroll
      for (int a = 0; a < 4; ++a)
        *(float4*)(to + 8 * a) = make_float4(s[4 * a] * cs, s[4 * a + 1] * cs, s[4 * a + 2] * cs, s[4 * a + 3] * cs);
    }
  }
  __device__ __forceinline__ static void total(const Params& p, const Block& b, int col, const float2& ml) {
    if constexpr (MASS) *(float2*)(p.norms + (size_t)b.g * p.cols + col) = ar_norm(ml.x, ml.y);
  }
};

// Many columns (aw_many): 256 of 64 fp16 drafts over a prefix of 32768 rows, 8 kv heads of 128, 60 us, 0.86 PFLOP/s with the
// probabilities' two planes counted; a chunk of 1024 fp32 positions over 2900 rows 121 us, 0.94 with both planes of all, of
// 1021 fp16 ones over 7001 rows 196, 0.96; bound as the window attention's chunks.
template <int HD, bool HALF, bool MASS, int WQ, int WK, int D>
__global__ __launch_bounds__(64 * WQ * WK, WQ * WK / 4) void attn_rows_kernel(AttnRowsParams p) {
  aw_many<ArLine<HD, HALF, MASS>, HD, HALF, WQ, WK, D>(p);
}

// Few columns (aw_few): one token over 32700 rows (134 MB) 33 us, 4.1 TB/s, 30 without keeping the scores; the tails of 64
// drafts (131 MB, 0 to 999 rows each) 36. Two blocks a CU up to 128 dims, though a few registers then go to memory: 24
// drafts over 4001 rows 20 us in all, 24 with one block a CU, where the token is as fast.
template <int HD, bool HALF, bool MASS>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void attn_rows_few_kernel(AttnRowsParams p) {
  aw_few<ArLine<HD, HALF, MASS>, HD, HALF>(p);
}

// The parts of a (row, head) joined by one wave: a lane has the reference and the sum of parts lane and lane + 64, so
// that all of a column's loads are on their way at once. A column of a draft that takes no part is not written.
template <int HD, bool HALF, bool MASS>
__device__ __forceinline__ void ar_join(const AttnRowsParams& p, int row, int head, int lane) {
  constexpr int E = HD / 64, MANY = 16;               // dims a lane; parts a time
  typedef typename std::conditional<HALF, _Float16, float>::type io_t;
  const int g = aw_row(p, head), col = row * p.rep + head - g * p.rep, seq = row / p.n;
  int have, fresh;
  const bool takes = ar_sequence(p, seq, have, fresh) && row - seq * p.n < fresh;
  const size_t all = (size_t)p.nsplit * p.n_kv * p.cols, step = (size_t)p.n_kv * p.cols, at = (size_t)g * p.cols + col;
  const float2* ml = (const float2*)((const float*)p.work + all * HD) + at * p.nsplit;
  const float* po = (const float*)p.work + at * HD + E * lane;
  float2 a[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    a[k] = make_float2(-INFINITY, 0.f);
    if (lane + 64 * k < p.nsplit) a[k] = ml[lane + 64 * k];
  }
  io_t gate[E], out[E];
  if (p.gate) __builtin_memcpy(gate, (const io_t*)p.gate + (size_t)row * p.gate_stride + (size_t)head * p.gate_head_stride + E * lane, sizeof gate);
  float x[MANY][E], f[2], o[E] = {};
  auto load = [&](int s0) AW_INLINE {
#pragma unroll
    for (int k = 0; k < MANY; ++k)
      if (s0 + k < p.nsplit) __builtin_memcpy(x[k], po + (size_t)(s0 + k) * step * HD, sizeof x[k]);
  };
  load(0);
  const float M = wave_max(fmaxf(a[0].x, a[1].x));
#pragma unroll
  for (int k = 0; k < 2; ++k) f[k] = aw_rescale(a[k].x, M);
  const float l = wave_sum(a[0].y * f[0] + a[1].y * f[1]);
  for (int s0 = 0;;) {
#pragma unroll
    for (int k = 0; k < MANY; ++k)
      if (s0 + k < p.nsplit) {
        const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(s0 < 64 ? f[0] : f[1]), (s0 + k) & 63));
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] += x[k][i] * w;
      }
    s0 += MANY;
    if (s0 >= p.nsplit) break;
    load(s0);
  }
  if (!takes) return;
  const float inv = 1.0f / l;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float v = o[i] * inv;
    out[i] = (io_t)(p.gate ? v * sigmoidf_((float)gate[i]) : v);
  }
  __builtin_memcpy((io_t*)p.out + (size_t)row * p.out_stride + (size_t)head * HD + E * lane, out, sizeof out);
  if (MASS && lane == 0) *(float2*)(p.norms + at) = ar_norm(M, l);
}

// Few columns: the masses of four keys a thread, from the scores that the attention kept. The columns' parts are joined
// anew by every block: `per` lanes a column.
constexpr int kArMassKeys = 1024;
__device__ __forceinline__ void ar_mass_few(const AttnRowsParams& p, int block, float2* norm) {
  const int kb = block / p.n_kv, g = block - kb * p.n_kv, x0 = kb * kArMassKeys + threadIdx.x;
  const int per = p.cols <= 4 ? 64 : p.cols <= 8 ? 32 : p.cols <= 16 ? 16 : 8, c = (int)threadIdx.x / per, first = threadIdx.x % per;
  // What does not wait for the norms: the first columns' scores and the masses there are (of slots, rows or not).
  constexpr int PRE = 4;
  const float* s = p.scores + (size_t)g * p.cols * p.score_ld;
  float* const m = p.mass + (size_t)g * p.tail_slots;
  float pre[PRE][4], old[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int x = min(x0 + 256 * k, p.tail_slots - 1);
    old[k] = m[x];
#pragma unroll
    for (int i = 0; i < PRE; ++i) pre[i][k] = s[min(i, p.cols - 1) * p.score_ld + x];
  }
  int have, fresh;
  if (!ar_sequence(p, 0, have, fresh)) return;
  const int N = have + fresh;
  if (kb * kArMassKeys >= N) return;
  if (p.nsplit > 1) {
    const size_t all = (size_t)p.nsplit * p.n_kv * p.cols;
    const float2* ml = (const float2*)((const float*)p.work + all * p.hd) + ((size_t)g * p.cols + min(c, p.cols - 1)) * p.nsplit;
    float M = -INFINITY, l = 0.f;
    for (int s0 = first; s0 < p.nsplit; s0 += 8 * per) {
      float2 a[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) a[k] = s0 + k * per < p.nsplit ? ml[s0 + k * per] : make_float2(-INFINITY, 0.f);
      float to = M;
#pragma unroll
      for (int k = 0; k < 8; ++k) to = fmaxf(to, a[k].x);
      l *= aw_rescale(M, to);
      M = to;
#pragma unroll
      for (int k = 0; k < 8; ++k) l += a[k].y * aw_rescale(a[k].x, M);
    }
    for (int o = 1; o < per; o <<= 1) {
      const float m1 = __shfl_xor(M, o, 64), l1 = __shfl_xor(l, o, 64), to = fmaxf(M, m1);
      l = l * aw_rescale(M, to) + l1 * aw_rescale(m1, to);
      M = to;
    }
    if (first == 0 && c < p.cols) norm[c] = ar_norm(M, l);
  } else if (first == 0 && c < p.cols) {
    norm[c] = *(const float2*)(p.norms + (size_t)g * p.cols + c);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int x = x0 + 256 * k;
    if (x >= N) return;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < PRE; ++i)
      if (i < p.cols) sum = fmaf(__builtin_amdgcn_exp2f(pre[i][k] - norm[i].x), norm[i].y, sum);
#pragma unroll 4
    for (int i = PRE; i < p.cols; ++i) sum = fmaf(__builtin_amdgcn_exp2f(s[i * p.score_ld + x] - norm[i].x), norm[i].y, sum);
    m[x] = x < have ? old[k] + sum : sum;
  }
}

// Up to 256 columns: the masses of 64 keys a block, each wave a quarter of the columns, the columns' parts joined by a thread
// each. A block of columns has left scores of the keys that it sees alone.
__device__ __forceinline__ void ar_mass_some(const AttnRowsParams& p, int block, float2* norm, float* part) {
  const int kb = block / p.n_kv, g = block - kb * p.n_kv, lane = threadIdx.x & 63, w = threadIdx.x >> 6, x = kb * 64 + lane;
  int have, fresh;
  if (!ar_sequence(p, 0, have, fresh)) return;
  const int N = have + fresh, c = threadIdx.x;
  if (kb * 64 >= N) return;
  if (c < p.cols) {
    if (p.nsplit > 1) {
      const size_t all = (size_t)p.nsplit * p.n_kv * p.cols;
      const float2* ml = (const float2*)((const float*)p.work + all * p.hd) + ((size_t)g * p.cols + c) * p.nsplit;
      float M = -INFINITY, l = 0.f;
      for (int s0 = 0; s0 < p.nsplit; s0 += 8) {
        float2 a[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) a[k] = s0 + k < p.nsplit ? ml[s0 + k] : make_float2(-INFINITY, 0.f);
        float to = M;
#pragma unroll
        for (int k = 0; k < 8; ++k) to = fmaxf(to, a[k].x);
        l *= aw_rescale(M, to);
        M = to;
#pragma unroll
        for (int k = 0; k < 8; ++k) l += a[k].y * aw_rescale(a[k].x, M);
      }
      norm[c] = ar_norm(M, l);
    } else {
      norm[c] = *(const float2*)(p.norms + (size_t)g * p.cols + c);
    }
  }
  __syncthreads();
  const float* s = p.scores + (size_t)g * p.cols * p.score_ld + min(x, p.tail_slots - 1);
  float sum = 0.f;
#pragma unroll 8
  for (int i = w; i < p.cols; i += 4) {
    const float e = fmaf(__builtin_amdgcn_exp2f(s[i * p.score_ld] - norm[i].x), norm[i].y, sum);
    sum = x <= have + aw_row(p, i) ? e : sum;
  }
  part[64 * w + lane] = sum;
  __syncthreads();
  if (w || x >= N) return;
  sum = part[lane] + part[64 + lane] + part[128 + lane] + part[192 + lane];
  float* m = p.mass + (size_t)g * p.tail_slots + x;
  *m = x < have ? *m + sum : sum;
}

// After the attention: the parts of each (row, head) joined (a wave each, blocks of four), the new rows into the
// tails' slots, and the masses of calls of few columns. Bound by latency: 13 parts of 24 drafts 4 us, 17 of 64 drafts 7 (18
// MB of parts), one token's 32 parts and 32700 masses of 8 kv heads 6.
template <int HD, bool HALF, bool MASS>
__global__ __launch_bounds__(256) void attn_rows_finish(AttnRowsParams p, int mass_blocks, int join_blocks) {
  __shared__ float2 norm[MASS ? kArMassColumns : 1];
  __shared__ float part[MASS ? 256 : 1];
  int pos = 0;
  if (MASS && !ar_position(p, pos)) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  // (First, so that a kv head's masses are added up on the XCD that has its scores.)
  if (MASS && (int)blockIdx.x < mass_blocks) {
    if (p.cols <= 32) ar_mass_few(p, blockIdx.x, norm);
    else ar_mass_some(p, blockIdx.x, norm, part);
    return;
  }
  const int block = (int)blockIdx.x - mass_blocks;
  if (block < join_blocks) {
    const unsigned id = block * 4 + w;              // below 2^23 + 4
    if (id >= (unsigned)(p.batch * p.n * p.n_head)) return;
    const int row = (int)(id / (unsigned)p.n_head);
    ar_join<HD, HALF, MASS>(p, row, (int)id - row * p.n_head, lane);
    return;
  }
  // 16 bytes of K and V a thread.
  constexpr int SEG = HD / 8;
  const long long id = (long long)(block - join_blocks) * 256 + threadIdx.x;
  if (id >= (long long)p.batch * p.n * p.n_kv * SEG) return;
  const unsigned at = (unsigned)(id / SEG);          // below 2^23
  const int sd = (int)(id % SEG) * 8, row = (int)(at / (unsigned)p.n_kv), g = (int)at - row * p.n_kv, seq = row / p.n;
  const int i = row - seq * p.n;
  int have, fresh;
  if (!ar_sequence(p, seq, have, fresh) || i >= fresh) return;
  const size_t slot = ((size_t)seq * p.n_kv + g) * p.tail_slots + have + i;
  const size_t from = (size_t)row * p.kv_stride + (size_t)g * HD + sd;
  *(uint4*)(p.ktail + slot * HD + sd) = *(const uint4*)(p.k + from);
  *(uint4*)(p.vtail + slot * HD + sd) = *(const uint4*)(p.v + from);
  if (MASS && sd == 0) p.positions[slot] = pos + i;
}

// Many columns: the scores once more, with the keys' rows in registers (KT tiles of 32 a wave) while the columns pass
// through LDS, 32 for each of CG groups of KW waves a step; a lane adds up its column's probabilities of its keys,
// lanes and groups are added at the end. (Columns that stayed while the keys passed would have to add up each key over
// the lanes.) The queries come as the attention left them, in operands' order, so that a step's bytes come straight
// into LDS and are read in a row. Eight waves, two a SIMD: the matrix instructions of one run beside the exponentials
// of both. Of 1024 fp32 positions of 32 heads of 128 over 2900 rows 65 us, 0.88 PFLOP/s with both planes counted, of
// 1021 fp16 ones over 7001 rows 84 us (four matrix instructions take a SIMD 66 ns, so that 28 and 31 us would be all of
// them without a pause); without the loads 9 and 12 us less. Scores and exponentials one after the other took 14 and
// 21 us more, masks in the loop 5 and 2.
constexpr int kArMassThreads = 512;
template <int HD, bool HALF>
struct ArMass {
  static constexpr int KT = HD == 256 ? 1 : 2, KW = HD == 256 ? 4 : 2, CG = 8 / KW;
  static constexpr int KEYS = 32 * KT * KW;                    // a block's
  static constexpr int NC = HD / 16, ALL = HALF ? NC : 2 * NC;  // KB of 32 columns' operands
  static_assert(KEYS == kArMassBlock && CG == ar_mass_group(HD), "the parts' layout");
  static constexpr int SB = HALF ? 2 : 1;                      // steps of CG column blocks a stage
  static constexpr int B = SB * CG * ALL * 1024;               // bytes of a stage
};
template <int HD, bool HALF>
__global__ __launch_bounds__(kArMassThreads, 2) void attn_mass_kernel(AttnRowsParams p) {
  using A = ArMass<HD, HALF>;
  __shared__ __align__(1024) uint8_t smem[2 * A::B];
  __shared__ float part[A::CG][A::KEYS];
  const int kb = blockIdx.x / (unsigned)p.n_kv, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int h = lane >> 5, j = lane & 31, kw = w % A::KW, cg = w / A::KW;
  ArBlock b;
  int pos, fresh;
  b.g = (int)blockIdx.x - kb * p.n_kv;
  b.seq = b.row0 = 0;
  b.tail = true;
  if (!ar_sequence(p, 0, b.cached, fresh) || !ar_position(p, pos)) return;
  b.cached = __builtin_amdgcn_readfirstlane(b.cached);
  b.N = b.cached + fresh;
  if (kb * A::KEYS >= b.N) return;
  const int x0 = kb * A::KEYS + 32 * A::KT * kw;
  const ArRows<HD> rows(p, b);
  half8_t kf[A::KT][A::NC];
#pragma unroll
  for (int t = 0; t < A::KT; ++t) {
    long long own;
    const long long at = rows.row(b, x0 + 32 * t + j, own);
    const char* kr = rows.kc + at + (rows.kd & own) + 16 * h;
#pragma unroll
    for (int k = 0; k < A::NC; ++k) kf[t][k] = *(const half8_t*)(kr + 32 * k);
  }
  // Columns before the first new row that sees the block's first key have nothing for it; the steps over the others are
  // shared by the parts.
  const int cbs = (p.cols + 31) / 32, from0 = max(0, kb * A::KEYS - b.cached) * p.rep / 32;
  const int every = (cbs - from0 + A::CG - 1) / A::CG, step0 = aw_share(every, blockIdx.y, gridDim.y);
  const int cb0 = from0 + step0 * A::CG, steps = aw_share(every, blockIdx.y + 1, gridDim.y) - step0;
  const char* planes = (const char*)p.planes + (size_t)b.g * cbs * A::ALL * 1024;
  const float4* norms = p.norms + (size_t)b.g * p.cols;
  const uint32_t lds = lds_address(smem);
  // The operands of the stage that step i begins, 1 KB a load of a wave; column blocks past the last are that one
  // again, its keys unseen.
  auto load = [&](int i) AW_INLINE {
    if (i >= steps) return;
    const uint32_t to = lds + (i / A::SB & 1) * A::B;
    for (int k = w; k < A::B / 1024; k += 8) {
      const int group = k / A::ALL;
      const size_t at = (size_t)min(cb0 + i * A::CG + group, cbs - 1) * A::ALL + (k - group * A::ALL);
      load_lds16(to + 1024 * k, uniform(planes + at * 1024), (uint32_t)lane * 16);
    }
  };
  float sum[A::KT][16] = {};
  // The scores of a wave's next 32 columns are taken while the exponentials of these run, some after each chunk's
  // products.
  f32x16_t s[A::KT];
  auto add = [&](const f32x16_t* of, int t, int e, const float4& norm) AW_INLINE {
    sum[t][e] = fmaf(__builtin_amdgcn_exp2f(fmaf(of[t][e], norm.z, -norm.x)), norm.y, sum[t][e]);
    asm volatile("" : "+v"(sum[t][e]));           // here, not where the sums are used next
  };
  auto scores = [&](int i, f32x16_t* to, auto beside) AW_INLINE {
    const uint32_t at = lds + i % (2 * A::SB) * (A::B / A::SB) + cg * A::ALL * 1024 + lane * 16;
    // Operands two steps ahead of their products; the barriers keep the steps as they stand here.
    auto operand = [&](int k) AW_INLINE { return lds_half8(at + 1024 * (HALF ? k : k % 2 * A::NC + k / 2)); };
    half8_t q[3] = {operand(0), operand(1), {}};
#pragma unroll
    for (int k = 0; k < A::ALL; ++k) {
      if (k + 2 < A::ALL) q[(k + 2) % 3] = operand(k + 2);
#pragma unroll
      for (int t = 0; t < A::KT; ++t)
        to[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[t][HALF ? k : k / 2], q[k % 3], k ? to[t] : f32x16_t{}, 0, 0, 0);
      beside(k);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto column = [&](int i) AW_INLINE { return (cb0 + i * A::CG + cg) * 32 + j; };
  auto norm_of = [&](int i) AW_INLINE { return norms[min(column(i), p.cols - 1)]; };
  load(0);
  float4 norm = norm_of(0), after = norm_of(1), now;
  wait_loads_and_block<0>();
  load(A::SB);
  if (steps > 0) scores(0, s, [](int) {});
  int i = 0;
  // Before a step's exponentials: where the next one begins a stage, its operands are there for every wave, and the
  // stage behind takes the place of what was read last.
  auto begin = [&]() AW_INLINE {
    now = norm;
    if ((i + 1) % A::SB == 0) {
      wait_loads_and_block<0>();
      load(i + 1 + A::SB);
    }
    norm = after;
    after = norm_of(i + 2);
  };
  // Steps up to number `to` with a mask: where new rows do not see the wave's keys, and the last one.
  auto masked = [&](int to) AW_INLINE {
    for (; i < to; ++i) {
      const int col = column(i), lim = col < p.cols ? b.cached + aw_row(p, col) + 1 : 0;
      begin();
#pragma unroll
      for (int t = 0; t < A::KT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (x0 + 32 * t + 8 * (e >> 2) + 4 * h + (e & 3) < lim) add(s, t, e, now);
      if (i + 1 < steps) scores(i + 1, s, [](int) {});
    }
  };
  auto whole = [&](f32x16_t* of, f32x16_t* next) AW_INLINE {
    begin();
    scores(i + 1, next, [&](int k) AW_INLINE {
#pragma unroll
      for (int x = k * 16 * A::KT / A::ALL; x < (k + 1) * 16 * A::KT / A::ALL; ++x) add(of, x / 16, x % 16, now);
    });
    ++i;
  };
  // Steps [i0, i1) are whole: every column sees every key of the wave, and another step follows.
  const int from = (max(0, x0 + 32 * A::KT - 1 - b.cached) * p.rep + 31) / 32;
  const int i0 = min(steps, max(0, from - cg - cb0 + A::CG - 1) / A::CG);
  const int i1 = max(i0, min(max(0, steps - 1), max(0, p.cols / 32 - cg - cb0 + A::CG - 1) / A::CG));
  masked(i0);
  f32x16_t next[A::KT];
  while (i + 1 < i1) {
    whole(s, next);
    whole(next, s);
  }
  if (i < i1) {
    whole(s, next);
#pragma unroll
    for (int t = 0; t < A::KT; ++t) s[t] = next[t];
  }
  masked(steps);
#pragma unroll
  for (int t = 0; t < A::KT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float v = row16_sum(sum[t][e]);
      v += __shfl_xor(v, 16, 64);
      if (j == 0) part[cg][32 * (A::KT * kw + t) + 8 * (e >> 2) + 4 * h + (e & 3)] = v;
    }
  __syncthreads();
  const int x = kb * A::KEYS + threadIdx.x;
  if (threadIdx.x >= A::KEYS || x >= b.N) return;
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < A::CG; ++i) v += part[i][threadIdx.x];
  if (gridDim.y > 1) {
    p.partial[((size_t)blockIdx.y * gridDim.x + blockIdx.x) * A::KEYS + threadIdx.x] = v;
    return;
  }
  float* m = p.mass + (size_t)b.g * p.tail_slots + x;
  *m = x < b.cached ? *m + v : v;
}

// The parts' sums of the columns into the masses, in order.
__global__ __launch_bounds__(kArMassBlock) void attn_mass_add(AttnRowsParams p, int parts) {
  const int kb = blockIdx.x / (unsigned)p.n_kv, g = (int)blockIdx.x - kb * p.n_kv, x = kb * kArMassBlock + threadIdx.x;
  int have, fresh, pos;
  if (!ar_sequence(p, 0, have, fresh) || !ar_position(p, pos) || x >= have + fresh) return;
  float v = 0.f;
  for (int y = 0; y < parts; ++y) v += p.partial[((size_t)y * gridDim.x + blockIdx.x) * kArMassBlock + threadIdx.x];
  float* m = p.mass + (size_t)g * p.tail_slots + x;
  *m = x < have ? *m + v : v;
}

// Launch ------------------------------------------------------------------------------------------

static_assert(kArTile == kAwKeys, "the plan's tiles");
// The rows that a tail has at most after the call.
static int ar_most_rows(const AttnRowsParams& p) { return p.state || p.lengths ? p.tail_slots : p.length + p.n; }
static ArCall ar_call(const AttnRowsParams& p) {
  return {p.half_io, p.batch, p.n, p.n_head, p.n_kv, p.hd, p.prefix, p.tail_slots, ar_most_rows(p)};
}

const char* attn_rows_refuses(const AttnRowsParams& p) {
  if (p.hd != 64 && p.hd != 128 && p.hd != 256) return "head_dim is not 64, 128 or 256";
  if (p.n_kv < 1 || p.n_head < 1 || p.n_head % p.n_kv) return "n_head is not a multiple of n_kv_head";
  if (p.n_head > 1024) return "more than 1024 heads";
  if (p.prefix_slots < 0 || p.prefix_slots > 1 << 30 || p.tail_slots < 1 || p.tail_slots > 1 << 30) return "slots outside [1, 2^30]";
  if ((long long)p.tail_slots * p.n_kv > 1 << 30 || (long long)p.prefix_slots * p.n_kv > 1 << 30) return "more than 2^30 slots of all kv heads";
  if (p.prefix < 0 || p.prefix > p.prefix_slots) return "prefix outside [0, prefix_slots]";
  // (Blocks of 256 threads, one a column at most, stay below a grid's 2^32 threads.)
  if (p.batch < 0 || p.n < 0 || (p.batch > 0 && (long long)p.n * p.n_head > (1 << 23) / p.batch)) return "too many rows";
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

const char* attn_mass_refuses(const AttnRowsParams& p) {
  if (const char* why = attn_rows_refuses(p)) return why;
  // (attn_mass_kernel's blocks, 512 threads for 128 keys of a kv head, stay below a grid's 2^32 threads.)
  if (((long long)p.tail_slots + kArMassBlock - 1) / kArMassBlock * p.n_kv * kArMassThreads >= 1ll << 32)
    return "2^30 slots of all kv heads or more";
  return nullptr;
}

// Parts of the prefix and of the tails: one split of each, or as many as kArPartRows allows.
static size_t ar_parts_bytes(const AttnRowsParams& p) {
  const long long rows = (long long)p.batch * p.n * p.n_head;
  return (size_t)(2 * std::min(std::max<long long>(rows, kArPartRows), kArMaxSplits * rows)) * (p.hd + 2) * 4;
}
static size_t ar_score_bytes(const AttnRowsParams& p) {
  const size_t column = (size_t)p.n_kv * ar_score_ld(p.tail_slots) * 4, cols = (size_t)p.n * (p.n_head / p.n_kv);
  return std::max(std::min<size_t>(cols, 32) * column, std::min(cols * column, kArScoreBytes));
}
size_t attn_rows_work_bytes(const AttnRowsParams& p) { return ar_parts_bytes(p); }
static size_t ar_norm_bytes(const AttnRowsParams& p) { return (size_t)p.n * p.n_head * sizeof(float4); }
static size_t ar_plane_bytes(const AttnRowsParams& p) {
  return (size_t)cdiv(p.n * (p.n_head / p.n_kv), 32) * 32 * p.n_kv * p.hd * (p.half_io ? 2 : 4);
}
// (Parts of the masses: at most kArCus blocks where there are several.)
constexpr size_t kArPartialBytes = (size_t)kArCus * kArMassBlock * 4;
size_t attn_mass_work_bytes(const AttnRowsParams& p) {
  return p.n ? ar_score_bytes(p) + ar_norm_bytes(p) + ar_plane_bytes(p) + kArPartialBytes : 0;
}

// One segment's blocks, or those of both (few columns each).
template <int HD, bool HALF, bool MASS>
static void ar_segment(AttnRowsParams& p, int wq, bool prefix, bool tail, hipStream_t s) {
  constexpr int WT = HD == 256 ? 4 : 8;             // waves of the kernel for many columns
  p.prefix_cb = cdiv(p.cols, 32 * wq);
  p.tail_cb = cdiv(p.n * p.rep, 32 * wq);
  p.prefix_blocks = prefix ? p.prefix_splits * p.prefix_cb * p.n_kv : 0;
  const dim3 grid(p.prefix_blocks + (tail ? p.batch * p.tail_cb * p.n_kv * p.tail_splits : 0));
  if (wq == 1) hipLaunchKernelGGL((attn_rows_few_kernel<HD, HALF, MASS>), grid, dim3(256), 0, s, p);
  else if (wq == 2) hipLaunchKernelGGL((attn_rows_kernel<HD, HALF, MASS, 2, WT / 2, HD == 64 ? 2 : 1>), grid, dim3(64 * WT), 0, s, p);
  else hipLaunchKernelGGL((attn_rows_kernel<HD, HALF, MASS, 4, WT / 4, 2>), grid, dim3(64 * WT), 0, s, p);
}

template <int HD, bool HALF, bool MASS>
static int ar_launch(AttnRowsParams& p, const ArCut& prefix, const ArCut& tail, hipStream_t s) {
  const bool both = prefix.splits == 0 || (prefix.wq == 1 && tail.wq == 1);
  if (!both) {
    ar_segment<HD, HALF, MASS>(p, prefix.wq, true, false, s);
    TRX_LAUNCHED();
  }
  ar_segment<HD, HALF, MASS>(p, tail.wq, both && prefix.splits > 0, true, s);
  TRX_LAUNCHED();
  const int join = p.nsplit > 1 ? (int)(((long long)p.batch * p.n * p.n_head + 3) / 4) : 0;
  const int append = (int)(((long long)p.batch * p.n * p.n_kv * (HD / 8) + 255) / 256);
  const int masses = p.scores ? cdiv(ar_most_rows(p), p.cols <= 32 ? kArMassKeys : 64) * p.n_kv : 0;
  hipLaunchKernelGGL((attn_rows_finish<HD, HALF, MASS>), dim3(masses + join + append), dim3(256), 0, s, p, masses, join);
  TRX_LAUNCHED();
  if constexpr (MASS) {
    if (!p.scores) {
      const int blocks = cdiv(ar_most_rows(p), kArMassBlock) * p.n_kv, parts = ar_mass_parts(ar_call(p));
      hipLaunchKernelGGL((attn_mass_kernel<HD, HALF>), dim3(blocks, parts), dim3(kArMassThreads), 0, s, p);
      TRX_LAUNCHED();
      if (parts > 1) {
        hipLaunchKernelGGL(attn_mass_add, dim3(blocks), dim3(kArMassBlock), 0, s, p, parts);
        TRX_LAUNCHED();
      }
    }
  }
  return TRX_OK;
}

template <int HD, bool HALF>
static int ar_launch(AttnRowsParams& p, const ArCut& prefix, const ArCut& tail, hipStream_t s) {
  return p.mass ? ar_launch<HD, HALF, true>(p, prefix, tail, s) : ar_launch<HD, HALF, false>(p, prefix, tail, s);
}

int launch_attn_rows(const AttnRowsParams& params, hipStream_t s) {
  AttnRowsParams p = params;
  const char* why = p.mass ? attn_mass_refuses(p) : attn_rows_refuses(p);
  TRX_CHECK(!why, TRX_E_INVALID, "attention over rows: %s", why);
  if (p.n == 0 || p.batch == 0) return TRX_OK;
  p.rep = p.n_head / p.n_kv;
  p.cols = p.batch * p.n * p.rep;
  p.rep_s = 32;
  while (1 << (p.rep_s - 32) < p.rep) ++p.rep_s;
  p.rep_m = ((1ull << p.rep_s) + p.rep - 1) / p.rep;
  ArCut prefix, tail;
  const ArCall call = ar_call(p);
  ar_plan(call, prefix, tail);
  p.prefix_splits = prefix.splits;
  p.tail_splits = tail.splits;
  p.nsplit = prefix.splits + tail.splits;
  if (p.mass) {
    char* at = (char*)p.work + ar_parts_bytes(p);
    const bool keeps = ar_keeps(call, tail);
    p.scores = keeps ? (float*)at : nullptr;
    p.score_ld = ar_score_ld(p.tail_slots);
    p.norms = (float4*)(at + ar_score_bytes(p));
    p.planes = keeps ? nullptr : at + ar_score_bytes(p) + ar_norm_bytes(p);
    p.partial = (float*)(at + ar_score_bytes(p) + ar_norm_bytes(p) + ar_plane_bytes(p));
  }
  if (p.half_io) {
    if (p.hd == 64) return ar_launch<64, true>(p, prefix, tail, s);
    if (p.hd == 128) return ar_launch<128, true>(p, prefix, tail, s);
    return ar_launch<256, true>(p, prefix, tail, s);
  }
  if (p.hd == 64) return ar_launch<64, false>(p, prefix, tail, s);
  if (p.hd == 128) return ar_launch<128, false>(p, prefix, tail, s);
  return ar_launch<256, false>(p, prefix, tail, s);
}

}  // namespace trx

using namespace trx;

#define TRX_API extern "C" __attribute__((visibility("default")))

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <class Shape>
static AttnRowsParams rows_params(const Shape* a, int batch, int n) {
  AttnRowsParams p = {};
  p.half_io = a->kind == TRX_KIND_F16;
  p.batch = batch;
  p.n = n;
  p.n_head = a->n_head;
  p.n_kv = a->n_kv_head;
  p.hd = a->head_dim;
  p.q_stride = a->q_stride;
  p.kv_stride = a->kv_stride;
  p.out_stride = a->out_stride;
  p.gate_stride = a->gate_stride;
  p.gate_head_stride = a->gate_head_stride;
  p.scale = a->scale;
  return p;
}
static AttnRowsParams shared_params(const trx_attn_shared_shape* a, int batch, int n, int prefix) {
  AttnRowsParams p = rows_params(a, batch, n);
  p.prefix_slots = a->prefix_slots;
  p.tail_slots = a->tail_slots;
  p.prefix = prefix;
  return p;
}
static AttnRowsParams mass_params(const trx_attn_mass_shape* a, int n) {
  AttnRowsParams p = rows_params(a, 1, n);
  p.tail_slots = a->slots;
  return p;
}

#define TRX_CHECK_SHAPE(shape, name)                                                                              \
  do {                                                                                                            \
    TRX_CHECK(shape, TRX_E_INVALID, name ": null shape");                                                         \
    TRX_CHECK((shape)->kind == TRX_KIND_F32 || (shape)->kind == TRX_KIND_F16, TRX_E_INVALID,                      \
              name ": kind %d is not F32 or F16", (shape)->kind);                                                 \
  } while (0)

TRX_API int trx_attn_shared_geometry(const trx_attn_shared_shape* shape, int batch, int n, int prefix, size_t* workspace_bytes) {
  TRX_CHECK_SHAPE(shape, "trx_attn_shared_geometry");
  TRX_CHECK(workspace_bytes, TRX_E_INVALID, "trx_attn_shared_geometry: null argument");
  const AttnRowsParams p = shared_params(shape, batch, n, prefix);
  const char* why = attn_rows_refuses(p);
  TRX_CHECK(!why, TRX_E_INVALID, "trx_attn_shared_geometry: %s", why);
  *workspace_bytes = attn_rows_work_bytes(p);
  return TRX_OK;
}

TRX_API int trx_attn_shared(const trx_attn_shared_shape* shape, int batch, int n, int prefix, const int32_t* lengths,
                            const int32_t* counts, const void* q, const uint16_t* k, const uint16_t* v,
                            const uint16_t* kprefix, const uint16_t* vprefix, uint16_t* ktail, uint16_t* vtail,
                            const void* gate, void* out, void* workspace, trx_stream_t s) {
  TRX_CHECK_SHAPE(shape, "trx_attn_shared");
  AttnRowsParams p = shared_params(shape, batch, n, prefix);
  p.gate = gate;
  const char* why = attn_rows_refuses(p);
  TRX_CHECK(!why, TRX_E_INVALID, "trx_attn_shared: %s", why);
  if (batch == 0 || n == 0) return TRX_OK;
  TRX_CHECK(lengths && q && k && v && ktail && vtail && out && workspace && (prefix == 0 || (kprefix && vprefix)),
            TRX_E_INVALID, "trx_attn_shared: null argument");
  TRX_CHECK(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(kprefix) && aligned16(vprefix) && aligned16(ktail) &&
            aligned16(vtail) && aligned16(gate) && aligned16(out) && aligned16(workspace), TRX_E_INVALID,
            "trx_attn_shared: a pointer is not 16-byte aligned");
  TRX_CHECK(((uintptr_t)lengths & 3) == 0 && ((uintptr_t)counts & 3) == 0, TRX_E_INVALID,
            "trx_attn_shared: lengths or counts are not 4-byte aligned");
  p.lengths = lengths;
  p.counts = counts;
  p.q = q;
  p.out = out;
  p.k = (const __half*)k;
  p.v = (const __half*)v;
  p.kprefix = (const __half*)kprefix;
  p.vprefix = (const __half*)vprefix;
  p.ktail = (__half*)ktail;
  p.vtail = (__half*)vtail;
  p.work = workspace;
  return launch_attn_rows(p, (hipStream_t)s);
}

TRX_API int trx_attn_mass_geometry(const trx_attn_mass_shape* shape, int n, size_t* workspace_bytes) {
  TRX_CHECK_SHAPE(shape, "trx_attn_mass_geometry");
  TRX_CHECK(workspace_bytes, TRX_E_INVALID, "trx_attn_mass_geometry: null argument");
  AttnRowsParams p = mass_params(shape, n);
  const char* why = attn_mass_refuses(p);
  TRX_CHECK(!why, TRX_E_INVALID, "trx_attn_mass_geometry: %s", why);
  *workspace_bytes = attn_rows_work_bytes(p) + attn_mass_work_bytes(p);
  return TRX_OK;
}

TRX_API int trx_attn_mass(const trx_attn_mass_shape* shape, int n, int count, int pos, const int32_t* state, const void* q,
                          const uint16_t* k, const uint16_t* v, uint16_t* kcache, uint16_t* vcache, float* mass,
                          int32_t* positions, const void* gate, void* out, void* workspace, trx_stream_t s) {
  TRX_CHECK_SHAPE(shape, "trx_attn_mass");
  AttnRowsParams p = mass_params(shape, n);
  p.gate = gate;
  const char* why = attn_mass_refuses(p);
  TRX_CHECK(!why, TRX_E_INVALID, "trx_attn_mass: %s", why);
  TRX_CHECK(n <= shape->slots, TRX_E_INVALID, "trx_attn_mass: %d rows, %d slots", n, shape->slots);
  TRX_CHECK(state || (count >= 0 && count <= shape->slots - n), TRX_E_INVALID, "trx_attn_mass: %d rows and %d new ones, %d slots",
            count, n, shape->slots);
  TRX_CHECK(state || (pos >= 0 && pos <= INT_MAX - n), TRX_E_INVALID, "trx_attn_mass: position %d", pos);
  if (n == 0) return TRX_OK;
  TRX_CHECK(q && k && v && kcache && vcache && mass && positions && out && workspace, TRX_E_INVALID,
            "trx_attn_mass: null argument");
  TRX_CHECK(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(kcache) && aligned16(vcache) && aligned16(gate) &&
            aligned16(out) && aligned16(workspace), TRX_E_INVALID, "trx_attn_mass: a pointer is not 16-byte aligned");
  TRX_CHECK(((uintptr_t)mass & 3) == 0 && ((uintptr_t)positions & 3) == 0 && ((uintptr_t)state & 3) == 0, TRX_E_INVALID,
            "trx_attn_mass: mass, positions or state are not 4-byte aligned");
  p.state = state;
  p.length = count;
  p.pos = pos;
  p.q = q;
  p.out = out;
  p.k = (const __half*)k;
  p.v = (const __half*)v;
  p.ktail = (__half*)kcache;
  p.vtail = (__half*)vcache;
  p.mass = mass;
  p.positions = positions;
  p.work = workspace;
  return launch_attn_rows(p, (hipStream_t)s);
}
