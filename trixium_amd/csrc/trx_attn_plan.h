// How a call of attention over rows is cut (trx_attn_rows.hip): the host's arithmetic alone, so that it compiles
// without HIP.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstddef>

namespace trx {

constexpr int kArTile = 32;                         // keys of a wave's tile (kAwKeys)
constexpr int kArCus = 256;
constexpr int kArMaxSplits = 64;
constexpr int kArPartRows = 32768;                  // (column, split) pairs of all kv heads that a split segment takes
constexpr int kArMassColumns = 256;                 // columns whose kept scores one block of keys adds up
constexpr int kArMassBlock = 128;                   // keys of a block that takes the scores again

// What the cut depends on.
struct ArCall {
  bool half_io;
  int batch, n, n_head, n_kv, hd, prefix;
  int slots;                   // of a tail
  int keys;                    // rows that a tail has at most after the call
};

// How a segment (the prefix under all columns, or the tails under their own) is cut: columns a block, in waves of 32
// (1: the kernel for few columns), and splits of the keys.
struct ArCut {
  int wq, splits;
};

inline int ar_ceil(long long a, long long b) { return (int)((a + b - 1) / b); }

// What a cut of a segment takes by this estimate, in microseconds, with `others` blocks beside it: a block takes a fixed
// part (its queries, the first rows' latency, the join of its waves, the outputs) and a step for each wk tiles of keys;
// a full chip makes a step 1.4 times as long. fp16 queries, one plane against fp32's two, leave three of four products, a step
// of wide blocks 0.72 as long. Measured (us; waves of columns and splits of the prefix, splits of the
// tails), the choice first:
//   24 drafts over 4001 rows and up to 300 of their own, 32 heads of 128, 8 kv heads: (1, 12; 1) 20; (1, 8; 1) 20,
//     (1, 4; 1) 25, (1, 16; 2) 27, (4, 32; 1) 35
//   64 over 32768 and up to 999, fp16: (4, 16; 1) 107; (4, 12; 1) 109, (2, 8; 1) 109, (4, 8; 1) 123, (1, 8; 1) 133
//   12 of 7 rows over 6001 and up to 200, fp16: (4, 10; 2) 39; (4, 8; 2) 39, (2, 4; 2) 40, (1, 8; 1) 41, (4, 6; 2) 42
//   8 over 2047 and up to 130, 24 heads of 256, 4 kv heads: (1, 16; 2) 20; (1, 8; 1) 23, (2, 16; 1) 39
//   one token with masses over 32700, fp16: 32 splits 38; 24 41, 64 41, 48 43, 16 49
//   27 with masses over 1900, 24 heads of 256: (1, 8) 27; (1, 10) 27, (1, 6) 30, (1, 4) 35, (2, 16) 41, (1, 12) 42
inline double ar_time(const ArCall& p, const ArCut& c, int units, int cols, int keys, long long others) {
  const int wk = c.wq == 1 ? 4 : (p.hd == 256 ? 4 : 8) / c.wq;
  const double fixed = c.wq == 1 ? 2 : 11;
  const double unit = c.wq == 1 ? p.hd / 64.0 : 1.35 * (p.half_io ? 0.72 : 1.0) * (p.hd == 64 ? 0.6 : 1.0);
  const double step = c.wq == 2 ? unit * (p.half_io ? 1.75 : p.hd == 256 ? 1.7 : 1.3) : unit;
  const long long blocks = (long long)units * ar_ceil(cols, 32 * c.wq) * p.n_kv * c.splits + others;
  const int steps = ar_ceil(ar_ceil(ar_ceil(keys, kArTile), c.splits), wk);
  const double full = (double)blocks / kArCus, rounds = full <= 1 ? 1 : 0.5 * (full + std::ceil(full));
  return rounds * (fixed + steps * step * (1 + 0.4 * std::min(full, 1.0)));
}

// f of every cut of a segment into splits that its parts have room for.
template <class F>
inline void ar_cuts(int wq, int keys, long long rows, F f) {
  for (int s : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, 64}) {
    if (s > 1 && (s > ar_ceil(keys, kArTile) || s * rows > kArPartRows)) return;
    f(ArCut{wq, s});
  }
}

inline void ar_plan(const ArCall& p, ArCut& prefix, ArCut& tail) {
  const int rep = p.n_head / p.n_kv, cols = p.n * rep, all = p.batch * cols, keys = p.keys;
  const long long rows = (long long)p.batch * p.n * p.n_head;
  const double part = 8.0 * rows * p.hd / 6e6;       // a part of every column written and read, at 6 TB/s
  // Each segment alone, one launch behind the other (a prefix brings the join with it). Up to 32 columns stay with the
  // kernel for few: wide blocks would leave most of theirs empty.
  double time = 0, least = 1e300;
  for (int wq : {1, 2, 4}) {
    if (wq > 1 && cols <= 32) break;
    ar_cuts(wq, keys, rows, [&](const ArCut& c) {
      const double t = ar_time(p, c, p.batch, cols, keys, 0) + (c.splits > 1 ? (p.prefix ? 0 : 2) + c.splits * part : 0);
      if (t < least) least = t, tail = c;
    });
  }
  prefix = {1, 0};
  if (p.prefix > 0) {
    time = least + 2;
    least = 1e300;
    for (int wq : {1, 2, 4}) {
      if (wq > 1 && all <= 32) break;
      ar_cuts(wq, p.prefix, rows, [&](const ArCut& c) {
        const double t = ar_time(p, c, 1, all, p.prefix, 0) + c.splits * part;
        if (t < least) least = t, prefix = c;
      });
    }
    time += least;
    // Both in one launch, of few columns a block.
    ar_cuts(1, keys, rows, [&](const ArCut& b) {
      const long long tails = (long long)p.batch * ar_ceil(cols, 32) * p.n_kv * b.splits;
      ar_cuts(1, p.prefix, rows, [&](const ArCut& a) {
        const long long prefixes = (long long)ar_ceil(all, 32) * p.n_kv * a.splits;
        const double t = std::max(ar_time(p, a, 1, all, p.prefix, tails), ar_time(p, b, p.batch, cols, keys, prefixes)) +
                         (a.splits + b.splits) * part;
        if (t < time) time = t, prefix = a, tail = b;
      });
    });
  }
}

// Floats from column to column of the kept scores.
inline long long ar_score_ld(int slots) { return ((long long)slots + 31) / 32 * 32; }

// Scores are kept of up to 32 columns, however long the cache, and of up to 256 in 16 MB. (27 positions of 24 heads of 256 over
// 1900 rows, 5 MB: 27 us, 36 where they are taken again; of 32 heads of 128 over 4000, 14 MB: 26 and 31; 60 of them, 31 MB: 41
// and 41.)
constexpr size_t kArScoreBytes = 16 << 20;
inline bool ar_keeps(const ArCall& p, const ArCut& tail) {
  const int cols = p.n * (p.n_head / p.n_kv);
  return cols <= 32 || (tail.wq == 1 && cols <= kArMassColumns && (size_t)cols * p.n_kv * ar_score_ld(p.slots) * 4 <= kArScoreBytes);
}

// Groups of column blocks that a block of the masses' kernel takes beside each other.
constexpr int ar_mass_group(int hd) { return hd == 256 ? 2 : 4; }
// Where the scores are taken again, few blocks of keys (a prompt's first chunk) share the columns as well, four steps at least
// each, and a small launch adds their sums up: 490 positions of 24 heads of 256 alone 64 us, 123 in one part; 538 of 32
// heads of 128 over 488 rows 68 and 81.
inline int ar_mass_parts(const ArCall& p) {
  const int blocks = ar_ceil(p.keys, kArMassBlock) * p.n_kv, cols = p.n * (p.n_head / p.n_kv);
  return std::max(1, std::min(kArCus / blocks, ar_ceil(ar_ceil(cols, 32), ar_mass_group(p.hd)) / 4));
}

}  // namespace trx
