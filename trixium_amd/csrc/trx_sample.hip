// One token per row of logits from the whole vocabulary: temperature, top-k, top-p, min-p, from a
// given uniform number.
//
// Tokens stand in the order of their logits, largest first, equal ones by index. The first top_k
// stay; of those the smallest prefix that holds top_p of their mass; of those the ones with at least
// min_p of the largest mass. The pick is the first in index order at which the mass that stayed passes
// u times its total.
//
// A token's mass e^((l - max) / T) is held as an integer of `frac` fractional bits (62 less the bits of
// the vocabulary's size, at most 51): sums of it are exact, so that neither the split over blocks nor
// the order of atomic additions can change a token. It is evaluated in 64 bits: the rounding of a
// 32-bit exponential would move a border between two tokens by far more than the sums do.
//
// No sort of the vocabulary: a histogram over 1024 steps of the logit's distance from the largest
// (counts and masses) finds the step that the cut falls into; the tokens of that step, or with a short
// list every token up to it, are gathered, and the cut is found among them by nine bits of (logit,
// index) at a time. A row is cut by one block, by the same rounds over the row itself (some seven readings a filter,
// twice that with both), where its cut step holds more than a row's gather (many equal or nearly
// equal logits) or tokens without mass, and where top_k and top_p are both set and the tokens up to top_k's step are
// more than that: what top_p asks for is not known before top_k's cut is. That is slow: top_k 5000 with top_p over
// 248320 logits 1406 us for one row, 1442 for 24, 1684 for 160; with top_k alone 36, 69, 187, with top_p alone 34, 81, 200.
//
// What bounds it: many rows, reading them (the largest logits, the histogram, the gather; for a row drawn from more
// than was gathered, the masses) and the 64-bit exponentials; a single row, six launches that wait for each other.
// us per launch, 160 rows of 248320 fp32 logits (159 MB) with top_p: 28 (5.7 TB/s), 59 (without the
// exponentials 42), 38, the cuts 20, masses 20, draws 9; one row of 151936: 4, 7, 7, 4, 2, 1.

#include "trx_sample.h"

#include <algorithm>

namespace trx {

constexpr int kSrBuckets = 1024;
constexpr int kSrGather = 4096;             // tokens a row's gather holds
constexpr int kSrBlockGather = 1024;        // of a block's, before it counts them into the row's
constexpr int kSrThreads = 256;             // of the kernels that stream a row
constexpr int kSrChunk = 4096;              // logits a block, at least
constexpr int kSrChunksMax = 256;
constexpr int kSrBlocks = 2048;
constexpr int kSrChunkParts = 16;           // of a chunk at most
constexpr int kSrRowThreads = 512;          // of the kernels with a block a row
constexpr int kSrParts = kSrRowThreads;     // of a row, whose masses the draw's block looks through
constexpr int kSrMaxVocab = 1 << 24;        // an index takes 24 bits beside the logit's 32

typedef unsigned long long u64;

// What a row's gather left to do.
enum { SR_DONE, SR_DRAW, SR_FULL, SR_EDGE, SR_ROW };

struct SrState {
  int mode, gathered;
  int by_k, unused;            // top_k leaves live tokens out
  u64 cut;                     // tokens below this (logit, index) are out
  u64 base;                    // EDGE: count or mass before the gathered step
  u64 total;                   // mass of every live token
  float u;
};

// The workspace of a row, in this order.
struct SrWork {
  u64* top;                    // [chunks] each chunk's largest (logit, index)
  u64* mass;                   // [kSrParts] mass that stayed
  u64* hmass;                  // [kSrBuckets]
  u64* item;                   // [kSrGather] gathered tokens
  SrState* st;
  uint32_t* hcount;            // [kSrBuckets]
  float* low;                  // [chunks] each chunk's smallest logit above -inf
};
constexpr size_t sr_row_bytes() {
  return (size_t)(kSrChunksMax + kSrParts) * 8 + (size_t)kSrBuckets * 8 + (size_t)kSrGather * 8 + sizeof(SrState) +
         (size_t)kSrBuckets * 4 + (size_t)kSrChunksMax * 4;
}
__device__ __forceinline__ SrWork sr_work(void* work, int row) {
  uint8_t* b = (uint8_t*)work + (size_t)row * sr_row_bytes();
  SrWork w;
  w.top = (u64*)b;
  w.mass = w.top + kSrChunksMax;
  w.hmass = w.mass + kSrParts;
  w.item = w.hmass + kSrBuckets;
  w.st = (SrState*)(w.item + kSrGather);
  w.hcount = (uint32_t*)(w.st + 1);
  w.low = (float*)(w.hcount + kSrBuckets);
  return w;
}

// A row's settings as they act.
struct SrRow {
  float temperature, top_p, min_p;
  int top_k;
  bool greedy, cut;
};
__device__ __forceinline__ SrRow sr_row(const SampleRowsParams& p, int row) {
  const trx_sampling s = p.rows[p.per_row ? row : 0];
  SrRow r;
  r.greedy = !(s.temperature > 0.f);
  r.temperature = s.temperature;
  r.top_k = s.top_k > 0 && s.top_k < p.vocab ? s.top_k : 0;
  r.top_p = s.top_p > 0.f && s.top_p < 1.f ? s.top_p : 1.f;
  r.min_p = s.min_p >= 0.f && s.min_p <= 1.f ? s.min_p : 0.f;
  r.cut = r.top_k > 0 || r.top_p < 1.f;
  return r;
}

// A logit as the order sees it: NaN counts as -inf, -0 as 0.
__device__ __forceinline__ float sr_clean(float l) { return l != l ? -INFINITY : l + 0.f; }
// (logit, index), larger for a token that stands before.
__device__ __forceinline__ u64 sr_key(float l, int i) {
  return (u64)ordered_bits(l) << 24 | (u64)(kSrMaxVocab - 1 - i);
}
__device__ __forceinline__ float sr_logit(u64 key) {
  const uint32_t b = (uint32_t)(key >> 24);
  return __uint_as_float(b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}
__device__ __forceinline__ int sr_index(u64 key) { return kSrMaxVocab - 1 - (int)(key & (kSrMaxVocab - 1)); }

// Masses and buckets of one row: the largest logit, log2(e) / T, buckets per unit of logit.
struct SrScale {
  double top, c2, per;
  int frac;
  bool inf;                    // the largest logit is +inf: those tokens share the mass
  bool dead;                   // tokens above -inf may have no mass; these are in the last bucket

  __device__ __forceinline__ SrScale(float M, float low, float T, int frac_) : frac(frac_) {
    top = M;
    inf = M == INFINITY;
    c2 = 1.44269504088896340736 / (double)T;
    const double end = (frac + 1) / c2;         // a mass of half a unit: below it, and rounded there, 0
    const double reach = fmin(end, top - (double)low);
    // (A mass above half a unit by 2^-36 of itself is one in spite of the roundings of y and of the series.)
    dead = inf || !(top - (double)low < end * (1.0 - 0x1p-40));
    per = !inf && reach > 0.0 ? kSrBuckets / reach : 0.0;
  }
  __device__ __forceinline__ u64 mass(float l) const {
    u64 m;
    masses<1>(&l, &m);
    return m;
  }
  // Of N logits side by side, their chains of products interleaved and without branches: one logit after the
  // other took twice as long.
  template <int N>
  __device__ __forceinline__ void masses(const float* l, u64* m) const {
    if (inf) {
#pragma unroll
      for (int i = 0; i < N; ++i) m[i] = l[i] == INFINITY ? 1ull << frac : 0;
      return;
    }
    // 2^y = 2^n 2^f, |f| <= 1/2: the series of e^(f ln 2) to the twelfth power is off by 2^-52.
    constexpr double k1 = 0.69314718055994530942, k2 = k1 * k1 / 2, k3 = k2 * k1 / 3, k4 = k3 * k1 / 4, k5 = k4 * k1 / 5,
                     k6 = k5 * k1 / 6, k7 = k6 * k1 / 7, k8 = k7 * k1 / 8, k9 = k8 * k1 / 9, k10 = k9 * k1 / 10,
                     k11 = k10 * k1 / 11, k12 = k11 * k1 / 12;
    constexpr double k[12] = {k11, k10, k9, k8, k7, k6, k5, k4, k3, k2, k1, 1.0};
    double f[N], w[N];
    int n[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const double y = fmax(((double)l[i] - top) * c2, -(double)(frac + 2));   // below: 0 as well
      const double t = y + 6755399441055744.0;  // 1.5 2^52: y rounded, in the low bits
      n[i] = (int)__double_as_longlong(t);
      f[i] = y - (t - 6755399441055744.0);
      w[i] = k12;
    }
#pragma unroll
    for (int j = 0; j < 12; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = fma(w[i], f[i], k[j]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // Times 2^(n + frac) on the exponent; rounded to an integer below 2^52 by the addition of 2^52 (a quarter
      // and a half go to 0).
      const double x = __longlong_as_double(__double_as_longlong(w[i]) + ((long long)(n[i] + frac) << 52));
      m[i] = (u64)__double_as_longlong(x + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
    }
  }
  __device__ __forceinline__ int bucket(float l) const {
    return (int)fminf((float)(((double)l - top) * -per), (float)(kSrBuckets - 1));
  }
  // Not above any logit of the buckets up to b (half a bucket of slack, then the float next to it).
  __device__ __forceinline__ float under(int b) const {
    return b >= kSrBuckets - 1 || !(per > 0.0) ? -INFINITY : (float)(top - (b + 1.5) / per);
  }
  // Not below any logit of the buckets from b on.
  __device__ __forceinline__ float over(int b) const { return (float)(top - (b - 0.5) / per); }
  // The smallest mass that min_p lets stay.
  __device__ __forceinline__ u64 floor_mass(float min_p) const {
    return (u64)ceil(ldexp((double)min_p, frac));
  }
};

// floor and ceil of x * total, 0 <= x < 1, exact.
__device__ __forceinline__ void sr_split(float x, uint32_t& m, int& e) {
  const uint32_t b = __float_as_uint(x), ex = b >> 23 & 0xFF;
  m = ex ? (b & 0x7FFFFF) | 0x800000 : b & 0x7FFFFF;
  e = 150 - (int)(ex ? ex : 1);               // x = m 2^-e
}
__device__ __forceinline__ u64 sr_floor(float x, u64 total) {
  uint32_t m;
  int e;
  sr_split(x, m, e);
  return e > 127 ? 0 : (u64)((unsigned __int128)total * m >> e);
}
__device__ __forceinline__ u64 sr_ceil(float x, u64 total) {
  uint32_t m;
  int e;
  sr_split(x, m, e);
  if (e > 100) return 1;                       // total < 2^62, m < 2^24
  return (u64)(((unsigned __int128)total * m + (((unsigned __int128)1 << e) - 1)) >> e);
}
// The mass that the draw has to pass: floor(u total), u outside [0, 1) at its nearest value there.
__device__ __forceinline__ u64 sr_target(float u, u64 total) {
  if (!(u > 0.f)) return 0;
  return u < 1.f ? sr_floor(u, total) : total - 1;
}

// The logits of a row in 16-byte pieces, whatever its alignment: `head` scalars before the first
// aligned one belong to chunk 0, the last piece is read by element.
template <class T>
struct SrLogits {
  static constexpr int E = 16 / sizeof(T);
  const T* row;
  int vocab, head;
  __device__ __forceinline__ SrLogits(const SampleRowsParams& p, int r) : vocab(p.vocab) {
    row = (const T*)p.logits + (size_t)r * p.ld;
    head = min((int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T), vocab);
  }
  __device__ __forceinline__ float at(int i) const { return sr_clean((float)row[i]); }
  __device__ __forceinline__ int end(int c, int chunk) const { return (int)min((long long)vocab, head + (c + 1ll) * chunk); }
  template <int THREADS, class F>
  __device__ __forceinline__ void each(int c, int chunk, F f) const {
    span<THREADS>(c * chunk, end(c, chunk), f, [] {});
  }
  // f(logits, index of the first) for every piece of E elements from the first-th behind the head on (0: the head
  // too) to before e1, over the block's threads; what a piece lacks is -inf. Four pieces a thread are on their way
  // while four are worked on; group() follows each four, in every thread.
  static constexpr int U = 4;
  template <int THREADS, class F, class G>
  __device__ __forceinline__ void span(int first, int e1, F f, G group) const {
    constexpr int S = THREADS * E * U;
    if (first == 0 && (int)threadIdx.x < head) {
      float v[E];
#pragma unroll
      for (int x = 1; x < E; ++x) v[x] = -INFINITY;
      v[0] = at(threadIdx.x);
      f(v, (int)threadIdx.x);
    }
    uint4 raw[U];
    auto load = [&](uint4* to, int g) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = g + (k * THREADS + (int)threadIdx.x) * E;
        if (i + E <= e1) to[k] = *(const uint4*)(row + i);
      }
    };
    load(raw, head + first);
    for (int g = head + first; g < e1; g += S) {
      uint4 next[U];
      if (g + S < e1) load(next, g + S);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = g + (k * THREADS + (int)threadIdx.x) * E;
        if (i >= e1) break;
        float v[E];
        if (i + E <= e1) {
          T x[E];
          __builtin_memcpy(x, &raw[k], 16);
#pragma unroll
          for (int j = 0; j < E; ++j) v[j] = sr_clean((float)x[j]);
        } else {
#pragma unroll
          for (int j = 0; j < E; ++j) v[j] = i + j < e1 ? at(i + j) : -INFINITY;
        }
        f(v, i);
      }
      group();
#pragma unroll
      for (int k = 0; k < U; ++k) raw[k] = next[k];
    }
  }
};

// The sum of this lane's value and those of the lanes before it: rows of 16 by shifts, then the rows' ends.
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_u64(u64 v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, true);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 wave_upto_u64(u64 v) {
  v += dpp_u64<0x111, 0xF>(v);                 // row_shr 1, 2, 4, 8
  v += dpp_u64<0x112, 0xF>(v);
  v += dpp_u64<0x114, 0xF>(v);
  v += dpp_u64<0x118, 0xF>(v);
  v += dpp_u64<0x142, 0xA>(v);                 // row_bcast 15 into rows 1 and 3
  v += dpp_u64<0x143, 0xC>(v);                 // row_bcast 31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ u64 wave_lane_u64(u64 v, int lane) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
__device__ __forceinline__ u64 wave_sum_u64(u64 v) { return wave_lane_u64(wave_upto_u64(v), 63); }
// The largest value of the wave (every lane gets it), the same way.
__device__ __forceinline__ u64 wave_max_u64(u64 v) {
  const auto up = [&](u64 x) __attribute__((always_inline)) { v = x > v ? x : v; };
  up(dpp_u64<0x111, 0xF>(v));
  up(dpp_u64<0x112, 0xF>(v));
  up(dpp_u64<0x114, 0xF>(v));
  up(dpp_u64<0x118, 0xF>(v));
  up(dpp_u64<0x142, 0xA>(v));
  up(dpp_u64<0x143, 0xC>(v));
  return wave_lane_u64(v, 63);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_min(float v) {
  return fminf(v, __int_as_float(__builtin_amdgcn_update_dpp(0x7F800000, __float_as_int(v), CTRL, ROWS, 0xF, false)));
}
__device__ __forceinline__ float wave_min(float v) {
  v = dpp_min<0x111, 0xF>(v);
  v = dpp_min<0x112, 0xF>(v);
  v = dpp_min<0x114, 0xF>(v);
  v = dpp_min<0x118, 0xF>(v);
  v = dpp_min<0x142, 0xA>(v);
  v = dpp_min<0x143, 0xC>(v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
// Sum over the block (every thread gets it); red holds a value a wave, of 16 at most.
__device__ __forceinline__ u64 block_sum_u64(u64 v, u64* red) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
  v = wave_upto_u64(v);
  __syncthreads();
  if (lane == 63) red[w] = v;
  __syncthreads();
  u64 t = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i < nw) t += red[i];
  return t;
}
// Sum of the values of the threads before this one, and of all.
__device__ __forceinline__ u64 block_before_u64(u64 v, u64* red, u64& all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
  const u64 x = wave_upto_u64(v);
  __syncthreads();
  if (lane == 63) red[w] = x;
  __syncthreads();
  u64 t = 0;
  all = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const u64 r = i < nw ? red[i] : 0;
    t += i < w ? r : 0;
    all += r;
  }
  return t + x - v;
}

// The row's largest (logit, index) and smallest logit from its chunks' (every thread gets them): the thread's
// share first, so that a kernel's first loads are on their way together.
struct SrExtremes {
  u64 t;
  float l;
  __device__ __forceinline__ SrExtremes(const SrWork& w, int chunks) : t(0), l(INFINITY) {
    for (int i = threadIdx.x; i < chunks; i += blockDim.x) {
      t = w.top[i] > t ? w.top[i] : t;
      l = fminf(l, w.low[i]);
    }
  }
  __device__ __forceinline__ void get(u64* red, u64& top, float& low) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, nw = min((int)blockDim.x, kSrChunksMax) >> 6;
    t = wave_max_u64(t);
    l = wave_min(l);
    __shared__ float lred[16];
    __syncthreads();
    if (lane == 0) red[wv] = t, lred[wv] = l;
    __syncthreads();
    for (int i = 0; i < nw; ++i) {             // (no chunk's thread is in a later wave)
      t = red[i] > t ? red[i] : t;
      l = fminf(l, lred[i]);
    }
    top = t;
    low = l;
  }
};

__device__ __forceinline__ bool sr_none(u64 top) { return sr_logit(top) == -INFINITY; }

// A decode position that computes no logits draws nothing.
__device__ __forceinline__ bool sr_gated(const SampleRowsParams& p) { return p.gate_pos && *p.gate_pos < *p.gate_from; }

__device__ __forceinline__ void sr_put(const SampleRowsParams& p, int row, int token, float logp) {
  p.tokens[row] = token;
  if (p.logp) p.logp[row] = logp;
  if (p.slot) *p.slot = (1ull << 32) | (u64)(0xFFFFFFFFu - (uint32_t)max(token, 0));
}

// 1. Every chunk's largest token and smallest logit; the row's histogram and state cleared.
template <class T>
__global__ __launch_bounds__(kSrThreads) void sample_extremes_kernel(SampleRowsParams p) {
  __shared__ u64 red[4];
  __shared__ float lred[4];
  if (sr_gated(p)) return;
  const int row = blockIdx.x / p.chunks, c = blockIdx.x - row * p.chunks, t = threadIdx.x;
  const SrWork w = sr_work(p.work, row);
  for (int i = c * kSrThreads + t; i < kSrBuckets; i += p.chunks * kSrThreads) w.hmass[i] = 0, w.hcount[i] = 0;
  if (c == 0 && t == 0) {
    *w.st = SrState{sr_row(p, row).cut ? SR_DONE : SR_DRAW, 0, 0, 0, 0, 0, 0, 0.f};
    if (!p.rng) {
      w.st->u = p.u[row];
    } else if (!sr_row(p, row).greedy) {
      uint32_t x = *p.rng;
      x ^= x << 13;
      x ^= x >> 17;
      x ^= x << 5;
      *p.rng = x;
      w.st->u = (float)(x >> 8) * (1.0f / 16777216.0f);
    }
  }
  const SrLogits<T> lg(p, row);
  u64 top = 0;
  float low = INFINITY;
  float best = -INFINITY;                      // the thread's largest logit, and where it stood first
  int where = 0;
  lg.template each<kSrThreads>(c, p.chunk, [&](const float* l, int i) {
#pragma unroll
    for (int x = 0; x < SrLogits<T>::E; ++x) {
      where = l[x] > best ? i + x : where;
      best = fmaxf(best, l[x]);
      low = fminf(low, l[x] > -INFINITY ? l[x] : INFINITY);
    }
  });
  top = wave_max_u64(sr_key(best, where));
  low = wave_min(low);
  if ((t & 63) == 0) red[t >> 6] = top, lred[t >> 6] = low;
  __syncthreads();
  if (t == 0) {
    for (int i = 1; i < 4; ++i) {
      top = red[i] > top ? red[i] : top;
      low = fminf(low, lred[i]);
    }
    w.top[c] = top;
    w.low[c] = low;
  }
}

// 2. The histogram of a row with a cut. The others need none; rows of the largest logit, and those with no logit
// to take, are done here.
template <class T>
__global__ __launch_bounds__(kSrThreads) void sample_histogram_kernel(SampleRowsParams p) {
  __shared__ u64 hm[kSrBuckets];
  __shared__ uint32_t hc[kSrBuckets];
  __shared__ u64 red[4];
  if (sr_gated(p)) return;
  const int row = blockIdx.x / p.chunks, c = blockIdx.x - row * p.chunks, t = threadIdx.x;
  const SrWork w = sr_work(p.work, row);
  const SrRow s = sr_row(p, row);
  if (c > 0 && (s.greedy || !s.cut)) return;
  u64 top;
  float low;
  SrExtremes(w, p.chunks).get(red, top, low);
  if (s.greedy || sr_none(top)) {
    if (c == 0 && t == 0) {
      w.st->mode = SR_DONE;
      if (sr_none(top)) sr_put(p, row, -1, NAN);
      else sr_put(p, row, sr_index(top), 0.f);
    }
    return;
  }
  if (!s.cut) return;
  for (int i = t; i < kSrBuckets; i += kSrThreads) hm[i] = 0, hc[i] = 0;
  __syncthreads();
  const SrScale sc(sr_logit(top), low, s.temperature, p.frac);
  constexpr int E = SrLogits<T>::E;
  SrLogits<T>(p, row).template each<kSrThreads>(c, p.chunk, [&](const float* l, int) {
    u64 m[E];
    int b[E];
#pragma unroll
    for (int x = 0; x < E; ++x) b[x] = sc.bucket(l[x]);
    sc.template masses<E>(l, m);
#pragma unroll
    for (int x = 0; x < E; ++x)
      if (m[x]) {
        atomicAdd(&hm[b[x]], m[x]);
        atomicAdd(&hc[b[x]], 1u);
      }
  });
  __syncthreads();
  for (int i = t; i < kSrBuckets; i += kSrThreads)
    if (hc[i]) {
      atomicAdd(w.hmass + i, hm[i]);
      atomicAdd(w.hcount + i, hc[i]);
    }
}

// Where a row's cut falls, from its histogram (256 threads, four buckets each; every thread gets it).
struct SrPlan {
  int mode, b0, b1;            // gather the buckets b0 .. b1
  bool by_k;
  u64 base, total;
};
constexpr int kSrOwn = kSrBuckets / kSrThreads;
__device__ SrPlan sr_plan(const SrWork& w, const SrRow& s, const u64* m, const uint32_t* n, u64* red) {
  __shared__ int bk_s, bp_s;
  __shared__ u64 base_s[4];
  const int t = threadIdx.x;
  constexpr int E = kSrOwn;
  u64 msum = 0, nsum = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    msum += m[i];
    nsum += n[i];
  }
  u64 total, live;
  u64 mb = block_before_u64(msum, red, total), nb = block_before_u64(nsum, red, live);
  if (t == 0) bk_s = bp_s = -1;
  __syncthreads();
  const bool by_k = s.top_k > 0 && (u64)s.top_k < live, by_p = s.top_p < 1.f;
  const u64 want_p = by_p ? sr_ceil(s.top_p, total) : 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    // One bucket takes the sum past each target.
    if (by_k && nb < (u64)s.top_k && nb + n[i] >= (u64)s.top_k) bk_s = E * t + i, base_s[0] = nb, base_s[1] = n[i];
    if (by_p && mb < want_p && mb + m[i] >= want_p) bp_s = E * t + i, base_s[2] = mb, base_s[3] = nb + n[i];
    nb += n[i];
    mb += m[i];
  }
  __syncthreads();
  SrPlan q;
  q.total = total;
  q.base = 0;
  q.b0 = 0;
  q.by_k = by_k;
  if (by_k) {
    q.b1 = bk_s;
    q.mode = base_s[0] + base_s[1] <= kSrGather ? SR_FULL : by_p || base_s[1] > kSrGather ? SR_ROW : SR_EDGE;
    if (q.mode == SR_EDGE) q.b0 = bk_s, q.base = base_s[0];
  } else if (by_p) {
    q.b1 = bp_s;
    const u64 here = w.hcount[q.b1];
    q.mode = base_s[3] <= kSrGather ? SR_FULL : here > kSrGather ? SR_ROW : SR_EDGE;
    if (q.mode == SR_EDGE) q.b0 = bp_s, q.base = base_s[2];
  } else {
    q.mode = SR_DRAW;                          // top_k takes every live token
    q.b1 = -1;
  }
  return q;
}

// 3. The tokens of the buckets that the cut's search needs.
template <class T>
__global__ __launch_bounds__(kSrThreads) void sample_gather_kernel(SampleRowsParams p) {
  __shared__ u64 red[4];
  if (sr_gated(p)) return;
  const int row = blockIdx.x / p.chunks, c = blockIdx.x - row * p.chunks, t = threadIdx.x;
  const SrWork w = sr_work(p.work, row);
  const SrRow s = sr_row(p, row);
  if (s.greedy || !s.cut) return;
  u64 top;
  float low;
  u64 m[kSrOwn];
  uint32_t n[kSrOwn];
#pragma unroll
  for (int i = 0; i < kSrOwn; ++i) m[i] = w.hmass[kSrOwn * t + i], n[i] = w.hcount[kSrOwn * t + i];
  SrExtremes(w, p.chunks).get(red, top, low);
  if (sr_none(top)) return;
  SrPlan q = sr_plan(w, s, m, n, red);
  const SrScale sc(sr_logit(top), low, s.temperature, p.frac);
  // Then every gathered token has a mass, without a look at it here (42 us instead of 39 for 160 rows of 248320).
  if (q.b1 == kSrBuckets - 1 && sc.dead) q.mode = SR_ROW;
  if (c == 0 && t == 0) {
    w.st->mode = q.mode;
    w.st->by_k = q.by_k;
    w.st->base = q.base;
    w.st->total = q.total;
  }
  if (q.mode != SR_FULL && q.mode != SR_EDGE) return;
  // The block's tokens together in LDS, so that it counts them into the row's once; past the buffer one by one.
  __shared__ u64 buf[kSrBlockGather];
  __shared__ int found, at_s;
  if (t == 0) found = 0;
  __syncthreads();
  const float least = sc.under(q.b1), most = q.b0 ? sc.over(q.b0) : INFINITY;
  SrLogits<T>(p, row).template each<kSrThreads>(c, p.chunk, [&](const float* l, int i) {
    bool some = false;
#pragma unroll
    for (int x = 0; x < SrLogits<T>::E; ++x) some |= (l[x] >= least) & (l[x] <= most);
    if (!some) return;
#pragma unroll
    for (int x = 0; x < SrLogits<T>::E; ++x) {
      if (l[x] < least || l[x] > most || l[x] == -INFINITY) continue;
      const int b = sc.bucket(l[x]);
      if (b < q.b0 || b > q.b1) continue;
      const u64 key = sr_key(l[x], i + x);
      const int at = atomicAdd(&found, 1);
      if (at < kSrBlockGather) {
        buf[at] = key;
      } else {
        const int g = atomicAdd(&w.st->gathered, 1);
        if (g < kSrGather) w.item[g] = key;
      }
    }
  });
  __syncthreads();
  const int count = min(found, kSrBlockGather);
  if (t == 0 && count) at_s = atomicAdd(&w.st->gathered, count);
  __syncthreads();
  for (int i = t; i < count; i += kSrThreads)
    if (at_s + i < kSrGather) w.item[at_s + i] = buf[i];
}

// The key at which the weights, added from the largest key down, reach `want`: BITS bits a round from the first
// in which lo and hi differ, between which every key with a weight lies, until one token is left.
// each(f) calls f(key, weight) over the thread's tokens.
struct SrSelect {
  u64 hist[kSrRowThreads], pick[2], key;
  uint32_t count[kSrRowThreads];
};
template <class Each>
__device__ u64 sr_select(Each each, u64 want, u64 lo, u64 hi, SrSelect& x, u64* red) {
  constexpr int BITS = __builtin_ctz(kSrRowThreads);  // a thread a bin
  const int t = threadIdx.x;
  int bits = lo == hi ? 0 : 64 - __clzll(lo ^ hi);
  u64 prefix = bits < 64 ? hi >> bits : 0;
  while (bits > 0) {
    const int shift = max(bits - BITS, 0), bins = 1 << (bits - shift), above = bits;
    x.hist[t] = 0;
    x.count[t] = 0;
    __syncthreads();
    each([&](u64 key, u64 wgt) {
      if (wgt && key >> above == prefix) {
        const int b = (int)(key >> shift) & (bins - 1);
        atomicAdd(&x.hist[b], wgt);
        atomicAdd(&x.count[b], 1u);
      }
    });
    __syncthreads();
    // Thread i holds the i-th bin from above.
    const int mine = bins - 1 - t;
    const u64 v = mine >= 0 ? x.hist[mine] : 0;
    u64 all;
    const u64 before = block_before_u64(v, red, all);
    if (mine >= 0 && before < want && before + v >= want) x.pick[0] = mine, x.pick[1] = before;
    __syncthreads();
    const int b = (int)x.pick[0];
    prefix = prefix << (bits - shift) | (u64)b;
    want -= x.pick[1];
    bits = shift;
    if (shift > 0 && x.count[b] == 1) {
      each([&](u64 key, u64 wgt) {
        if (wgt && key >> shift == prefix) x.key = key;
      });
      __syncthreads();
      prefix = x.key;
      bits = 0;
    }
    __syncthreads();
  }
  return prefix;
}
// The smallest and largest key with a weight, over the block.
template <class Each>
__device__ void sr_range(Each each, u64& lo, u64& hi, u64* red) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
  u64 a = ~0ull, b = 0;
  each([&](u64 key, u64 wgt) {
    a = wgt && key < a ? key : a;
    b = wgt && key > b ? key : b;
  });
  a = ~wave_max_u64(~a);
  b = wave_max_u64(b);
  __syncthreads();
  if (lane == 0) red[w] = a, red[w + nw] = b;
  __syncthreads();
  for (int i = 0; i < nw; ++i) {
    a = red[i] < a ? red[i] : a;
    b = red[nw + i] > b ? red[nw + i] : b;
  }
  __syncthreads();
  lo = a;
  hi = b;
}

__device__ __forceinline__ void sr_store(const SampleRowsParams& p, int row, const SrScale& sc, float T, float l, int i,
                                         u64 total) {
  const double d = sc.inf ? 0.0 : -(sc.top - (double)l) / (double)T;
  sr_put(p, row, i, p.logp ? (float)(d - log(ldexp((double)total, -sc.frac))) : 0.f);
}

// 4. A block a row: the cut, and the draw where every token that stayed was gathered. Bound by the barriers and by
// what every wave computes alike: 512 threads take 12.7 us for one row of 200 gathered tokens, 1024 15.6, 256 12.4; of
// 160 rows 20, 19, 26. Up to 64 tokens one wave compares each with each: 4.2 us against 10.7.
template <class T>
__global__ __launch_bounds__(kSrRowThreads) void sample_cut_kernel(SampleRowsParams p) {
  __shared__ u64 key_s[kSrGather], mass_s[kSrGather];
  __shared__ SrSelect sel;
  __shared__ u64 red[32];
  if (sr_gated(p)) return;
  const int row = blockIdx.x, t = threadIdx.x;
  const SrWork w = sr_work(p.work, row);
  const SrState st = *w.st;
  SrExtremes ends(w, p.chunks);
  constexpr int OWN = kSrGather / kSrRowThreads;
  u64 item[OWN];                               // the thread's gathered tokens (some past the last one)
#pragma unroll
  for (int i = 0; i < OWN; ++i) item[i] = w.item[t + i * kSrRowThreads];
  const SrRow s = sr_row(p, row);
  if (st.mode == SR_DONE || st.mode == SR_DRAW) return;
  u64 top;
  float low;
  ends.get(red, top, low);
  const SrScale sc(sr_logit(top), low, s.temperature, p.frac);
  if (st.mode == SR_ROW) {
    const SrLogits<T> lg(p, row);
    auto masses = [&](auto f) {
      lg.template each<kSrRowThreads>(0, p.vocab, [&](const float* l, int i) {
#pragma unroll
        for (int x = 0; x < SrLogits<T>::E; ++x) f(sr_key(l[x], i + x), sc.mass(l[x]));
      });
    };
    auto counts = [&](auto f) { masses([&](u64 key, u64 wgt) { f(key, wgt ? 1ull : 0ull); }); };
    const u64 lo = sr_key(low, kSrMaxVocab - 1);
    u64 cut = 0, total = st.total;
    if (st.by_k) {
      cut = sr_select(counts, (u64)s.top_k, lo, top, sel, red);
      u64 m = 0;
      masses([&](u64 key, u64 wgt) { m += key >= cut ? wgt : 0; });
      total = block_sum_u64(m, red);
    }
    if (s.top_p < 1.f) {
      const u64 c2 = sr_select(masses, sr_ceil(s.top_p, total), lo, top, sel, red);
      cut = c2 > cut ? c2 : cut;
    }
    if (t == 0) w.st->cut = cut, w.st->mode = SR_DRAW;
    return;
  }
  const int n = min(st.gathered, kSrGather);
  if (n <= 64) {
    // A wave's worth: every token's place in the order by comparing it with each of the others, no barriers.
    if (t >= 64) return;
    const u64 key = t < n ? item[0] : 0;
    u64 m = t < n ? sc.mass(sr_logit(key)) : 0, before = 0, total = st.total;
    int rank = 0;
    for (int i = 0; i < n; ++i) {
      const u64 k = wave_lane_u64(key, i), w = wave_lane_u64(m, i);
      rank += k > key && w;
      before += k > key ? w : 0;
    }
    if (st.mode == SR_EDGE) {
      const u64 want = (st.by_k ? (u64)s.top_k : sr_ceil(s.top_p, total)) - st.base;
      if (m && (st.by_k ? (u64)rank + 1 == want : before < want && before + m >= want)) w.st->cut = key;
      if (t == 0) w.st->mode = SR_DRAW;
      return;
    }
    if (st.by_k) {
      if (rank >= s.top_k) m = 0;
      total = wave_sum_u64(m);
    }
    if (s.top_p < 1.f && before >= sr_ceil(s.top_p, total)) m = 0;
    if (m < sc.floor_mass(s.min_p)) m = 0;
    total = wave_sum_u64(m);
    const u64 want = sr_target(st.u, total), place = key & (kSrMaxVocab - 1);
    before = 0;
    for (int i = 0; i < n; ++i) before += (wave_lane_u64(key, i) & (kSrMaxVocab - 1)) > place ? wave_lane_u64(m, i) : 0;
    if (m && before <= want && want < before + m) sr_store(p, row, sc, s.temperature, sr_logit(key), sr_index(key), total);
    if (t == 0) w.st->mode = SR_DONE;
    return;
  }
#pragma unroll
  for (int i = 0; i < OWN; ++i)
    if (t + i * kSrRowThreads < n) {
      key_s[t + i * kSrRowThreads] = item[i];
      mass_s[t + i * kSrRowThreads] = sc.mass(sr_logit(item[i]));
    }
  __syncthreads();
  u64 lo, hi;
  sr_range([&](auto f) {
    for (int i = t; i < n; i += kSrRowThreads) f(key_s[i], mass_s[i]);
  }, lo, hi, red);
  // The cut by count, the cut by mass, the draw, each a search.
  const bool edge = st.mode == SR_EDGE;
  u64 total = st.total;
#pragma unroll 1
  for (int stage = 0; stage < 3; ++stage) {
    if (stage == 0 ? !st.by_k : stage == 1 && (edge ? st.by_k : s.top_p >= 1.f)) continue;
    if (!edge && (stage == 2 || (stage == 1 && st.by_k))) {
      const u64 least = stage == 2 ? sc.floor_mass(s.min_p) : 0;
      u64 m = 0;
      for (int i = t; i < n; i += kSrRowThreads) {  // (a thread's own tokens)
        if (mass_s[i] < least) mass_s[i] = 0;
        m += mass_s[i];
      }
      total = block_sum_u64(m, red);
    }
    u64 want = stage == 0 ? (u64)s.top_k : stage == 1 ? sr_ceil(s.top_p, total) : sr_target(st.u, total) + 1;
    if (edge) want -= st.base;
    // The draw goes in index order: by the index part of the keys alone, which falls as the index rises.
    const u64 part = stage == 2 ? (u64)(kSrMaxVocab - 1) : ~0ull;
    if (stage == 2) lo = kSrMaxVocab - p.vocab, hi = kSrMaxVocab - 1;
    const u64 key = sr_select([&](auto f) {
      for (int i = t; i < n; i += kSrRowThreads) {
        const u64 m = mass_s[i];
        f(key_s[i] & part, stage == 0 && m ? 1 : m);
      }
    }, want, lo, hi, sel, red);
    if (edge) {
      if (t == 0) w.st->cut = key, w.st->mode = SR_DRAW;
      return;
    }
    for (int i = t; i < n; i += kSrRowThreads) {
      if (stage < 2 && key_s[i] < key) mass_s[i] = 0;
      if (stage == 2 && mass_s[i] && (key_s[i] & part) == key)
        sr_store(p, row, sc, s.temperature, sr_logit(key_s[i]), sr_index(key), total);
    }
  }
  if (t == 0) w.st->mode = SR_DONE;
}

// 5. The mass that stayed in each part of a chunk, for the rows not yet drawn.
template <class T>
__global__ __launch_bounds__(kSrThreads) void sample_mass_kernel(SampleRowsParams p) {
  __shared__ u64 red[4];
  __shared__ u64 part[kSrChunkParts][kSrThreads / 64];
  if (sr_gated(p)) return;
  const int row = blockIdx.x / p.chunks, c = blockIdx.x - row * p.chunks, t = threadIdx.x;
  const SrWork w = sr_work(p.work, row);
  if (w.st->mode != SR_DRAW) return;
  const SrRow s = sr_row(p, row);
  const u64 cut = w.st->cut;
  u64 top;
  float low;
  SrExtremes(w, p.chunks).get(red, top, low);
  const SrScale sc(sr_logit(top), low, s.temperature, p.frac);
  const u64 least = sc.floor_mass(s.min_p);
  // (logit, index) at least `cut`: above its logit, or that and no later than its index.
  const float edge = cut ? sr_logit(cut) : -INFINITY;
  const int last = cut ? sr_index(cut) : kSrMaxVocab;
  const SrLogits<T> lg(p, row);
  constexpr int E = SrLogits<T>::E;
  u64 sum = 0;                                 // (the block's sums only at the end: no barriers between the parts)
  int left = p.part, i = 0;
  lg.template span<kSrThreads>(c * p.chunk, lg.end(c, p.chunk), [&](const float* l, int at) {
    u64 m[E];
    sc.template masses<E>(l, m);
#pragma unroll
    for (int x = 0; x < E; ++x)
      sum += (m[x] >= least) & ((l[x] > edge) | ((l[x] == edge) & (at + x <= last))) ? m[x] : 0;
  }, [&] {
    left -= kSrThreads * E * SrLogits<T>::U;
    if (left > 0) return;
    sum = wave_upto_u64(sum);
    if ((t & 63) == 63) part[i][t >> 6] = sum;
    sum = 0;
    left = p.part;
    ++i;
  });
  sum = wave_upto_u64(sum);                    // of a part that the row's end cuts short
  if (i < p.parts && (t & 63) == 63) part[i][t >> 6] = sum;
  for (++i; i < p.parts; ++i)
    if ((t & 63) == 63) part[i][t >> 6] = 0;
  __syncthreads();
  if (t < p.parts) w.mass[c * p.parts + t] = part[t][0] + part[t][1] + part[t][2] + part[t][3];
}

// 6. The part that the draw falls into, and the token in it.
template <class T>
__global__ __launch_bounds__(kSrRowThreads) void sample_draw_kernel(SampleRowsParams p) {
  __shared__ u64 red[16], before_s;
  __shared__ int part_s;
  if (sr_gated(p)) return;
  const int row = blockIdx.x, t = threadIdx.x;
  const SrWork w = sr_work(p.work, row);
  if (w.st->mode != SR_DRAW) return;
  const SrRow s = sr_row(p, row);
  const u64 cut = w.st->cut;
  u64 top;
  float low;
  SrExtremes(w, p.chunks).get(red, top, low);
  const SrScale sc(sr_logit(top), low, s.temperature, p.frac);
  const u64 least = sc.floor_mass(s.min_p);
  const u64 mc = t < p.chunks * p.parts ? w.mass[t] : 0;
  u64 total;
  const u64 bc = block_before_u64(mc, red, total);
  u64 want = sr_target(w.st->u, total);
  if (bc <= want && want < bc + mc) part_s = t, before_s = bc;
  __syncthreads();
  want -= before_s;
  const SrLogits<T> lg(p, row);
  const int c = part_s / p.parts, first = c * p.chunk + (part_s - c * p.parts) * p.part;
  const int i1 = min(lg.end(c, p.chunk), lg.end(0, first + p.part));
  for (int i0 = first ? lg.head + first : 0; i0 < i1; i0 += 4 * kSrRowThreads) {
    u64 m[4], sum = 0;
    float l[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + 4 * t + k;
      l[k] = i < i1 ? lg.at(i) : -INFINITY;
    }
    sc.template masses<4>(l, m);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + 4 * t + k;
      if (m[k] < least || sr_key(l[k], min(i, i1 - 1)) < cut) m[k] = 0;
      sum += m[k];
    }
    u64 all, b = block_before_u64(sum, red, all);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (b <= want && want < b + m[k]) sr_store(p, row, sc, s.temperature, l[k], i0 + 4 * t + k, total);
      b += m[k];
    }
    if (want < all) return;
    want -= all;
  }
}

// The repetition penalty --------------------------------------------------------------------------

constexpr int kPenaltyWindow = 64;          // positions at most (a thread each)

__global__ __launch_bounds__(kSrThreads) void penalty_kernel(PenaltyParams p) {
  const int pos = *p.pos;
  if (pos < *p.head_from) return;
  const int t = threadIdx.x, i0 = blockIdx.x * kSrChunk, i1 = min(p.vocab, i0 + kSrChunk);
  for (int i = i0 + t; i < i1; i += kSrThreads) p.out[i] = p.logits[i];
  __syncthreads();                           // the block's own copies first
  const int j = pos - t;
  if (t >= min(p.window, kPenaltyWindow) || j < 0) return;
  const int tok = p.tokens[j % p.ring];
  if (tok < i0 || tok >= i1) return;
  const float v = p.logits[tok], rep = *p.repetition;
  p.out[tok] = v > 0.f ? v / rep : v * rep;  // of a token that stands twice, twice the same value
}

int launch_penalty(const PenaltyParams& p, hipStream_t s) {
  TRX_CHECK(p.vocab > 0 && p.window >= 0 && p.window <= kPenaltyWindow, TRX_E_INVALID, "penalty: bad parameters");
  hipLaunchKernelGGL(penalty_kernel, dim3(cdiv(p.vocab, kSrChunk)), dim3(kSrThreads), 0, s, p);
  TRX_LAUNCHED();
  return TRX_OK;
}

// Launch ------------------------------------------------------------------------------------------

const char* sample_rows_refuses(int n, int vocab) {
  if (vocab < 1 || vocab > kSrMaxVocab) return "vocab outside [1, 2^24]";
  if (n < 0 || n > 1 << 20) return "more than 2^20 rows";
  return nullptr;
}

size_t sample_rows_work_bytes(int n, int vocab) { return (size_t)n * sr_row_bytes(); }

template <class T>
static int sr_launch(const SampleRowsParams& p, hipStream_t s) {
  const dim3 grid(p.n * p.chunks), block(kSrThreads), rows(p.n), row_block(kSrRowThreads);
  hipLaunchKernelGGL(sample_extremes_kernel<T>, grid, block, 0, s, p);
  TRX_LAUNCHED();
  hipLaunchKernelGGL(sample_histogram_kernel<T>, grid, block, 0, s, p);
  TRX_LAUNCHED();
  hipLaunchKernelGGL(sample_gather_kernel<T>, grid, block, 0, s, p);
  TRX_LAUNCHED();
  hipLaunchKernelGGL(sample_cut_kernel<T>, rows, row_block, 0, s, p);
  TRX_LAUNCHED();
  hipLaunchKernelGGL(sample_mass_kernel<T>, grid, block, 0, s, p);
  TRX_LAUNCHED();
  hipLaunchKernelGGL(sample_draw_kernel<T>, rows, row_block, 0, s, p);
  TRX_LAUNCHED();
  return TRX_OK;
}

int launch_sample_rows(const SampleRowsParams& params, hipStream_t s) {
  SampleRowsParams p = params;
  const char* why = sample_rows_refuses(p.n, p.vocab);
  TRX_CHECK(!why, TRX_E_INVALID, "sampling: %s", why);
  if (p.n == 0) return TRX_OK;
  // About eight blocks a CU: many rows take long chunks (a chunk's histogram goes into the row's by atomics, as
  // many as it has buckets), few rows short ones. 160 rows of 248320, with 1024, 2048, 4096 blocks in all: 212,
  // 195, 187 us; 24 rows of 151936: 77, 78, 103. One row, with chunks of at least 1024, 2048, 4096: 45, 40, 40.
  const int most = std::min(kSrChunksMax, std::max(1, cdiv(kSrBlocks, p.n)));
  p.chunk = kSrChunk * cdiv(cdiv(p.vocab, kSrChunk), most);
  p.chunks = cdiv(p.vocab, p.chunk);
  const int group = kSrThreads * SrLogits<float>::U * (p.half ? SrLogits<_Float16>::E : SrLogits<float>::E);
  p.part = group * cdiv(cdiv(p.chunk, group), std::min(kSrChunkParts, kSrParts / p.chunks));
  p.parts = cdiv(p.chunk, p.part);
  int bits = 0;
  while ((1 << bits) < p.vocab) ++bits;
  p.frac = std::min(51, 62 - bits);
  return p.half ? sr_launch<_Float16>(p, s) : sr_launch<float>(p, s);
}

}  // namespace trx

using namespace trx;

#define TRX_API extern "C" __attribute__((visibility("default")))

TRX_API int trx_sample_rows_geometry(int vocab, int n, size_t* workspace_bytes) {
  TRX_CHECK(workspace_bytes, TRX_E_INVALID, "trx_sample_rows_geometry: null argument");
  const char* why = sample_rows_refuses(n, vocab);
  TRX_CHECK(!why, TRX_E_INVALID, "trx_sample_rows_geometry: %s", why);
  *workspace_bytes = sample_rows_work_bytes(n, vocab);
  return TRX_OK;
}

TRX_API int trx_sample_rows(const void* logits, int kind, int n, int vocab, int64_t ld, const trx_sampling* rows,
                            int per_row, const float* u, int32_t* tokens, float* logp, void* workspace,
                            trx_stream_t s) {
  TRX_CHECK(kind == TRX_KIND_F32 || kind == TRX_KIND_F16, TRX_E_INVALID, "trx_sample_rows: kind %d is not F32 or F16", kind);
  const char* why = sample_rows_refuses(n, vocab);
  TRX_CHECK(!why, TRX_E_INVALID, "trx_sample_rows: %s", why);
  TRX_CHECK(ld >= vocab, TRX_E_INVALID, "trx_sample_rows: rows of %lld values, %d tokens", (long long)ld, vocab);
  if (n == 0) return TRX_OK;
  TRX_CHECK(logits && rows && u && tokens && workspace, TRX_E_INVALID, "trx_sample_rows: null argument");
  TRX_CHECK(((uintptr_t)logits & (kind == TRX_KIND_F32 ? 3 : 1)) == 0 && ((uintptr_t)rows & 3) == 0 &&
            ((uintptr_t)u & 3) == 0 && ((uintptr_t)tokens & 3) == 0 && ((uintptr_t)logp & 3) == 0 &&
            ((uintptr_t)workspace & 15) == 0, TRX_E_INVALID, "trx_sample_rows: a pointer is not aligned");
  SampleRowsParams p = {};
  p.logits = logits;
  p.half = kind == TRX_KIND_F16;
  p.n = n;
  p.vocab = vocab;
  p.ld = ld;
  p.rows = rows;
  p.per_row = per_row != 0;
  p.u = u;
  p.tokens = tokens;
  p.logp = logp;
  p.work = workspace;
  return launch_sample_rows(p, (hipStream_t)s);
}
