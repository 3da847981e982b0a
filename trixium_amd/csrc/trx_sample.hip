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
// list every token up to it, are gathered, and the cut is found among them by eight bits of (logit,
// index) at a time. A row whose cut step holds more than a block gathers (many equal or nearly equal
// logits) is cut by the same rounds over the row itself.

#include "trx_sample.h"

#include <algorithm>

namespace trx {

constexpr int kSrBuckets = 1024;
constexpr int kSrGather = 4096;             // tokens a row's gather holds
constexpr int kSrThreads = 256;             // of the kernels that stream a row
constexpr int kSrChunk = 4096;              // logits a block, at least
constexpr int kSrChunksMax = 256;
constexpr int kSrRowThreads = 1024;         // of the kernels with a block a row
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
  u64* mass;                   // [chunks] mass that stayed
  u64* hmass;                  // [kSrBuckets]
  u64* item;                   // [kSrGather] gathered tokens
  SrState* st;
  uint32_t* hcount;            // [kSrBuckets]
  float* low;                  // [chunks] each chunk's smallest logit above -inf
};
constexpr size_t sr_row_bytes() {
  return (size_t)kSrChunksMax * 16 + (size_t)kSrBuckets * 8 + (size_t)kSrGather * 8 + sizeof(SrState) +
         (size_t)kSrBuckets * 4 + (size_t)kSrChunksMax * 4;
}
__device__ __forceinline__ SrWork sr_work(void* work, int row) {
  uint8_t* b = (uint8_t*)work + (size_t)row * sr_row_bytes();
  SrWork w;
  w.top = (u64*)b;
  w.mass = w.top + kSrChunksMax;
  w.hmass = w.mass + kSrChunksMax;
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

  __device__ __forceinline__ SrScale(float M, float low, float T, int frac_) : frac(frac_) {
    top = M;
    inf = M == INFINITY;
    c2 = 1.44269504088896340736 / (double)T;
    const double reach = fmin((frac + 1) / c2, top - (double)low);   // below it a mass is 0
    per = !inf && reach > 0.0 ? kSrBuckets / reach : 0.0;
  }
  __device__ __forceinline__ u64 mass(float l) const {
    if (inf) return l == INFINITY ? 1ull << frac : 0;
    const double y = -(top - (double)l) * c2;
    if (!(y >= -(double)(frac + 1))) return 0;
    // 2^y = 2^n e^(f ln 2), |f| <= 1/2: the series to the twelfth power is off by 2^-52.
    const double n = rint(y), f = (y - n) * 0.69314718055994530942;
    double w = 1.0 / 479001600.0;
    w = fma(w, f, 1.0 / 39916800.0);
    w = fma(w, f, 1.0 / 3628800.0);
    w = fma(w, f, 1.0 / 362880.0);
    w = fma(w, f, 1.0 / 40320.0);
    w = fma(w, f, 1.0 / 5040.0);
    w = fma(w, f, 1.0 / 720.0);
    w = fma(w, f, 1.0 / 120.0);
    w = fma(w, f, 1.0 / 24.0);
    w = fma(w, f, 1.0 / 6.0);
    w = fma(w, f, 0.5);
    w = fma(w, f, 1.0);
    w = fma(w, f, 1.0);
    // Rounded to an integer below 2^52 by the addition of 2^52.
    const double v = ldexp(w, (int)n + frac) + 4503599627370496.0;
    return (u64)__double_as_longlong(v) & 0xFFFFFFFFFFFFFull;
  }
  __device__ __forceinline__ int bucket(float l) const {
    return min(kSrBuckets - 1, (int)fmin((top - (double)l) * per, (double)kSrBuckets));
  }
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
  __device__ __forceinline__ int begin(int c, int chunk) const { return c ? min(vocab, head + c * chunk) : 0; }
  __device__ __forceinline__ int end(int c, int chunk) const { return (int)min((long long)vocab, head + (c + 1ll) * chunk); }
  // f(logit, index) for every element of chunk c, over the block's threads.
  template <int THREADS, class F>
  __device__ __forceinline__ void each(int c, int chunk, F f) const {
    if (c == 0 && (int)threadIdx.x < head) f(at(threadIdx.x), (int)threadIdx.x);
    const int e1 = end(c, chunk);
    constexpr int U = 4;
    for (int i0 = head + c * chunk + (int)threadIdx.x * E; i0 < e1; i0 += THREADS * E * U) {
      uint4 raw[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = i0 + k * THREADS * E;
        if (i + E <= e1) raw[k] = *(const uint4*)(row + i);
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = i0 + k * THREADS * E;
        if (i + E <= e1) {
          T v[E];
          __builtin_memcpy(v, &raw[k], 16);
#pragma unroll
          for (int x = 0; x < E; ++x) f(sr_clean((float)v[x]), i + x);
        } else {
          for (int x = i; x < e1; ++x) f(at(x), x);
        }
      }
    }
  }
};

__device__ __forceinline__ u64 wave_max_u64(u64 v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const u64 x = __shfl_xor(v, o, 64);
    v = x > v ? x : v;
  }
  return v;
}
__device__ __forceinline__ float wave_min(float v) { return -wave_max(-v); }
__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// Sum over the block (every thread gets it); red holds a value a wave.
__device__ __forceinline__ u64 block_sum_u64(u64 v, u64* red) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
  v = wave_sum_u64(v);
  __syncthreads();
  if (lane == 0) red[w] = v;
  __syncthreads();
  u64 t = 0;
  for (int i = 0; i < nw; ++i) t += red[i];
  return t;
}
// Sum of the values of the threads before this one.
__device__ __forceinline__ u64 block_before_u64(u64 v, u64* red) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  u64 x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) red[w] = x;
  __syncthreads();
  u64 t = 0;
  for (int i = 0; i < w; ++i) t += red[i];
  return t + x - v;
}

// The row's largest (logit, index) and smallest logit from its chunks' (every thread gets them).
__device__ __forceinline__ void sr_extremes(const SrWork& w, int chunks, u64* red, u64& top, float& low) {
  u64 t = 0;
  float l = INFINITY;
  for (int i = threadIdx.x; i < chunks; i += blockDim.x) {
    t = w.top[i] > t ? w.top[i] : t;
    l = fminf(l, w.low[i]);
  }
  t = wave_max_u64(t);
  l = wave_min(l);
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, nw = blockDim.x >> 6;
  __shared__ float lred[16];
  __syncthreads();
  if (lane == 0) red[wv] = t, lred[wv] = l;
  __syncthreads();
  for (int i = 0; i < nw; ++i) {
    t = red[i] > t ? red[i] : t;
    l = fminf(l, lred[i]);
  }
  top = t;
  low = l;
}

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
    *w.st = SrState{SR_DONE, 0, 0, 0, 0, 0, 0, 0.f};
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
  lg.template each<kSrThreads>(c, p.chunk, [&](float l, int i) {
    const u64 k = sr_key(l, i);
    top = k > top ? k : top;
    if (l > -INFINITY) low = fminf(low, l);
  });
  top = wave_max_u64(top);
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

// 2. The histogram of a row with a cut; the others need none (the largest logit's row is done here).
template <class T>
__global__ __launch_bounds__(kSrThreads) void sample_histogram_kernel(SampleRowsParams p) {
  __shared__ u64 hm[kSrBuckets];
  __shared__ uint32_t hc[kSrBuckets];
  __shared__ u64 red[4];
  if (sr_gated(p)) return;
  const int row = blockIdx.x / p.chunks, c = blockIdx.x - row * p.chunks, t = threadIdx.x;
  const SrWork w = sr_work(p.work, row);
  const SrRow s = sr_row(p, row);
  u64 top;
  float low;
  sr_extremes(w, p.chunks, red, top, low);
  if (s.greedy || sr_none(top)) {
    if (c == 0 && t == 0) {
      if (sr_none(top)) sr_put(p, row, -1, NAN);
      else sr_put(p, row, sr_index(top), 0.f);
    }
    return;
  }
  if (!s.cut) {
    if (c == 0 && t == 0) w.st->mode = SR_DRAW;
    return;
  }
  for (int i = t; i < kSrBuckets; i += kSrThreads) hm[i] = 0, hc[i] = 0;
  __syncthreads();
  const SrScale sc(sr_logit(top), low, s.temperature, p.frac);
  SrLogits<T>(p, row).template each<kSrThreads>(c, p.chunk, [&](float l, int) {
    const u64 m = sc.mass(l);
    if (m) {
      const int b = sc.bucket(l);
      atomicAdd(&hm[b], m);
      atomicAdd(&hc[b], 1u);
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
__device__ SrPlan sr_plan(const SrWork& w, const SrRow& s, u64* red) {
  __shared__ int bk_s, bp_s;
  __shared__ u64 base_s[4], total_s[2];
  const int t = threadIdx.x;
  constexpr int E = kSrBuckets / kSrThreads;
  u64 m[E], msum = 0;
  uint32_t n[E];
  u64 nsum = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    m[i] = w.hmass[E * t + i];
    n[i] = w.hcount[E * t + i];
    msum += m[i];
    nsum += n[i];
  }
  u64 mb = block_before_u64(msum, red), nb = block_before_u64(nsum, red);
  if (t == kSrThreads - 1) total_s[0] = mb + msum, total_s[1] = nb + nsum;
  if (t == 0) bk_s = bp_s = -1;
  __syncthreads();
  const u64 total = total_s[0], live = total_s[1];
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
  u64 top;
  float low;
  sr_extremes(w, p.chunks, red, top, low);
  if (s.greedy || sr_none(top) || !s.cut) return;
  const SrPlan q = sr_plan(w, s, red);
  if (c == 0 && t == 0) {
    w.st->mode = q.mode;
    w.st->by_k = q.by_k;
    w.st->base = q.base;
    w.st->total = q.total;
  }
  if (q.mode != SR_FULL && q.mode != SR_EDGE) return;
  const SrScale sc(sr_logit(top), low, s.temperature, p.frac);
  SrLogits<T>(p, row).template each<kSrThreads>(c, p.chunk, [&](float l, int i) {
    if (!sc.mass(l)) return;
    const int b = sc.bucket(l);
    if (b < q.b0 || b > q.b1) return;
    const int at = atomicAdd(&w.st->gathered, 1);
    if (at < kSrGather) w.item[at] = sr_key(l, i);
  });
}

// The (logit, index) at which the weights, added from the largest key down, reach `want`: eight bits a
// round from the highest that differ. each(f) calls f(key, weight) over the thread's tokens.
template <class Each>
__device__ u64 sr_select(Each each, u64 want, int bits, u64* hist, u64* red) {
  __shared__ u64 pick_s[2];
  const int t = threadIdx.x;
  u64 prefix = 0;
  for (int shift = bits - 8; shift >= 0; shift -= 8) {
    if (t < 256) hist[t] = 0;
    __syncthreads();
    each([&](u64 key, u64 wgt) {
      if (wgt && (shift + 8 >= 64 ? 0 : key >> (shift + 8)) == prefix) atomicAdd(&hist[key >> shift & 255], wgt);
    });
    __syncthreads();
    // Thread i holds bin 255 - i.
    const u64 v = t < 256 ? hist[255 - t] : 0;
    const u64 before = block_before_u64(v, red);
    if (t < 256 && before < want && before + v >= want) pick_s[0] = 255 - t, pick_s[1] = before;
    __syncthreads();
    prefix = prefix << 8 | pick_s[0];
    want -= pick_s[1];
    __syncthreads();
  }
  return prefix;
}

__device__ __forceinline__ void sr_store(const SampleRowsParams& p, int row, const SrScale& sc, float T, float l, int i,
                                         u64 total) {
  const double d = sc.inf ? 0.0 : -(sc.top - (double)l) / (double)T;
  sr_put(p, row, i, p.logp ? (float)(d - log(ldexp((double)total, -sc.frac))) : 0.f);
}

// 4. A block a row: the cut, and the draw where every token that stayed was gathered.
template <class T>
__global__ __launch_bounds__(kSrRowThreads) void sample_cut_kernel(SampleRowsParams p) {
  __shared__ u64 key_s[kSrGather], mass_s[kSrGather];
  __shared__ u64 hist[256], red[16];
  if (sr_gated(p)) return;
  const int row = blockIdx.x, t = threadIdx.x;
  const SrWork w = sr_work(p.work, row);
  const SrState st = *w.st;
  if (st.mode == SR_DONE || st.mode == SR_DRAW) return;
  const SrRow s = sr_row(p, row);
  u64 top;
  float low;
  sr_extremes(w, p.chunks, red, top, low);
  const SrScale sc(sr_logit(top), low, s.temperature, p.frac);
  constexpr int KB = 56;                       // bits of a key
  if (st.mode == SR_ROW) {
    const SrLogits<T> lg(p, row);
    auto counts = [&](auto f) {
      for (int c = 0; c < p.chunks; ++c)
        lg.template each<kSrRowThreads>(c, p.chunk, [&](float l, int i) { f(sr_key(l, i), sc.mass(l) ? 1ull : 0ull); });
    };
    auto masses = [&](auto f) {
      for (int c = 0; c < p.chunks; ++c)
        lg.template each<kSrRowThreads>(c, p.chunk, [&](float l, int i) { f(sr_key(l, i), sc.mass(l)); });
    };
    u64 cut = 0, total = st.total;
    if (st.by_k) {
      cut = sr_select(counts, (u64)s.top_k, KB, hist, red);
      u64 m = 0;
      masses([&](u64 key, u64 wgt) { m += key >= cut ? wgt : 0; });
      total = block_sum_u64(m, red);
    }
    if (s.top_p < 1.f) {
      const u64 c2 = sr_select(masses, sr_ceil(s.top_p, total), KB, hist, red);
      cut = c2 > cut ? c2 : cut;
    }
    if (t == 0) w.st->cut = cut, w.st->mode = SR_DRAW;
    return;
  }
  const int n = min(st.gathered, kSrGather);
  for (int i = t; i < n; i += kSrRowThreads) {
    const u64 k = w.item[i];
    key_s[i] = k;
    mass_s[i] = sc.mass(sr_logit(k));
  }
  __syncthreads();
  auto masses = [&](auto f) {
    for (int i = t; i < n; i += kSrRowThreads) f(key_s[i], mass_s[i]);
  };
  auto counts = [&](auto f) {
    for (int i = t; i < n; i += kSrRowThreads) f(key_s[i], mass_s[i] ? 1ull : 0ull);
  };
  auto keep = [&](u64 cut) {                   // a thread's own tokens
    for (int i = t; i < n; i += kSrRowThreads)
      if (key_s[i] < cut) mass_s[i] = 0;
  };
  if (st.mode == SR_EDGE) {
    const u64 cut = st.by_k ? sr_select(counts, (u64)s.top_k - st.base, KB, hist, red)
                             : sr_select(masses, sr_ceil(s.top_p, st.total) - st.base, KB, hist, red);
    if (t == 0) w.st->cut = cut, w.st->mode = SR_DRAW;
    return;
  }
  u64 total = st.total;
  if (st.by_k) {
    keep(sr_select(counts, (u64)s.top_k, KB, hist, red));
    u64 m = 0;
    masses([&](u64, u64 wgt) { m += wgt; });
    total = block_sum_u64(m, red);
  }
  if (s.top_p < 1.f) keep(sr_select(masses, sr_ceil(s.top_p, total), KB, hist, red));
  const u64 least = sc.floor_mass(s.min_p);
  u64 m = 0;
  for (int i = t; i < n; i += kSrRowThreads) {
    if (mass_s[i] < least) mass_s[i] = 0;
    m += mass_s[i];
  }
  total = block_sum_u64(m, red);
  // In index order: the index part of the keys alone, which falls as the index rises.
  auto by_index = [&](auto f) {
    for (int i = t; i < n; i += kSrRowThreads) f(key_s[i] & (kSrMaxVocab - 1), mass_s[i]);
  };
  const u64 pick = sr_select(by_index, sr_target(st.u, total) + 1, 24, hist, red);
  for (int i = t; i < n; i += kSrRowThreads)
    if (mass_s[i] && (key_s[i] & (kSrMaxVocab - 1)) == pick) sr_store(p, row, sc, s.temperature, sr_logit(key_s[i]), sr_index(pick), total);
  if (t == 0) w.st->mode = SR_DONE;
}

// 5. Each chunk's mass that stayed, for the rows not yet drawn.
template <class T>
__global__ __launch_bounds__(kSrThreads) void sample_mass_kernel(SampleRowsParams p) {
  __shared__ u64 red[4];
  if (sr_gated(p)) return;
  const int row = blockIdx.x / p.chunks, c = blockIdx.x - row * p.chunks, t = threadIdx.x;
  const SrWork w = sr_work(p.work, row);
  if (w.st->mode != SR_DRAW) return;
  const SrRow s = sr_row(p, row);
  const u64 cut = w.st->cut;
  u64 top;
  float low;
  sr_extremes(w, p.chunks, red, top, low);
  const SrScale sc(sr_logit(top), low, s.temperature, p.frac);
  const u64 least = sc.floor_mass(s.min_p);
  u64 sum = 0;
  SrLogits<T>(p, row).template each<kSrThreads>(c, p.chunk, [&](float l, int i) {
    const u64 m = sc.mass(l);
    if (m >= least && sr_key(l, i) >= cut) sum += m;
  });
  sum = block_sum_u64(sum, red);
  if (t == 0) w.mass[c] = sum;
}

// 6. The chunk that the draw falls into, and the token in it.
template <class T>
__global__ __launch_bounds__(kSrRowThreads) void sample_draw_kernel(SampleRowsParams p) {
  __shared__ u64 red[16], before_s;
  __shared__ int chunk_s;
  if (sr_gated(p)) return;
  const int row = blockIdx.x, t = threadIdx.x;
  const SrWork w = sr_work(p.work, row);
  if (w.st->mode != SR_DRAW) return;
  const SrRow s = sr_row(p, row);
  const u64 cut = w.st->cut;
  u64 top;
  float low;
  sr_extremes(w, p.chunks, red, top, low);
  const SrScale sc(sr_logit(top), low, s.temperature, p.frac);
  const u64 least = sc.floor_mass(s.min_p);
  const u64 mc = t < p.chunks ? w.mass[t] : 0;
  const u64 total = block_sum_u64(mc, red);
  u64 want = sr_target(w.st->u, total);
  const u64 bc = block_before_u64(mc, red);
  if (bc <= want && want < bc + mc) chunk_s = t, before_s = bc;
  __syncthreads();
  want -= before_s;
  const SrLogits<T> lg(p, row);
  const int c = chunk_s, i1 = lg.end(c, p.chunk);
  for (int i0 = lg.begin(c, p.chunk); i0 < i1; i0 += 4 * kSrRowThreads) {
    u64 m[4], sum = 0;
    float l[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + 4 * t + k;
      l[k] = i < i1 ? lg.at(i) : -INFINITY;
      m[k] = sc.mass(l[k]);
      if (m[k] < least || sr_key(l[k], min(i, i1 - 1)) < cut) m[k] = 0;
      sum += m[k];
    }
    u64 b = block_before_u64(sum, red);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (b <= want && want < b + m[k]) sr_store(p, row, sc, s.temperature, l[k], i0 + 4 * t + k, total);
      b += m[k];
    }
    const u64 all = block_sum_u64(sum, red);
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
  p.chunk = kSrChunk * std::max(1, cdiv(cdiv(p.vocab, kSrChunk), kSrChunksMax));
  p.chunks = cdiv(p.vocab, p.chunk);
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
