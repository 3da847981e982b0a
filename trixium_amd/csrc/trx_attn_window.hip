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

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <limits.h>

namespace trx {

constexpr int kAwKeys = 32;                 // keys per wave and stage
constexpr float kAwBias = 7.f;              // log2 of the largest probability's fp16 value, less 8
constexpr float kAwRaise = 8.f;
constexpr float kLog2e = 1.44269504088896341f;

#define AW_INLINE __attribute__((always_inline))   // a call would keep its arrays in memory

typedef _Float16 half2v_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef short s16x2_t __attribute__((ext_vector_type(2)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

// LDS rows of a stage stand one after the other as the loads deliver them (64 lanes times 16 bytes in a row),
// a row's 16-byte pieces in an order that spreads the reads over the banks: piece c of row r at place
// c ^ swizzle(r).
template <int HD>
struct AwLds {
  static constexpr int ROW = 2 * HD;                // bytes
  // K rows are read 16 bytes a lane, a row a lane: sixteen rows take sixteen places.
  __device__ __forceinline__ static int k_swizzle(int r) { return HD == 64 ? (r >> 1) & 7 : r & 15; }
  // V rows are read transposed, 64 bytes of each of four rows at a time: the four take four places.
  __device__ __forceinline__ static int v_swizzle(int r) { return HD == 64 ? (r >> 1 & 1) << 2 : (r & 3) << 2; }
};

// 16 bytes a lane from global memory straight into LDS, the wave's 1024 bytes in lane order at `lds` (uniform).
// Counted by vmcnt like a load; wait_loads_and_block stands between it and the reads of what it brings, and
// between the reads of what it replaces and itself.
__device__ __forceinline__ void load_lds16(uint32_t lds, const char* g) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(g));
}
__device__ __forceinline__ void load_lds16(uint32_t lds, const char* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base));
}
// A pointer that every lane holds alike, as the uniform base of a load.
__device__ __forceinline__ const char* uniform(const char* p) {
  const uint64_t a = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a), hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
  return (const char*)((uint64_t)hi << 32 | lo);
}
// Until at most N of this wave's loads are outstanding and its LDS reads are done; then the block's barrier.
template <int N>
__device__ __forceinline__ void wait_loads_and_block() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

typedef __attribute__((address_space(3))) uint8_t lds_byte;
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
__device__ __forceinline__ half8_t lds_half8(uint32_t at) {
  return *(const __attribute__((address_space(3))) half8_t*)(uintptr_t)at;
}

// Four consecutive keys of one dim a lane: within 16 lanes, lane l gives the address of key l / 4, dims
// 4 (l % 4) .. + 3, and takes dim l of the four keys.
__device__ __forceinline__ half4_t lds_read_tr(uint32_t at) {
  typedef __attribute__((address_space(3))) s16x4_t lds_t;
  return __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(uintptr_t)at));
}

// The first position, and whether the call has positions that the ring's arithmetic holds.
__device__ __forceinline__ bool aw_pos(const AttnWindowParams& p, int& pos) {
  pos = p.pos_dev ? *p.pos_dev : p.pos;
  return pos >= 0 && pos <= INT_MAX - p.n;
}

// Largest of a lane's value and that of lane ^ 32.
__device__ __forceinline__ float both_halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// fp16 of a - hi.lo and b - hi.hi, each rounded once.
__device__ __forceinline__ uint32_t rest_h(uint32_t hi, float a, float b) {
  uint32_t r;
  asm("v_fma_mixlo_f16 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(hi), "v"(a));
  asm("v_fma_mixhi_f16 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(r) : "v"(hi), "v"(b));
  return r;
}

// All ones in the halves of two fp16 values that are finite.
__device__ __forceinline__ uint32_t finite_h(uint32_t two) {
  const s16x2_t x = __builtin_bit_cast(s16x2_t, two & 0x7FFF7FFFu) - (short)0x7C00;
  return __builtin_bit_cast(uint32_t, x >> 15);
}

// The position's row of a column: column / rep by a product (columns below 2^25, rep_m = 2^rep_s / rep rounded up,
// 2^rep_s at least 2^32 rep: exact).
__device__ __forceinline__ int aw_row(const AttnWindowParams& p, int column) {
  return (int)((unsigned long long)(unsigned)column * p.rep_m >> p.rep_s);
}
// The first of a split's share of `count` stages (count below 2^26, at most 64 splits).
__device__ __forceinline__ int aw_share(int count, int split, int splits) {
  return (int)((unsigned)count * (unsigned)split / (unsigned)splits);
}

// What the waves of a block know of their work: the call's first position and the block's keys, numbered
// x in [0, N): position x below ns (the sinks), else x - ns + lo.
struct AwBlock {
  int pos, g, sp, c0;          // first position; kv head; split; first column
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
  b.sp = blockIdx.y;
  b.c0 = (int)cb * columns;
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

  __device__ __forceinline__ AwRows(const AttnWindowParams& p, int g) : kv_stride(p.kv_stride), pin(p.pin) {
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

// The queries of a wave's columns in the B operand's layout: dims 16 c + 8 h .. + 7.
template <int HD, bool HALF>
struct AwQuery {
  static constexpr int NC = HD / 16;
  half8_t hi[NC], lo[HALF ? 1 : NC];

  // piece(i): 16 bytes of the lane's query, from element (HALF ? 8 : 4) i on. Returns the powers of two per
  // unit of raw score.
  template <class Piece>
  __device__ __forceinline__ float take(float scale, int h, Piece piece) {
    const float cs = scale * kLog2e;
    if constexpr (HALF) {
#pragma unroll
      for (int k = 0; k < NC; ++k) hi[k] = __builtin_bit_cast(half8_t, piece(2 * k + h));
      return cs;
    } else {
      typedef float f32x4_t __attribute__((ext_vector_type(4)));
      float amax = 0.f;
#pragma unroll
      for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const f32x4_t a = __builtin_bit_cast(f32x4_t, piece(4 * k + 2 * h + i));
          amax = fmaxf(amax, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w))));
        }
      amax = both_halves_max(amax);
      int e = 0;
      if (amax > 0.f && amax < INFINITY) {
        frexpf(amax, &e);                         // amax < 2^e
        e = min(max(14 - e, -114), 100);
      }
      const float up = ldexpf(1.f, e);
#pragma unroll
      for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const f32x4_t a = __builtin_bit_cast(f32x4_t, piece(4 * k + 2 * h + i));
#pragma unroll
          for (int l = 0; l < 4; ++l) {
            const float x = a[l] * up;
            const _Float16 top = (_Float16)x;
            hi[k][4 * i + l] = top;
            lo[k][4 * i + l] = (_Float16)(x - (float)top);
          }
        }
      return ldexpf(cs, -e);
    }
  }
};

// What takes a part's sums from its reference to the larger one that the parts are joined at. Never 0, so that
// an infinity (add_seen's) stays one where the part's largest score lies far below, or is -inf: a finite sum is
// below 2^57, and what 2^-126 leaves of it far below the other parts' rounding. A part without a key: its sums are 0.
__device__ __forceinline__ float aw_rescale(float from, float to) {
  return from == to ? 1.f : fmaxf(__builtin_amdgcn_exp2f(from - to), 0x1p-126f);
}

// A wave's running maximum, sums and outputs of its 32 columns. TWO: the probabilities' second plane.
template <int HD, bool HALF, bool TWO>
struct AwWave {
  static constexpr int NC = HD / 16, NDT = HD / 32;      // chunks of 16 dims; output tiles of 32
  f32x16_t o[NDT];
  float cs;                                      // powers of two per unit of raw score
  uint32_t finite;                               // zeros: halves that add_masked left out
  float m, l;                                    // the reference in raw scores; the sum of this lane's keys

  __device__ __forceinline__ void init(float cs_) {
    cs = cs_;
    m = -INFINITY;
    l = 0.f;
    finite = ~0u;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[dt][e] = 0.f;
  }

  // Scores of 32 keys: key(c) is chunk c of this lane's key row (the A operand: row j, dims 16 c + 8 h ..),
  // hi(c) and lo(c) of its queries. Register e of a lane is key 8 (e / 4) + 4 h + e % 4 of the column.
  template <class Key, class Hi, class Lo>
  __device__ __forceinline__ static f32x16_t scores(Key key, Hi hi, Lo lo) {
    f32x16_t s;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const half8_t a = key(c);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, hi(c), s, 0, 0, 0);
      if constexpr (!HALF) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, lo(c), s, 0, 0, 0);
    }
    return s;
  }

  // -inf at the keys that the column does not see; the bits of the others.
  __device__ __forceinline__ uint32_t mask(const AwBlock& b, int window, int t, int x0, int h, f32x16_t& s) const {
    uint32_t vis = 0;
    const int last = t - b.lo + b.ns;              // the number of the column's own position: key x is last - x before
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int x = x0 + 8 * (e >> 2) + 4 * h + (e & 3);
      const bool ok = x < b.ns ? x <= t : (unsigned)(last - x) < (unsigned)window;
      s[e] = ok ? s[e] : -INFINITY;
      vis |= (uint32_t)ok << e;
    }
    return vis;
  }

  // The reference follows the tile's maximum where that exceeds it by 2^8.
  __device__ __forceinline__ void raise(const f32x16_t& s) {
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[e]);
    mx = both_halves_max(mx);
    const bool up = (mx - m) * cs > kAwRaise;     // also the first key seen (m = -inf); not where none was
    if (__any(up)) {
      const float mn = up ? mx : m;
      // m = -inf: nothing summed yet (o and l are zero).
      const float corr = up && m > -INFINITY ? __builtin_amdgcn_exp2f((m - mn) * cs) : 1.f;
      l *= corr;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] *= corr;
      m = mn;
    }
  }

  // Probabilities in the B operand's layout: keys 16 kh + 4 h .. + 3 and 16 kh + 8 + 4 h .. + 3.
  __device__ __forceinline__ void probabilities(const f32x16_t& s, half8_t* ph, half8_t* pl) {
    // A column that has seen no key yet: every s is -inf, every probability 0.
    const float ref = kAwBias - (m == -INFINITY ? 0.f : m * cs);
#pragma unroll
    for (int kh = 0; kh < 2; ++kh) {
      uint32_t hi[4], lw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x2_t pe = {__builtin_amdgcn_exp2f(fmaf(s[8 * kh + 2 * i], cs, ref)),
                            __builtin_amdgcn_exp2f(fmaf(s[8 * kh + 2 * i + 1], cs, ref))};
        l += pe.x + pe.y;
        hi[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(pe, half2v_t));
        if constexpr (TWO) lw[i] = rest_h(hi[i], pe.x, pe.y);
      }
      ph[kh] = __builtin_bit_cast(half8_t, u32x4_t{hi[0], hi[1], hi[2], hi[3]});
      if constexpr (TWO) pl[kh] = __builtin_bit_cast(half8_t, u32x4_t{lw[0], lw[1], lw[2], lw[3]});
    }
  }

  // V^T rows 32 dt + j of a tile of V rows in LDS, in the probabilities' order of keys. tr (aw_tr): the lane's
  // place in the tile's first rows.
  __device__ __forceinline__ static half8_t values(uint32_t tr, int dt, int kh) {
    const uint32_t a0 = (tr ^ (uint32_t)(64 * dt)) + 16 * kh * AwLds<HD>::ROW;
    const half4_t x = lds_read_tr(a0), y = lds_read_tr(a0 + 8 * AwLds<HD>::ROW);
    return half8_t{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  }

  __device__ __forceinline__ void add(uint32_t tr, const half8_t* ph, const half8_t* pl) {
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int kh = 0; kh < 2; ++kh) {
        const half8_t a = values(tr, dt, kh);
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[kh], o[dt], 0, 0, 0);
        if constexpr (TWO) o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[kh], o[dt], 0, 0, 0);
      }
  }

  // The same where some key is hidden from some column. An infinity or NaN in its V must reach the
  // columns that see it and no other: it leaves the product (0 * inf is NaN), and add_seen puts it in at the end.
  __device__ __forceinline__ void add_masked(uint32_t tr, const half8_t* ph, const half8_t* pl) {
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int kh = 0; kh < 2; ++kh) {
        u32x4_t raw = __builtin_bit_cast(u32x4_t, values(tr, dt, kh));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t f = finite_h(raw[i]);
          raw[i] &= f;
          finite &= f;
        }
        const half8_t a = __builtin_bit_cast(half8_t, raw);
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[kh], o[dt], 0, 0, 0);
        if constexpr (TWO) o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[kh], o[dt], 0, 0, 0);
      }
  }

  // Whether a value was left out of a product, or a sum is infinite or NaN: an infinity's product with a
  // probability's second plane, or with one that vanished, is not the infinity that the sum has to hold.
  __device__ __forceinline__ bool stray() const {
    float z = 0.f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) z = fmaf(o[dt][e], 0.f, z);
    return __any(finite != ~0u || !(z == 0.f));
  }
  // Then: the sums without what is not finite, for add_seen. (NaN scores are in the sum of the probabilities.)
  __device__ __forceinline__ void drop_strays() {
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[dt][e] = fabsf(o[dt][e]) < INFINITY ? o[dt][e] : 0.f;
  }
  // The infinities and NaNs of the tile of keys from x0 on into the sums of the columns that see them, by a
  // product of their places with the keys seen: inf counts 1, -inf 64, NaN 4096, so 16 keys' counts do not mix.
  __device__ __forceinline__ void add_seen(const AwBlock& b, const AwRows<HD>& rows, int window, int t, int x0, int lane) {
    const int h = lane >> 5, j = lane & 31;
    f32x16_t none = {};
    const uint32_t vis = mask(b, window, t, x0, h, none);
#pragma unroll 1
    for (int kh = 0; kh < 2; ++kh) {
      const uint16_t* row[8];
      half8_t seen;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        long long fresh;
        const long long at = rows.row(b, x0 + 16 * kh + 8 * (i >> 2) + 4 * h + (i & 3), fresh);
        row[i] = (const uint16_t*)(rows.vc + at + (rows.vd & fresh)) + j;
        seen[i] = (_Float16)(float)(vis >> (8 * kh + i) & 1);
      }
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        half8_t at;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t v = row[i][32 * dt], n = v & 0x7FFFu;
          at[i] = (_Float16)(n < 0x7C00u ? 0.f : n > 0x7C00u ? 4096.f : v == n ? 1.f : 64.f);
        }
        const f32x16_t c = __builtin_amdgcn_mfma_f32_32x32x16_f16(at, seen, f32x16_t{}, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t n = (uint32_t)c[e];
          o[dt][e] += ((n & 63) ? INFINITY : 0.f) + ((n & 4032) ? -INFINITY : 0.f) + (n >> 12 ? NAN : 0.f);
        }
      }
    }
  }

  // The sums of WK waves that took other keys of the same columns, joined into those of wk = 0 through
  // jb (a barrier has passed since its memory was read last). True where this wave holds the result.
  static constexpr int W = NDT * 16 + 2;
  template <int WQ, int WK>
  __device__ __forceinline__ bool join(float* jb, int wq, int wk, int lane, float& mref) {
    if (wk > 0) {
      float* b = jb + (size_t)((wk - 1) * WQ + wq) * W * 64 + lane;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) b[(dt * 16 + e) * 64] = o[dt][e];
      b[(W - 2) * 64] = mref;
      b[(W - 1) * 64] = l;
    }
    __syncthreads();
    if (wk > 0) return false;
    float M = mref;
#pragma unroll
    for (int i = 0; i < WK - 1; ++i) M = fmaxf(M, jb[((size_t)(i * WQ + wq) * W + W - 2) * 64 + lane]);
    const float f0 = aw_rescale(mref, M);
    l *= f0;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[dt][e] *= f0;
#pragma unroll 1
    for (int i = 0; i < WK - 1; ++i) {
      const float* b = jb + (size_t)(i * WQ + wq) * W * 64 + lane;
      const float fi = aw_rescale(b[(W - 2) * 64], M);
      l += b[(W - 1) * 64] * fi;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] += b[(dt * 16 + e) * 64] * fi;
    }
    mref = M;
    return true;
  }

  // The outputs of the wave's columns, or with several splits their sums ([split][kv head][column], the
  // reference in powers of two and the sum behind all outputs). Through LDS (32 rows of HD + 4 floats of the
  // wave's own), so that a wave writes whole rows: 16 bytes of each of 64 rows at a time took the epilogue
  // four times as long.
  __device__ __forceinline__ void finish(const AttnWindowParams& p, const AwBlock& b, int first, int lane, float mref,
                                         float* own) const {
    constexpr int ST = HD + 4, L = HD / 4, CP = 64 / L;   // lanes a row; rows at a time
    const int h = lane >> 5, j = lane & 31;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int a4 = 0; a4 < 4; ++a4)
        *(float4*)(own + j * ST + dt * 32 + 8 * a4 + 4 * h) =
            make_float4(o[dt][4 * a4], o[dt][4 * a4 + 1], o[dt][4 * a4 + 2], o[dt][4 * a4 + 3]);
    if (h == 0) *(float2*)(own + j * ST + HD) = make_float2(mref, l);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    int col = first + lane / L, row = aw_row(p, col), in = col - row * p.rep;  // the column's position and head
    const int rows = aw_row(p, CP), heads = CP - rows * p.rep;
#pragma unroll 4
    for (int c = lane / L; c < 32; c += CP, col += CP) {
      if (col >= p.cols) break;
      const float4 x = *(const float4*)(own + c * ST + 4 * (lane % L));
      const float2 ml = *(const float2*)(own + c * ST + HD);
      put(p, b, col, row, b.g * p.rep + in, 4 * (lane % L), x, ml);
      row += rows;
      in += heads;
      if (in >= p.rep) in -= p.rep, ++row;
    }
  }
  // Four dims of a column: its output, or its split's sums (the lane of dim 0 also the reference and the sum).
  __device__ __forceinline__ static void put(const AttnWindowParams& p, const AwBlock& b, int col, int row, int head, int d0,
                                             const float4& x, const float2& ml) {
    if (p.nsplit > 1) {
      const size_t all = (size_t)p.nsplit * p.n_kv * p.cols, at = ((size_t)b.sp * p.n_kv + b.g) * p.cols + col;
      *(float4*)((float*)p.work + at * HD + d0) = x;
      if (d0 == 0) *((float2*)((float*)p.work + all * HD) + at) = ml;
      return;
    }
    const float inv = 1.0f / ml.y;
    float v[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
    const size_t orow = (size_t)row * p.out_stride + head * HD + d0;
    const size_t grow = (size_t)row * p.gate_stride + (size_t)head * p.gate_head_stride + d0;
    if constexpr (HALF) {
      if (p.gate) {
        const half4_t gv = *(const half4_t*)((const _Float16*)p.gate + grow);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] *= sigmoidf_((float)gv[k]);
      }
      *(half4_t*)((_Float16*)p.out + orow) = half4_t{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    } else {
      if (p.gate) {
        const float4 gv = *(const float4*)((const float*)p.gate + grow);
        v[0] *= sigmoidf_(gv.x);
        v[1] *= sigmoidf_(gv.y);
        v[2] *= sigmoidf_(gv.z);
        v[3] *= sigmoidf_(gv.w);
      }
      *(float4*)((float*)p.out + orow) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
};

// The lane's place in transposed reads of a tile of V rows at `tile`: key (lane / 4) % 4 + 4 h, dims
// 16 (lane / 16 % 2) + 4 (lane % 4), the row's swizzle applied (its tile begins at a multiple of 32 rows).
template <int HD>
__device__ __forceinline__ uint32_t aw_tr(uint32_t tile, int lane) {
  const int r = 4 * (lane >> 5) + ((lane >> 2) & 3);
  return tile + r * AwLds<HD>::ROW + (AwLds<HD>::v_swizzle(r) << 4) + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
}

// Many columns: WQ waves of columns times WK waves of keys. A stage of keys (32 for each of the WK) comes
// into LDS once, D stages ahead of its use, by loads that pass no registers; the scores of the next stage are
// taken while this one's exponentials run, so a stage's K comes with the V of the stage before. One barrier a
// stage: behind it the rows that the stage before last read are replaced.
// Bound by the matrix instructions and what of the vector and LDS work does not run beside them: a whole stage of
// 128 dims with fp32 queries takes 3.3k cycles, of which 2.1k are matrix instructions (fp16: 2.2k and 1.0k); the
// products reach 0.80 PFLOP/s over 1024 positions x 32 heads of 128 with a window of 2048 (two planes counted; the
// launch 86 us), 0.73 over 1021 with a window of 6000 and fp16 queries (139 us). Eight waves, so that a SIMD has
// two (four of 256 dims: a wave's registers). Tried and slower: two tiles of columns a wave (200 against 139 us
// then), two stages a barrier (equal), one of a SIMD's waves half a stage behind the other (98 against 90).
// What is rare stands outside the loop, which the instruction cache then holds: 64 against 28 KB of code were
// 95 against 88 us, and 15 us of 115 with 256 dims, where it had cost spilled registers.
template <int HD, bool HALF, int WQ, int WK, int D>
__global__ __launch_bounds__(64 * WQ * WK, WQ * WK / 4) void attn_window_kernel(AttnWindowParams p) {
  using Wave = AwWave<HD, HALF, !HALF>;
  using Lds = AwLds<HD>;
  constexpr int NW = WQ * WK;
  constexpr int SR = WK * kAwKeys;                // keys a stage
  constexpr int SEG = HD / 8, RPI = 64 / SEG;     // 16-byte pieces a row; rows a load of a wave
  constexpr int PP = SR / RPI / NW;               // a wave's loads of a stage's K (or V)
  static_assert(SR % (RPI * NW) == 0, "whole loads");
  constexpr int B = SR * Lds::ROW;                // bytes of a stage's K (or V)
  constexpr int RING = (D + 1) * B;               // of the stages held
  constexpr size_t OWN = (size_t)Wave::W * 64 * 4;
  constexpr size_t JOIN = (size_t)(WK > 1 ? WK - 1 : 1) * WQ * OWN;
  constexpr int QROW = HD * (HALF ? 2 : 4), QP = QROW / 16;  // bytes of a query; its 16-byte pieces
  constexpr size_t QB = (size_t)32 * WQ * QROW, KEEP = QB > JOIN ? QB : JOIN;
  __shared__ __align__(1024) uint8_t smem[2 * RING > KEEP ? 2 * RING : KEEP];

  int pos;
  if (!aw_pos(p, pos)) return;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), wq = w % WQ, wk = w / WQ;
  const int h = lane >> 5, j = lane & 31;
  const AwBlock b = aw_block(p, pos, 32 * WQ);
  const AwColumn c(p, b, b.c0 + 32 * wq, j);
  const AwRows<HD> rows(p, b.g);
  const int stages = (b.N + SR - 1) / SR;
  const int st0 = aw_share(stages, b.sp, p.nsplit), st1 = aw_share(stages, b.sp + 1, p.nsplit);
  const uint32_t ks = lds_address(smem), vs = ks + RING;

  // The block's queries come through LDS too, whole rows at a time and once for the WK waves: 16 bytes of each
  // of 32 rows at a time, by every wave, took as long as five stages.
  AwQuery<HD, HALF> q;
  Wave v;
  {
    auto swizzle = [](int r) { return QP >= 16 ? r & 15 : r >> 1 & 7; };
    for (int i = w; i < (int)(QB / 1024); i += NW) {
      const int r = (64 * i + lane) / QP, piece = lane % QP, col = min(b.c0 + r, p.cols - 1), row = aw_row(p, col);
      const size_t at = (size_t)row * p.q_stride + (b.g * p.rep + col - row * p.rep) * HD;
      load_lds16(ks + 1024 * i, (const char*)p.q + at * (HALF ? 2 : 4) + 16 * (piece ^ swizzle(r)));
    }
    wait_loads_and_block<0>();
    const uint32_t mine = ks + (32 * wq + j) * QROW;
    v.init(q.take(p.scale, h, [&](int i) { return __builtin_bit_cast(u32x4_t, lds_half8(mine + 16 * (i ^ swizzle(j)))); }));
    wait_loads_and_block<0>();
  }

  // Load i of a wave: rows RPI (w + i NW) .. of the stage, a lane's piece of them. Stages of evenly spaced
  // rows (all but a few) follow each other by one addition: the address arithmetic of every stage took a
  // quarter of its time.
  constexpr int NO = HD == 256 && NW == 4 ? 2 : 1;  // loads after which a row's swizzle is the same again
  struct Stream {
    const char* base;                             // the stage's first row
    uint32_t step;                                // bytes from row to row
    int left;                                     // stages to come that follow evenly
    uint32_t off[NO];                             // a lane's pieces
  };
  auto send = [&](const Stream& f, uint32_t lds) AW_INLINE {
#pragma unroll
    for (int i = 0; i < PP; ++i)
      load_lds16(lds + 1024 * (w + i * NW), uniform(f.base + (size_t)f.step * (i / NO * NO * RPI * NW)), f.off[i % NO]);
  };
  auto next = [&](Stream& f, uint32_t lds) AW_INLINE {
    f.base += (size_t)f.step * SR;
    send(f, lds);
  };
  auto load = [&](int st, Stream& f, const char* ring, long long dist, uint32_t lds, auto swizzle) AW_INLINE {
    if (f.left > 0) {
      --f.left;
      next(f, lds);
      return;
    }
    long long at = 0;
    bool own = false;
    uint32_t step = 0;
    f.left = rows.flat(b, st * SR, SR, at, own, step) - 1;
    const int lrow = lane / SEG, lpiece = lane % SEG;
    if (f.left < 0) {
#pragma unroll 1
      for (int i = 0; i < PP; ++i) {
        const int r = RPI * (w + i * NW) + lrow;
        long long fresh;
        const long long row = rows.row(b, st * SR + r, fresh);
        load_lds16(lds + 1024 * (w + i * NW), ring + row + (dist & fresh) + 16 * (lpiece ^ swizzle(r)));
      }
      return;
    }
    f.base = uniform(ring + at + (own ? dist : 0));
    f.step = __builtin_amdgcn_readfirstlane(step);
#pragma unroll
    for (int i = 0; i < NO; ++i) {
      const int r = RPI * (w + i * NW) + lrow;
      f.off[i] = (uint32_t)r * step + 16 * (lpiece ^ swizzle(r));
    }
    send(f, lds);
  };
  // Stage st's rows take the places in turn. The K of a stage past the last one are its last key's.
  Stream fk, fv;
  fk.left = fv.left = 0;
  auto load_k = [&](int st, uint32_t at) AW_INLINE { load(st, fk, rows.kc, rows.kd, ks + at, Lds::k_swizzle); };
  auto load_v = [&](int st, uint32_t at) AW_INLINE { load(st, fv, rows.vc, rows.vd, vs + at, Lds::v_swizzle); };
  auto after = [](uint32_t at) { return at + B >= (uint32_t)RING ? 0u : at + B; };
  uint32_t kl = D * B, vl = D * B;                // places of the next rows to be loaded
  if (st0 < st1) {
    load_k(st0, 0);
    load_v(st0, 0);
    load_k(st0 + 1, B);
    if (D == 2 && st0 + 1 < st1) {
      load_v(st0 + 1, B);
      load_k(st0 + 2, 2 * B);
    }
    kl = 0;                                       // K of stage st0 + D + 1: st0's place
  }
  // This lane's key row of a stage (its pieces are places apart by their bits), and its place in V.
  const uint32_t kt = ks + (wk * kAwKeys + j) * Lds::ROW + 16 * (h ^ Lds::k_swizzle(j));
  const uint32_t tr = aw_tr<HD>(vs + wk * kAwKeys * Lds::ROW, lane);
  uint32_t kp = 0, vp = 0;                        // places of the next stage's K and of this one's V
  f32x16_t s = {};
  auto scores = [&]() AW_INLINE {
    const uint32_t k = kt + kp;
    kp = after(kp);
    return Wave::scores([&](int c) { return lds_half8(k ^ (32 * c)); }, [&](int c) { return q.hi[c]; },
                        [&](int c) { return q.lo[HALF ? 0 : c]; });
  };
  auto mask = [&](int st) AW_INLINE { v.mask(b, p.window, c.t, st * SR + wk * kAwKeys, h, s); };
  // Stages whose keys every column of the wave sees whole: [a0, a1). The others, at the sinks and at both ends
  // of the window, mask their scores.
  const int first = wk * kAwKeys - b.ns + b.lo;   // position of stage st's first key of the wave: first + SR st
  const int a0 = min(st1, max(st0, (max(b.lo, c.w_last - p.window + 1) - first + SR - 1) / SR));
  const int a1 = max(a0, min(st1, c.w_first + 1 - kAwKeys < first ? 0 : (c.w_first + 1 - kAwKeys - first) / SR + 1));
  if (st0 < st1) {
    wait_loads_and_block<0>();
    s = scores();
    mask(st0);
  }
  // Before stage st: its V and the next stage's K are there for every wave, and the rows D stages on take the
  // place of the ones that the stage before it read.
  auto stage = [&](int st) AW_INLINE {
    if (D == 2 && st + 1 < st1) wait_loads_and_block<2 * PP>();
    else wait_loads_and_block<0>();
    if (st + D < st1) {
      load_v(st + D, vl);
      load_k(st + D + 1, kl);
      vl = after(vl);
      kl = after(kl);
    }
  };
  half8_t ph[2], pl[2];
  for (int st = st0; st < st1; ++st) {
    // Whole stages while the rows to be loaded follow evenly: no branches, so that the loads and what they need
    // stand among the products. (The last whole stage's next scores may need a mask: it is not among these. The
    // rows may go past the split's last stage, not past the block's keys.)
    int flow = st < a0 ? 0 : min(a1 - 1 - st, min(fk.left, fv.left));
    if (flow > 0) {
      fk.left -= flow;
      fv.left -= flow;
      st += flow;
      for (; flow > 0; --flow) {
        wait_loads_and_block<D == 2 ? 2 * PP : 0>();
        v.raise(s);
        const f32x16_t s1 = scores();
        next(fv, vs + vl);
        next(fk, ks + kl);
        vl = after(vl);
        kl = after(kl);
        v.probabilities(s, ph, pl);
        v.add(tr + vp, ph, pl);
        vp = after(vp);
        s = s1;
      }
    }
    stage(st);
    v.raise(s);
    v.probabilities(s, ph, pl);
    v.add_masked(tr + vp, ph, pl);
    vp = after(vp);
    if (st + 1 < st1) {
      s = scores();
      mask(st + 1);
    }
  }
  if (v.stray()) {
    v.drop_strays();
    for (int st = st0; st < st1; ++st) v.add_seen(b, rows, p.window, c.t, st * SR + wk * kAwKeys, lane);
  }
  v.l += __shfl_xor(v.l, 32, 64);
  float mref = v.m == -INFINITY ? -INFINITY : v.m * v.cs;
  // Every wave's reads are done, and the K loaded past the last stage has arrived.
  wait_loads_and_block<0>();
  if constexpr (WK > 1)
    if (!v.template join<WQ, WK>((float*)smem, wq, wk, lane, mref)) return;
  v.finish(p, b, b.c0 + 32 * wq, lane, mref, (float*)(smem + wq * OWN));
}

// Few columns (a token, a short turn): the keys are the long axis. Each of a block's four waves takes 32
// keys at a time by itself, without barriers: its K rows come straight into the operand's registers, its V
// rows through LDS of its own (to be read transposed), both one tile ahead; the queries, the same for
// all four, lie in LDS to leave the registers to the rows. Bound by the rows' latency and
// bytes, the joins and, for short windows, the two launches: one position over 32768 keys (134 MB) 26 us, 5.3 TB/s,
// and 6 in the second launch; over 1024 keys (4.2 MB) 10 and 3.
template <int HD, bool HALF>
__global__ __launch_bounds__(256, 1) void attn_window_few_kernel(AttnWindowParams p) {
  using Wave = AwWave<HD, HALF, true>;
  using Lds = AwLds<HD>;
  constexpr int WK = 4, SEG = HD / 8;
  constexpr int PP = kAwKeys * SEG / 64, RPP = 64 / SEG;  // a lane's 16-byte pieces of V; rows between them
  constexpr int VB = kAwKeys * Lds::ROW, QS = HD + 8;
  constexpr int QROW = HD * (HALF ? 2 : 4), QP = QROW / 16;  // bytes of a query; its 16-byte pieces
  constexpr size_t STAGE = (size_t)WK * VB, PLANES = (HALF ? 1 : 2) * 32 * QS * 2, JOIN = (size_t)WK * 64 * Wave::W * 4;
  static_assert(32 * QROW <= STAGE, "the queries as they come fit where the V rows will be");
  __shared__ __align__(1024) uint8_t smem[STAGE + PLANES > JOIN ? STAGE + PLANES : JOIN];
  _Float16* const qs = (_Float16*)(smem + STAGE);

  int pos;
  if (!aw_pos(p, pos)) return;
  const int lane = threadIdx.x & 63, wk = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5, j = lane & 31;
  const AwBlock b = aw_block(p, pos, 32);
  const AwColumn c(p, b, b.c0, j);
  const AwRows<HD> rows(p, b.g);
  const int tiles = (b.N + kAwKeys - 1) / kAwKeys;
  const int i0 = aw_share(tiles, b.sp, p.nsplit) + wk, i1 = aw_share(tiles, b.sp + 1, p.nsplit);
  const int columns = min(32, p.cols - b.c0), mine = min(j, columns - 1);
  uint8_t* const vs = smem + wk * VB;
  const int srow = lane / SEG, piece = lane % SEG;
  const uint32_t tr = aw_tr<HD>(lds_address(vs), lane);

  half8_t kf[Wave::NC];
  u32x4_t vr[PP];
  long long at = 0;                               // of the lane's key: its row's distance, and 1 if it is the call's own
  auto load_k = [&](int i) AW_INLINE {
    long long fresh;
    at = rows.row(b, i * kAwKeys + j, fresh) - fresh;
    const char* r = rows.kc + (at + fresh) + (rows.kd & fresh) + 16 * h;
#pragma unroll
    for (int k = 0; k < Wave::NC; ++k) kf[k] = *(const half8_t*)(r + 32 * k);
  };
  auto load_v = [&](int) AW_INLINE {              // the tile that load_k took last
#pragma unroll
    for (int k = 0; k < PP; ++k) {
      if (k % 4 == 0) __builtin_amdgcn_sched_barrier(0);  // (a few addresses at a time)
      const long long a = __shfl(at, srow + k * RPP, 64);
      vr[k] = *(const u32x4_t*)(rows.vc + (a & ~1ll) + (rows.vd & -(a & 1)) + 16 * piece);
    }
  };
  // The queries there are, whole rows at a time, into LDS, beside the first rows; then their planes.
  auto swizzle = [](int r) { return QP >= 16 ? r & 15 : r >> 1 & 7; };
  for (int i = wk; 1024 * i < columns * QROW; i += WK) {
    const int r = min((64 * i + lane) / QP, columns - 1), row = aw_row(p, b.c0 + r);
    const size_t at = (size_t)row * p.q_stride + (b.g * p.rep + b.c0 + r - row * p.rep) * HD;
    load_lds16(lds_address(smem) + 1024 * i, (const char*)p.q + at * (HALF ? 2 : 4) + 16 * (lane % QP ^ swizzle((64 * i + lane) / QP)));
  }
  if (i0 < i1) {
    load_k(i0);
    load_v(i0);
  }
  wait_loads_and_block<0>();
  Wave v;
  {
    AwQuery<HD, HALF> q;
    const uint32_t at = lds_address(smem) + mine * QROW;
    v.init(q.take(p.scale, h, [&](int i) { return __builtin_bit_cast(u32x4_t, lds_half8(at + 16 * (i ^ swizzle(mine)))); }));
#pragma unroll
    for (int k = 0; k < Wave::NC; ++k)
      if (k % WK == wk) {
        *(half8_t*)(qs + j * QS + 16 * k + 8 * h) = q.hi[k];
        if constexpr (!HALF) *(half8_t*)(qs + 32 * QS + j * QS + 16 * k + 8 * h) = q.lo[k];
      }
  }
  __syncthreads();
  const _Float16* const qr = qs + j * QS + 8 * h;
  for (int i = i0; i < i1; i += WK) {
    f32x16_t s = Wave::scores([&](int k) { return kf[k]; }, [&](int k) { return *(const half8_t*)(qr + 16 * k); },
                              [&](int k) { return *(const half8_t*)(qr + 32 * QS + 16 * k); });
    const bool more = i + WK < i1;
    if (more) load_k(i + WK);
    // Whether every column of the wave sees every key (a second form of the products is more than the registers
    // hold with 256 dims).
    const int x0 = i * kAwKeys, u0 = x0 - b.ns + b.lo;
    const bool whole = HD < 256 && x0 >= b.ns && u0 > c.w_last - p.window && u0 <= c.w_first - (kAwKeys - 1);
    if (!whole) v.mask(b, p.window, c.t, x0, h, s);
    v.raise(s);
    half8_t ph[2], pl[2];
    v.probabilities(s, ph, pl);
    // The wave's own tile: its stores before its reads, its last reads (their products issued) before these
    // stores; LDS serves a wave in order.
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int k = 0; k < PP; ++k)
      *(u32x4_t*)(vs + (srow + k * RPP) * Lds::ROW + 16 * (piece ^ Lds::v_swizzle(srow + k * RPP))) = vr[k];
    if (more) load_v(i + WK);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (whole) v.add(tr, ph, pl);
    else v.add_masked(tr, ph, pl);
  }
  if (v.stray()) {
    v.drop_strays();
    for (int i = i0; i < i1; i += WK) v.add_seen(b, rows, p.window, c.t, i * kAwKeys, lane);
  }
  v.l += __shfl_xor(v.l, 32, 64);
  float mref = v.m == -INFINITY ? -INFINITY : v.m * v.cs;
  // The four waves' sums joined, each wave's share of the dims.
  __syncthreads();                                // every wave's reads are done
  float* const jb = (float*)smem + lane;
  if (j < columns) {
    float* const to = jb + (size_t)wk * Wave::W * 64;
#pragma unroll
    for (int dt = 0; dt < Wave::NDT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) to[(dt * 16 + e) * 64] = v.o[dt][e];
    to[(Wave::W - 2) * 64] = mref;
    to[(Wave::W - 1) * 64] = v.l;
  }
  __syncthreads();
  if (j >= columns) return;
  float M = -INFINITY, l = 0.f, f[WK];
#pragma unroll
  for (int i = 0; i < WK; ++i) M = fmaxf(M, f[i] = jb[((size_t)i * Wave::W + Wave::W - 2) * 64]);
#pragma unroll
  for (int i = 0; i < WK; ++i) {
    f[i] = aw_rescale(f[i], M);
    l += jb[((size_t)i * Wave::W + Wave::W - 1) * 64] * f[i];
  }
  constexpr int OWN = Wave::NDT >= WK ? Wave::NDT / WK : 1;
#pragma unroll
  for (int d = 0; d < OWN; ++d) {
    const int dt = wk * OWN + d;
    if (dt >= Wave::NDT) return;
    float x[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = 0.f;
#pragma unroll
    for (int i = 0; i < WK; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] += jb[((size_t)i * Wave::W + dt * 16 + e) * 64] * f[i];
#pragma unroll
    for (int a4 = 0; a4 < 4; ++a4)
      Wave::put(p, b, b.c0 + j, c.row, c.head, dt * 32 + 8 * a4 + 4 * h,
                make_float4(x[4 * a4], x[4 * a4 + 1], x[4 * a4 + 2], x[4 * a4 + 3]), make_float2(M, l));
  }
}

// After the attention: the splits of each (position, head) joined (a wave each, blocks of four), and
// the call's last rows of K and V into their slots.
template <int HD, bool HALF>
__global__ __launch_bounds__(256) void attn_window_finish(AttnWindowParams p, int join_blocks) {
  int pos;
  if (!aw_pos(p, pos)) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if ((int)blockIdx.x < join_blocks) {
    constexpr int E = HD / 64;                     // dims a lane: E lane .. + E - 1
    const unsigned id = blockIdx.x * 4 + w;         // below 2^25 + 4
    if (id >= (unsigned)(p.n * p.n_head)) return;
    const int row = (int)(id / (unsigned)p.n_head), head = (int)id - row * p.n_head, g = aw_row(p, head);
    const int col = row * p.rep + head - g * p.rep;
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
