// The tiles of attention on the matrix cores that the operators over KV caches share (trx_attn_window.hip,
// trx_attn_rows.hip): columns, which are (position, head) pairs of one kv head, against tiles of 32 keys, with a
// running maximum and sum. The mathematics and the precision stand in trx_attn_window.hip.
//
// Where the keys lie and which column sees which is a class Layout's, with
//   Params: q, gate, out, their strides, scale, work, rep and n_kv, nsplit (parts of a column's keys), cols (all
//     columns of a kv head), and rep_m, rep_s for the division by rep;
//   Block: g, its kv head; c0 and end, its first column and that behind the last one; N, its keys, numbered
//     0 .. N - 1; split of splits, its share of them, and sp, the part that its sums are;
//   Rows: the places of the keys' rows (row, flat); Column: row, head and the columns it stands with;
//   block (false: nothing to do), sight (whether a column sees a key), whole (stages that every column of a wave
//     sees whole), all_see (one tile); and what a layout may keep of the work: query (a chunk of a wave's, as operands),
//     scored (a tile's scores, in calls of few columns), total (of a column that one block finishes: its maximum and
//     sum);
//   TWO: whether fp16 calls of many columns take the probabilities' second plane, as all others do.
#pragma once

#include "trx_internal.h"

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
template <class Params>
__device__ __forceinline__ int aw_row(const Params& p, int column) {
  return (int)((unsigned long long)(unsigned)column * p.rep_m >> p.rep_s);
}
// The first of a split's share of `count` stages (count times splits below 2^32).
__device__ __forceinline__ int aw_share(int count, int split, int splits) {
  return (int)((unsigned)count * (unsigned)split / (unsigned)splits);
}

// The queries of a wave's columns in the B operand's layout: dims 16 c + 8 h .. + 7.
template <int HD, bool HALF>
struct AwQuery {
  static constexpr int NC = HD / 16;
  typedef float f32x4_t __attribute__((ext_vector_type(4)));
  half8_t hi[NC], lo[HALF ? 1 : NC];

  // piece(i): 16 bytes of the lane's query, from element (HALF ? 8 : 4) i on. The powers of two per unit of raw score,
  // and what the elements are multiplied by before they are rounded.
  template <class Piece>
  __device__ __forceinline__ static float unit(float scale, int h, Piece piece, float& up) {
    const float cs = scale * kLog2e;
    up = 1.f;
    if constexpr (HALF) return cs;
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
      frexpf(amax, &e);                           // amax < 2^e
      e = min(max(14 - e, -114), 100);
    }
    up = ldexpf(1.f, e);
    return ldexpf(cs, -e);
  }
  // Chunk k of both planes.
  template <class Piece>
  __device__ __forceinline__ static void chunk(int k, int h, float up, Piece piece, half8_t& hi, half8_t& lo) {
    if constexpr (HALF) {
      hi = __builtin_bit_cast(half8_t, piece(2 * k + h));
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const f32x4_t a = __builtin_bit_cast(f32x4_t, piece(4 * k + 2 * h + i));
#pragma unroll
        for (int l = 0; l < 4; ++l) {
          const float x = a[l] * up;
          const _Float16 top = (_Float16)x;
          hi[4 * i + l] = top;
          lo[4 * i + l] = (_Float16)(x - (float)top);
        }
      }
    }
  }
  template <class Piece>
  __device__ __forceinline__ float take(float scale, int h, Piece piece) {
    float up;
    const float cs = unit(scale, h, piece, up);
#pragma unroll
    for (int k = 0; k < NC; ++k) chunk(k, h, up, piece, hi[k], lo[HALF ? 0 : k]);
    return cs;
  }
};

// What takes a part's sums from its reference to the larger one that the parts are joined at. Never 0, so that
// an infinity (add_seen's) stays one where the part's largest score lies far below, or is -inf: a finite sum is
// below 2^57, and what 2^-126 leaves of it far below the other parts' rounding. A part without a key: its sums are 0.
__device__ __forceinline__ float aw_rescale(float from, float to) {
  return from == to ? 1.f : fmaxf(__builtin_amdgcn_exp2f(from - to), 0x1p-126f);
}

// A wave's running maximum, sums and outputs of its 32 columns. TWO: the probabilities' second plane.
template <class Layout, int HD, bool HALF, bool TWO>
struct AwWave {
  using Params = typename Layout::Params;
  using Block = typename Layout::Block;
  using Rows = typename Layout::Rows;
  using Column = typename Layout::Column;
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
  __device__ __forceinline__ uint32_t mask(const Params& p, const Block& b, const Column& c, int x0, int h, f32x16_t& s) const {
    uint32_t vis = 0;
    const auto sight = Layout::sight(p, b, c);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const bool ok = sight(x0 + 8 * (e >> 2) + 4 * h + (e & 3));
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
  __device__ __forceinline__ void add_seen(const Params& p, const Block& b, const Rows& rows, const Column& c, int x0, int lane) {
    const int h = lane >> 5, j = lane & 31;
    f32x16_t none = {};
    const uint32_t vis = mask(p, b, c, x0, h, none);
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
        const f32x16_t found = __builtin_amdgcn_mfma_f32_32x32x16_f16(at, seen, f32x16_t{}, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t n = (uint32_t)found[e];
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
  __device__ __forceinline__ void finish(const Params& p, const Block& b, int first, int lane, float mref, float* own) const {
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
      if (col >= b.end) break;
      const float4 x = *(const float4*)(own + c * ST + 4 * (lane % L));
      const float2 ml = *(const float2*)(own + c * ST + HD);
      put(p, b, col, row, b.g * p.rep + in, 4 * (lane % L), x, ml);
      row += rows;
      in += heads;
      if (in >= p.rep) in -= p.rep, ++row;
    }
  }
  // Four dims of a column: its output, or its split's sums (the lane of dim 0 also the reference and the sum).
  __device__ __forceinline__ static void put(const Params& p, const Block& b, int col, int row, int head, int d0, const float4& x,
                                             const float2& ml) {
    if (p.nsplit > 1) {
      const size_t all = (size_t)p.nsplit * p.n_kv * p.cols, at = ((size_t)b.sp * p.n_kv + b.g) * p.cols + col;
      *(float4*)((float*)p.work + at * HD + d0) = x;
      if (d0 == 0) *((float2*)((float*)p.work + all * HD) + Layout::sum_at(p, b, col, at)) = ml;
      return;
    }
    if (d0 == 0) Layout::total(p, b, col, ml);
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
template <class Layout, int HD, bool HALF, int WQ, int WK, int D>
__device__ __forceinline__ void aw_many(const typename Layout::Params& p) {
  using Wave = AwWave<Layout, HD, HALF, !HALF || Layout::TWO>;
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

  typename Layout::Block b;
  if (!Layout::block(p, 32 * WQ, b)) return;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), wq = w % WQ, wk = w / WQ;
  const int h = lane >> 5, j = lane & 31;
  const typename Layout::Column c(p, b, b.c0 + 32 * wq, j);
  const typename Layout::Rows rows(p, b);
  const int stages = (b.N + SR - 1) / SR;
  const int st0 = aw_share(stages, b.split, b.splits), st1 = aw_share(stages, b.split + 1, b.splits);
  const uint32_t ks = lds_address(smem), vs = ks + RING;

  // The block's queries come through LDS too, whole rows at a time and once for the WK waves: 16 bytes of each
  // of 32 rows at a time, by every wave, took as long as five stages.
  AwQuery<HD, HALF> q;
  Wave v;
  {
    auto swizzle = [](int r) { return QP >= 16 ? r & 15 : r >> 1 & 7; };
    for (int i = w; i < (int)(QB / 1024); i += NW) {
      const int r = (64 * i + lane) / QP, piece = lane % QP, col = min(b.c0 + r, b.end - 1), row = aw_row(p, col);
      const size_t at = (size_t)row * p.q_stride + (b.g * p.rep + col - row * p.rep) * HD;
      load_lds16(ks + 1024 * i, (const char*)p.q + at * (HALF ? 2 : 4) + 16 * (piece ^ swizzle(r)));
    }
    wait_loads_and_block<0>();
    const uint32_t mine = ks + (32 * wq + j) * QROW;
    v.init(q.take(p.scale, h, [&](int i) { return __builtin_bit_cast(u32x4_t, lds_half8(mine + 16 * (i ^ swizzle(j)))); }));
    if (wk == 0) {
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) Layout::query(p, b, b.c0 + 32 * wq, lane, k, q.hi[k], q.lo[HALF ? 0 : k], v.cs);
    }
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
  auto mask = [&](int st) AW_INLINE { v.mask(p, b, c, st * SR + wk * kAwKeys, h, s); };
  // Stages whose keys every column of the wave sees whole: [a0, a1). The others, at the sinks and at both ends
  // of the window, mask their scores.
  int a0, a1;
  Layout::whole(p, b, c, wk * kAwKeys, SR, a0, a1);
  a0 = min(st1, max(st0, a0));
  a1 = max(a0, min(st1, a1));
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
    for (int st = st0; st < st1; ++st) v.add_seen(p, b, rows, c, st * SR + wk * kAwKeys, lane);
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
template <class Layout, int HD, bool HALF>
__device__ __forceinline__ void aw_few(const typename Layout::Params& p) {
  using Wave = AwWave<Layout, HD, HALF, true>;
  using Lds = AwLds<HD>;
  constexpr int WK = 4, SEG = HD / 8;
  constexpr int PP = kAwKeys * SEG / 64, RPP = 64 / SEG;  // a lane's 16-byte pieces of V; rows between them
  constexpr int VB = kAwKeys * Lds::ROW, QS = HD + 8;
  constexpr int QROW = HD * (HALF ? 2 : 4), QP = QROW / 16;  // bytes of a query; its 16-byte pieces
  constexpr size_t STAGE = (size_t)WK * VB, PLANES = (HALF ? 1 : 2) * 32 * QS * 2, JOIN = (size_t)WK * 64 * Wave::W * 4;
  static_assert(32 * QROW <= STAGE, "the queries as they come fit where the V rows will be");
  __shared__ __align__(1024) uint8_t smem[STAGE + PLANES > JOIN ? STAGE + PLANES : JOIN];
  _Float16* const qs = (_Float16*)(smem + STAGE);

  typename Layout::Block b;
  if (!Layout::block(p, 32, b)) return;
  const int lane = threadIdx.x & 63, wk = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5, j = lane & 31;
  const typename Layout::Column c(p, b, b.c0, j);
  const typename Layout::Rows rows(p, b);
  const int tiles = (b.N + kAwKeys - 1) / kAwKeys;
  const int i0 = aw_share(tiles, b.split, b.splits) + wk, i1 = aw_share(tiles, b.split + 1, b.splits);
  const int columns = min(32, b.end - b.c0), mine = min(j, columns - 1);
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
    // (Each wave a share of the chunks: all of them by every wave took 1 us with 256 dims.)
    using Query = AwQuery<HD, HALF>;
    const uint32_t at = lds_address(smem) + mine * QROW;
    auto piece = [&](int i) AW_INLINE { return __builtin_bit_cast(u32x4_t, lds_half8(at + 16 * (i ^ swizzle(mine)))); };
    float up;
    v.init(Query::unit(p.scale, h, piece, up));
#pragma unroll
    for (int i = 0; i < Wave::NC / WK; ++i) {
      const int k = WK * i + wk;
      half8_t hi, lo;
      Query::chunk(k, h, up, piece, hi, lo);
      *(half8_t*)(qs + j * QS + 16 * k + 8 * h) = hi;
      if constexpr (!HALF) *(half8_t*)(qs + 32 * QS + j * QS + 16 * k + 8 * h) = lo;
      Layout::query(p, b, b.c0, lane, k, hi, lo, v.cs);
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
    const int x0 = i * kAwKeys;
    const bool whole = HD < 256 && Layout::all_see(p, b, c, x0);
    if (!whole) v.mask(p, b, c, x0, h, s);
    if (j < columns) Layout::scored(p, b, b.c0 + j, x0 + 4 * h, s, v.cs);
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
    for (int i = i0; i < i1; i += WK) v.add_seen(p, b, rows, c, i * kAwKeys, lane);
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
}  // namespace trx
