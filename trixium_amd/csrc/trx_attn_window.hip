// Attention of the next n positions over a KV ring, with a sliding window and a few first positions
// that stay visible (sinks). A query at position t sees V(t) = {u <= t : u < sinks or u > t - window}:
//   o_t = sum_{u in V(t)} e^{scale q_t.k_u - m} v_u / sum_{u in V(t)} e^{scale q_t.k_u - m},
// m the largest score, one pass over the keys with a running maximum and sum.
//
// Columns: a (position, head of the kv head) pair each, 32 a wave, so the heads that share K and V
// read them once. A block takes WQ waves of columns times WK waves of keys: every stage of
// WK * 32 keys goes into LDS once, the WK waves of a column take 32 of them each, and are joined at the
// end. With few columns (WQ = 1) the keys are the long axis: they are split over the block's waves
// and over blocks, joined by attn_window_finish.
// The keys any query of the block sees are numbered in order (the sinks, then the window from the
// first query's on): tiles of that numbering never hold rows outside it, whatever the ring's seam.
//
// Products on the matrix cores (v_mfma_f32_32x32x16_f16), K and V as the ring holds them:
//   S^T = K Q^T: fp32 queries enter as two fp16 planes of q * 2^e (e per query: the largest element
//   below 2^14), so a score is the fp32 dot product to 2^-22; fp16 queries as they are.
//   O^T += V^T P^T: P^T stands in the score registers in the operand's layout but for the order of
//   the keys, which V^T, read transposed from LDS, follows. fp32 outputs: P in two fp16 planes
//   (2^-22); fp16 outputs: one (2^-12 a probability at most, a quarter step of the output, and
//   independent from key to key).
// Probabilities are 2^(s - r + 7) against a reference r that follows the running maximum only where
// that exceeds it by 2^8: at most 2^15 (finite in fp16), and those that vanish in fp16 are below 2^-32
// of the largest.

#include "trx_attn_window.h"

#include <algorithm>
#include <limits.h>

namespace trx {

constexpr int kAwKeys = 32;                 // keys per wave and stage
constexpr float kAwBias = 7.f;              // log2 of the largest probability's fp16 value, less 8
constexpr float kAwRaise = 8.f;
constexpr float kLog2e = 1.44269504088896341f;

typedef _Float16 half2v_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

// LDS row strides in halves. K rows are read 16 bytes a lane, a row a lane: one 16-byte step a row
// spreads them over the banks. V rows are read transposed, 64 bytes of a row by each 8 lanes: rows 64
// bytes apart modulo the 256 of the banks.
template <int HD> struct AwLds {
  static constexpr int KS = HD + 8, VS = HD + 32;
};

// Four consecutive keys of one dim a lane: within 16 lanes, lane l gives the address of key l / 4, dims
// 4 (l % 4) .. + 3, and takes dim l of the four keys.
__device__ __forceinline__ half4_t lds_read_tr(const _Float16* p) {
  typedef __attribute__((address_space(3))) s16x4_t lds_t;
  const s16x4_t r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(__attribute__((address_space(3))) void*)p);
  return __builtin_bit_cast(half4_t, r);
}

// The first position, and whether the call has positions that the ring's arithmetic holds.
__device__ __forceinline__ bool aw_pos(const AttnWindowParams& p, int& pos) {
  pos = p.pos_dev ? *p.pos_dev : p.pos;
  return pos >= 0 && pos <= INT_MAX - p.n;
}

__device__ __forceinline__ bool nonfinite_h(uint32_t two) {
  return (two & 0x7C00u) == 0x7C00u || (two & 0x7C000000u) == 0x7C000000u;
}

template <int HD, bool HALF, int WQ, int WK, int NBUF>
__global__ __launch_bounds__(64 * WQ * WK, WQ * WK / 4) void attn_window_kernel(AttnWindowParams p) {
  constexpr int T = 64 * WQ * WK;                 // threads
  constexpr int SR = WK * kAwKeys;                // keys a stage
  constexpr int KS = AwLds<HD>::KS, VS = AwLds<HD>::VS;
  constexpr int NC = HD / 16, NDT = HD / 32;      // chunks of 16 dims; output tiles of 32
  constexpr int SEG = HD / 8, PP = SR * SEG / T;  // 16-byte pieces a row; a thread's pieces
  static_assert(SR * SEG % T == 0 && T % SEG == 0, "whole pieces");
  constexpr int RPP = T / SEG;                    // rows between a thread's pieces
  constexpr int KB = SR * KS, VB = SR * VS;       // halves of a buffer
  constexpr size_t JOIN = (size_t)(WK - 1) * WQ * 64 * (NDT * 16 + 2) * 4;
  constexpr size_t STAGE = (size_t)NBUF * (KB + VB) * 2;
  __shared__ __align__(16) uint8_t smem[STAGE > JOIN ? STAGE : JOIN];
  _Float16* const ks = (_Float16*)smem;
  _Float16* const vs = ks + NBUF * KB;

  int pos;
  if (!aw_pos(p, pos)) return;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, wq = w % WQ, wk = w / WQ;
  const int h = lane >> 5, j = lane & 31;
  // A kv head's blocks stay on the XCDs of its number (blocks go round-robin over them): its K and V
  // are read into few L2s.
  const int g = blockIdx.x % p.n_kv, rest = blockIdx.x / p.n_kv;
  const int sp = rest % p.nsplit, qt = rest / p.nsplit;
  const int c0 = qt * 32 * WQ;                    // the block's first column
  const int rep = p.rep, last_col = p.cols - 1;
  const int t_first = pos + c0 / rep, t_last = pos + min(c0 + 32 * WQ - 1, last_col) / rep;
  const int ns = min(p.sinks, t_last + 1);
  const int lo = max(ns, t_first - p.window + 1);
  const int N = ns + (t_last + 1 - lo);
  const int stages = (N + SR - 1) / SR;
  const int st0 = (int)((long long)stages * sp / p.nsplit), st1 = (int)((long long)stages * (sp + 1) / p.nsplit);

  // This lane's column, and the range of positions of the wave's columns.
  const int cw = c0 + 32 * wq, col = cw + j;
  const bool cvalid = col <= last_col, wvalid = cw <= last_col;
  const int row = min(col, last_col) / rep, head = g * rep + (min(col, last_col) - row * rep);
  const int t = pos + row;
  const int tw_first = pos + min(cw, last_col) / rep, tw_last = pos + min(cw + 31, last_col) / rep;

  // Queries in the B operand's layout (dims 16 c + 8 h .. + 7).
  half8_t qh[NC], ql[HALF ? 1 : NC];
  float cs = p.scale * kLog2e;
  if constexpr (HALF) {
    const _Float16* qr = (const _Float16*)p.q + (size_t)row * p.q_stride + head * HD + 8 * h;
#pragma unroll
    for (int c = 0; c < NC; ++c) qh[c] = *(const half8_t*)(qr + 16 * c);
  } else {
    const float* qr = (const float*)p.q + (size_t)row * p.q_stride + head * HD + 8 * h;
    float amax = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float4 a = *(const float4*)(qr + 16 * c), b = *(const float4*)(qr + 16 * c + 4);
      amax = fmaxf(amax, fmaxf(fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w))),
                               fmaxf(fmaxf(fabsf(b.x), fabsf(b.y)), fmaxf(fabsf(b.z), fabsf(b.w)))));
    }
    amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
    int e = 0;
    if (amax > 0.f && amax < INFINITY) {
      frexpf(amax, &e);                           // amax < 2^e
      e = min(max(14 - e, -114), 100);
    }
    const float up = ldexpf(1.f, e);
    cs = ldexpf(cs, -e);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float4 a = *(const float4*)(qr + 16 * c), b = *(const float4*)(qr + 16 * c + 4);
      const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float x = v[k] * up;
        const _Float16 hi = (_Float16)x;
        qh[c][k] = hi;
        ql[c][k] = (_Float16)(x - (float)hi);
      }
    }
  }

  // A thread's rows of a stage: RPP apart, 16 bytes at sd.
  const int srow = tid / SEG, sd = (tid % SEG) * 8;
  const int R = p.slots - p.pin, ub = max(lo, p.pin);
  const int roff = (int)((unsigned)(ub - p.pin) % (unsigned)R);   // ring offset of position ub
  const char* const kc = (const char*)(p.kcache + (size_t)g * p.slots * HD + sd);
  const char* const vc = (const char*)(p.vcache + (size_t)g * p.slots * HD + sd);
  // The call's own rows as distances from the ring's: one address a load, whichever side it reads.
  const long long kd = (const char*)(p.k + g * HD + sd) - kc, vd = (const char*)(p.v + g * HD + sd) - vc;
  u32x4_t kr[PP], vr[PP];
  auto load = [&](int st) {
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      // Past the last key: that key again (masked).
      const int x = min(st * SR + srow + i * RPP, N - 1);
      const int u = x < ns ? x : x - ns + lo;
      const int ro = roff + (u - ub);               // u - ub < window <= R
      const int slot = u < p.pin ? u : p.pin + (ro >= R ? ro - R : ro);
      const int fresh = u < pos ? 0 : -1;
      const long long at = 2ll * (fresh ? u - pos : slot) * (fresh ? p.kv_stride : HD);
      kr[i] = *(const u32x4_t*)(kc + at + (kd & (long long)fresh));
      vr[i] = *(const u32x4_t*)(vc + at + (vd & (long long)fresh));
    }
  };
  auto store = [&](int buf) {
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      *(u32x4_t*)(ks + buf * KB + (srow + i * RPP) * KS + sd) = kr[i];
      *(u32x4_t*)(vs + buf * VB + (srow + i * RPP) * VS + sd) = vr[i];
    }
  };

  f32x16_t o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[dt][e] = 0.f;
  float m = -INFINITY, l = 0.f;                   // the reference in raw scores; the sum of this lane's keys
  // The lane's part of a transposed read's address: key (lane / 4) % 4 (+ 4 h), dims 16 (lane / 16 % 2) + 4 (lane % 4).
  const int tr_row = 4 * h + ((lane >> 2) & 3), tr_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);

  if (st0 < st1) load(st0);
  for (int st = st0, buf = 0; st < st1; ++st, buf = NBUF == 2 ? buf ^ 1 : 0) {
    if (NBUF == 1) __syncthreads();               // the last stage's reads are done
    store(buf);
    if (st + 1 < st1) load(st + 1);
    __syncthreads();
    // This wave's 32 keys, numbered x0 ..: positions x (the sinks) or x - ns + lo.
    const int x0 = st * SR + wk * kAwKeys, u0 = x0 - ns + lo;
    if (!wvalid || x0 >= N) continue;
    if (x0 >= ns && (u0 > tw_last || u0 + kAwKeys - 1 <= tw_first - p.window)) continue;
    const bool whole = x0 + kAwKeys <= ns ? x0 + kAwKeys - 1 <= tw_first
                                          : x0 >= ns && u0 > tw_last - p.window && u0 + kAwKeys - 1 <= tw_first;
    const _Float16* kt = ks + buf * KB + wk * kAwKeys * KS;
    const _Float16* vt = vs + buf * VB + wk * kAwKeys * VS;
    f32x16_t s, sl;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = sl[e] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const half8_t a = *(const half8_t*)(kt + j * KS + 16 * c + 8 * h);
      if constexpr (HALF) {
        if (c & 1) sl = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[c], sl, 0, 0, 0);
        else s = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[c], s, 0, 0, 0);
      } else {
        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[c], s, 0, 0, 0);
        sl = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[c], sl, 0, 0, 0);
      }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] += sl[e];
    // Register e of a lane is key 8 (e / 4) + 4 h + e % 4.
    uint32_t vis = 0xFFFFu;
    if (!whole) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int x = x0 + 8 * (e >> 2) + 4 * h + (e & 3), u = x - ns + lo;
        const bool ok = x < ns ? x <= t : u <= t && u > t - p.window;
        if (!ok) {
          s[e] = -INFINITY;
          vis &= ~(1u << e);
        }
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[e]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const bool raise = (mx - m) * cs > kAwRaise || (m == -INFINITY && mx > -INFINITY);
    if (__any(raise)) {
      const float mn = raise ? mx : m;
      // m = -inf: nothing summed yet (o and l are zero).
      const float corr = raise && m > -INFINITY ? __builtin_amdgcn_exp2f((m - mn) * cs) : 1.f;
      l *= corr;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] *= corr;
      m = mn;
    }
    // A column that has seen no key yet: every s is -inf, every probability 0.
    const float ref = kAwBias - (m == -INFINITY ? 0.f : m * cs);
    half8_t ph[2], pl[HALF ? 1 : 2];
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const f32x2_t pe = {__builtin_amdgcn_exp2f(fmaf(s[e], cs, ref)), __builtin_amdgcn_exp2f(fmaf(s[e + 1], cs, ref))};
      l += pe.x + pe.y;
      const half2v_t hi = __builtin_convertvector(pe, half2v_t);
      ph[e >> 3][e & 7] = hi.x;
      ph[e >> 3][(e & 7) + 1] = hi.y;
      if constexpr (!HALF) {
        const f32x2_t rest2 = pe - __builtin_convertvector(hi, f32x2_t);
        const half2v_t lw = __builtin_convertvector(rest2, half2v_t);
        pl[e >> 3][e & 7] = lw.x;
        pl[e >> 3][(e & 7) + 1] = lw.y;
      }
    }
    if (whole) {
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int kh = 0; kh < 2; ++kh) {
          // V^T rows 32 dt + j, keys 16 kh + 4 h .. + 3 and 16 kh + 8 + 4 h .. + 3.
          const _Float16* a0 = vt + (16 * kh + tr_row) * VS + 32 * dt + tr_col;
          const half4_t x = lds_read_tr(a0), y = lds_read_tr(a0 + 8 * VS);
          const half8_t a = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[kh], o[dt], 0, 0, 0);
          if constexpr (!HALF) o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[kh], o[dt], 0, 0, 0);
        }
    } else {
      // Some key is hidden from some column. An infinity or NaN in its V must reach the columns that
      // see it and no other: it leaves the product (0 * inf is NaN), and joins the columns' sums by
      // a product of the visible keys with its places.
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int kh = 0; kh < 2; ++kh) {
          const _Float16* a0 = vt + (16 * kh + tr_row) * VS + 32 * dt + tr_col;
          const half4_t x = lds_read_tr(a0), y = lds_read_tr(a0 + 8 * VS);
          half8_t a = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
          const uint4 raw = __builtin_bit_cast(uint4, a);
          if (__any(nonfinite_h(raw.x) || nonfinite_h(raw.y) || nonfinite_h(raw.z) || nonfinite_h(raw.w))) {
            half8_t seen;
#pragma unroll
            for (int i = 0; i < 8; ++i) seen[i] = (vis >> (8 * kh + i)) & 1 ? (_Float16)1.f : (_Float16)0.f;
            const float put[3] = {INFINITY, -INFINITY, NAN};
#pragma unroll
            for (int cls = 0; cls < 3; ++cls) {
              half8_t at;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const uint32_t b = __builtin_bit_cast(uint16_t, (_Float16)a[i]);
                const bool hit = cls == 0 ? b == 0x7C00u : cls == 1 ? b == 0xFC00u : (b & 0x7FFFu) > 0x7C00u;
                at[i] = hit ? (_Float16)1.f : (_Float16)0.f;
              }
              f32x16_t c;
#pragma unroll
              for (int e = 0; e < 16; ++e) c[e] = 0.f;
              c = __builtin_amdgcn_mfma_f32_32x32x16_f16(at, seen, c, 0, 0, 0);
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (c[e] > 0.f) o[dt][e] += put[cls];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint32_t b = __builtin_bit_cast(uint16_t, (_Float16)a[i]);
              if ((b & 0x7C00u) == 0x7C00u) a[i] = (_Float16)0.f;
            }
          }
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[kh], o[dt], 0, 0, 0);
          if constexpr (!HALF) o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[kh], o[dt], 0, 0, 0);
        }
    }
  }
  l += __shfl_xor(l, 32, 64);
  float mref = m == -INFINITY ? -INFINITY : m * cs;      // in powers of two, for the joins

  if constexpr (WK > 1) {
    // The waves of other keys hand their sums to the first of their columns.
    float* jb = (float*)smem;
    constexpr int W = NDT * 16 + 2;
    __syncthreads();                                     // the last stage's reads are done
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
    if (wk > 0) return;
    float M = mref;
#pragma unroll
    for (int i = 0; i < WK - 1; ++i) M = fmaxf(M, jb[((size_t)(i * WQ + wq) * W + W - 2) * 64 + lane]);
    const float w0 = mref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mref - M);
    // A wave that saw no key leaves nothing (its sums are zero).
    const float f0 = mref == M ? 1.f : w0;
    l *= f0;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[dt][e] *= f0;
    for (int i = 0; i < WK - 1; ++i) {
      const float* b = jb + (size_t)(i * WQ + wq) * W * 64 + lane;
      const float mi = b[(W - 2) * 64];
      const float fi = mi == -INFINITY ? 0.f : mi == M ? 1.f : __builtin_amdgcn_exp2f(mi - M);
      l += b[(W - 1) * 64] * fi;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] += b[(dt * 16 + e) * 64] * fi;
    }
    mref = M;
  }
  if (!cvalid) return;
  if (p.nsplit > 1) {
    // This split's sums: [split][kv head][column], the reference and the sum behind all outputs.
    const size_t at = ((size_t)sp * p.n_kv + g) * p.cols + col, all = (size_t)p.nsplit * p.n_kv * p.cols;
    float* po = (float*)p.work + at * HD;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int a4 = 0; a4 < 4; ++a4)
        *(float4*)(po + dt * 32 + 8 * a4 + 4 * h) =
            make_float4(o[dt][4 * a4], o[dt][4 * a4 + 1], o[dt][4 * a4 + 2], o[dt][4 * a4 + 3]);
    if (h == 0) *((float2*)((float*)p.work + all * HD) + at) = make_float2(mref, l);
    return;
  }
  const float inv = 1.0f / l;
  const size_t orow = (size_t)row * p.out_stride + head * HD;
  const size_t grow = (size_t)row * p.gate_stride + (size_t)head * p.gate_head_stride;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int a4 = 0; a4 < 4; ++a4) {
      const int d0 = dt * 32 + 8 * a4 + 4 * h;
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = o[dt][4 * a4 + i] * inv;
      if constexpr (HALF) {
        if (p.gate) {
          const half4_t gv = *(const half4_t*)((const _Float16*)p.gate + grow + d0);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] *= sigmoidf_((float)gv[i]);
        }
        *(half4_t*)((_Float16*)p.out + orow + d0) = half4_t{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
      } else {
        if (p.gate) {
          const float4 gv = *(const float4*)((const float*)p.gate + grow + d0);
          v[0] *= sigmoidf_(gv.x);
          v[1] *= sigmoidf_(gv.y);
          v[2] *= sigmoidf_(gv.z);
          v[3] *= sigmoidf_(gv.w);
        }
        *(float4*)((float*)p.out + orow + d0) = make_float4(v[0], v[1], v[2], v[3]);
      }
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
    const long long id = (long long)blockIdx.x * 4 + w;
    if (id >= (long long)p.n * p.n_head) return;
    const int row = (int)(id / p.n_head), head = (int)(id - (long long)row * p.n_head), g = head / p.rep;
    const int col = row * p.rep + head - g * p.rep;
    const size_t all = (size_t)p.nsplit * p.n_kv * p.cols, step = (size_t)p.n_kv * p.cols;
    const size_t at = (size_t)g * p.cols + col;
    const float2* ml = (const float2*)((const float*)p.work + all * HD) + at;
    const float* po = (const float*)p.work + at * HD + E * lane;
    float M = -INFINITY;
    for (int s = lane; s < p.nsplit; s += 64) M = fmaxf(M, ml[s * step].x);
    M = wave_max(M);
    float l = 0.f, o[E];
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = 0.f;
    for (int s = 0; s < p.nsplit; ++s) {
      const float2 a = ml[s * step];
      const float f = a.x == -INFINITY ? 0.f : a.x == M ? 1.f : __builtin_amdgcn_exp2f(a.x - M);
      l += a.y * f;
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] += po[s * step * HD + i] * f;
    }
    const float inv = 1.0f / l;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int d = E * lane + i;
      float v = o[i] * inv;
      const size_t gi = (size_t)row * p.gate_stride + (size_t)head * p.gate_head_stride + d;
      const size_t oi = (size_t)row * p.out_stride + (size_t)head * HD + d;
      if constexpr (HALF) {
        if (p.gate) v *= sigmoidf_((float)((const _Float16*)p.gate)[gi]);
        ((_Float16*)p.out)[oi] = (_Float16)v;
      } else {
        if (p.gate) v *= sigmoidf_(((const float*)p.gate)[gi]);
        ((float*)p.out)[oi] = v;
      }
    }
    return;
  }
  // Rows pos .. pos + n - 1, 16 bytes of K and V a thread. A ring row that a later row of the call
  // replaces is left out.
  constexpr int SEG = HD / 8;
  const int R = p.slots - p.pin;
  const long long id = (long long)(blockIdx.x - join_blocks) * 256 + threadIdx.x;
  const long long pieces = (long long)p.n * p.n_kv * SEG;
  if (id >= pieces) return;
  const int sd = (int)(id % SEG) * 8, g = (int)(id / SEG % p.n_kv), r = (int)(id / SEG / p.n_kv), u = pos + r;
  if (u >= p.pin && p.n - r > R) return;
  const int slot = u < p.pin ? u : p.pin + (int)((unsigned)(u - p.pin) % (unsigned)R);
  const size_t to = ((size_t)g * p.slots + slot) * HD + sd, from = (size_t)r * p.kv_stride + (size_t)g * HD + sd;
  *(uint4*)(p.kcache + to) = *(const uint4*)(p.k + from);
  *(uint4*)(p.vcache + to) = *(const uint4*)(p.v + from);
}

// Launch ------------------------------------------------------------------------------------------

constexpr int kAwCus = 256;
constexpr int kAwMaxSplits = 64;

// Few columns: one wave of columns, four of keys; else four of columns, two of keys.
static bool aw_few(const AttnWindowParams& p) { return (long long)p.n * (p.n_head / p.n_kv) <= 32; }

// Splits of the keys: the count whose rounds of blocks (a block a CU) times stages a block, with a
// stage's worth for a split's join, is least.
static int aw_splits(const AttnWindowParams& p, long long keys, int most) {
  const bool few = aw_few(p);
  const int wq = few ? 1 : 4, sr = (few ? 4 : 2) * kAwKeys;
  const long long blocks = (long long)cdiv(p.n * (p.n_head / p.n_kv), 32 * wq) * p.n_kv;
  const long long stages = (keys + sr - 1) / sr;
  int best = 1;
  long long cost = LLONG_MAX;
  for (int s = 1; s <= most && s <= stages; ++s) {
    const long long c = (blocks * s + kAwCus - 1) / kAwCus * ((stages + s - 1) / s + (s > 1 ? 1 : 0));
    if (c < cost) cost = c, best = s;
  }
  return best;
}

static long long aw_keys(const AttnWindowParams& p) {
  const int wq = aw_few(p) ? 1 : 4, rep = p.n_head / p.n_kv;
  const long long span = std::min<long long>(p.n, (32 * wq + rep - 1) / rep + 1);
  return (long long)p.sinks + p.window + span - 1;
}

const char* attn_window_refuses(const AttnWindowParams& p) {
  if (p.hd != 64 && p.hd != 128 && p.hd != 256) return "head_dim is not 64, 128 or 256";
  if (p.n_kv < 1 || p.n_head < 1 || p.n_head % p.n_kv) return "n_head is not a multiple of n_kv_head";
  if (p.n_head > 1024) return "more than 1024 heads";
  if (p.slots > 1 << 30) return "more than 2^30 slots";
  if (p.pin < 0 || p.slots <= p.pin) return "pin outside [0, slots)";
  if (p.sinks < 0 || p.sinks > p.pin) return "sinks outside [0, pin]";
  if (p.window < 1 || p.window > p.slots - p.pin) return "window outside [1, slots - pin]";
  if (p.n < 0 || (long long)p.n * p.n_head > (1 << 28)) return "too many positions";
  if (!(p.scale > 0.f && p.scale < INFINITY)) return "scale is not positive and finite";
  const int q4 = p.half_io ? 8 : 4, o4 = 4;
  if (p.q_stride < p.n_head * p.hd || p.q_stride % q4) return "q_stride";
  if (p.kv_stride < p.n_kv * p.hd || p.kv_stride % 8) return "kv_stride";
  if (p.out_stride < p.n_head * p.hd || p.out_stride % o4) return "out_stride";
  if (p.gate && (p.gate_head_stride < p.hd || p.gate_head_stride % o4 || p.gate_stride % o4 ||
                 p.gate_stride < (long long)(p.n_head - 1) * p.gate_head_stride + p.hd))
    return "gate strides";
  return nullptr;
}

size_t attn_window_work_bytes(const AttnWindowParams& p) {
  if (p.n == 0) return 0;
  const int s = aw_splits(p, aw_keys(p), kAwMaxSplits);
  return s > 1 ? (size_t)s * p.n * p.n_head * (p.hd + 2) * 4 : 0;
}

template <int HD, bool HALF>
static void aw_dispatch(const AttnWindowParams& p, hipStream_t s) {
  if (aw_few(p)) {
    const dim3 grid(p.n_kv * p.nsplit);
    hipLaunchKernelGGL((attn_window_kernel<HD, HALF, 1, 4, HD == 256 ? 1 : 2>), grid, dim3(256), 0, s, p);
  } else {
    const dim3 grid(cdiv(p.cols, 128) * p.n_kv * p.nsplit);
    hipLaunchKernelGGL((attn_window_kernel<HD, HALF, 4, 2, 2>), grid, dim3(512), 0, s, p);
  }
}

template <int HD, bool HALF>
static int aw_launch(const AttnWindowParams& p, hipStream_t s) {
  aw_dispatch<HD, HALF>(p, s);
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
  // The workspace holds the splits of a full window; a ring that is still filling takes no more.
  const int most = aw_splits(p, aw_keys(p), kAwMaxSplits);
  p.nsplit = p.pos_dev ? most : aw_splits(p, std::min<long long>(aw_keys(p), (long long)p.pos + p.n), most);
  if (p.half_io) {
    if (p.hd == 64) return aw_launch<64, true>(p, s);
    if (p.hd == 128) return aw_launch<128, true>(p, s);
    return aw_launch<256, true>(p, s);
  }
  if (p.hd == 64) return aw_launch<64, false>(p, s);
  if (p.hd == 128) return aw_launch<128, false>(p, s);
  return aw_launch<256, false>(p, s);
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
  TRX_CHECK(workspace || attn_window_work_bytes(p) == 0, TRX_E_INVALID, "trx_attn_window: null workspace");
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
