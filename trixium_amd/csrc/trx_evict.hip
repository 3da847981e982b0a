// Eviction from a cache with masses (trx_kv_evict): of the `count` rows of a kv head the `keep` foremost stay, first
// those at positions that are kept, slot rising (their masses do not count), then the others, mass falling and slot
// rising; and the rows that stay past slot keep move into the slots of those that go below it. Nothing else moves, so a
// token's eviction touches one row, and rows are read at slots from keep on and written at slots below it: no order of
// blocks matters.
//
// Selection: a row's key is 32 bits that order as the rows do and 32 of its slot, so that no two are equal; the
// keep-th largest is found by its bits, 11, 11 and 10 at a time, most significant first, each from a histogram of the
// rows that share the bits before it (integers: exact), until 64 rows share them (masses: after 22 bits as a rule).
// A block per kv head, its keys in LDS as far as they fit and read again for every step past that. It leaves a bit a
// row, whether the row is a hole or moves, and the numbers of both before every 64 rows, from which the copying
// threads find their rows. One row alone that goes is looked for directly.

#include "trx_internal.h"

#include <algorithm>

namespace trx {

constexpr int kEvThreads = 1024, kEvWaves = kEvThreads / 64;
constexpr int kEvOwnMoves = 128;            // rows that the selecting block moves itself

#define AW_INLINE __attribute__((always_inline))

struct EvictParams {
  __half *kcache, *vcache;     // [n_kv][slots][hd]
  float* mass;                 // [n_kv][slots]
  int* positions;              // [n_kv][slots]
  const int* state;            // {count, pos} on the device, or null
  int count, pos, keep, sinks, recent;
  int n_kv, hd, slots;
  void* work;                  // an EvictMoves a kv head
};

// What moves in a kv head. Its slots are cut into kEvWaves runs of `rounds` times 64; of 64 slots each, a bit for every
// slot below keep whose row goes (a hole) and every other whose row stays (it moves), and how many of both stand
// before them in the run.
struct EvictMoves {
  int n, rounds;
  int2 run[kEvWaves];          // holes and moves before each run
};
// (Fours of rounds, so that four keys a lane are looked at a time.)
__host__ __device__ inline int ev_rounds(int rows) { return (int)(((long long)rows + 4 * kEvThreads - 1) / (4 * kEvThreads)) * 4; }
__host__ __device__ inline size_t ev_moves_bytes(int slots) { return sizeof(EvictMoves) + (size_t)ev_rounds(slots) * kEvWaves * 16; }
struct EvictLists {
  EvictMoves* head;
  unsigned long long* bits;    // of every 64 slots
  int2* before;
  __device__ __forceinline__ EvictLists(const EvictParams& p, int g) {
    char* at = (char*)p.work + g * ev_moves_bytes(p.slots);
    head = (EvictMoves*)at;
    bits = (unsigned long long*)(at + sizeof(EvictMoves));
    before = (int2*)(bits + (size_t)ev_rounds(p.slots) * kEvWaves);
  }
  // The slot of hole or (MOVE) of moving row j.
  template <bool MOVE>
  __device__ __forceinline__ int find(const EvictParams& p, int j) const {
    auto of = [](const int2& c) AW_INLINE { return MOVE ? c.y : c.x; };
    int run = 0;
#pragma unroll
    for (int i = 1; i < kEvWaves; ++i) run += of(head->run[i]) <= j;
    j -= of(head->run[run]);
    const int2* b = before + (size_t)run * head->rounds;
    int lo = 0, hi = head->rounds;                // the last of them with at most j before it
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (of(b[mid]) <= j) lo = mid;
      else hi = mid;
    }
    j -= of(b[lo]);
    const int u = (run * head->rounds + lo) * 64;
    unsigned long long m = bits[(size_t)run * head->rounds + lo];
    // (64 slots on both sides of keep hold both kinds.)
    const int low = min(max(p.keep - u, 0), 64);
    const unsigned long long holes = low == 64 ? ~0ull : (1ull << low) - 1;
    m &= MOVE ? ~holes : holes;
    int bit = 0;
#pragma unroll
    for (int w = 32; w; w /= 2) {
      const int n = __popcll(m & ((1ull << w) - 1));
      if (j >= n) {
        j -= n;
        bit += w;
        m >>= w;
      }
    }
    return u + bit;
  }
};

__device__ __forceinline__ bool ev_state(const EvictParams& p, int& count, int& pos) {
  count = p.state ? p.state[0] : p.count;
  pos = p.state ? p.state[1] : p.pos;
  return count > p.keep && count <= p.slots && pos >= 0;
}

// Rows that are kept first, then by mass, then NaN; 0 is below every row's key.
__device__ __forceinline__ uint32_t ev_key(const EvictParams& p, int pos, float mass, int position) {
  if (position < p.sinks || position >= pos - p.recent) return ~0u;
  return mass != mass ? 1u : ordered_bits(mass + 0.f);     // (-0 is 0)
}

// Row `from` of a kv head to slot `to`: 16 bytes of K and V a thread (d: the dim).
__device__ __forceinline__ void ev_move(const EvictParams& p, int g, int from, int to, int d) {
  const size_t a = (size_t)g * p.slots + from, b = (size_t)g * p.slots + to;
  *(uint4*)(p.kcache + b * p.hd + d) = *(const uint4*)(p.kcache + a * p.hd + d);
  *(uint4*)(p.vcache + b * p.hd + d) = *(const uint4*)(p.vcache + a * p.hd + d);
  if (d == 0) {
    p.mass[b] = p.mass[a];
    p.positions[b] = p.positions[a];
  }
}

// One row goes: the smallest key, of equal ones the last slot, its slot to the last row. A block per kv head; of 4096 rows
// 4.6 us, the latency of the loads, of two steps over the block and of the row that moves.
__global__ __launch_bounds__(kEvThreads) void evict_one_kernel(EvictParams p) {
  __shared__ unsigned long long least[kEvWaves];
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const float* mass = p.mass + (size_t)g * p.slots;
  const int* position = p.positions + (size_t)g * p.slots;
  unsigned long long mine = ~0ull;
#pragma unroll 8
  for (int u = tid; u < p.count; u += kEvThreads) {
    const unsigned long long k = (unsigned long long)ev_key(p, p.pos, mass[u], position[u]) << 32 | ~(uint32_t)u;
    mine = min(mine, k);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) mine = min(mine, (unsigned long long)__shfl_xor((long long)mine, o, 64));
  if (lane == 0) least[w] = mine;
  __syncthreads();
  mine = least[lane % kEvWaves];
#pragma unroll
  for (int o = kEvWaves / 2; o; o >>= 1) mine = min(mine, (unsigned long long)__shfl_xor((long long)mine, o, 64));
  const int to = (int)~(uint32_t)mine;
  if (to < p.keep && tid < p.hd / 8) ev_move(p, g, p.keep, to, 8 * tid);
}

// R: keys a thread has in LDS (0: none, they are read again). OWN: the block moves its rows itself.
// Bound by one CU: its loads (32768 rows of 8 kv heads, 2 MB: 9 us with the first histogram beside them), then its vector
// instructions, each some 0.2 us over the rows: 7 for what follows of the cut, 5 for the bits; 23 in all while the masses
// are in the Infinity Cache, 27 from HBM. Keys in
// registers took 51 (unrolled steps, each fetched once), lists of rows in place of the bits 20 more.
template <int R, bool OWN>
__global__ __launch_bounds__(kEvThreads) void evict_select_kernel(EvictParams p) {
  __shared__ uint32_t held[R ? R * kEvThreads : 1];
  __shared__ int bins[2048];
  __shared__ int2 runs[kEvWaves];
  __shared__ int waves[kEvWaves];
  __shared__ uint32_t found[3];
  __shared__ unsigned long long shared[64];
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const EvictLists lists(p, g);
  int count, pos;
  if (!ev_state(p, count, pos)) {
    if (!OWN && tid == 0) lists.head->n = 0;
    return;
  }
  const float* mass = p.mass + (size_t)g * p.slots;
  const int* position = p.positions + (size_t)g * p.slots;
  // Each wave a run of slots, 64 at a time; rows past the last have a key of 0.
  const int rounds = ev_rounds(count), first_u = w * rounds * 64 + lane;
  // f(slot, key), the lanes of a wave together, from memory, sixteen rounds' loads in flight; rounds [from, to) of them.
  auto read = [&](int from, int to, auto f) AW_INLINE {
    for (int i = from; i < to; i += 16) {
      float m[16];
      int q[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int u = min(first_u + 64 * (i + k), count - 1);
        m[k] = mass[u];
        q[k] = position[u];
      }
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int u = first_u + 64 * (i + k);
        if (i + k < to) f(u, u < count ? ev_key(p, pos, m[k], q[k]) : 0u);
      }
    }
  };
  auto each = [&](int from, int to, auto f) AW_INLINE {
    if constexpr (R > 0) {
      for (int i = from; i < to; i += 4) {
        const uint32_t* k = held + first_u + 64 * i;
        const uint32_t a = k[0], b = k[64], c = k[128], d = k[192];
        f(first_u + 64 * i, a);
        f(first_u + 64 * i + 64, b);
        f(first_u + 64 * i + 128, c);
        f(first_u + 64 * i + 192, d);
      }
    } else {
      read(from, to, f);
    }
  };
  // One row more in its bin, of the lanes where `is`. (Many rows alike, as those whose positions are kept, would wait
  // for each other.)
  auto tally = [&](bool is, int bin) AW_INLINE {
    const unsigned long long all = __ballot(is);
    if (!all) return;
    const int first = __builtin_amdgcn_readlane(bin, (int)__builtin_ctzll(all));
    if (__ballot(is && bin == first) == all) {
      if (lane == 0) atomicAdd(&bins[first], __popcll(all));
    } else if (is) {
      atomicAdd(&bins[bin], 1);
    }
  };
  // The keep-th largest key {top, low} (low: of ~slot), bit by bit: of the rows that share the bits known so far, `same`,
  // the `need` largest stay.
  uint32_t top = 0, low = 0, known_top = 0, known_low = 0;
  int need = p.keep, same = count;
#pragma unroll 1
  for (int step = 0; step < 6; ++step) {
    const int third = step % 3, shift = third == 0 ? 21 : third == 1 ? 10 : 0, last = third == 2 ? 1023 : 2047;
    bins[tid] = bins[tid + kEvThreads] = 0;
    __syncthreads();
    if (step == 0) {
      read(0, rounds, [&](int u, uint32_t k) AW_INLINE {
        if constexpr (R > 0) held[u] = k;
        tally(k != 0, k >> 21);
      });
    } else if (step < 3) {
      each(0, rounds, [&](int u, uint32_t k) AW_INLINE { tally(k != 0 && (k & known_top) == top, k >> shift & last); });
    } else {
      each(0, rounds, [&](int u, uint32_t k) AW_INLINE { tally(k == top && (~(uint32_t)u & known_low) == low, ~(uint32_t)u >> shift & last); });
    }
    __syncthreads();
    // Two bins a thread, from the largest down.
    const int hi = 2047 - 2 * tid, a = bins[hi], b = bins[hi - 1];
    int upto = a + b;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o, 64);
      if (lane >= o) upto += v;
    }
    if (lane == 63) waves[w] = upto;
    __syncthreads();
    int before = upto - a - b;
    for (int i = 0; i < w; ++i) before += waves[i];
    const bool one = before < need && need <= before + a, two = before + a < need && need <= before + a + b;
    if (one || two) {
      found[0] = (uint32_t)(one ? hi : hi - 1) << shift;
      found[1] = need - before - (one ? 0 : a);
      found[2] = one ? a : b;
    }
    __syncthreads();
    (step < 3 ? top : low) |= found[0];
    (step < 3 ? known_top : known_low) |= (uint32_t)last << shift;
    need = (int)found[1];
    same = (int)found[2];
    if (same <= 64 || same == need) break;
  }
  if (same != need) {
    // The rows that share them into LDS, the need-th largest of them by one wave.
    if (tid == 0) bins[0] = 0;
    __syncthreads();
    each(0, rounds, [&](int u, uint32_t k) AW_INLINE {
      if (k != 0 && (k & known_top) == top && (~(uint32_t)u & known_low) == low)
        shared[atomicAdd(&bins[0], 1)] = (unsigned long long)k << 32 | ~(uint32_t)u;
    });
    __syncthreads();
    if (w == 0) {
      const unsigned long long mine = lane < same ? shared[lane] : 0;
      int larger = 0;
      for (int i = 0; i < same; ++i) larger += shared[i] > mine;
      if (lane < same && larger == need - 1) {
        found[0] = (uint32_t)(mine >> 32);
        found[1] = (uint32_t)mine;
      }
    }
    __syncthreads();
    top = found[0];
    low = found[1];
  }
  // A hole: below keep and does not stay. A row that moves: past it and stays. (Past the last row neither.) Lane i
  // keeps the bits of the i-th of 64 rounds.
  int holes = 0, moved = 0;
  for (int r = 0; r < rounds; r += 64) {
    unsigned long long mine = 0;
    int i = 0;
    each(r, min(r + 64, rounds), [&](int u, uint32_t k) AW_INLINE {
      const bool stays = k > top || (k == top && ~(uint32_t)u >= low);
      const unsigned long long bits = __ballot(stays != (u < p.keep));
      mine = lane == i ? bits : mine;
      ++i;
    });
    const int under = min(max(p.keep - (first_u - lane + 64 * (r + lane)), 0), 64);
    const int h = __popcll(under == 64 ? mine : mine & ((1ull << under) - 1)), m = __popcll(mine) - h;
    int hs = h, ms = m;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int a = __shfl_up(hs, o, 64), b = __shfl_up(ms, o, 64);
      if (lane >= o) hs += a, ms += b;
    }
    if (r + lane < rounds) {
      const size_t at = (size_t)w * rounds + r + lane;
      lists.bits[at] = mine;
      lists.before[at] = make_int2(holes + hs - h, moved + ms - m);
    }
    holes += __shfl(hs, 63, 64);
    moved += __shfl(ms, 63, 64);
  }
  if (lane == 0) runs[w] = make_int2(holes, moved);
  __syncthreads();
  int n = 0;
  for (int i = 0; i < kEvWaves; ++i) n += runs[i].x;
  if (tid < kEvWaves) {
    int2 b = make_int2(0, 0);
    for (int i = 0; i < tid; ++i) b.x += runs[i].x, b.y += runs[i].y;
    lists.head->run[tid] = b;
    lists.head->n = n;
    lists.head->rounds = rounds;
  }
  if constexpr (OWN) {
    __syncthreads();
    const int seg = p.hd / 8;
    for (int i = tid; i < n * seg; i += kEvThreads)
      ev_move(p, g, lists.find<true>(p, i / seg), lists.find<false>(p, i / seg), i % seg * 8);
  }
}

// 16 bytes of K and V a thread, which looks for its rows itself: a chain of some eight loads, 5 us for 3600 rows of each of 8
// kv heads (15 MB read), 17 where they come from HBM.
__global__ __launch_bounds__(256) void evict_move_kernel(EvictParams p) {
  const int g = blockIdx.x % (unsigned)p.n_kv, seg = p.hd / 8;
  const EvictLists lists(p, g);
  const int n = lists.head->n;
  const unsigned step = gridDim.x / (unsigned)p.n_kv * 256;
  for (size_t i = blockIdx.x / (unsigned)p.n_kv * 256 + threadIdx.x; i < (size_t)n * seg; i += step) {
    const int j = (int)(i / seg);
    ev_move(p, g, lists.find<true>(p, j), lists.find<false>(p, j), (int)(i % seg) * 8);
  }
}

template <int R>
static void ev_select(const EvictParams& p, bool own, hipStream_t s) {
  if (own) hipLaunchKernelGGL((evict_select_kernel<R, true>), dim3(p.n_kv), dim3(kEvThreads), 0, s, p);
  else hipLaunchKernelGGL((evict_select_kernel<R, false>), dim3(p.n_kv), dim3(kEvThreads), 0, s, p);
}

static int launch_evict(const EvictParams& p, hipStream_t s) {
  const int count = p.state ? p.slots : p.count, most = std::min(p.keep, count - p.keep);  // rows, and moves, at most
  if (!p.state && count - p.keep == 1) {
    hipLaunchKernelGGL(evict_one_kernel, dim3(p.n_kv), dim3(kEvThreads), 0, s, p);
    TRX_LAUNCHED();
    return TRX_OK;
  }
  const bool own = most <= kEvOwnMoves;
  if (count <= 4 * kEvThreads) ev_select<4>(p, own, s);
  else if (count <= 32 * kEvThreads) ev_select<32>(p, own, s);
  else ev_select<0>(p, own, s);
  TRX_LAUNCHED();
  if (own) return TRX_OK;
  const long long blocks = ((long long)most * (p.hd / 8) + 255) / 256;
  hipLaunchKernelGGL(evict_move_kernel, dim3((int)std::min(blocks, 256ll) * p.n_kv), dim3(256), 0, s, p);
  TRX_LAUNCHED();
  return TRX_OK;
}

static const char* evict_refuses(const trx_attn_mass_shape& a) {
  if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return "head_dim is not 64, 128 or 256";
  if (a.n_kv_head < 1 || a.n_head < 1 || a.n_head % a.n_kv_head) return "n_head is not a multiple of n_kv_head";
  if (a.n_head > 1024) return "more than 1024 heads";
  if (a.slots < 1 || a.slots > 1 << 30) return "slots outside [1, 2^30]";
  if ((long long)a.slots * a.n_kv_head > 1 << 30) return "more than 2^30 slots of all kv heads";
  return nullptr;
}

}  // namespace trx

using namespace trx;

#define TRX_API extern "C" __attribute__((visibility("default")))

TRX_API int trx_kv_evict_geometry(const trx_attn_mass_shape* shape, size_t* workspace_bytes) {
  TRX_CHECK(shape && workspace_bytes, TRX_E_INVALID, "trx_kv_evict_geometry: null argument");
  const char* why = evict_refuses(*shape);
  TRX_CHECK(!why, TRX_E_INVALID, "trx_kv_evict_geometry: %s", why);
  *workspace_bytes = shape->n_kv_head * ev_moves_bytes(shape->slots);
  return TRX_OK;
}

TRX_API int trx_kv_evict(const trx_attn_mass_shape* shape, int count, int pos, const int32_t* state, int keep, int sinks,
                         int recent, uint16_t* kcache, uint16_t* vcache, float* mass, int32_t* positions, void* workspace,
                         trx_stream_t s) {
  TRX_CHECK(shape, TRX_E_INVALID, "trx_kv_evict: null shape");
  const char* why = evict_refuses(*shape);
  TRX_CHECK(!why, TRX_E_INVALID, "trx_kv_evict: %s", why);
  TRX_CHECK(keep >= 1 && keep <= shape->slots, TRX_E_INVALID, "trx_kv_evict: keep %d outside [1, %d]", keep, shape->slots);
  TRX_CHECK(sinks >= 0 && recent >= 0, TRX_E_INVALID, "trx_kv_evict: sinks %d, recent %d", sinks, recent);
  TRX_CHECK(state || (count >= 0 && count <= shape->slots), TRX_E_INVALID, "trx_kv_evict: %d rows, %d slots", count, shape->slots);
  TRX_CHECK(state || pos >= 0, TRX_E_INVALID, "trx_kv_evict: position %d", pos);
  if (!state && count <= keep) return TRX_OK;
  TRX_CHECK(kcache && vcache && mass && positions && workspace, TRX_E_INVALID, "trx_kv_evict: null argument");
  TRX_CHECK((((uintptr_t)kcache | (uintptr_t)vcache | (uintptr_t)workspace) & 15) == 0, TRX_E_INVALID,
            "trx_kv_evict: a pointer is not 16-byte aligned");
  TRX_CHECK((((uintptr_t)mass | (uintptr_t)positions | (uintptr_t)state) & 3) == 0, TRX_E_INVALID,
            "trx_kv_evict: mass, positions or state are not 4-byte aligned");
  EvictParams p = {};
  p.kcache = (__half*)kcache;
  p.vcache = (__half*)vcache;
  p.mass = mass;
  p.positions = positions;
  p.state = state;
  p.count = count;
  p.pos = pos;
  p.keep = keep;
  p.sinks = sinks;
  p.recent = recent;
  p.n_kv = shape->n_kv_head;
  p.hd = shape->head_dim;
  p.slots = shape->slots;
  p.work = workspace;
  return launch_evict(p, (hipStream_t)s);
}
