// Eviction from a cache with masses (trx_kv_evict): of the `count` rows of a kv head the `keep` foremost stay, in the
// order (at a position that is kept, mass falling, slot rising), and the rows that stay past slot keep move into
// the slots of those that go below it. Nothing else moves, so a token's eviction touches one row, and rows are read
// at slots from keep on and written at slots below it: no order of blocks matters.
//
// Selection: a row's key is 32 bits that order as the rows do; the keep-th largest is found by its bytes, most
// significant first, each from a histogram of the rows that share the bytes before it (integers: exact). A block
// per kv head; then one that copies rows.

#include "trx_internal.h"

#include <algorithm>

namespace trx {

constexpr int kEvThreads = 1024, kEvWaves = kEvThreads / 64;

struct EvictParams {
  __half *kcache, *vcache;     // [n_kv][slots][hd]
  float* mass;                 // [n_kv][slots]
  int* positions;              // [n_kv][slots]
  const int* state;            // {count, pos} on the device, or null
  int count, pos, keep, sinks, recent;
  int n_kv, hd, slots;
  int* moves;                  // [n_kv] the number of moves, then [n_kv][2][slots / 2] to and from
};

__device__ __forceinline__ bool ev_state(const EvictParams& p, int& count, int& pos) {
  count = p.state ? p.state[0] : p.count;
  pos = p.state ? p.state[1] : p.pos;
  return count > p.keep && count <= p.slots && pos >= 0;
}
__device__ __forceinline__ int* ev_list(const EvictParams& p, int g) { return p.moves + p.n_kv + (size_t)g * (p.slots / 2) * 2; }

// Rows that are kept first, then by mass; 0: NaN.
__device__ __forceinline__ uint32_t ev_key(const EvictParams& p, int pos, float mass, int position) {
  if (position < p.sinks || position >= pos - p.recent) return ~0u;
  return mass != mass ? 0u : ordered_bits(mass + 0.f);     // (-0 is 0)
}

__global__ __launch_bounds__(kEvThreads) void evict_select_kernel(EvictParams p) {
  __shared__ int bins[256];
  __shared__ int part[3][kEvWaves];
  __shared__ uint32_t found[2];
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int count, pos;
  if (!ev_state(p, count, pos)) {
    if (tid == 0) p.moves[g] = 0;
    return;
  }
  const float* mass = p.mass + (size_t)g * p.slots;
  const int* position = p.positions + (size_t)g * p.slots;
  auto key = [&](int u) { return ev_key(p, pos, mass[u], position[u]); };
  // The keep-th largest key, and how many rows that have it stay.
  uint32_t top = 0;
  int need = p.keep;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) bins[tid] = 0;
    __syncthreads();
    const uint32_t known = shift == 24 ? 0u : ~0u << (shift + 8);
    for (int u = tid; u < count; u += kEvThreads) {
      const uint32_t k = key(u);
      if ((k & known) == top) atomicAdd(&bins[k >> shift & 255], 1);
    }
    __syncthreads();
    if (w == 0) {
      // Four bins a lane, from the largest down.
      int n[4], sum = 0;
      for (int i = 0; i < 4; ++i) sum += n[i] = bins[255 - 4 * lane - i];
      int upto = sum;
      for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(upto, o, 64);
        if (lane >= o) upto += v;
      }
      int before = upto - sum;
      for (int i = 0; i < 4; ++i) {
        if (before < need && need <= before + n[i]) {
          found[0] = top | (uint32_t)(255 - 4 * lane - i) << shift;
          found[1] = need - before;
        }
        before += n[i];
      }
    }
    __syncthreads();
    top = found[0];
    need = (int)found[1];
  }
  // Each wave a run of slots: its rows that have the key, then its holes below keep and its rows past it.
  const int run = (count + kEvThreads - 1) / kEvThreads * 64, u0 = w * run, u1 = min(count, u0 + run);
  int equal = 0;
  for (int u = u0 + lane; u < u0 + run; u += 64) equal += __popcll(__ballot(u < u1 && key(u) == top));
  if (lane == 0) part[0][w] = equal;
  __syncthreads();
  int first = 0;
  for (int i = 0; i < w; ++i) first += part[0][i];
  const unsigned long long below = (1ull << lane) - 1;
  // What to do with row u: 0 nothing, 1 a hole, 2 moves.
  auto role = [&](int u, int& before) {
    const uint32_t k = u < u1 ? key(u) : 0u;
    const unsigned long long e = __ballot(u < u1 && k == top);
    const bool stays = k > top || (k == top && before + __popcll(e & below) < need);
    before += __popcll(e);
    return u >= u1 ? 0 : u < p.keep ? (stays ? 0 : 1) : (stays ? 2 : 0);
  };
  int holes = 0, moved = 0, before = first;
  for (int u = u0 + lane; u < u0 + run; u += 64) {
    const int r = role(u, before);
    holes += __popcll(__ballot(r == 1));
    moved += __popcll(__ballot(r == 2));
  }
  if (lane == 0) part[1][w] = holes, part[2][w] = moved;
  __syncthreads();
  int hole = 0, move = 0;
  for (int i = 0; i < w; ++i) hole += part[1][i], move += part[2][i];
  int *to = ev_list(p, g), *from = to + p.slots / 2;
  before = first;
  for (int u = u0 + lane; u < u0 + run; u += 64) {
    const int r = role(u, before);
    const unsigned long long a = __ballot(r == 1), b = __ballot(r == 2);
    if (r == 1) to[hole + __popcll(a & below)] = u;
    if (r == 2) from[move + __popcll(b & below)] = u;
    hole += __popcll(a);
    move += __popcll(b);
  }
  if (w == kEvWaves - 1 && lane == 0) p.moves[g] = hole;
}

// 16 bytes of K and V a thread.
__global__ __launch_bounds__(256) void evict_move_kernel(EvictParams p) {
  const int g = blockIdx.x % (unsigned)p.n_kv, seg = p.hd / 8, n = p.moves[g];
  const int *to = ev_list(p, g), *from = to + p.slots / 2;
  const unsigned step = gridDim.x / (unsigned)p.n_kv * 256;
  for (size_t i = blockIdx.x / (unsigned)p.n_kv * 256 + threadIdx.x; i < (size_t)n * seg; i += step) {
    const int m = (int)(i / seg), d = (int)(i % seg) * 8;
    const size_t a = (size_t)g * p.slots + from[m], b = (size_t)g * p.slots + to[m];
    *(uint4*)(p.kcache + b * p.hd + d) = *(const uint4*)(p.kcache + a * p.hd + d);
    *(uint4*)(p.vcache + b * p.hd + d) = *(const uint4*)(p.vcache + a * p.hd + d);
    if (d == 0) {
      p.mass[b] = p.mass[a];
      p.positions[b] = p.positions[a];
    }
  }
}

static int launch_evict(const EvictParams& p, hipStream_t s) {
  hipLaunchKernelGGL(evict_select_kernel, dim3(p.n_kv), dim3(kEvThreads), 0, s, p);
  TRX_LAUNCHED();
  const long long most = (long long)std::min(p.keep, (p.state ? p.slots : p.count) - p.keep) * (p.hd / 8);
  hipLaunchKernelGGL(evict_move_kernel, dim3((int)std::min(std::max((most + 255) / 256, 1ll), 256ll) * p.n_kv), dim3(256), 0, s, p);
  TRX_LAUNCHED();
  return TRX_OK;
}

static const char* evict_refuses(const trx_attn_mass_shape& a) {
  if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return "head_dim is not 64, 128 or 256";
  if (a.n_kv_head < 1 || a.n_head < 1 || a.n_head % a.n_kv_head) return "n_head is not a multiple of n_kv_head";
  if (a.n_head > 1024) return "more than 1024 heads";
  if (a.slots < 1 || a.slots > 1 << 30) return "slots outside [1, 2^30]";
  return nullptr;
}

}  // namespace trx

using namespace trx;

#define TRX_API extern "C" __attribute__((visibility("default")))

TRX_API int trx_kv_evict_geometry(const trx_attn_mass_shape* shape, size_t* workspace_bytes) {
  TRX_CHECK(shape && workspace_bytes, TRX_E_INVALID, "trx_kv_evict_geometry: null argument");
  const char* why = evict_refuses(*shape);
  TRX_CHECK(!why, TRX_E_INVALID, "trx_kv_evict_geometry: %s", why);
  *workspace_bytes = 4 * ((size_t)shape->n_kv_head + (size_t)shape->n_kv_head * (shape->slots / 2) * 2);
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
  p.moves = (int*)workspace;
  return launch_evict(p, (hipStream_t)s);
}
