// Ring caches in 4 bits, written for gfx950 (MI355X): tokens into them (uttt_kv_commit4), their values out of them
// (uttt_kv_values4), whole caches over others' (uttt_kv_fork4).  A block of 32 slots (fp4.h, uttt_decode.h) is the unit of all
// three: it lies together in memory, and the codes of its values are words over 8 slots.
#include <algorithm>

#include "../../include/uttt_decode.h"
#include "fp4.h"
#include "uttt_host.h"

namespace uttt {
namespace {

constexpr int kSlots = 32;

struct Commit4Args {
  int heads, n_nodes, path, sink_blocks, ring_blocks, window, sinks;
  const void *k, *v;
  int64_t s_l, s_n, s_t, s_h;  // elements
  const int32_t* nodes;
  int64_t path_stride;
  const int32_t* counts;
  char* cache;
  int64_t c_l, c_n;  // bytes
  const int64_t* positions;
};

// Eight neighbours as they lie in memory, and in fp32.
template <typename T>
struct Eight {
  u32x4 raw[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Eight<T> load8(const T* p) {
  Eight<T> e;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) e.raw[i] = reinterpret_cast<const u32x4*>(p)[i];
  return e;
}

template <typename T>
__device__ __forceinline__ void widen8(const Eight<T>& e, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    v[j] = sizeof(T) == 2 ? bf16_of(e.raw[0][(j >> 1) & 3], j & 1) : __uint_as_float(e.raw[(int)sizeof(T) / 2 - 1 ? j >> 2 : 0][j & 3]);
}

// Codes (a word) and scale of a group that four neighbouring lanes hold, eight values each.
__device__ __forceinline__ uint32_t quantise8(const float (&v)[8], bf16& scale) {
  float largest = 0.f;
  bool fine = true;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    largest = fmaxf(largest, fabsf(v[j]));
    fine &= fabsf(v[j]) < INFINITY;
  }
  largest = fine ? largest : INFINITY;
  largest = fmaxf(largest, __shfl_xor(largest, 1, 64));
  largest = fmaxf(largest, __shfl_xor(largest, 2, 64));
  scale = fp4_scale(largest, largest < INFINITY);
  return fp4_codes(v, to_f32(scale));
}

// Where a slot's scale stands among its group's.
__device__ __forceinline__ int scale_place(int slot) { return ((slot & 15) >> 2) * 8 + (slot >> 4) * 4 + (slot & 3); }

// One block of slots per workgroup: the first wave takes the keys, the second the values.  A wave finds which token each of
// its 32 slots takes, reads their rows (neighbouring lanes a row's neighbouring pieces), quantises, and turns the codes through LDS
// to the cache's words; slots that no token takes keep their bits.  Prompts of 1024 tokens into 6 layers of 4 requests, 4
// heads of 128: 17 us (3.8 TB/s), bound by finding scales and quotients (571 vector instructions a wave); one token into 12
// layers 4.1 us of latency.  Grid (blocks that a path can touch, requests x heads, layers).
template <typename T, int HD>
__global__ void __launch_bounds__(128) k_kv_commit4(const Commit4Args a) {
  constexpr int kRow = HD / 8, kPasses = kSlots * kRow / 64;  // pieces of a row, and a lane's of the block
  __shared__ uint32_t codes[2][kSlots][kRow + 1];
  const int n = blockIdx.y / a.heads, head = blockIdx.y % a.heads, l = blockIdx.z;
  const int64_t pos = a.positions[n];
  const int count = a.counts ? min(max(a.counts[n], 0), a.path) : a.path;
  if (pos < 0 || count == 0) return;
  // the steps of the path that take sinks, then the ring's
  const int first = (int)min((int64_t)count, max((int64_t)a.sinks - pos, (int64_t)0)), ring = count - first;
  const int64_t past = max(pos + first - a.sinks, (int64_t)0);
  // a 64-bit remainder costs hundreds of instructions
  const int r0 = past >> 32 ? (int)(past % a.window) : (int)((uint32_t)past % (uint32_t)a.window);
  const int sink_from = (int)min(pos, (int64_t)a.sinks), sink0 = sink_from / kSlots;
  const int sink_n = first > 0 ? (sink_from + first - 1) / kSlots - sink0 + 1 : 0;
  const int ring0 = r0 / kSlots;
  int ring_n = 0;
  if (ring >= a.window) {
    ring_n = a.ring_blocks;
  } else if (ring > 0) {
    const int end = r0 + ring;
    ring_n = end <= a.window ? (end - 1) / kSlots - ring0 + 1
                             : min(a.ring_blocks, a.ring_blocks - ring0 + (end - a.window - 1) / kSlots + 1);
  }
  const int c = blockIdx.x;
  if (c >= sink_n + ring_n) return;
  const bool sink = c < sink_n;
  int block = sink ? sink0 + c : ring0 + (c - sink_n);  // of its region
  if (!sink && block >= a.ring_blocks) block -= a.ring_blocks;
  const int lane = threadIdx.x & 63, r = lane & 15, h = lane >> 4, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const bool values = w != 0;
  // the node that slot `lane & 31` of the block takes, -1: none
  int mine = -1;
  {
    const int slot = block * kSlots + (lane & 31);
    int step = -1;
    if (sink) {
      if (slot >= sink_from && slot < sink_from + first) step = slot - sink_from;
    } else if (slot < a.window) {
      int d = slot >= r0 ? slot - r0 : slot - r0 + a.window;
      if (d < ring) {
        if (ring > a.window) d += (ring - 1 - d) / a.window * a.window;  // the last of the slot's steps
        step = first + d;
      }
    }
    if (step >= 0) {
      mine = a.nodes ? a.nodes[n * a.path_stride + step] : step;
      if (mine >= a.n_nodes) mine = -1;
    }
  }
  char* at = a.cache + l * a.c_l + n * a.c_n +
             ((int64_t)head * (a.sink_blocks + a.ring_blocks) + (sink ? 0 : a.sink_blocks) + block) * (36 * HD);
  const T* src = static_cast<const T*>(values ? a.v : a.k) + l * a.s_l + n * a.s_n + head * a.s_h + 8 * (lane % kRow);
  char* scales = at + 32 * HD + (values ? 2 * HD : 0);
  Eight<T> row[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int node = __shfl(mine, (i * 64 + lane) / kRow, 64);
    row[i] = Eight<T>{};
    if (node >= 0) row[i] = load8(src + node * a.s_t);
  }
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int slot = (i * 64 + lane) / kRow, piece = lane % kRow;
    const bool taken = __shfl(mine, slot, 64) >= 0;
    if (!__any(taken)) continue;
    float v[8];
    widen8(row[i], v);
    bf16 s;
    codes[w][slot][piece] = quantise8(v, s);
    if (taken && (piece & 3) == 0) *reinterpret_cast<bf16*>(scales + (piece >> 2) * 64 + scale_place(slot) * 2) = s;
  }
  __syncthreads();
  if (!values) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int slot = 16 * t + r;
      if (__shfl(mine, slot, 64) < 0) continue;
      uint32_t words[HD / 32];
#pragma unroll
      for (int g = 0; g < HD / 32; ++g) words[g] = codes[0][slot][4 * g + h];
      if constexpr (HD == 64)
        *reinterpret_cast<u32x2*>(at + 16 * lane + 8 * t) = u32x2{words[0], words[1]};
      else
        *reinterpret_cast<u32x4*>(at + 1024 * t + 16 * lane) = u32x4{words[0], words[1], words[2], words[3]};
    }
    return;
  }
  uint32_t taken = 0;  // the nibbles of this lane's words that are new
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int node = __shfl(mine, 16 * (j >> 2) + 4 * h + (j & 3), 64);
    taken |= node >= 0 ? 15u << (4 * j) : 0u;
  }
  if (taken == 0) return;
#pragma unroll
  for (int q = 0; q < HD / 64; ++q) {
    u32x4* to = reinterpret_cast<u32x4*>(at + 16 * HD + 1024 * q + 16 * lane);
    u32x4 out{0u, 0u, 0u, 0u};
    if (taken != ~0u) out = *to;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = 16 * (4 * q + i) + r;
      uint32_t word = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        word |= (codes[1][16 * (j >> 2) + 4 * h + (j & 3)][e >> 3] >> (4 * (e & 7)) & 15u) << (4 * j);
      out[i] = (out[i] & ~taken) | (word & taken);
    }
    *to = out;
  }
}

__global__ void __launch_bounds__(kThreads) k_kv_advance4(int64_t* positions, const int32_t* counts, int n, int path) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i < n && positions[i] >= 0) positions[i] += counts ? min(max(counts[i], 0), path) : path;
}

struct Values4Args {
  int heads, sink_blocks, ring_blocks;
  int64_t window, sinks;
  const char* cache;
  int64_t c_l, c_n;
  void *k, *v;
};

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    bf16x8 t;
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = static_cast<bf16>(v[j]);
    *reinterpret_cast<bf16x8*>(p) = t;
  } else {
    *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
  }
}

// A block per workgroup, keys and values a wave each; values turn through LDS so that both store eight neighbours.  Bound by its
// stores: the prompts' caches above 13.5 us (4.8 TB/s with the reads).
// Grid (blocks, requests x heads, layers).
template <typename T, int HD>
__global__ void __launch_bounds__(128) k_kv_values4(const Values4Args a) {
  __shared__ __align__(16) uint8_t codes[kSlots][HD + 8];
  const int n = blockIdx.y / a.heads, head = blockIdx.y % a.heads, l = blockIdx.z, blocks = a.sink_blocks + a.ring_blocks;
  const int n_req = gridDim.y / a.heads;
  const char* at = a.cache + l * a.c_l + n * a.c_n + ((int64_t)head * blocks + blockIdx.x) * (36 * HD);
  const int lane = threadIdx.x & 63, r = lane & 15, h = lane >> 4;
  const bool values = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) != 0;
  const bool sink = (int)blockIdx.x < a.sink_blocks;
  const int64_t slot0 = (int64_t)(sink ? blockIdx.x : blockIdx.x - a.sink_blocks) * kSlots;
  const int held = (int)min((int64_t)kSlots, (sink ? a.sinks : a.window) - slot0);
  T* out = static_cast<T*>(values ? a.v : a.k) +
           ((((int64_t)l * n_req + n) * a.heads + head) * (a.sinks + a.window) + (sink ? slot0 : a.sinks + slot0)) * HD;
  u32x4 piece[HD / 64];
#pragma unroll
  for (int q = 0; q < HD / 64; ++q)
    piece[q] = *reinterpret_cast<const u32x4*>(at + (values ? 16 * HD : 0) + 1024 * q + 16 * lane);
  if (values) {
#pragma unroll
    for (int w = 0; w < HD / 16; ++w)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        codes[16 * (j >> 2) + 4 * h + (j & 3)][16 * w + r] = piece[w >> 2][w & 3] >> (4 * j) & 15u;
  }
  __syncthreads();
  const char* scales = at + 32 * HD + (values ? 2 * HD : 0);
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int g = 0; g < HD / 32; ++g) {
      const int slot = 16 * t + r, w = t * (HD / 32) + g;
      const float s = to_f32(*reinterpret_cast<const bf16*>(scales + g * 64 + scale_place(slot) * 2));
      uint32_t word = piece[w >> 2][w & 3];
      if (values) {
        const uint2 b = *reinterpret_cast<const uint2*>(&codes[slot][32 * g + 8 * h]);
        word = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) word |= ((j < 4 ? b.x >> (8 * j) : b.y >> (8 * (j - 4))) & 15u) << (4 * j);
      }
      const bf16x8 c = fp4_values(word);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_f32(c[j]) * s;
      if (slot < held) store8(out + (int64_t)slot * HD + 32 * g + 8 * h, v);
    }
}

constexpr int kMaxFork4 = 128;

struct Fork4Args {
  int n_req, block_pieces, sink_blocks;
  int64_t blocks, slab, sinks;  // slab: pieces of a request of one layer
  const int32_t* sources;
  char* cache;
  int64_t c_l, c_n;  // bytes
  const int64_t* positions;
};

// A thread owns a piece of every request's slab and loads all that move before it stores any: any map is safe in
// place, without scratch memory.  Blocks that hold no token of the source stay.  Grid (pieces of a slab, layers).
template <typename V, int N>
__global__ void __launch_bounds__(kThreads) k_kv_fork4(const Fork4Args a) {
  const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.slab) return;
  const int64_t block = c / a.block_pieces % a.blocks;
  const int64_t from = block < a.sink_blocks ? block * kSlots : a.sinks + (block - a.sink_blocks) * kSlots;  // its first token
  char* base = a.cache + (int64_t)blockIdx.y * a.c_l + c * (int64_t)sizeof(V);
  V piece[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    piece[n] = V{};
    if (n < a.n_req) {
      const int s = a.sources[n];
      if (s != n && s >= 0 && s < a.n_req && (!a.positions || from < a.positions[s]))
        piece[n] = *reinterpret_cast<const V*>(base + s * a.c_n);
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (n < a.n_req) {
      const int s = a.sources[n];
      if (s != n && s >= 0 && s < a.n_req && (!a.positions || from < a.positions[s]))
        *reinterpret_cast<V*>(base + n * a.c_n) = piece[n];
    }
  }
}

__global__ void __launch_bounds__(kMaxFork4) k_kv_fork4_positions(int64_t* positions, const int32_t* sources, int n_req) {
  const int n = threadIdx.x;
  const int s = n < n_req ? sources[n] : -1;
  const bool moved = s != n && s >= 0 && s < n_req;
  const int64_t p = moved ? positions[s] : 0;
  __syncthreads();
  if (moved) positions[n] = p;
}

// What the three calls ask of a cache that they write or read.
struct CacheShape {
  int64_t layers, n_req, heads, hd, window, sinks, c_l, c_n;
  const void* cache;
  int64_t sink_blocks() const { return (sinks + kSlots - 1) / kSlots; }
  int64_t ring_blocks() const { return (window + kSlots - 1) / kSlots; }
  int64_t slab() const { return heads * (sink_blocks() + ring_blocks()) * 36 * hd; }  // bytes
};

int check_cache(const CacheShape& s, bool written) {
  UTTT_REQUIRE(s.layers >= 1 && s.layers <= 65535 && s.n_req >= 1 && s.heads >= 1 && s.heads <= 65535 &&
                   s.n_req <= 65535 && s.n_req * s.heads <= 65535,
               "layers, or requests x heads, out of range");
  UTTT_REQUIRE(s.hd == 64 || s.hd == 128, "head_dim must be 64 or 128 (got %lld)", (long long)s.hd);
  UTTT_REQUIRE(s.window >= 1 && s.window <= (1LL << 28) && s.sinks >= 0 && s.sinks <= (1LL << 28),
               "window must be in [1, 2^28] and sinks in [0, 2^28]");
  UTTT_REQUIRE(s.cache != nullptr && aligned16(s.cache) && s.c_l % 16 == 0 && s.c_n % 16 == 0,
               "the cache must be non-NULL and 16-byte aligned with strides of whole 16-byte pieces");
  if (!written) return UTTT_OK;
  const int64_t slab = s.slab();
  // the nearer of the two dimensions lies inside the other, whose strides reach past its last cache
  const bool inside = s.c_l >= s.c_n;  // requests inside layers
  const int64_t near = inside ? s.c_n : s.c_l, far = inside ? s.c_l : s.c_n, n_near = inside ? s.n_req : s.layers;
  const bool apart = s.n_req == 1 || s.layers == 1
                         ? (s.n_req == 1 || s.c_n >= slab) && (s.layers == 1 || s.c_l >= slab)
                         : near >= slab && (far - slab) / near >= n_near - 1;
  UTTT_REQUIRE(apart, "the requests' caches must not overlap");
  return UTTT_OK;
}

template <typename T, int HD>
void launch_commit4(const Commit4Args& m, dim3 grid, hipStream_t st) {
  hipLaunchKernelGGL((k_kv_commit4<T, HD>), grid, dim3(128), 0, st, m);
}

template <typename T, int HD>
void launch_values4(const Values4Args& m, dim3 grid, hipStream_t st) {
  hipLaunchKernelGGL((k_kv_values4<T, HD>), grid, dim3(128), 0, st, m);
}

}  // namespace
}  // namespace uttt

using namespace uttt;

extern "C" int uttt_kv_commit4(const uttt_kv_commit4_args* a, uttt_stream_t stream) {
  UTTT_REQUIRE(a != nullptr, "args is NULL");
  const CacheShape s{a->layers, a->n_req, a->n_kv_heads, a->head_dim, a->window, a->sinks, a->cache_stride_l, a->cache_stride_n,
                     a->cache};
  if (const int rc = check_cache(s, true)) return rc;
  UTTT_REQUIRE(a->act_dtype == UTTT_DTYPE_F32 || a->act_dtype == UTTT_DTYPE_BF16, "bad act_dtype");
  UTTT_REQUIRE(a->n_nodes >= 1 && a->n_nodes <= (1LL << 24) && a->path >= 1 && a->path <= (1LL << 24) &&
                   (a->nodes != nullptr || a->path <= a->n_nodes),
               "node or path counts out of range");
  UTTT_REQUIRE(a->k_nodes && a->v_nodes && a->positions, "pointers must be non-NULL");
  const int64_t vec = a->act_dtype == UTTT_DTYPE_BF16 ? 8 : 4;
  UTTT_REQUIRE(aligned16(a->k_nodes) && aligned16(a->v_nodes) && a->nodes_stride_l % vec == 0 && a->nodes_stride_n % vec == 0 &&
                   a->nodes_stride_t % vec == 0 && a->nodes_stride_h % vec == 0,
               "nodes must be 16-byte aligned with strides of whole 16-byte pieces");
  Commit4Args m{};
  m.heads = (int)a->n_kv_heads; m.n_nodes = (int)a->n_nodes; m.path = (int)a->path;
  m.sink_blocks = (int)s.sink_blocks(); m.ring_blocks = (int)s.ring_blocks();
  m.window = (int)a->window; m.sinks = (int)a->sinks;
  m.k = a->k_nodes; m.v = a->v_nodes;
  m.s_l = a->nodes_stride_l; m.s_n = a->nodes_stride_n; m.s_t = a->nodes_stride_t; m.s_h = a->nodes_stride_h;
  m.nodes = a->nodes; m.path_stride = a->path_stride; m.counts = a->counts;
  m.cache = static_cast<char*>(a->cache); m.c_l = a->cache_stride_l; m.c_n = a->cache_stride_n;
  m.positions = a->positions;
  // a run of A slots reaches ceil(A / 32) + 1 blocks, and one more where the ring's last block is cut short
  const int64_t steps = (a->path + kSlots - 1) / kSlots;
  const int64_t most = std::min(s.sink_blocks(), steps + 1) + std::min(s.ring_blocks(), steps + 2);
  const dim3 grid((unsigned)most, (unsigned)(a->n_req * a->n_kv_heads), (unsigned)a->layers);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool b16 = a->act_dtype == UTTT_DTYPE_BF16;
  if (a->head_dim == 64)
    b16 ? launch_commit4<bf16, 64>(m, grid, st) : launch_commit4<float, 64>(m, grid, st);
  else
    b16 ? launch_commit4<bf16, 128>(m, grid, st) : launch_commit4<float, 128>(m, grid, st);
  if (a->advance)
    hipLaunchKernelGGL(k_kv_advance4, dim3((unsigned)((a->n_req + kThreads - 1) / kThreads)), dim3(kThreads), 0, st, a->positions,
                       a->counts, (int)a->n_req, m.path);
  return launch_status("uttt_kv_commit4");
}

extern "C" int uttt_kv_values4(const uttt_kv_values4_args* a, uttt_stream_t stream) {
  UTTT_REQUIRE(a != nullptr, "args is NULL");
  const CacheShape s{a->layers, a->n_req, a->n_kv_heads, a->head_dim, a->window, a->sinks, a->cache_stride_l, a->cache_stride_n,
                     a->cache};
  if (const int rc = check_cache(s, false)) return rc;
  UTTT_REQUIRE(a->act_dtype == UTTT_DTYPE_F32 || a->act_dtype == UTTT_DTYPE_BF16, "bad act_dtype");
  UTTT_REQUIRE(a->k && a->v && aligned16(a->k) && aligned16(a->v), "k and v must be non-NULL and 16-byte aligned");
  Values4Args m{};
  m.heads = (int)a->n_kv_heads; m.sink_blocks = (int)s.sink_blocks(); m.ring_blocks = (int)s.ring_blocks();
  m.window = a->window; m.sinks = a->sinks;
  m.cache = static_cast<const char*>(a->cache); m.c_l = a->cache_stride_l; m.c_n = a->cache_stride_n;
  m.k = a->k; m.v = a->v;
  const dim3 grid((unsigned)(s.sink_blocks() + s.ring_blocks()), (unsigned)(a->n_req * a->n_kv_heads), (unsigned)a->layers);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool b16 = a->act_dtype == UTTT_DTYPE_BF16;
  if (a->head_dim == 64)
    b16 ? launch_values4<bf16, 64>(m, grid, st) : launch_values4<float, 64>(m, grid, st);
  else
    b16 ? launch_values4<bf16, 128>(m, grid, st) : launch_values4<float, 128>(m, grid, st);
  return launch_status("uttt_kv_values4");
}

extern "C" int uttt_kv_fork4(const uttt_kv_fork4_args* a, uttt_stream_t stream) {
  UTTT_REQUIRE(a != nullptr, "args is NULL");
  const CacheShape s{a->layers, a->n_req, a->n_kv_heads, a->head_dim, a->window, a->sinks, a->cache_stride_l, a->cache_stride_n,
                     a->cache};
  if (const int rc = check_cache(s, true)) return rc;
  UTTT_REQUIRE(a->n_req <= kMaxFork4, "at most %d requests", kMaxFork4);
  UTTT_REQUIRE(a->sources != nullptr, "sources must be non-NULL");
  // A thread holds a piece of every request: pieces shrink so that 128 of them fit its registers.  us with these and with the
  // next smaller ones (and registers for twice the requests), any map: 24 layers of 1024 slots, 4 heads of 128, 4 requests 19.3 and
  // 25.9, 16 65 and 76, 32 208 and 237; 12 layers of 512 slots, 4 heads of 64, 17 requests 15.2 and 26.5, 64 79 and 97, 128 176.
  const int64_t piece = a->n_req <= 32 ? 16 : a->n_req <= 64 ? 8 : 4;
  Fork4Args m{};
  m.n_req = (int)a->n_req; m.block_pieces = (int)(36 * a->head_dim / piece); m.sink_blocks = (int)s.sink_blocks();
  m.blocks = s.sink_blocks() + s.ring_blocks(); m.slab = s.slab() / piece; m.sinks = a->sinks;
  m.sources = a->sources;
  m.cache = static_cast<char*>(a->cache); m.c_l = a->cache_stride_l; m.c_n = a->cache_stride_n;
  m.positions = a->positions;
  const int64_t blocks = (m.slab + kThreads - 1) / kThreads;
  UTTT_REQUIRE(blocks <= 0x7fffffffLL, "caches too large for one launch");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)blocks, (unsigned)a->layers);
  if (a->n_req <= 16)
    hipLaunchKernelGGL((k_kv_fork4<u32x4, 16>), grid, dim3(kThreads), 0, st, m);
  else if (a->n_req <= 32)
    hipLaunchKernelGGL((k_kv_fork4<u32x4, 32>), grid, dim3(kThreads), 0, st, m);
  else if (a->n_req <= 64)
    hipLaunchKernelGGL((k_kv_fork4<u32x2, 64>), grid, dim3(kThreads), 0, st, m);
  else
    hipLaunchKernelGGL((k_kv_fork4<uint32_t, 128>), grid, dim3(kThreads), 0, st, m);
  if (a->positions)
    hipLaunchKernelGGL(k_kv_fork4_positions, dim3(1), dim3(kMaxFork4), 0, st, a->positions, a->sources, (int)a->n_req);
  return launch_status("uttt_kv_fork4");
}
