// Copies between the ring caches of batched decoding, written for gfx950 (MI355X): the accepted nodes of a
// draft into every layer's ring (uttt_kv_commit), and whole requests' caches over others' (uttt_kv_fork).
#include <algorithm>

#include "../../include/uttt_serve.h"
#include "uttt_device.h"
#include "uttt_host.h"

namespace uttt {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct CommitArgs {
  int layers, heads, n_nodes, path, pieces;  // pieces: 16-byte pieces of a head's row
  int64_t window, sinks, slots;
  const u32x4 *k_nodes, *v_nodes;
  int64_t nodes_l, nodes_n;  // strides in pieces
  const int32_t* nodes;
  int64_t path_stride;
  const int32_t* counts;
  u32x4 *k_ring, *v_ring;
  int64_t ring_l, ring_n;
  const int64_t* positions;
};

// One 16-byte piece of a key and of the value beside it per thread, a node's row of a head in consecutive
// threads, all layers in one launch: bound by the bytes where there are many (24 layers, 32 requests, paths of up to
// 64 nodes of 4 heads x 128 bf16 21 us, 4.7 TB/s), by the launch where there are few (2.3 us).
// Grid (pieces of all layers and path steps, requests).
__global__ void __launch_bounds__(kThreads) k_kv_commit(const CommitArgs a) {
  const int n = blockIdx.y;
  const int64_t pos = a.positions[n];
  const int count = min(max(a.counts[n], 0), a.path);
  int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int p = (int)(i % a.pieces);
  i /= a.pieces;
  const int h = (int)(i % a.heads);
  i /= a.heads;
  const int step = (int)(i % a.path), l = (int)(i / a.path);
  if (l >= a.layers || step >= count || pos < 0) return;
  const int node = a.nodes[n * a.path_stride + step];
  if (node < 0 || node >= a.n_nodes) return;
  const int64_t at = pos + step;
  int64_t slot = at;
  if (at >= a.sinks) {
    if (step + a.window < count) return;  // a later step of this path takes the same slot
    slot = a.sinks + (at - a.sinks) % a.window;
  }
  const int64_t from = l * a.nodes_l + n * a.nodes_n + ((int64_t)node * a.heads + h) * a.pieces + p;
  const int64_t to = l * a.ring_l + n * a.ring_n + (h * a.slots + slot) * a.pieces + p;
  const u32x4 k = a.k_nodes[from], v = a.v_nodes[from];
  a.k_ring[to] = k;
  a.v_ring[to] = v;
}

__global__ void __launch_bounds__(kThreads) k_kv_advance(int64_t* positions, const int32_t* counts, int n, int path) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i < n && positions[i] >= 0) positions[i] += min(max(counts[i], 0), path);
}

struct ForkArgs {
  int n_req, row_pieces;  // pieces of a slot's row
  int64_t slots, slab;    // pieces of a request's slab of one layer
  const int32_t* sources;
  char *k_ring, *v_ring;
  int64_t ring_l, ring_n;  // strides in pieces
  const int64_t* positions;
};

// A thread owns one piece of a slab, in every request: it loads the pieces of all requests that move
// before it stores any, and no other thread touches them, so any map of sources is safe in place, without scratch
// memory.  Bound by the bytes: 16 requests of 24 layers of 4 heads x 1028 slots x 128 bf16 exchanged at random take 249
// us, 4.5 TB/s read and written.  grid (pieces of a slab, 2 x layers).
template <typename V, int N>
__global__ void __launch_bounds__(kThreads) k_kv_fork(const ForkArgs a) {
  const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.slab) return;
  const int64_t slot = c / a.row_pieces % a.slots;
  V* base = reinterpret_cast<V*>(blockIdx.y & 1 ? a.v_ring : a.k_ring) + (int64_t)(blockIdx.y >> 1) * a.ring_l + c;
  V piece[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    piece[n] = V{};
    if (n < a.n_req) {
      const int s = a.sources[n];
      if (s != n && s >= 0 && s < a.n_req && slot < a.positions[s]) piece[n] = base[s * a.ring_n];
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (n < a.n_req) {
      const int s = a.sources[n];
      if (s != n && s >= 0 && s < a.n_req && slot < a.positions[s]) base[n * a.ring_n] = piece[n];
    }
  }
}

constexpr int kMaxFork = 128;

__global__ void __launch_bounds__(kMaxFork) k_kv_fork_positions(int64_t* positions, const int32_t* sources, int n_req) {
  const int n = threadIdx.x;
  const int s = n < n_req ? sources[n] : -1;
  const bool moved = s != n && s >= 0 && s < n_req;
  const int64_t p = moved ? positions[s] : 0;
  __syncthreads();
  if (moved) positions[n] = p;
}

// Whether the requests' slabs of all layers, which the call writes, lie apart.
bool slabs_apart(int64_t layers, int64_t stride_l, int64_t n_req, int64_t stride_n, int64_t slab) {
  if (n_req == 1 || layers == 1)
    return (n_req == 1 || stride_n >= slab) && (layers == 1 || stride_l >= slab);
  return stride_l >= stride_n ? stride_n >= slab && stride_l / n_req >= stride_n
                              : stride_l >= slab && stride_n / layers >= stride_l;
}

}  // namespace
}  // namespace uttt

using namespace uttt;

extern "C" int uttt_kv_commit(const uttt_kv_commit_args* a, uttt_stream_t stream) {
  UTTT_REQUIRE(a != nullptr, "args is NULL");
  UTTT_REQUIRE(a->layers >= 1 && a->layers <= 65535 && a->n_req >= 1 && a->n_req <= 65535, "layers / requests out of range");
  UTTT_REQUIRE(a->n_kv_heads >= 1 && a->n_kv_heads <= 65535 && a->n_nodes >= 1 && a->n_nodes <= 65535 && a->path >= 1 &&
                   a->path <= 65535,
               "head, node or path counts out of range");
  UTTT_REQUIRE(a->window >= 1 && a->window <= (1LL << 40) && a->sinks >= 0 && a->sinks <= (1LL << 40),
               "window must be >= 1 and sinks >= 0");
  UTTT_REQUIRE(a->act_dtype == UTTT_DTYPE_F32 || a->act_dtype == UTTT_DTYPE_BF16, "bad act_dtype");
  const int64_t vec = a->act_dtype == UTTT_DTYPE_BF16 ? 8 : 4;
  UTTT_REQUIRE(a->head_dim >= vec && a->head_dim <= 65536 && a->head_dim % vec == 0,
               "head_dim must be whole 16-byte pieces");
  UTTT_REQUIRE(a->k_nodes && a->v_nodes && a->nodes && a->counts && a->k_ring && a->v_ring && a->positions,
               "pointers must be non-NULL");
  UTTT_REQUIRE(aligned16(a->k_nodes) && aligned16(a->v_nodes) && aligned16(a->k_ring) && aligned16(a->v_ring) &&
                   a->nodes_stride_l % vec == 0 && a->nodes_stride_n % vec == 0 && a->ring_stride_l % vec == 0 &&
                   a->ring_stride_n % vec == 0,
               "nodes and rings must be 16-byte aligned with strides of whole pieces");
  UTTT_REQUIRE((double)a->n_kv_heads * (double)(a->sinks + a->window) * (double)a->head_dim < (double)(1LL << 60) &&
                   slabs_apart(a->layers, a->ring_stride_l, a->n_req, a->ring_stride_n,
                               a->n_kv_heads * (a->sinks + a->window) * a->head_dim),
               "the requests' rings must not overlap");
  CommitArgs m{};
  m.layers = (int)a->layers; m.heads = (int)a->n_kv_heads; m.n_nodes = (int)a->n_nodes; m.path = (int)a->path;
  m.pieces = (int)(a->head_dim / vec);
  m.window = a->window; m.sinks = a->sinks; m.slots = a->sinks + a->window;
  m.k_nodes = static_cast<const u32x4*>(a->k_nodes); m.v_nodes = static_cast<const u32x4*>(a->v_nodes);
  m.nodes_l = a->nodes_stride_l / vec; m.nodes_n = a->nodes_stride_n / vec;
  m.nodes = a->nodes; m.path_stride = a->path_stride; m.counts = a->counts;
  m.k_ring = static_cast<u32x4*>(a->k_ring); m.v_ring = static_cast<u32x4*>(a->v_ring);
  m.ring_l = a->ring_stride_l / vec; m.ring_n = a->ring_stride_n / vec;
  m.positions = a->positions;
  const double total = (double)a->layers * a->path * a->n_kv_heads * m.pieces;
  UTTT_REQUIRE(total < (double)(1LL << 38), "too many pieces for one launch");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t blocks = ((int64_t)total + kThreads - 1) / kThreads;
  hipLaunchKernelGGL(k_kv_commit, dim3((unsigned)blocks, (unsigned)a->n_req), dim3(kThreads), 0, st, m);
  if (a->advance)
    hipLaunchKernelGGL(k_kv_advance, dim3((unsigned)((a->n_req + kThreads - 1) / kThreads)), dim3(kThreads), 0, st,
                       a->positions, a->counts, (int)a->n_req, m.path);
  return launch_status("uttt_kv_commit");
}

extern "C" int uttt_kv_fork(const uttt_kv_fork_args* a, uttt_stream_t stream) {
  UTTT_REQUIRE(a != nullptr, "args is NULL");
  UTTT_REQUIRE(a->layers >= 1 && a->layers <= 32767, "layers out of range");
  UTTT_REQUIRE(a->n_req >= 1 && a->n_req <= kMaxFork, "at most %d requests", kMaxFork);
  UTTT_REQUIRE(a->n_kv_heads >= 1 && a->n_kv_heads <= 65535 && a->slots >= 1 && a->slots <= (1LL << 31),
               "head or slot counts out of range");
  UTTT_REQUIRE(a->act_dtype == UTTT_DTYPE_F32 || a->act_dtype == UTTT_DTYPE_BF16, "bad act_dtype");
  const int64_t size = a->act_dtype == UTTT_DTYPE_BF16 ? 2 : 4, vec = 16 / size;
  UTTT_REQUIRE(a->head_dim >= vec && a->head_dim <= 65536 && a->head_dim % vec == 0,
               "head_dim must be whole 16-byte pieces");
  UTTT_REQUIRE(a->sources && a->k_ring && a->v_ring && a->positions, "pointers must be non-NULL");
  UTTT_REQUIRE(aligned16(a->k_ring) && aligned16(a->v_ring) && a->ring_stride_l % vec == 0 && a->ring_stride_n % vec == 0,
               "rings must be 16-byte aligned with strides of whole pieces");
  UTTT_REQUIRE((double)a->n_kv_heads * (double)a->slots * (double)a->head_dim < (double)(1LL << 60) &&
                   slabs_apart(a->layers, a->ring_stride_l, a->n_req, a->ring_stride_n, a->n_kv_heads * a->slots * a->head_dim),
               "the requests' rings must not overlap");
  // A thread holds a piece of every request, so the kernel for more requests has more registers and fewer waves, and pieces
  // shrink so that 128 of them fit.  12 layers of 4 heads x 516 slots x 64 bf16, us, the kernel of its size and the next
  // larger: 16 requests 18 and 57 (of 64), 32 requests 55 and 89, 64 requests with pieces of 8 bytes 189 and of 16 191,
  // 128 with 4 bytes 540 and with 8 602 (one for up to 4 requests gave 8.8 for 9.0 and is not kept).
  const int64_t piece = a->n_req <= 32 ? 16 : a->n_req <= 64 ? 8 : 4, per = piece / size;
  ForkArgs m{};
  m.n_req = (int)a->n_req; m.row_pieces = (int)(a->head_dim / per);
  m.slots = a->slots; m.slab = a->n_kv_heads * a->slots * m.row_pieces;
  m.sources = a->sources;
  m.k_ring = static_cast<char*>(a->k_ring); m.v_ring = static_cast<char*>(a->v_ring);
  m.ring_l = a->ring_stride_l / per; m.ring_n = a->ring_stride_n / per;
  m.positions = a->positions;
  const int64_t blocks = (m.slab + kThreads - 1) / kThreads;
  UTTT_REQUIRE(blocks <= 0x7fffffffLL, "slabs too large for one launch");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)blocks, (unsigned)(2 * a->layers));
  if (a->n_req <= 16)
    hipLaunchKernelGGL((k_kv_fork<u32x4, 16>), grid, dim3(kThreads), 0, st, m);
  else if (a->n_req <= 32)
    hipLaunchKernelGGL((k_kv_fork<u32x4, 32>), grid, dim3(kThreads), 0, st, m);
  else if (a->n_req <= 64)
    hipLaunchKernelGGL((k_kv_fork<u32x2, 64>), grid, dim3(kThreads), 0, st, m);
  else
    hipLaunchKernelGGL((k_kv_fork<uint32_t, 128>), grid, dim3(kThreads), 0, st, m);
  hipLaunchKernelGGL(k_kv_fork_positions, dim3(1), dim3(kMaxFork), 0, st, a->positions, a->sources, (int)a->n_req);
  return launch_status("uttt_kv_fork");
}
