// Attention of a few new tokens per request over ring caches with sink slots, gfx950 (MI355X): a tree of drafted
// tokens, or the one token of a decode step.  Cache layout, visibility and the tree's positions: uttt_serve.h.
//
// One pass over the cache with the running maximum and sum of a softmax, split over a request's slots and
// joined: the rows of a (request, kv head) are its nodes times the query heads that share the keys, 32 rows to a
// unit.  bf16 (k_swa_tree_mm): a workgroup takes U units over a range of 64-slot tiles, each of its four waves
// a quarter of the tiles in LDS of its own, so the waves run without barriers: a wave's K tile is loaded
// while it multiplies weights and values, its V tile while it forms scores.  Both products run on
// v_mfma_f32_32x32x16_bf16 with the scores transposed (S^T = K Q^T: a query per lane, its softmax inside
// the lane and one exchange with the lane 32 away; the rounded weights are the B operand of O^T = V^T P^T as
// they lie).  The new tokens' keys are one more tile, rotated by the whole workgroup into the last wave's
// buffers.  The waves' results meet in LDS, the splits' in a second launch.
//
// Roundings: weights to bf16 as a MFMA operand (sums are formed from the unrounded ones); rotated
// queries are carried as two bf16 terms, so they cost no accuracy beside the keys' own bf16; the new keys are rotated
// in fp32 and rounded once.
//
// Slots that no node of the request may see (unwritten, or out of the window for all) are zeroed in LDS.
// Where a tile's values are seen by some nodes only and hold infinities or NaN, weights of 0 must not meet
// them: that tile's second product is formed with selections instead of MFMA.
#include <math.h>

#include <algorithm>

#include "../../include/uttt_serve.h"
#include "uttt_device.h"
#include "uttt_host.h"

namespace uttt {
namespace {

constexpr int kMaxNodes = 64;
constexpr int kWaves = 4;

struct TreeArgs {
  int n_req, n_kv_heads, rep, nodes, rows;  // rows: nodes * rep
  int groups, nsplit;                       // workgroups along the rows of a (request, kv head), splits of its slots
  int window, sinks, slots;
  int write_ring;
  float scale;
  const int64_t* positions;
  const int32_t *parents, *counts;
  const float *cos_table, *sin_table;
  int64_t table_len;
  const void* q; int64_t q_n, q_t, q_h;
  const void* k; int64_t k_n, k_t, k_h;
  const void* v; int64_t v_n, v_t, v_h;
  void *k_ring, *v_ring; int64_t ring_n;
  void* out; int64_t o_n, o_t, o_h;
  void *k_nodes, *v_nodes;
  float *part_o, *part_ml;  // per (request, kv head, split, row): unnormalised output; maximum (log2 units) and sum
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)uniform((int)x) | (uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32);
}
__device__ __forceinline__ uint64_t shfl64(uint64_t v, int lane) {
  const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)v, lane, 64), hi = (uint32_t)__shfl((int)(uint32_t)(v >> 32), lane, 64);
  return (uint64_t)hi << 32 | lo;
}

// A request's tree, one node per lane.
struct Tree {
  uint64_t sees;  // of this lane's node: the nodes that it sees (ancestors and itself, within the window)
  int depth;      // of this lane's node
  int deepest;    // of the request's nodes
  bool bad;       // a parent that is neither -1 nor an earlier node, or a position out of range
};

__device__ __forceinline__ Tree read_tree(const TreeArgs& a, int n, int count, int64_t pos, int lane) {
  Tree t;
  int up = -1;
  bool bad = false;
  if (lane < count) {
    up = a.parents != nullptr ? a.parents[(int64_t)n * a.nodes + lane] : lane - 1;
    bad = up < -1 || up >= lane;
    if (bad) up = -1;
  }
  // paths to the root by doubling: `up` is the ancestor 2^i steps away
  t.sees = lane < count ? 1ull << lane : 0;
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    const uint64_t above = shfl64(t.sees, max(up, 0));
    const int next = __shfl(up, max(up, 0), 64);
    if (up >= 0) {
      t.sees |= above;
      up = next;
    }
  }
  t.depth = max((int)__popcll(t.sees) - 1, 0);
  int d = t.depth;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) d = max(d, __shfl_xor(d, off, 64));
  t.deepest = uniform(d);
  t.bad = __any(bad) || pos < 0 || (a.cos_table != nullptr && pos + t.deepest >= a.table_len);
  if (t.deepest >= a.window && !t.bad) {  // ancestors out of the window
    for (int j = 0; j < count; ++j) {
      const int dj = __shfl(t.depth, j, 64);
      if (t.depth - dj >= a.window && pos + dj >= a.sinks) t.sees &= ~(1ull << j);
    }
  }
  return t;
}

// What a request's cache holds, as ages: slot sinks + i holds the token of age (cur - i) mod window, the
// newest cached one having age 0.
struct Ring {
  int used;   // slots that hold tokens are those below
  int cur, held;  // of the newest token; ages below `held` exist
};

__device__ __forceinline__ Ring read_ring(const TreeArgs& a, int64_t pos) {
  Ring r;
  r.used = (int)min(max(pos, (int64_t)0), (int64_t)a.slots);
  r.cur = pos > a.sinks ? (int)((pos - 1 - a.sinks) % a.window) : 0;
  r.held = (int)min(max(pos - a.sinks, (int64_t)0), (int64_t)a.window);
  return r;
}

// The ages that a node of depth d sees are those below visible_age(d): a node of depth d sees window - 1 - d
// cached tokens behind the sinks.
__device__ __forceinline__ int visible_age(const TreeArgs& a, const Ring& r, int d) { return min(r.held, a.window - 1 - d); }

// Which of the slots s0 .. s0 + 63 hold a sink or an age below lim: ages run backwards from slot sinks + cur and on
// from the last slot.
__device__ __forceinline__ uint64_t seen_slots(const TreeArgs& a, const Ring& r, int s0, int lim) {
  const int newest = a.sinks + r.cur - s0, oldest = newest - max(lim, 0) + 1, start = a.sinks - s0;
  const int over = max(start - oldest, 0);  // slots of the part that wraps
  return bit_range(-s0, min(a.sinks, r.used) - s0) | bit_range(max(oldest, start), newest + 1) |
         bit_range(a.slots - s0 - over, a.slots - s0);
}

// This workgroup's work.  Row groups of one (request, kv head, split) read the same slots: their ids are 8
// apart, so they run on one XCD and share its L2.
struct Place {
  int n, kvh, split, group;
  bool valid;
};
__device__ __forceinline__ Place place_of(const TreeArgs& a) {
  const int x = blockIdx.x % kXcds, q = blockIdx.x / kXcds;
  const int i = q / a.groups * kXcds + x;
  Place p;
  p.group = q % a.groups;
  p.split = i % a.nsplit;
  p.kvh = i / a.nsplit % a.n_kv_heads;
  p.n = i / a.nsplit / a.n_kv_heads;
  p.valid = p.n < a.n_req;
  return p;
}

__device__ __forceinline__ int64_t part_row(const TreeArgs& a, const Place& p, int row) {
  return (((int64_t)p.n * a.n_kv_heads + p.kvh) * a.nsplit + p.split) * a.rows + row;
}

// NaN for rows [row0, row1) of a request that cannot be computed
template <typename T, int HD>
__device__ __forceinline__ void refuse_rows(const TreeArgs& a, const Place& p, int row0, int row1) {
  for (int i = threadIdx.x; i < (row1 - row0) * HD; i += kThreads) {
    const int row = row0 + i / HD, e = i % HD;
    if (a.nsplit == 1)
      static_cast<T*>(a.out)[p.n * a.o_n + row / a.rep * a.o_t + (p.kvh * a.rep + row % a.rep) * a.o_h + e] =
          from_f32<T>(NAN);
    else if (e == 0)
      a.part_ml[2 * part_row(a, p, row)] = NAN;
  }
}

// where the new key / value row of node t goes, or NULL
template <typename T, int HD>
__device__ __forceinline__ T* node_row(const TreeArgs& a, const Place& p, void* nodes, void* ring, int t, int64_t pos) {
  if (a.write_ring) {
    const int64_t slot = pos < a.sinks ? pos : a.sinks + (pos - a.sinks) % a.window;
    return static_cast<T*>(ring) + p.n * a.ring_n + ((int64_t)p.kvh * a.slots + slot) * HD;
  }
  return static_cast<T*>(nodes) + (((int64_t)p.n * a.nodes + t) * a.n_kv_heads + p.kvh) * HD;
}

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

__device__ __forceinline__ bool finite16(const uint4& v) {  // eight bf16
  auto ok = [](uint32_t x) { return (x & 0x7f80u) != 0x7f80u && (x & 0x7f800000u) != 0x7f800000u; };
  return ok(v.x) && ok(v.y) && ok(v.z) && ok(v.w);
}

template <int HD, int U>
__global__ void __launch_bounds__(kThreads, HD == 64 ? 2 : 1) k_swa_tree_mm(const TreeArgs a) {
  constexpr int NT = HD / 64, NB = HD / 32, KS = HD / 16;
  constexpr int TILE = NT * 8192;  // K (or V) of 64 slots
  constexpr int LOADS = NT * 8;    // 1 KB loads of a tile
  constexpr int RED = HD + 4;      // floats of a query's row when the waves' results meet
  constexpr float kLog2e = 1.4426950408889634f;
  static_assert(kWaves * 32 * RED * 4 <= kWaves * 2 * TILE, "the waves' results fit the tiles' LDS");
  __shared__ __align__(1024) char lds[kWaves * 2 * TILE];
  __shared__ float red_ml[kWaves][32][2];
  __shared__ int tree_odd;  // the new values hold infinities or NaN
  const Place p = place_of(a);
  if (!p.valid) return;
  const int w = uniform((int)threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const int count = a.counts != nullptr ? min(max(uniform(a.counts[p.n]), 0), a.nodes) : a.nodes;
  const int row0 = p.group * 32 * U, row1 = min(row0 + 32 * U, count * a.rep);
  if (row0 >= row1) return;
  const bool first = p.split == 0;

  // ---- this wave's tiles: 64 slots each, in LDS of its own
  const uint32_t k_lds = lds_addr(lds) + (uint32_t)(w * 2 * TILE), v_lds = k_lds + TILE;
  const bf16* kr = static_cast<const bf16*>(a.k_ring) + p.n * a.ring_n + (int64_t)p.kvh * a.slots * HD;
  const bf16* vr = static_cast<const bf16*>(a.v_ring) + p.n * a.ring_n + (int64_t)p.kvh * a.slots * HD;
  const int voff_k[2] = {row_src_off(0, lane, HD), row_src_off(1, lane, HD) - 16 * HD};
  const int voff_v = slab_src_off(0, lane, HD);
  auto issue = [&](const bf16* ring, uint32_t dst, int tile, bool is_k) {
    const int n = max(min(a.slots - tile * 64, 64), 0);  // slots past the ring read as zeros
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const __amdgpu_buffer_rsrc_t rs =
          buffer_rsrc(ring + (int64_t)tile * 64 * HD + 64 * t, (uint32_t)max(n * HD * 2 - 128 * t, 0));
#pragma unroll
      for (int g = 0; g < 8; ++g)
        buffer_load_lds_raw(rs, lds_ptr(dst + (uint32_t)(t * 8192 + g * 1024)), 16,
                            (is_k ? voff_k[g & 1] : voff_v) + g * 16 * HD, 0, 0, 0);
    }
  };
  // the tile a wave starts with needs no position in the first split: ask for it at once (the last wave
  // starts with the new tokens there)
  const bool early = first && w < kWaves - 1;
  if (early) {
    issue(kr, k_lds, w, true);
    issue(vr, v_lds, w, false);
  }
  if (threadIdx.x == 0) tree_odd = 0;
  const int64_t pos = uniform(a.positions[p.n]);
  const Tree tree = read_tree(a, p.n, count, pos, lane);
  if (tree.bad) {
    refuse_rows<bf16, HD>(a, p, row0, row1);
    wait_vmcnt<0>();  // no LDS write of this workgroup's loads outlives it
    return;
  }
  const Ring ring = read_ring(a, pos);
  const int ntiles = (ring.used + 63) / 64;
  const int t_begin = (int)((int64_t)ntiles * p.split / a.nsplit), t_end = (int)((int64_t)ntiles * (p.split + 1) / a.nsplit);
  // wave w takes places w, w + kWaves, .. of the split's list; the first split's has the new tokens at place
  // kWaves - 1, whether or not its cache reaches that far
  auto tile_at = [&](int i) { return t_begin + (first && i >= kWaves ? i - 1 : i); };
  auto has = [&](int i) { return (first && i == kWaves - 1) || tile_at(i) < t_end; };

  // ---- queries: row r of each unit, dims 16 s + 8 h .. + 7 in fragment s; rotated ones as two terms
  const bool turned = a.cos_table != nullptr;
  bf16x8 qf[U][KS], ql[U][KS];
  int lim[U];
  uint64_t sees[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int row = row0 + 32 * u + r;
    const bool ok = row < row1;
    const int t = ok ? row / a.rep : 0, head = p.kvh * a.rep + (ok ? row % a.rep : 0);
    const int d = __shfl(tree.depth, t, 64);
    sees[u] = shfl64(tree.sees, t);
    lim[u] = visible_age(a, ring, d);
    const bf16* qr = static_cast<const bf16*>(a.q) + p.n * a.q_n + t * a.q_t + head * a.q_h + 8 * h;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qf[u][s] = ok ? *reinterpret_cast<const bf16x8*>(qr + 16 * s) : bf16x8{};
      ql[u][s] = bf16x8{};
    }
    if (turned) {
      const float* cr = a.cos_table + (pos + d) * HD + 8 * h;
      const float* sr = a.sin_table + (pos + d) * HD + 8 * h;
#pragma unroll
      for (int s = 0; s < KS / 2; ++s) {
        f32x4 c[2], sn[2];
        c[0] = *reinterpret_cast<const f32x4*>(cr + 16 * s);
        c[1] = *reinterpret_cast<const f32x4*>(cr + 16 * s + 4);
        sn[0] = *reinterpret_cast<const f32x4*>(sr + 16 * s);
        sn[1] = *reinterpret_cast<const f32x4*>(sr + 16 * s + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float lo = to_f32((bf16)qf[u][s][e]), hi = to_f32((bf16)qf[u][s + KS / 2][e]);
          const float ce = c[e >> 2][e & 3], se = sn[e >> 2][e & 3];
          const float x = lo * ce - hi * se, y = hi * ce + lo * se;
          const bf16 xh = from_f32<bf16>(x), yh = from_f32<bf16>(y);
          qf[u][s][e] = xh;
          qf[u][s + KS / 2][e] = yh;
          ql[u][s][e] = from_f32<bf16>(x - to_f32(xh));
          ql[u][s + KS / 2][e] = from_f32<bf16>(y - to_f32(yh));
        }
      }
    }
  }

  // ---- the new tokens' tile, by all waves into the last one's buffers (row tile for K, slab for V)
  if (first) {
    constexpr int HP = HD / 16;  // pairs of 16-byte pieces of a key
    char* kt = lds + (kWaves - 1) * 2 * TILE;
    char* vt = kt + TILE;
    const bool keep = p.group == 0 && (a.write_ring || a.k_nodes != nullptr);
    const bf16* kn = static_cast<const bf16*>(a.k) + p.n * a.k_n + p.kvh * a.k_h;
    const bf16* vn = static_cast<const bf16*>(a.v) + p.n * a.v_n + p.kvh * a.v_h;
#pragma unroll
    for (int i = 0; i < 64 * HP / kThreads; ++i) {
      const int idx = threadIdx.x + i * kThreads, t = idx / HP, pc = idx % HP;
      const int d = __shfl(tree.depth, t, 64);
      bf16x8 lo{}, hi{};
      if (t < count) {
        lo = *reinterpret_cast<const bf16x8*>(kn + t * a.k_t + 8 * pc);
        hi = *reinterpret_cast<const bf16x8*>(kn + t * a.k_t + HD / 2 + 8 * pc);
        if (turned) {
          const float* cr = a.cos_table + (pos + d) * HD + 8 * pc;
          const float* sr = a.sin_table + (pos + d) * HD + 8 * pc;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = to_f32((bf16)lo[e]), y = to_f32((bf16)hi[e]);
            lo[e] = from_f32<bf16>(x * cr[e] - y * sr[e]);
            hi[e] = from_f32<bf16>(y * cr[e] + x * sr[e]);
          }
        }
        if (keep) {
          bf16* to = node_row<bf16, HD>(a, p, a.k_nodes, a.k_ring, t, pos);
          *reinterpret_cast<bf16x8*>(to + 8 * pc) = lo;
          *reinterpret_cast<bf16x8*>(to + HD / 2 + 8 * pc) = hi;
        }
      }
      const int ph = pc + HP;  // piece of the second half
      *reinterpret_cast<bf16x8*>(kt + (pc >> 3) * 8192 + t * 128 + (((pc & 7) ^ row_swz(t)) * 16)) = lo;
      *reinterpret_cast<bf16x8*>(kt + (ph >> 3) * 8192 + t * 128 + (((ph & 7) ^ row_swz(t)) * 16)) = hi;
    }
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 64 * 2 * HP / kThreads; ++i) {
      const int idx = threadIdx.x + i * kThreads, t = idx / (2 * HP), pc = idx % (2 * HP);
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (t < count) {
        x = *reinterpret_cast<const uint4*>(vn + t * a.v_t + 8 * pc);
        odd |= !finite16(x);
        if (keep) *reinterpret_cast<uint4*>(node_row<bf16, HD>(a, p, a.v_nodes, a.v_ring, t, pos) + 8 * pc) = x;
      }
      *reinterpret_cast<uint4*>(vt + (pc >> 3) * 8192 + t * 128 + (((pc & 7) ^ slab_swz(t)) * 16)) = x;
    }
    __syncthreads();  // tree_odd is 0 before it is set
    if (odd) tree_odd = 1;
    __syncthreads();
  }

  // ---- the tiles
  uint32_t ka[4], va[NB];
#pragma unroll
  for (int s = 0; s < 4; ++s) ka[s] = row_frag_addr(k_lds, 0, lane, s);
  {
    // transposing reads in the accumulator's key order: half h takes keys 4 h .. + 3, then 8 + 4 h ..
    const int g = lane >> 4, j16 = lane & 15, t = 4 * (g >> 1) + (j16 >> 2);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int c = 32 * (i & 1) + 16 * (g & 1) + 4 * (j16 & 3);
      va[i] = v_lds + (uint32_t)((i / 2) * 8192 + t * 128 + (((c >> 3) ^ slab_swz(t)) * 16) + (c & 7) * 2);
    }
  }
  const float c2 = a.scale * kLog2e;
  float m[U], l[U];
  f32x16 o[U][NB];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    m[u] = -INFINITY;
    l[u] = 0.f;
#pragma unroll
    for (int i = 0; i < NB; ++i) zero(o[u][i]);
  }
  const int lim_any = visible_age(a, ring, 0), lim_all = visible_age(a, ring, tree.deepest);

  bool loaded = early;  // this wave's next ring tile is on its way
  for (int i = w; has(i); i += kWaves) {
    const bool is_tree = first && i == kWaves - 1;
    const int tile = tile_at(i), s0 = tile * 64;
    const bool more = has(i + kWaves);
    if (!is_tree) {
      if (!loaded) {
        issue(kr, k_lds, tile, true);
        issue(vr, v_lds, tile, false);
      }
      wait_vmcnt<LOADS>();  // K has landed, V may still be on its way
    }
    f32x16 s[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      zero(s[u][0]);
      zero(s[u][1]);
    }
#pragma unroll
    for (int ks = 0; ks < KS; ks += 2) {
      bf16x8 f0[2], f1[2];
      const uint32_t at0 = ka[ks & 3] + (uint32_t)((ks >> 2) * 8192), at1 = ka[(ks + 1) & 3] + (uint32_t)((ks >> 2) * 8192);
      f0[0] = lds_read_bf16x8<0>(at0);
      f0[1] = lds_read_bf16x8<4096>(at0);
      f1[0] = lds_read_bf16x8<0>(at1);
      f1[1] = lds_read_bf16x8<4096>(at1);
      asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(f0[0]), "+v"(f0[1]), "+v"(f1[0]), "+v"(f1[1]));
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          s[u][kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f0[kb], qf[u][ks], s[u][kb], 0, 0, 0);
          s[u][kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f1[kb], qf[u][ks + 1], s[u][kb], 0, 0, 0);
        }
        if (turned) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            s[u][kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f0[kb], ql[u][ks], s[u][kb], 0, 0, 0);
            s[u][kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f1[kb], ql[u][ks + 1], s[u][kb], 0, 0, 0);
          }
        }
      }
    }
    pin_loads();
    // every K read is back: the next tile's K on its way
    const int next = more ? tile_at(i + kWaves) : 0;
    if (more) issue(kr, k_lds, next, true);

    // ---- masks
    uint64_t any = ~0ull, all = 0;  // keys that some node sees, that all see
    if (!is_tree) {
      any = seen_slots(a, ring, s0, lim_any);
      all = seen_slots(a, ring, s0, lim_all);
    }
    if (all != ~0ull) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint64_t vis = is_tree ? sees[u] : seen_slots(a, ring, s0, lim[u]);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) mask_keys(s[u][kb], (uint32_t)(vis >> (32 * kb)));
      }
    }
    // ---- softmax of the tile
    bf16x8 pw[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float tm = s[u][0][0];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) tm = fmaxf(tm, s[u][kb][e]);
      tm = fmaxf(tm, other_half(tm));
      if (__any(tm > m[u])) {
        const float m_new = fmaxf(m[u], tm);
        const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[u] - m_new) * c2);
        m[u] = m_new;
        l[u] *= corr;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[u][b][e] *= corr;
      }
      const float base = m[u] == -INFINITY ? 0.f : m[u] * c2;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][kb][e], c2, -base));
          l[u] += x;
          s[u][kb][e] = x;
          pw[u][2 * kb + (e >> 3)][e & 7] = from_f32<bf16>(x);
        }
    }
    // ---- values
    bool odd = is_tree && tree_odd != 0;
    if (!is_tree) {
      if (more)
        wait_vmcnt<LOADS>();
      else
        wait_vmcnt<0>();
      pin_loads();
      if (any != ~0ull) {  // rows that no node sees: zeros
        for (int t = lane >> 3; t < 64; t += 8)
          if (!((any >> t) & 1)) {
#pragma unroll
            for (int b = 0; b < NT; ++b)
              *reinterpret_cast<uint4*>(lds + (w * 2 + 1) * TILE + b * 8192 + t * 128 + (lane & 7) * 16) =
                  make_uint4(0u, 0u, 0u, 0u);
          }
      }
      if (any != all) {  // rows that some nodes see: infinities or NaN must not meet the others' zeros
        bool bad = false;
        if (((any & ~all) >> lane) & 1) {
#pragma unroll
          for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int j = 0; j < 8; ++j)
              bad |= !finite16(*reinterpret_cast<const uint4*>(lds + (w * 2 + 1) * TILE + b * 8192 + lane * 128 + j * 16));
        }
        odd = __any(bad);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    if (!odd) {
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        i16x4 f[2 * NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint32_t at = va[b] + (uint32_t)(ks * 2048);
          f[2 * b] = lds_read_tr16<0>(at);
          f[2 * b + 1] = lds_read_tr16<1024>(at);
        }
        if constexpr (NB == 4)
          asm volatile("s_waitcnt lgkmcnt(0)"
                       : "+v"(f[0]), "+v"(f[1]), "+v"(f[2]), "+v"(f[3]), "+v"(f[4]), "+v"(f[5]), "+v"(f[6]), "+v"(f[7]));
        else
          asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(f[0]), "+v"(f[1]), "+v"(f[2]), "+v"(f[3]));
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const bf16x8 vf =
              __builtin_bit_cast(bf16x8, __builtin_shufflevector(f[2 * b], f[2 * b + 1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
          for (int u = 0; u < U; ++u) o[u][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pw[u][ks], o[u][b], 0, 0, 0);
        }
      }
    } else {
      // the weights through this wave's K buffer (whatever was on its way there lands first and is asked for
      // again), a key at a time, selected
      wait_vmcnt<0>();
      pin_loads();
      float* ps = reinterpret_cast<float*>(lds + w * 2 * TILE);
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) ps[(32 * kb + acc_row(e)) * 32 + r] = s[u][kb][e];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        for (int key = 0; key < 64; ++key) {
          const float x = ps[key * 32 + r];
          const char* row = lds + (w * 2 + 1) * TILE + key * 128;
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int d = 32 * (b & 1) + 8 * (e >> 2) + 4 * h + (e & 3);
              const float y = to_f32(*reinterpret_cast<const bf16*>(row + (b >> 1) * 8192 + (((d >> 3) ^ slab_swz(key)) * 16) + (d & 7) * 2));
              o[u][b][e] = x > 0.f ? __builtin_fmaf(x, y, o[u][b][e]) : o[u][b][e];
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      if (more) issue(kr, k_lds, next, true);
    }
    pin_loads();
    if (more) issue(vr, v_lds, next, false);
    loaded = more;
  }
  if (early && !has(w)) wait_vmcnt<0>();  // an early tile that the request does not have

  // ---- the waves' results meet, unit by unit
  float* red = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    __syncthreads();
    l[u] += other_half(l[u]);
    if (h == 0) {
      red_ml[w][r][0] = m[u];
      red_ml[w][r][1] = l[u];
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<f32x4*>(red + (w * 32 + r) * RED + 32 * b + 2 * e + 4 * h) =
            f32x4{o[u][b][e], o[u][b][e + 1], o[u][b][e + 2], o[u][b][e + 3]};
    __syncthreads();
    for (int idx = threadIdx.x; idx < 32 * HD / 4; idx += kThreads) {
      const int qr = idx / (HD / 4), e = idx % (HD / 4) * 4, row = row0 + 32 * u + qr;
      if (row >= row1) continue;
      float mm = -INFINITY;
#pragma unroll
      for (int x = 0; x < kWaves; ++x) mm = fmaxf(mm, red_ml[x][qr][0]);
      float den = 0.f;
      f32x4 num{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < kWaves; ++x) {
        const float f = red_ml[x][qr][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((red_ml[x][qr][0] - mm) * c2);
        const f32x4 y = *reinterpret_cast<const f32x4*>(red + (x * 32 + qr) * RED + e);
        den += f * red_ml[x][qr][1];
        if (f != 0.f) num += f * y;
      }
      if (a.nsplit == 1) {
        const float inv = 1.0f / den;
        bf16* og = static_cast<bf16*>(a.out) + p.n * a.o_n + row / a.rep * a.o_t + (p.kvh * a.rep + row % a.rep) * a.o_h + e;
        bf16 y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = from_f32<bf16>(num[j] * inv);
        *reinterpret_cast<uint2*>(og) = *reinterpret_cast<const uint2*>(y);
      } else {
        const int64_t at = part_row(a, p, row);
        *reinterpret_cast<f32x4*>(a.part_o + at * HD + e) = num;
        if (e == 0) {
          a.part_ml[2 * at] = mm * c2;
          a.part_ml[2 * at + 1] = den;
        }
      }
    }
  }
}

// The splits of a row joined: four output elements per thread.
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads) k_swa_tree_join(const TreeArgs a) {
  const int64_t idx = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int e = (int)(idx % (HD / 4)) * 4;
  int64_t i = idx / (HD / 4);
  const int row = (int)(i % a.rows);
  i /= a.rows;
  const int kvh = (int)(i % a.n_kv_heads), n = (int)(i / a.n_kv_heads);
  if (n >= a.n_req) return;
  const int count = a.counts != nullptr ? min(max(a.counts[n], 0), a.nodes) : a.nodes;
  if (row >= count * a.rep) return;
  const int64_t at = ((int64_t)n * a.n_kv_heads + kvh) * a.nsplit * a.rows + row;
  float m = -INFINITY;
  bool bad = false;
  for (int s = 0; s < a.nsplit; ++s) {
    const float x = a.part_ml[2 * (at + (int64_t)s * a.rows)];
    bad |= x != x;
    m = fmaxf(m, x);
  }
  float den = 0.f;
  f32x4 num{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.nsplit; ++s) {
    const int64_t b = at + (int64_t)s * a.rows;
    const float x = a.part_ml[2 * b];
    if (!bad && x != -INFINITY) {
      const float f = __builtin_amdgcn_exp2f(x - m);
      den += f * a.part_ml[2 * b + 1];
      num += f * *reinterpret_cast<const f32x4*>(a.part_o + b * HD + e);
    }
  }
  T* og = static_cast<T*>(a.out) + n * a.o_n + row / a.rep * a.o_t + (kvh * a.rep + row % a.rep) * a.o_h + e;
  const float inv = bad ? NAN : 1.0f / den;
#pragma unroll
  for (int j = 0; j < 4; ++j) og[j] = from_f32<T>(num[j] * inv);
}

// fp32 operands: the same walk with v_mfma_f32_16x16x4f32 and operands straight from memory into registers, for
// research and parity runs.  A workgroup takes 16 rows; its waves take 16 keys each of a 64-key tile and meet at the
// end.  A lane's float4 along a row serves four k steps (dims 16 j + 4 g + i for lane group g, step i), and
// the weights pass through LDS from the scores' layout (a lane: four queries, one key) to the A operand's
// (one query, four keys).
template <int HD>
__global__ void __launch_bounds__(kThreads) k_swa_tree_f32(const TreeArgs a) {
  constexpr int NJ = HD / 16, LK = HD + 4, RED = HD + 4;
  constexpr float kLog2e = 1.4426950408889634f;
  __shared__ __align__(16) float kt[64 * LK];  // the new keys, rotated; at the end the waves' results
  __shared__ __align__(16) float ps[kWaves][16][20];
  __shared__ float red_ml[kWaves][16][2];
  static_assert(kWaves * 16 * RED <= 64 * LK, "the waves' results fit the new keys' LDS");
  const Place p = place_of(a);
  if (!p.valid) return;
  const int w = uniform((int)threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int count = a.counts != nullptr ? min(max(uniform(a.counts[p.n]), 0), a.nodes) : a.nodes;
  const int row0 = p.group * 16, row1 = min(row0 + 16, count * a.rep);
  if (row0 >= row1) return;
  const int64_t pos = uniform(a.positions[p.n]);
  const Tree tree = read_tree(a, p.n, count, pos, lane);
  if (tree.bad) {
    refuse_rows<float, HD>(a, p, row0, row1);
    return;
  }
  const Ring ring = read_ring(a, pos);
  const int ntiles = (ring.used + 63) / 64;
  const int t_begin = (int)((int64_t)ntiles * p.split / a.nsplit), t_end = (int)((int64_t)ntiles * (p.split + 1) / a.nsplit);
  const bool turned = a.cos_table != nullptr, first = p.split == 0;
  // queries: row c, dims 16 j + 4 g .. + 3
  f32x4 q[NJ];
  {
    const int row = row0 + c;
    const bool ok = row < row1;
    const int t = ok ? row / a.rep : 0, head = p.kvh * a.rep + (ok ? row % a.rep : 0);
    const int d = __shfl(tree.depth, t, 64);
    const float* qr = static_cast<const float*>(a.q) + p.n * a.q_n + t * a.q_t + head * a.q_h + 4 * g;
#pragma unroll
    for (int j = 0; j < NJ; ++j) q[j] = ok ? *reinterpret_cast<const f32x4*>(qr + 16 * j) : f32x4{0.f, 0.f, 0.f, 0.f};
    if (turned) {
      const float* cr = a.cos_table + (pos + d) * HD + 4 * g;
      const float* sr = a.sin_table + (pos + d) * HD + 4 * g;
#pragma unroll
      for (int j = 0; j < NJ / 2; ++j) {
        const f32x4 ce = *reinterpret_cast<const f32x4*>(cr + 16 * j), se = *reinterpret_cast<const f32x4*>(sr + 16 * j);
        const f32x4 x = q[j], y = q[j + NJ / 2];
        q[j] = x * ce - y * se;
        q[j + NJ / 2] = y * ce + x * se;
      }
    }
  }
  // scores' layout: this lane's rows 4 g + i
  int lim[4];
  uint64_t sees[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = min(row0 + 4 * g + i, row1 - 1) / a.rep;
    lim[i] = visible_age(a, ring, __shfl(tree.depth, t, 64));
    sees[i] = shfl64(tree.sees, t);
  }
  const int lim_any = visible_age(a, ring, 0), lim_all = visible_age(a, ring, tree.deepest);
  const float* kn = static_cast<const float*>(a.k) + p.n * a.k_n + p.kvh * a.k_h;
  const float* vn = static_cast<const float*>(a.v) + p.n * a.v_n + p.kvh * a.v_h;
  if (first) {
    const bool keep = p.group == 0 && (a.write_ring || a.k_nodes != nullptr);
    for (int idx = threadIdx.x; idx < 64 * HD / 2; idx += kThreads) {
      const int t = idx / (HD / 2), e = idx % (HD / 2);  // a wave stays within one or two nodes
      const int d = __shfl(tree.depth, t, 64);
      float lo = 0.f, hi = 0.f;
      if (t < count) {
        lo = kn[t * a.k_t + e];
        hi = kn[t * a.k_t + HD / 2 + e];
        if (turned) {
          const float ce = a.cos_table[(pos + d) * HD + e], se = a.sin_table[(pos + d) * HD + e];
          const float x = lo, y = hi;
          lo = x * ce - y * se;
          hi = y * ce + x * se;
        }
        if (keep) {
          float* to = node_row<float, HD>(a, p, a.k_nodes, a.k_ring, t, pos);
          to[e] = lo;
          to[HD / 2 + e] = hi;
          to = node_row<float, HD>(a, p, a.v_nodes, a.v_ring, t, pos);
          to[e] = vn[t * a.v_t + e];
          to[HD / 2 + e] = vn[t * a.v_t + HD / 2 + e];
        }
      }
      kt[t * LK + e] = lo;
      kt[t * LK + HD / 2 + e] = hi;
    }
    __syncthreads();
  }
  const float* kr = static_cast<const float*>(a.k_ring) + p.n * a.ring_n + (int64_t)p.kvh * a.slots * HD;
  const float* vr = static_cast<const float*>(a.v_ring) + p.n * a.ring_n + (int64_t)p.kvh * a.slots * HD;
  const float c2 = a.scale * kLog2e;
  float m[4], l[4];
  f32x4 o[NJ];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int tile = first ? t_begin - 1 : t_begin; tile < t_end; ++tile) {
    const bool is_tree = tile < t_begin;
    const int s0 = is_tree ? 16 * w : tile * 64 + 16 * w;  // this wave's 16 keys
    // which of them some row sees, and all
    const uint32_t any = (uint32_t)(is_tree ? bit_range(0, count - s0) : seen_slots(a, ring, s0, lim_any)) & 0xffffu;
    const uint32_t all = is_tree ? 0u : (uint32_t)seen_slots(a, ring, s0, lim_all) & 0xffffu;
    if (any == 0) continue;
    const bool any_c = (any >> c) & 1;
    f32x4 s{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      f32x4 k{0.f, 0.f, 0.f, 0.f};
      if (is_tree)
        k = *reinterpret_cast<const f32x4*>(kt + (s0 + c) * LK + 16 * j + 4 * g);
      else if (any_c)
        k = *reinterpret_cast<const f32x4*>(kr + (int64_t)(s0 + c) * HD + 16 * j + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) s = __builtin_amdgcn_mfma_f32_16x16x4f32(q[j][i], k[i], s, 0, 0, 0);
    }
    // values: keys 4 g + i, dims 16 j + c
    f32x4 v[NJ];
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = s0 + 4 * g + i;
      const bool ok = (any >> (4 * g + i)) & 1, part = !((all >> (4 * g + i)) & 1);
      const float* row = is_tree ? vn + key * a.v_t : vr + (int64_t)key * HD;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        v[j][i] = ok ? row[16 * j + c] : 0.f;
        odd |= part && !(fabsf(v[j][i]) < INFINITY);
      }
    }
    odd = __any(odd);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool vis = ((is_tree ? sees[i] >> s0 : seen_slots(a, ring, s0, lim[i])) >> c) & 1;
      s[i] = vis ? s[i] : -INFINITY;
      float mx = s[i];
#pragma unroll
      for (int off = 1; off < 16; off <<= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
      const float m_new = fmaxf(m[i], mx);
      const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[i] - m_new) * c2);
      m[i] = m_new;
      const float x = s[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((s[i] - m_new) * c2);
      l[i] = l[i] * corr + x;  // this lane's keys; the lanes of a row meet at the end
#pragma unroll
      for (int j = 0; j < NJ; ++j) o[j][i] *= corr;
      ps[w][4 * g + i][c] = x;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    if (!odd) {
      const f32x4 pa = *reinterpret_cast<const f32x4*>(&ps[w][c][4 * g]);
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(pa[i], v[j][i], o[j], 0, 0, 0);
    } else {  // a key at a time, selected: 0 weights must not meet infinities or NaN
      for (int key = 0; key < 16; ++key) {
        if (!((any >> key) & 1)) continue;
        const float* row = is_tree ? vn + (s0 + key) * a.v_t : vr + (int64_t)(s0 + key) * HD;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = ps[w][4 * g + i][key];
#pragma unroll
          for (int j = 0; j < NJ; ++j) o[j][i] = x > 0.f ? __builtin_fmaf(x, row[16 * j + c], o[j][i]) : o[j][i];
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();  // the new keys are read
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) l[i] += __shfl_xor(l[i], off, 64);
    if (c == 0) {
      red_ml[w][4 * g + i][0] = m[i];
      red_ml[w][4 * g + i][1] = l[i];
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) kt[(w * 16 + 4 * g + i) * RED + 16 * j + c] = o[j][i];
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < 16 * HD; idx += kThreads) {
    const int qr = idx / HD, e = idx % HD, row = row0 + qr;
    if (row >= row1) continue;
    float mm = -INFINITY;
#pragma unroll
    for (int x = 0; x < kWaves; ++x) mm = fmaxf(mm, red_ml[x][qr][0]);
    float den = 0.f, num = 0.f;
#pragma unroll
    for (int x = 0; x < kWaves; ++x) {
      const float f = red_ml[x][qr][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((red_ml[x][qr][0] - mm) * c2);
      den += f * red_ml[x][qr][1];
      if (f != 0.f) num += f * kt[(x * 16 + qr) * RED + e];
    }
    if (a.nsplit == 1) {
      static_cast<float*>(a.out)[p.n * a.o_n + row / a.rep * a.o_t + (p.kvh * a.rep + row % a.rep) * a.o_h + e] = num / den;
    } else {
      const int64_t at = part_row(a, p, row);
      a.part_o[at * HD + e] = num;
      if (e == 0) {
        a.part_ml[2 * at] = mm * c2;
        a.part_ml[2 * at + 1] = den;
      }
    }
  }
}

// Workgroups' shape: rows of a workgroup, workgroups along a (request, kv head)'s rows, splits of its slots.
struct TreePlan {
  int units, groups, nsplit;
};

constexpr int kMaxTreeSplits = 64;

TreePlan plan_tree(int64_t n_req, int64_t n_heads, int64_t n_kv_heads, int64_t nodes, int64_t head_dim, int64_t slots,
                   bool b16) {
  TreePlan p;
  const int64_t rows = n_heads / n_kv_heads * nodes;
  p.units = 1;
  const int64_t per = b16 ? 32 * p.units : 16;
  p.groups = (int)((rows + per - 1) / per);
  const int64_t base = n_req * n_kv_heads * p.groups, tiles = (slots + 63) / 64;
  const int64_t want = head_dim == 64 ? 512 : 256, least = 8;  // workgroups, tiles of a split
  p.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({(want + base - 1) / base, tiles / least, (int64_t)kMaxTreeSplits}));
  return p;
}

template <int HD>
void launch_tree(const TreeArgs& m, const TreePlan& p, bool b16, hipStream_t st) {
  const int64_t lists = (int64_t)m.n_req * m.n_kv_heads * m.nsplit;
  const dim3 grid((unsigned)((lists + kXcds - 1) / kXcds * kXcds * m.groups));
  if (!b16)
    hipLaunchKernelGGL(k_swa_tree_f32<HD>, grid, dim3(kThreads), 0, st, m);
  else
    hipLaunchKernelGGL((k_swa_tree_mm<HD, 1>), grid, dim3(kThreads), 0, st, m);
  if (m.nsplit > 1) {
    const int64_t n = (int64_t)m.n_req * m.n_kv_heads * m.rows * (HD / 4);
    const dim3 jg((unsigned)((n + kThreads - 1) / kThreads));
    if (b16)
      hipLaunchKernelGGL((k_swa_tree_join<bf16, HD>), jg, dim3(kThreads), 0, st, m);
    else
      hipLaunchKernelGGL((k_swa_tree_join<float, HD>), jg, dim3(kThreads), 0, st, m);
  }
}

}  // namespace
}  // namespace uttt

using namespace uttt;

extern "C" size_t uttt_swa_tree_workspace(int64_t n_req, int64_t n_heads, int64_t n_kv_heads, int64_t nodes,
                                          int64_t head_dim, int64_t slots, int32_t act_dtype) {
  if (n_req < 1 || n_kv_heads < 1 || n_heads < n_kv_heads || nodes < 1 || head_dim < 1 || slots < 1) return 0;
  const TreePlan p = plan_tree(n_req, n_heads, n_kv_heads, nodes, head_dim, slots, act_dtype == UTTT_DTYPE_BF16);
  if (p.nsplit == 1) return 16;
  return sizeof(float) * (size_t)p.nsplit * (size_t)n_req * (size_t)n_heads * (size_t)nodes * (size_t)(head_dim + 2);
}

extern "C" int uttt_swa_tree(const uttt_swa_tree_args* a, uttt_stream_t stream) {
  UTTT_REQUIRE(a != nullptr, "args is NULL");
  UTTT_REQUIRE(a->head_dim == 64 || a->head_dim == 128, "head_dim must be 64 or 128 (got %lld)", (long long)a->head_dim);
  UTTT_REQUIRE(a->n_req >= 1 && a->n_req <= (1LL << 20) && a->n_kv_heads >= 1 && a->n_kv_heads <= 65535 &&
                   a->n_heads >= 1 && a->n_heads <= 65535 && a->n_heads % a->n_kv_heads == 0,
               "bad request / head counts");
  UTTT_REQUIRE(a->nodes >= 1 && a->nodes <= kMaxNodes, "nodes must be in [1, %d]", kMaxNodes);
  UTTT_REQUIRE(a->window >= 1 && a->window <= (1LL << 28) && a->sinks >= 0 && a->sinks <= (1LL << 28),
               "window or sinks out of range");
  UTTT_REQUIRE(a->act_dtype == UTTT_DTYPE_F32 || a->act_dtype == UTTT_DTYPE_BF16, "bad act_dtype");
  UTTT_REQUIRE(a->scale > 0.f, "scale must be > 0");
  UTTT_REQUIRE(a->positions && a->q && a->k_new && a->v_new && a->k_ring && a->v_ring && a->out,
               "pointers must be non-NULL");
  UTTT_REQUIRE(a->write_ring ? a->nodes == 1 && !a->k_nodes && !a->v_nodes : (a->k_nodes == nullptr) == (a->v_nodes == nullptr),
               "write_ring takes one node and no node buffers; node buffers come in pairs");
  UTTT_REQUIRE((a->cos_table == nullptr) == (a->sin_table == nullptr), "cos/sin tables must both be given or both NULL");
  const int64_t vec = a->act_dtype == UTTT_DTYPE_BF16 ? 8 : 4;
  auto whole = [vec](int64_t x, int64_t y, int64_t z) { return x % vec == 0 && y % vec == 0 && z % vec == 0; };
  UTTT_REQUIRE(aligned16(a->q) && aligned16(a->k_new) && aligned16(a->v_new) && aligned16(a->k_ring) &&
                   aligned16(a->v_ring) && aligned16(a->out) && aligned16(a->k_nodes) && aligned16(a->v_nodes) &&
                   aligned16(a->cos_table) && aligned16(a->sin_table) && whole(a->q_stride_n, a->q_stride_t, a->q_stride_h) &&
                   whole(a->k_stride_n, a->k_stride_t, a->k_stride_h) && whole(a->v_stride_n, a->v_stride_t, a->v_stride_h) &&
                   whole(a->o_stride_n, a->o_stride_t, a->o_stride_h) && a->ring_stride_n % vec == 0,
               "operands must be 16-byte aligned with strides of whole 16-byte pieces");
  const bool b16 = a->act_dtype == UTTT_DTYPE_BF16;
  const int64_t slots = a->window + a->sinks;
  const TreePlan p = plan_tree(a->n_req, a->n_heads, a->n_kv_heads, a->nodes, a->head_dim, slots, b16);
  UTTT_REQUIRE((a->n_req * a->n_kv_heads * p.nsplit + kXcds) * p.groups <= 0x7fffffffLL &&
                   a->n_req * a->n_heads * a->nodes * (a->head_dim / 4) / kThreads < 0x7fffffffLL,
               "too many requests for one launch");
  UTTT_REQUIRE(p.nsplit == 1 || (a->workspace != nullptr && aligned16(a->workspace) &&
                                 a->workspace_bytes >= uttt_swa_tree_workspace(a->n_req, a->n_heads, a->n_kv_heads, a->nodes,
                                                                               a->head_dim, slots, a->act_dtype)),
               "tree attention workspace too small");
  TreeArgs m{};
  m.n_req = (int)a->n_req; m.n_kv_heads = (int)a->n_kv_heads; m.rep = (int)(a->n_heads / a->n_kv_heads);
  m.nodes = (int)a->nodes; m.rows = m.rep * m.nodes;
  m.groups = p.groups; m.nsplit = p.nsplit;
  m.window = (int)a->window; m.sinks = (int)a->sinks; m.slots = (int)slots;
  m.write_ring = a->write_ring; m.scale = a->scale;
  m.positions = a->positions; m.parents = a->parents; m.counts = a->counts;
  m.cos_table = a->cos_table; m.sin_table = a->sin_table; m.table_len = a->table_len;
  m.q = a->q; m.q_n = a->q_stride_n; m.q_t = a->q_stride_t; m.q_h = a->q_stride_h;
  m.k = a->k_new; m.k_n = a->k_stride_n; m.k_t = a->k_stride_t; m.k_h = a->k_stride_h;
  m.v = a->v_new; m.v_n = a->v_stride_n; m.v_t = a->v_stride_t; m.v_h = a->v_stride_h;
  m.k_ring = a->k_ring; m.v_ring = a->v_ring; m.ring_n = a->ring_stride_n;
  m.out = a->out; m.o_n = a->o_stride_n; m.o_t = a->o_stride_t; m.o_h = a->o_stride_h;
  m.k_nodes = a->k_nodes; m.v_nodes = a->v_nodes;
  if (p.nsplit > 1) {
    m.part_o = static_cast<float*>(a->workspace);
    m.part_ml = m.part_o + (int64_t)p.nsplit * a->n_req * a->n_heads * a->nodes * a->head_dim;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->head_dim == 64)
    launch_tree<64>(m, p, b16, st);
  else
    launch_tree<128>(m, p, b16, st);
  return launch_status("uttt_swa_tree");
}
