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
// buffers.  The waves' results meet in LDS, the splits' in a second launch.  Long caches are bound by their bytes (32
// requests over 4096 slots of head_dim 128, bf16: 44 us and 4 for the join, 5.1 TB/s), single requests by the chain
// of latencies (one over 512 slots of head_dim 64: 11.4 us).
//
// Roundings: weights to bf16 as a MFMA operand (sums are formed from the unrounded ones); rotated
// queries are carried as two bf16 terms, so they cost no accuracy beside the keys' own bf16; the new keys are rotated
// in fp32 and rounded once.
//
// Slots that no node of the request may see (unwritten, or out of the window for all) are zeroed in LDS.
// Where values that some nodes see and others do not hold infinities or NaN, weights of 0 must not meet them: those
// rows are computed again, a row per wave and only over the keys it sees (selected_row; slow, and rare).
#include <math.h>

#include <algorithm>

#include "../../include/uttt_serve.h"
#include "uttt_device.h"
#include "uttt_host.h"

namespace uttt {
namespace {

constexpr int kMaxNodes = 64;
constexpr float kLog2e = 1.4426950408889634f;
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
  int used;       // slots that hold tokens are those below
  int cur, held;  // of the newest token; ages below `held` exist
};

// The slots outside every node's view start behind the newest token and may go on from the window's first slot:
// [from, to) and [sinks, over).
struct Edge {
  int from, to, over;
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

__device__ __forceinline__ Edge read_edge(const TreeArgs& a, const Ring& r, int lim_all) {
  Edge e;
  e.from = r.used < a.sinks ? r.used : a.sinks + r.cur + 1;
  e.to = e.from + a.window - max(lim_all, 0);
  e.over = a.sinks + max(e.to - a.slots, 0);
  if (r.used < a.sinks) e.to = a.slots;
  return e;
}
// whether every node sees the 64 slots from s0
__device__ __forceinline__ bool clean_tile(const TreeArgs& a, const Edge& e, int s0) {
  return s0 + 64 <= a.slots && (s0 + 64 <= e.from || s0 >= e.to) && (e.over == a.sinks || s0 + 64 <= a.sinks || s0 >= e.over);
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

template <typename T>
__device__ __forceinline__ T* out_row(const TreeArgs& a, const Place& p, int row) {
  return static_cast<T*>(a.out) + p.n * a.o_n + row / a.rep * a.o_t + (p.kvh * a.rep + row % a.rep) * a.o_h;
}

// NaN for rows [row0, row1) of a request that cannot be computed
template <typename T, int HD>
__device__ __forceinline__ void refuse_rows(const TreeArgs& a, const Place& p, int row0, int row1, int threads) {
  for (int i = threadIdx.x; i < (row1 - row0) * HD; i += threads) {
    const int row = row0 + i / HD, e = i % HD;
    if (a.nsplit == 1)
      out_row<T>(a, p, row)[e] = from_f32<T>(NAN);
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

// LDS bytes of 64 keys (or values): HD / 64 row tiles (slabs) of 8 KB
template <int HD>
constexpr int kTileBytes = HD / 64 * 8192;

// The 1 KB loads g of the HD / 8 that bring a tile of 64 slots of a (request, kv head)'s keys or values into LDS, as a row
// tile (K) or a slab (V).  Slots past the ring read as zeros.
template <int HD, bool K>
struct TileLoad {
  __amdgpu_buffer_rsrc_t ring;
  int even, odd;  // this lane's piece of row groups 0 and 1, less the group's own offset
  __device__ __forceinline__ TileLoad(const void* base, int slots, int lane)
      : ring(buffer_rsrc(base, (uint32_t)(slots * HD * 2))),
        even(K ? row_src_off(0, lane, HD) : slab_src_off(0, lane, HD)),
        odd(K ? row_src_off(1, lane, HD) - 16 * HD : even) {}
  __device__ __forceinline__ void issue(uint32_t dst, int tile, int g) const {
    const int rg = g & 7;
    buffer_load_lds_raw(ring, lds_ptr(dst + (uint32_t)(g * 1024)), 16,
                        (rg & 1 ? odd : even) + (tile * 128 * HD + rg * 16 * HD + (g >> 3) * 128), 0, 0, 0);
  }
};

// 32 rows of a (request, kv head) in one wave: a query per lane (both halves of the wave hold it), its softmax and its
// output, transposed (o[b][e]: dim 32 b + 8 (e / 4) + 4 h + e % 4).
template <int HD>
struct Unit {
  static constexpr int NB = HD / 32, KS = HD / 16;
  bf16x8 qf[KS], ql[KS];  // dims 16 s + 8 h .. + 7 in fragment s; rotated queries as two terms
  int lim;                // ages below it are seen
  uint64_t sees;          // nodes that are seen
  float m, l;
  f32x16 o[NB];

  __device__ __forceinline__ void load(const TreeArgs& a, const Place& p, const Tree& tree, const Ring& ring, int64_t pos,
                                       int row, int row1) {
    const int h = (threadIdx.x & 63) >> 5;
    const bool ok = row < row1;
    const int t = ok ? row / a.rep : 0, head = p.kvh * a.rep + (ok ? row % a.rep : 0);
    const int d = __shfl(tree.depth, t, 64);
    sees = shfl64(tree.sees, t);
    lim = visible_age(a, ring, d);
    const bf16* qr = static_cast<const bf16*>(a.q) + p.n * a.q_n + t * a.q_t + head * a.q_h + 8 * h;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qf[s] = ok ? *reinterpret_cast<const bf16x8*>(qr + 16 * s) : bf16x8{};
      ql[s] = bf16x8{};
    }
    if (a.cos_table != nullptr) {
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
          const float lo = to_f32((bf16)qf[s][e]), hi = to_f32((bf16)qf[s + KS / 2][e]);
          const float ce = c[e >> 2][e & 3], se = sn[e >> 2][e & 3];
          const float x = lo * ce - hi * se, y = hi * ce + lo * se;
          const bf16 xh = from_f32<bf16>(x), yh = from_f32<bf16>(y);
          qf[s][e] = xh;
          qf[s + KS / 2][e] = yh;
          ql[s][e] = from_f32<bf16>(x - to_f32(xh));
          ql[s + KS / 2][e] = from_f32<bf16>(y - to_f32(yh));
        }
      }
    }
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) zero(o[b]);
  }

  // s = K Q^T of a tile of 64 keys (a row tile at LDS address k)
  __device__ __forceinline__ void scores(f32x16 (&s)[2], uint32_t k, bool two_terms) const {
    const int lane = threadIdx.x & 63;
    zero(s[0]);
    zero(s[1]);
    bf16x8 f[2][4];
    auto read = [&](bf16x8(&x)[4], int ks) {
      const uint32_t at = k + (uint32_t)((ks >> 2) * 8192);
      const uint32_t at0 = row_frag_addr(at, 0, lane, ks & 3), at1 = row_frag_addr(at, 0, lane, (ks + 1) & 3);
      x[0] = lds_read_bf16x8<0>(at0);
      x[1] = lds_read_bf16x8<4096>(at0);
      x[2] = lds_read_bf16x8<0>(at1);
      x[3] = lds_read_bf16x8<4096>(at1);
    };
    read(f[0], 0);
#pragma unroll
    for (int ks = 0; ks < KS; ks += 2) {
      bf16x8(&x)[4] = f[(ks >> 1) & 1];
      if (ks + 2 < KS) {
        read(f[((ks >> 1) + 1) & 1], ks + 2);
        asm volatile("s_waitcnt lgkmcnt(4)" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));
      } else {
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));
      }
      s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[0], qf[ks], s[0], 0, 0, 0);
      s[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[1], qf[ks], s[1], 0, 0, 0);
      s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[2], qf[ks + 1], s[0], 0, 0, 0);
      s[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[3], qf[ks + 1], s[1], 0, 0, 0);
      if (two_terms) {
        s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[0], ql[ks], s[0], 0, 0, 0);
        s[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[1], ql[ks], s[1], 0, 0, 0);
        s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[2], ql[ks + 1], s[0], 0, 0, 0);
        s[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[3], ql[ks + 1], s[1], 0, 0, 0);
      }
    }
  }

  // the tile's weights, rounded, as the B operand of the second product
  __device__ __forceinline__ void softmax(const f32x16 (&s)[2], bf16x8 (&p)[4], float c2) {
    float tm = s[0][0];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) tm = fmaxf(tm, s[kb][e]);
    tm = fmaxf(tm, other_half(tm));
    if (__any(tm > m)) {
      const float m_new = fmaxf(m, tm);
      const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - m_new) * c2);
      m = m_new;
      l *= corr;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[b][e] *= corr;
    }
    const float base = m == -INFINITY ? 0.f : m * c2;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][e], c2, -base));
        l += x;
        p[2 * kb + (e >> 3)][e & 7] = from_f32<bf16>(x);
      }
  }

  // o += V^T P^T of a tile (a slab at LDS address v), keys in the accumulator's order: half h reads keys 4 h .. + 3, then
  // 8 + 4 h .. of each 16
  __device__ __forceinline__ void values(const bf16x8 (&p)[4], uint32_t v) {
    const int lane = threadIdx.x & 63, g = lane >> 4, j16 = lane & 15, t = 4 * (g >> 1) + (j16 >> 2);
    uint32_t va[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int c = 32 * (b & 1) + 16 * (g & 1) + 4 * (j16 & 3);
      va[b] = v + (uint32_t)((b / 2) * 8192 + t * 128 + (((c >> 3) ^ slab_swz(t)) * 16) + (c & 7) * 2);
    }
    i16x4 f[2][2 * NB];
    auto read = [&](i16x4(&x)[2 * NB], int ks) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        x[2 * b] = lds_read_tr16<0>(va[b] + (uint32_t)(ks * 2048));
        x[2 * b + 1] = lds_read_tr16<1024>(va[b] + (uint32_t)(ks * 2048));
      }
    };
    auto wait = [&](i16x4(&x)[2 * NB], bool more) {
      if constexpr (NB == 4) {
        if (more)
          asm volatile("s_waitcnt lgkmcnt(8)"
                       : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]), "+v"(x[6]), "+v"(x[7]));
        else
          asm volatile("s_waitcnt lgkmcnt(0)"
                       : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]), "+v"(x[6]), "+v"(x[7]));
      } else {
        if (more)
          asm volatile("s_waitcnt lgkmcnt(4)" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));
        else
          asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));
      }
    };
    read(f[0], 0);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      i16x4(&x)[2 * NB] = f[ks & 1];
      if (ks < 3) read(f[(ks + 1) & 1], ks + 1);
      wait(x, ks < 3);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x[2 * b], x[2 * b + 1], 0, 1, 2, 3, 4, 5, 6, 7));
        o[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, p[ks], o[b], 0, 0, 0);
      }
    }
  }
};

// (x of this lane's dims lane, lane + 64, ..) rotated; HD 64 has a pair's halves 32 lanes apart
template <int HD>
__device__ __forceinline__ void rotate_row(const TreeArgs& a, float (&x)[HD / 64], int64_t at) {
  if (a.cos_table == nullptr) return;
  const int e = (threadIdx.x & 63) & (HD / 2 - 1);
  const float c = a.cos_table[at * HD + e], s = a.sin_table[at * HD + e];
  if constexpr (HD == 64) {
    const float y = other_half(x[0]);
    x[0] = (threadIdx.x & 63) < 32 ? x[0] * c - y * s : x[0] * c + y * s;
  } else {
    const float lo = x[0], hi = x[1];
    x[0] = lo * c - hi * s;
    x[1] = hi * c + lo * s;
  }
}

// One row by one wave over the keys that it sees, of tiles [t_begin, t_end) and, with `nodes`, of the new tokens: nothing
// else is touched.  Writes what the tiled kernels write.
template <int HD>
__device__ __forceinline__ void selected_row(const TreeArgs& a, const Place& p, const Tree& tree, const Ring& ring, int64_t pos,
                                             int row, int t_begin, int t_end, bool nodes) {
  constexpr int E = HD / 64;
  const int lane = threadIdx.x & 63, t = row / a.rep;
  const int d = uniform(__shfl(tree.depth, t, 64));
  const uint64_t sees = shfl64(tree.sees, t);
  const int lim = visible_age(a, ring, d);
  const float c2 = a.scale * kLog2e;
  float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    q[i] = to_f32(static_cast<const bf16*>(a.q)[p.n * a.q_n + t * a.q_t + (p.kvh * a.rep + row % a.rep) * a.q_h + lane + 64 * i]);
    o[i] = 0.f;
  }
  rotate_row<HD>(a, q, pos + d);
  auto take = [&](const float(&k)[E], const bf16* v) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) s += q[i] * k[i];
    s = wave_sum(s) * c2;
    const float m_new = fmaxf(m, s), corr = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
    const float x = s == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s - m_new);
    l = l * corr + x;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = o[i] * corr + x * to_f32(v[lane + 64 * i]);
    m = m_new;
  };
  const int64_t base = p.n * a.ring_n + (int64_t)p.kvh * a.slots * HD;
#pragma unroll 1
  for (int tile = t_begin; tile < t_end; ++tile) {
    uint64_t seen = seen_slots(a, ring, tile * 64, lim);
#pragma unroll 1
    while (seen != 0) {
      const int64_t at = base + ((int64_t)tile * 64 + __builtin_ctzll(seen)) * HD;
      seen &= seen - 1;
      float k[E];
#pragma unroll
      for (int i = 0; i < E; ++i) k[i] = to_f32(static_cast<const bf16*>(a.k_ring)[at + lane + 64 * i]);
      take(k, static_cast<const bf16*>(a.v_ring) + at);
    }
  }
  uint64_t seen = nodes ? sees : 0;
#pragma unroll 1
  while (seen != 0) {
    const int j = __builtin_ctzll(seen);
    seen &= seen - 1;
    float k[E];
#pragma unroll
    for (int i = 0; i < E; ++i) k[i] = to_f32(static_cast<const bf16*>(a.k)[p.n * a.k_n + j * a.k_t + p.kvh * a.k_h + lane + 64 * i]);
    rotate_row<HD>(a, k, pos + __shfl(tree.depth, j, 64));
#pragma unroll
    for (int i = 0; i < E; ++i) k[i] = to_f32(from_f32<bf16>(k[i]));
    take(k, static_cast<const bf16*>(a.v) + p.n * a.v_n + j * a.v_t + p.kvh * a.v_h);
  }
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if (a.nsplit == 1)
      out_row<bf16>(a, p, row)[lane + 64 * i] = from_f32<bf16>(o[i] / l);
    else
      a.part_o[part_row(a, p, row) * HD + lane + 64 * i] = o[i];
  }
  if (a.nsplit > 1 && lane == 0) {
    a.part_ml[2 * part_row(a, p, row)] = l == l ? m : NAN;
    a.part_ml[2 * part_row(a, p, row) + 1] = l;
  }
}

// The new tokens' tile (keys rotated; a row tile, then a slab) by all threads, kept for the caller by the first row
// group.  Whether the values hold infinities or NaN comes back through `odd` (LDS, 0 before); ends with a barrier.
template <int HD, int THREADS>
__device__ __forceinline__ void new_tile(const TreeArgs& a, const Place& p, const Tree& tree, int count, int64_t pos,
                                         char* kt, char* vt, int* odd) {
  constexpr int HP = HD / 16;  // pairs of 16-byte pieces of a key
  const bool keep = p.group == 0 && (a.write_ring || a.k_nodes != nullptr);
  const bf16* kn = static_cast<const bf16*>(a.k) + p.n * a.k_n + p.kvh * a.k_h;
  const bf16* vn = static_cast<const bf16*>(a.v) + p.n * a.v_n + p.kvh * a.v_h;
#pragma unroll 1
  for (int idx = threadIdx.x; idx < 64 * HP; idx += THREADS) {
    const int t = idx / HP, pc = idx % HP;
    const int d = __shfl(tree.depth, t, 64);
    bf16x8 lo{}, hi{};
    if (t < count) {
      lo = *reinterpret_cast<const bf16x8*>(kn + t * a.k_t + 8 * pc);
      hi = *reinterpret_cast<const bf16x8*>(kn + t * a.k_t + HD / 2 + 8 * pc);
      if (a.cos_table != nullptr) {
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
  bool bad = false;
#pragma unroll 2
  for (int idx = threadIdx.x; idx < 64 * 2 * HP; idx += THREADS) {
    const int t = idx / (2 * HP), pc = idx % (2 * HP);
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (t < count) {
      x = *reinterpret_cast<const uint4*>(vn + t * a.v_t + 8 * pc);
      bad |= !finite16(x);
      if (keep) *reinterpret_cast<uint4*>(node_row<bf16, HD>(a, p, a.v_nodes, a.v_ring, t, pos) + 8 * pc) = x;
    }
    *reinterpret_cast<uint4*>(vt + (pc >> 3) * 8192 + t * 128 + (((pc & 7) ^ slab_swz(t)) * 16)) = x;
  }
  if (bad) *odd = 1;
  __syncthreads();
}

// What of a tile of slots some node sees (`any`) and all see (`all`); then the values' slab in LDS: rows that no node
// sees are zeroed, and whether rows that only some see hold infinities or NaN comes back.
template <int HD>
__device__ __forceinline__ bool guard_values(char* vt, uint64_t any, uint64_t all) {
  const int lane = threadIdx.x & 63;
  const uint64_t none = ~any, part = any & ~all;
  bool bad = false;
#pragma unroll 4
  for (int i = 0; i < HD / 8; ++i) {  // 8 rows at a time, a 16-byte piece per lane
    const int t = 8 * (i & 7) + (lane >> 3);
    uint4* piece = reinterpret_cast<uint4*>(vt + (i >> 3) * 8192 + t * 128 + (lane & 7) * 16);
    if ((none >> t) & 1)
      *piece = make_uint4(0u, 0u, 0u, 0u);
    else if ((part >> t) & 1)
      bad |= !finite16(*piece);
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  return __any(bad);
}

// The keys of a tile that a unit's rows see, as a mask; -inf for the others' scores.
__device__ __forceinline__ void mask_tile(f32x16 (&s)[2], uint64_t seen) {
  mask_keys(s[0], (uint32_t)seen);
  mask_keys(s[1], (uint32_t)(seen >> 32));
}

// One unit, its keys spread over the workgroup's waves.
template <int HD>
__global__ void __launch_bounds__(kThreads, HD == 64 ? 2 : 1) k_swa_tree_mm(const TreeArgs a) {
  constexpr int NB = HD / 32;
  constexpr int TILE = kTileBytes<HD>, LOADS = TILE / 1024;
  constexpr int RED = HD + 4;  // floats of a query's row when the waves' results meet
  static_assert(kWaves * 32 * RED * 4 <= kWaves * 2 * TILE, "the waves' results fit the tiles' LDS");
  __shared__ __align__(1024) char lds[kWaves * 2 * TILE];  // a K tile and a V slab per wave
  __shared__ float red_ml[kWaves][32][2];
  __shared__ int odd_values;  // values that only some rows see hold infinities or NaN
  const Place p = place_of(a);
  if (!p.valid) return;
  const int w = uniform((int)threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const int count = a.counts != nullptr ? min(max(uniform(a.counts[p.n]), 0), a.nodes) : a.nodes;
  const int row0 = p.group * 32, row1 = min(row0 + 32, count * a.rep);
  if (row0 >= row1) return;
  const bool first = p.split == 0;

  char* kt = lds + w * 2 * TILE;
  char* vt = kt + TILE;
  const uint32_t k_lds = lds_addr(kt), v_lds = k_lds + TILE;
  const int64_t slab = p.n * a.ring_n + (int64_t)p.kvh * a.slots * HD;
  const TileLoad<HD, true> k_load(static_cast<const bf16*>(a.k_ring) + slab, a.slots, lane);
  const TileLoad<HD, false> v_load(static_cast<const bf16*>(a.v_ring) + slab, a.slots, lane);
  auto issue_k = [&](int tile) {
#pragma unroll
    for (int g = 0; g < LOADS; ++g) k_load.issue(k_lds, tile, g);
  };
  auto issue_v = [&](int tile) {
#pragma unroll
    for (int g = 0; g < LOADS; ++g) v_load.issue(v_lds, tile, g);
  };
  // the tile a wave starts with needs no position in the first split: ask for it at once (the last wave
  // starts with the new tokens there)
  const bool early = first && w < kWaves - 1;
  if (early) {
    issue_k(w);
    issue_v(w);
  }
  const int64_t pos = uniform(a.positions[p.n]);
  const Tree tree = read_tree(a, p.n, count, pos, lane);
  if (tree.bad) {
    refuse_rows<bf16, HD>(a, p, row0, row1, kThreads);
    wait_vmcnt<0>();  // no LDS write of this workgroup's loads outlives it
    return;
  }
  if (threadIdx.x == 0) odd_values = 0;
  const Ring ring = read_ring(a, pos);
  const int ntiles = (ring.used + 63) / 64;
  const int t_begin = (int)((int64_t)ntiles * p.split / a.nsplit), t_end = (int)((int64_t)ntiles * (p.split + 1) / a.nsplit);
  // wave w takes places w, w + kWaves, .. of the split's list; the first split's has the new tokens at place
  // kWaves - 1, whether or not its cache reaches that far
  auto tile_at = [&](int i) { return t_begin + (first && i >= kWaves ? i - 1 : i); };
  auto has = [&](int i) { return (first && i == kWaves - 1) || tile_at(i) < t_end; };

  const bool turned = a.cos_table != nullptr;
  Unit<HD> u;
  u.load(a, p, tree, ring, pos, row0 + r, row1);
  __syncthreads();  // odd_values is 0
  if (first) new_tile<HD, kThreads>(a, p, tree, count, pos, lds + (kWaves - 1) * 2 * TILE, lds + (kWaves - 1) * 2 * TILE + TILE,
                                    &odd_values);
  const float c2 = a.scale * kLog2e;
  const int lim_any = visible_age(a, ring, 0), lim_all = visible_age(a, ring, tree.deepest);
  const Edge edge = read_edge(a, ring, lim_all);

  bool loaded = early;  // this wave's next ring tile is on its way
  for (int i = w; has(i); i += kWaves) {
    const bool is_tree = first && i == kWaves - 1;
    const int tile = tile_at(i), s0 = tile * 64;
    const bool more = has(i + kWaves);
    if (!is_tree) {
      if (!loaded) {
        issue_k(tile);
        issue_v(tile);
      }
      wait_vmcnt<LOADS>();  // K has landed, V may still be on its way
    }
    f32x16 s[2];
    u.scores(s, k_lds, turned);
    pin_loads();
    // every K read is back: the next tile's K on its way
    const int next = more ? tile_at(i + kWaves) : 0;
    if (more) issue_k(next);
    const bool clean = !is_tree && clean_tile(a, edge, s0);
    if (!clean) mask_tile(s, is_tree ? u.sees : seen_slots(a, ring, s0, u.lim));
    bf16x8 pw[4];
    u.softmax(s, pw, c2);
    if (!is_tree) {
      if (more)
        wait_vmcnt<LOADS>();
      else
        wait_vmcnt<0>();
      pin_loads();
      if (!clean && guard_values<HD>(vt, seen_slots(a, ring, s0, lim_any), seen_slots(a, ring, s0, lim_all))) odd_values = 1;
    }
    u.values(pw, v_lds);
    pin_loads();
    if (more) issue_v(next);
    loaded = more;
  }
  if (early && !has(w)) wait_vmcnt<0>();  // an early tile that the request does not have

  // ---- the waves' results meet
  float* red = reinterpret_cast<float*>(lds);
  __syncthreads();
  u.l += other_half(u.l);
  if (h == 0) {
    red_ml[w][r][0] = u.m;
    red_ml[w][r][1] = u.l;
  }
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 16; e += 4)
      *reinterpret_cast<f32x4*>(red + (w * 32 + r) * RED + 32 * b + 2 * e + 4 * h) =
          f32x4{u.o[b][e], u.o[b][e + 1], u.o[b][e + 2], u.o[b][e + 3]};
  __syncthreads();
  if (odd_values != 0) {
#pragma unroll 1
    for (int row = row0 + w; row < row1; row += kWaves) selected_row<HD>(a, p, tree, ring, pos, row, t_begin, t_end, first);
    return;
  }
  for (int idx = threadIdx.x; idx < 32 * HD / 4; idx += kThreads) {
    const int qr = idx / (HD / 4), e = idx % (HD / 4) * 4, row = row0 + qr;
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
      bf16 y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = from_f32<bf16>(num[j] * inv);
      *reinterpret_cast<uint2*>(out_row<bf16>(a, p, row) + e) = *reinterpret_cast<const uint2*>(y);
    } else {
      const int64_t at = part_row(a, p, row);
      *reinterpret_cast<f32x4*>(a.part_o + at * HD + e) = num;
      if (e == 0) {
        a.part_ml[2 * at] = den == den ? mm * c2 : NAN;
        a.part_ml[2 * at + 1] = den;
      }
    }
  }
}

// A unit per wave, the workgroup's eight waves sharing each tile in LDS: for so many rows that reading the cache again for
// every 32 of them would cost more than it brings.  The two waves of a SIMD work half a tile apart, a barrier
// per half: while one forms scores the other is at its weights and values, so matrix and vector units are busy
// at once.  (Weights alone against both products, the other cut, leaves the weights' half waiting: 3200 cycles
// a half at head_dim 128.)  K has three slots and V four: a wave asks for tile t + 2 ahead of its scores of tile t
// (every wave has left what those slots held), and the tile it asked for before is home by the end of that half,
// one half before the first wave needs it.  16 trees of 64 nodes, 4096 slots: 67 us (435 TFLOP/s; MFMA busy for a
// quarter of it, the softmax's vector work for as much again) and 8 for the join.
constexpr int kWideWaves = 8;

__device__ __forceinline__ void half_barrier() {
  pin_loads();
  __builtin_amdgcn_s_barrier();
  pin_loads();
}

template <int HD>
__global__ void __launch_bounds__(kWideWaves * 64, 1) k_swa_tree_wide(const TreeArgs a) {
  constexpr int NB = HD / 32, TILE = kTileBytes<HD>, PER = TILE / 1024 / kWideWaves;  // loads of a wave
  __shared__ __align__(1024) char lds[7 * TILE];  // three K tiles, four V slabs
  __shared__ int tree_odd;                        // the new values hold infinities or NaN
  const Place p = place_of(a);
  if (!p.valid) return;
  const int w = uniform((int)threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const int count = a.counts != nullptr ? min(max(uniform(a.counts[p.n]), 0), a.nodes) : a.nodes;
  const int row0 = p.group * 32 * kWideWaves, row1 = min(row0 + 32 * kWideWaves, count * a.rep);
  if (row0 >= row1) return;
  const bool first = p.split == 0, late = w >= kWideWaves / 2;
  const int64_t slab = p.n * a.ring_n + (int64_t)p.kvh * a.slots * HD;
  const TileLoad<HD, true> k_load(static_cast<const bf16*>(a.k_ring) + slab, a.slots, lane);
  const TileLoad<HD, false> v_load(static_cast<const bf16*>(a.v_ring) + slab, a.slots, lane);
  const uint32_t k_lds = lds_addr(lds), v_lds = k_lds + 3 * TILE;
  const int64_t pos = uniform(a.positions[p.n]);
  const Tree tree = read_tree(a, p.n, count, pos, lane);
  if (tree.bad) {
    refuse_rows<bf16, HD>(a, p, row0, row1, kWideWaves * 64);
    return;
  }
  if (threadIdx.x == 0) tree_odd = 0;
  const Ring ring = read_ring(a, pos);
  const int ntiles = (ring.used + 63) / 64;
  const int t_begin = (int)((int64_t)ntiles * p.split / a.nsplit), t_end = (int)((int64_t)ntiles * (p.split + 1) / a.nsplit);
  // the list: the new tokens (the first split's), then the slots' tiles
  const int lead = first ? 1 : 0, listed = lead + t_end - t_begin;
  // this wave's share of place i
  auto issue_k = [&](int i) {
#pragma unroll
    for (int x = 0; x < PER; ++x) k_load.issue(k_lds + (uint32_t)(i % 3 * TILE), t_begin + i - lead, w + kWideWaves * x);
  };
  auto issue_v = [&](int i) {
#pragma unroll
    for (int x = 0; x < PER; ++x) v_load.issue(v_lds + (uint32_t)(i % 4 * TILE), t_begin + i - lead, w + kWideWaves * x);
  };
  if (!first && listed > 0) {
    issue_k(0);
    issue_v(0);
  }
  if (listed > 1) {
    issue_k(1);
    issue_v(1);
  }
  if (first) {
    __syncthreads();  // tree_odd is 0
    new_tile<HD, kWideWaves * 64>(a, p, tree, count, pos, lds, lds + 3 * TILE, &tree_odd);
  }
  Unit<HD> u;
  u.load(a, p, tree, ring, pos, row0 + 32 * w + r, row1);
  const float c2 = a.scale * kLog2e;
  const int lim_any = visible_age(a, ring, 0), lim_all = visible_age(a, ring, tree.deepest);
  const Edge edge = read_edge(a, ring, lim_all);
  const bool turned = a.cos_table != nullptr;
  bool odd = first && tree_odd != 0;
  wait_vmcnt<0>();
  half_barrier();
  if (late) half_barrier();
  for (int t = 0; t < listed; ++t) {
    if (t + 2 < listed) {
      issue_k(t + 2);
      issue_v(t + 2);
    }
    f32x16 s[2];
    u.scores(s, k_lds + (uint32_t)(t % 3 * TILE), turned);
    // formed in this half: the barrier alone would not keep the arithmetic from sinking below it
    asm volatile("" : "+v"(s[0]), "+v"(s[1]));
    if (t + 2 < listed)  // place t + 1 has landed
      wait_vmcnt<2 * PER>();
    else
      wait_vmcnt<0>();
    half_barrier();
    const int s0 = (t_begin + t - lead) * 64;
    const bool clean = t >= lead && clean_tile(a, edge, s0);
    if (!clean) mask_tile(s, t < lead ? u.sees : seen_slots(a, ring, s0, u.lim));
    bf16x8 pw[4];
    u.softmax(s, pw, c2);
    if (t >= lead && !clean)  // every wave writes the same zeros
      odd |= guard_values<HD>(lds + (3 + t % 4) * TILE, seen_slots(a, ring, s0, lim_any), seen_slots(a, ring, s0, lim_all));
    u.values(pw, v_lds + (uint32_t)(t % 4 * TILE));
    half_barrier();
  }
  if (!late) half_barrier();
  if (odd) {
    const int last = min(row0 + 32 * (w + 1), row1);
#pragma unroll 1
    for (int row = row0 + 32 * w; row < last; ++row) selected_row<HD>(a, p, tree, ring, pos, row, t_begin, t_end, first);
    return;
  }
  const int row = row0 + 32 * w + r;
  if (row >= row1) return;
  u.l += other_half(u.l);
  if (a.nsplit == 1) {
    const float inv = 1.0f / u.l;
    bf16* og = out_row<bf16>(a, p, row) + 4 * h;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        bf16 y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = from_f32<bf16>(u.o[b][e + j] * inv);
        *reinterpret_cast<uint2*>(og + 32 * b + 2 * e) = *reinterpret_cast<const uint2*>(y);
      }
  } else {
    const int64_t at = part_row(a, p, row);
    if (h == 0) {
      a.part_ml[2 * at] = u.l == u.l ? u.m * c2 : NAN;
      a.part_ml[2 * at + 1] = u.l;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<f32x4*>(a.part_o + at * HD + 32 * b + 2 * e + 4 * h) =
            f32x4{u.o[b][e], u.o[b][e + 1], u.o[b][e + 2], u.o[b][e + 3]};
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

// the largest of 16 lanes, in all of them, through DPP rotations
__device__ __forceinline__ float row_max(float v) {
  auto turned = [](float x, auto by) __attribute__((always_inline)) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + decltype(by)::value, 0xF, 0xF, false));
  };
  v = fmaxf(v, turned(v, std::integral_constant<int, 8>{}));
  v = fmaxf(v, turned(v, std::integral_constant<int, 4>{}));
  v = fmaxf(v, turned(v, std::integral_constant<int, 2>{}));
  return fmaxf(v, turned(v, std::integral_constant<int, 1>{}));
}

// fp32 operands: the same walk with v_mfma_f32_16x16x4f32 and operands straight from memory into registers, for
// research and parity runs.  A workgroup takes 16 rows; its waves take 16 keys each of a 64-key tile and meet at the
// end.  A lane's float4 along a row serves four k steps (dims 16 j + 4 g + i for lane group g, step i), and
// the weights pass through LDS from the scores' layout (a lane: four queries, one key) to the A operand's
// (one query, four keys).  Few requests are bound by the tiles' latency, so a tile's loads are issued at once and
// without branches, for head_dim 64 (where registers allow it beside two waves of a SIMD) the keys a tile ahead, and
// tiles that every row sees whole skip all masks: one request over 512 slots 34 -> 16 us, 32 over 4096 of head_dim
// 128 227 -> 91 us (5.0 TB/s), 16 trees of 64 nodes over as many 743 -> 440 us (66 TFLOP/s, the 16 rows of a
// workgroup use each key for 16 products only).
template <int HD>
__global__ void __launch_bounds__(kThreads, 2) k_swa_tree_f32(const TreeArgs a) {
  constexpr int NJ = HD / 16, LK = HD + 4, RED = HD + 4;
  constexpr bool AHEAD = HD == 64;
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
    refuse_rows<float, HD>(a, p, row0, row1, kThreads);
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
  // scores' layout: the nodes of this lane's rows 4 g + i, a byte each
  uint32_t of_rows = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) of_rows |= (uint32_t)(min(row0 + 4 * g + i, row1 - 1) / a.rep) << (8 * i);
  const int lim_any = visible_age(a, ring, 0), lim_all = visible_age(a, ring, tree.deepest);
  const float* kn = static_cast<const float*>(a.k) + p.n * a.k_n + p.kvh * a.k_h;
  const float* vn = static_cast<const float*>(a.v) + p.n * a.v_n + p.kvh * a.v_h;
  if (first) {
    const bool keep = p.group == 0 && (a.write_ring || a.k_nodes != nullptr);
    for (int base = 0; base < count * (HD / 2); base += kThreads) {  // scores with rows past the nodes are masked
      const int idx = base + threadIdx.x, t = idx / (HD / 2), e = idx % (HD / 2);  // a wave stays within one or two nodes
      const int d = __shfl(tree.depth, t, 64);
      if (t >= count) continue;
      float lo = kn[t * a.k_t + e], hi = kn[t * a.k_t + HD / 2 + e];
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

  // A tile's keys, dims 16 j + 4 g + i of key c, come a tile ahead, its values, dims 16 j + c of keys 4 g + i, while its
  // scores are formed: every load is made, from a slot that exists, and what no row sees is left out behind it.
  const Edge edge = read_edge(a, ring, lim_all);
  f32x4 k_next[NJ];
  auto fetch_keys = [&](int tile) __attribute__((always_inline)) {
    if (tile < t_begin) return;
    const float* row = kr + (int64_t)min(tile * 64 + 16 * w + c, a.slots - 1) * HD + 4 * g;
#pragma unroll
    for (int j = 0; j < NJ; ++j) k_next[j] = *reinterpret_cast<const f32x4*>(row + 16 * j);
  };
  const int t_first = first ? t_begin - 1 : t_begin;
  if (AHEAD) fetch_keys(t_first);
  for (int tile = t_first; tile < t_end; ++tile) {
    const bool is_tree = tile < t_begin;
    const int s0 = is_tree ? 16 * w : tile * 64 + 16 * w;  // this wave's 16 keys
    if (!AHEAD) fetch_keys(tile);
    f32x4 k[NJ], v[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) k[j] = k_next[j];
    const bool clean = !is_tree && clean_tile(a, edge, tile * 64);
    uint32_t any = 0xffffu, all = 0xffffu;  // which of the keys some row sees, and all
    if (!clean) {
      any = (uint32_t)(is_tree ? bit_range(0, count - s0) : seen_slots(a, ring, s0, lim_any)) & 0xffffu;
      all = is_tree ? 0u : (uint32_t)seen_slots(a, ring, s0, lim_all) & 0xffffu;
    }
    if (any == 0) {
      if (AHEAD && tile + 1 < t_end) fetch_keys(tile + 1);
      continue;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = s0 + 4 * g + i;
      const float* row = is_tree ? vn + min(key, count - 1) * a.v_t : vr + (int64_t)min(key, a.slots - 1) * HD;
#pragma unroll
      for (int j = 0; j < NJ; ++j) v[j][i] = row[16 * j + c];
    }
    if (AHEAD && tile + 1 < t_end) fetch_keys(tile + 1);
    if (is_tree) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) k[j] = *reinterpret_cast<const f32x4*>(kt + (s0 + c) * LK + 16 * j + 4 * g);
    }
    // two sums side by side: half as long a chain, and half as many roundings in a row
    f32x4 s{0.f, 0.f, 0.f, 0.f}, s_odd{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NJ; j += 2)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s = __builtin_amdgcn_mfma_f32_16x16x4f32(q[j][i], k[j][i], s, 0, 0, 0);
        s_odd = __builtin_amdgcn_mfma_f32_16x16x4f32(q[j + 1][i], k[j + 1][i], s_odd, 0, 0, 0);
      }
    s += s_odd;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!clean) {
        const int t = (of_rows >> (8 * i)) & 63;
        const uint64_t seen =
            is_tree ? shfl64(tree.sees, t) >> s0 : seen_slots(a, ring, s0, visible_age(a, ring, __shfl(tree.depth, t, 64)));
        const bool vis = (seen >> c) & 1;
        s[i] = vis ? s[i] : -INFINITY;
      }
      const float m_new = fmaxf(m[i], row_max(s[i]));
      const float m_scaled = m_new * c2;  // its rounding is the row's, the exponents have one of their own
      const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(__builtin_fmaf(m[i], c2, -m_scaled));
      m[i] = m_new;
      const float x = s[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c2, -m_scaled));
      l[i] = l[i] * corr + x;  // this lane's keys; the lanes of a row meet at the end
#pragma unroll
      for (int j = 0; j < NJ; ++j) o[j][i] *= corr;
      ps[w][4 * g + i][c] = x;
    }
    bool odd = false;
    if (!clean) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool ok = (any >> (4 * g + i)) & 1, part = !((all >> (4 * g + i)) & 1);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          v[j][i] = ok ? v[j][i] : 0.f;
          odd |= part && !(fabsf(v[j][i]) < INFINITY);
        }
      }
      odd = __any(odd);
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
      out_row<float>(a, p, row)[e] = num / den;
    } else {
      const int64_t at = part_row(a, p, row);
      a.part_o[at * HD + e] = num;
      if (e == 0) {
        a.part_ml[2 * at] = den == den ? mm * c2 : NAN;
        a.part_ml[2 * at + 1] = den;
      }
    }
  }
}

// Workgroups' shape: units of 32 rows that share a workgroup's tiles (1: k_swa_tree_mm, 8: k_swa_tree_wide; 0: 16 fp32
// rows), workgroups along a (request, kv head)'s rows, splits of its slots.
struct TreePlan {
  int units, groups, nsplit;
};

constexpr int kMaxTreeSplits = 64;

TreePlan plan_tree(int64_t n_req, int64_t n_heads, int64_t n_kv_heads, int64_t nodes, int64_t head_dim, int64_t slots,
                   bool b16) {
  TreePlan p;
  const int64_t rows = n_heads / n_kv_heads * nodes, lists = n_req * n_kv_heads, tiles = (slots + 63) / 64;
  p.units = b16 ? 1 : 0;
  // Many rows of many lists share their tiles (16 trees of 64 nodes over 4096 slots of head_dim 128: 109 us apart, 75 shared;
  // of 40 nodes 99, 67; 8 trees of 64 57, 55; below, units alone: 4 trees of 64 41 apart, 50 shared, 16 of 24 56, 61; a unit of
  // head_dim 64 has half the work for a barrier: 16 of 64 43 apart, 63 shared)
  if (b16 && head_dim == 128 && rows > 128 && lists * ((rows + 31) / 32) >= 256) p.units = kWideWaves;
  const int64_t per = b16 ? 32 * p.units : 16;
  p.groups = (int)((rows + per - 1) / per);
  const int64_t base = lists * p.groups;
  // Splits that fill the card's `want` places for workgroups once, of at least `least` tiles each: a split costs its part of
  // the second launch, and a second round of workgroups as much as the first.  A tile of the slower walks (fp32,
  // head_dim 128) is worth a shorter split.  Measured, us:
  //   want of half / this / twice: 32 decoding requests over 4096 slots of head_dim 128, bf16 49.2 / 47.1 / 50.7; 16 trees
  //     of 64 nodes over as many 97.5 / 76.9 / 92.0
  //   192 workgroups of head_dim 128 left whole / in two (16 trees of 24 nodes): 55 / 69
  //   least of 4 / 8: fp32, one request over 512 slots 16.0 / 20.8, 3 over 761 of head_dim 128 22.2 / 35.4; bf16 of
  //     head_dim 128, 3 over 761 16.8 / 19.9, one tree of 8 nodes over 1024 19.3 / 20.5, one request over 4096 22.4 / 21.1;
  //     bf16 of head_dim 64, one request over 512 12.2 / 11.6, 5 trees of 38 nodes over 697 15.4 / 11.9
  const int64_t want = head_dim == 64 ? 512 : 256, least = b16 && head_dim == 64 ? 8 : 4;
  p.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({want / base, tiles / least, (int64_t)kMaxTreeSplits}));
  return p;
}

template <int HD>
void launch_tree(const TreeArgs& m, const TreePlan& p, bool b16, hipStream_t st) {
  const int64_t lists = (int64_t)m.n_req * m.n_kv_heads * m.nsplit;
  const dim3 grid((unsigned)((lists + kXcds - 1) / kXcds * kXcds * m.groups));
  if (p.units == 0)
    hipLaunchKernelGGL(k_swa_tree_f32<HD>, grid, dim3(kThreads), 0, st, m);
  else if (p.units == 1)
    hipLaunchKernelGGL(k_swa_tree_mm<HD>, grid, dim3(kThreads), 0, st, m);
  else if constexpr (HD == 128)
    hipLaunchKernelGGL(k_swa_tree_wide<HD>, grid, dim3(kWideWaves * 64), 0, st, m);
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
  UTTT_REQUIRE(a->window >= 1 && a->window <= (1LL << 28) && a->sinks >= 0 && a->sinks <= (1LL << 28) &&
                   (a->window + a->sinks) * a->head_dim * 4 < (1LL << 31),
               "window or sinks out of range (a request's keys of one head must stay below 2 GB)");
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
  UTTT_REQUIRE(!a->write_ring || a->n_req == 1 || a->ring_stride_n >= a->n_kv_heads * slots * a->head_dim,
               "the requests' rings must not overlap");
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
