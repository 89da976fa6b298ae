// Attention of new tokens (a decode step's one, or a tree of drafted ones) over ring caches in 4 bits, written for gfx950
// (MI355X).
//
// The rows of a (request, kv head), nodes times query heads, share its keys.  Per block of 32 slots and 16 rows, in registers
// and without LDS:
//   S^T = K q^T        two 16 x 16 tiles: a lane has the scores of one row (its column r) with 8 slots; the codes are the
//                      operand, a group's scale multiplies the group's fp32 products as they are added up
//   P   = 2^(S - m)    one pass with a running maximum that only moves when a score passes it by 2^8
//   O^T = V^T (P s)^T  the values' scales go onto the weights, a group of 32 elements at a time; a lane's 8 weights
//                      are the operand as they are, since the cache keeps its words of 8 slots in that order
// Rows of q are rotated in fp32, scaled, and carried as bf16 parts: two (16 bits) for bf16 activations, three (all 24) for fp32;
// weights are rounded to bf16 for bf16 activations (as attention over 16-bit rings has them: an error of 2.2e-3 against 64 bits
// where the result's own rounding is 1.65e-3; a second part would double the values' products) and carried as three parts for fp32;
// sums are those of the unrounded ones.
// The new tokens themselves are keys in LDS, in their own precision; a single one stays in registers.
//
// 32 requests over 4096 slots, 16 heads on 4 of 128: 21 us and 4 of the join, 2.9 TB/s (fp32 activations 32 us).  What bounds it
// is vector work, half of the SIMD cycles: per block 64 conversions of codes, as many scales unpacked and applied to scores, then to
// weights; a tile has 16 columns of which 4 heads to a kv head fill 4.  One request over 512 slots: 7.4 us of latency.  Trees of
// more than 16 rows walk the cache once per 16 (16 trees of 64 nodes 118 us).
#include <algorithm>
#include <type_traits>

#include "../../include/uttt_decode.h"
#include "fp4.h"
#include "uttt_host.h"

namespace uttt {
namespace {

constexpr int kSlots = 32;
constexpr int kMaxNodes4 = 64;
constexpr int kMaxSplits4 = 64;
constexpr int kJoin = 4;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kSlack = 8.f;  // weights of up to 2^8 before the maximum moves

struct Tree4Args {
  int n_req, n_kv_heads, rep, nodes, rows, groups, nsplit;
  int window, sinks, sink_blocks, ring_blocks;
  float scale;  // times log2 e
  const int64_t* positions;
  const int32_t *parents, *counts;
  const float *cos_table, *sin_table;
  int64_t table_len;
  const void* q;
  int64_t q_n, q_t, q_h;
  const void* k;
  int64_t k_n, k_t, k_h;
  const void* v;
  int64_t v_n, v_t, v_h;
  const char* cache;
  int64_t c_n;
  void* out;
  int64_t o_n, o_t, o_h;
  void *k_nodes, *v_nodes;
  int64_t nodes_n;
  float *part_o, *part_ml;
};

// What a request's tree is, each lane a node: its ancestors and itself that it sees, its depth.
struct Tree {
  int64_t pos;
  int count, depth, deepest;
  uint64_t sees;
  bool bad;
};

__device__ __forceinline__ uint64_t shfl64(uint64_t x, int lane) {
  return (uint64_t)(uint32_t)__shfl((int)(uint32_t)x, lane, 64) | (uint64_t)(uint32_t)__shfl((int)(uint32_t)(x >> 32), lane, 64)
                                                                       << 32;
}

__device__ __forceinline__ Tree read_tree(const Tree4Args& a, int n) {
  Tree t;
  const int lane = threadIdx.x & 63;
  t.pos = a.positions[n];
  t.count = a.counts ? min(max(a.counts[n], 0), a.nodes) : a.nodes;
  t.bad = t.pos < 0;
  uint64_t path = lane < t.count ? 1ull << lane : 0;
  if (a.parents != nullptr) {
    int up = lane < t.count ? a.parents[(int64_t)n * a.nodes + lane] : -1;
    const bool wrong = up < -1 || up >= lane;
    t.bad |= __any(lane < t.count && wrong);
    up = wrong || lane >= t.count ? -1 : up;
    for (int reach = 1; reach < t.count; reach *= 2) {  // twice as far up with every round
      const int from = max(up, 0);
      const uint64_t more = shfl64(path, from);
      const int next = __shfl(up, from, 64);
      path |= up >= 0 ? more : 0;
      up = up >= 0 ? next : -1;
    }
  } else if (lane < t.count) {
    path = ~0ull >> (63 - lane);
  }
  t.depth = max(__popcll(path) - 1, 0);
  int deepest = lane < t.count ? t.depth : 0;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) deepest = max(deepest, __shfl_xor(deepest, off, 64));
  t.deepest = deepest;
  if (a.cos_table != nullptr && t.count > 0) t.bad |= t.pos >= a.table_len - deepest;
  if (deepest >= a.window) {  // ancestors may be out of the window
    for (int j = 0; j < t.count; ++j) {
      const int dj = __shfl(t.depth, j, 64);
      if (t.depth - dj >= a.window && t.pos >= a.sinks - dj) path &= ~(1ull << j);
    }
  }
  t.sees = path;
  return t;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    const bf16x8 t = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32(t[j]);
  } else {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = a[j];
      v[4 + j] = b[j];
    }
  }
}

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

// KT: new tokens that fit, 1 (which needs no LDS), 32 or 64; W: waves.  A tree of 24 nodes over 1024 slots of 128 takes 18.5 us with
// room for 32 and 19.3 for 64, shorter heads the same.
template <typename T, int HD, int KT, int W>
struct Smem4 {
  static constexpr int kParts = sizeof(T) == 2 ? 1 : 3;
  static constexpr int kKeys = KT == 1 ? 0 : kParts * KT * (HD + 8) * 2;    // [part][node][HD + 8]
  static constexpr int kValues = KT == 1 ? 0 : kParts * HD * (KT + 8) * 2;  // [part][HD][KT + 8]
  static constexpr int kMeet = W * 16 * (HD + 4) * 4;    // [wave][row][HD + 4]
  static constexpr int kBytes = kKeys + kValues > kMeet ? kKeys + kValues : kMeet;
};

template <typename T, int HD, int KT, int W>
__global__ void __launch_bounds__(W * 64, W == 4 ? 2 : 1) k_swa_tree4(const Tree4Args a) {
  constexpr int G = HD / 32, D = HD / 16;
  constexpr int QP = sizeof(T) == 2 ? 2 : 3, PP = sizeof(T) == 2 ? 1 : 3, KP = PP;
  using S = Smem4<T, HD, KT, W>;
  __shared__ __align__(16) char smem[S::kBytes];
  __shared__ float ml[W][16][2];
  __shared__ int odd, odd_keys;  // new values, new keys that are not finite
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, h = lane >> 4;
  int id = blockIdx.x;
  const int group = id % a.groups;
  id /= a.groups;
  const int split = id % a.nsplit;
  id /= a.nsplit;
  const int kvh = id % a.n_kv_heads, n = id / a.n_kv_heads;
  const int row0 = group * 16;
  // a lane's row of q: elements 32 g + 8 h .. (of one node per request on its way before anything else is known)
  float x[G][8];
  auto load_q = [&](int node, int head) {
    const T* qp = static_cast<const T*>(a.q) + n * a.q_n + node * a.q_t + head * a.q_h + 8 * h;
#pragma unroll
    for (int g = 0; g < G; ++g) load8(qp + 32 * g, x[g]);
  };
  if (KT == 1) load_q(0, kvh * a.rep + min(row0 + r, a.rep - 1));
  const Tree tree = read_tree(a, n);
  const int live = tree.count * a.rep;  // rows of nodes that exist, a node's heads together
  if (row0 >= live) return;
  const int row = min(row0 + r, live - 1), node = row / a.rep, head = kvh * a.rep + row % a.rep;
  T* out = static_cast<T*>(a.out);
  const int n_heads = a.n_kv_heads * a.rep;
  if (tree.bad) {
    for (int i = threadIdx.x; i < 16 * HD; i += W * 64) {
      const int ri = row0 + i / HD, e = i % HD;
      if (ri >= live) break;
      const int nd = ri / a.rep, hd = kvh * a.rep + ri % a.rep;
      if (a.nsplit == 1) {
        out[n * a.o_n + nd * a.o_t + hd * a.o_h + e] = from_f32<T>(NAN);
      } else {
        const int64_t at = (((int64_t)split * a.n_req + n) * n_heads + hd) * a.nodes + nd;
        a.part_o[at * HD + e] = 0.f;
        if (e == 0) {
          a.part_ml[2 * at] = 0.f;
          a.part_ml[2 * at + 1] = NAN;
        }
      }
    }
    return;
  }
  const int depth = __shfl(tree.depth, node, 64);
  const uint64_t sees = shfl64(tree.sees, node);

  // the cached tokens: blocks of sinks, then of the ring, a wave every fourth of this split's
  const int sink_held = (int)min(tree.pos, (int64_t)a.sinks);
  const int ring_held = (int)min(max(tree.pos - a.sinks, (int64_t)0), (int64_t)a.window);
  // the slot that the next token takes (a 64-bit remainder costs hundreds of instructions)
  const int64_t past = max(tree.pos - a.sinks, (int64_t)0);
  const int newest = past >> 32 ? (int)(past % a.window) : (int)((uint32_t)past % (uint32_t)a.window);
  const int sink_n = (sink_held + kSlots - 1) / kSlots, total = sink_n + (ring_held + kSlots - 1) / kSlots;
  const int begin = (int)((int64_t)total * split / a.nsplit), end = (int)((int64_t)total * (split + 1) / a.nsplit);
  const char* cache = a.cache + n * a.c_n + (int64_t)kvh * (a.sink_blocks + a.ring_blocks) * (36 * HD);
  struct Block {
    u32x4 kc[HD / 64], vc[HD / 64], ks[G], vs[G];
  };
  auto fetch = [&](int b) {
    Block x;
    const char* at = cache + (int64_t)(b < sink_n ? b : a.sink_blocks + b - sink_n) * (36 * HD);
#pragma unroll
    for (int q = 0; q < HD / 64; ++q) x.kc[q] = *reinterpret_cast<const u32x4*>(at + 1024 * q + 16 * lane);
#pragma unroll
    for (int g = 0; g < G; ++g) x.ks[g] = *reinterpret_cast<const u32x4*>(at + 32 * HD + 64 * g + 16 * h);
#pragma unroll
    for (int q = 0; q < HD / 64; ++q) x.vc[q] = *reinterpret_cast<const u32x4*>(at + 16 * HD + 1024 * q + 16 * lane);
#pragma unroll
    for (int g = 0; g < G; ++g) x.vs[g] = *reinterpret_cast<const u32x4*>(at + 34 * HD + 64 * g + 16 * h);
    return x;
  };
  const int age_limit = min(ring_held, a.window - 1 - depth);  // tokens of the ring that this row sees, from the newest on
  const int age_clean = min(ring_held, a.window - 1 - tree.deepest);
  constexpr bool kAhead = sizeof(T) == 2 || HD == 64;  // three parts of 128 elements leave no registers to load ahead
  Block next{};
  if (kAhead && begin + w < end) next = fetch(begin + w);

  f32x4 o[D];
#pragma unroll
  for (int d = 0; d < D; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  // the row rotated, scaled, in parts
  bf16x8 qf[G][QP];
  {
    if (KT > 1) load_q(node, head);
    const int64_t at = (tree.pos + depth) * HD + 8 * h;
    const bool single = KT == 1 && split == 0 && w == 0;  // this wave takes the one new token
    const int64_t k_at = n * a.k_n + kvh * a.k_h + 8 * h;
    float k[G][8];
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (single) load8(static_cast<const T*>(a.k) + k_at + 32 * g, k[g]);
#pragma unroll
    for (int g = 0; g < G / 2; ++g) {
      if (a.cos_table == nullptr) break;
      float c0[8], s0[8], c1[8], s1[8];
      load8(a.cos_table + at + 32 * g, c0);
      load8(a.sin_table + at + 32 * g, s0);
      load8(a.cos_table + at + 32 * (g + G / 2), c1);
      load8(a.sin_table + at + 32 * (g + G / 2), s1);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float lo = x[g][j], hi = x[g + G / 2][j];
        x[g][j] = fmaf(lo, c0[j], -(hi * s0[j]));
        x[g + G / 2][j] = fmaf(hi, c1[j], lo * s1[j]);
        if (single) {
          const float k0 = k[g][j], k1 = k[g + G / 2][j];
          k[g][j] = fmaf(k0, c0[j], -(k1 * s0[j]));
          k[g + G / 2][j] = fmaf(k1, c1[j], k0 * s1[j]);
        }
      }
    }
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[g][j] *= a.scale;
        bf16 p[QP];
        bf16_parts(x[g][j], p);
#pragma unroll
        for (int i = 0; i < QP; ++i) qf[g][i][j] = p[i];
      }
    if (single) {  // the one new token is seen by every row: the softmax starts with it
      float s = 0.f;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf(x[g][j], to_f32(from_f32<T>(k[g][j])), s);
      s += __shfl_xor(s, 16, 64);
      s += __shfl_xor(s, 32, 64);
      m = s;
      l = h == 0 ? (fabsf(s) < INFINITY ? 1.f : s == -INFINITY ? 0.f : NAN) : 0.f;  // at -inf its value goes with the first rescale
      const T* vp = static_cast<const T*>(a.v) + n * a.v_n + kvh * a.v_h;
#pragma unroll
      for (int d = 0; d < D; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][i] = to_f32(vp[16 * d + 4 * h + i]);
      if (a.k_nodes != nullptr && group == 0 && r == 0) {
        const int64_t to = n * a.nodes_n + (int64_t)kvh * HD + 8 * h;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float v[8];
          load8(vp + 32 * g + 8 * h, v);
          store8(static_cast<T*>(a.k_nodes) + to + 32 * g, k[g]);
          store8(static_cast<T*>(a.v_nodes) + to + 32 * g, v);
        }
      }
    }
  }

  // the new tokens' keys, rotated and rounded, and values into LDS (and out, for the caches)
  bf16* keys = reinterpret_cast<bf16*>(smem);
  bf16* vals = reinterpret_cast<bf16*>(smem + S::kKeys);
  if (threadIdx.x == 0) odd = odd_keys = 0;
  if (KT > 1 && split == 0) {
    __syncthreads();
    bool strange = false, strange_keys = false;
    for (int i = threadIdx.x; i < KT * (HD / 16); i += W * 64) {
      const int nd = i / (HD / 16), e = i % (HD / 16) * 8;  // elements e .. and HD / 2 + e ..
      float k0[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, k1[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      float v0[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, v1[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      const int dn = __shfl(tree.depth, nd & 63, 64);
      if (nd < tree.count) {
        const T* kp = static_cast<const T*>(a.k) + n * a.k_n + nd * a.k_t + kvh * a.k_h + e;
        const T* vp = static_cast<const T*>(a.v) + n * a.v_n + nd * a.v_t + kvh * a.v_h + e;
        load8(kp, k0);
        load8(kp + HD / 2, k1);
        load8(vp, v0);
        load8(vp + HD / 2, v1);
        if (a.cos_table != nullptr) {
          const int64_t at = (tree.pos + dn) * HD + e;
          float c0[8], s0[8], c1[8], s1[8];
          load8(a.cos_table + at, c0);
          load8(a.sin_table + at, s0);
          load8(a.cos_table + at + HD / 2, c1);
          load8(a.sin_table + at + HD / 2, s1);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float lo = k0[j], hi = k1[j];
            k0[j] = fmaf(lo, c0[j], -(hi * s0[j]));
            k1[j] = fmaf(hi, c1[j], lo * s1[j]);
          }
        }
        if (a.k_nodes != nullptr && group == 0) {
          const int64_t to = n * a.nodes_n + ((int64_t)nd * a.n_kv_heads + kvh) * HD + e;
          store8(static_cast<T*>(a.k_nodes) + to, k0);
          store8(static_cast<T*>(a.k_nodes) + to + HD / 2, k1);
          store8(static_cast<T*>(a.v_nodes) + to, v0);
          store8(static_cast<T*>(a.v_nodes) + to + HD / 2, v1);
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        bf16 p[KP];
        bf16_parts(k0[j], p);
        strange_keys |= !(fabsf(to_f32(p[0])) < INFINITY);
#pragma unroll
        for (int i = 0; i < KP; ++i) keys[(i * KT + nd) * (HD + 8) + e + j] = p[i];
        bf16_parts(k1[j], p);
        strange_keys |= !(fabsf(to_f32(p[0])) < INFINITY);
#pragma unroll
        for (int i = 0; i < KP; ++i) keys[(i * KT + nd) * (HD + 8) + HD / 2 + e + j] = p[i];
        // what is not finite is left out of the products and added to the rows that see it
        const bool fine0 = fabsf(v0[j]) < INFINITY, fine1 = fabsf(v1[j]) < INFINITY;
        strange |= !fine0 || !fine1;
        bf16_parts(fine0 ? v0[j] : 0.f, p);
#pragma unroll
        for (int i = 0; i < KP; ++i) vals[(i * HD + e + j) * (KT + 8) + nd] = p[i];
        bf16_parts(fine1 ? v1[j] : 0.f, p);
#pragma unroll
        for (int i = 0; i < KP; ++i) vals[(i * HD + HD / 2 + e + j) * (KT + 8) + nd] = p[i];
      }
    }
    if (strange) odd = 1;
    if (strange_keys) odd_keys = 1;
  }

  // the softmax's step: scores (masked: -inf) of 8 keys to weights, the sums so far rescaled where the maximum moves
  auto weigh = [&](float (&s)[8], auto clean) {
    float mx = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    if (__any(mx > m + kSlack)) {
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float to = fmaxf(m, mx), f = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - to);
      m = to;
      l *= f;
#pragma unroll
      for (int d = 0; d < D; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][i] *= f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float e = __builtin_amdgcn_exp2f(s[j] - m);
      s[j] = !decltype(clean)::value && s[j] == -INFINITY ? 0.f : e;
      l += s[j];
    }
  };

  // One block: every slot seen by every row (CLEAN), or each by itself.
  auto attend = [&](const Block& x, auto clean, int first, bool sink) {
    constexpr bool CLEAN = decltype(clean)::value;
    float s[8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * t + i] = 0.f;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const bf16x8 k = fp4_values(x.kc[(t * G + g) >> 2][(t * G + g) & 3]);
        f32x4 y{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < QP; ++i) y = mfma16(k, qf[g][i], y);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * t + i] = fmaf(bf16_of(x.ks[g][2 * t + (i >> 1)], i & 1), y[i], s[4 * t + i]);
      }
    }
    if constexpr (!CLEAN) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int slot = first + 16 * (j >> 2) + 4 * h + (j & 3);
        const int age = slot < newest ? newest - 1 - slot : newest - 1 - slot + a.window;
        const bool seen = sink ? slot < sink_held : slot < a.window && age < age_limit;
        s[j] = seen ? s[j] : -INFINITY;
      }
    }
    weigh(s, clean);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      bf16x8 p[PP];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float z = s[j] * bf16_of(x.vs[g][j >> 1], j & 1);
        if constexpr (!CLEAN) z = s[j] == 0.f ? 0.f : z;  // scales of slots that are not seen may be anything
        bf16 part[PP];
        bf16_parts(z, part);
#pragma unroll
        for (int i = 0; i < PP; ++i) p[i][j] = part[i];
      }
#pragma unroll
      for (int d = 2 * g; d < 2 * g + 2; ++d) {
        const bf16x8 v = fp4_values(x.vc[d >> 2][d & 3]);
#pragma unroll
        for (int i = 0; i < PP; ++i) o[d] = mfma16(v, p[i], o[d]);
      }
    }
  };
  for (int b = begin + w; b < end; b += W) {
    const Block now = kAhead ? next : fetch(b);
    if (kAhead && b + W < end) next = fetch(b + W);
    const bool sink = b < sink_n;
    const int first = (sink ? b : b - sink_n) * kSlots;  // the block's first slot in its region
    // ages fall from the block's first slot on, unless the newest slot lies inside
    const int oldest = first < newest ? newest - 1 - first : newest - 1 - first + a.window;
    if (sink ? first + kSlots <= sink_held
             : first + kSlots <= a.window && !(first < newest && newest < first + kSlots) && oldest < age_clean)
      attend(now, std::true_type{}, first, sink);
    else
      attend(now, std::false_type{}, first, sink);
  }

  if (KT > 1 && split == 0) {
    __syncthreads();
    const int b = w;  // of the new tokens' blocks
    if (b * kSlots < min(KT, tree.count)) {
      float s[8];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x4 y{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int i = 0; i < KP; ++i) {
            const bf16x8 k = *reinterpret_cast<const bf16x8*>(keys + (i * KT + b * kSlots + 16 * t + r) * (HD + 8) + 32 * g + 8 * h);
#pragma unroll
            for (int x = 0; x < QP; ++x)
              if (KP == 1 || i + x < QP) y = mfma16(k, qf[g][x], y);  // products below 2^-24 of the whole are left out
          }
        if (odd_keys) {  // an infinite key times a part of q that is 0 is NaN: the first part, 0 only where q is, has the score
          f32x4 z{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int g = 0; g < G; ++g)
            z = mfma16(*reinterpret_cast<const bf16x8*>(keys + (b * kSlots + 16 * t + r) * (HD + 8) + 32 * g + 8 * h), qf[g][0], z);
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = fabsf(z[i]) < INFINITY ? y[i] : z[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = b * kSlots + 16 * t + 4 * h + i;
          s[4 * t + i] = (sees >> key) & 1 ? y[i] : -INFINITY;
        }
      }
      weigh(s, std::false_type{});
      bf16x8 p[PP];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        bf16 part[PP];
        bf16_parts(s[j], part);
#pragma unroll
        for (int i = 0; i < PP; ++i) p[i][j] = part[i];
      }
#pragma unroll
      for (int d = 0; d < D; ++d)
#pragma unroll
        for (int x = 0; x < KP; ++x) {
          const bf16* vp = vals + (x * HD + 16 * d + r) * (KT + 8) + b * kSlots + 4 * h;
          const bf16x4 lo = *reinterpret_cast<const bf16x4*>(vp), hi = *reinterpret_cast<const bf16x4*>(vp + 16);
          const bf16x8 v{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
          for (int i = 0; i < PP; ++i)
            if (i + x < PP) o[d] = mfma16(v, p[i], o[d]);
        }
      if (odd) {  // infinities and NaN among the values, a key at a time, where its weight is not 0
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll 1
          for (int hh = 0; hh < 4; ++hh) {
            const float x = __shfl(s[j], 16 * hh + r, 64);
            const int key = b * kSlots + 16 * (j >> 2) + 4 * hh + (j & 3);
            if (key >= tree.count) continue;
            const T* vp = static_cast<const T*>(a.v) + n * a.v_n + key * a.v_t + kvh * a.v_h + 4 * h;
#pragma unroll
            for (int d = 0; d < D; ++d)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float v = to_f32(vp[16 * d + i]);
                o[d][i] = x != 0.f && !(fabsf(v) < INFINITY) ? fmaf(x, v, o[d][i]) : o[d][i];
              }
          }
      }
    }
  }

  // the waves meet
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  __syncthreads();
  float* meet = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int d = 0; d < D; ++d) *reinterpret_cast<f32x4*>(meet + (w * 16 + r) * (HD + 4) + 16 * d + 4 * h) = o[d];
  if (h == 0) {
    ml[w][r][0] = m;
    ml[w][r][1] = l;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * HD; i += W * 64) {
    const int rr = i / HD, e = i % HD, ri = row0 + rr;
    if (ri >= live) break;
    float top = -INFINITY, den = 0.f, num = 0.f;
#pragma unroll
    for (int x = 0; x < W; ++x) top = fmaxf(top, ml[x][rr][0]);
#pragma unroll
    for (int x = 0; x < W; ++x) {
      const float f = ml[x][rr][0] == -INFINITY ? (ml[x][rr][1] == 0.f ? 0.f : NAN) : __builtin_amdgcn_exp2f(ml[x][rr][0] - top);
      den = fmaf(f, ml[x][rr][1], den);
      num = f == 0.f ? num : fmaf(f, meet[(x * 16 + rr) * (HD + 4) + e], num);
    }
    const int nd = ri / a.rep, hd = kvh * a.rep + ri % a.rep;
    if (a.nsplit == 1) {
      out[n * a.o_n + nd * a.o_t + hd * a.o_h + e] = from_f32<T>(num / den);
    } else {
      const int64_t at = (((int64_t)split * a.n_req + n) * n_heads + hd) * a.nodes + nd;
      a.part_o[at * HD + e] = num;
      if (e == 0) {
        a.part_ml[2 * at] = top;
        a.part_ml[2 * at + 1] = den;
      }
    }
  }
}

// The splits' sums of a row meet: four elements per thread.  4 us of latency.
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads) k_swa_tree4_join(const Tree4Args a) {
  const int n_heads = a.n_kv_heads * a.rep;
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x, rows = (int64_t)a.n_req * n_heads * a.nodes;
  const int64_t row = at / (HD / 4);
  const int e = (int)(at % (HD / 4)) * 4;
  if (row >= rows) return;
  const int node = (int)(row % a.nodes), head = (int)(row / a.nodes % n_heads), n = (int)(row / a.nodes / n_heads);
  if (a.counts != nullptr && node >= a.counts[n]) return;
  float top = -INFINITY, den = 0.f;
  f32x4 num{0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < a.nsplit; s0 += kJoin) {  // the loads of kJoin splits at once
    float2 ml[kJoin];
    f32x4 o[kJoin];
#pragma unroll
    for (int u = 0; u < kJoin; ++u) {
      const int64_t part = min(s0 + u, a.nsplit - 1) * rows + row;
      ml[u] = *reinterpret_cast<const float2*>(a.part_ml + 2 * part);
      o[u] = *reinterpret_cast<const f32x4*>(a.part_o + part * HD + e);
    }
    float next = top;
#pragma unroll
    for (int u = 0; u < kJoin; ++u) next = s0 + u < a.nsplit ? fmaxf(next, ml[u].x) : next;
    const float back = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - next);
    top = next;
    den = den == 0.f ? 0.f : den * back;
#pragma unroll
    for (int i = 0; i < 4; ++i) num[i] = back == 0.f ? 0.f : num[i] * back;
#pragma unroll
    for (int u = 0; u < kJoin; ++u) {
      if (s0 + u >= a.nsplit) break;
      const float f = ml[u].x == -INFINITY ? (ml[u].y == 0.f ? 0.f : NAN) : __builtin_amdgcn_exp2f(ml[u].x - top);
      den = fmaf(f, ml[u].y, den);
#pragma unroll
      for (int i = 0; i < 4; ++i) num[i] = f == 0.f ? num[i] : fmaf(f, o[u][i], num[i]);
    }
  }
  T* out = static_cast<T*>(a.out) + n * a.o_n + node * a.o_t + head * a.o_h + e;
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = from_f32<T>(num[i] / den);
}

struct Plan4 {
  int groups, nsplit, waves;
};

// Workgroups to 256, of at least 20 blocks, of eight waves where they fit that number.  Measured, us: one token of 32
// requests over 4096 slots of 128 for 16 heads on 4: to 256 workgroups 25.2, to 512 27.0, to 1024 34.4; 8 such 17.5, 17.6,
// 17.0; one 15.2, 15.4, 14.6; 32 over 1024 slots of 64, 12 and 20 blocks at least: 11.3, 9.8.  Waves, four and eight to a
// workgroup: 256 workgroups (32 over 4096) 28.0 and 25.2, (64 over 1024 of 128) 17.5 and 16.0, 4 (one over 512) 7.8 and
// 7.4; 384 (96 over 1024) 22.8 and 27.6, 1024 (trees of 64 nodes) 118 and 141.
Plan4 plan_tree4(int64_t n_req, int64_t n_heads, int64_t n_kv_heads, int64_t nodes, int64_t blocks) {
  Plan4 p;
  p.groups = (int)((n_heads / n_kv_heads * nodes + 15) / 16);
  const int64_t base = n_req * n_kv_heads * p.groups;
  p.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({256 / base, blocks / 20, (int64_t)kMaxSplits4}));
  p.waves = base * p.nsplit <= 256 ? 8 : 4;
  return p;
}

int64_t blocks_of(int64_t window, int64_t sinks) { return (window + kSlots - 1) / kSlots + (sinks + kSlots - 1) / kSlots; }

template <typename T, int HD, int KT>
void launch_tree4(const Tree4Args& m, int waves, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)m.n_req * m.n_kv_heads * m.nsplit * m.groups));
  if (waves == 4)
    hipLaunchKernelGGL((k_swa_tree4<T, HD, KT, 4>), grid, dim3(256), 0, st, m);
  else
    hipLaunchKernelGGL((k_swa_tree4<T, HD, KT, 8>), grid, dim3(512), 0, st, m);
}

template <typename T, int HD>
void launch_tree4(const Tree4Args& m, int waves, hipStream_t st) {
  if (m.nodes == 1)
    launch_tree4<T, HD, 1>(m, waves, st);
  else if (m.nodes <= 32)
    launch_tree4<T, HD, 32>(m, waves, st);
  else
    launch_tree4<T, HD, 64>(m, waves, st);
  if (m.nsplit > 1) {
    const int64_t n = (int64_t)m.n_req * m.n_kv_heads * m.rows * (HD / 4);
    hipLaunchKernelGGL((k_swa_tree4_join<T, HD>), dim3((unsigned)((n + kThreads - 1) / kThreads)), dim3(kThreads), 0, st, m);
  }
}

}  // namespace
}  // namespace uttt

using namespace uttt;

extern "C" size_t uttt_swa_tree4_workspace(int64_t n_req, int64_t n_heads, int64_t n_kv_heads, int64_t nodes,
                                           int64_t head_dim, int64_t window, int64_t sinks) {
  if (n_req < 1 || n_kv_heads < 1 || n_heads < n_kv_heads || nodes < 1 || head_dim < 1 || window < 1 || sinks < 0) return 0;
  const Plan4 p = plan_tree4(n_req, n_heads, n_kv_heads, nodes, blocks_of(window, sinks));
  if (p.nsplit == 1) return 16;
  return sizeof(float) * (size_t)p.nsplit * (size_t)n_req * (size_t)n_heads * (size_t)nodes * (size_t)(head_dim + 2);
}

extern "C" int uttt_swa_tree4(const uttt_swa_tree4_args* a, uttt_stream_t stream) {
  UTTT_REQUIRE(a != nullptr, "args is NULL");
  UTTT_REQUIRE(a->head_dim == 64 || a->head_dim == 128, "head_dim must be 64 or 128 (got %lld)", (long long)a->head_dim);
  UTTT_REQUIRE(a->n_req >= 1 && a->n_req <= (1LL << 20) && a->n_kv_heads >= 1 && a->n_kv_heads <= 65535 &&
                   a->n_heads >= 1 && a->n_heads <= 65535 && a->n_heads % a->n_kv_heads == 0,
               "bad request / head counts");
  UTTT_REQUIRE(a->nodes >= 1 && a->nodes <= kMaxNodes4, "nodes must be in [1, %d]", kMaxNodes4);
  UTTT_REQUIRE(a->window >= 1 && a->window <= (1LL << 28) && a->sinks >= 0 && a->sinks <= (1LL << 28),
               "window must be in [1, 2^28] and sinks in [0, 2^28]");
  UTTT_REQUIRE(a->act_dtype == UTTT_DTYPE_F32 || a->act_dtype == UTTT_DTYPE_BF16, "bad act_dtype");
  UTTT_REQUIRE(a->scale > 0.f && a->scale < INFINITY, "scale must be > 0");
  UTTT_REQUIRE(a->positions && a->q && a->k_new && a->v_new && a->cache && a->out, "pointers must be non-NULL");
  UTTT_REQUIRE((a->k_nodes == nullptr) == (a->v_nodes == nullptr), "node buffers come in pairs");
  UTTT_REQUIRE((a->cos_table == nullptr) == (a->sin_table == nullptr), "cos/sin tables must both be given or both NULL");
  const int64_t vec = a->act_dtype == UTTT_DTYPE_BF16 ? 8 : 4;
  auto whole = [vec](int64_t x, int64_t y, int64_t z) { return x % vec == 0 && y % vec == 0 && z % vec == 0; };
  UTTT_REQUIRE(aligned16(a->q) && aligned16(a->k_new) && aligned16(a->v_new) && aligned16(a->cache) && aligned16(a->k_nodes) &&
                   aligned16(a->v_nodes) && aligned16(a->cos_table) && aligned16(a->sin_table) &&
                   whole(a->q_stride_n, a->q_stride_t, a->q_stride_h) && whole(a->k_stride_n, a->k_stride_t, a->k_stride_h) &&
                   whole(a->v_stride_n, a->v_stride_t, a->v_stride_h) && a->nodes_stride_n % vec == 0 && a->cache_stride_n % 16 == 0,
               "operands must be 16-byte aligned with strides of whole 16-byte pieces");
  const Plan4 p = plan_tree4(a->n_req, a->n_heads, a->n_kv_heads, a->nodes, blocks_of(a->window, a->sinks));
  UTTT_REQUIRE(a->n_req * a->n_kv_heads * p.nsplit * p.groups <= 0x7fffffffLL &&
                   a->n_req * a->n_heads * a->nodes * (a->head_dim / 4) / kThreads < 0x7fffffffLL,
               "too many requests for one launch");
  UTTT_REQUIRE(p.nsplit == 1 || (a->workspace != nullptr && aligned16(a->workspace) &&
                                 a->workspace_bytes >= uttt_swa_tree4_workspace(a->n_req, a->n_heads, a->n_kv_heads, a->nodes,
                                                                                a->head_dim, a->window, a->sinks)),
               "tree attention workspace too small");
  Tree4Args m{};
  m.n_req = (int)a->n_req; m.n_kv_heads = (int)a->n_kv_heads; m.rep = (int)(a->n_heads / a->n_kv_heads);
  m.nodes = (int)a->nodes; m.rows = m.rep * m.nodes;
  m.groups = p.groups; m.nsplit = p.nsplit;
  m.window = (int)a->window; m.sinks = (int)a->sinks;
  m.sink_blocks = (int)((a->sinks + kSlots - 1) / kSlots); m.ring_blocks = (int)((a->window + kSlots - 1) / kSlots);
  m.scale = a->scale * kLog2e;
  m.positions = a->positions; m.parents = a->parents; m.counts = a->counts;
  m.cos_table = a->cos_table; m.sin_table = a->sin_table; m.table_len = a->table_len;
  m.q = a->q; m.q_n = a->q_stride_n; m.q_t = a->q_stride_t; m.q_h = a->q_stride_h;
  m.k = a->k_new; m.k_n = a->k_stride_n; m.k_t = a->k_stride_t; m.k_h = a->k_stride_h;
  m.v = a->v_new; m.v_n = a->v_stride_n; m.v_t = a->v_stride_t; m.v_h = a->v_stride_h;
  m.cache = static_cast<const char*>(a->cache); m.c_n = a->cache_stride_n;
  m.out = a->out; m.o_n = a->o_stride_n; m.o_t = a->o_stride_t; m.o_h = a->o_stride_h;
  m.k_nodes = a->k_nodes; m.v_nodes = a->v_nodes; m.nodes_n = a->nodes_stride_n;
  if (p.nsplit > 1) {
    m.part_o = static_cast<float*>(a->workspace);
    m.part_ml = m.part_o + (int64_t)p.nsplit * a->n_req * a->n_heads * a->nodes * a->head_dim;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool b16 = a->act_dtype == UTTT_DTYPE_BF16;
  if (a->head_dim == 64)
    b16 ? launch_tree4<bf16, 64>(m, p.waves, st) : launch_tree4<float, 64>(m, p.waves, st);
  else
    b16 ? launch_tree4<bf16, 128>(m, p.waves, st) : launch_tree4<float, 128>(m, p.waves, st);
  return launch_status("uttt_swa_tree4");
}
