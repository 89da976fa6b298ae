// Products with weights in 4 bits for the rows of a decode step, written for gfx950 (MI355X): y = x W^T with one matrix
// for all rows (slow projections, LM head) or one per request (the frozen fast-weight readout).
//
// Per group of 32 columns a 16 x 32 piece of W is one MFMA operand, converted from its codes (fp4.h); the group's scale, one
// per row of W, multiplies the fp32 products as they are added up:  y[m][n] = sum_g s[n][g] (x[m][g] . c[n][g]).  x is the
// other operand as it is (bf16), or in bf16 parts that add up to it: three for fp32, two where bf16 activations were multiplied
// by a norm's weight or are the hidden values of a readout (16 bits, where the model's own path has 8).
//
// One row (k_gemv4): the row lies in LDS, its parts are rows of one operand, and a wave streams a block of 16 rows of W, or its
// part of the columns.  More rows (k_prod4): a wave takes NT blocks of 16 rows of W for 16 MT rows of x, whose
// operands come from memory (L2) and serve all NT; parts are made beforehand (k_parts4).
#include <algorithm>

#include "../../include/uttt_decode.h"
#include "fp4.h"
#include "uttt_host.h"

namespace uttt {
namespace {

constexpr int kBlockBytes = 1152;  // 16 x 128 of W
constexpr int kMaxWaves4 = 8;
constexpr int kCounterPitch = 64;  // a row's counter has a cache line of its own
constexpr int kRowLds = 49152;  // bytes of a row's parts that k_gemv4 takes

// Eight neighbours of a row from column k0 on, zeros from k on.  Rows lie anywhere: 16-byte loads need no alignment here.
typedef bf16x8 bf16x8_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

// A row's eight neighbours that end with the row, to those from column k0 on.
__device__ __forceinline__ bf16x8 tail_x8(bf16x8 v, int k0, int k) {
  typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
  const u64x2 q = __builtin_bit_cast(u64x2, v);
  const int over = min(max(k0 + 8 - k, 0), 8), bits = 16 * (over & 3);
  const uint64_t low = over >= 4 ? q.y : q.x, high = over >= 4 ? 0 : q.y;
  const u64x2 y{low >> bits | (high << 1) << (63 - bits), high >> bits};
  return __builtin_bit_cast(bf16x8, over == 8 ? u64x2{0, 0} : y);
}

__device__ __forceinline__ bf16x8 load_x8(const bf16* row, int k0, int k) {
  bf16x8 v;
  if (k0 + 8 <= k) {
    v = *reinterpret_cast<const bf16x8_any*>(row + k0);
  } else if (k >= 8) {
    v = tail_x8(*reinterpret_cast<const bf16x8_any*>(row + k - 8), k0, k);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k0 + j < k ? row[k0 + j] : static_cast<bf16>(0.f);
  }
  return v;
}

template <typename X>
__device__ __forceinline__ void load_x8(const X* row, int k0, int k, float (&v)[8]) {
  if constexpr (sizeof(X) == 2) {
    const bf16x8 t = load_x8(row, k0, k);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32(t[j]);
  } else if (k0 + 8 <= k) {
    const f32x4 a = *reinterpret_cast<const f32x4_any*>(row + k0), b = *reinterpret_cast<const f32x4_any*>(row + k0 + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = a[j];
      v[4 + j] = b[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k0 + j < k ? to_f32(row[k0 + j]) : 0.f;
  }
}

template <int P>
__device__ __forceinline__ void parts8(const float (&v)[8], bf16x8 (&out)[P]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    bf16 p[P];
    bf16_parts(v[j], p);
#pragma unroll
    for (int i = 0; i < P; ++i) out[i][j] = p[i];
  }
}

__device__ __forceinline__ float silu(float x) { return x / (1.f + __expf(-x)); }

// The sum over a workgroup of up to kMaxWaves4 waves.
__device__ __forceinline__ float group_sum(float v, float* scratch, int waves) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < waves; ++i) s += scratch[i];
  return s;
}

// ---------------------------------------------------------------------------
// out = x' + LN(z), one row per workgroup: z and x stay in registers between the sums and the result
// ---------------------------------------------------------------------------
struct Norm4Args {
  int d;
  float eps, x_eps;
  const float* z;  // (B, T, d)
  const void* x;
  int64_t xs_b, xs_t;
  const void* gain;  // (d,) of x's type, or null: x' = RMSNorm(x) times it
  const float *ln_w, *ln_b;
  void* out;
  int64_t os_b, os_t;
};

// AGENT: z was stored by other workgroups of this launch, past their caches, and is read the same way
template <typename T, int NT, bool AGENT>
__device__ __forceinline__ void readout_norm(const Norm4Args& a, const float* z, const T* x, T* out, float* scratch) {
  constexpr int kEach = 4096 / NT;
  float v[kEach], xv[kEach];
  float sum = 0.f, squares = 0.f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int e = threadIdx.x + i * NT;
    v[i] = 0.f;
    if (e < a.d) {
      if constexpr (AGENT)
        v[i] = __hip_atomic_load(z + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      else
        v[i] = z[e];
    }
    xv[i] = e < a.d ? to_f32(x[e]) : 0.f;
    sum += v[i];
    squares = fmaf(xv[i], xv[i], squares);
  }
  const float mean = group_sum(sum, scratch, NT / 64) / (float)a.d;
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const float g = (int)threadIdx.x + i * NT < a.d ? v[i] - mean : 0.f;
    far = fmaf(g, g, far);
  }
  const float rs = 1.f / sqrtf(group_sum(far, scratch, NT / 64) / (float)a.d + a.eps);
  float xr = 1.f;
  if (a.gain != nullptr) xr = 1.f / sqrtf(group_sum(squares, scratch, NT / 64) / (float)a.d + a.x_eps);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int e = threadIdx.x + i * NT;
    if (e >= a.d) break;
    float y = xv[i];
    if (a.gain != nullptr) y *= xr * to_f32(static_cast<const T*>(a.gain)[e]);
    out[e] = from_f32<T>(y + ((v[i] - mean) * rs * a.ln_w[e] + a.ln_b[e]));
  }
}

// Grid (T, B).  Latency: 3 us for 32 rows of 768.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_readout4_norm(const Norm4Args a) {
  __shared__ float scratch[kMaxWaves4];
  const int t = blockIdx.x, b = blockIdx.y;
  readout_norm<T, kThreads, false>(a, a.z + ((int64_t)b * gridDim.x + t) * a.d, static_cast<const T*>(a.x) + b * a.xs_b + t * a.xs_t,
                                   static_cast<T*>(a.out) + b * a.os_b + t * a.os_t, scratch);
}

// ---------------------------------------------------------------------------
// one row
// ---------------------------------------------------------------------------
enum class Row { kLinear, kSwiglu, kDown };

struct Gemv4Args {
  int n, k, blocks, tiles, split;  // split: waves that divide a tile's columns
  float x_eps;
  const void* x;  // (k,) per batch; kDown: bf16 parts (P, k)
  int64_t xs_b;
  const void* gain;
  const char* w[2];
  int64_t ws_b[2];
  const void* r;
  void* out;  // kSwiglu: bf16 parts (P, n) per batch; kDown: z
  int64_t os_b;
  unsigned* counters;  // (B,): kSwiglu clears them, kDown counts a row's workgroups
  Norm4Args norm;
};

// A tile of 16 rows of W per `split` waves, 4 waves at least to a workgroup: x's parts are read from LDS as rows of the operand,
// so that one product serves them all, and the codes go from memory into the product.  Bound by reading W where there
// is much of it: a row by 32000 x 2048 7.8 us (4.7 TB/s), readouts of 32 x (2048, 5504) 115 us (5.3 TB/s, partly from the infinity
// cache); by latency where not: 3.4 us by 1280 x 768, a readout of 768 x 2048 5 + 6.  Grid (tiles, batch).
template <typename X, typename T, int P, Row MODE>
__global__ void __launch_bounds__(kMaxWaves4 * 64) k_gemv4(const Gemv4Args a) {
  constexpr int S = MODE == Row::kSwiglu ? 2 : 1;
  constexpr int U = 2;  // blocks of columns loaded ahead
  extern __shared__ __align__(16) char lds[];
  __shared__ float red[kMaxWaves4][S][16];
  __shared__ float scratch[kMaxWaves4];
  __shared__ int last;
  const int waves = blockDim.x >> 6, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r = lane & 15, h = lane >> 4, b = blockIdx.y;
  const int per = waves / a.split, tile = blockIdx.x * per + w / a.split, part = w % a.split;
  const int begin = a.blocks * part / a.split, end = a.blocks * (part + 1) / a.split;
  const char* wp[S];
#pragma unroll
  for (int s = 0; s < S; ++s) wp[s] = a.w[s] + b * a.ws_b[s] + (int64_t)min(tile, a.tiles - 1) * a.blocks * kBlockBytes;
  u32x4 code[2][U][S];
  u32x2 scale[2][U][S];
  auto fetch = [&](int kb, u32x4 (&c)[U][S], u32x2 (&f)[U][S]) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const char* at = wp[s] + (int64_t)min(kb + u, end - 1) * kBlockBytes;
        c[u][s] = *reinterpret_cast<const u32x4*>(at + lane * 16);
        f[u][s] = *reinterpret_cast<const u32x2*>(at + 1024 + r * 8);
      }
  };
  fetch(begin, code[0], scale[0]);
  if (MODE == Row::kSwiglu && blockIdx.x == 0 && threadIdx.x == 0) a.counters[b * kCounterPitch] = 0;

  // the row's parts into LDS, a part every `pitch` bytes (shifted by half the banks), zeros behind k
  const int wide = a.blocks * 128, pitch = wide * 2 + 64;
  float squares = 0.f;
  for (int k0 = threadIdx.x * 8; k0 < wide; k0 += blockDim.x * 8) {
    bf16x8 p[P];
    if constexpr (MODE == Row::kDown) {
#pragma unroll
      for (int i = 0; i < P; ++i) p[i] = load_x8(static_cast<const bf16*>(a.x) + b * a.xs_b + (int64_t)i * a.k, k0, a.k);
    } else {
      float v[8];
      load_x8(static_cast<const X*>(a.x) + b * a.xs_b, k0, a.k, v);
      if (a.x_eps > 0.f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) squares = fmaf(v[j], v[j], squares);
      }
      if (a.gain != nullptr) {
        float g[8];
        load_x8(static_cast<const X*>(a.gain), k0, a.k, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= g[j];
      }
      parts8(v, p);
    }
#pragma unroll
    for (int i = 0; i < P; ++i) *reinterpret_cast<bf16x8*>(lds + i * pitch + k0 * 2) = p[i];
  }
  float norm = 1.f;
  if (MODE != Row::kDown && a.x_eps > 0.f) norm = rsqrtf(group_sum(squares, scratch, waves) / (float)a.k + a.x_eps);
  __syncthreads();

  const char* xp = lds + (P == 1 ? 0 : min(r, P - 1) * pitch) + 16 * h;  // rows of the operand: the parts
  float y[S];
#pragma unroll
  for (int s = 0; s < S; ++s) y[s] = 0.f;
  auto blocks = [&](int kb, const u32x4 (&c)[U][S], const u32x2 (&f)[U][S]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (kb + u >= end) break;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const bf16x8 x = *reinterpret_cast<const bf16x8*>(xp + (kb + u) * 256 + 64 * g);
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const f32x4 t = mfma16(x, fp4_values(c[u][s][g]), f32x4{0.f, 0.f, 0.f, 0.f});
          const float scale = bf16_of(f[u][s][g >> 1], g & 1);
#pragma unroll
          for (int i = 0; i < P; ++i) y[s] = fmaf(scale, t[i], y[s]);
        }
      }
    }
  };
  for (int kb = begin; kb < end; kb += 2 * U) {
    fetch(kb + U, code[1], scale[1]);
    blocks(kb, code[0], scale[0]);
    fetch(kb + 2 * U, code[0], scale[0]);
    blocks(kb + U, code[1], scale[1]);
  }
  if (h == 0) {
#pragma unroll
    for (int s = 0; s < S; ++s) red[w][s][r] = y[s];
  }
  __syncthreads();
  if ((int)threadIdx.x < per * 16) {
    const int t = threadIdx.x >> 4, n = (blockIdx.x * per + t) * 16 + (threadIdx.x & 15);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      y[s] = 0.f;
      for (int q = 0; q < a.split; ++q) y[s] += red[t * a.split + q][s][threadIdx.x & 15];
      y[s] *= norm;
    }
    if (n < a.n) {
      if constexpr (MODE == Row::kLinear) {
        if (a.r != nullptr) y[0] += to_f32(static_cast<const T*>(a.r)[n]);
        static_cast<T*>(a.out)[n] = from_f32<T>(y[0]);
      } else if constexpr (MODE == Row::kSwiglu) {
        constexpr int HP = sizeof(T) == 2 ? 2 : 3;
        bf16 p[HP];
        bf16_parts(silu(y[1]) * y[0], p);
#pragma unroll
        for (int i = 0; i < HP; ++i) (static_cast<bf16*>(a.out) + b * a.os_b)[(int64_t)i * a.n + n] = p[i];
      } else {
        __hip_atomic_store(static_cast<float*>(a.out) + b * a.os_b + n, y[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
  if constexpr (MODE == Row::kDown) {
    // A row's last workgroup normalises it: stores past the caches, every thread waits for its own, then the row's count goes
    // up; the last one reads past the caches.  The launch before cleared the counts.
    wait_vmcnt<0>();
    __syncthreads();
    if (threadIdx.x == 0)
      last = __hip_atomic_fetch_add(a.counters + b * kCounterPitch, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    const float* z = static_cast<const float*>(a.out) + b * a.os_b;
    const T* x = static_cast<const T*>(a.norm.x) + b * a.norm.xs_b;
    T* out = static_cast<T*>(a.norm.out) + b * a.norm.os_b;
    if (waves == 4)
      readout_norm<T, 256, true>(a.norm, z, x, out, scratch);
    else
      readout_norm<T, 512, true>(a.norm, z, x, out, scratch);
  }
}

// ---------------------------------------------------------------------------
// more rows
// ---------------------------------------------------------------------------
// Rows of x in parts lie in the operands' order, so that a wave reads each as 1 KB: per batch, 16 rows and 32 columns the parts
// one after the other, in each 16 bytes for lane 16 h + r, row r's columns 8 h .. 8 h + 7.  Columns are padded with zeros
// to whole 64; rows behind the last hold anything.
__host__ __device__ __forceinline__ int64_t parts_of_batch(int64_t m, int64_t k, int parts) {  // elements
  return (m + 15) / 16 * 16 * ((k + 63) / 64 * 64) * parts;
}
__device__ __forceinline__ int64_t part_place(int m, int k, int part, int groups, int parts) {
  return ((((int64_t)(m >> 4) * groups + (k >> 5)) * parts + part) * 64 + ((k & 31) >> 3) * 16 + (m & 15)) * 8 + (k & 7);
}

struct Parts4Args {
  int m, k;
  float x_eps;
  const void* x;
  int64_t xs_b, xs_m;
  const void* gain;
  bf16* out;
  unsigned* counters;  // of the product that follows, cleared here
  int n_counters;
};

constexpr int kPartsColumns = kThreads * 8;

// Rows as bf16 parts, RMS-normalised and multiplied by the norm's weight where there is one.  Grid (m, columns, B); every
// workgroup of a row forms its sum of squares.  Latency: 61 rows of 5501 fp32 values 3 to 5 us.
template <typename X, int P>
__global__ void __launch_bounds__(kThreads) k_parts4(const Parts4Args a) {
  __shared__ float scratch[kMaxWaves4];
  const int m = blockIdx.x, b = blockIdx.z, wide = (a.k + 63) / 64 * 64;
  const X* row = static_cast<const X*>(a.x) + b * a.xs_b + m * a.xs_m;
  if (m == 0 && blockIdx.y == 0 && b == 0)
    for (int i = threadIdx.x; i < a.n_counters; i += kThreads) a.counters[i * kCounterPitch] = 0;
  float norm = 1.f;
  if (a.x_eps > 0.f) {
    float squares = 0.f;
    for (int k0 = threadIdx.x * 8; k0 < a.k; k0 += kThreads * 8) {
      float v[8];
      load_x8(row, k0, a.k, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) squares = fmaf(v[j], v[j], squares);
    }
    norm = rsqrtf(group_sum(squares, scratch, kThreads / 64) / (float)a.k + a.x_eps);
  }
  const int k0 = blockIdx.y * kPartsColumns + threadIdx.x * 8;
  if (k0 >= wide) return;
  float v[8];
  load_x8(row, k0, a.k, v);
  if (a.gain != nullptr) {
    float g[8];
    load_x8(static_cast<const X*>(a.gain), k0, a.k, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= g[j];
  }
  if (a.x_eps > 0.f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= norm;
  }
  bf16x8 p[P];
  parts8(v, p);
  bf16* out = a.out + b * parts_of_batch(a.m, a.k, P);
#pragma unroll
  for (int i = 0; i < P; ++i) *reinterpret_cast<bf16x8*>(out + part_place(m, k0, i, wide / 32, P)) = p[i];
}

struct Prod4Args {
  int m, n, k, blocks;
  float x_eps;    // > 0 (one part): rows of x are RMS-normalised
  const bf16* x;  // one part: rows; more: operands (parts_of_batch)
  int64_t xs_b, xs_m;
  const char* w[2];
  int64_t ws_b[2];
  const void* r;
  int64_t rs_m;
  void* out;  // SWIGLU: the next product's operands
  int64_t os_b, os_m;
  int nsplit;          // > 1: workgroups that divide the columns of the same rows and tiles
  float* part;         // their sums, (group, split, 16 MT rows, 16 NT columns)
  unsigned* counters;  // of a group's splits that have stored theirs
};

constexpr int kMaxSplits = 8;
constexpr int kSplitGroups = 256;        // at least two splits each
constexpr int kSplitFloats = 32 * 64;    // of a workgroup

// Products whose columns may be divided over workgroups.
constexpr bool splits(int parts, int nt, int w, bool swiglu) { return parts == 3 && nt == 4 && w == 4 && !swiglu; }

// A product's element (m, n): the result, or with SWIGLU (y up, `gate` the gate's) the next product's operands.
template <typename O, bool SWIGLU>
__device__ __forceinline__ void finish_row(const Prod4Args& a, int b, int m, int n, float y, float gate) {
  if (m >= a.m || n >= a.n) return;
  if constexpr (SWIGLU) {
    constexpr int HP = sizeof(O) == 2 ? 2 : 3;
    bf16 p[HP];
    bf16_parts(silu(gate) * y, p);
    bf16* out = static_cast<bf16*>(a.out) + b * parts_of_batch(a.m, a.n, HP);
#pragma unroll
    for (int q = 0; q < HP; ++q) out[part_place(m, n, q, a.n / 32, HP)] = p[q];
  } else {
    if (a.r != nullptr) y += to_f32(static_cast<const O*>(a.r)[(int64_t)m * a.rs_m + n]);
    (static_cast<O*>(a.out) + b * a.os_b)[(int64_t)m * a.os_m + n] = from_f32<O>(y);
  }
}

// Grid (n / (16 NT), m / (16 MT), batch); the W waves divide the columns and meet in LDS.  Operands are loaded 64 columns
// ahead, pieces of the weights 128.  Rows of one part go through LDS, a wave's own, 8 lanes to 128 bytes of a row: read as
// operands, where neighbouring lanes are different rows, every lane would be an access of its own (32 rows by 8000 x 2048
// took 12 us for 7).  Latency at a few hundred tiles: 32 rows by 768 x 768 3.7 us, by 2048 x 2048 5.
template <typename O, int P, int MT, int NT, int W, bool SWIGLU>
__global__ void __launch_bounds__(W * 64, W == 4 ? 2 : 1) k_prod4(const Prod4Args a) {
  constexpr int kStage = P == 1 ? W * MT * 2048 : 0, kMeet = W * NT * MT * 1024;
  __shared__ __align__(16) char lds[kStage > kMeet ? kStage : kMeet];
  __shared__ float squares[W][MT * 16];
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r = lane & 15, h = lane >> 4;
  constexpr int TILES = SWIGLU ? NT / 2 : NT;  // tiles of n
  constexpr bool kSplits = splits(P, NT, W, SWIGLU);
  const int nsplit = kSplits ? a.nsplit : 1, split = kSplits ? blockIdx.x % nsplit : 0;
  const int tiles = (a.n + 15) >> 4, tile0 = blockIdx.x / nsplit * TILES, m0 = blockIdx.y * (16 * MT), b = blockIdx.z;
  const char* wp[NT];
#pragma unroll
  for (int s = 0; s < NT; ++s) {
    const int which = SWIGLU ? s & 1 : 0, tile = min(tile0 + (SWIGLU ? s >> 1 : s), tiles - 1);
    wp[s] = a.w[which] + b * a.ws_b[which] + (int64_t)tile * a.blocks * kBlockBytes;
  }
  f32x4 acc[NT][MT], gram[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    gram[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < NT; ++s) acc[s][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  struct Weights {
    u32x4 code[NT];
    u32x2 scale[NT];
  };
  auto weights = [&](int kb) {
    Weights v;
#pragma unroll
    for (int s = 0; s < NT; ++s) {
      const char* at = wp[s] + (int64_t)kb * kBlockBytes;
      v.code[s] = *reinterpret_cast<const u32x4*>(at + lane * 16);
      v.scale[s] = *reinterpret_cast<const u32x2*>(at + 1024 + r * 8);
    }
    return v;
  };
  // 64 columns of x: pieces of rows on their way to LDS (one part), or operands
  struct Ahead {
    bf16x8 x[2 * MT * P];
  };
  const bf16* base = a.x + b * a.xs_b;
  const int groups = (a.k + 63) / 64 * 2;
  auto ahead = [&](int half) {
    Ahead v;
    if constexpr (P == 1) {
      const int k0 = half * 64 + 8 * (lane & 7);
      const bool plain = half * 64 + 64 <= a.k;
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) {
        const bf16* row = base + (int64_t)min(m0 + 8 * i + (lane >> 3), a.m - 1) * a.xs_m;
        v.x[i] = plain ? *reinterpret_cast<const bf16x8_any*>(row + k0) : load_x8(row, k0, a.k);
      }
    } else {
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const int rows = min(m0 + 16 * t, (a.m - 1) & ~15);  // a block of 16 rows that there is
          const bf16* at = base + (((int64_t)(rows >> 4) * groups + 2 * half + g) * P) * 512 + lane * 8;
#pragma unroll
          for (int i = 0; i < P; ++i) v.x[(g * MT + t) * P + i] = *reinterpret_cast<const bf16x8*>(at + i * 512);
        }
    }
    return v;
  };
  char* stage = lds + w * (MT * 2048);
  auto multiply = [&](const Ahead& v, const Weights& q, int half) {
    bf16x8 x[2][MT][P];
    if constexpr (P == 1) {  // piece p of row t lies in slot p ^ (t / 2 mod 8)
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) {
        const int t = 8 * i + (lane >> 3);
        *reinterpret_cast<bf16x8*>(stage + t * 128 + (((lane & 7) ^ row_swz(t)) * 16)) = v.x[i];
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const int row = 16 * t + r;
          x[g][t][0] = *reinterpret_cast<const bf16x8*>(stage + row * 128 + (((4 * g + h) ^ row_swz(row)) * 16));
        }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    } else {
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int i = 0; i < P; ++i) x[g][t][i] = v.x[(g * MT + t) * P + i];
    }
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      if (P == 1 && a.x_eps > 0.f) {  // a row's sum of squares: the diagonal of x x^T
#pragma unroll
        for (int t = 0; t < MT; ++t) gram[t] = mfma16(x[g][t][0], x[g][t][0], gram[t]);
      }
#pragma unroll
      for (int s = 0; s < NT; ++s) {
        const bf16x8 c = fp4_values(half ? q.code[s][2 + g] : q.code[s][g]);
        const float f = bf16_of(half ? q.scale[s][1] : q.scale[s][0], g);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          f32x4 y{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < P; ++i) y = mfma16(x[g][t][i], c, y);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[s][t][i] = fmaf(f, y[i], acc[s][t][i]);
        }
      }
    }
  };
  const int part = split * W + w, parts = nsplit * W;
  const int begin = a.blocks * part / parts, end = a.blocks * (part + 1) / parts, halves = (a.k + 63) >> 6;
  if (begin < end) {
    Weights next = weights(begin);
    Ahead first = ahead(2 * begin);
    for (int kb = begin; kb < end; ++kb) {
      const Weights now = next;
      const bool both = 2 * kb + 1 < halves;  // the last block may have 64 columns only
      const Ahead second = ahead(both ? 2 * kb + 1 : 2 * kb);
      next = weights(min(kb + 1, end - 1));
      multiply(first, now, 0);
      first = ahead(min(2 * kb + 2, 2 * end - 2));
      if (both) multiply(second, now, 1);
    }
  }
  if (P == 1 && a.x_eps > 0.f && r >> 2 == h) {
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const float lo = r & 1 ? gram[t][1] : gram[t][0], hi = r & 1 ? gram[t][3] : gram[t][2];
      squares[w][16 * t + r] = r & 2 ? hi : lo;
    }
  }
  __syncthreads();
  float* red = reinterpret_cast<float*>(lds);  // [wave][tile][4 t + i][lane]
#pragma unroll
  for (int s = 0; s < NT; ++s)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[((w * NT + s) * (MT * 4) + 4 * t + i) * 64 + lane] = acc[s][t][i];
  __syncthreads();
  constexpr int kOuts = MT * TILES * 4 / W > 0 ? MT * TILES * 4 / W : 1;  // of a thread: 16 TILES neighbours of 16 MT rows
  const int group = blockIdx.y * (gridDim.x / nsplit) + blockIdx.x / nsplit;
  float* sums = kSplits && nsplit > 1 ? a.part + (int64_t)group * nsplit * kSplitFloats : nullptr;
#pragma unroll
  for (int o = 0; o < kOuts; ++o) {
    const int idx = threadIdx.x + o * W * 64, nn = idx & 15, s = (idx >> 4) % TILES, mm = idx / (16 * TILES);
    if (mm >= 16 * MT) break;
    const int i = 4 * (mm >> 4) + (mm & 3), l = ((mm & 15) >> 2) * 16 + nn;
    float y = 0.f, gate = 0.f;
#pragma unroll
    for (int q = 0; q < W; ++q) {
      y += red[((q * NT + (SWIGLU ? 2 * s : s)) * (MT * 4) + i) * 64 + l];
      if (SWIGLU) gate += red[((q * NT + 2 * s + 1) * (MT * 4) + i) * 64 + l];
    }
    if (P == 1 && a.x_eps > 0.f) {
      float q2 = 0.f;
#pragma unroll
      for (int q = 0; q < W; ++q) q2 += squares[q][mm];
      y *= rsqrtf(q2 / (float)a.k + a.x_eps);
    }
    if (kSplits && sums != nullptr)
      __hip_atomic_store(sums + split * kSplitFloats + idx, y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    else
      finish_row<O, SWIGLU>(a, b, m0 + mm, (tile0 + s) * 16 + nn, y, gate);
  }
  if constexpr (kSplits) {
    if (sums == nullptr) return;
    // The group's last workgroup adds up, in the splits' order: stores past the caches, every thread waits for its own, then the
    // group's count goes up; the last one reads past the caches.  The launch before cleared the counts.
    __shared__ bool last;
    wait_vmcnt<0>();
    __syncthreads();
    if (threadIdx.x == 0)
      last = (int)__hip_atomic_fetch_add(a.counters + group * kCounterPitch, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
             nsplit - 1;
    __syncthreads();
    if (!last) return;
    float v[kMaxSplits][kOuts];
#pragma unroll
    for (int q = 0; q < kMaxSplits; ++q)
#pragma unroll
      for (int o = 0; o < kOuts; ++o)
        v[q][o] = __hip_atomic_load(sums + min(q, nsplit - 1) * kSplitFloats + threadIdx.x + o * W * 64, __ATOMIC_RELAXED,
                                    __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (int o = 0; o < kOuts; ++o) {
      const int idx = threadIdx.x + o * W * 64, nn = idx & 15, s = (idx >> 4) % TILES, mm = idx / (16 * TILES);
      float y = v[0][o];
#pragma unroll
      for (int q = 1; q < kMaxSplits; ++q) y += q < nsplit ? v[q][o] : 0.f;
      finish_row<O, SWIGLU>(a, b, m0 + mm, (tile0 + s) * 16 + nn, y, 0.f);
    }
  }
}

// Many blocks of W: WN waves beside each other take NT blocks of 16 rows each and share x, which passes through LDS in
// steps that all of them load together; 8 / WN such teams divide the columns.  Of 32 rows by 32000 x 2048 the operands of x
// are then a fourth of what every wave would fetch for itself; 12.1 us (13.5 with the norm, whose sums are products too), 64 rows
// 17.8 (20.6).  No single rate bounds it: the bytes are 8.2 us, the vector instructions (3000 a SIMD) 5, the products under 2; 250
// workgroups of eight waves are one a unit, so that nothing else runs while a step's barrier and its loads are waited for.
// Rows of 8 columns or more.
// Grid (n / (16 NT WN), m / (16 MT), batch).
template <typename O, int MT, int NT, int WN>
__global__ void __launch_bounds__(512, 2) k_share4(const Prod4Args a) {
  constexpr int WK = 8 / WN;
  constexpr int H = WN == 4 ? 2 : 1;            // halves (64 columns) of a step
  constexpr int kStep = H * 2 * MT * 1024;      // bytes of a step of x
  constexpr int kEach = kStep / 1024 / WN;      // 1 KB pieces of it that a wave loads: 8 rows of 64 columns
  static_assert(kStep % (1024 * WN) == 0, "a team loads a step together");
  constexpr int kStage = WK * 2 * kStep, kMeet = 8 * NT * MT * 1024;
  __shared__ __align__(16) char lds[kStage > kMeet ? kStage : kMeet];
  __shared__ float squares[WK][MT * 16];
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wn = w % WN, wk = w / WN;
  const int lane = threadIdx.x & 63, r = lane & 15, h = lane >> 4;
  const int tiles = (a.n + 15) >> 4, tile0 = (blockIdx.x * WN + wn) * NT, m0 = blockIdx.y * (16 * MT), b = blockIdx.z;
  const char* wp[NT];
#pragma unroll
  for (int s = 0; s < NT; ++s) wp[s] = a.w[0] + b * a.ws_b[0] + (int64_t)min(tile0 + s, tiles - 1) * a.blocks * kBlockBytes;
  f32x4 acc[NT][MT], gram[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    gram[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < NT; ++s) acc[s][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  struct Weights {
    u32x4 code[NT];
    u32x2 scale[NT];
  };
  const int begin = a.blocks * wk / WK, end = a.blocks * (wk + 1) / WK, halves = (a.k + 63) >> 6;
  const int steps = (a.blocks + WK - 1) / WK * (2 / H);  // of the longest team
  const bf16* base = a.x + b * a.xs_b;
  auto weights = [&](int kb) {
    Weights v;
    kb = min(kb, max(end - 1, 0));
#pragma unroll
    for (int s = 0; s < NT; ++s) {
      const char* at = wp[s] + (int64_t)kb * kBlockBytes;
      v.code[s] = *reinterpret_cast<const u32x4*>(at + lane * 16);
      v.scale[s] = *reinterpret_cast<const u32x2*>(at + 1024 + r * 8);
    }
    return v;
  };
  struct Pieces {
    bf16x8 x[kEach];
  };
  auto load = [&](int half0) {
    Pieces v;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int piece = i * WN + wn, half = min(half0 + piece / (2 * MT), halves - 1), k0 = half * 64 + 8 * (lane & 7);
      const bf16* row = base + (int64_t)min(m0 + 8 * (piece % (2 * MT)) + (lane >> 3), a.m - 1) * a.xs_m;
      v.x[i] = *reinterpret_cast<const bf16x8_any*>(row + min(k0, a.k - 8));
    }
    return v;
  };
  auto store = [&](Pieces v, int buf, int half0) {
    char* to = lds + (wk * 2 + buf) * kStep;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int piece = i * WN + wn, t = 8 * (piece % (2 * MT)) + (lane >> 3);
      const int half = min(half0 + piece / (2 * MT), halves - 1);
      if (half * 64 + 64 > a.k) v.x[i] = tail_x8(v.x[i], half * 64 + 8 * (lane & 7), a.k);
      *reinterpret_cast<bf16x8*>(to + piece / (2 * MT) * (MT * 2048) + t * 128 + (((lane & 7) ^ row_swz(t)) * 16)) = v.x[i];
    }
  };
  auto multiply = [&](const Weights& q, int buf, int local, int half) {  // `half` of the block of columns, `local` of the step
    const char* from = lds + (wk * 2 + buf) * kStep + local * (MT * 2048);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      bf16x8 x[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int row = 16 * t + r;
        x[t] = *reinterpret_cast<const bf16x8*>(from + row * 128 + (((4 * g + h) ^ row_swz(row)) * 16));
      }
      if (a.x_eps > 0.f && wn == 0) {  // a row's sum of squares: the diagonal of x x^T
#pragma unroll
        for (int t = 0; t < MT; ++t) gram[t] = mfma16(x[t], x[t], gram[t]);
      }
#pragma unroll
      for (int s = 0; s < NT; ++s) {
        const bf16x8 c = fp4_values(half ? q.code[s][2 + g] : q.code[s][g]);
        const float f = bf16_of(half ? q.scale[s][1] : q.scale[s][0], g);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const f32x4 y = mfma16(x[t], c, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[s][t][i] = fmaf(f, y[i], acc[s][t][i]);
        }
      }
    }
  };
  // Step i of a team is in buffer i mod 2.  Behind the barrier that opens it nobody reads the other one any more, which
  // takes step i + 1; the pieces of the four steps behind it and the next weights are on their way meanwhile.
  constexpr int kWeights = H == 2 ? 4 : 2;
  Weights q[kWeights];
  Pieces pieces[4];
  // loads come back in order: what the first step needs goes first
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    pieces[u] = load(2 * begin + u * H);
    if (u < kWeights) q[u] = weights(begin + u);
  }
  store(pieces[0], 0, 2 * begin);
  pieces[0] = load(2 * begin + 4 * H);
  for (int i0 = 0; i0 < steps; i0 += 4) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u;
      if (i >= steps) break;
      __syncthreads();
      store(pieces[(u + 1) & 3], (u + 1) & 1, 2 * begin + (i + 1) * H);
      pieces[(u + 1) & 3] = load(2 * begin + (i + 5) * H);
      const int kb = begin + i * H / 2;
      if constexpr (H == 2) {
        if (kb < end) {
          multiply(q[u], u & 1, 0, 0);
          if (2 * kb + 1 < halves) multiply(q[u], u & 1, 1, 1);
        }
        q[u] = weights(kb + 4);
      } else {
        if (kb < end && ((u & 1) == 0 || 2 * kb + 1 < halves)) multiply(q[u >> 1], u & 1, 0, u & 1);
        if (u & 1) q[u >> 1] = weights(kb + 2);
      }
    }
  }
  if (a.x_eps > 0.f && wn == 0 && r >> 2 == h) {
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const float lo = r & 1 ? gram[t][1] : gram[t][0], hi = r & 1 ? gram[t][3] : gram[t][2];
      squares[wk][16 * t + r] = r & 2 ? hi : lo;
    }
  }
  __syncthreads();
  float* red = reinterpret_cast<float*>(lds);  // [team][wave of it][tile][4 t + i][lane]
#pragma unroll
  for (int s = 0; s < NT; ++s)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[((w * NT + s) * (MT * 4) + 4 * t + i) * 64 + lane] = acc[s][t][i];
  __syncthreads();
  constexpr int kCols = 16 * NT * WN, kOuts = MT * 16 * kCols / 512 > 0 ? MT * 16 * kCols / 512 : 1;
#pragma unroll
  for (int o = 0; o < kOuts; ++o) {
    const int idx = threadIdx.x + o * 512, col = idx % kCols, mm = idx / kCols;
    if (mm >= 16 * MT) break;
    const int nn = col & 15, s = (col >> 4) % NT, of_n = (col >> 4) / NT;
    const int i = 4 * (mm >> 4) + (mm & 3), l = ((mm & 15) >> 2) * 16 + nn;
    float y = 0.f;
#pragma unroll
    for (int q = 0; q < WK; ++q) y += red[(((q * WN + of_n) * NT + s) * (MT * 4) + i) * 64 + l];
    if (a.x_eps > 0.f) {
      float q2 = 0.f;
#pragma unroll
      for (int q = 0; q < WK; ++q) q2 += squares[q][mm];
      y *= rsqrtf(q2 / (float)a.k + a.x_eps);
    }
    finish_row<O, false>(a, b, m0 + mm, blockIdx.x * kCols + col, y, 0.f);
  }
}

template <typename X, int P>
void launch_parts(const Parts4Args& x, int batch, hipStream_t st) {
  const dim3 grid((unsigned)x.m, (unsigned)((x.k + kPartsColumns - 1) / kPartsColumns), (unsigned)batch);
  hipLaunchKernelGGL((k_parts4<X, P>), grid, dim3(kThreads), 0, st, x);
}

template <typename O, int P, int NT, int W, bool SWIGLU>
void launch_rows(const Prod4Args& p, int batch, hipStream_t st) {
  const int tiles = (p.n + 15) / 16, per = SWIGLU ? NT / 2 : NT;
  const int mt = p.m <= 16 ? 1 : p.m <= 32 || P > 1 ? 2 : 4;
  const int nsplit = splits(P, NT, W, SWIGLU) ? p.nsplit : 1;
  const dim3 grid((unsigned)((tiles + per - 1) / per * nsplit), (unsigned)((p.m + 16 * mt - 1) / (16 * mt)), (unsigned)batch);
  const dim3 block(W * 64);
  if (mt == 1)
    hipLaunchKernelGGL((k_prod4<O, P, 1, NT, W, SWIGLU>), grid, block, 0, st, p);
  else if (mt == 2)
    hipLaunchKernelGGL((k_prod4<O, P, 2, NT, W, SWIGLU>), grid, block, 0, st, p);
  else if constexpr (P == 1)
    hipLaunchKernelGGL((k_prod4<O, P, 4, NT, W, SWIGLU>), grid, block, 0, st, p);
}

template <typename O, int NT, int WN>
void launch_share(const Prod4Args& p, int batch, hipStream_t st) {
  const int tiles = (p.n + 15) / 16, per = NT * WN, mt = p.m <= 16 ? 1 : p.m <= 32 ? 2 : 4;
  const dim3 grid((unsigned)((tiles + per - 1) / per), (unsigned)((p.m + 16 * mt - 1) / (16 * mt)), (unsigned)batch);
  if (mt == 1)
    hipLaunchKernelGGL((k_share4<O, 1, NT, WN>), grid, dim3(512), 0, st, p);
  else if (mt == 2)
    hipLaunchKernelGGL((k_share4<O, 2, NT, WN>), grid, dim3(512), 0, st, p);
  else
    hipLaunchKernelGGL((k_share4<O, 4, NT, WN>), grid, dim3(512), 0, st, p);
}

// Measured, us, for rows x (n, k): one part, 32 x (32000, 2048): waves for themselves, 4 blocks of W each 17.1, sharing x,
// teams of 4 with 2 blocks each 12.1, of 4 with one block 12.6, of 2 with one 16.8 (8 rows 9.5, 9.1, 10.4; 64 rows 17.8, 23.1, 32.3);
// 32 x (16000, 2048): teams of 4 with 2 blocks 12.7, of 2 with one 10.1 (64 rows 16.4, 16.8, of 4 with one block 12.1);
// 32 x (5504, 2048): eight waves for themselves 7.3, teams of 2 6.8; of 2048 columns alike.  More rows convert W again for
// every 64 of them: 128 x (32000, 2048) 41, 256 77, 1024 298, where the library's product of 16-bit weights takes 26, 33 and 102 (64
// rows 23 and 23); 1024 x (1280, 768) 12.4 and 8.7.
// Three parts, which already are in the operands' order: 32 x (32000, 2048) sharing 23.8, for themselves 4 blocks each 21.5; 61 x
// (1999, 5501) sharing 30, eight waves to a block 29, 16 27.  What bounds that last one is x, read once per workgroup: 4 blocks of W
// each and the columns divided over 8 workgroups instead 18.8 (with the rows' parts 24.0 before), 32 x (2048, 5504) 14.3 for 19.8, 5 x
// (100, 11000) 10.3 for 19.1; of few columns it is the second exchange that costs (7 x (300, 1000) 7.9 for 6.5): from 16 blocks of
// columns on, 4 a workgroup.
template <typename O, int P>
void launch_linear_rows(const Prod4Args& p, int batch, hipStream_t st) {
  const int64_t tiles = (p.n + 15) / 16 * batch * ((p.m + 31) / 32);
  if constexpr (P == 1) {
    if (tiles >= 1536 && p.k >= 8)
      launch_share<O, 2, 4>(p, batch, st);
    else if (tiles >= 192 && p.k >= 8)
      launch_share<O, 1, 2>(p, batch, st);
    else
      launch_rows<O, P, 1, 8, false>(p, batch, st);
  } else if (tiles >= 768 || p.nsplit > 1) {
    launch_rows<O, P, 4, 4, false>(p, batch, st);
  } else if (p.blocks >= 16) {
    launch_rows<O, P, 1, 16, false>(p, batch, st);
  } else {
    launch_rows<O, P, 1, 8, false>(p, batch, st);
  }
}

template <typename X, typename T, int P, Row MODE>
void launch_gemv(Gemv4Args g, int batch, hipStream_t st) {
  g.tiles = (g.n + 15) / 16;
  // waves enough to fill half of the card's 4096 places, as far as a tile has columns to divide (4096, 2048 and 1024 waves are
  // within 10% of each other)
  g.split = 1;
  while (g.split < kMaxWaves4 && 2 * g.split <= g.blocks && (int64_t)g.tiles * batch * g.split < 2048) g.split *= 2;
  const int waves = std::max(4, g.split), per = waves / g.split;
  const size_t lds = (size_t)P * ((size_t)g.blocks * 256 + 64);
  const dim3 grid((unsigned)((g.tiles + per - 1) / per), (unsigned)batch);
  hipLaunchKernelGGL((k_gemv4<X, T, P, MODE>), grid, dim3(waves * 64), lds, st, g);
}

int64_t padded(int64_t k) { return (k + 127) / 128 * 128; }

// Bytes of a row's parts in k_gemv4's LDS.
int64_t row_lds(int64_t k, int parts) { return parts * (padded(k) * 2 + 64); }

bool whole_pieces(const void* p, int64_t a, int64_t b, int64_t vec) { return aligned16(p) && a % vec == 0 && b % vec == 0; }

// Where a readout's buffers lie in its workspace: hidden parts, z, counters, and x's parts (several tokens).
struct Readout4Layout {
  bool single;
  size_t hidden, z, counters, parts, total;
  Readout4Layout(int64_t B, int64_t T, int64_t D, int64_t F) {
    single = T == 1 && row_lds(F, 3) <= kRowLds;
    hidden = 0;
    z = align_up((size_t)B * parts_of_batch(T, F, 3) * 2);
    counters = z + align_up((size_t)B * T * D * 4);
    parts = counters + align_up((size_t)B * kCounterPitch * 4);
    total = parts + (single ? 0 : align_up((size_t)B * parts_of_batch(T, D, 3) * 2));
  }
};

// Where a product's buffers lie in its workspace: x's parts, the sums of splits and their counters.
struct Linear4Layout {
  size_t sums, counters, total;
  Linear4Layout(int64_t m, int64_t k) {
    sums = align_up((size_t)parts_of_batch(m, k, 3) * 2);
    counters = sums + (size_t)2 * kSplitGroups * kSplitFloats * 4;
    total = counters + (size_t)kSplitGroups * kCounterPitch * 4;
  }
};

// One token a row: two launches, each row's last workgroup of the second normalising it.  More: products of rows in parts, with
// SwiGLU four waves to a workgroup (32 rows of 4 tokens, 768 x 2048: 40 us, with eight 50; 16 of 8 28.5 and 32; one of 16, 2048 x
// 5504: 24 to 27 either way).  What bounds those is a launch or two more than one token has, the parts' and the norm's, and x's operands
// from memory for every two blocks of W (32 rows of one token 25, of 16 43, of 64 103, where W is read and converted twice).
template <typename T>
void launch_readout4(const uttt_readout4_args* a, hipStream_t st) {
  constexpr int HP = sizeof(T) == 2 ? 2 : 3;  // parts of the hidden values
  const int D = (int)a->d_model, F = (int)a->d_ff, M = (int)a->tokens, B = (int)a->batch;
  const Readout4Layout at(B, M, D, F);
  char* ws = static_cast<char*>(a->workspace);
  bf16* hidden = reinterpret_cast<bf16*>(ws + at.hidden);
  float* z = reinterpret_cast<float*>(ws + at.z);
  Norm4Args n{};
  n.d = D; n.eps = a->eps; n.x_eps = a->x_norm_eps;
  n.z = z;
  n.x = a->x; n.xs_b = a->x_stride_b; n.xs_t = a->x_stride_t;
  n.gain = a->x_norm_weight;
  n.ln_w = a->ln_weight; n.ln_b = a->ln_bias;
  n.out = a->out; n.os_b = a->out_stride_b; n.os_t = a->out_stride_t;
  const char *up = static_cast<const char*>(a->w_up), *gate = static_cast<const char*>(a->w_gate),
             *down = static_cast<const char*>(a->w_down);
  if (at.single) {
    Gemv4Args g{};
    g.n = F; g.k = D; g.blocks = (D + 127) / 128;
    g.x = a->x; g.xs_b = a->x_stride_b; g.gain = a->x_norm_weight;
    g.x_eps = a->x_norm_weight ? a->x_norm_eps : 0.f;
    g.w[0] = up; g.ws_b[0] = a->w_up_stride; g.w[1] = gate; g.ws_b[1] = a->w_gate_stride;
    g.out = hidden; g.os_b = (int64_t)HP * F;
    g.counters = reinterpret_cast<unsigned*>(ws + at.counters);
    bool whole = false;  // bf16 as it is
    if constexpr (sizeof(T) == 2) {
      whole = g.gain == nullptr;
      if (whole) launch_gemv<T, T, 1, Row::kSwiglu>(g, B, st);
    }
    if (!whole) launch_gemv<T, T, HP, Row::kSwiglu>(g, B, st);
    Gemv4Args d{};
    d.n = D; d.k = F; d.blocks = (F + 127) / 128;
    d.x = hidden; d.xs_b = (int64_t)HP * F;
    d.w[0] = down; d.ws_b[0] = a->w_down_stride;
    d.out = z; d.os_b = D;
    d.counters = g.counters;
    d.norm = n;
    launch_gemv<bf16, T, HP, Row::kDown>(d, B, st);
    return;
  }
  Prod4Args p{};
  p.nsplit = 1;
  p.m = M; p.n = F; p.k = D; p.blocks = (D + 127) / 128;
  p.w[0] = up; p.ws_b[0] = a->w_up_stride; p.w[1] = gate; p.ws_b[1] = a->w_gate_stride;
  p.out = hidden;
  bool whole = false;  // bf16 as it is
  if constexpr (sizeof(T) == 2) {
    whole = a->x_norm_weight == nullptr;
    if (whole) {
      p.x = static_cast<const bf16*>(a->x); p.xs_b = a->x_stride_b; p.xs_m = a->x_stride_t;
      launch_rows<T, 1, 2, 4, true>(p, B, st);
    }
  }
  if (!whole) {
    Parts4Args x{};
    x.m = M; x.k = D;
    x.x_eps = a->x_norm_weight ? a->x_norm_eps : 0.f;
    x.x = a->x; x.xs_b = a->x_stride_b; x.xs_m = a->x_stride_t;
    x.gain = a->x_norm_weight;
    x.out = reinterpret_cast<bf16*>(ws + at.parts);
    launch_parts<T, HP>(x, B, st);
    p.x = x.out; p.xs_b = parts_of_batch(M, D, HP);
    launch_rows<T, HP, 2, 4, true>(p, B, st);
  }
  Prod4Args q{};
  q.nsplit = 1;
  q.m = M; q.n = D; q.k = F; q.blocks = (F + 127) / 128;
  q.x = hidden; q.xs_b = parts_of_batch(M, F, HP);
  q.w[0] = down; q.ws_b[0] = a->w_down_stride;
  q.out = z; q.os_b = (int64_t)M * D; q.os_m = D;
  launch_linear_rows<float, HP>(q, B, st);
  hipLaunchKernelGGL(k_readout4_norm<T>, dim3(M, B), dim3(kThreads), 0, st, n);
}

}  // namespace
}  // namespace uttt

using namespace uttt;

extern "C" int uttt_decode_abi_version(void) { return UTTT_DECODE_ABI_VERSION; }

extern "C" size_t uttt_linear4_workspace(int64_t m, int64_t k, int32_t act_dtype) {
  if (m < 1 || k < 1 || act_dtype == UTTT_DTYPE_BF16 || (m == 1 && row_lds(k, 3) <= kRowLds)) return 0;
  return Linear4Layout(m, k).total;
}

extern "C" int uttt_linear4(const uttt_linear4_args* a, uttt_stream_t stream) {
  UTTT_REQUIRE(a != nullptr, "args is NULL");
  UTTT_REQUIRE(a->act_dtype == UTTT_DTYPE_F32 || a->act_dtype == UTTT_DTYPE_BF16, "bad act_dtype");
  UTTT_REQUIRE(a->m >= 1 && a->m <= (1 << 20) && a->n >= 1 && a->n <= (1 << 24) && a->k >= 1 && a->k <= (1 << 20),
               "m, n and k must be in [1, 2^20], [1, 2^24] and [1, 2^20]");
  UTTT_REQUIRE(a->x_eps >= 0.f && a->x_eps < INFINITY, "x_eps must be finite and >= 0 (0: no norm)");
  UTTT_REQUIRE(a->x && a->w && a->out, "x, w and out must be non-NULL");
  UTTT_REQUIRE(aligned16(a->w), "w must be 16-byte aligned");
  UTTT_REQUIRE((a->m == 1 || (a->x_row_stride >= a->k && a->out_row_stride >= a->n)) &&
                   (a->residual == nullptr || a->m == 1 || a->residual_row_stride >= a->n),
               "row strides must cover k and n");
  const bool b16 = a->act_dtype == UTTT_DTYPE_BF16;
  const size_t parts = uttt_linear4_workspace(a->m, a->k, a->act_dtype);
  UTTT_REQUIRE(parts == 0 || (a->workspace != nullptr && aligned16(a->workspace) && a->workspace_bytes >= parts),
               "workspace too small for the rows' parts");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->m == 1 && row_lds(a->k, b16 ? 1 : 3) <= kRowLds) {
    Gemv4Args g{};
    g.n = (int)a->n; g.k = (int)a->k; g.blocks = (int)((a->k + 127) / 128);
    g.x_eps = a->x_eps;
    g.x = a->x;
    g.w[0] = static_cast<const char*>(a->w);
    g.r = a->residual;
    g.out = a->out;
    if (b16)
      launch_gemv<bf16, bf16, 1, Row::kLinear>(g, 1, st);
    else
      launch_gemv<float, float, 3, Row::kLinear>(g, 1, st);
    return launch_status("uttt_linear4");
  }
  Prod4Args p{};
  p.nsplit = 1;
  p.m = (int)a->m; p.n = (int)a->n; p.k = (int)a->k; p.blocks = (int)((a->k + 127) / 128);
  p.x_eps = a->x_eps;
  p.x = static_cast<const bf16*>(a->x); p.xs_m = a->x_row_stride;
  p.w[0] = static_cast<const char*>(a->w);
  p.r = a->residual; p.rs_m = a->residual_row_stride;
  p.out = a->out; p.os_m = a->out_row_stride;
  if (!b16) {
    Parts4Args x{};
    x.m = p.m; x.k = p.k;
    x.x_eps = a->x_eps;
    x.x = a->x; x.xs_m = a->x_row_stride;
    x.out = static_cast<bf16*>(a->workspace);
    p.x = x.out;
    const Linear4Layout at(a->m, a->k);
    const int64_t groups = (a->n + 63) / 64 * ((a->m + 31) / 32);
    if (p.blocks >= 16)
      p.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({(int64_t)kMaxSplits, 2 * kSplitGroups / groups, p.blocks / 4}));
    p.part = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + at.sums);
    p.counters = x.counters = reinterpret_cast<unsigned*>(static_cast<char*>(a->workspace) + at.counters);
    x.n_counters = p.nsplit > 1 ? (int)groups : 0;
    launch_parts<float, 3>(x, 1, st);
  }
  if (b16)
    launch_linear_rows<bf16, 1>(p, 1, st);
  else
    launch_linear_rows<float, 3>(p, 1, st);
  return launch_status("uttt_linear4");
}

extern "C" size_t uttt_readout4_workspace(int64_t batch, int64_t tokens, int64_t d_model, int64_t d_ff) {
  if (batch < 1 || tokens < 1 || d_model < 1 || d_ff < 1) return 0;
  return Readout4Layout(batch, tokens, d_model, d_ff).total;
}

extern "C" int uttt_readout4(const uttt_readout4_args* a, uttt_stream_t stream) {
  UTTT_REQUIRE(a != nullptr, "args is NULL");
  UTTT_REQUIRE(a->act_dtype == UTTT_DTYPE_F32 || a->act_dtype == UTTT_DTYPE_BF16, "bad act_dtype");
  UTTT_REQUIRE(a->batch >= 1 && a->batch <= 65535 && a->tokens >= 1 && a->tokens <= (1 << 20),
               "batch must be in [1, 65535], tokens in [1, 2^20]");
  UTTT_REQUIRE(a->d_model >= 64 && a->d_model <= 4096 && a->d_model % 64 == 0 && a->d_ff >= 64 && a->d_ff <= (1 << 20) &&
                   a->d_ff % 64 == 0,
               "d_model and d_ff must be multiples of 64, d_model <= 4096, d_ff <= 2^20");
  UTTT_REQUIRE(a->eps > 0.f && (a->x_norm_weight == nullptr || a->x_norm_eps > 0.f), "eps must be > 0");
  UTTT_REQUIRE(a->x && a->w_up && a->w_gate && a->w_down && a->ln_weight && a->ln_bias && a->out,
               "pointers must be non-NULL");
  const bool b16 = a->act_dtype == UTTT_DTYPE_BF16;
  UTTT_REQUIRE(whole_pieces(a->x, a->x_stride_b, a->x_stride_t, b16 ? 8 : 4) && aligned16(a->x_norm_weight),
               "x and its norm's weight must be 16-byte aligned with strides of whole 16-byte pieces");
  UTTT_REQUIRE(aligned16(a->w_up) && aligned16(a->w_gate) && aligned16(a->w_down) && a->w_up_stride % 16 == 0 &&
                   a->w_gate_stride % 16 == 0 && a->w_down_stride % 16 == 0,
               "weights must be 16-byte aligned");
  UTTT_REQUIRE(a->workspace != nullptr && aligned16(a->workspace) &&
                   a->workspace_bytes >= uttt_readout4_workspace(a->batch, a->tokens, a->d_model, a->d_ff),
               "readout workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (b16)
    launch_readout4<bf16>(a, st);
  else
    launch_readout4<float>(a, st);
  return launch_status("uttt_readout4");
}
