// Next-token sampling of a decode step, written for gfx950 (MI355X): temperature, top-k, min-p and top-p with
// settings per row, from given uniform numbers; one launch, no sort.  The rules stand at uttt_sample_select.
//
// With w_i = 2^(c (x_i - max)), c = log2(e) / temperature, every rule keeps a prefix of the order (logit
// descending, id ascending), so the kept set is a cut (key, ties): the ids whose logit lies above the key's,
// and the first `ties` of those at it.  Passes over the row, one workgroup each:
//   1. the largest logit (rows that fit are kept in LDS for the passes behind);
//   2. the ids within 16 factors of two of the top (up to 24 where the row is flat, 43.5 where a top_k may lie there), listed
//      per stretch of the row (16, one per wave) so that their weights are formed with all lanes busy; their histogram of
//      counts and masses over x (2048 bins); and where top_p takes its share of it, the mass of the whole row, all of whose ids
//      are weighed for it.  When the cut lies further down, again over all ids whose weight is not 0;
//   3. the bin in which the count or the mass passes its bound: the stretches' masses ahead of it from the lists (where one
//      overflowed, from the row), and its ids, which are ranked against each other.  When they are many (equal or
//      nearly equal logits), the bin's range of keys is divided further first;
//   4. a scan of the list of the stretch that holds the chosen id, inside one wave.
// Without a cut 3 is a pass that weighs the whole row; without a list of the stretch (no cut, or many ids kept) 4 weighs
// 16 parts of it first.
//
// Bound by the arithmetic of the weights: some 25 instructions an id, 18 us a pass over 131072 of them on the one compute
// unit that has a row, beside 20 us to read it.  One row of 21478 bf16 takes 20 us (2.8 for pass 1, 10 for pass 2, 3 for 3),
// 256 rows of 131072 fp32 with mixed settings 117 to 164 us by their settings, the flattest of them (temperature 1.5, top_p
// near 1) last; all at temperature 0.7 and top_p 0.9 95 us.  Finding the cut's bin from counts alone, to weigh each id once, was
// slower (199 us for 150): it has to weigh every id with a bin again, not only those that may be kept.
//
// The sums decide between neighbouring ids, so weights are formed in 64 bits and added as integers in units of
// 2^-42 of the largest weight: exact whatever the order, so atomics in any order give equal bits.  (fp64 and
// unpacked fp32 arithmetic issue at the same rate here.)
#include <math.h>

#include <algorithm>

#include "../../include/uttt_serve.h"
#include "uttt_device.h"
#include "uttt_host.h"

namespace uttt {
namespace {

typedef unsigned long long u64;

struct SampleArgs {
  int vocab, limit;
  uint64_t low;  // excluded ids below 64, as a bit mask
  int n_high;    // excluded ids of 64 and above
  int high[8];
  const void* logits;
  int64_t rs;
  const float *uniforms, *temperature;
  const int32_t* top_k;
  const float *top_p, *min_p;
  int64_t* out;
  float* logprob;
  int64_t* advance;
};

constexpr int kSmpThreads = 1024, kSmpWaves = kSmpThreads / 64;
constexpr int kBins = 2 * kSmpThreads;  // two per thread in the scan
constexpr int kList = kSmpThreads;  // ids that are ranked against each other, one per thread
// Ids of each 64: from so many on they are weighed in place.  From 8, 24, 48 on: 256 x 131072 mixed 137, 133, 129 us (other
// settings 181, 163, 163), 64 x 50000 46.7, 46.3, 46.3.
constexpr int kDense = 24;
// Rows up to this size stay in LDS.  Staged and not: 1 x 21478 20.0 and 20.1 us, 64 x 30000 mixed 34.9 and 36.4.
constexpr int kStageBytes = 60 * 1024;
constexpr int kKeptStaged = 256, kKept = 512;

// order-preserving key of a logit that is not NaN; -0 and +0 are equal
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// 2^t for t <= 0 (0 for NaN) in units of 2^-42, to the nearest unit: 2^f, |f| <= 1/2, by its Taylor series to degree 10
// (2.2e-13 off at the ends), the whole part of t straight into the exponent
__device__ __forceinline__ u64 weight_units(double t) {
  t = __builtin_fmax(t, -60.0);  // far below half a unit
  const double kRound = 6755399441055744.0;  // 1.5 2^52: adding it leaves the nearest integer in the low bits
  const double shifted = t + kRound;
  const double f = t - (shifted - kRound);
  constexpr double kL = 0.6931471805599453, kL2 = kL * kL, kL4 = kL2 * kL2;
  double p = kL4 * kL4 * kL2 / 3628800;
  p = __builtin_fma(p, f, kL4 * kL4 * kL / 362880);
  p = __builtin_fma(p, f, kL4 * kL4 / 40320);
  p = __builtin_fma(p, f, kL4 * kL2 * kL / 5040);
  p = __builtin_fma(p, f, kL4 * kL2 / 720);
  p = __builtin_fma(p, f, kL4 * kL / 120);
  p = __builtin_fma(p, f, kL4 / 24);
  p = __builtin_fma(p, f, kL2 * kL / 6);
  p = __builtin_fma(p, f, kL2 / 2);
  p = __builtin_fma(p, f, kL);
  p = __builtin_fma(p, f, 1.0);
  const u64 scaled = __builtin_bit_cast(u64, p) + ((u64)(uint32_t)((int)__builtin_bit_cast(u64, shifted) + 42) << 52);
  // adding 2^52 rounds to whole units, which are then the low bits
  const double u = __builtin_bit_cast(double, scaled) + 4503599627370496.0;
  return __builtin_bit_cast(u64, u) & 0xfffffffffffffull;
}

// Sums over lanes through DPP operands: within rows of 16 lanes by shifts, then the rows' last lanes to the rows behind.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp0(uint32_t v) {  // 0 where the source lane does not exist
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp0(u64 v) {
  return (u64)dpp0<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | dpp0<CTRL, ROWS>((uint32_t)v);
}
template <typename V>
__device__ __forceinline__ V row_scan(V v) {  // inclusive, 16 lanes
  v += dpp0<0x111, 0xF>(v);
  v += dpp0<0x112, 0xF>(v);
  v += dpp0<0x114, 0xF>(v);
  return v + dpp0<0x118, 0xF>(v);
}
template <typename V>
__device__ __forceinline__ V wave_scan(V v) {  // inclusive, 64 lanes
  v = row_scan(v);
  v += dpp0<0x142, 0xA>(v);
  return v + dpp0<0x143, 0xC>(v);
}
__device__ __forceinline__ uint32_t of_lane(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ u64 of_lane(u64 v, int lane) {
  return (u64)of_lane((uint32_t)(v >> 32), lane) << 32 | of_lane((uint32_t)v, lane);
}

// A cut: ids with a larger key are kept, and the first `ties` of those with this key.
struct Cut {
  uint32_t key;
  int ties;
  u64 mass;  // of what it keeps
};

// kept: ids of one wave's stretch that are listed
template <int KEPT>
struct Shared {
  u64 mass[kBins];
  uint32_t count[kBins];
  u64 mass2[kBins];  // of a range of keys inside one bin
  uint32_t count2[kBins];
  float kept_logit[kSmpWaves][KEPT];  // the ids of a wave's stretch that have a bin, in their order
  int kept_id[kSmpWaves][KEPT];
  int kept_n[kSmpWaves];  // -1: the list holds only the last of them
  u64 wave_mass[kSmpWaves], scan_mass[kSmpWaves];
  uint32_t wave_count[kSmpWaves], scan_count[kSmpWaves];
  float wave_best[kSmpWaves], wave_sum[kSmpWaves];
  uint32_t list_key[kList];
  int list_id[kList];
  u64 list_mass[kList];
  uint32_t n, kmin, kmax, before_count;
  u64 before_mass;
  int bin, best;
  u64 kept;
  uint32_t cut_key;
  int cut_ties;
};

// ids that are left out, and those below 0, read as -inf
template <int VEC>
__device__ __forceinline__ void leave_out(const SampleArgs& a, float (&v)[VEC], int i) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    bool out = i + e < 64 && (i + e < 0 || ((a.low >> (i + e)) & 1));
    for (int k = 0; k < a.n_high; ++k) out |= i + e == a.high[k];
    v[e] = out ? -INFINITY : v[e];
  }
}

// f(values, first id) for places [lo, hi) of the row in order, VEC to a lane; U steps of 64 VEC in flight.  The id is the
// place less `off`.  What a step has past hi reads as -inf.
template <typename T, int VEC, int U, bool RAW, typename F>
__device__ __forceinline__ void scan_ids(const SampleArgs& a, const T* x, int off, int lo, int hi, int lane, F&& f) {
  typedef T vec_t __attribute__((ext_vector_type(VEC)));
#pragma unroll 1
  for (int b = lo; b < hi; b += 64 * VEC * U) {
    vec_t v[U];
    const bool whole = b + 64 * VEC * U <= hi;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = b + (u * 64 + lane) * VEC;
      if (whole || i + VEC <= hi) {
        v[u] = *reinterpret_cast<const vec_t*>(x + i);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[u][e] = i + e < hi ? x[i + e] : from_f32<T>(-INFINITY);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = b + (u * 64 + lane) * VEC - off;
      float y[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) y[e] = to_f32((T)v[u][e]);
      if (RAW && (b < 64 + off || a.n_high > 0)) leave_out<VEC>(a, y, i);
      f(y, i);
    }
  }
}

// STAGED: the row stays in LDS behind the first pass, without the ids that are left out.
template <typename T, bool STAGED>
__global__ void __launch_bounds__(kSmpThreads) k_sample_select(const SampleArgs a) {
  constexpr int KEPT = STAGED ? kKeptStaged : kKept, VEC = 16 / (int)sizeof(T);
  __shared__ Shared<KEPT> s;
  __shared__ __align__(16) T stage[STAGED ? kStageBytes / sizeof(T) : 1];
  constexpr int W = STAGED ? 8 / (int)sizeof(T) : VEC > 4 ? 4 : VEC;  // ids to a lane in the passes behind the first
  constexpr float kFarthest = 43.5f;  // factors of two below the top from where on weights are 0 units, half of 2^-42 not reached
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Places count from the 16-byte boundary at or before the row's first id, so that rows of any alignment are read in
  // whole 16-byte pieces (256 rows of 131071 fp32 at temperature 0.7: 43 us less than
  // one id at a time); ids from the place `off` on.
  const T* x = static_cast<const T*>(a.logits) + (int64_t)row * a.rs;
  const int off = __builtin_amdgcn_readfirstlane((int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)));
  const int places = a.limit + off;
  x -= off;
  // a wave's stretch of the row
  constexpr int kStep = 64;  // whole pieces; short rows still reach many waves
  const int stretch = ((places + kSmpWaves - 1) / kSmpWaves + kStep - 1) / kStep * kStep;
  const int lo = min(w * stretch, places), hi = min(lo + stretch, places);
  const float temp = a.temperature[row], uniform = a.uniforms[row];
  const int top_k = a.top_k != nullptr ? a.top_k[row] : 0;
  const float top_p = a.top_p != nullptr ? a.top_p[row] : 1.f, min_given = a.min_p != nullptr ? a.min_p[row] : 0.f;
  const float min_p = min_given > 0.f ? fminf(min_given, 1.f) : 0.f;  // NaN is off
  auto scan = [&](int from, int to, auto&& f) __attribute__((always_inline)) {
    if constexpr (STAGED)
      scan_ids<T, W, 1, false>(a, stage, off, from, to, lane, f);
    else
      scan_ids<T, W, 2, true>(a, x, off, from, to, lane, f);
  };

  // ---- the largest logit; NaN makes it NaN
  float top = -INFINITY, mean = 0.f;
  bool nan = false;
  scan_ids<T, VEC, 4, true>(a, x, off, lo, hi, lane, [&](const float(&v)[VEC], int i) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      top = fmaxf(top, v[e]);
      nan |= v[e] != v[e];
      mean += v[e] > -INFINITY ? v[e] : 0.f;
    }
    if constexpr (STAGED) {
      typedef T vec_t __attribute__((ext_vector_type(VEC)));
      vec_t y;
#pragma unroll
      for (int e = 0; e < VEC; ++e) y[e] = from_f32<T>(v[e]);
      if (i + off < hi) *reinterpret_cast<vec_t*>(stage + (i + off)) = y;  // past the last id: -inf
    }
  });
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    top = fmaxf(top, __shfl_xor(top, off, 64));
    mean += __shfl_xor(mean, off, 64);
  }
  if (__any(nan)) top = NAN;
  if (lane == 0) {
    s.wave_best[w] = top;
    s.wave_sum[w] = mean;
  }
  for (int i = tid; i < kBins; i += kSmpThreads) {
    s.mass[i] = 0;
    s.count[i] = 0;
  }
  if (tid == 0) s.best = 0x7fffffff;
  __syncthreads();
  top = -INFINITY;
  mean = 0.f;
  nan = false;
#pragma unroll 4
  for (int q = 0; q < kSmpWaves; ++q) {
    const float v = s.wave_best[q];
    nan |= v != v;
    top = fmaxf(top, v);
    mean += s.wave_sum[q];
  }
  const bool greedy = !(temp > 1e-5f);
  if (greedy || nan || !(fabsf(top) < INFINITY)) {  // the lowest id of the largest value (NaN above all)
    int best = 0x7fffffff;
    scan(lo, hi, [&](const float(&v)[W], int i) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < W; ++e)
        if (nan ? v[e] != v[e] : v[e] == top) best = min(best, i + e);
    });
    if (best != 0x7fffffff) atomicMin(&s.best, best);
    __syncthreads();
    if (tid == 0) {
      a.out[row] = s.best == 0x7fffffff ? 0 : max(s.best, 0);  // below 0 where all are -inf
      if (a.logprob != nullptr) a.logprob[row] = greedy ? 0.f : NAN;
      if (a.advance != nullptr) a.advance[row] += 1;
    }
    return;
  }

  const double c = 1.4426950408889634 / (double)temp, dtop = (double)top;
  const bool by_count = top_k > 0 && top_k < a.limit, by_mass = top_p < 1.f;
  const u64 least = min_p > 0.f ? (u64)__builtin_ceil((double)min_p * 4398046511104.0) : 1;
  auto weight = [&](float v) __attribute__((always_inline)) -> u64 {
    u64 u = weight_units(((double)v - dtop) * c);
    if (least > 1) u = u >= least ? u : 0;
    return u;
  };
  // The bins of the first round reach 16 factors of two down, in which a cut lies that most of the mass is ahead of; where
  // the row's mean is that near, so that much of the mass is around it, 4 past the mean; and 2/5 of the way to the mean
  // for top_k, whose ids may weigh next to nothing.  Reaching 16 always, rows whose cut lies further down take both
  // rounds: 256 x 131072 of deviation 3 at temperature 1.5 and top_p 0.99 230 us, for 154 so; with top_k 50 at temperature 0.2 87, for
  // 64 (64 x 32000 26.5, for 27.5).
  const float to_mean = (top - mean / (float)a.limit) * (float)c;
  float reach = to_mean < 20.f ? fmaxf(16.f, to_mean + 4.f) : 16.f;
  if (by_count && to_mean > 40.f) reach = fminf(0.4f * to_mean, kFarthest);
  // half the difference: a whole one may pass the type's largest number, where a high temperature still gives it weight
  float per_half = (float)c * (2.f * (float)kBins / reach);  // bins to two units of the logits
  const float half_top = 0.5f * top;
  auto place = [&](float v) __attribute__((always_inline)) { return __builtin_fmaf(v, -0.5f, half_top) * per_half; };

  Cut cut{0, 0x7fffffff, 0};  // keeps everything
  bool masses = false;        // the stretches' masses up to the cut are known
  int kept = 0;               // ids in this wave's list
  bool complete = false;      // it holds all it should
  u64 whole = 0;              // the row's mass; at the end the kept ids'
  if (by_count || by_mass) {
    // f(logits, first id, weights, which of them) for the ids of this wave's list, a lane each
    auto each_listed = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll 1
      for (int b = 0; b < kept; b += 64)
        if (b + lane < kept) {
          const float v[1] = {s.kept_logit[w][b + lane]};
          const u64 u[1] = {weight(v[0])};
          const bool in[1] = {true};
          f(v, s.kept_id[w][b + lane], u, in);
        }
    };
    // append the ids of a step that `in` marks to this wave's list, which f takes when they do not fit, and at the end; f
    // takes a step with many marked ids at once.  u: the step's weights, when it is `weighed`
    auto append = [&](const float(&v)[W], int i, const bool(&in)[W], bool weighed, u64(&u)[W], auto&& f) __attribute__((always_inline)) {
      uint32_t mine = 0;
      int more = 0;
#pragma unroll
      for (int e = 0; e < W; ++e) {
        mine += in[e];
        more += __popcll(__ballot(in[e]));
      }
      if (more == 0) return;
      if (more >= kDense * W) {
        if (!weighed) {
#pragma unroll
          for (int e = 0; e < W; ++e) u[e] = weight(v[e]);
        }
        f(v, i, u, in);
        complete = false;
        return;
      }
      const uint32_t upto = wave_scan(mine);
      if (kept + more > KEPT) {
        each_listed(f);
        kept = 0;
        complete = false;
      }
      int at = kept + (int)(upto - mine);
#pragma unroll
      for (int e = 0; e < W; ++e) {
        if (in[e]) {
          s.kept_logit[w][at] = v[e];
          s.kept_id[w][at] = i + e;
        }
        at += in[e];
      }
      kept += more;
    };
    // the same for all ids that have a bin: from the list when it is complete, else from the row
    auto each_binned = [&](auto&& f) __attribute__((always_inline)) {
      if (complete) {
        each_listed(f);
        return;
      }
      scan(lo, hi, [&](const float(&v)[W], int i) __attribute__((always_inline)) {
#pragma unroll 1
        for (int e = 0; e < W; ++e) {
          const float ve = e == 0 ? v[0] : e == 1 ? v[1 % W] : e == 2 ? v[2 % W] : v[3 % W];
          if (!(place(ve) < (float)kBins)) continue;
          const float v1[1] = {ve};
          const u64 u1[1] = {weight(ve)};
          const bool in1[1] = {true};
          f(v1, i + e, u1, in1);
        }
      });
    };
    // Counts and masses of the bins, and the whole mass.  Ids further down are a part of that (`tail`; else they have no weight,
    // min_p leaves them out, or top_p's share is not of them), so every id is weighed then.  fp32 exponentials for them were
    // faster (1 x 21478 16.5 us for 20, 256 x 131072 at temperature 0.7 77 for 95) and moved cuts.
    auto histogram = [&](bool tail) __attribute__((always_inline)) {
      u64 sum = 0;
      kept = 0;
      complete = true;
      auto count = [&](const auto& v, int, const auto& u, const auto& in) __attribute__((always_inline)) {
        constexpr int M = sizeof(v) / sizeof(float);
        if (by_mass) {
#pragma unroll
          for (int e = 0; e < M; ++e) {
            if (!tail) sum += in[e] ? u[e] : 0;
            if (in[e]) atomicAdd(&s.mass[(int)place(v[e])], u[e]);
          }
        }
        if (by_count) {
#pragma unroll
          for (int e = 0; e < M; ++e)
            if (in[e]) atomicAdd(&s.count[(int)place(v[e])], 1u);
        }
      };
      scan(lo, hi, [&](const float(&v)[W], int i) __attribute__((always_inline)) {
        bool in[W];
        u64 u[W];
#pragma unroll
        for (int e = 0; e < W; ++e) in[e] = place(v[e]) < (float)kBins;
        if (tail) {
#pragma unroll
          for (int e = 0; e < W; ++e) {
            u[e] = weight(v[e]);
            sum += u[e];
          }
        }
        append(v, i, in, tail, u, count);
      });
      each_listed(count);
      sum = wave_scan(sum);
      if (lane == 63) s.wave_mass[w] = sum;
      __syncthreads();
      whole = of_lane(row_scan(s.wave_mass[lane & 15]), 15);
    };
    // the bin with the last kept id (s.bin, -1: none), and what lies ahead of it: the bound-th id, or the last one
    // whose mass ahead is within the bound
    auto find = [&](const u64* mass, const uint32_t* count, u64 mass0, uint32_t count0, bool counts, u64 bound) __attribute__((always_inline)) {
      const u64 m0 = mass[2 * tid], m1 = mass[2 * tid + 1];
      const uint32_t n0 = count[2 * tid], n1 = count[2 * tid + 1];
      u64 m = wave_scan(m0 + m1);
      uint32_t n = wave_scan(n0 + n1);
      if (lane == 63) {
        s.scan_mass[w] = m;
        s.scan_count[w] = n;
      }
      if (tid == 0) s.bin = -1;
      __syncthreads();
      m -= m0 + m1;
      n -= n0 + n1;
      if (w > 0) {
        m += of_lane(row_scan(s.scan_mass[lane & 15]), w - 1);
        n += of_lane(row_scan(s.scan_count[lane & 15]), w - 1);
      }
      m += mass0;
      n += count0;
      const bool in0 = counts ? n < bound && bound <= n + n0 : m <= bound && bound < m + m0;
      const bool in1 = counts ? n + n0 < bound && bound <= n + n0 + n1 : m + m0 <= bound && bound < m + m0 + m1;
      if (in0 || in1) {
        s.bin = 2 * tid + (in0 ? 0 : 1);
        s.before_mass = in0 ? m : m + m0;
        s.before_count = in0 ? n : n + n0;
      }
      __syncthreads();
      const int bin = s.bin;
      __syncthreads();
      return bin;
    };
    auto add_to_list = [&](uint32_t k, int id, u64 u) __attribute__((always_inline)) {
      const uint32_t at = atomicAdd(&s.n, 1u);
      if (at < kList) {
        s.list_key[at] = k;
        s.list_id[at] = id;
        s.list_mass[at] = u;
      }
    };
    auto start_list = [&]() __attribute__((always_inline)) {
      if (tid == 0) {
        s.n = 0;
        s.kmin = 0xffffffffu;
        s.kmax = 0;
      }
      __syncthreads();
    };
    auto end_list = [&](uint32_t mn, uint32_t mx) __attribute__((always_inline)) {
      if (mn <= mx) {
        atomicMin(&s.kmin, mn);
        atomicMax(&s.kmax, mx);
      }
      __syncthreads();
    };
    // the ids of one bin with keys in [kmin, kmax]: how many, the first kList, the range of their keys
    auto gather = [&](int bin, uint32_t kmin, uint32_t kmax) __attribute__((always_inline)) {
      start_list();
      uint32_t mn = 0xffffffffu, mx = 0;
      each_binned([&](const float(&v)[1], int i, const u64(&u)[1], const bool(&)[1]) __attribute__((always_inline)) {
        const float d = place(v[0]);
        if (!(d >= (float)bin && d < (float)(bin + 1))) return;
        const uint32_t k = key_of(v[0]);
        if (k < kmin || k > kmax) return;
        mn = min(mn, k);
        mx = max(mx, k);
        add_to_list(k, i, u[0]);
      });
      end_list(mn, mx);
    };
    // the same for a whole bin, and per stretch the mass of the bins ahead
    auto collect = [&](int bin) __attribute__((always_inline)) {
      start_list();
      uint32_t mn = 0xffffffffu, mx = 0;
      u64 sum = 0;
      auto weigh = [&](const auto& v, int i, const auto& u, const auto& in) __attribute__((always_inline)) {
        constexpr int M = sizeof(v) / sizeof(float);
        bool here = false, at[M];
#pragma unroll
        for (int e = 0; e < M; ++e) {
          const float d = place(v[e]);
          sum += in[e] && d < (float)bin ? u[e] : 0;
          at[e] = in[e] && d >= (float)bin && d < (float)(bin + 1);
          here |= at[e];
        }
        if (!here) return;
#pragma unroll
        for (int e = 0; e < M; ++e) {
          if (!at[e]) continue;
          const uint32_t k = key_of(v[e]);
          mn = min(mn, k);
          mx = max(mx, k);
          add_to_list(k, i + e, u[e]);
        }
      };
      if (!complete) {  // list again, now only what may be kept
        kept = 0;
        complete = true;
        scan(lo, hi, [&](const float(&v)[W], int i) __attribute__((always_inline)) {
          bool in[W];
          u64 u[W];
#pragma unroll
          for (int e = 0; e < W; ++e) in[e] = place(v[e]) < (float)(bin + 1);
          append(v, i, in, false, u, weigh);
        });
      }
      each_listed(weigh);
      sum = wave_scan(sum);
      if (lane == 63) {
        s.wave_mass[w] = sum;
        s.wave_count[w] = 0;
        s.kept_n[w] = complete ? kept : -1;
      }
      end_list(mn, mx);
    };
    // the cut inside a bin that find() named
    auto resolve = [&](int bin, bool counts, u64 bound, bool ahead) __attribute__((always_inline)) -> Cut {
      u64 mass0 = s.before_mass;
      uint32_t count0 = s.before_count;
      if (ahead)
        collect(bin);
      else
        gather(bin, 0, 0xffffffffu);
      masses = ahead && s.n <= kList;
      uint32_t kmin = s.kmin, kmax = s.kmax;
      while (s.n > kList && kmin != kmax) {
        const int shift = max(0, 32 - 11 - __builtin_clz(kmax - kmin));
        for (int i = tid; i < kBins; i += kSmpThreads) {
          s.mass2[i] = 0;
          s.count2[i] = 0;
        }
        __syncthreads();
        each_binned([&](const float(&v)[1], int, const u64(&u)[1], const bool(&)[1]) __attribute__((always_inline)) {
          const float d = place(v[0]);
          if (!(d >= (float)bin && d < (float)(bin + 1))) return;
          const uint32_t k = key_of(v[0]);
          if (k < kmin || k > kmax) return;
          const int b = (int)((kmax - k) >> shift);
          atomicAdd(&s.mass2[b], u[0]);
          atomicAdd(&s.count2[b], 1u);
        });
        __syncthreads();
        const int part = find(s.mass2, s.count2, mass0, count0, counts, bound);
        if (part < 0) break;  // the bound lies inside the bin, so one of its parts has it
        mass0 = s.before_mass;
        count0 = s.before_count;
        const uint32_t hi_key = kmax - ((uint32_t)part << shift), width = (1u << shift) - 1;
        const uint32_t lo_key = hi_key - kmin > width ? hi_key - width : kmin;
        gather(bin, lo_key, hi_key);
        kmin = s.kmin;
        kmax = s.kmax;
      }
      Cut r;
      const int n = (int)min(s.n, (uint32_t)kList);
      if (kmin == kmax) {  // equal logits: a number of them
        const u64 u = weight(of_key(kmin));
        const u64 all = s.n;
        u64 t = counts ? bound - count0 : u != 0 ? (bound - mass0) / u + 1 : all;
        t = t < all ? t : all;
        r.key = kmin;
        r.ties = (int)t;
        r.mass = mass0 + t * u;
      } else {
        if (tid == 0) {
          s.kept = 0;
          s.cut_key = 0xffffffffu;
          s.cut_ties = 0;
        }
        __syncthreads();
        bool keep = false;
        uint32_t k = 0;
        if (tid < n) {
          k = s.list_key[tid];
          const int id = s.list_id[tid];
          u64 m = mass0;
          uint32_t cnt = count0;
#pragma unroll 4
          for (int j = 0; j < n; ++j) {
            const uint32_t kj = s.list_key[j];
            if (kj > k || (kj == k && s.list_id[j] < id)) {
              m += s.list_mass[j];
              ++cnt;
            }
          }
          keep = counts ? cnt < bound : m <= bound;
          if (keep) {
            atomicAdd(&s.kept, s.list_mass[tid]);
            atomicMin(&s.cut_key, k);
          }
        }
        __syncthreads();
        if (keep && k == s.cut_key) atomicAdd(&s.cut_ties, 1);
        __syncthreads();
        r.key = s.cut_key;
        r.ties = s.cut_ties;
        r.mass = mass0 + s.kept;
      }
      if (masses && tid < n) {  // the bin's own part of the stretches' masses, and its ids at the cut
        const int q = (s.list_id[tid] + off) / stretch;
        if (s.list_key[tid] > r.key) atomicAdd(&s.wave_mass[q], s.list_mass[tid]);
        if (s.list_key[tid] == r.key) atomicAdd(&s.wave_count[q], 1u);
      }
      __syncthreads();
      return r;
    };
#pragma unroll 1
    for (int round = 0; round < 2; ++round) {
      // ids without a bin lie 16 factors of two down or more: they weigh at most 2^26 units
      histogram(by_mass && !by_count && round == 0 && least <= 1ull << 27);
      u64 bound = (u64)((double)fmaxf(top_p, 0.f) * (double)whole);  // top_p of the row's mass
      bool found = true;
      if (by_count) {
        const int bin = find(s.mass, s.count, 0, 0, true, (u64)top_k);
        if (bin >= 0) {
          cut = resolve(bin, true, (u64)top_k, !by_mass);
          bound = (u64)((double)fmaxf(top_p, 0.f) * (double)cut.mass);  // or of what top_k keeps
        } else {
          found = false;  // it lies further down, or among ids of weight 0, or there are fewer ids than top_k
        }
      }
      if (by_mass && (found || round == 1)) {
        const int bin = find(s.mass, s.count, 0, 0, false, bound);
        found = bin >= 0;
        if (found) {
          const Cut p = resolve(bin, false, bound, true);
          if (p.key > cut.key || (p.key == cut.key && p.ties < cut.ties))
            cut = p;
          else
            masses = false;
        }
      }
      if (found || round == 1) break;
      per_half = (float)c * (2.f * (float)kBins / kFarthest);
      __syncthreads();
      for (int i = tid; i < kBins; i += kSmpThreads) {
        s.mass[i] = 0;
        s.count[i] = 0;
      }
      __syncthreads();
    }
  }

  // ---- the kept mass of parts [lo, hi) of the row, one per wave: above the cut's key, and ids at it
  const float at_cut = cut.key != 0 ? of_key(cut.key) : -INFINITY;
  const u64 tie_mass = cut.key != 0 ? weight(at_cut) : 0;
  auto part_mass = [&](int p_lo, int p_hi) __attribute__((always_inline)) {
    u64 m = 0;
    uint32_t t = 0;
    scan(p_lo, p_hi, [&](const float(&v)[W], int) __attribute__((always_inline)) {
      float most = v[0];
#pragma unroll
      for (int e = 1; e < W; ++e) most = fmaxf(most, v[e]);
      if (!(most >= at_cut)) return;
      u64 u[W];
#pragma unroll
      for (int e = 0; e < W; ++e) u[e] = weight(v[e]);
#pragma unroll
      for (int e = 0; e < W; ++e) {
        m += v[e] > at_cut ? u[e] : 0;
        t += v[e] == at_cut;
      }
    });
    m = wave_scan(m);
    t = wave_scan(t);
    __syncthreads();
    if (lane == 63) {
      s.wave_mass[w] = m;
      s.wave_count[w] = t;
    }
    __syncthreads();
  };
  const u64 max_ties = (u64)cut.ties;
  auto with_ties = [&](u64 ties, u64 more) __attribute__((always_inline)) {  // mass of `more` ids at the cut's key behind `ties` of them
    const u64 left = ties < max_ties ? max_ties - ties : 0;
    return (more < left ? more : left) * tie_mass;
  };
  if (!masses) part_mass(lo, hi);
  const float uf = uniform > 0.f ? fminf(uniform, 0.99999994f) : 0.f;
  u64 want = 0, ahead = 0, ties_ahead = 0;
  // the part whose mass first exceeds `want`, and the mass and ties ahead of it; lane q of a row of 16 has part q
  auto pick = [&](bool first) __attribute__((always_inline)) {
    const u64 mine = s.wave_mass[lane & 15], t = s.wave_count[lane & 15];
    const u64 t_end = ties_ahead + row_scan(t);
    const u64 m_end = ahead + row_scan(mine + with_ties(t_end - t, t));
    if (first) {
      const u64 total = of_lane(m_end, 15);
      want = (u64)((double)uf * (double)total);
      want = want < total ? want : total - 1;
      whole = total;
    }
    const uint32_t over = (uint32_t)__ballot(m_end > want) & 0xffffu;
    const int found = over != 0 ? __builtin_ctz(over) : 15;
    if (found > 0) {
      ahead = of_lane(m_end, found - 1);
      ties_ahead = of_lane(t_end, found - 1);
    }
    return found;
  };
  const int q = pick(true);
  int q0 = 0, q1 = masses ? s.kept_n[q] : -1;
  const bool listed = q1 >= 0;
  if (!listed) {
    const int p0 = min(q * stretch, places), p1 = min(p0 + stretch, places);
    const int part = ((p1 - p0 + kSmpWaves - 1) / kSmpWaves + kStep - 1) / kStep * kStep;
    const int q_lo = min(p0 + w * part, p1);
    part_mass(q_lo, min(q_lo + part, p1));
    q0 = min(p0 + pick(false) * part, p1);
    q1 = min(q0 + part, p1);
  }
  if (w != 0) return;
  // ---- inside one wave: 64 ids at a time, of the stretch's list or of a part of the row
  u64 m = ahead, t = ties_ahead;
  int token = -1;
#pragma unroll 1
  for (int b = q0; b < q1 && token < 0; b += 64) {
    const int i = b + lane;
    float v[1] = {-INFINITY};
    if (i < q1) {
      if (listed) {
        v[0] = s.kept_logit[q][i];
      } else if constexpr (STAGED) {
        v[0] = to_f32(stage[i]);
      } else {
        v[0] = to_f32(x[i]);
        leave_out<1>(a, v, i - off);
      }
    }
    u64 u = v[0] > at_cut ? weight(v[0]) : 0;
    const bool tie = v[0] == at_cut && tie_mass != 0;
    const u64 tied = __ballot(tie);
    if (tie) u = t + __popcll(tied & ((1ull << lane) - 1)) < max_ties ? tie_mass : 0;
    const u64 sum = wave_scan(u);
    const u64 over = __ballot(m + sum > want);
    if (over != 0) {
      token = b + __builtin_ctzll(over);
      token = listed ? s.kept_id[q][token] : token - off;
    }
    m += of_lane(sum, 63);
    t += __popcll(tied);
  }
  if (lane == 0) {
    token = token < 0 ? 0 : token;  // integers add up the same way at every level, so one is found
    a.out[row] = token;
    // log(w / total): the weight's own exponent, not its rounded units
    float divisor = temp;
    asm volatile("" : "+v"(divisor));  // its 64-bit form is made here, not kept in registers through the passes
    if (a.logprob != nullptr)
      a.logprob[row] = (float)(((double)to_f32(x[token + off]) - dtop) / (double)divisor - log((double)whole * 0x1p-42));
    if (a.advance != nullptr) a.advance[row] += 1;
  }
}

template <typename T>
void launch_sample(const SampleArgs& s, int64_t rows, hipStream_t st) {
  const dim3 grid((unsigned)rows), block(kSmpThreads);
  if ((int64_t)s.limit * (int64_t)sizeof(T) <= kStageBytes - 16)
    hipLaunchKernelGGL((k_sample_select<T, true>), grid, block, 0, st, s);
  else
    hipLaunchKernelGGL((k_sample_select<T, false>), grid, block, 0, st, s);
}

}  // namespace
}  // namespace uttt

using namespace uttt;

extern "C" int uttt_serve_abi_version(void) { return UTTT_SERVE_ABI_VERSION; }

extern "C" int uttt_sample_select(const uttt_sample_args* a, uttt_stream_t stream) {
  UTTT_REQUIRE(a != nullptr, "args is NULL");
  UTTT_REQUIRE(a->rows >= 1 && a->rows <= 65535, "rows must be in [1, 65535]");
  UTTT_REQUIRE(a->vocab >= 1 && a->vocab <= (1LL << 20), "vocab must be in [1, 2^20]");
  UTTT_REQUIRE(a->dtype == UTTT_DTYPE_BF16 || a->dtype == UTTT_DTYPE_F32, "logits must be bf16 or fp32");
  UTTT_REQUIRE(a->n_banned >= 0 && a->n_banned <= 8, "at most 8 excluded ids");
  for (int k = 0; k < a->n_banned; ++k) UTTT_REQUIRE(a->banned[k] >= 0, "excluded ids must be >= 0");
  UTTT_REQUIRE(a->logits != nullptr && a->out != nullptr && a->uniforms != nullptr && a->temperature != nullptr,
               "logits, uniforms, temperature and out must be non-NULL");
  UTTT_REQUIRE(a->row_stride >= a->vocab || a->row_stride == 0, "the row stride must cover vocab, or be 0 for one row for all");
  SampleArgs s{};
  s.vocab = (int)a->vocab;
  for (int k = 0; k < a->n_banned; ++k) {
    if (a->banned[k] < 64)
      s.low |= uint64_t(1) << a->banned[k];
    else
      s.high[s.n_high++] = a->banned[k];
  }
  s.limit = (int)std::min<int64_t>(a->active_limit < 0 ? a->vocab : a->active_limit, a->vocab);
  s.logits = a->logits; s.rs = a->row_stride;
  s.uniforms = a->uniforms; s.temperature = a->temperature;
  s.top_k = a->top_k; s.top_p = a->top_p; s.min_p = a->min_p;
  s.out = a->out; s.logprob = a->logprob; s.advance = a->advance;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->dtype == UTTT_DTYPE_BF16)
    launch_sample<bf16>(s, a->rows, st);
  else
    launch_sample<float>(s, a->rows, st);
  return launch_status("uttt_sample_select");
}
