// Beam search's choice, written for gfx950 (MI355X): the `beams` best continuations of every group of beams.
//
// value(b, v) = score_b + (x_bv - max_b) - log sum_v exp(x_bv - max_b), formed in 64 bits from logits in their own
// precision, so that the order of candidates of different beams is the definition's; the exponentials are fp32 ones (their
// errors average out far below what separates two beams), their sums 64-bit ones.
//
// Within a row the order is that of (logit, id), so the first launch, a workgroup per stretch of a row with the stretch in
// registers, finds each stretch's maximum, sum and `beams` best by (logit, id) alone.  No sort: the beams-th largest of a
// wave's 64 lane maxima, found bit by bit with ballots, is a bound that at least `beams` elements reach; the few that
// reach the largest bound of the waves are listed in LDS and ranked against each other.  The second launch, a workgroup per
// group, does the same with the stretches' best and their values.
#include <algorithm>

#include "../../include/uttt_decode.h"
#include "uttt_device.h"
#include "uttt_host.h"

namespace uttt {
namespace {

constexpr int kMaxBeams = 32;
constexpr int kPer = 16;                     // elements of a thread
constexpr int kStretch = kThreads * kPer;    // of a workgroup
constexpr int kListed = 1024;                // elements at the bound that LDS holds; more (equal logits) are chosen one by one
constexpr int kMergeThreads = 1024;

struct BeamArgs {
  int rows, beams, splits, n_banned;
  int64_t vocab, limit;
  int banned[8];
  const void* logits;
  int64_t row_stride;
  const float* scores;
  const int32_t* ended_in;
  int64_t eos, pad;
  int64_t* tokens;
  int32_t* sources;
  float* out_scores;
  int32_t* ended_out;
  double* sums;      // (rows, splits)
  uint64_t* best;    // (rows, splits, beams): ordered logit above, ~id below; 0: none
  float* tops;       // (rows, splits)
};

// Floats in the order of unsigned integers (NaN apart), and back.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t ordered(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  return u >> 63 ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ double unordered(uint64_t k) {
  return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k));
}

// The largest key that at least `want` lanes reach.
__device__ __forceinline__ uint32_t reached_by(uint32_t key, int want) {
  uint32_t t = 0;
#pragma unroll
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t next = t | 1u << bit;
    if (__popcll(__ballot(key >= next)) >= want) t = next;
  }
  return t;
}

__device__ __forceinline__ uint64_t wave_max64(uint64_t x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint64_t y = (uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)x, off, 64) |
                       (uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)(x >> 32), off, 64) << 32;
    x = x > y ? x : y;
  }
  return x;
}

// Grid (stretches, rows).
template <typename T>
__global__ void __launch_bounds__(kThreads) k_beam_part(const BeamArgs a) {
  constexpr int kVec = Lanes16<T>::kVec;
  __shared__ uint64_t list[kListed];
  __shared__ uint64_t wide[kThreads / 64];
  __shared__ float tops[kThreads / 64];
  __shared__ double sums[kThreads / 64];
  __shared__ uint32_t bounds[kThreads / 64];
  __shared__ int listed;
  const int row = blockIdx.y, split = blockIdx.x, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (a.ended_in != nullptr && a.ended_in[row] != 0) return;  // its one continuation needs no logit
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  const int64_t base = (int64_t)split * kStretch;
  const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  float v[kPer];
  // element j of a thread is id base + at(j); 16-byte pieces where the row allows them, single ones otherwise
  auto at = [&](int j) {
    return aligned ? ((j / kVec) * kThreads + (int)threadIdx.x) * kVec + j % kVec : j * kThreads + (int)threadIdx.x;
  };
  if (aligned && base + kStretch <= a.vocab) {
    uint4 piece[kPer / kVec];
#pragma unroll
    for (int c = 0; c < kPer / kVec; ++c) piece[c] = *reinterpret_cast<const uint4*>(x + base + at(c * kVec));
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = Lanes16<T>::get(piece[j / kVec], j % kVec);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = base + at(j) < a.vocab ? to_f32(x[base + at(j)]) : -INFINITY;
  }
  if (threadIdx.x == 0) listed = 0;
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int64_t id = base + at(j);
    bool out = id >= a.limit;
    for (int i = 0; i < a.n_banned; ++i) out |= id == a.banned[i];
    v[j] = out ? -INFINITY : v[j] + 0.f;  // -0 is 0: the order is the values'
    top = fmaxf(top, v[j]);
  }
  const uint32_t mine = reached_by(ordered(top), a.beams);
  const float wave_top = wave_max(top);
  if (lane == 0) {
    bounds[w] = mine;
    tops[w] = wave_top;
  }
  __syncthreads();
  const uint32_t bound = max(max(bounds[0], bounds[1]), max(bounds[2], bounds[3]));
  const float all = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  double sum = 0.0;
  const uint32_t none = ordered(-INFINITY);
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    sum += (double)(v[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((v[j] - all) * 1.44269504088896340736f));
    const uint32_t k = ordered(v[j]);
    if (k >= bound && k > none) {
      const int i = atomicAdd(&listed, 1);
      if (i < kListed) list[i] = (uint64_t)k << 32 | (uint32_t)~(uint32_t)(base + at(j));
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if (lane == 0) sums[w] = sum;
  __syncthreads();
  const int64_t part = (int64_t)row * a.splits + split;
  if (threadIdx.x == 0) {
    a.sums[part] = sums[0] + sums[1] + sums[2] + sums[3];
    a.tops[part] = all;
  }
  uint64_t* best = a.best + part * a.beams;
  const int n = listed;
  if (n <= kListed) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint64_t k = list[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += list[j] > k;
      if (rank < a.beams) best[rank] = k;
    }
    for (int i = n + threadIdx.x; i < a.beams; i += kThreads) best[i] = 0;
    return;
  }
  uint64_t last = ~0ull;
  for (int i = 0; i < a.beams; ++i) {  // the best below the last one
    uint64_t found = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const uint64_t k = (uint64_t)ordered(v[j]) << 32 | (uint32_t)~(uint32_t)(base + at(j));
      if (v[j] > -INFINITY && k < last && k > found) found = k;
    }
    found = wave_max64(found);
    if (lane == 0) wide[w] = found;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kThreads / 64; ++j) found = found > wide[j] ? found : wide[j];
    if (threadIdx.x == 0) best[i] = found;
    last = found;
    __syncthreads();
  }
}

// Candidates are ordered by their values, of equal ones by the place of (beam, id) in the group.
__device__ __forceinline__ bool better(uint64_t v, uint32_t p, uint64_t w, uint32_t q) { return v > w || (v == w && p < q); }

// Grid (groups).
__global__ void __launch_bounds__(kMergeThreads) k_beam_merge(const BeamArgs a) {
  constexpr int kWaves = kMergeThreads / 64;
  __shared__ uint64_t values[kListed];
  __shared__ uint32_t places[kListed];
  __shared__ double add[kMaxBeams];  // score_b - log sum_b
  __shared__ float tops[kMaxBeams];
  __shared__ int kind[kMaxBeams];  // 0: offers none, 1: its ids, 2: ended
  __shared__ uint32_t bounds[kWaves];
  __shared__ uint64_t wide_v[kWaves];
  __shared__ uint32_t wide_p[kWaves];
  __shared__ int listed;
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int row0 = blockIdx.x * a.beams;
  if (threadIdx.x == 0) listed = 0;
  for (int b = w; b < a.beams; b += kWaves) {
    const int row = row0 + b;
    const float score = a.scores[row];
    const bool over = a.ended_in != nullptr && a.ended_in[row] != 0;
    float top = -INFINITY;
    double sum = 0.0;
    if (!over) {
      for (int s = lane; s < a.splits; s += 64) top = fmaxf(top, a.tops[(int64_t)row * a.splits + s]);
      top = wave_max(top);
      for (int s = lane; s < a.splits; s += 64) {
        const float t = a.tops[(int64_t)row * a.splits + s];
        const double part = a.sums[(int64_t)row * a.splits + s];
        // NaN sums stay NaN: a row with NaN offers nothing
        sum += t == -INFINITY ? part : part * exp((double)t - (double)top);
      }
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    }
    if (lane == 0) {
      const bool finite = fabsf(score) < INFINITY;
      kind[b] = !finite ? 0 : over ? 2 : fabsf(top) < INFINITY && sum > 0.0 && sum < (double)INFINITY ? 1 : 0;
      tops[b] = top;
      add[b] = over ? (double)score + 0.0 : (double)score - log(sum);
    }
  }
  __syncthreads();
  const int per = a.splits * a.beams, total = a.beams * per;
  // candidate i: its key and place; 0: none
  auto look = [&](int i, uint32_t& place) -> uint64_t {
    const int b = i / per, j = i - b * per;
    place = ~0u;
    if (kind[b] == 0) return 0;
    if (kind[b] == 2) {
      place = (uint32_t)(b * a.vocab + a.pad);
      return j == 0 ? ordered(add[b]) : 0;
    }
    const uint64_t k = a.best[(int64_t)(row0 + b) * per + j];
    if (k == 0) return 0;
    place = (uint32_t)(b * a.vocab) + (uint32_t)~(uint32_t)k;
    return ordered(((double)unordered((uint32_t)(k >> 32)) - (double)tops[b]) + add[b]);
  };
  uint32_t high = 0, place;
  for (int i = threadIdx.x; i < total; i += kMergeThreads) high = max(high, (uint32_t)(look(i, place) >> 32));
  const uint32_t mine = reached_by(high, a.beams);
  if (lane == 0) bounds[w] = mine;
  __syncthreads();
  uint32_t bound = 0;
#pragma unroll
  for (int j = 0; j < kWaves; ++j) bound = max(bound, bounds[j]);
  for (int i = threadIdx.x; i < total; i += kMergeThreads) {
    const uint64_t v = look(i, place);
    if (v != 0 && (uint32_t)(v >> 32) >= bound) {
      const int to = atomicAdd(&listed, 1);
      if (to < kListed) {
        values[to] = v;
        places[to] = place;
      }
    }
  }
  __syncthreads();
  const int n = listed;
  auto emit = [&](int rank, uint64_t v, uint32_t p) {
    const int b = (int)(p / a.vocab);
    const int64_t token = p - b * a.vocab;
    a.tokens[row0 + rank] = token;
    a.sources[row0 + rank] = row0 + b;
    a.out_scores[row0 + rank] = (float)unordered(v);
    if (a.ended_out) a.ended_out[row0 + rank] = kind[b] == 2 || token == a.eos;
  };
  int found = 0;
  if (n <= kListed) {
    for (int i = threadIdx.x; i < n; i += kMergeThreads) {
      const uint64_t v = values[i];
      const uint32_t p = places[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += better(values[j], places[j], v, p);
      if (rank < a.beams) emit(rank, v, p);
    }
    found = min(n, a.beams);
  } else {
    uint64_t last_v = ~0ull;
    uint32_t last_p = 0;
    for (; found < a.beams; ++found) {  // the best behind the last one
      uint64_t v = 0;
      uint32_t p = ~0u;
      for (int i = threadIdx.x; i < total; i += kMergeThreads) {
        const uint64_t c = look(i, place);
        if (c != 0 && better(last_v, last_p, c, place) && better(c, place, v, p)) {
          v = c;
          p = place;
        }
      }
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) {
        const uint64_t ov = (uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)v, off, 64) |
                            (uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)(v >> 32), off, 64) << 32;
        const uint32_t op = (uint32_t)__shfl_xor((int)p, off, 64);
        if (better(ov, op, v, p)) {
          v = ov;
          p = op;
        }
      }
      if (lane == 0) {
        wide_v[w] = v;
        wide_p[w] = p;
      }
      __syncthreads();
      for (int j = 0; j < kWaves; ++j)
        if (better(wide_v[j], wide_p[j], v, p)) {
          v = wide_v[j];
          p = wide_p[j];
        }
      if (threadIdx.x == 0) emit(found, v, p);  // more than kListed candidates: there are enough
      last_v = v;
      last_p = p;
      __syncthreads();
    }
  }
  for (int i = found + threadIdx.x; i < a.beams; i += kMergeThreads) {
    a.tokens[row0 + i] = a.pad;
    a.sources[row0 + i] = row0 + i;
    a.out_scores[row0 + i] = -INFINITY;
    if (a.ended_out) a.ended_out[row0 + i] = 1;
  }
}

int64_t stretches(int64_t vocab) { return (vocab + kStretch - 1) / kStretch; }

}  // namespace
}  // namespace uttt

using namespace uttt;

extern "C" size_t uttt_beam_select_workspace(int64_t rows, int64_t vocab, int64_t beams) {
  if (rows < 1 || vocab < 1 || beams < 1) return 0;
  return (size_t)rows * (size_t)stretches(vocab) * (8 * (size_t)beams + 8 + 4);
}

extern "C" int uttt_beam_select(const uttt_beam_select_args* a, uttt_stream_t stream) {
  UTTT_REQUIRE(a != nullptr, "args is NULL");
  UTTT_REQUIRE(a->dtype == UTTT_DTYPE_F32 || a->dtype == UTTT_DTYPE_BF16, "bad dtype");
  UTTT_REQUIRE(a->beams >= 1 && a->beams <= kMaxBeams, "beams must be in [1, %d]", kMaxBeams);
  UTTT_REQUIRE(a->rows >= 1 && a->rows <= 65535 && a->rows % a->beams == 0,
               "rows must be a multiple of beams in [1, 65535] (got %lld)", (long long)a->rows);
  UTTT_REQUIRE(a->vocab >= 1 && a->vocab <= (1 << 20), "vocab must be in [1, 2^20]");
  UTTT_REQUIRE(a->n_banned >= 0 && a->n_banned <= 8, "at most 8 excluded ids");
  UTTT_REQUIRE(a->pad >= 0 && a->pad < a->vocab, "pad must be an id of the vocabulary");
  UTTT_REQUIRE(a->logits && a->scores && a->tokens && a->sources && a->out_scores, "pointers must be non-NULL");
  UTTT_REQUIRE(a->rows == 1 || a->row_stride >= a->vocab, "the row stride must cover the vocabulary");
  UTTT_REQUIRE(a->workspace != nullptr && aligned16(a->workspace) &&
                   a->workspace_bytes >= uttt_beam_select_workspace(a->rows, a->vocab, a->beams),
               "beam workspace too small");
  BeamArgs m{};
  m.rows = (int)a->rows; m.beams = (int)a->beams; m.n_banned = a->n_banned;
  m.vocab = a->vocab;
  m.limit = a->active_limit < 0 ? a->vocab : std::min(a->active_limit, a->vocab);
  m.splits = (int)std::max<int64_t>(1, stretches(m.limit));
  for (int i = 0; i < 8; ++i) m.banned[i] = a->banned[i];
  m.logits = a->logits; m.row_stride = a->row_stride;
  m.scores = a->scores; m.ended_in = a->ended_in;
  m.eos = a->eos; m.pad = a->pad;
  m.tokens = a->tokens; m.sources = a->sources; m.out_scores = a->out_scores; m.ended_out = a->ended_out;
  m.best = static_cast<uint64_t*>(a->workspace);
  m.sums = reinterpret_cast<double*>(m.best + (int64_t)m.rows * m.splits * m.beams);
  m.tops = reinterpret_cast<float*>(m.sums + (int64_t)m.rows * m.splits);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)m.splits, (unsigned)m.rows);
  if (a->dtype == UTTT_DTYPE_BF16)
    hipLaunchKernelGGL(k_beam_part<bf16>, grid, dim3(kThreads), 0, st, m);
  else
    hipLaunchKernelGGL(k_beam_part<float>, grid, dim3(kThreads), 0, st, m);
  hipLaunchKernelGGL(k_beam_merge, dim3((unsigned)(m.rows / m.beams)), dim3(kMergeThreads), 0, st, m);
  return launch_status("uttt_beam_select");
}
