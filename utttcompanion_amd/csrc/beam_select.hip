// Beam search's choice, written for gfx950 (MI355X): the `beams` best continuations of every group of beams.
//
// value(b, v) = score_b + (x_bv - max_b) - log sum_v exp(x_bv - max_b), formed in 64 bits from logits in their own precision and
// the row's sum.  Within a row the order is exact.  Between rows it is the definition's where two values differ by more than the
// sums' errors: exponentials are fp32 ones of fp32 differences, added up by sixteens in fp32 and from there on in 64
// bits.  A term is off by 2^-24 (2.25 d + 2) of itself, d its distance from the top (difference, product with log2 e,
// exponential; log(vocab) at most on average), sixteen of them by 2^-20, and a thread's sum by up to 2^-23 more each time its top
// moves: 2^-15 at most, where logits rise all through a row of 2^20, and 2^-23 where they are as random as a model's.
//
// Within a row the order is that of (logit, id), so the first launch, a workgroup per part of a row, finds each part's maximum,
// sum and `beams` best by (logit, id) alone.  No sort: the beams-th largest of a wave's 64 lane maxima, found bit by bit
// with ballots, is a bound that at least `beams` elements reach; the few that reach it are listed in LDS and, at the end,
// ranked against each other.  16 x 16 rows of 131072 fp32 ids take 24 to 26 us, what reading them takes (5.2 TB/s).  Rows off 16
// bytes, and a row's last stretch, are read element by element: both launches 60 us at 16 x 16 x 131073 bf16 ids, 31 at 131072 (fp32
// 38 and 35; 16 x 4 of 50001 13.7 and 12.4).
// The second launch, a workgroup per group, does the same with the parts' best and their values: 5 to 8 us of latency, some
// 30 more for many beams whose scores lie far apart (one group of 32 of 131072 ids 54 to 71 for both launches).
#include <algorithm>

#include "../../include/uttt_decode.h"
#include "uttt_device.h"
#include "uttt_host.h"

namespace uttt {
namespace {

constexpr int kMaxBeams = 32;
constexpr int kPer = 16;                     // elements of a thread
constexpr int kStretch = kThreads * kPer;    // of a workgroup
constexpr int kListed = 512;                 // elements at the bound that a list holds; more are chosen one by one
constexpr int kMergeThreads = 1024;
// Workgroups that parts of rows are cut into, where there are fewer rows.  Both launches, us, with 512, 1024 and 2048: 16 x 16
// beams of 131072 ids 37.8, 38.6, 41.9; one group of 16 of them 23.7, 22.8, 28.8; 64 x 4 of 50000 21.9, 19.6, 22.4.
constexpr int kFill = 1024;
constexpr float kLog2e = 1.44269504088896340736f;

struct BeamArgs {
  int rows, beams, parts, n_banned;
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
  double* sums;      // (rows, parts)
  uint64_t* best;    // (rows, parts, beams): ordered logit above, ~id below; 0: none
  float* tops;       // (rows, parts)
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

// The largest key of BITS upper bits that at least `want` lanes reach.
template <int BITS>
__device__ __forceinline__ uint32_t reached_by(uint32_t key, int want) {
  uint32_t t = 0;
#pragma unroll
  for (int bit = 31; bit >= 32 - BITS; --bit) {
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

// Grid (parts of a row, rows).  A part's stretches pass through registers, the next one on its way: each thread keeps the
// maximum and the sum of what it has seen, each wave the bound that its lanes' maxima give (it only rises, so what is not listed
// when it passes by is never among the best) and the list of what reached it.  The waves meet at the end.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_beam_part(const BeamArgs a) {
  constexpr int kVec = Lanes16<T>::kVec, kWaves = kThreads / 64;
  __shared__ uint64_t lists[kWaves][kListed];
  __shared__ uint64_t best_of[kListed];
  __shared__ uint64_t wide[kWaves];
  __shared__ float tops[kWaves];
  __shared__ double sums[kWaves];
  __shared__ uint32_t bounds[kWaves];
  __shared__ int counts[kWaves];
  __shared__ int chosen;
  const int row = blockIdx.y, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (a.ended_in != nullptr && a.ended_in[row] != 0) return;  // its one continuation needs no logit
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const int limit = (int)a.limit, vocab = (int)a.vocab;
  const int all = (limit + kStretch - 1) / kStretch;
  const int begin = (int)((int64_t)all * blockIdx.x / a.parts), end = (int)((int64_t)all * (blockIdx.x + 1) / a.parts);
  // element j of a thread is id base + at(j); 16-byte pieces where the row allows them, single ones otherwise
  auto at = [&](int j) {
    return aligned ? ((j / kVec) * kThreads + (int)threadIdx.x) * kVec + j % kVec : j * kThreads + (int)threadIdx.x;
  };
  struct Values {
    float v[kPer];
  };
  auto load = [&](int i) {
    Values r;
    const int base = i * kStretch;
    if (aligned && base + kStretch <= vocab) {
      uint4 piece[kPer / kVec];
#pragma unroll
      for (int c = 0; c < kPer / kVec; ++c) piece[c] = *reinterpret_cast<const uint4*>(x + base + at(c * kVec));
#pragma unroll
      for (int j = 0; j < kPer; ++j) r.v[j] = Lanes16<T>::get(piece[j / kVec], j % kVec);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) r.v[j] = base + at(j) < vocab ? to_f32(x[base + at(j)]) : -INFINITY;
    }
    return r;
  };
  // ids that are out of use as -inf; -0 as 0: the order is the values'
  auto prepare = [&](Values& r, int i) {
    const int base = i * kStretch;
#pragma unroll
    for (int j = 0; j < kPer; ++j) r.v[j] += 0.f;
    if (base + kStretch > limit) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) r.v[j] = base + at(j) >= limit ? -INFINITY : r.v[j];
    }
    for (int q = 0; q < a.n_banned; ++q) {
      const int id = a.banned[q] - base;
      if (id < 0 || id >= kStretch) continue;
#pragma unroll
      for (int j = 0; j < kPer; ++j) r.v[j] = at(j) == id ? -INFINITY : r.v[j];
    }
  };
  float top = -INFINITY;
  double sum = 0.0;
  uint32_t bound = 0;
  int count = 0;  // of this wave's list
  Values next;
  if (begin < end) next = load(begin);
  for (int i = begin; i < end; ++i) {
    Values now = next;
    if (i + 1 < end) next = load(i + 1);
    prepare(now, i);
    float high = top;
#pragma unroll
    for (int j = 0; j < kPer; ++j) high = fmaxf(high, now.v[j]);
    bound = max(bound, reached_by<16>(ordered(high), a.beams));
    const float least = fmaxf(unordered(max(bound, ordered(-INFINITY))), -3.402823466e38f);
    float part = 0.f;
    const float from = high == -INFINITY ? 0.f : high;  // differences first: a rounded product would move the whole sum
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      part += __builtin_amdgcn_exp2f((now.v[j] - from) * kLog2e);
      const uint64_t here = __ballot(now.v[j] >= least);
      if (here != 0) {
        const int to = count + __popcll(here & ((1ull << lane) - 1));
        if (now.v[j] >= least && to < kListed)
          lists[w][to] = (uint64_t)ordered(now.v[j]) << 32 | (uint32_t)~(uint32_t)(i * kStretch + at(j));
        count += __popcll(here);
      }
    }
    sum = (top == high ? sum : sum * (double)__builtin_amdgcn_exp2f((top - from) * kLog2e)) + (double)part;
    top = high;
  }
  const float wave_top = wave_max(top);
  if (lane == 0) {
    bounds[w] = bound;
    tops[w] = wave_top;
    counts[w] = count;
  }
  if (threadIdx.x == 0) chosen = 0;
  __syncthreads();
  const uint32_t reach = max(max(bounds[0], bounds[1]), max(bounds[2], bounds[3]));
  const float over = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const int64_t place = (int64_t)row * a.parts + blockIdx.x;
  uint64_t* best = a.best + place * a.beams;
  // a thread without a finite maximum has seen nothing, or NaN
  sum = top == -INFINITY ? (sum == sum ? 0.0 : sum) : sum * (double)__builtin_amdgcn_exp2f((top - over) * kLog2e);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if (lane == 0) sums[w] = sum;
  const bool fits = max(max(counts[0], counts[1]), max(counts[2], counts[3])) <= kListed;
  if (fits) {
    for (int i = lane; i < count; i += 64) {
      const uint64_t k = lists[w][i];
      if ((uint32_t)(k >> 32) >= reach) {
        const int to = atomicAdd(&chosen, 1);
        if (to < kListed) best_of[to] = k;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    a.sums[place] = sums[0] + sums[1] + sums[2] + sums[3];
    a.tops[place] = over;
  }
  const int n = chosen;
  if (fits && n <= kListed) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint64_t k = best_of[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += best_of[j] > k;
      if (rank < a.beams) best[rank] = k;
    }
    for (int i = n + threadIdx.x; i < a.beams; i += kThreads) best[i] = 0;
    return;
  }
  uint64_t last = ~0ull;
  for (int q = 0; q < a.beams; ++q) {  // too many equal logits for the lists: the best below the last one, each by another pass
    uint64_t found = 0;
    for (int i = begin; i < end; ++i) {
      Values now = load(i);
      prepare(now, i);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const uint64_t k = (uint64_t)ordered(now.v[j]) << 32 | (uint32_t)~(uint32_t)(i * kStretch + at(j));
        if (now.v[j] > -INFINITY && k < last && k > found) found = k;
      }
    }
    found = wave_max64(found);
    if (lane == 0) wide[w] = found;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kWaves; ++j) found = found > wide[j] ? found : wide[j];
    if (threadIdx.x == 0) best[q] = found;
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
  __shared__ uint32_t bounds[kWaves], shares[kWaves], highs[kWaves];
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
      for (int s = lane; s < a.parts; s += 64) top = fmaxf(top, a.tops[(int64_t)row * a.parts + s]);
      top = wave_max(top);
      for (int s = lane; s < a.parts; s += 64) {
        const float t = a.tops[(int64_t)row * a.parts + s];
        const double part = a.sums[(int64_t)row * a.parts + s];
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
  const int per = a.parts * a.beams, total = a.beams * per;
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
  uint32_t high = 0, place, bound = 0;
  for (int i = threadIdx.x; i < total; i += kMergeThreads) high = max(high, (uint32_t)(look(i, place) >> 32));
  const uint32_t mine = reached_by<32>(high, a.beams);
  if (lane == 0) bounds[w] = mine;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kWaves; ++j) bound = max(bound, bounds[j]);
  int n;
  // Where more reach it than the list holds (beams of very different scores, equal logits), what a share of the `beams` reaches
  // in every wave is another bound; then bounds are halved towards a higher one that `beams` still reach.  One group of 32 beams
  // of 131072 bf16 ids: 54 to 71 us, choosing its 32 one by one 660.
  for (uint32_t over = ~0u, tries = 0;; ++tries) {
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
    n = listed;
    if (n <= kListed) break;
    uint32_t next = bound;
    if (tries == 0) {
      const uint32_t share = reached_by<32>(high, (a.beams + kWaves - 1) / kWaves);
      uint32_t highest = high;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) highest = max(highest, (uint32_t)__shfl_xor((int)highest, off, 64));
      if (lane == 0) {
        shares[w] = share;
        highs[w] = highest;
      }
      __syncthreads();
      uint32_t common = ~0u;
      over = 0;
#pragma unroll
      for (int j = 0; j < kWaves; ++j) {
        common = min(common, shares[j]);
        over = max(over, highs[j] + 1);
      }
      next = max(bound, common);
    }
    while (next == bound && over - next > 1) {
      const uint32_t mid = next + (over - next) / 2;
      int reached = 0;
      for (int i = threadIdx.x; i < total; i += kMergeThreads) reached += (uint32_t)(look(i, place) >> 32) >= mid;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) reached += __shfl_xor(reached, off, 64);
      if (lane == 0) bounds[w] = reached;
      __syncthreads();
      reached = 0;
#pragma unroll
      for (int j = 0; j < kWaves; ++j) reached += bounds[j];
      __syncthreads();
      if (reached < a.beams)
        over = mid;
      else
        next = mid;
    }
    if (next == bound) break;  // equal ones
    bound = next;
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
  }
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

// Parts of a row: as many as fill the card, a stretch at least each.
int64_t row_parts(int64_t rows, int64_t vocab) {
  return std::max<int64_t>(1, std::min<int64_t>((vocab + kStretch - 1) / kStretch, kFill / rows));
}

}  // namespace
}  // namespace uttt

using namespace uttt;

extern "C" size_t uttt_beam_select_workspace(int64_t rows, int64_t vocab, int64_t beams) {
  if (rows < 1 || vocab < 1 || beams < 1) return 0;
  return (size_t)rows * (size_t)row_parts(rows, vocab) * (8 * (size_t)beams + 8 + 4);
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
  m.parts = (int)row_parts(a->rows, m.limit);
  for (int i = 0; i < 8; ++i) m.banned[i] = a->banned[i];
  m.logits = a->logits; m.row_stride = a->row_stride;
  m.scores = a->scores; m.ended_in = a->ended_in;
  m.eos = a->eos; m.pad = a->pad;
  m.tokens = a->tokens; m.sources = a->sources; m.out_scores = a->out_scores; m.ended_out = a->ended_out;
  m.best = static_cast<uint64_t*>(a->workspace);
  m.sums = reinterpret_cast<double*>(m.best + (int64_t)m.rows * m.parts * m.beams);
  m.tops = reinterpret_cast<float*>(m.sums + (int64_t)m.rows * m.parts);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)m.parts, (unsigned)m.rows);
  if (a->dtype == UTTT_DTYPE_BF16)
    hipLaunchKernelGGL(k_beam_part<bf16>, grid, dim3(kThreads), 0, st, m);
  else
    hipLaunchKernelGGL(k_beam_part<float>, grid, dim3(kThreads), 0, st, m);
  hipLaunchKernelGGL(k_beam_merge, dim3((unsigned)(m.rows / m.beams)), dim3(kMergeThreads), 0, st, m);
  return launch_status("uttt_beam_select");
}
