// Next-token sampling of a decode step, written for gfx950 (MI355X): temperature, top-k, min-p and top-p with
// settings per row, from given uniform numbers; one launch, no sort.  The rules stand at uttt_sample_select.
//
// With w_i = 2^(c (x_i - max)), c = log2(e) / temperature, every rule keeps a prefix of the order (logit
// descending, id ascending), so the kept set is a cut (key, ties): the ids whose logit lies above the key's,
// and the first `ties` of those at it.  A cut is found from a histogram of counts and masses over x (bins of 1/48 of a
// factor of two), then inside the one bin where the count or the mass passes its bound: its few ids are
// ranked against each other, or, when there are many, its range of keys is divided again.  The token is
// found by the kept mass of 16 stretches of the row, one per wave, then of 16 parts of the stretch that holds
// it, then by a scan inside one wave.
//
// The sums decide between neighbouring ids, so weights are formed in 64 bits (2^f by its Taylor series to
// degree 10, 2^-42 off) and added as integers in units of 2^-42 of the largest weight: exact whatever the order, so
// atomics in any order give equal bits.
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
constexpr float kBinsPerOctave = 48.f;  // kBins / 48 > 42: every weight that is not 0 has a bin of its own width
constexpr int kList = 256;

__device__ __forceinline__ bool excluded(const SampleArgs& a, int i) {
  if (i < 64) return (a.low >> i) & 1;
  bool m = false;
  for (int k = 0; k < a.n_high; ++k) m |= i == a.high[k];
  return m;
}

// order-preserving key of a logit that is not NaN; -0 and +0 are equal
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// 2^t for t <= 0 in units of 2^-42, to the nearest unit
__device__ __forceinline__ u64 weight_units(double t) {
  if (!(t > -44.0)) return 0;
  const double n = __builtin_rint(t), f = (t - n) * 0.6931471805599453;
  double p = 1.0 / 3628800;
  p = __builtin_fma(p, f, 1.0 / 362880);
  p = __builtin_fma(p, f, 1.0 / 40320);
  p = __builtin_fma(p, f, 1.0 / 5040);
  p = __builtin_fma(p, f, 1.0 / 720);
  p = __builtin_fma(p, f, 1.0 / 120);
  p = __builtin_fma(p, f, 1.0 / 24);
  p = __builtin_fma(p, f, 1.0 / 6);
  p = __builtin_fma(p, f, 0.5);
  p = __builtin_fma(p, f, 1.0);
  p = __builtin_fma(p, f, 1.0);
  // adding 2^52 rounds to whole units, which are then the low bits
  const double u = __builtin_ldexp(p, (int)n + 42) + 4503599627370496.0;
  return __builtin_bit_cast(u64, u) & 0xfffffffffffffull;
}

__device__ __forceinline__ u64 shfl_up64(u64 v, int off) {
  const uint32_t lo = __shfl_up((uint32_t)v, off, 64), hi = __shfl_up((uint32_t)(v >> 32), off, 64);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 shfl_xor64(u64 v, int off) {
  const uint32_t lo = __shfl_xor((uint32_t)v, off, 64), hi = __shfl_xor((uint32_t)(v >> 32), off, 64);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += shfl_xor64(v, off);
  return v;
}

// A cut: ids with a larger key are kept, and the first `ties` of those with this key.
struct Cut {
  uint32_t key;
  int ties;
  u64 mass;  // of what it keeps
};

struct Shared {
  u64 mass[kBins];
  uint32_t count[kBins];
  u64 mass2[kBins];  // of a range of keys inside one bin
  uint32_t count2[kBins];
  u64 wave_mass[kSmpWaves];
  uint32_t wave_count[kSmpWaves];
  float wave_best[kSmpWaves];
  int wave_id[kSmpWaves];
  uint32_t list_key[kList];
  int list_id[kList];
  u64 list_mass[kList];
  uint32_t n, kmin, kmax, before_count;
  u64 before_mass;
  int bin;
  u64 kept;
  uint32_t cut_key;
  int cut_ties;
  int token;
};

// ids [lo, hi) of the row, in order, VEC at a time and 64 VEC to a wave step, kUnroll steps in flight
template <typename T, int VEC, int kUnroll, typename F>
__device__ __forceinline__ void scan_ids(const T* x, int lo, int hi, int lane, F&& f) {
  typedef T vec_t __attribute__((ext_vector_type(VEC)));
  for (int b = lo; b < hi; b += 64 * VEC * kUnroll) {
    vec_t v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = b + (u * 64 + lane) * VEC;
      if (i + VEC <= hi) {
        v[u] = *reinterpret_cast<const vec_t*>(x + i);
      } else if (i < hi) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[u][e] = i + e < hi ? x[i + e] : x[i];
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = b + (u * 64 + lane) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (i + e < hi) f(to_f32(v[u][e]), i + e);
    }
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kSmpThreads) k_sample_select(const SampleArgs a) {
  __shared__ Shared s;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const T* x = static_cast<const T*>(a.logits) + (int64_t)row * a.rs;
  // a wave's stretch of the row
  constexpr int kStep = 64 * VEC;
  const int stretch = ((a.limit + kSmpWaves - 1) / kSmpWaves + kStep - 1) / kStep * kStep;
  const int lo = min(w * stretch, a.limit), hi = min(lo + stretch, a.limit);

  // ---- the largest logit (NaN above all, ties to the lowest id), as a greedy choice has it
  float bv = -INFINITY;
  int bi = 0x7fffffff;
  auto take = [&](float v, int i) {
    const bool vn = v != v, bn = bv != bv;
    const bool ahead = vn != bn ? vn : (!vn && v != bv) ? v > bv : i < bi;
    if (ahead) {
      bv = v;
      bi = i;
    }
  };
  scan_ids<T, VEC, 16 / VEC < 4 ? 16 / VEC : 4>(x, lo, hi, lane, [&](float v, int i) { take(excluded(a, i) ? -INFINITY : v, i); });
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) take(__shfl_xor(bv, off, 64), __shfl_xor(bi, off, 64));
  if (lane == 0) {
    s.wave_best[w] = bv;
    s.wave_id[w] = bi;
  }
  for (int i = tid; i < kBins; i += kSmpThreads) {
    s.mass[i] = 0;
    s.count[i] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kSmpWaves; ++q) take(s.wave_best[q], s.wave_id[q]);
  const float temp = a.temperature[row], top = bv;
  const bool greedy = !(temp > 1e-5f), odd = !(fabsf(top) < INFINITY);
  if (greedy || odd) {
    if (tid == 0) {
      a.out[row] = bi == 0x7fffffff ? 0 : bi;
      if (a.logprob != nullptr) a.logprob[row] = greedy ? 0.f : NAN;
      if (a.advance != nullptr) a.advance[row] += 1;
    }
    return;
  }

  const double c = 1.4426950408889634 / (double)temp, dtop = (double)top;
  const int top_k = a.top_k != nullptr ? a.top_k[row] : 0;
  const float top_p = a.top_p != nullptr ? a.top_p[row] : 1.f, min_p = a.min_p != nullptr ? a.min_p[row] : 0.f;
  const bool by_count = top_k > 0 && top_k < a.limit, by_mass = top_p < 1.f;
  const u64 least = min_p > 0.f ? (u64)__builtin_ceil(fmin((double)min_p, 1.0) * 4398046511104.0) : 1;
  auto weight = [&](float v) -> u64 {
    const u64 u = weight_units(((double)v - dtop) * c);
    return u >= least ? u : 0;
  };
  const float per_unit = fminf((float)c * kBinsPerOctave, 3e38f);
  auto bin_of = [&](float v) { return (int)fminf((top - v) * per_unit, (float)(kBins - 1)); };

  Cut cut{0, 0x7fffffff, 0};  // keeps everything
  if (by_count || by_mass) {
    scan_ids<T, VEC, 1>(x, lo, hi, lane, [&](float v, int i) {
      if (excluded(a, i)) return;
      const int b = bin_of(v);
      const u64 u = weight(v);
      if (u != 0) atomicAdd(&s.mass[b], u);
      if (by_count) atomicAdd(&s.count[b], 1u);
    });
    __syncthreads();
    // what lies ahead of each thread's two bins, and where the bound falls; `bound` counts or mass
    auto find = [&](const u64* mass, const uint32_t* count, u64 mass0, uint32_t count0, bool counts, u64 bound) {
      const u64 m0 = mass[2 * tid], m1 = mass[2 * tid + 1];
      const uint32_t n0 = count[2 * tid], n1 = count[2 * tid + 1];
      u64 m = m0 + m1;
      uint32_t n = n0 + n1;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const u64 pm = shfl_up64(m, off);
        const uint32_t pn = __shfl_up(n, off, 64);
        if (lane >= off) {
          m += pm;
          n += pn;
        }
      }
      if (lane == 63) {
        s.wave_mass[w] = m;
        s.wave_count[w] = n;
      }
      if (tid == 0) s.bin = -1;
      __syncthreads();
      m -= m0 + m1;
      n -= n0 + n1;
      u64 total = mass0;
#pragma unroll
      for (int q = 0; q < kSmpWaves; ++q) {
        const u64 wm = s.wave_mass[q];
        total += wm;
        if (q < w) {
          m += wm;
          n += s.wave_count[q];
        }
      }
      m += mass0;
      n += count0;
      if (!counts && bound == ~0ull) bound = (u64)((double)fmaxf(top_p, 0.f) * (double)total);
      // the bin with the last kept id: the bound-th, or the last whose mass ahead is within the bound
      const bool in0 = counts ? n < bound && bound <= n + n0 : m <= bound && bound < m + m0;
      const bool in1 = counts ? n + n0 < bound && bound <= n + n0 + n1 : m + m0 <= bound && bound < m + m0 + m1;
      if (in0 || in1) {
        s.bin = 2 * tid + (in0 ? 0 : 1);
        s.before_mass = in0 ? m : m + m0;
        s.before_count = in0 ? n : n + n0;
      }
      __syncthreads();
      return bound;
    };
    // the ids of one bin (and range of keys): how many, the first kList, the range of their keys
    auto gather = [&](int bin, uint32_t kmin, uint32_t kmax) {
      if (tid == 0) {
        s.n = 0;
        s.kmin = 0xffffffffu;
        s.kmax = 0;
      }
      __syncthreads();
      uint32_t mn = 0xffffffffu, mx = 0;
      scan_ids<T, VEC, 1>(x, lo, hi, lane, [&](float v, int i) {
        if (bin_of(v) != bin || excluded(a, i)) return;
        const uint32_t k = key_of(v);
        if (k < kmin || k > kmax) return;
        mn = min(mn, k);
        mx = max(mx, k);
        const uint32_t at = atomicAdd(&s.n, 1u);
        if (at < kList) {
          s.list_key[at] = k;
          s.list_id[at] = i;
          s.list_mass[at] = weight(v);
        }
      });
      if (mn <= mx) {
        atomicMin(&s.kmin, mn);
        atomicMax(&s.kmax, mx);
      }
      __syncthreads();
    };
    // the cut inside the bin that find() left
    auto resolve = [&](bool counts, u64 bound) -> Cut {
      const int bin = s.bin;
      u64 mass0 = s.before_mass;
      uint32_t count0 = s.before_count;
      __syncthreads();
      gather(bin, 0, 0xffffffffu);
      uint32_t kmin = s.kmin, kmax = s.kmax;
      while (s.n > kList && kmin != kmax) {
        const int shift = max(0, 32 - 11 - __builtin_clz(kmax - kmin));
        for (int i = tid; i < kBins; i += kSmpThreads) {
          s.mass2[i] = 0;
          s.count2[i] = 0;
        }
        __syncthreads();
        scan_ids<T, VEC, 1>(x, lo, hi, lane, [&](float v, int i) {
          if (bin_of(v) != bin || excluded(a, i)) return;
          const uint32_t k = key_of(v);
          if (k < kmin || k > kmax) return;
          const int b = (int)((kmax - k) >> shift);
          const u64 u = weight(v);
          if (u != 0) atomicAdd(&s.mass2[b], u);
          atomicAdd(&s.count2[b], 1u);
        });
        __syncthreads();
        find(s.mass2, s.count2, mass0, count0, counts, bound);
        if (s.bin < 0) break;  // the bound lies inside the bin, so one of its parts has it
        const uint32_t b = (uint32_t)s.bin;
        mass0 = s.before_mass;
        count0 = s.before_count;
        const uint32_t hi_key = kmax - (b << shift), width = (1u << shift) - 1;
        const uint32_t lo_key = hi_key - kmin > width ? hi_key - width : kmin;
        __syncthreads();
        gather(bin, lo_key, hi_key);
        kmin = s.kmin;
        kmax = s.kmax;
      }
      Cut r;
      if (kmin == kmax) {  // equal logits: a number of them
        const u64 u = weight(of_key(kmin));
        const u64 n = s.n;
        u64 t = counts ? bound - count0 : u != 0 ? (bound - mass0) / u + 1 : n;
        t = t < n ? t : n;
        r.key = kmin;
        r.ties = (int)t;
        r.mass = mass0 + t * u;
      } else {
        const int n = (int)s.n;
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
      __syncthreads();
      return r;
    };
    u64 limit_mass = ~0ull;  // top_p of the row's mass, or of what top_k keeps
    if (by_count) {
      find(s.mass, s.count, 0, 0, true, (u64)top_k);
      if (s.bin >= 0) {  // else fewer ids than top_k
        cut = resolve(true, (u64)top_k);
        limit_mass = (u64)((double)fmaxf(top_p, 0.f) * (double)cut.mass);
      }
    }
    if (by_mass) {
      const u64 bound = find(s.mass, s.count, 0, 0, false, limit_mass);
      if (s.bin >= 0) {
        const Cut p = resolve(false, bound);
        if (p.key > cut.key || (p.key == cut.key && p.ties < cut.ties)) cut = p;
      }
    }
  }

  // ---- the kept mass of parts [lo, hi) of the row, one per wave: above the cut's key, and ids at it
  const u64 tie_mass = cut.key != 0 ? weight(of_key(cut.key)) : 0;
  auto part_mass = [&](int p_lo, int p_hi) {
    u64 m = 0;
    uint32_t t = 0;
    scan_ids<T, VEC, 1>(x, p_lo, p_hi, lane, [&](float v, int i) {
      const uint32_t k = key_of(v);
      if (k < cut.key || excluded(a, i)) return;
      if (k == cut.key)
        ++t;
      else
        m += weight(v);
    });
    m = wave_sum64(m);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) t += __shfl_xor(t, off, 64);
    __syncthreads();
    if (lane == 0) {
      s.wave_mass[w] = m;
      s.wave_count[w] = t;
    }
    __syncthreads();
  };
  const u64 max_ties = (u64)cut.ties;
  auto with_ties = [&](u64 ties, u64 more) {  // mass of `more` ids at the cut's key behind `ties` of them
    const u64 left = ties < max_ties ? max_ties - ties : 0;
    return (more < left ? more : left) * tie_mass;
  };
  part_mass(lo, hi);
  u64 total = 0, ties = 0;
#pragma unroll
  for (int q = 0; q < kSmpWaves; ++q) {
    total += s.wave_mass[q] + with_ties(ties, s.wave_count[q]);
    ties += s.wave_count[q];
  }
  float uf = a.uniforms[row];
  uf = uf > 0.f ? fminf(uf, 0.99999994f) : 0.f;
  u64 want = (u64)((double)uf * (double)total);
  want = want < total ? want : total - 1;
  // the part whose mass first exceeds `want`, and the mass and ties ahead of it
  u64 ahead = 0, ties_ahead = 0;
  auto pick = [&]() {
    u64 m = ahead, t = ties_ahead;
    int found = kSmpWaves - 1;
    bool done = false;
#pragma unroll
    for (int q = 0; q < kSmpWaves; ++q) {
      if (!done) {
        const u64 next = m + s.wave_mass[q] + with_ties(t, s.wave_count[q]);
        if (next > want) {
          found = q;
          done = true;
        } else {
          m = next;
          t += s.wave_count[q];
        }
      }
    }
    ahead = m;
    ties_ahead = t;
    return found;
  };
  const int p0 = min(pick() * stretch, a.limit), p1 = min(p0 + stretch, a.limit);
  const int part = ((p1 - p0 + kSmpWaves - 1) / kSmpWaves + kStep - 1) / kStep * kStep;
  {
    const int q_lo = min(p0 + w * part, p1);
    part_mass(q_lo, min(q_lo + part, p1));
  }
  const int q0 = min(p0 + pick() * part, p1), q1 = min(q0 + part, p1);
  if (w != 0) return;
  // ---- inside one wave: 64 ids at a time
  u64 m = ahead, t = ties_ahead;
  int token = -1;
  for (int b = q0; b < q1 && token < 0; b += 64) {
    const int i = b + lane;
    u64 u = 0;
    uint32_t tie = 0;
    if (i < q1 && !excluded(a, i)) {
      const float v = to_f32(x[i]);
      const uint32_t k = key_of(v);
      if (k > cut.key) u = weight(v);
      tie = k == cut.key;
    }
    const u64 tied = __ballot(tie);
    const u64 before = t + __popcll(tied & ((1ull << lane) - 1));
    if (tie) u = before < max_ties ? tie_mass : 0;
    u64 sum = u;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const u64 p = shfl_up64(sum, off);
      if (lane >= off) sum += p;
    }
    const u64 over = __ballot(m + sum > want);
    if (over != 0) {
      token = b + __builtin_ctzll(over);
    }
    m += (u64)(uint32_t)__shfl((uint32_t)(sum >> 32), 63, 64) << 32 | (uint32_t)__shfl((uint32_t)sum, 63, 64);
    t += __popcll(tied);
  }
  if (lane == 0) {
    token = token < 0 ? bi : token;
    a.out[row] = token;
    // log(w / total): the weight's own exponent, not its rounded units
    if (a.logprob != nullptr)
      a.logprob[row] = (float)(((double)to_f32(x[token]) - dtop) / (double)temp - log((double)total * 0x1p-42));
    if (a.advance != nullptr) a.advance[row] += 1;
  }
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
  UTTT_REQUIRE(a->row_stride >= a->vocab, "the row stride must cover vocab");
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
  const dim3 grid((unsigned)a->rows);
  const bool bf = a->dtype == UTTT_DTYPE_BF16;
  const bool vec = aligned16(a->logits) && (a->rows == 1 || a->row_stride % 4 == 0);
  if (bf && vec)
    hipLaunchKernelGGL((k_sample_select<bf16, 4>), grid, dim3(kSmpThreads), 0, st, s);
  else if (bf)
    hipLaunchKernelGGL((k_sample_select<bf16, 1>), grid, dim3(kSmpThreads), 0, st, s);
  else if (vec)
    hipLaunchKernelGGL((k_sample_select<float, 4>), grid, dim3(kSmpThreads), 0, st, s);
  else
    hipLaunchKernelGGL((k_sample_select<float, 1>), grid, dim3(kSmpThreads), 0, st, s);
  return launch_status("uttt_sample_select");
}
