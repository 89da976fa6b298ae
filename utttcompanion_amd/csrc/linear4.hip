// Products with weights in 4 bits for the rows of a decode step, written for gfx950 (MI355X): y = x W^T with one matrix
// for all rows (slow projections, LM head) or one per request (the frozen fast-weight readout).
//
// Per group of 32 columns a 16 x 32 piece of W is one MFMA operand, converted from its codes (fp4.h); the group's scale, one
// per row of W, multiplies the fp32 products as they are added up:  y[m][n] = sum_g s[n][g] (x[m][g] . c[n][g]).  x is an
// operand as it is (bf16), or in bf16 parts that add up to it: three for fp32, two where bf16 activations were multiplied by a
// norm's weight or are the fp32 hidden values of a readout (16 bits, where the model's own path has 8).
//
// A workgroup takes NT blocks of 16 rows of W and 16 MT rows of x; its waves divide the columns and meet in LDS.
#include <algorithm>

#include "../../include/uttt_decode.h"
#include "fp4.h"
#include "uttt_host.h"

namespace uttt {
namespace {

constexpr int kBlockBytes = 1152;  // 16 x 128 of W
constexpr int kMaxWaves4 = 8;

struct Prod4Args {
  int m, n, k, blocks;  // blocks of 128 columns
  int aligned;          // x: 16-byte pieces
  float x_eps;          // > 0: rows of x are RMS-normalised
  const void* x;
  int64_t xs_b, xs_m;
  const void* gain;  // (k,) of x's type, or null: multiplies x's columns after the norm
  const char* w[2];
  int64_t ws_b[2];
  const void* r;
  int64_t rs_m;
  void* out;
  int64_t os_b, os_m;
};

// Eight neighbours of a row from column k0 on, zeros from k on.
__device__ __forceinline__ bf16x8 load_x8(const bf16* row, int k0, int k, bool aligned) {
  bf16x8 v;
  if (aligned && k0 + 8 <= k) {
    v = *reinterpret_cast<const bf16x8*>(row + k0);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k0 + j < k ? row[k0 + j] : static_cast<bf16>(0.f);
  }
  return v;
}

template <typename X>
__device__ __forceinline__ void load_x8(const X* row, int k0, int k, bool aligned, float (&v)[8]) {
  if constexpr (sizeof(X) == 2) {
    const bf16x8 t = load_x8(row, k0, k, aligned);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32(t[j]);
  } else if (aligned && k0 + 8 <= k) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(row + k0), b = *reinterpret_cast<const f32x4*>(row + k0 + 4);
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

template <typename X, typename O, int PARTS, int MT, int NT, bool SWIGLU>
__global__ void __launch_bounds__(kMaxWaves4 * 64) k_prod4(const Prod4Args a) {
  __shared__ float red[kMaxWaves4][MT * 4][64];
  __shared__ float squares[kMaxWaves4][MT * 16];
  const int waves = blockDim.x >> 6, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r = lane & 15, h = lane >> 4;
  const int tiles = (a.n + 15) >> 4, tile0 = blockIdx.x * (SWIGLU ? 1 : NT), m0 = blockIdx.y * (16 * MT), b = blockIdx.z;
  const X* x = static_cast<const X*>(a.x) + b * a.xs_b;
  const X* gain = static_cast<const X*>(a.gain);
  const char* wp[NT];
#pragma unroll
  for (int s = 0; s < NT; ++s) {
    const int tile = SWIGLU ? tile0 : min(tile0 + s, tiles - 1);
    wp[s] = a.w[SWIGLU ? s : 0] + b * a.ws_b[SWIGLU ? s : 0] + (int64_t)tile * a.blocks * kBlockBytes;
  }
  const X* row[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) row[t] = x + (int64_t)min(m0 + 16 * t + r, a.m - 1) * a.xs_m;
  f32x4 acc[NT][MT];
  float ss[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    ss[t] = 0.f;
#pragma unroll
    for (int s = 0; s < NT; ++s) acc[s][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int begin = a.blocks * w / waves, end = a.blocks * (w + 1) / waves;
  for (int kb = begin; kb < end; ++kb) {
    u32x4 code[NT];
    u32x2 scale[NT];
#pragma unroll
    for (int s = 0; s < NT; ++s) {
      code[s] = *reinterpret_cast<const u32x4*>(wp[s] + (int64_t)kb * kBlockBytes + lane * 16);
      scale[s] = *reinterpret_cast<const u32x2*>(wp[s] + (int64_t)kb * kBlockBytes + 1024 + r * 8);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int k0 = kb * 128 + 32 * g + 8 * h;
      bf16x8 xf[MT][PARTS];
      float gv[8];
      if (gain != nullptr) load_x8(gain, k0, a.k, true, gv);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if constexpr (sizeof(X) == 2 && PARTS == 1) {
          xf[t][0] = load_x8(row[t], k0, a.k, a.aligned);
          if (a.x_eps > 0.f) {
#pragma unroll
            for (int j = 0; j < 8; ++j) ss[t] = fmaf(to_f32(xf[t][0][j]), to_f32(xf[t][0][j]), ss[t]);
          }
        } else {
          float v[8];
          load_x8(row[t], k0, a.k, a.aligned, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            ss[t] = fmaf(v[j], v[j], ss[t]);
            if (gain != nullptr) v[j] *= gv[j];
            bf16 p[PARTS];
            bf16_parts(v[j], p);
#pragma unroll
            for (int i = 0; i < PARTS; ++i) xf[t][i][j] = p[i];
          }
        }
      }
#pragma unroll
      for (int s = 0; s < NT; ++s) {
        const bf16x8 c = fp4_values(code[s][g]);
        const float f = bf16_of(scale[s][g >> 1], g & 1);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          f32x4 y{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < PARTS; ++i) y = mfma16(xf[t][i], c, y);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[s][t][i] = fmaf(f, y[i], acc[s][t][i]);
        }
      }
    }
  }
  if (a.x_eps > 0.f) {
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      ss[t] += __shfl_xor(ss[t], 16, 64);
      ss[t] += __shfl_xor(ss[t], 32, 64);
      if (h == 0) squares[w][16 * t + r] = ss[t];
    }
  }
  constexpr int kOuts = (MT * 256 + 63) / 64;  // outputs of a thread, at one wave
  float kept[SWIGLU ? kOuts : 1];
#pragma unroll
  for (int s = 0; s < NT; ++s) {
    __syncthreads();
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[w][4 * t + i][lane] = acc[s][t][i];
    __syncthreads();
    const int n0 = (SWIGLU ? tile0 : tile0 + s) * 16;
#pragma unroll
    for (int o = 0; o < kOuts; ++o) {
      const int idx = threadIdx.x + o * (int)blockDim.x;
      if (idx >= MT * 256) break;
      const int nn = idx & 15, mm = idx >> 4, i = 4 * (mm >> 4) + (mm & 3), l = ((mm & 15) >> 2) * 16 + nn;
      float y = 0.f;
      for (int q = 0; q < waves; ++q) y += red[q][i][l];
      if (a.x_eps > 0.f) {
        float q2 = 0.f;
        for (int q = 0; q < waves; ++q) q2 += squares[q][mm];
        y *= rsqrtf(q2 / (float)a.k + a.x_eps);
      }
      if constexpr (SWIGLU) {
        if (s == 0) {
          kept[o] = y;
          continue;
        }
        y = y / (1.f + __expf(-y)) * kept[o];
      }
      if (m0 + mm >= a.m || n0 + nn >= a.n) continue;
      const int64_t row_m = m0 + mm;
      if (a.r != nullptr) y += to_f32(static_cast<const O*>(a.r)[row_m * a.rs_m + n0 + nn]);
      (static_cast<O*>(a.out) + b * a.os_b)[row_m * a.os_m + n0 + nn] = from_f32<O>(y);
    }
  }
}

struct Norm4Args {
  int d;
  float eps, x_eps;
  const float* z;  // (B, T, d)
  const void* x;
  int64_t xs_b, xs_t;
  const void* gain;
  const float *ln_w, *ln_b;
  void* out;
  int64_t os_b, os_t;
};

// out = x' + LN(z), one row per workgroup (T, B): z and x stay in registers between the sums and the result.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_readout4_norm(const Norm4Args a) {
  __shared__ float scratch[4];
  const int t = blockIdx.x, b = blockIdx.y;
  const float* z = a.z + ((int64_t)b * gridDim.x + t) * a.d;
  const T* x = static_cast<const T*>(a.x) + b * a.xs_b + t * a.xs_t;
  T* out = static_cast<T*>(a.out) + b * a.os_b + t * a.os_t;
  float v[16], xv[16];
  float sum = 0.f, squares = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int e = threadIdx.x + i * kThreads;
    v[i] = e < a.d ? z[e] : 0.f;
    xv[i] = e < a.d ? to_f32(x[e]) : 0.f;
    sum += v[i];
    squares = fmaf(xv[i], xv[i], squares);
  }
  const float mean = block_sum(sum, scratch) / (float)a.d;
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float g = threadIdx.x + i * kThreads < a.d ? v[i] - mean : 0.f;
    far = fmaf(g, g, far);
  }
  const float rs = 1.f / sqrtf(block_sum(far, scratch) / (float)a.d + a.eps);
  float xr = 1.f;
  if (a.gain != nullptr) xr = 1.f / sqrtf(block_sum(squares, scratch) / (float)a.d + a.x_eps);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int e = threadIdx.x + i * kThreads;
    if (e >= a.d) break;
    float y = xv[i];
    if (a.gain != nullptr) y *= xr * to_f32(static_cast<const T*>(a.gain)[e]);
    out[e] = from_f32<T>(y + ((v[i] - mean) * rs * a.ln_w[e] + a.ln_b[e]));
  }
}

template <typename X, typename O, int PARTS, int NT, bool SWIGLU>
void launch_prod4(const Prod4Args& p, int batch, hipStream_t st) {
  const int tiles = (p.n + 15) / 16, units = SWIGLU ? tiles : (tiles + NT - 1) / NT;
  const int waves = std::min(p.blocks, 4);
  const int mt = p.m <= 16 ? 1 : p.m <= 32 || PARTS > 1 ? 2 : 4;
  const dim3 grid((unsigned)units, (unsigned)((p.m + 16 * mt - 1) / (16 * mt)), (unsigned)batch), block(waves * 64);
  if (mt == 1)
    hipLaunchKernelGGL((k_prod4<X, O, PARTS, 1, NT, SWIGLU>), grid, block, 0, st, p);
  else if (mt == 2)
    hipLaunchKernelGGL((k_prod4<X, O, PARTS, 2, NT, SWIGLU>), grid, block, 0, st, p);
  else if constexpr (PARTS == 1)  // 64 rows of several parts do not fit the registers
    hipLaunchKernelGGL((k_prod4<X, O, PARTS, 4, NT, SWIGLU>), grid, block, 0, st, p);
}

bool whole_pieces(const void* p, int64_t a, int64_t b, int64_t vec) { return aligned16(p) && a % vec == 0 && b % vec == 0; }

}  // namespace
}  // namespace uttt

using namespace uttt;

extern "C" int uttt_decode_abi_version(void) { return UTTT_DECODE_ABI_VERSION; }

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
  Prod4Args p{};
  p.m = (int)a->m; p.n = (int)a->n; p.k = (int)a->k; p.blocks = (int)((a->k + 127) / 128);
  p.aligned = whole_pieces(a->x, a->m == 1 ? 0 : a->x_row_stride, 0, b16 ? 8 : 4);
  p.x_eps = a->x_eps;
  p.x = a->x; p.xs_m = a->x_row_stride;
  p.w[0] = static_cast<const char*>(a->w);
  p.r = a->residual; p.rs_m = a->residual_row_stride;
  p.out = a->out; p.os_m = a->out_row_stride;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (b16)
    launch_prod4<bf16, bf16, 1, 1, false>(p, 1, st);
  else
    launch_prod4<float, float, 3, 1, false>(p, 1, st);
  return launch_status("uttt_linear4");
}

extern "C" size_t uttt_readout4_workspace(int64_t batch, int64_t tokens, int64_t d_model, int64_t d_ff) {
  if (batch < 1 || tokens < 1 || d_model < 1 || d_ff < 1) return 0;
  return sizeof(float) * (size_t)batch * (size_t)tokens * (size_t)(d_model + d_ff);
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
  const int D = (int)a->d_model, F = (int)a->d_ff, T = (int)a->tokens, B = (int)a->batch;
  float* hidden = static_cast<float*>(a->workspace);
  float* z = hidden + (int64_t)B * T * F;
  hipStream_t st = static_cast<hipStream_t>(stream);
  Prod4Args p{};
  p.m = T; p.n = F; p.k = D; p.blocks = (D + 127) / 128;
  p.aligned = 1;
  p.x = a->x; p.xs_b = a->x_stride_b; p.xs_m = a->x_stride_t;
  p.gain = a->x_norm_weight;
  p.x_eps = a->x_norm_weight ? a->x_norm_eps : 0.f;
  p.w[0] = static_cast<const char*>(a->w_up); p.ws_b[0] = a->w_up_stride;
  p.w[1] = static_cast<const char*>(a->w_gate); p.ws_b[1] = a->w_gate_stride;
  p.out = hidden; p.os_b = (int64_t)T * F; p.os_m = F;
  if (!b16)
    launch_prod4<float, float, 3, 2, true>(p, B, st);
  else if (p.gain)
    launch_prod4<bf16, float, 2, 2, true>(p, B, st);
  else
    launch_prod4<bf16, float, 1, 2, true>(p, B, st);
  Prod4Args q{};
  q.m = T; q.n = D; q.k = F; q.blocks = (F + 127) / 128;
  q.aligned = 1;
  q.x = hidden; q.xs_b = (int64_t)T * F; q.xs_m = F;
  q.w[0] = static_cast<const char*>(a->w_down); q.ws_b[0] = a->w_down_stride;
  q.out = z; q.os_b = (int64_t)T * D; q.os_m = D;
  if (b16)
    launch_prod4<float, float, 2, 1, false>(q, B, st);
  else
    launch_prod4<float, float, 3, 1, false>(q, B, st);
  Norm4Args n{};
  n.d = D; n.eps = a->eps; n.x_eps = a->x_norm_eps;
  n.z = z;
  n.x = a->x; n.xs_b = a->x_stride_b; n.xs_t = a->x_stride_t;
  n.gain = a->x_norm_weight;
  n.ln_w = a->ln_weight; n.ln_b = a->ln_bias;
  n.out = a->out; n.os_b = a->out_stride_b; n.os_t = a->out_stride_t;
  if (b16)
    hipLaunchKernelGGL(k_readout4_norm<bf16>, dim3(T, B), dim3(kThreads), 0, st, n);
  else
    hipLaunchKernelGGL(k_readout4_norm<float>, dim3(T, B), dim3(kThreads), 0, st, n);
  return launch_status("uttt_readout4");
}
