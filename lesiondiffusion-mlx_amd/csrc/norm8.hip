// Root-mean-square norm with the residual's addition, into the input's type or into 8-bit rows, and
// the same 8-bit rows of a tensor as it is.
//
//   s = T(x + residual)            (stored where asked for; x itself without a residual)
//   y = s / sqrt(mean(s^2) + eps) * gamma
//   y rounded to T, or per row and 128 columns to e4m3 codes and a power of two (quant8.h)
//
// One pass: a row's values stay in registers between the sum of squares and the output (beyond 8,192 columns
// they are read twice), a wave a row up to 1,024 columns and a workgroup beyond. Bound by memory: 16,384 rows
// of 4,096 in bf16 with residual and 8-bit rows 85 us (5.5 TB/s) on tensors that no cache holds; called again on the
// same ones 72 (part of them still in the 256 MB behind the L2s), plain 39, 8-bit rows of a tensor as it is 36 and 30.
#include "quant8.h"

namespace ldx {
namespace {

struct NormArgs {
  const void* x; int64_t xp;
  const void* r; int64_t rp;      // residual or null
  void* s; int64_t sp;            // sum or null
  const float* gamma; float eps;  // null gamma: no norm
  void* y; int64_t yp;            // T output or null
  uint8_t* codes; int64_t cp;     // 8-bit output
  uint8_t* scales; int64_t ep;
  int64_t rows;
  int C, kb;                      // features; 128-column blocks
  double per_C;                   // 1 / C
};

// Sum (float, double) / largest over a row's threads: a wave, or the four waves of the workgroup through red.
template <int TPR, bool MAX, typename F>
__device__ __forceinline__ F row_reduce(F v, double* red) {
  if constexpr (MAX) v = wave_max(v);
  else v = wave_sum(v);
  if constexpr (TPR > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (F)red[0];
#pragma unroll
    for (int i = 1; i < TPR / 64; i++) v = MAX ? (F)fmax(v, (F)red[i]) : v + (F)red[i];
  }
  return v;
}

// Values c .. c + 7 of a row, zero past C; with a residual, the rounded sum (also stored, past the caches
// where it is not read again).
template <bool STREAM = true, typename T>
__device__ __forceinline__ void take8(const NormArgs& a, const T* x, const T* r, T* s, int c, float (&f)[8]) {
  if (c + 8 <= a.C) {
    load8(x + c, f);
    if (r) {
      float g[8];
      load8(r + c, g);
#pragma unroll
      for (int i = 0; i < 8; i++) f[i] = (float)(T)(f[i] + g[i]);
      if (s) {
        if constexpr (STREAM) stream8(s + c, f);
        else store8(s + c, f);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; i++) {
    f[i] = 0.f;
    if (c + i < a.C) {
      f[i] = (float)x[c + i];
      if (r) {
        f[i] = (float)(T)(f[i] + (float)r[c + i]);
        if (s) s[c + i] = (T)f[i];
      }
    }
  }
}

// 1 / sqrt of a row as two numbers, to 2^-45.
struct Root {
  float hi, lo;
};

// f rstd g to 2^-40 as the nearest fp32 number y and what is left.
__device__ __forceinline__ Root product(float f, Root rstd, float g) {
  const float t = f * rstd.hi, y = t * g;
  const float e = __builtin_fmaf(f, rstd.lo, __builtin_fmaf(f, rstd.hi, -t));
  const float r = __builtin_fmaf(e, g, __builtin_fmaf(t, g, -y)), z = y + r;
  return fabsf(y) < __builtin_inff() ? Root{z, r - (z - y)} : Root{y, 0.f};
}

// The product as the neighbour with an odd last bit where it lies between two fp32 numbers: rounded again,
// to a code or past a scale's limit, it goes where the exact product would.
__device__ __forceinline__ float product_odd(float f, Root rstd, float g) {
  const Root y = product(f, rstd, g);
  const int z = __float_as_int(y.hi), away = (unsigned)(z ^ __float_as_int(y.lo)) >> 31;   // 1: the product is nearer 0
  return y.lo != 0.f ? __int_as_float((z - away) | 1) : y.hi;
}

// The output of values c .. c + 7: a 16-lane row holds a block of 128.
template <typename T, bool NORM, bool Q8>
__device__ __forceinline__ void give8(const NormArgs& a, int64_t row, int c, Root rstd, float (&f)[8]) {
  if constexpr (NORM) {
    float g[8], x[8];
    if (c + 8 <= a.C) {
      load8(a.gamma + c, g);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) g[i] = c + i < a.C ? a.gamma[c + i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
      x[i] = f[i];
      f[i] = x[i] * rstd.hi * g[i];   // within three last places of the product: enough for 16 bits
    }
    if constexpr (Q8) {
      // What codes and scales round at has 19 zero bits at its end: only values within three of such a number
      // need more (a wave in 100; zeros do, too). Of 67 million codes about 8 then differ from exact
      // arithmetic's (what fp32 sums of squares leave), 43 without, for 2 us of 71.
      unsigned least = ~0u;
#pragma unroll
      for (int i = 0; i < 8; i++) least = min(least, ((unsigned)__float_as_int(f[i]) + 3u) << 13);
      if (__any(c < a.C && least <= 6u << 13)) {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = product_odd(x[i], rstd, g[i]);
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; i++) f[i] = product(x[i], rstd, g[i]).hi;
    }
  }
  if constexpr (Q8) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(f[i]));
    m = row16_max(m);
    const int b = scale_byte(m);
    const float inv = inverse_of(b);
    if (c < a.kb * kBlock8) {
      const i32x2 w = {encode4(f[0], f[1], f[2], f[3], inv), encode4(f[4], f[5], f[6], f[7], inv)};
      __builtin_nontemporal_store(w, reinterpret_cast<i32x2*>(a.codes + row * a.cp + c));
      if (c % kBlock8 == 0) a.scales[row * a.ep + c / kBlock8] = (uint8_t)b;
    }
  } else {
    T* y = (T*)a.y + row * a.yp;
    if (c + 8 <= a.C) {
      stream8(y + c, f);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (c + i < a.C) y[c + i] = (T)f[i];
    }
  }
}

// 1 / sqrt(mean + eps) of a row from its sum of squares, for values that are first multiplied by g: 1
// but where the squares pass fp32 although the values do not (bf16 and fp32 beyond 2^64 / sqrt(C));
// there the power of two that brings the largest value to 1..4, and the squares are taken again. (Squares
// below fp32 are nothing beside eps, 1e-30 at least.)
template <int TPR, typename Square>
__device__ __forceinline__ Root row_rstd(const NormArgs& a, double ss, float amax, double* red, float& g,
                                         Square squares) {
  g = 1.f;
  if (!(ss <= 3.0e38)) {   // uniform over the row's threads
    amax = row_reduce<TPR, true>(amax, red);
    if (amax < __builtin_inff()) {
      g = inverse_of(min(max(__float_as_int(amax) >> 23, 1), 253));
      ss = row_reduce<TPR, false>((double)squares(g), red);
    }
  }
  const double v = ss * a.per_C + (double)a.eps * g * g, r = __builtin_amdgcn_rsqf((float)v);
  const double s = r + 0.5 * r * (1.0 - v * r * r);   // a step of Newton's from fp32's root
  const float hi = (float)s;
  return v < __builtin_inf() ? Root{hi, (float)(s - hi)} : Root{(float)r, 0.f};
}

template <int N>
__device__ __forceinline__ void times(float (&f)[N], float g) {
  if (g != 1.f)
#pragma unroll
    for (int i = 0; i < N; i++) f[i] *= g;
}

// TPR threads a row, NCH groups of eight consecutive values each; NCH = 0 takes rows of any length and
// reads them twice.
template <typename T, int TPR, int NCH, bool NORM, bool Q8>
__global__ __launch_bounds__(256) void norm8_kernel(NormArgs a) {
  __shared__ double red[4];
  constexpr int RPB = 256 / TPR;
  const int t = threadIdx.x % TPR;
  const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * RPB + threadIdx.x / TPR;
  if (row >= a.rows) return;   // whole waves
  const T* x = (const T*)a.x + row * a.xp;
  const T* r = a.r ? (const T*)a.r + row * a.rp : nullptr;
  T* s = a.s ? (T*)a.s + row * a.sp : nullptr;
  if constexpr (NCH > 0) {
    float f[NCH][8];
    float ss = 0.f, amax = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; k++) take8(a, x, r, s, (k * TPR + t) * 8, f[k]);
    Root rstd = {1.f, 0.f};
    float g = 1.f;
    if constexpr (NORM) {
#pragma unroll
      for (int k = 0; k < NCH; k++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
          ss += f[k][i] * f[k][i];
          amax = fmaxf(amax, fabsf(f[k][i]));
        }
      rstd = row_rstd<TPR>(a, row_reduce<TPR, false>((double)ss, red), amax, red, g, [&](float by) {
        float q = 0.f;
#pragma unroll
        for (int k = 0; k < NCH; k++)
#pragma unroll
          for (int i = 0; i < 8; i++) q += (f[k][i] * by) * (f[k][i] * by);
        return q;
      });
#pragma unroll
      for (int k = 0; k < NCH; k++) times(f[k], g);
    }
#pragma unroll
    for (int k = 0; k < NCH; k++) give8<T, NORM, Q8>(a, row, (k * TPR + t) * 8, rstd, f[k]);
  } else {
    // Whole workgroup rounds, so that the lanes of a block of 128 stay together.
    const int rounds = (a.kb * kBlock8 + TPR * 8 - 1) / (TPR * 8);
    Root rstd = {1.f, 0.f};
    float g = 1.f;
    if constexpr (NORM) {
      // Eights in fp32 and their sum in fp64, however many there are.
      double ss = 0.0;
      float amax = 0.f, f[8];
      for (int k = 0; k < rounds; k++) {
        take8<false>(a, x, r, s, (k * TPR + t) * 8, f);
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          q += f[i] * f[i];
          amax = fmaxf(amax, fabsf(f[i]));
        }
        ss += q;
      }
      // Read again: the sum that this thread stored, since it may have been stored over x or r.
      const T* x2 = r && s ? s : x;
      const T* r2 = r && s ? nullptr : r;
      rstd = row_rstd<TPR>(a, row_reduce<TPR, false>(ss, red), amax, red, g, [&](float by) {
        double all = 0.0;
        float h[8];
        for (int k = 0; k < rounds; k++) {
          take8(a, x2, r2, (T*)nullptr, (k * TPR + t) * 8, h);
          float q = 0.f;
#pragma unroll
          for (int i = 0; i < 8; i++) q += (h[i] * by) * (h[i] * by);
          all += q;
        }
        return all;
      });
      for (int k = 0; k < rounds; k++) {
        take8(a, x2, r2, (T*)nullptr, (k * TPR + t) * 8, f);
        times(f, g);
        give8<T, NORM, Q8>(a, row, (k * TPR + t) * 8, rstd, f);
      }
    } else {
      float f[8];
      for (int k = 0; k < rounds; k++) {
        take8(a, x, r, s, (k * TPR + t) * 8, f);
        give8<T, NORM, Q8>(a, row, (k * TPR + t) * 8, rstd, f);
      }
    }
  }
  if constexpr (Q8)   // the bytes that pad a row's scales to four: 1.0
    if (t < (int)(-a.kb & 3)) a.scales[row * a.ep + a.kb + t] = 127;
}

template <typename T, bool NORM, bool Q8>
void launch(const NormArgs& a, hipStream_t st) {
  const int n = Q8 ? a.kb * kBlock8 : a.C;
  // (A launch's axis takes 2^32 threads.)
  const auto grid = [](int64_t n) { return n <= 1 << 22 ? dim3((unsigned)n) : dim3(1 << 22, (unsigned)((n + (1 << 22) - 1) >> 22)); };
  const dim3 wide = grid(a.rows), narrow = grid((a.rows + 3) / 4), block(256);
  if (n <= 512)
    hipLaunchKernelGGL((norm8_kernel<T, 64, 1, NORM, Q8>), narrow, block, 0, st, a);
  else if (n <= 1024)
    hipLaunchKernelGGL((norm8_kernel<T, 64, 2, NORM, Q8>), narrow, block, 0, st, a);
  else if (n <= 2048)
    hipLaunchKernelGGL((norm8_kernel<T, 256, 1, NORM, Q8>), wide, block, 0, st, a);
  else if (n <= 4096)
    hipLaunchKernelGGL((norm8_kernel<T, 256, 2, NORM, Q8>), wide, block, 0, st, a);
  else if (n <= 8192)
    hipLaunchKernelGGL((norm8_kernel<T, 256, 4, NORM, Q8>), wide, block, 0, st, a);
  else
    hipLaunchKernelGGL((norm8_kernel<T, 256, 0, NORM, Q8>), wide, block, 0, st, a);
}

template <bool NORM, bool Q8>
int launch_any(const NormArgs& a, int dtype, hipStream_t st, const char* what) {
  if (dtype == LDX_DTYPE_F16) launch<f16, NORM, Q8>(a, st);
  else if (dtype == LDX_DTYPE_BF16) launch<bf16, NORM, Q8>(a, st);
  else launch<float, NORM, Q8>(a, st);
  return check_launch(what);
}

// Rows of `rows` elements apart by `pitch` within one allocation that int64 byte offsets reach.
int check_rows(const char* what, int64_t rows, int64_t features, int dtype) {
  if (dtype != LDX_DTYPE_F16 && dtype != LDX_DTYPE_BF16 && dtype != LDX_DTYPE_F32)
    return fail("%s: dtype %d is not LDX_DTYPE_F16, LDX_DTYPE_BF16 or LDX_DTYPE_F32", what, dtype);
  if (rows < 1 || rows > 0x7fffffff) return fail("%s: %lld rows", what, (long long)rows);
  if (features < 1 || features > (1 << 28)) return fail("%s: %lld features", what, (long long)features);
  return LDX_OK;
}

int check_codes(const char* what, const void* codes, int64_t cp, const void* scales, int64_t ep, int kb) {
  if (!scales) return fail("%s: null pointer", what);
  if (cp < (int64_t)kb * kBlock8 || cp % 16 || ep < ((kb + 3) & ~3) || ep % 4)
    return fail("%s: pitches %lld, %lld do not hold %d blocks of %d", what, (long long)cp, (long long)ep, kb, kBlock8);
  if ((uintptr_t)codes % 16 || (uintptr_t)scales % 4) return fail("%s: codes or scales not aligned", what);
  return LDX_OK;
}

}  // namespace
}  // namespace ldx

using namespace ldx;

extern "C" int ldx_rms_norm(const ldx_rms_norm_args* p, void* stream) {
  if (!p || !p->x || !p->gamma || (!p->y && !p->codes)) return fail("rms_norm: null pointer");
  if (int rc = check_rows("rms_norm", p->rows, p->features, p->dtype)) return rc;
  if (p->y && p->codes) return fail("rms_norm: one output, y or codes");
  if (p->sum && !p->residual) return fail("rms_norm: a sum needs a residual");
  const int C = p->features, kb = (C + kBlock8 - 1) / kBlock8;
  if (p->x_pitch < C || (p->residual && p->residual_pitch < C) || (p->sum && p->sum_pitch < C) ||
      (p->y && p->y_pitch < C))
    return fail("rms_norm: row pitch below %d features", C);
  if (!(p->eps >= 1e-30f && p->eps <= 1e30f)) return fail("rms_norm: eps %g", (double)p->eps);
  if (p->codes)
    if (int rc = check_codes("rms_norm", p->codes, p->codes_pitch, p->scales, p->scales_pitch, kb)) return rc;
  const NormArgs a = {p->x, p->x_pitch, p->residual, p->residual_pitch, p->sum, p->sum_pitch, p->gamma, p->eps,
                      p->y, p->y_pitch, (uint8_t*)p->codes, p->codes_pitch, (uint8_t*)p->scales, p->scales_pitch,
                      p->rows, C, kb, 1.0 / C};
  hipStream_t st = as_stream(stream);
  return p->codes ? launch_any<true, true>(a, p->dtype, st, "rms_norm")
                  : launch_any<true, false>(a, p->dtype, st, "rms_norm");
}

extern "C" int ldx_quantize8(const void* x, int64_t xp, int64_t rows, int32_t features, int32_t dtype, void* codes,
                             int64_t cp, void* scales, int64_t ep, void* stream) {
  if (!x || !codes) return fail("quantize8: null pointer");
  if (int rc = check_rows("quantize8", rows, features, dtype)) return rc;
  const int kb = (features + kBlock8 - 1) / kBlock8;
  if (xp < features) return fail("quantize8: row pitch below %d features", features);
  if (int rc = check_codes("quantize8", codes, cp, scales, ep, kb)) return rc;
  NormArgs a = {};
  a.x = x; a.xp = xp;
  a.codes = (uint8_t*)codes; a.cp = cp;
  a.scales = (uint8_t*)scales; a.ep = ep;
  a.rows = rows; a.C = features; a.kb = kb;
  return launch_any<false, true>(a, dtype, as_stream(stream), "quantize8");
}
