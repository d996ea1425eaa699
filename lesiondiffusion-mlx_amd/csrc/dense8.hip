// Products of 8-bit rows: y = act(x w^T + bias + residual), x and w e4m3 codes with a power of two per
// row and 128 columns.
#include "quant8.h"

namespace ldx {
namespace {

struct Dense8Args {
  const uint8_t* x; int64_t xp;
  const uint8_t* xs; int64_t xsp;
  const uint8_t* w; int64_t wp;
  const uint8_t* ws; int64_t wsp;
  const float* bias;
  const void* res; int64_t rp;
  void* y; int64_t yp;
  int64_t M;
  int O, kb, act, dtype;
};

__device__ __forceinline__ float gelu_f(float v) { return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f)); }

__device__ __forceinline__ float act_f(float v, int act) {
  if (act == LDX_ACT_GELU) return gelu_f(v);
  if (act == LDX_ACT_SILU) return v / (1.0f + expf(-v));
  return v;
}

// Eight codes with their scale (its power of two, as fp32) as bf16 values: both fit exactly.
__device__ __forceinline__ bf16x8 widen8(int lo, int hi, float s) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
  return (bf16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// D(16 x 16) += A(16 x 128) B(128 x 16) of one block of 128: lane l holds 32 codes of A row l % 16 and of
// B column l % 16 and the scale bytes of that row and column (all four quarters of k share them, so the
// order of k within the block is free as long as A and B agree); D column l % 16, rows 4 (l / 16) + i.
// EXACT: the same from bf16 operands, whose products the instruction adds within 24 bits.
template <bool EXACT>
__device__ __forceinline__ f32x4 block16(i32x8 a, i32x8 b, f32x4 c, int sa, int sb) {
  if constexpr (!EXACT) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
  } else {
    const float fa = scale_of(sa), fb = scale_of(sb);
#pragma unroll
    for (int i = 0; i < 4; i++)
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(a[2 * i], a[2 * i + 1], fa),
                                                  widen8(b[2 * i], b[2 * i + 1], fb), c, 0, 0, 0);
    return c;
  }
}

template <typename T>
__device__ __forceinline__ void finish(const Dense8Args& a, int64_t m, int o, float v) {
  if (a.bias) v += a.bias[o];
  if (a.res) v += (float)((const T*)a.res)[m * a.rp + o];
  ((T*)a.y)[m * a.yp + o] = (T)act_f(v, a.act);
}

// One 16 x 16 tile a workgroup, its blocks of 128 dealt to the waves and their sums added in wave order.
constexpr int kTileWaves = 4;

template <typename T>
__global__ __launch_bounds__(64 * kTileWaves) void dense8_tile_kernel(Dense8Args a) {
  constexpr bool EXACT = sizeof(T) == 4;
  __shared__ float part[kTileWaves][16][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const unsigned no = (unsigned)(a.O + 15) / 16;
  const int64_t m0 = (int64_t)(blockIdx.x / no) * 16;
  const int o0 = (int)(blockIdx.x % no) * 16;
  const int64_t m = m0 + r < a.M ? m0 + r : a.M - 1;
  const int o = o0 + r < a.O ? o0 + r : a.O - 1;
  const uint8_t* w = a.w + o * a.wp + 16 * g;
  const uint8_t* x = a.x + m * a.xp + 16 * g;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int k = wave; k < a.kb; k += kTileWaves) {
    i32x8 A, B;
    reinterpret_cast<i32x4*>(&A)[0] = *reinterpret_cast<const i32x4*>(w + k * kBlock8);
    reinterpret_cast<i32x4*>(&A)[1] = *reinterpret_cast<const i32x4*>(w + k * kBlock8 + 64);
    reinterpret_cast<i32x4*>(&B)[0] = *reinterpret_cast<const i32x4*>(x + k * kBlock8);
    reinterpret_cast<i32x4*>(&B)[1] = *reinterpret_cast<const i32x4*>(x + k * kBlock8 + 64);
    acc = block16<EXACT>(A, B, acc, a.ws[o * a.wsp + k], a.xs[m * a.xsp + k]);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) part[wave][r][4 * g + i] = acc[i];
  __syncthreads();
  const int tm = threadIdx.x >> 4, to = threadIdx.x & 15;
  float v = part[0][tm][to];
#pragma unroll
  for (int i = 1; i < kTileWaves; i++) v += part[i][tm][to];
  if (m0 + tm < a.M && o0 + to < a.O) finish<T>(a, m0 + tm, o0 + to, v);
}

template <typename T>
void launch(const Dense8Args& a, hipStream_t st) {
  const int64_t tiles = (a.M + 15) / 16 * ((a.O + 15) / 16);
  hipLaunchKernelGGL(dense8_tile_kernel<T>, dim3((unsigned)tiles), dim3(64 * kTileWaves), 0, st, a);
}

int check_operand(const char* name, const void* codes, int64_t cp, const void* scales, int64_t sp, int kb) {
  if (!codes || !scales) return fail("dense8: null pointer");
  if (cp < (int64_t)kb * kBlock8 || cp % 16 || sp < ((kb + 3) & ~3) || sp % 4)
    return fail("dense8: %s pitches %lld, %lld do not hold %d blocks of %d", name, (long long)cp, (long long)sp, kb,
                kBlock8);
  if ((uintptr_t)codes % 16 || (uintptr_t)scales % 4) return fail("dense8: %s codes or scales not aligned", name);
  return LDX_OK;
}

}  // namespace
}  // namespace ldx

using namespace ldx;

extern "C" int ldx_dense8(const ldx_dense8_args* p, void* stream) {
  if (!p || !p->y) return fail("dense8: null pointer");
  if (p->rows < 1 || p->rows > 0x7fffffff || p->features < 1 || p->features > (1 << 28) || p->out_features < 1 ||
      p->out_features > (1 << 28))
    return fail("dense8: %lld rows, %d features, %d outputs", (long long)p->rows, p->features, p->out_features);
  if (p->dtype != LDX_DTYPE_F16 && p->dtype != LDX_DTYPE_BF16 && p->dtype != LDX_DTYPE_F32)
    return fail("dense8: dtype %d is not LDX_DTYPE_F16, LDX_DTYPE_BF16 or LDX_DTYPE_F32", p->dtype);
  if (p->act != LDX_ACT_NONE && p->act != LDX_ACT_GELU && p->act != LDX_ACT_SILU) return fail("dense8: act %d", p->act);
  if ((p->rows + 15) / 16 * ((p->out_features + 15) / 16) > 0x7fffffff)
    return fail("dense8: %lld x %d outputs are more than one launch takes", (long long)p->rows, p->out_features);
  const int kb = (p->features + kBlock8 - 1) / kBlock8;
  if (int rc = check_operand("x", p->x_codes, p->x_pitch, p->x_scales, p->x_scales_pitch, kb)) return rc;
  if (int rc = check_operand("w", p->w_codes, p->w_pitch, p->w_scales, p->w_scales_pitch, kb)) return rc;
  if (p->y_pitch < p->out_features || (p->residual && p->residual_pitch < p->out_features))
    return fail("dense8: row pitch below %d outputs", p->out_features);
  const Dense8Args a = {(const uint8_t*)p->x_codes, p->x_pitch, (const uint8_t*)p->x_scales, p->x_scales_pitch,
                        (const uint8_t*)p->w_codes, p->w_pitch, (const uint8_t*)p->w_scales, p->w_scales_pitch,
                        p->bias, p->residual, p->residual_pitch, p->y, p->y_pitch, p->rows, p->out_features, kb,
                        p->act, p->dtype};
  hipStream_t st = as_stream(stream);
  if (p->dtype == LDX_DTYPE_F16) launch<f16>(a, st);
  else if (p->dtype == LDX_DTYPE_BF16) launch<bf16>(a, st);
  else launch<float>(a, st);
  return check_launch("dense8");
}
