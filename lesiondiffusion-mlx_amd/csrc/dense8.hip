// Products of 8-bit rows: y = act(x w^T + bias + residual), x and w e4m3 codes with a power of two per
// row and 128 columns.
#include <type_traits>

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

// exp(-x) as 2^hi * (1 + lo), lo the part of x log2(e) that its rounding to hi left.
__device__ __forceinline__ float exp_neg(float x) {
  const float hi = x * -1.44269504f;
  const float lo = __builtin_fmaf(x, -1.44269504f, -hi) - x * 1.92596299e-8f;
  return __builtin_amdgcn_exp2f(hi) * __builtin_fmaf(lo, 0.693147181f, 1.0f);
}

// GELU without the cancellation of 1 + erf for negative v: v Q(|v|) there and v (1 - Q(v)) otherwise,
// Q(v) = erfc(v / sqrt 2) / 2 = t exp(p(t) - v^2 / 2) / 2, t = 1 / (1 + 0.4 v / sqrt 2), where p is a
// least-squares Chebyshev fit of log(erfc(x) exp(x^2) / t) for x up to 12 (to 1.1e-7; beyond 64 Q is 0 and v
// itself must not be squared). Branchless: the library's erff and expf in the eight-wide epilogue were 20 KB
// of code.
__device__ __forceinline__ float gelu_f(float v) {
  const float u = fminf(fabsf(v), 64.f), t = __builtin_amdgcn_rcpf(__builtin_fmaf(u, 0.4f * 0.70710678f, 1.0f));
  float p = -0.213728147f;
  p = __builtin_fmaf(p, t, 0.955197486f);
  p = __builtin_fmaf(p, t, -1.5495496f);
  p = __builtin_fmaf(p, t, 1.07216591f);
  p = __builtin_fmaf(p, t, -0.493939286f);
  p = __builtin_fmaf(p, t, 0.321830446f);
  p = __builtin_fmaf(p, t, 0.394323262f);
  p = __builtin_fmaf(p, t, 1.00245476f);
  p = __builtin_fmaf(p, t, -1.48875494f);
  const float hu = 0.5f * u, sq = hu * u, rest = __builtin_fmaf(hu, u, -sq);   // v^2 / 2 = sq + rest
  const float e = exp_neg(sq) * __builtin_amdgcn_exp2f((p - rest) * 1.44269504f);
  const float q = 0.5f * t * e;
  return v * (v < 0.f ? q : 1.0f - q);
}

// v / (1 + exp(-v)); 0 from where exp(-v) passes fp32, v = -88.72 (values of 3e-37 and less). The divisor is quartered:
// from v = -87.34 on its reciprocal is no normal number, and v_rcp_f32 gives 0 for such.
__device__ __forceinline__ float silu8_f(float v) {
  const float e = exp_neg(fminf(fmaxf(v, -120.f), 120.f));   // beyond: 0 and v
  return v * (0.25f * __builtin_amdgcn_rcpf(__builtin_fmaf(0.25f, e, 0.25f)));
}

__device__ __forceinline__ float act_f(float v, int act) {
  if (act == LDX_ACT_GELU) return gelu_f(v);
  if (act == LDX_ACT_SILU) return silu8_f(v);
  return v;
}

// Eight codes with their scale (its power of two, as fp32, of whose bits the conversion takes the byte: 0 is 2^-127 and
// 255 NaN) as bf16 values, which hold them exactly from 2^-130 to 2^128; digits below 2^-133 are rounded off.
__device__ __forceinline__ bf16x8 widen8(int lo, int hi, float s) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
  return (bf16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Outputs o .. o + 7 of row m, as many as there are.
template <typename T>
__device__ __forceinline__ void finish8(const Dense8Args& a, int64_t m, int o, float (&v)[8]) {
  T* y = (T*)a.y + m * a.yp + o;
  if (o + 8 <= a.O) {
    float f[8];
    if (a.bias) {
      load8(a.bias + o, f);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] += f[i];
    }
    if (a.res) {
      load8((const T*)a.res + m * a.rp + o, f);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] += f[i];
    }
    if (a.act == LDX_ACT_GELU) {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = gelu_f(v[i]);
    } else if (a.act == LDX_ACT_SILU) {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = silu8_f(v[i]);
    }
    if constexpr (sizeof(T) == 2) stream8(y, v);   // (fp32's lines leave in two halves: 167 -> 220 us)
    else store8(y, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (o + i >= a.O) break;
      float f = v[i];
      if (a.bias) f += a.bias[o + i];
      if (a.res) f += (float)((const T*)a.res)[m * a.rp + o + i];
      y[i] = (T)act_f(f, a.act);
    }
  }
}

// The tile of workgroup l of nt x mt. Workgroups l and l + 8 share an XCD: each XCD gets a contiguous range
// of tiles, in which bands of four rows of tiles run along the outputs, so that what it holds at a time is
// near a square.
__device__ __forceinline__ void tile_of(unsigned l, unsigned nt, unsigned mt, unsigned& tm, unsigned& tn) {
  const unsigned tiles = nt * mt, x = l % 8, per = tiles / 8, extra = tiles % 8;
  const unsigned idx = x * per + (x < extra ? x : extra) + l / 8;
  constexpr unsigned BAND = 4;
  const unsigned band = idx / (BAND * nt), first = band * BAND;
  const unsigned high = mt - first < BAND ? mt - first : BAND, in = idx - band * BAND * nt;
  tm = first + in % high;
  tn = in / high;
}

// ----------------------------------------------------------------------------------- few tiles
//
// Where few tiles launch, a block's turn (DMA, barrier, LDS reads, a handful of products) is bound by its
// latencies, not by any rate. Here a workgroup's W waves take blocks of k of their own: each has a ring of
// S blocks (32 FN outputs + 32 FM rows of 128 bytes, swizzled as below), no barrier until the end, and the
// sums of the whole tile, which are added through LDS in wave order.
// (64 x 4,096 x 4,096 7.4 us, 18 with the shared blocks of the next kernel; 77 x 768 x 512 4.6 and 5.7. With a few rows
// most of a block's places are empty, and 4,096 outputs are 128 workgroups, on half of the CUs: 4 x 4,096 x 4,096 6.0.)
template <int FN, int FM, int W, int S>
struct SplitTile {
  static constexpr int TN = 32 * FN, TM = 32 * FM;
  static constexpr int DATA = (TN + TM) * kBlock8, SLOT = DATA + 512;   // 64 dwords of scales each
  static constexpr int DMAS = 4 * (FN + FM) + 2;
  static constexpr int PITCH = TN + 4, OUT = W * TM * PITCH * 4;
  static constexpr int RING = W * S * SLOT, LDS = RING > OUT ? RING : OUT;
  static_assert(LDS <= 160 * 1024, "tile");
};

template <typename T, int FN, int FM, int W, int S>
__global__ __launch_bounds__(64 * W) void dense8_split_kernel(Dense8Args a, unsigned nt, unsigned mt) {
  typedef SplitTile<FN, FM, W, S> B;
  constexpr bool EXACT = sizeof(T) == 4;
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, h = lane >> 5;
  unsigned tm, tn;
  tile_of(blockIdx.x, nt, mt, tm, tn);
  const int64_t m0 = (int64_t)tm * B::TM;
  const int o0 = (int)tn * B::TN;
  const int mrows = (int)(a.M - m0 < B::TM ? a.M - m0 : B::TM), orows = a.O - o0 < B::TN ? a.O - o0 : B::TN;
  // Rows past the operand's last read as zeros (the buffer ends there).
  const i32x4 wr = dma_rsrc(a.w + o0 * a.wp, (unsigned)(orows * a.wp));
  const i32x4 xr = dma_rsrc(a.x + m0 * a.xp, (unsigned)(mrows * a.xp));
  const i32x4 wsr = dma_rsrc(a.ws + o0 * a.wsp, (unsigned)(orows * a.wsp));
  const i32x4 xsr = dma_rsrc(a.xs + m0 * a.xsp, (unsigned)(mrows * a.xsp));
  uint8_t* ring = lds + wave * S * B::SLOT;
  const unsigned base = lds_offset(ring);
  unsigned wv[2], xv[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const unsigned row = 8 * i + lane / 8, unit = (lane % 8) ^ (row / 2 % 8);
    wv[i] = lane / 8 * (unsigned)a.wp + unit * 16;
    xv[i] = lane / 8 * (unsigned)a.xp + unit * 16;
  }
  const int steps = (a.kb - wave + W - 1) / W;   // blocks wave, wave + W, ..
  const auto fetch = [&](int i) {
    const unsigned k = wave + W * i, to = base + i % S * B::SLOT, at = k * kBlock8;
    dma_buffer_b32(wsr, lane * (unsigned)a.wsp, k & ~3u, to + B::DATA);
    dma_buffer_b32(xsr, lane * (unsigned)a.xsp, k & ~3u, to + B::DATA + 256);
#pragma unroll
    for (int e = 0; e < 4 * FN; e++) dma_buffer_b128(wr, wv[e & 1], e * 8 * (unsigned)a.wp + at, to + e * 1024);
#pragma unroll
    for (int e = 0; e < 4 * FM; e++) dma_buffer_b128(xr, xv[e & 1], e * 8 * (unsigned)a.xp + at, to + (4 * FN + e) * 1024);
  };
  f32x16 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; i++)
#pragma unroll
    for (int j = 0; j < FM; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;
  unsigned unit[4];
#pragma unroll
  for (int p = 0; p < 4; p++) unit[p] = (unsigned)r * kBlock8 + (((2 * p + h) ^ (r / 2 % 8)) * 16);

#pragma unroll
  for (int i = 0; i < S; i++)
    if (i < steps) fetch(i);
  for (int i = 0; i < steps; i++) {
    if (S > 1 && i + S <= steps) vmcnt_wait<(S - 1) * B::DMAS>();   // block i has come, S - 1 are on their way
    else vmcnt_wait<0>();
    asm volatile("" ::: "memory");
    const uint8_t* s = ring + i % S * B::SLOT;
    i32x8 fr[2][FN + FM];
    int sc[FN + FM];
#pragma unroll
    for (int f = 0; f < FN + FM; f++) {
#pragma unroll
      for (int p = 0; p < 4; p++) {
        const i32x4 v = *reinterpret_cast<const i32x4*>(s + f * 32 * kBlock8 + unit[p]);
#pragma unroll
        for (int e = 0; e < 4; e++) fr[p / 2][f][p % 2 * 4 + e] = v[e];
      }
      const int row = f < FN ? f * 32 + r : 64 + (f - FN) * 32 + r;
      sc[f] = reinterpret_cast<const int*>(s + B::DATA)[row] >> (8 * ((wave + W * i) & 3));
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);   // the reads have returned: the slot is free
    asm volatile("" ::: "memory");
    if (i + S < steps) fetch(i + S);
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
      for (int f = 0; f < FN; f++)
#pragma unroll
        for (int j = 0; j < FM; j++) {
          if constexpr (!EXACT) {
            acc[f][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fr[c][f], fr[c][FN + j], acc[f][j], 0, 0, 0, sc[f],
                                                                       0, sc[FN + j]);
          } else {
#pragma unroll
            for (int p = 0; p < 4; p++)
              acc[f][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                  widen8(fr[c][f][2 * p], fr[c][f][2 * p + 1], scale_of(sc[f] & 255)),
                  widen8(fr[c][FN + j][2 * p], fr[c][FN + j][2 * p + 1], scale_of(sc[FN + j] & 255)), acc[f][j], 0, 0, 0);
          }
        }
#pragma unroll
    for (int f = 0; f < FN; f++)
#pragma unroll
      for (int j = 0; j < FM; j++) asm volatile("" : "+a"(acc[f][j]));
  }

  ring_barrier();
  float* out = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int f = 0; f < FN; f++)
#pragma unroll
    for (int j = 0; j < FM; j++)
#pragma unroll
      for (int q = 0; q < 4; q++)
        *reinterpret_cast<f32x4*>(out + (wave * B::TM + j * 32 + r) * B::PITCH + f * 32 + 8 * q + 4 * h) =
            (f32x4){acc[f][j][4 * q], acc[f][j][4 * q + 1], acc[f][j][4 * q + 2], acc[f][j][4 * q + 3]};
  __syncthreads();
  for (int e = threadIdx.x; e < B::TM * 4 * FN; e += 64 * W) {
    const int row = e / (4 * FN), col = e % (4 * FN) * 8;
    if (row >= mrows || col >= orows) continue;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; w++) {
      const f32x4* p = reinterpret_cast<const f32x4*>(out + (w * B::TM + row) * B::PITCH + col);
      const f32x4 lo = p[0], hi = p[1];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        v[i] += lo[i];
        v[4 + i] += hi[i];
      }
    }
    finish8<T>(a, m0 + row, o0 + col, v);
  }
}

template <typename T, int FN, int FM, int W, int S>
int launch_split(const Dense8Args& a, hipStream_t st) {
  typedef SplitTile<FN, FM, W, S> B;
  const unsigned nt = (unsigned)((a.O + B::TN - 1) / B::TN), mt = (unsigned)((a.M + B::TM - 1) / B::TM);
  const auto kern = dense8_split_kernel<T, FN, FM, W, S>;
  if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, B::LDS) != hipSuccess)
    return check_launch("dense8: set LDS size");
  hipLaunchKernelGGL(kern, dim3(nt * mt), dim3(64 * W), B::LDS, st, a, nt, mt);
  return check_launch("dense8");
}

// ------------------------------------------------------------------------------ large products
//
// A workgroup of 2 x 2 waves takes 64 FN outputs x 64 FM rows, a wave 32 FN x 32 FM of them in 32 x 32
// accumulators. The operands' rows of a block (128 bytes) come into LDS by DMA, a ring of S stages;
// whole 128-byte lines, since 64-byte pieces arrive at 18 TB/s and lines at 24 (every CU loading from
// L2). Of row r the 16-byte unit u stands at u ^ (r / 2 % 8), so that the 16 lanes which read one unit of
// 16 rows meet all 64 banks once.
//
// With one wave a SIMD nothing else hides what a wave issues between its matrix instructions: the LDS
// reads of the next half block go one by one between the products of this one, and with the second half's
// the DMAs into the stage that all waves have then read.
//
// Scales come by DMA too, four blocks' bytes (a dword a row) at a time.
//
// 8,192 x 4,096 x 8,192 in bf16 207 to 233 us (2.66 to 2.36 PF/s) in 256 x 256 tiles, of which a block's
// turn is 1.28 us and the result's way out 9 us a tile; 2,048^3 12.7 us in 128 x 128 tiles. fp32 results, on
// bf16 instructions, 422 and 25.6 us.

constexpr int kHalf8 = kBlock8 / 2;

template <int FN, int FM, int S>
struct BigTile {
  static constexpr int TN = 64 * FN, TM = 64 * FM;
  static constexpr int STAGE = (TN + TM) * kBlock8;
  static constexpr int SCALES = (TN + TM) * 4;
  static constexpr int DMAS = 2 * (FN + FM);      // 1 KB (8 rows) each, per wave and block
  static constexpr int READS = 2 * (FN + FM);     // per half block
  // The result leaves through LDS: a wave's JP x 32 rows of 32 FN outputs, padded by 16 bytes.
  static constexpr int JP = FN == 4 ? 2 : 1, PITCH = 32 * FN + 4, OUT = 4 * JP * 32 * PITCH * 4;
  static constexpr int GROUPS = S == 2 ? 2 : 4;   // of four blocks' scales; S / 4 + 2 are in use at a time
  static constexpr int RING = S * STAGE + GROUPS * SCALES;
  static constexpr int LDS = RING > OUT ? RING : OUT;
  static_assert(FM % JP == 0 && LDS <= 160 * 1024, "tile");
};

template <typename T, int FN, int FM, int S>
__global__ __launch_bounds__(256) void dense8_big_kernel(Dense8Args a, unsigned nt, unsigned mt) {
  typedef BigTile<FN, FM, S> B;
  constexpr bool EXACT = sizeof(T) == 4;
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, h = lane >> 5, wn = wave >> 1, wm = wave & 1;
  unsigned tm, tn;
  tile_of(blockIdx.x, nt, mt, tm, tn);
  const int64_t m0 = (int64_t)tm * B::TM;
  const int o0 = (int)tn * B::TN;
  const int mrows = (int)(a.M - m0 < B::TM ? a.M - m0 : B::TM), orows = a.O - o0 < B::TN ? a.O - o0 : B::TN;
  // Rows past the operand's last read as zeros (the buffer ends there).
  const i32x4 wr = dma_rsrc(a.w + o0 * a.wp, (unsigned)(orows * a.wp));
  const i32x4 xr = dma_rsrc(a.x + m0 * a.xp, (unsigned)(mrows * a.xp));
  const i32x4 wsr = dma_rsrc(a.ws + o0 * a.wsp, (unsigned)(orows * a.wsp));
  const i32x4 xsr = dma_rsrc(a.xs + m0 * a.xsp, (unsigned)(mrows * a.xsp));
  const unsigned base = lds_offset(lds);
  // A lane's place in a DMA of eight rows; its unit depends on whether the eight is an odd one.
  unsigned wv[2], xv[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const unsigned row = 8 * i + lane / 8, unit = (lane % 8) ^ (row / 2 % 8);
    wv[i] = lane / 8 * (unsigned)a.wp + unit * 16;
    xv[i] = lane / 8 * (unsigned)a.xp + unit * 16;
  }
  const unsigned wstep = 8 * (unsigned)a.wp, xstep = 8 * (unsigned)a.xp;
  // DMA i of this wave for block k.
  const auto dma = [&](int k, int i) {
    const unsigned to = base + (k % S) * B::STAGE, at = k * kBlock8;
    if (i < 2 * FN) {
      const unsigned e = wave * 2 * FN + i;
      dma_buffer_b128(wr, wv[i & 1], e * wstep + at, to + e * 1024);
    } else {
      const unsigned e = wave * 2 * FM + i - 2 * FN;
      dma_buffer_b128(xr, xv[i & 1], e * xstep + at, to + (B::TN / 8 + e) * 1024);
    }
  };
  // Scales of blocks k .. k + 3.
  const auto dma_scales = [&](int k) {
    if (k & 3) return;
    const unsigned to = base + S * B::STAGE + (k / 4 % B::GROUPS) * B::SCALES;
#pragma unroll
    for (int i = 0; i < FN + FM; i++) {
      if (i % 4 != wave) continue;
      const unsigned row = (unsigned)(i * 64 + lane);
      if (i < FN) dma_buffer_b32(wsr, row * (unsigned)a.wsp, (unsigned)k, to + i * 256);
      else dma_buffer_b32(xsr, (row - B::TN) * (unsigned)a.xsp, (unsigned)k, to + i * 256);
    }
  };

  f32x16 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; i++)
#pragma unroll
    for (int j = 0; j < FM; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;

  // Units 2 p + h (p = 0, 1 in the block's first half) of the lane's row of the wave's first fragments.
  unsigned wu[4], xu[4];
#pragma unroll
  for (int p = 0; p < 4; p++) {
    const unsigned u = (unsigned)r * kBlock8 + (((2 * p + h) ^ (r / 2 % 8)) * 16);
    wu[p] = wn * FN * 32 * kBlock8 + u;
    xu[p] = (B::TN + wm * FM * 32) * kBlock8 + u;
  }
  i32x8 fw[2][FN], fx[2][FM];
  // LDS read i of half c of block k.
  const auto read = [&](int k, int c, int i) {
    const uint8_t* s = lds + (k % S) * B::STAGE;
    const int f = i / 2, p = i % 2;
    const i32x4 v = *reinterpret_cast<const i32x4*>(f < FN ? s + wu[2 * c + p] + f * 32 * kBlock8
                                                           : s + xu[2 * c + p] + (f - FN) * 32 * kBlock8);
    i32x8& to = f < FN ? fw[c][f < FN ? f : 0] : fx[c][f < FN ? 0 : f - FN];
#pragma unroll
    for (int e = 0; e < 4; e++) to[4 * p + e] = v[e];
  };
  int sn[FN], sx[FM];
  const auto scales = [&](int k) {
    const int* s = reinterpret_cast<const int*>(lds + S * B::STAGE + (k / 4 % B::GROUPS) * B::SCALES);
#pragma unroll
    for (int i = 0; i < FN; i++) sn[i] = s[(wn * FN + i) * 32 + r];
#pragma unroll
    for (int j = 0; j < FM; j++) sx[j] = s[B::TN + (wm * FM + j) * 32 + r];
  };
  // Products of half c of block k; between them the reads of the half block after it and, with MORE in
  // the second half, the DMAs of block k + S.
  const auto products = [&](int k, auto half, auto more) {
    constexpr int c = decltype(half)::value;
    constexpr bool MORE = c == 1 && decltype(more)::value;
    constexpr int N = EXACT ? 4 : FN * FM;
    const auto beside = [&](int s) {
#pragma unroll
      for (int i = s * B::READS / N; i < (s + 1) * B::READS / N; i++) read(k + c, 1 - c, i);
      if constexpr (MORE)
#pragma unroll
        for (int i = s * B::DMAS / N; i < (s + 1) * B::DMAS / N; i++) dma(k + S, i);
    };
    if constexpr (MORE) dma_scales(k + S);
    if constexpr (!EXACT) {
#pragma unroll
      for (int s = 0; s < N; s++) {
        const int i = s / FM, j = s % FM;
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fw[c][i], fx[c][j], acc[i][j], 0, 0, 0, sn[i], 0,
                                                                   sx[j]);
        beside(s);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int p = 0; p < 4; p++) {
        bf16x8 bw[FN];
#pragma unroll
        for (int i = 0; i < FN; i++) bw[i] = widen8(fw[c][i][2 * p], fw[c][i][2 * p + 1], scale_of(sn[i] & 255));
        beside(p);
#pragma unroll
        for (int j = 0; j < FM; j++) {
          const bf16x8 bx = widen8(fx[c][j][2 * p], fx[c][j][2 * p + 1], scale_of(sx[j] & 255));
#pragma unroll
          for (int i = 0; i < FN; i++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bw[i], bx, acc[i][j], 0, 0, 0);
        }
      }
    }
    // The products stay in this half block: without this the compiler sinks them past the branches below.
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
      for (int j = 0; j < FM; j++) asm volatile("" : "+a"(acc[i][j]));
    if constexpr (c == 1) {
      if ((k & 3) == 3) {
        scales(k + 1);   // past the last block: old bytes, not used
      } else {
#pragma unroll
        for (int i = 0; i < FN; i++) sn[i] = (int)((unsigned)sn[i] >> 8);
#pragma unroll
        for (int j = 0; j < FM; j++) sx[j] = (int)((unsigned)sx[j] >> 8);
      }
    }
  };
  constexpr std::integral_constant<int, 0> half0{};
  constexpr std::integral_constant<int, 1> half1{};

#pragma unroll
  for (int k = 0; k < S; k++)
    if (k < a.kb) {
      dma_scales(k);
#pragma unroll
      for (int i = 0; i < B::DMAS; i++) dma(k, i);
    }
  if (a.kb >= S) vmcnt_wait<(S - 1) * B::DMAS>();
  else vmcnt_wait<0>();
  ring_barrier();
#pragma unroll
  for (int i = 0; i < B::READS; i++) read(0, 0, i);
  scales(0);
  int k = 0;
  for (; k + S < a.kb; k++) {
    products(k, half0, std::true_type{});
    // Block k + 1 has come (S - 2 more are on their way), and behind the barrier every wave has read block k.
    vmcnt_wait<(S - 2) * B::DMAS>();
    ring_barrier();
    products(k, half1, std::true_type{});
  }
  for (; k < a.kb; k++) {   // the last S: the reads past the end take old bytes, not used
    products(k, half0, std::false_type{});
    if (S > 2 && k + S == a.kb) vmcnt_wait<(S - 2) * B::DMAS>();
    else vmcnt_wait<0>();
    ring_barrier();
    products(k, half1, std::false_type{});
  }

  // A lane holds outputs 8 q + 4 h + e of row r of each 32 x 32. Through LDS a wave takes whole rows of its
  // 32 FN outputs, eight to a lane, in one rolled loop (the epilogue unrolled over the accumulators was
  // so much code that a 256 x 256 tile spent 20 us in it).
  ring_barrier();
  float* out = reinterpret_cast<float*>(lds) + wave * B::JP * 32 * B::PITCH;
#pragma unroll
  for (int j0 = 0; j0 < FM; j0 += B::JP) {
#pragma unroll
    for (int j = 0; j < B::JP; j++)
#pragma unroll
      for (int i = 0; i < FN; i++)
#pragma unroll
        for (int q = 0; q < 4; q++)
          *reinterpret_cast<f32x4*>(out + (j * 32 + r) * B::PITCH + i * 32 + 8 * q + 4 * h) =
              (f32x4){acc[i][j0 + j][4 * q], acc[i][j0 + j][4 * q + 1], acc[i][j0 + j][4 * q + 2], acc[i][j0 + j][4 * q + 3]};
    __builtin_amdgcn_wave_barrier();
    constexpr int PER = 4 * FN;   // lanes a row
#pragma unroll 4
    for (int row = lane / PER; row < B::JP * 32; row += 64 / PER) {
      const float* f = out + row * B::PITCH + lane % PER * 8;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = f[e];
      const int64_t m = m0 + (wm * FM + j0) * 32 + row;
      if (m < a.M) finish8<T>(a, m, o0 + wn * FN * 32 + lane % PER * 8, v);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <typename T, int FN, int FM, int S>
int launch_big(const Dense8Args& a, hipStream_t st) {
  typedef BigTile<FN, FM, S> B;
  const unsigned nt = (unsigned)((a.O + B::TN - 1) / B::TN), mt = (unsigned)((a.M + B::TM - 1) / B::TM);
  const auto kern = dense8_big_kernel<T, FN, FM, S>;
  if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, B::LDS) != hipSuccess)
    return check_launch("dense8: set LDS size");
  hipLaunchKernelGGL(kern, dim3(nt * mt), dim3(256), B::LDS, st, a, nt, mt);
  return check_launch("dense8");
}

// Which kernel: the one of least estimated time. A call's time was measured as a sum of a fixed part, one
// for each round of workgroups (places: as many as the CUs hold at once), for each block of a workgroup's
// steps in a round, and for the workgroups and their steps by how full the rounds are -- fitted to 130 random
// shapes (1 to 8,192 rows, 64 to 8,192 features and outputs) per kernel; the choices are within 0.6 % (16-bit
// results) and 1.2 % (fp32) of the fastest on average, 20 % at most. us.
// An activation adds to a round, and to the tiles of the two large ones, what one wave a SIMD takes for all of
// its tile's results: without that 2.8 % from the fastest on average, 54 % at most, with it 1.1 and 31 (GELU).
struct Cost {
  float fixed, round, step, work, tile;   // the last two per full round
  float act, act_tile;
};

constexpr int64_t kMostTiles = 1 << 23;   // of a launch: 2^31 threads

inline double estimate(const Cost& c, bool act, int64_t M, int64_t O, int kb, int tm, int tn, int places, int waves) {
  const double tiles = (double)((M + tm - 1) / tm) * (double)((O + tn - 1) / tn), full = tiles / places;
  if (tiles > (double)kMostTiles && tm < 256) return 1e30;
  const double rounds = (double)(int64_t)(full + 0.999999), steps = (kb + waves - 1) / waves;
  return c.fixed + c.round * rounds + c.step * rounds * steps + c.work * full * steps + c.tile * full +
         (act ? c.act * rounds + c.act_tile * full : 0.0);
}

template <bool EXACT>
int choose(bool act, int64_t M, int64_t O, int kb) {
  constexpr Cost big4 = EXACT ? Cost{9.80f, 2.11f, 2.267f, 0.298f, 14.97f, 15.5f, 3.4f}
                              : Cost{10.78f, 1.97f, 0.981f, 0.299f, 9.03f, 15.5f, 3.4f};
  constexpr Cost big2 = EXACT ? Cost{5.22f, 0.f, 0.740f, 0.654f, 9.33f, 2.8f, 4.4f}
                              : Cost{5.16f, 0.f, 0.411f, 0.546f, 4.85f, 2.8f, 4.4f};
  constexpr Cost big1 = EXACT ? Cost{4.06f, 0.f, 0.366f, 0.169f, 2.83f, 0.9f, 0.3f}
                              : Cost{3.51f, 0.62f, 0.208f, 0.174f, 1.50f, 0.9f, 0.3f};
  constexpr Cost split2 = EXACT ? Cost{3.21f, 1.27f, 1.010f, 0.092f, 1.56f, 0.9f, 0.1f}
                              : Cost{3.10f, 1.60f, 0.677f, 0.192f, 0.80f, 0.9f, 0.1f};
  constexpr Cost split1 = EXACT ? Cost{3.66f, 0.f, 0.468f, 0.267f, 1.16f, 0.5f, 0.f}
                              : Cost{3.65f, 0.01f, 0.339f, 0.327f, 0.91f, 0.5f, 0.f};
  const double t[5] = {estimate(split1, act, M, O, kb, 32, 32, 512, 4), estimate(split2, act, M, O, kb, 64, 64, 256, 4),
                       estimate(big1, act, M, O, kb, 64, 64, 512, 1), estimate(big2, act, M, O, kb, 128, 128, 512, 1),
                       estimate(big4, act, M, O, kb, 256, 256, 256, 1)};
  int best = 0;
  for (int i = 1; i < 5; i++)
    if (t[i] < t[best]) best = i;
  return best;
}

template <typename T>
int launch(const Dense8Args& a, hipStream_t st) {
  switch (choose<sizeof(T) == 4>(a.act != LDX_ACT_NONE, a.M, a.O, a.kb)) {
    case LDX_DENSE8_OWN_32: return launch_split<T, 1, 1, 4, 2>(a, st);
    case LDX_DENSE8_OWN_64: return launch_split<T, 2, 2, 4, 2>(a, st);
    case LDX_DENSE8_SHARED_64: return launch_big<T, 1, 1, 4>(a, st);
    case LDX_DENSE8_SHARED_128: return launch_big<T, 2, 2, 2>(a, st);
    default: return launch_big<T, 4, 4, 2>(a, st);
  }
}

int check_operand(const char* name, const void* codes, int64_t cp, const void* scales, int64_t sp, int kb) {
  if (!codes || !scales) return fail("dense8: null pointer");
  if (cp < (int64_t)kb * kBlock8 || cp > (1 << 22) || cp % 16 || sp < ((kb + 3) & ~3) || sp > (1 << 22) || sp % 4)
    return fail("dense8: %s pitches %lld, %lld do not hold %d blocks of %d", name, (long long)cp, (long long)sp, kb,
                kBlock8);
  if ((uintptr_t)codes % 16 || (uintptr_t)scales % 4) return fail("dense8: %s codes or scales not aligned", name);
  return LDX_OK;
}

int check_call(const ldx_dense8_args* p) {
  if (!p || !p->y) return fail("dense8: null pointer");
  if (p->rows < 1 || p->rows > 0x7fffffff || p->features < 1 || p->features > (1 << 22) || p->out_features < 1 ||
      p->out_features > (1 << 28))
    return fail("dense8: %lld rows, %d features, %d outputs", (long long)p->rows, p->features, p->out_features);
  if (p->dtype != LDX_DTYPE_F16 && p->dtype != LDX_DTYPE_BF16 && p->dtype != LDX_DTYPE_F32)
    return fail("dense8: dtype %d is not LDX_DTYPE_F16, LDX_DTYPE_BF16 or LDX_DTYPE_F32", p->dtype);
  if (p->act != LDX_ACT_NONE && p->act != LDX_ACT_GELU && p->act != LDX_ACT_SILU) return fail("dense8: act %d", p->act);
  if ((p->rows + 255) / 256 * ((p->out_features + 255) / 256) > kMostTiles)
    return fail("dense8: %lld x %d outputs are more than one launch takes", (long long)p->rows, p->out_features);
  const int kb = (p->features + kBlock8 - 1) / kBlock8;
  if (int rc = check_operand("x", p->x_codes, p->x_pitch, p->x_scales, p->x_scales_pitch, kb)) return rc;
  if (int rc = check_operand("w", p->w_codes, p->w_pitch, p->w_scales, p->w_scales_pitch, kb)) return rc;
  if (p->y_pitch < p->out_features || (p->residual && p->residual_pitch < p->out_features))
    return fail("dense8: row pitch below %d outputs", p->out_features);
  return LDX_OK;
}

}  // namespace
}  // namespace ldx

using namespace ldx;

extern "C" int ldx_dense8_kernel(const ldx_dense8_args* p) {
  if (int rc = check_call(p)) return rc;
  const int kb = (p->features + kBlock8 - 1) / kBlock8;
  return p->dtype == LDX_DTYPE_F32 ? choose<true>(p->act != LDX_ACT_NONE, p->rows, p->out_features, kb)
                                   : choose<false>(p->act != LDX_ACT_NONE, p->rows, p->out_features, kb);
}

extern "C" int ldx_dense8(const ldx_dense8_args* p, void* stream) {
  if (int rc = check_call(p)) return rc;
  const int kb = (p->features + kBlock8 - 1) / kBlock8;
  const Dense8Args a = {(const uint8_t*)p->x_codes, p->x_pitch, (const uint8_t*)p->x_scales, p->x_scales_pitch,
                        (const uint8_t*)p->w_codes, p->w_pitch, (const uint8_t*)p->w_scales, p->w_scales_pitch,
                        p->bias, p->residual, p->residual_pitch, p->y, p->y_pitch, p->rows, p->out_features, kb,
                        p->act, p->dtype};
  hipStream_t st = as_stream(stream);
  return p->dtype == LDX_DTYPE_F16 ? launch<f16>(a, st) : p->dtype == LDX_DTYPE_BF16 ? launch<bf16>(a, st) : launch<float>(a, st);
}
