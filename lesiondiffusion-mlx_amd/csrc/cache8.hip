// A cache of keys and values held in 8 bits (quant8.h), in pages of 64 tokens with one scale per page
// and head for the keys and one for the values: writing new tokens, and the attention that reads it.
#include "quant8.h"

namespace ldx {
namespace {

// ---------------------------------------------------------------------------------------- append

struct AppendArgs {
  uint8_t* codes[2];     // keys (pages, H, 64, D), values (pages, H, D, 64)
  uint8_t* scales[2];    // (pages, H)
  const void* src[2];
  int64_t st[2][3];      // batch, token, head strides of the new keys / values
  int pages, H, D, tokens;
  const int32_t* table; int64_t tp; int width;
  const int32_t* starts;
  const int32_t* counts;
};

// A code under scale byte `from` as a code under the larger byte `to`: exact, but for the rounding of
// those that become subnormal.
__device__ __forceinline__ int recode4(int w, int from, int to) {
  const float s = scale_of(max(127 + from - to, 1));   // 2^-126 and less: every code rounds to zero
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  return encode4(lo[0], lo[1], hi[0], hi[1], s);
}

// One page's new tokens of one head, keys or values: their largest magnitude, the page's scale, the
// codes. Values go through LDS, where they are turned channel by token.
template <typename T>
__global__ __launch_bounds__(256) void append8_kernel(AppendArgs a) {
  __shared__ float red[4];
  __shared__ __align__(16) uint8_t turned[256 * 64];
  const int b = blockIdx.z, h = blockIdx.y >> 1, which = blockIdx.y & 1, tid = threadIdx.x;
  const int start = a.starts[b];
  const int n = a.counts ? min(a.counts[b], a.tokens) : a.tokens;
  if (start < 0 || n <= 0) return;
  const int64_t end = (int64_t)start + n;
  const int64_t slot = start / kPage8 + (int64_t)blockIdx.x, first = slot * kPage8;
  if (first >= end || slot >= a.width) return;
  const int page = a.table[b * a.tp + slot];
  if ((unsigned)page >= (unsigned)a.pages) return;
  const int lo = (int)max(start - first, (int64_t)0), hi = (int)min(end - first, (int64_t)kPage8);
  const int units = a.D / 8, chunks = (hi - lo) * units;   // eight channels of a token each
  const T* src = (const T*)a.src[which] + b * a.st[which][0] + (first + lo - start) * a.st[which][1] + h * a.st[which][2];
  const int64_t tok = a.st[which][1];
  float amax = 0.f;
  for (int c = tid; c < chunks; c += 256) {
    float f[8];
    load8(src + c / units * tok + c % units * 8, f);
#pragma unroll
    for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(f[i]));
  }
  amax = wave_max(amax);
  if ((tid & 63) == 0) red[tid >> 6] = amax;
  __syncthreads();
  amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  uint8_t* scale = a.scales[which] + (int64_t)page * a.H + h;
  uint8_t* codes = a.codes[which] + ((int64_t)page * a.H + h) * a.D * kPage8;
  const int was = *scale;
  int to = scale_byte(amax);
  const bool rises = lo > 0 && to > was;
  if (lo > 0 && to < was) to = was;
  const float inv = inverse_of(min(to, 253));
  __syncthreads();   // every thread has read the old scale
  if (tid == 0) *scale = (uint8_t)to;
  if (which == 0) {
    if (rises)
      for (int c = tid; c < lo * a.D / 4; c += 256) {
        int* w = reinterpret_cast<int*>(codes) + c;
        *w = recode4(*w, was, to);
      }
    for (int c = tid; c < chunks; c += 256) {
      float f[8];
      load8(src + c / units * tok + c % units * 8, f);
      const i32x2 w = {encode4(f[0], f[1], f[2], f[3], inv), encode4(f[4], f[5], f[6], f[7], inv)};
      *reinterpret_cast<i32x2*>(codes + (lo + c / units) * a.D + c % units * 8) = w;
    }
    return;
  }
  for (int c = tid; c < chunks; c += 256) {
    float f[8];
    load8(src + c / units * tok + c % units * 8, f);
    const int w0 = encode4(f[0], f[1], f[2], f[3], inv), w1 = encode4(f[4], f[5], f[6], f[7], inv);
    uint8_t* t = turned + c % units * 8 * kPage8 + lo + c / units;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      t[i * kPage8] = (uint8_t)(w0 >> (8 * i));
      t[(i + 4) * kPage8] = (uint8_t)(w1 >> (8 * i));
    }
  }
  __syncthreads();
  // Four tokens of a channel at a time: older ones (re-coded where the scale rises) below lo, new ones
  // up to hi, the rest as it is.
  const int g0 = rises ? 0 : lo / 4, g1 = (hi + 3) / 4, per = g1 - g0;
  for (int c = tid; c < a.D * per; c += 256) {
    const int at = c / per * kPage8 + (g0 + c % per) * 4, t0 = (g0 + c % per) * 4;
    int w = *reinterpret_cast<const int*>(turned + at);
    if (t0 < lo || t0 + 4 > hi) {
      const int old = *reinterpret_cast<const int*>(codes + at);
      const int kept = rises ? recode4(old, was, to) : old;
      unsigned m = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const unsigned byte = 0xffu << (8 * i);
        const unsigned v = t0 + i < lo ? (unsigned)kept : t0 + i < hi ? (unsigned)w : (unsigned)old;
        m |= v & byte;
      }
      w = (int)m;
    }
    *reinterpret_cast<int*>(codes + at) = w;
  }
}

// ------------------------------------------------------------------------------------- attention

struct Attend8Args {
  const uint8_t* k; const uint8_t* v;
  const uint8_t* ks; const uint8_t* vs;
  int pages, H;
  const void* q; int64_t qs[3];
  void* o; int64_t os[3];
  int G, lq, rows;       // query heads per cache head; queries; G * lq
  float scale;           // times log2(e)
  const int32_t* table; int64_t tp; int width;
  const int32_t* lengths;
  const int32_t* starts;
  int splits;
  float* part;           // splits > 1: [b][h][row][split] of D sums, then of (m, l)
};

template <typename T>
struct Vec8;
template <>
struct Vec8<f16> { typedef f16x8 V; };
template <>
struct Vec8<bf16> { typedef bf16x8 V; };

__device__ __forceinline__ f32x4 mfma_q(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_q(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// Eight codes as they stand (scale 1): e4m3's values fit fp16 and bf16 exactly.
__device__ __forceinline__ void codes_as(int lo, int hi, f16x8& r) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
  const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
  r = (f16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ void codes_as(int lo, int hi, bf16x8& r) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
  r = (bf16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The keys that a query sees: limit = min(length, start + i + 1) with starts, the length without.
__device__ __forceinline__ int key_limit(const Attend8Args& a, int len, int64_t start, int row) {
  if (!a.starts) return len;
  const int64_t c = start + row / a.G + 1;
  return (int)(c < 0 ? 0 : c < len ? c : len);
}

// The 0x80 bit of every byte of w that holds a NaN code.
__device__ __forceinline__ unsigned nan_bytes(int w) {
  return (((unsigned)w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// S^T = K Q^T per page, on 16 x 16 x 32 products: lane l holds query column l % 16. Key row m of key tile
// t is the page's token 16 (m / 4) + 4 t + m % 4, so that the scores a lane receives (rows 4 g + i, g =
// l / 16, tiles t = 0..3) are those of tokens 16 g + 4 t + i: sixteen in a row, the order in which a lane
// reads the turned values, and the probabilities go into the second product as they lie.
//
// The scales stay out of the operands: the keys' goes into the softmax scale, the values' onto each page's
// sum as it is added to the running one, so that probabilities (at most 1) are what fp16 rounds.
constexpr int kAttendWaves = 4;

template <typename T, int D>
__global__ __launch_bounds__(64 * kAttendWaves) void attend8_kernel(Attend8Args a) {
  typedef typename Vec8<T>::V V8;
  constexpr int ND = D / 16;              // channel tiles
  constexpr int NK = D / 32;              // products per key tile
  __shared__ float sm[kAttendWaves][16], sl[kAttendWaves][16];
  __shared__ float sacc[kAttendWaves][16][D + 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int b = blockIdx.z, split = blockIdx.x, tiles = (a.rows + 15) / 16;
  const int h = blockIdx.y / tiles, row0 = blockIdx.y % tiles * 16;
  const int row = row0 + r;
  const bool real = row < a.rows;
  const int raw = a.lengths[b];
  const bool too_long = raw > (int64_t)a.width * kPage8;
  const int len = too_long || raw < 0 ? 0 : raw;
  const int64_t start = a.starts ? a.starts[b] : 0;
  const int limit = real ? key_limit(a, len, start, row) : 0;
  const int least = key_limit(a, len, start, row0);                                // the tile's first row
  const int most = key_limit(a, len, start, min(row0 + 15, a.rows - 1));           // and its last
  const int npages = (most + kPage8 - 1) / kPage8;
  const int chunk = (npages + a.splits - 1) / a.splits;
  const int p0 = split * chunk, p1 = min(p0 + chunk, npages);

  V8 q[NK];
  if (real) {
    const T* qp = (const T*)a.q + b * a.qs[0] + (int64_t)(row / a.G) * a.qs[1] + (int64_t)(h * a.G + row % a.G) * a.qs[2];
    // D >= 64: the products 2 j and 2 j + 1 take channels 64 j + 16 g + 0..7 and + 8..15, so that a
    // key's bytes are read 16 at a time.
#pragma unroll
    for (int j = 0; j < NK; j++) {
      const int c = D == 32 ? 8 * g : 64 * (j / 2) + 16 * g + 8 * (j % 2);
      __builtin_memcpy(&q[j], qp + c, 16);
    }
  } else {
#pragma unroll
    for (int j = 0; j < NK; j++) q[j] = V8{};
  }

  f32x4 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; d++) acc[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
  float m = -__builtin_inff(), l = 0.f;

  for (int p = p0 + wave; p < p1; p += kAttendWaves) {
    int page = a.table[b * a.tp + p];
    const bool missing = (unsigned)page >= (unsigned)a.pages;
    if (missing) page = 0;
    const int64_t at = (int64_t)page * a.H + h;
    const uint8_t* kp = a.k + at * (kPage8 * D);
    const uint8_t* vp = a.v + at * (kPage8 * D);
    const float vscale = scale_of(a.vs[at]);
    const float kscale = missing ? __builtin_nanf("") : a.scale * scale_of(a.ks[at]);
    const int base = p * kPage8 + 16 * g;   // the lane's first token
    float s[16];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      f32x4 c = {0.f, 0.f, 0.f, 0.f};
      const uint8_t* kr = kp + (16 * (r >> 2) + 4 * t + (r & 3)) * D;
      if constexpr (D == 32) {
        const i32x2 w = *reinterpret_cast<const i32x2*>(kr + 8 * g);
        V8 kv;
        codes_as(w[0], w[1], kv);
        c = mfma_q(kv, q[0], c);
      } else {
#pragma unroll
        for (int j = 0; j < NK / 2; j++) {
          const i32x4 w = *reinterpret_cast<const i32x4*>(kr + 64 * j + 16 * g);
          V8 kv;
          codes_as(w[0], w[1], kv);
          c = mfma_q(kv, q[2 * j], c);
          codes_as(w[2], w[3], kv);
          c = mfma_q(kv, q[2 * j + 1], c);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; i++) s[4 * t + i] = c[i] * kscale;
    }
    const bool cut = p * kPage8 + kPage8 > least;   // some query does not see the whole page
    if (cut) {
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (base + i >= limit) s[i] = -__builtin_inff();
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; i++) mx = fmaxf(mx, s[i]);
    const auto x16 = __builtin_amdgcn_permlane16_swap(__float_as_int(mx), __float_as_int(mx), false, false);
    mx = fmaxf(__int_as_float(x16[0]), __int_as_float(x16[1]));
    const auto x32 = __builtin_amdgcn_permlane32_swap(__float_as_int(mx), __float_as_int(mx), false, false);
    mx = fmaxf(__int_as_float(x32[0]), __int_as_float(x32[1]));
    const float mn = fmaxf(m, mx);
    const float ref = mn == -__builtin_inff() ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    m = mn;
    l *= alpha;
    f16x8 pr[2];
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const float e = __builtin_amdgcn_exp2f(s[i] - ref);
      l += e;
      pr[i / 8][i % 8] = (f16)e;
    }
#pragma unroll
    for (int d = 0; d < ND; d++) {
      i32x4 w = *reinterpret_cast<const i32x4*>(vp + (16 * d + r) * kPage8 + 16 * g);
      bool poisoned = false;
      f16x8 seen[2];
      if (cut) {
        // Tokens behind the sequence are whatever was there: zero them. Tokens that only some of the
        // queries see may be NaN, and zero times NaN is not zero: they are taken out of the product, and
        // a product of their places with 1 for each token seen says which sums they belong in.
        const int left = len - base;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int n = left - 4 * i;
          if (n < 4) w[i] = n <= 0 ? 0 : w[i] & (int)(0xffffffffu >> (32 - 8 * n));
          nan = nan || nan_bytes(w[i]) != 0;
        }
        poisoned = __any(nan);
      }
      f32x4 c = {0.f, 0.f, 0.f, 0.f};
      f32x4 marks = {0.f, 0.f, 0.f, 0.f};
      if (poisoned) {
#pragma unroll
        for (int i = 0; i < 16; i++) seen[i / 8][i % 8] = base + i < limit ? (f16)1.f : (f16)0.f;
        f16x8 mk[2];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const unsigned nb = nan_bytes(w[i]);
#pragma unroll
          for (int j = 0; j < 4; j++) mk[i / 2][i % 2 * 4 + j] = (nb >> (8 * j)) & 0x80 ? (f16)1.f : (f16)0.f;
          w[i] &= ~(int)((nb >> 7) * 255u);
        }
        marks = mfma16(mk[0], seen[0], marks);
        marks = mfma16(mk[1], seen[1], marks);
      }
      f16x8 v0, v1;
      codes_as(w[0], w[1], v0);
      codes_as(w[2], w[3], v1);
      c = mfma16(v0, pr[0], c);
      c = mfma16(v1, pr[1], c);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (poisoned && marks[i] > 0.f) c[i] = __builtin_nanf("");
        acc[d][i] = acc[d][i] * alpha + c[i] * vscale;
      }
    }
  }
  // l over the four lane groups of a query, then the waves' states through LDS.
  const auto l16 = __builtin_amdgcn_permlane16_swap(__float_as_int(l), __float_as_int(l), false, false);
  l = __int_as_float(l16[0]) + __int_as_float(l16[1]);
  const auto l32 = __builtin_amdgcn_permlane32_swap(__float_as_int(l), __float_as_int(l), false, false);
  l = __int_as_float(l32[0]) + __int_as_float(l32[1]);
  if (g == 0) {
    sm[wave][r] = m;
    sl[wave][r] = l;
  }
#pragma unroll
  for (int d = 0; d < ND; d++) *reinterpret_cast<f32x4*>(&sacc[wave][r][16 * d + 4 * g]) = acc[d];
  __syncthreads();
  const int64_t bh = (int64_t)b * a.H + h;
  for (int e = threadIdx.x; e < 16 * D / 4; e += 64 * kAttendWaves) {
    const int er = e / (D / 4), ec = e % (D / 4) * 4, orow = row0 + er;
    if (orow >= a.rows) continue;
    float mt = sm[0][er];
#pragma unroll
    for (int w = 1; w < kAttendWaves; w++) mt = fmaxf(mt, sm[w][er]);
    const float ref = mt == -__builtin_inff() ? 0.f : mt;
    float lt = 0.f;
    f32x4 ot = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kAttendWaves; w++) {
      const float f = __builtin_amdgcn_exp2f(sm[w][er] - ref);
      lt += sl[w][er] * f;
      ot += *reinterpret_cast<const f32x4*>(&sacc[w][er][ec]) * f;
    }
    if (too_long) lt = __builtin_nanf("");
    if (a.splits > 1) {
      const int64_t at = (bh * a.rows + orow) * a.splits + split;
      const int64_t all = (int64_t)gridDim.z * a.H * a.rows * a.splits;
      *reinterpret_cast<f32x4*>(a.part + at * D + ec) = ot;
      if (ec == 0) {
        a.part[all * D + 2 * at] = ref;
        a.part[all * D + 2 * at + 1] = lt;
      }
      continue;
    }
    const float inv = lt == 0.f ? 0.f : 1.f / lt;
    T* op = (T*)a.o + b * a.os[0] + (int64_t)(orow / a.G) * a.os[1] + (int64_t)(h * a.G + orow % a.G) * a.os[2] + ec;
#pragma unroll
    for (int i = 0; i < 4; i++) op[i] = (T)(ot[i] * inv);
  }
}

// Joins the splits of a row: a thread takes four channels.
template <typename T, int D>
__global__ __launch_bounds__(256) void attend8_merge_kernel(Attend8Args a, int64_t total) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t at = e / (D / 4);
  if (at >= total) return;
  const int c = (int)(e % (D / 4)) * 4;
  const float* ml = a.part + total * a.splits * D + at * a.splits * 2;
  float mt = -__builtin_inff();
  for (int s = 0; s < a.splits; s++)
    if (ml[2 * s + 1] != 0.f) mt = fmaxf(mt, ml[2 * s]);
  float lt = 0.f;
  f32x4 ot = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; s++) {
    if (ml[2 * s + 1] == 0.f) continue;   // a split without a token that the row sees
    const float f = __builtin_amdgcn_exp2f(ml[2 * s] - mt);
    lt += ml[2 * s + 1] * f;
    ot += *reinterpret_cast<const f32x4*>(a.part + (at * a.splits + s) * D + c) * f;
  }
  const float inv = lt == 0.f ? 0.f : 1.f / lt;
  const int64_t bh = at / a.rows;
  const int row = (int)(at % a.rows), h = (int)(bh % a.H);
  T* op = (T*)a.o + bh / a.H * a.os[0] + (int64_t)(row / a.G) * a.os[1] + (int64_t)(h * a.G + row % a.G) * a.os[2] + c;
#pragma unroll
  for (int i = 0; i < 4; i++) op[i] = (T)(ot[i] * inv);
}

template <typename T, int D>
void launch_d(const Attend8Args& a, int batch, hipStream_t st) {
  const dim3 grid((unsigned)a.splits, (unsigned)(a.H * ((a.rows + 15) / 16)), (unsigned)batch);
  hipLaunchKernelGGL((attend8_kernel<T, D>), grid, dim3(64 * kAttendWaves), 0, st, a);
  if (a.splits > 1) {
    const int64_t total = (int64_t)batch * a.H * a.rows;
    hipLaunchKernelGGL((attend8_merge_kernel<T, D>), dim3((unsigned)((total * (D / 4) + 255) / 256)), dim3(256), 0, st, a,
                       total);
  }
}

template <typename T>
void launch_t(const Attend8Args& a, int D, int batch, hipStream_t st) {
  if (D == 32) launch_d<T, 32>(a, batch, st);
  else if (D == 64) launch_d<T, 64>(a, batch, st);
  else if (D == 128) launch_d<T, 128>(a, batch, st);
  else launch_d<T, 256>(a, batch, st);
}

int check_cache(const char* what, const ldx_cache8& c) {
  if (!c.k || !c.v || !c.k_scales || !c.v_scales) return fail("%s: null pointer", what);
  if (c.pages < 1 || c.heads < 1 || c.heads > 8192) return fail("%s: %d pages, %d heads", what, c.pages, c.heads);
  if (c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)
    return fail("%s: head_dim %d is not 32, 64, 128 or 256", what, c.head_dim);
  if ((uintptr_t)c.k % 16 || (uintptr_t)c.v % 16) return fail("%s: codes not aligned", what);
  return LDX_OK;
}

// Workgroups that a sequence's pages are spread over: enough that the launch fills the card.
int split_count(const ldx_cache8_attention_args* p) {
  const int64_t rows = (int64_t)p->q_len * (p->q_heads / p->cache.heads);
  const int64_t groups = (int64_t)p->batch * p->cache.heads * ((rows + 15) / 16);
  int64_t s = 1024 / groups;
  const int64_t most = (p->width + kAttendWaves - 1) / kAttendWaves;
  if (s > most) s = most;
  if (s > 64) s = 64;
  return s < 1 ? 1 : (int)s;
}

size_t split_bytes(const ldx_cache8_attention_args* p, int splits) {
  if (splits < 2) return 0;
  const size_t rows = (size_t)p->q_len * (p->q_heads / p->cache.heads);
  return (size_t)p->batch * p->cache.heads * rows * splits * (p->cache.head_dim + 2) * sizeof(float);
}

int check_attention(const ldx_cache8_attention_args* p) {
  if (!p || !p->q || !p->o || !p->table || !p->lengths) return fail("cache8_attention: null pointer");
  if (int rc = check_cache("cache8_attention", p->cache)) return rc;
  if (p->dtype != LDX_DTYPE_F16 && p->dtype != LDX_DTYPE_BF16)
    return fail("cache8_attention: dtype %d is not LDX_DTYPE_F16 or LDX_DTYPE_BF16", p->dtype);
  if (p->batch < 1 || p->batch > 65535 || p->q_len < 1 || p->width < 1 || p->width > (1 << 24))
    return fail("cache8_attention: batch %d, %d queries, %d pages a sequence", p->batch, p->q_len, p->width);
  if (p->q_heads < 1 || p->q_heads % p->cache.heads)
    return fail("cache8_attention: %d query heads over %d cache heads", p->q_heads, p->cache.heads);
  const int64_t rows = (int64_t)p->q_len * (p->q_heads / p->cache.heads);
  if ((rows + 15) / 16 * p->cache.heads > 65535)
    return fail("cache8_attention: %d queries of %d heads are more than one launch takes", p->q_len, p->q_heads);
  if (p->table_pitch < p->width) return fail("cache8_attention: table pitch below %d", p->width);
  if (!(p->scale > -1e30f && p->scale < 1e30f)) return fail("cache8_attention: scale %g", (double)p->scale);
  return LDX_OK;
}

}  // namespace
}  // namespace ldx

using namespace ldx;

extern "C" int ldx_cache8_append(const ldx_cache8_append_args* p, void* stream) {
  if (!p || !p->k || !p->v || !p->table || !p->starts) return fail("cache8_append: null pointer");
  if (int rc = check_cache("cache8_append", p->cache)) return rc;
  if (p->dtype != LDX_DTYPE_F16 && p->dtype != LDX_DTYPE_BF16 && p->dtype != LDX_DTYPE_F32)
    return fail("cache8_append: dtype %d is not LDX_DTYPE_F16, LDX_DTYPE_BF16 or LDX_DTYPE_F32", p->dtype);
  if (p->batch < 1 || p->batch > 65535 || p->tokens < 1 || p->width < 1 || p->width > (1 << 24))
    return fail("cache8_append: batch %d, %d tokens, %d pages a sequence", p->batch, p->tokens, p->width);
  if (p->table_pitch < p->width) return fail("cache8_append: table pitch below %d", p->width);
  AppendArgs a = {{(uint8_t*)p->cache.k, (uint8_t*)p->cache.v},
                  {(uint8_t*)p->cache.k_scales, (uint8_t*)p->cache.v_scales},
                  {p->k, p->v},
                  {{p->k_stride[0], p->k_stride[1], p->k_stride[2]}, {p->v_stride[0], p->v_stride[1], p->v_stride[2]}},
                  p->cache.pages, p->cache.heads, p->cache.head_dim, p->tokens,
                  p->table, p->table_pitch, p->width, p->starts, p->counts};
  const unsigned slots = (unsigned)((p->tokens + 2 * (int64_t)kPage8 - 2) / kPage8);
  const dim3 grid(slots, 2 * (unsigned)p->cache.heads, (unsigned)p->batch);
  hipStream_t st = as_stream(stream);
  if (p->dtype == LDX_DTYPE_F16) hipLaunchKernelGGL(append8_kernel<f16>, grid, dim3(256), 0, st, a);
  else if (p->dtype == LDX_DTYPE_BF16) hipLaunchKernelGGL(append8_kernel<bf16>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(append8_kernel<float>, grid, dim3(256), 0, st, a);
  return check_launch("cache8_append");
}

extern "C" size_t ldx_cache8_attention_workspace_bytes(const ldx_cache8_attention_args* p) {
  return check_attention(p) == LDX_OK ? split_bytes(p, split_count(p)) : 0;
}

extern "C" int ldx_cache8_attention(const ldx_cache8_attention_args* p, void* stream) {
  if (int rc = check_attention(p)) return rc;
  int splits = split_count(p);
  if (splits > 1 && (!p->workspace || p->workspace_bytes < split_bytes(p, splits))) splits = 1;
  if (splits > 1 && (uintptr_t)p->workspace % 16) return fail("cache8_attention: workspace not aligned");
  const int G = p->q_heads / p->cache.heads;
  const Attend8Args a = {(const uint8_t*)p->cache.k, (const uint8_t*)p->cache.v, (const uint8_t*)p->cache.k_scales,
                         (const uint8_t*)p->cache.v_scales, p->cache.pages, p->cache.heads,
                         p->q, {p->q_stride[0], p->q_stride[1], p->q_stride[2]},
                         p->o, {p->o_stride[0], p->o_stride[1], p->o_stride[2]},
                         G, p->q_len, G * p->q_len, p->scale * 1.4426950408889634f,
                         p->table, p->table_pitch, p->width, p->lengths, p->starts, splits, (float*)p->workspace};
  hipStream_t st = as_stream(stream);
  if (p->dtype == LDX_DTYPE_F16) launch_t<f16>(a, p->cache.head_dim, p->batch, st);
  else launch_t<bf16>(a, p->cache.head_dim, p->batch, st);
  return check_launch("cache8_attention");
}
