// A cache of keys and values held in 4 bits, in pages of 64 tokens: OCP e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6
// and their negatives) with a power of two (E8M0) for each 32 channels of a token. Writing new tokens, reading
// them back, and the attention that reads the cache.
//
// Keys and values lie alike: codes (pages, H, 64, D / 2), two channels in a byte, the even one in its lower half,
// and scales (pages, H, D / 32, 64), a block's tokens side by side: a lane of the attention reads those of 16
// tokens at once. A scale per token is what lets a token be written without touching older ones, which in 4 bits
// would lose too much by being rounded again.
#include "attend_parts.h"

namespace ldx {
namespace {

constexpr int kPage4 = LDX_PAGE4;
constexpr int kBlock4 = LDX_BLOCK4;
static_assert(kPage4 == kPage8, "attend_parts.h counts pages of 64 tokens");

// The scale byte of a block with largest magnitude amax = 1.m * 2^(E - 127): the least b from 1 on with amax <= 6 *
// 2^(b - 127) = 1.5 * 2^(b - 125). Zeros get 127. At most 252: values past 6 * 2^125, which the next scale's larger
// codes would round to 2^128, are held as that. NaN and infinite blocks get 255, which is NaN.
__device__ __forceinline__ int scale4_byte(float amax) {
  const int bits = __float_as_int(amax);
  if (bits >= 0x7f800000) return 255;
  if (bits == 0) return 127;
  const int b = (bits >> 23) - 2 + ((bits & 0x7fffff) > 0x400000 ? 1 : 0);
  return min(max(b, 1), 252);
}

// Eight values times the inverse scale as eight codes (round to nearest even, magnitudes past 6 as 6).
__device__ __forceinline__ unsigned encode8(const float (&f)[8], float inv) {
  unsigned w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[0] * inv, f[1] * inv, 1.f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[2] * inv, f[3] * inv, 1.f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[4] * inv, f[5] * inv, 1.f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[6] * inv, f[7] * inv, 1.f, 3);
}

// The widening conversions take a scale's exponent bits alone, as E8M0 (0 is 2^-127, 255 gives NaN): a scale byte goes
// there by one rotation of the word that holds it, whatever lands beside it.
__device__ __forceinline__ float scale_at(int word, int byte) {
  return __int_as_float((int)__builtin_amdgcn_alignbit((unsigned)word, (unsigned)word, 8 * byte + 9));
}

// ------------------------------------------------------------------------------ append and read

struct Store4Args {
  uint8_t* codes[2];     // keys, values (pages, H, 64, D / 2)
  uint8_t* scales[2];    // (pages, H, D / 32, 64)
  void* x[2];            // what is appended, or where it is read to
  int64_t st[2][3];      // its batch, token, head strides
  int pages, H, tokens;
  const int32_t* table; int64_t tp; int width;
  const int32_t* starts;
  const int32_t* counts;   // append: tokens of each sequence
  const int32_t* lengths;  // read: tokens that a sequence holds
  bool fill;               // read: zeros behind them
};

// A workgroup takes the tokens that stand in one page, of a head's keys or values: a lane eight channels, four of them a
// block, whose largest magnitude they find among themselves. 2 x 4,001 tokens of 8 heads of 64 in fp16 6.6 us, 3.1
// TB/s with the launch; a token of each of 48 sequences of 8 heads of 128 3.2 us, which is the launch.
template <typename T, int D>
__global__ __launch_bounds__(256) void append4_kernel(Store4Args a) {
  constexpr int UNITS = D / 8;   // eight channels, a lane each; four lanes hold a block
  const int b = blockIdx.z, h = blockIdx.y >> 1, which = blockIdx.y & 1, tid = threadIdx.x;
  const int start = a.starts[b];
  const int n = a.counts ? min(a.counts[b], a.tokens) : a.tokens;
  if (start < 0 || n <= 0) return;
  const int64_t end = (int64_t)start + n, slot = start / kPage4 + (int64_t)blockIdx.x, first = slot * kPage4;
  if (first >= end || slot >= a.width) return;
  const int page = a.table[b * a.tp + slot];
  if ((unsigned)page >= (unsigned)a.pages) return;
  const int lo = (int)max(start - first, (int64_t)0), hi = (int)min(end - first, (int64_t)kPage4);
  const int64_t at = (int64_t)page * a.H + h, tok = a.st[which][1];
  uint8_t* codes = a.codes[which] + at * (kPage4 * D / 2);
  uint8_t* scales = a.scales[which] + at * (kPage4 * D / kBlock4);
  const T* src = (const T*)a.x[which] + b * a.st[which][0] + (first + lo - start) * tok + h * a.st[which][2];
  for (int c = tid; c < (hi - lo) * UNITS; c += 256) {
    const int t = c / UNITS, u = c % UNITS;
    float f[8];
    load8(src + t * tok + u * 8, f);
    float amax = 0.f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      amax = fmaxf(amax, fabsf(f[i]));
      nan |= f[i] != f[i];
    }
    if (nan) amax = __builtin_inff();
    amax = fmaxf(amax, dpp_f<0xB1>(amax));   // quad_perm 1 0 3 2
    amax = fmaxf(amax, dpp_f<0x4E>(amax));   // quad_perm 2 3 0 1
    const int s = scale4_byte(amax);
    *reinterpret_cast<unsigned*>(codes + (lo + t) * (D / 2) + u * 4) = s == 255 ? 0u : encode8(f, inverse_of(s));
    if (u % 4 == 0) scales[u / 4 * kPage4 + lo + t] = (uint8_t)s;
  }
}

// Eight codes times their scale in T, to memory of any alignment, past the caches' retention.
template <typename T>
struct Pair;
template <>
struct Pair<f16> {
  template <int SEL>
  static __device__ __forceinline__ f16x2 of(unsigned w, float s) { return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, SEL); }
};
template <>
struct Pair<bf16> {
  template <int SEL>
  static __device__ __forceinline__ bf16x2 of(unsigned w, float s) { return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, SEL); }
};
template <>
struct Pair<float> {
  template <int SEL>
  static __device__ __forceinline__ f32x2 of(unsigned w, float s) { return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, SEL); }
};
template <typename T>
__device__ __forceinline__ void decode8(unsigned w, float s, T* p) {
  typedef T V __attribute__((ext_vector_type(8)));
  typedef V Unaligned __attribute__((aligned(sizeof(T))));
  const auto a = Pair<T>::template of<0>(w, s), b = Pair<T>::template of<1>(w, s), c = Pair<T>::template of<2>(w, s),
             d = Pair<T>::template of<3>(w, s);
  const V v = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  __builtin_nontemporal_store(v, reinterpret_cast<Unaligned*>(p));
}

// A lane takes eight channels as in append4_kernel: a word of codes and a byte of scales in, 16 or 32 bytes out, which are
// what bounds it: 4 x 24,000 tokens of 8 heads of 128 as bf16 76 us, 6.5 TB/s (101 with stores that stay in the caches).
template <typename T, int D>
__global__ __launch_bounds__(256) void read4_kernel(Store4Args a) {
  constexpr int UNITS = D / 8;
  const int b = blockIdx.z, h = blockIdx.y >> 1, which = blockIdx.y & 1, tid = threadIdx.x;
  const int64_t start = a.starts ? a.starts[b] : 0;
  // Row i is token start + i; the workgroup takes rows of one page, the first of them maybe less than whole.
  const int64_t slot = (start >= 0 ? start / kPage4 : -((-start + kPage4 - 1) / kPage4)) + blockIdx.x, first = slot * kPage4;
  const int64_t lo = max(start, first), hi = min(start + a.tokens, first + kPage4);
  if (lo >= hi) return;
  const int64_t len = a.lengths[b];
  const bool within = slot >= 0 && slot < a.width;
  const int page = within ? a.table[b * a.tp + slot] : -1;
  const bool missing = (unsigned)page >= (unsigned)a.pages;
  const int64_t at = (int64_t)(missing ? 0 : page) * a.H + h, tok = a.st[which][1];
  const uint8_t* codes = a.codes[which] + at * (kPage4 * D / 2);
  const uint8_t* scales = a.scales[which] + at * (kPage4 * D / kBlock4);
  T* dst = (T*)a.x[which] + b * a.st[which][0] + h * a.st[which][2];
  for (int c = tid; c < (int)(hi - lo) * UNITS; c += 256) {
    const int u = c % UNITS;
    const int64_t t = lo + c / UNITS;
    const bool held = t >= 0 && t < len;
    if (!held && !a.fill) continue;
    const int place = (int)(t - first);
    const unsigned w = held && !missing ? *reinterpret_cast<const unsigned*>(codes + place * (D / 2) + u * 4) : 0u;
    const int s = !held ? 127 : missing ? 255 : scales[u / 4 * kPage4 + place];
    decode8(w, __int_as_float(s << 23), dst + (t - start) * tok + u * 8);
  }
}

template <typename T, bool READ>
void launch_store(const Store4Args& a, int D, dim3 grid, hipStream_t st) {
  if constexpr (READ) {
    if (D == 32) hipLaunchKernelGGL((read4_kernel<T, 32>), grid, dim3(256), 0, st, a);
    else if (D == 64) hipLaunchKernelGGL((read4_kernel<T, 64>), grid, dim3(256), 0, st, a);
    else if (D == 128) hipLaunchKernelGGL((read4_kernel<T, 128>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((read4_kernel<T, 256>), grid, dim3(256), 0, st, a);
  } else {
    if (D == 32) hipLaunchKernelGGL((append4_kernel<T, 32>), grid, dim3(256), 0, st, a);
    else if (D == 64) hipLaunchKernelGGL((append4_kernel<T, 64>), grid, dim3(256), 0, st, a);
    else if (D == 128) hipLaunchKernelGGL((append4_kernel<T, 128>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((append4_kernel<T, 256>), grid, dim3(256), 0, st, a);
  }
}

// ------------------------------------------------------------------------------------- attention

struct Attend4Args {
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
  int splits, chunk;     // parts of a sequence; least pages of a part
  int tile;              // rows of a workgroup
  float* part;           // splits > 1: [b][h][row][split] of D sums, then of (m, l)
};

__device__ __forceinline__ f32x4 mfma16b(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// Eight codes times a scale as bf16, which holds them exactly.
__device__ __forceinline__ bf16x8 widen8(unsigned w, float s) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3);
  return (bf16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Two codes (byte SEL of a word) times a scale, as a word of two bf16.
template <int SEL>
__device__ __forceinline__ unsigned widen2(unsigned w, float s) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, SEL));
}
__device__ __forceinline__ unsigned widen2(unsigned w, float s, int sel) {
  return sel == 0 ? widen2<0>(w, s) : sel == 1 ? widen2<1>(w, s) : sel == 2 ? widen2<2>(w, s) : widen2<3>(w, s);
}

// A number as two bf16: its upper half, cut off, and what is left, rounded: 16 bits of it.
__device__ __forceinline__ void split2(float x, float y, unsigned& hi, unsigned& lo) {
  const unsigned a = (unsigned)__float_as_int(x), b = (unsigned)__float_as_int(y);
  hi = __builtin_amdgcn_perm(b, a, 0x07060302);
  const bf16x2 l = {(bf16)(x - __int_as_float((int)(a & 0xffff0000u))), (bf16)(y - __int_as_float((int)(b & 0xffff0000u)))};
  lo = __builtin_bit_cast(unsigned, l);
}

// The 0x80 bit of every scale byte of 253 and more: NaN, and blocks whose values may pass fp32.
__device__ __forceinline__ unsigned beyond_bytes(int w) {
  return (((unsigned)w & 0x7f7f7f7fu) + 0x03030303u) & (unsigned)w & 0x80808080u;
}

// A query's reference for its exponentials follows its maximum only where that passes it by more than this (in
// powers of two): the sums are seldom multiplied then.
constexpr float kLag = 8.f;
constexpr int kWaves4 = 4;

// S^T = K Q^T per page on 16 x 16 x 32 products: lane l holds query column l % 16, g = l / 16. Key row m of key tile t
// is the page's token 16 (m / 4) + 4 t + m % 4, so that the scores a lane receives (rows 4 g + i, tiles t) are those
// of tokens 16 g + 4 t + i, sixteen in a row, and the probabilities go into the second product as they lie. There lane l
// holds the values of the same tokens for channels l % 16 * (D / 16) .. of each, D / 32 bytes a token, of which tile d
// of O^T takes the d-th: eight tokens' bytes are widened and their 16-bit halves sorted by channel.
//
// Operands are bf16, which holds a code times any scale exactly; a 16-bit query of more digits and the probabilities
// go in as two of them, 16 bits in all. Sums are fp32.
//
// A page's keys are asked for when the last one's scores are made and its values when the last one's products are, so
// that a wave keeps a page on its way. Bound by memory: a query of 8 x 4 heads of 128 for each of 32 sequences of 4,000 to
// 16,384 tokens 78 us and 5 for the join, 4.6 TB/s, 69 with nearly no arithmetic left in it; of 4 x 8 heads behind 200,000
// tokens 26 and 5.
template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves4, D == 256 ? 1 : 2) void attend4_kernel(Attend4Args a) {
  constexpr int ND = D / 16;              // channel tiles; channels of a lane's values
  constexpr int NK = D / 32;              // products per key tile; words of a lane's part of a key
  constexpr int QP = sizeof(T) == 2 && __is_same(T, f16) ? 2 : 1;   // parts of a query
  constexpr int NB = D == 256 ? 2 : 1;    // blocks of a lane's part of a key
  constexpr int VW = D == 256 ? 2 : 1;    // words of a lane's part of a token's values
  __shared__ float sm[kWaves4][16], sl[kWaves4][16];
  __shared__ __align__(16) float sacc[kWaves4][16][D + 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int b = blockIdx.z, split = blockIdx.x % a.splits, tiles = (a.rows + 15) / 16, tile = blockIdx.x / a.splits;
  const int h = tile / tiles, row0 = tile % tiles * 16;
  const int row = row0 + r;
  const bool real = row < a.rows;
  const int raw = a.lengths[b];
  const bool too_long = raw > (int64_t)a.width * kPage4;
  const int len = too_long || raw < 0 ? 0 : raw;
  const int64_t start = a.starts ? a.starts[b] : 0;
  const int limit = real ? key_limit(a, len, start, row) : 0;
  const int least = key_limit(a, len, start, row0);                                // the tile's first row
  const int most = key_limit(a, len, start, min(row0 + 15, a.rows - 1));           // and its last
  const int npages = (most + kPage4 - 1) / kPage4;
  const int chunk = max((npages + a.splits - 1) / a.splits, a.chunk);
  const int p0 = a.splits > 1 ? split * chunk : 0, p1 = a.splits > 1 ? min(p0 + chunk, npages) : npages;
  if (p0 >= p1 && split > 0) return;   // the join knows that there is no such part

  bf16x8 q[QP][NK];
  {
    const T* qp = (const T*)a.q + b * a.qs[0] + (int64_t)(row / a.G) * a.qs[1] + (int64_t)(h * a.G + row % a.G) * a.qs[2];
#pragma unroll
    for (int j = 0; j < NK; j++) {
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (real) load8(qp + D / 4 * g + 8 * j, f);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const bf16 hi = (bf16)f[e];
        q[0][j][e] = hi;
        if constexpr (QP == 2) q[1][j][e] = (bf16)(f[e] - (float)hi);
      }
    }
  }

  float acc[ND][4];
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int i = 0; i < 4; i++) acc[d][i] = 0.f;
  float m = -__builtin_inff(), l = 0.f;
  int poison = 0;   // bit i: the lane's query sees a value of NaN in block i of its channels' ones

  const int32_t* table = a.table + b * a.tp;
  const unsigned koff = (unsigned)(16 * (r >> 2) + (r & 3)) * (D / 2) + (D / 8) * g;
  const unsigned voff = (unsigned)(16 * g) * (D / 2) + (D / 32) * r;
  const unsigned ksoff = (unsigned)(D / 4 * g / kBlock4) * kPage4 + 16 * (r >> 2);
  const unsigned vsoff = (unsigned)(ND * r / kBlock4) * kPage4 + 16 * g;
  const int kbyte = r & 3;
  unsigned kc[4][NK];   // a page's keys
  i32x4 ks[NB], vs;
  unsigned vc[16][VW];  // and its values
  struct Place {
    int64_t at;
    bool missing;
  };
  const auto place = [&](int page) {
    const bool missing = (unsigned)page >= (unsigned)a.pages;
    return Place{(int64_t)(missing ? 0 : page) * a.H + h, missing};
  };
  const auto load_k = [&](Place t, int p) {
    const __amdgpu_buffer_rsrc_t kr = make_rsrc(a.k + t.at * (kPage4 * D / 2), p < p1 ? (unsigned)(kPage4 * D / 2) : 0u);
    const __amdgpu_buffer_rsrc_t sr = make_rsrc(a.ks + t.at * (kPage4 * NK), p < p1 ? (unsigned)(kPage4 * NK) : 0u);
#pragma unroll
    for (int i = 0; i < NB; i++) ks[i] = buffer_load16<i32x4>(sr, ksoff, i * kPage4);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (NK == 1) {
        kc[i][0] = __builtin_amdgcn_raw_buffer_load_b32(kr, koff, 4 * i * (D / 2), 0);
      } else if constexpr (NK == 2) {
        const auto w = __builtin_amdgcn_raw_buffer_load_b64(kr, koff, 4 * i * (D / 2), 0);
        kc[i][0] = w[0];
        kc[i][1] = w[1];
      } else {
#pragma unroll
        for (int j = 0; j < NK / 4; j++) {
          const u32x4 w = buffer_load16<u32x4>(kr, koff, 4 * i * (D / 2) + 16 * j);
#pragma unroll
          for (int x = 0; x < 4; x++) kc[i][4 * j + x] = w[x];
        }
      }
    }
  };
  const auto load_v = [&](Place t, int p) {
    const __amdgpu_buffer_rsrc_t vr = make_rsrc(a.v + t.at * (kPage4 * D / 2), p < p1 ? (unsigned)(kPage4 * D / 2) : 0u);
    const __amdgpu_buffer_rsrc_t sr = make_rsrc(a.vs + t.at * (kPage4 * NK), p < p1 ? (unsigned)(kPage4 * NK) : 0u);
    vs = buffer_load16<i32x4>(sr, vsoff);
#pragma unroll
    for (int x = 0; x < 16; x++) {
      if constexpr (D == 32) vc[x][0] = __builtin_amdgcn_raw_buffer_load_b8(vr, voff, x * (D / 2), 0);
      else if constexpr (D == 64) vc[x][0] = __builtin_amdgcn_raw_buffer_load_b16(vr, voff, x * (D / 2), 0);
      else if constexpr (D == 128) vc[x][0] = __builtin_amdgcn_raw_buffer_load_b32(vr, voff, x * (D / 2), 0);
      else {
        const auto w = __builtin_amdgcn_raw_buffer_load_b64(vr, voff, x * (D / 2), 0);
        vc[x][0] = w[0];
        vc[x][VW - 1] = w[1];
      }
    }
  };

  // Page numbers are known two rounds ahead; behind the last page the last one's is read again.
  const int last = max(p1 - 1, 0);
  const auto entry = [&](int p) { return table_entry(table, min(p, last)); };
  int p = p0 + wave;
  Place now = place(entry(p)), next = place(entry(p + kWaves4));
  int after = entry(p + 2 * kWaves4);
  load_k(now, p);
  load_v(now, p);
  for (; p < p1; p += kWaves4) {
    const int base = p * kPage4 + 16 * g;   // the lane's first token
    float s[16];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NK; j++) {
        const float f = __int_as_float((int)__builtin_amdgcn_alignbit((unsigned)ks[j * NB / NK][t], (unsigned)ks[j * NB / NK][t], 8 * kbyte + 9));
        const bf16x8 kv = widen8(kc[t][j], f);
#pragma unroll
        for (int x = 0; x < QP; x++) o = mfma16b(kv, q[x][j], o);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) s[4 * t + i] = o[i] * a.scale;
      __builtin_amdgcn_sched_barrier(0);   // one tile's widened codes at a time
    }
    load_k(next, p + kWaves4);
    __builtin_amdgcn_sched_barrier(0);
    if (now.missing && p * kPage4 < limit) l = __builtin_nanf("");   // (page 0 was read in a missing one's place)
    const bool cut = p * kPage4 + kPage4 > least;   // some query does not see the whole page
    if (cut) {
      int left = limit - base;
      pin_value(left);
#pragma unroll
      for (int i = 0; i < 16; i++) s[i] = i < left ? s[i] : -__builtin_inff();
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 15; i += 2) mx = max3_f(mx, s[i], s[i + 1]);
    mx = max3_f(mx, s[15], s[15]);
    const auto x16 = __builtin_amdgcn_permlane16_swap(__float_as_int(mx), __float_as_int(mx), false, false);
    mx = max3_f(__int_as_float(x16[0]), __int_as_float(x16[1]), __int_as_float(x16[1]));
    const auto x32 = __builtin_amdgcn_permlane32_swap(__float_as_int(mx), __float_as_int(mx), false, false);
    const float mn = max3_f(m, __int_as_float(x32[0]), __int_as_float(x32[1]));
    float ref = m == -__builtin_inff() ? 0.f : m;
    if (__any(mn - m > kLag)) {
      ref = mn == -__builtin_inff() ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m - ref);
      l *= alpha;
#pragma unroll
      for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[d][i] *= alpha;
      m = mn;
    }
    u32x4 ph[2], pl[2];
    float lp = 0.f;   // the page's own sum, so that small ones do not go one by one into a large one
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float e0 = __builtin_amdgcn_exp2f(s[i] - ref), e1 = __builtin_amdgcn_exp2f(s[i + 1] - ref);
      lp += e0 + e1;
      unsigned hi, lo;
      split2(e0, e1, hi, lo);
      ph[i / 8][i % 8 / 2] = hi;
      pl[i / 8][i % 8 / 2] = lo;
    }
    l += lp;
    if (cut) {
      // Tokens that only some of the queries see may have values of NaN, and those behind the sequence anything; zero
      // times NaN is not zero. Such blocks get a scale of 1, and the queries that see them NaN, at the end.
      unsigned beyond = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) beyond |= beyond_bytes(vs[i]);
      if (__any(beyond != 0)) {
        const uint8_t* sp = a.vs + now.at * (kPage4 * NK) + (D / 4 * g / kBlock4) * kPage4;
#pragma unroll 1
        for (int t = 0; t < kPage4; t++)
#pragma unroll
          for (int i = 0; i < NB; i++)
            if (sp[i * kPage4 + t] >= 253 && p * kPage4 + t < limit) poison |= 1 << i;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const unsigned mask = (beyond_bytes(vs[i]) >> 7) * 255u;
          vs[i] = (int)(((unsigned)vs[i] & ~mask) | (0x7f7f7f7fu & mask));
        }
      }
    }
#pragma unroll
    for (int d = 0; d < ND; d += 2) {   // the two channels of a byte
      f32x4 o0 = {acc[d][0], acc[d][1], acc[d][2], acc[d][3]}, o1 = {acc[d + 1][0], acc[d + 1][1], acc[d + 1][2], acc[d + 1][3]};
#pragma unroll
      for (int u = 0; u < 2; u++) {
        u32x4 v0, v1;
#pragma unroll
        for (int x = 0; x < 8; x += 2) {
          const int t = 8 * u + x;
          const unsigned e = widen2(vc[t][d / 8], scale_at(vs[t / 4], t % 4), d % 8 / 2);
          const unsigned f = widen2(vc[t + 1][d / 8], scale_at(vs[(t + 1) / 4], (t + 1) % 4), d % 8 / 2);
          v0[x / 2] = __builtin_amdgcn_perm(f, e, 0x05040100);
          v1[x / 2] = __builtin_amdgcn_perm(f, e, 0x07060302);
        }
        const bf16x8 hi = __builtin_bit_cast(bf16x8, ph[u]), lo = __builtin_bit_cast(bf16x8, pl[u]);
        o0 = mfma16b(__builtin_bit_cast(bf16x8, v0), hi, o0);
        o1 = mfma16b(__builtin_bit_cast(bf16x8, v1), hi, o1);
        o0 = mfma16b(__builtin_bit_cast(bf16x8, v0), lo, o0);
        o1 = mfma16b(__builtin_bit_cast(bf16x8, v1), lo, o1);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        acc[d][i] = o0[i];
        acc[d + 1][i] = o1[i];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    load_v(next, p + kWaves4);
    __builtin_amdgcn_sched_barrier(0);
    now = next;
    next = place(after);
    after = entry(p + 3 * kWaves4);
  }

  // Lane (r, g) holds channels (4 g + i) ND + d of query r.
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const bool bad = poison >> (NB == 1 ? 0 : i / 2) & 1;
      sacc[wave][r][(4 * g + i) * ND + d] = bad ? __builtin_nanf("") : acc[d][i];
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
  __syncthreads();
  const int64_t bh = (int64_t)b * a.H + h;
  for (int e = threadIdx.x; e < 16 * D / 4; e += 64 * kWaves4) {
    const int er = e / (D / 4), ec = e % (D / 4) * 4, orow = row0 + er;
    if (orow >= a.rows) continue;
    float mt = sm[0][er];
#pragma unroll
    for (int w = 1; w < kWaves4; w++) mt = fmaxf(mt, sm[w][er]);
    const float ref = mt == -__builtin_inff() ? 0.f : mt;
    float lt = 0.f;
    f32x4 ot = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves4; w++) {
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
    put4<T>(a, b, h, orow, ec, ot, lt);
  }
}

// ------------------------------------------------------------------- many queries of a cache head
//
// A workgroup takes 128 rows (queries x grouped heads), a wave 32 of them, and shares each page through LDS as 16-bit
// operands, so that a code is widened once for all of them. S^T = K Q^T and O^T += V^T P^T on 32 x 32 x 16 products: lane
// l holds query column l % 32, h = l / 32. Row 8 q + 4 h + i of a 32-token key tile is its token 16 h + 4 q + i, so that
// the scores a lane receives are 16 tokens in a row and the probabilities go into the second product as they lie. Row 8 q +
// 4 h + i of a value tile is its channel 16 (q / 2) + 8 h + 4 (q % 2) + i, so that a lane's results are eight channels in a
// row.
//
// Keys are widened to the queries' type and values to fp16, which holds a code times 2^-23 to 2^8 exactly; probabilities
// are rounded to fp16. A page with scales outside of that (of its keys only where queries are fp16) is widened to bf16
// instead, with fp16 queries and the probabilities in two parts.
//
// A round takes the probabilities of page p between the products that make page p + 1's scores, and page p's values'
// products between the widening of later pages' codes, an instruction of the matrix units and some of the vector units in
// turn. (One after the other, 2,048 causal queries of 8 x 4 heads of 128 behind 8,192 tokens 445 us, so 345 to 380, 820 to
// 900 TF/s; 2,000 of 4 x 4 heads of 64 behind 8,000 tokens 130 and 7 for the join, of 256 1,160 and 540, of 32 97 and 6, with
// three waves a SIMD (two 109, four, which spill registers, 160).)
//
// At head width 64 a page takes a SIMD 1,650 cycles for 32 rows, 515 of which its matrix units work and 880 its vector units. Of
// the time that a CU is busy its vector units, matrix units and LDS work 67, 20 and 20 % at head width 32, 53, 31 and 27 at 64,
// 50, 52 and 45 at 128, 33, 27 and 24 at 256 (one wave a SIMD): but at 128 no more than one after the other would. The waves of a
// workgroup meet at a barrier each page and so run the same part of it at the same time.
constexpr int kWideRows = 128;
// A query's reference is this much below its maximum, and lags kLag behind it: probabilities reach 2^15, and fp16 holds
// those from 2^-21 of the largest on to 2^-11 of themselves and smaller ones to 2^-32 of it, so that many small ones
// beside a dominant one keep their weight.
constexpr float kRaise = 7.f;

__device__ __forceinline__ f32x16 mfma_w(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma_w(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Whether a word holds only scale bytes 104 to 135, whose codes fp16 holds: their upper three bits, 24 more. (A byte of 232
// and more carries into its neighbour, but gives itself away.)
__device__ __forceinline__ bool within_fp16(int w) { return (((unsigned)w + 0x18181818u) & 0xe0e0e0e0u) == 0x80808080u; }

// l and eight probabilities, as the products take them (their sum in fp32), so that rounding moves both sides of the
// quotient alike. Two at a time: half the additions of fp32 numbers.
__device__ __forceinline__ float sum8(f16x8 p, float l) {
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    l = __builtin_amdgcn_fdot2((f16x2){p[i], p[i + 1]}, (f16x2){(f16)1.f, (f16)1.f}, l, false);
  return l;
}

// Two codes (byte sel of a word) times a scale, as a word of two T.
template <typename T>
__device__ __forceinline__ unsigned pair_of(unsigned w, float s, int sel) {
  return sel == 0   ? __builtin_bit_cast(unsigned, Pair<T>::template of<0>(w, s))
         : sel == 1 ? __builtin_bit_cast(unsigned, Pair<T>::template of<1>(w, s))
         : sel == 2 ? __builtin_bit_cast(unsigned, Pair<T>::template of<2>(w, s))
                    : __builtin_bit_cast(unsigned, Pair<T>::template of<3>(w, s));
}

template <int N>
struct Const {
  static constexpr int value = N;
};

template <typename T>
struct Vec8;
template <>
struct Vec8<f16> { typedef f16x8 V; };
template <>
struct Vec8<bf16> { typedef bf16x8 V; };

// LDS holds keys in fragment order (a lane's 16 bytes at its place): 16 widening lanes write pieces j of 256 / D keys, and a
// fragment's pad moves its 16-byte places by 256 / D a piece. Values lie as they do in the cache, a token's channels in a
// row, and are turned as they are read, four tokens of 32 channels by 32 lanes (rows of 64 bytes past a multiple of 256, or
// 64 short of one, so that the four meet all banks once).
template <int D>
struct WideLds {
  static constexpr int KF = 1024 + 4096 / D, KEYS = 2 * (D / 16) * KF, VROW = D == 32 ? 64 : 2 * D + 64;
};

template <typename T, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : D == 32 ? 3 : 2) void attend4_wide_kernel(Attend4Args a) {
  typedef typename Vec8<T>::V V8;
  constexpr int NJ = D / 16;               // products per key tile
  constexpr int NT = D / 32;               // channel tiles; blocks
  constexpr int RAW = D == 32 ? 1 : D / 64;   // 8-byte pieces of a page's keys (values) that a thread widens
  constexpr int CHECK = D == 256 ? 2 : 1;  // words of a page's key (value) scales that a lane looks at
  typedef WideLds<D> L;
  extern __shared__ __align__(16) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, hh = lane >> 5;
  const int b = blockIdx.z, split = blockIdx.x % a.splits, tiles = (a.rows + kWideRows - 1) / kWideRows;
  const int tile = blockIdx.x / a.splits;
  const int h = tile / tiles, row0 = (tiles - 1 - tile % tiles) * kWideRows;   // causal: longest first
  const int wrow = row0 + 32 * wave, row = wrow + r;
  const bool real = row < a.rows;
  const int raw = a.lengths[b];
  const bool too_long = raw > (int64_t)a.width * kPage4;
  const int len = too_long || raw < 0 ? 0 : raw;
  const int64_t start = a.starts ? a.starts[b] : 0;
  const int limit = real ? key_limit(a, len, start, row) : 0;
  const int least = wrow < a.rows ? key_limit(a, len, start, wrow) : 0;                             // of the wave
  const int wmost = wrow < a.rows ? key_limit(a, len, start, min(wrow + 31, a.rows - 1)) : 0;
  const int most = key_limit(a, len, start, min(row0 + kWideRows, a.rows) - 1);                     // of the tile
  const int npages = (most + kPage4 - 1) / kPage4;
  const int chunk = max((npages + a.splits - 1) / a.splits, a.chunk);
  const int p0 = a.splits > 1 ? split * chunk : 0, p1 = a.splits > 1 ? min(p0 + chunk, npages) : npages;
  if (p0 >= p1 && split > 0) return;   // the join knows that there is no such part

  V8 q[NJ];
  {
    const T* qp = (const T*)a.q + b * a.qs[0] + (int64_t)(row / a.G) * a.qs[1] + (int64_t)(h * a.G + row % a.G) * a.qs[2];
    const float sign = a.scale > 0.f ? 1.f : a.scale < 0.f ? -1.f : 0.f;   // the size goes into the exponentials
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (real) load8(qp + 16 * j + 8 * hh, f);
#pragma unroll
      for (int e = 0; e < 8; e++) q[j][e] = (T)(f[e] * sign);
    }
  }
  const float scale = a.scale == 0.f ? 1.f : fabsf(a.scale);
  f32x16 acc[NT];
#pragma unroll
  for (int d = 0; d < NT; d++)
#pragma unroll
    for (int e = 0; e < 16; e++) acc[d][e] = 0.f;
  float m = -__builtin_inff(), l = 0.f;
  unsigned poison = 0;   // bit d: the lane's query sees a value of NaN in channel tile d

  const int32_t* table = a.table + b * a.tp;
  const auto entry = [&](int p) { return table_entry(table, min(p, p1 - 1)); };
  const auto place = [&](int page) { return (int64_t)((unsigned)page >= (unsigned)a.pages ? 0 : page) * a.H + h; };

  // A thread's pieces of a page's keys, and of another's values.
  struct Raw {
    i32x2 codes[RAW];
    int scale[RAW];
  };
  Raw kraw, vraw;
  // At head width 32 there are 128 pieces, for two waves: the others have the values'.
  const int vid = D == 32 ? tid ^ 128 : tid;
  const auto load = [&](const uint8_t* codes, const uint8_t* scales, int64_t at, int id, Raw& raw) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t cr = make_rsrc(codes + at * (kPage4 * D / 2), kPage4 * D / 2);
    const __amdgpu_buffer_rsrc_t sr = make_rsrc(scales + at * (kPage4 * NT), kPage4 * NT);
    const unsigned soff = id % NJ / 2 * kPage4 + id / NJ;   // (256 / NJ tokens on for the next piece)
#pragma unroll
    for (int i = 0; i < RAW; i++) {
      raw.codes[i] = __builtin_bit_cast(i32x2, __builtin_amdgcn_raw_buffer_load_b64(cr, id * 8, 2048 * i, 0));
      raw.scale[i] = __builtin_amdgcn_raw_buffer_load_b8(sr, soff, 256 / NJ * i, 0);
    }
  };
  // A page's scales, which every wave looks at, so that all take the page alike. (At head widths 64 and 32 the other lanes
  // read behind them, zeros, which stand for nothing.)
  struct Check {
    int word[CHECK];
  };
  const auto ask = [&](const uint8_t* scales, int64_t at, Check& c) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t sr = make_rsrc(scales + at * (kPage4 * NT), kPage4 * NT);
#pragma unroll
    for (int i = 0; i < CHECK; i++) c.word[i] = __builtin_amdgcn_raw_buffer_load_b32(sr, lane * 4, 256 * i, 0);
  };
  // Whether page p needs more than fp16. Tokens behind all that the rows see say nothing.
  const auto is_odd = [&](int p, Check& c) __attribute__((always_inline)) {
    if (p * kPage4 + kPage4 > most) {
      const int mine = most - p * kPage4 - lane * 4 % kPage4;
      const unsigned keep = mine >= 4 ? ~0u : mine <= 0 ? 0u : ~0u >> (32 - 8 * mine);
#pragma unroll
      for (int i = 0; i < CHECK; i++) c.word[i] = (int)(((unsigned)c.word[i] & keep) | (0x7f7f7f7fu & ~keep));
    }
    bool bad = false;
#pragma unroll
    for (int i = 0; i < CHECK; i++) bad |= !within_fp16(c.word[i]);
    return (bool)__any(bad && lane < 16 * NT);
  };
  const auto times = [&](float f) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < NT; d++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[d][e] *= f;
  };
  // Widen half x of a thread's piece i of the keys, or the values, into buffer `to`.
  const auto widen_key = [&](uint8_t* to, int i, int x, auto kt) __attribute__((always_inline)) {
    typedef decltype(kt) KT;
    if (D == 32 && wave >= 2) return;
    const int e = tid + 256 * i, key = e / NJ, j = e % NJ;
    const int t = key & 31, at = 8 * (t >> 2 & 3) + 4 * (t >> 4) + (t & 3);   // the token's row of its tile
    const float s = __int_as_float(kraw.scale[i] << 23);
    u32x4 w;
#pragma unroll
    for (int y = 0; y < 4; y++) w[y] = pair_of<KT>((unsigned)kraw.codes[i][x], s, y);
    *reinterpret_cast<u32x4*>(to + ((key >> 5) * NJ + j) * L::KF + at * 16 + 512 * x) = w;
  };
  const auto widen_value = [&](uint8_t* to, int left, int i, int x, auto vt) __attribute__((always_inline)) {
    typedef decltype(vt) VT;
    if (D == 32 && wave < 2) return;
    const int e = vid + 256 * i, key = e / NJ, j = e % NJ;
    // Values of tokens that none of the rows sees get a scale of 1: probabilities of 0 times anything finite; in bf16
    // those of NaN (and past fp32), too, see below.
    const bool one = key >= left || (__is_same(VT, bf16) && vraw.scale[i] >= 253);
    const float s = __int_as_float((one ? 127 : vraw.scale[i]) << 23);
    const int flip = (D == 256 ? j >> 3 : D == 128 ? j >> 2 : D == 64 ? key : key >> 2) & 1;   // 16 lanes write 16 bytes each, half of them first halves
    const int c0 = vraw.codes[i][x], c1 = vraw.codes[i][1 - x];
    const unsigned codes = (unsigned)(flip ? c1 : c0);
    u32x4 w;
#pragma unroll
    for (int y = 0; y < 4; y++) w[y] = pair_of<VT>(codes, s, y);
    *reinterpret_cast<u32x4*>(to + key * L::VROW + j * 32 + 16 * (x ^ flip)) = w;
  };
  const auto widen_keys = [&](uint8_t* to, auto kt) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2 * RAW; i++) widen_key(to, i / 2, i % 2, kt);
  };
  const auto widen_values = [&](uint8_t* to, int left, auto vt) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2 * RAW; i++) widen_value(to, left, i / 2, i % 2, vt);
  };
  // Eight tokens, 32 t + 16 h + 8 u .., of the channel that is row r of tile d, in 16 bits: lane l % 16 of 16 hands in
  // where four channels of a token stand and gets a channel of four tokens.
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  typedef __attribute__((address_space(3))) s16x4* lds4;
  const unsigned turned = (16 * hh + (lane & 15) / 4) * L::VROW + 2 * (16 * (lane >> 4 & 1) + 8 * (lane & 1) + 4 * (lane >> 1 & 1));
  const auto values = [&](const uint8_t* vb, int d, int t, int u) __attribute__((always_inline)) {
    const unsigned at = lds_offset(vb) + turned + (32 * t + 8 * u) * L::VROW + 64 * d;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)at);
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)(at + 4 * L::VROW));
    return (s16x8){x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  };

  struct Scores {
    f32x16 t[2];   // tiles of 32 tokens
  };
  const auto product = [&](const uint8_t* kb, Scores& sv) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) sv.t[t][e] = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; j++) {
#pragma unroll
      for (int t = 0; t < 2; t++)
        sv.t[t] = mfma_w(*reinterpret_cast<const V8*>(kb + lane * 16 + (t * NJ + j) * L::KF), q[j], sv.t[t]);
      if (j % 2) __builtin_amdgcn_sched_barrier(0);   // bounds the operands read ahead
    }
  };
  // The same of keys in bf16, and queries in two parts, made anew for each such page so that they do not stay in registers.
  const auto product_odd = [&](const uint8_t* kb, Scores& sv) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) sv.t[t][e] = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      V8 w = q[j];
      pin_value(w);
      bf16x8 hi, lo;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        hi[e] = (bf16)(float)w[e];
        lo[e] = (bf16)((float)w[e] - (float)hi[e]);
      }
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const bf16x8 kv = *reinterpret_cast<const bf16x8*>(kb + lane * 16 + (t * NJ + j) * L::KF);
        sv.t[t] = mfma_w(kv, lo, mfma_w(kv, hi, sv.t[t]));
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // A page's scores as exponents below the lane's reference, which is moved where it has to be.
  const auto exponents = [&](int p, bool missing, Scores& s, float& kc) __attribute__((always_inline)) {
    const int base = p * kPage4 + 16 * hh;   // score e of tile t is token base + 32 t + e
    if (missing && p * kPage4 < limit) l = __builtin_nanf("");   // (page 0 was read in a missing one's place)
    if (p * kPage4 + kPage4 > least) {
      int left = limit - base;
      pin_value(left);
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) s.t[t][e] = 32 * t + e < left ? s.t[t][e] : -__builtin_inff();
    }
    float mx = max3_f(s.t[0][0], s.t[1][0], s.t[0][1]);
    mx = max3_f(mx, s.t[1][1], s.t[1][1]);
#pragma unroll
    for (int e = 2; e < 16; e++) mx = max3_f(mx, s.t[0][e], s.t[1][e]);
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_int(mx), __float_as_int(mx), false, false);
    float mn = max3_f(m, __builtin_fmaf(__int_as_float(x[0]), scale, -kRaise),
                      __builtin_fmaf(__int_as_float(x[1]), scale, -kRaise));
    // A score goes into the exponential times the scale and unrounded, its reference does not: what the reference's
    // rounding left out, up to 2^-24 of it, moves a query's probabilities by one factor, which must not leave fp16.
    // Beyond 2^20 scores are rounded first, the reference never lags, and it is taken from the largest score as that is
    // rounded, so that the two are at most 8 apart, whatever number scores are multiples of. (Rounded by itself it would be 16
    // below, and the probability infinite in fp16, for 7 in 16 of the largest scores from 2^27 to 2^28.)
    const bool far = __any(fabsf(mn) >= 0x1p20f && mn != -__builtin_inff());
    kc = far ? 1.f : scale;
    if (__builtin_expect(far, 0)) {
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) s.t[t][e] *= scale;
      float a0 = __int_as_float(x[0]) * scale, a1 = __int_as_float(x[1]) * scale;
      pin_value(a0);   // (or the compiler makes one rounding of the two)
      pin_value(a1);
      mn = max3_f(m, a0 - kRaise, a1 - kRaise);
    }
    float ref = m == -__builtin_inff() ? 0.f : m;
    if (__any(mn - m > (far ? 0.f : kLag))) {
      ref = mn == -__builtin_inff() ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m - ref);
      l *= alpha;
      times(alpha);
      m = mn;
    }
    return ref;
  };
  const auto two = [&](const Scores& s, int i, float kc, float ref) __attribute__((always_inline)) {   // probabilities 2 i, 2 i + 1
    const f16x2 p = {(f16)__builtin_amdgcn_exp2f(__builtin_fmaf(s.t[i / 8][2 * i % 16], kc, -ref)),
                     (f16)__builtin_amdgcn_exp2f(__builtin_fmaf(s.t[i / 8][2 * i % 16 + 1], kc, -ref))};
    return p;
  };
  const auto probabilities = [&](const Scores& s, float kc, float ref, f16x8 (&pr)[4]) __attribute__((always_inline)) {
    float lp = 0.f;   // the page's own sum, so that small ones do not go one by one into a large one
#pragma unroll
    for (int i = 0; i < 4; i++) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const f16x2 p = two(s, 4 * i + e, kc, ref);
        pr[i][2 * e] = p[0], pr[i][2 * e + 1] = p[1];
      }
      lp = sum8(pr[i], lp);
      pin_value(lp);
      __builtin_amdgcn_sched_barrier(0);
    }
    l += lp;
  };
  const auto add_values = [&](const uint8_t* vb, const f16x8 (&pr)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int d = 0; d < NT; d++) {
        acc[d] = mfma_w(__builtin_bit_cast(f16x8, values(vb, d, i / 2, i % 2)), pr[i], acc[d]);
        if (d % 2) __builtin_amdgcn_sched_barrier(0);
      }
  };
  // A page's probabilities between the next page's products, and its values' products between the widening of codes, to
  // kto and vto (of the page's `left` tokens that count). A product's operand is read two products ahead.
  const auto both = [&](const Scores& now, Scores& next, float kc, float ref, const uint8_t* kb, const uint8_t* vb, uint8_t* kto,
                        uint8_t* vto, int left) __attribute__((always_inline)) {
    constexpr int NK = 2 * NJ, NV = 4 * NT, AHEAD = D <= 64 ? 3 : 2;
    const auto key = [&](int i) __attribute__((always_inline)) {
      return *reinterpret_cast<const V8*>(kb + lane * 16 + (i % 2 * NJ + i / 2) * L::KF);
    };
    const auto value = [&](int i) __attribute__((always_inline)) { return values(vb, i % NT, i / NT / 2, i / NT % 2); };
    f16x8 pr[4];
    float lp = 0.f;
    V8 k[AHEAD];
    s16x8 v[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; i++) k[i] = key(i);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) next.t[t][e] = 0.f;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < NK; i++) {
      next.t[i % 2] = mfma_w(k[i % AHEAD], q[i / 2], next.t[i % 2]);
      if (i + AHEAD < NK) k[i % AHEAD] = key(i + AHEAD);
      else v[i + AHEAD - NK] = value(i + AHEAD - NK);
#pragma unroll
      for (int x = i * 16 / NK; x < (i + 1) * 16 / NK; x++) {   // sixteen pairs
        const f16x2 p = two(now, x, kc, ref);
        pr[x / 4][2 * x % 8] = p[0], pr[x / 4][2 * x % 8 + 1] = p[1];
        lp = __builtin_amdgcn_fdot2(p, (f16x2){(f16)1.f, (f16)1.f}, lp, false);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    l += lp;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      acc[i % NT] = mfma_w(__builtin_bit_cast(f16x8, v[i % AHEAD]), pr[i / NT], acc[i % NT]);
      if (i + AHEAD < NV) v[i % AHEAD] = value(i + AHEAD);
#pragma unroll
      for (int x = i * 4 * RAW / NV; x < (i + 1) * 4 * RAW / NV; x++) {   // halves of pieces
        if (x < 2 * RAW) widen_key(kto, x / 2, x % 2, T());
        else widen_value(vto, left, (x - 2 * RAW) / 2, x % 2, f16());
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // The same of values in bf16. Those of NaN were left out of LDS: the queries that see them get it at the end.
  const auto add_odd = [&](int p, int64_t at, const uint8_t* vb, const Scores& s, float kc, float ref) __attribute__((always_inline)) {
    float lp = 0.f;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        u32x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s.t[t][8 * u + e], kc, -ref));
          const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s.t[t][8 * u + e + 1], kc, -ref));
          lp += x + y;
          unsigned xy, left;
          split2(x, y, xy, left);
          hi[e / 2] = xy;
          lo[e / 2] = left;
        }
#pragma unroll
        for (int d = 0; d < NT; d++) {
          const bf16x8 v = __builtin_bit_cast(bf16x8, values(vb, d, t, u));
          acc[d] = mfma_w(v, __builtin_bit_cast(bf16x8, lo), mfma_w(v, __builtin_bit_cast(bf16x8, hi), acc[d]));
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    l += lp;
    // Few such pages hold a NaN: all scales are looked at with scalar loads, a word at a time, before a lane looks for its own
    // query. (Vector loads there, or the words held from the page's start, moved registers of the ordinary rounds: 2 % of
    // their time at head width 128 and 6 at 256.)
    const uint8_t* vs = a.vs + at * (kPage4 * NT);
    const scalar_ints words = (scalar_ints)(uintptr_t)vs;
    unsigned beyond = 0;
#pragma unroll 1
    for (int i = 0; i < kPage4 * NT / 4; i += 16)
#pragma unroll
      for (int j = 0; j < 16; j++) beyond |= beyond_bytes(words[i + j]);
    if (beyond)
#pragma unroll 1
      for (int i = 0; i < kPage4 * NT; i++)
        if (vs[i] >= 253 && p * kPage4 + i % kPage4 < limit) poison |= 1u << i / kPage4;
  };

  if (p0 < p1) {
    // Round p takes the exponentials of page p's scores, made in the round before, while the matrix units make page p + 1's,
    // and adds its values while page p + 2's keys and p + 1's values are widened. Keys of p + 3 and values of p + 2 are on
    // their way.
    uint8_t* const keys[2] = {lds, lds + L::KEYS};
    uint8_t* const vals[2] = {lds + 2 * L::KEYS, lds + 2 * L::KEYS + kPage4 * L::VROW};
    int pages[5];   // numbers of pages p .. p + 4
#pragma unroll
    for (int i = 0; i < 5; i++) pages[i] = entry(p0 + i);
    constexpr bool EXACT = __is_same(T, bf16);   // keys of any scale are what they are
    const auto keys_at = [&](int i) __attribute__((always_inline)) { load(a.k, a.ks, place(pages[i]), tid, kraw); };
    const auto values_at = [&](int i) __attribute__((always_inline)) { load(a.v, a.vs, place(pages[i]), vid, vraw); };
    int p = p0;
    Scores s0, s1;
    Check kc0, kc1, vc0, vc1;   // of the keys and values that this round and the next one widen
    keys_at(0);
    values_at(0);
    ask(a.ks, place(pages[0]), kc0);
    ask(a.ks, place(pages[1]), kc1);
    ask(a.vs, place(pages[0]), vc0);
    bool odd = (!EXACT && (is_odd(p0, kc0) | is_odd(p0 + 1, kc1))) | is_odd(p0, vc0);
    if (__builtin_expect(!odd, 1)) {
      widen_keys(keys[0], T());
      widen_values(vals[0], most - p0 * kPage4, f16());
      keys_at(1);
      ring_barrier();
      product(keys[0], s0);
      widen_keys(keys[1], T());
      if (!EXACT) ask(a.ks, place(pages[2]), kc0);
      ask(a.vs, place(pages[1]), vc0);
      keys_at(2);
      values_at(1);
      if (!EXACT) ask(a.ks, place(pages[3]), kc1);
      ask(a.vs, place(pages[2]), vc1);
      const auto round = [&](auto parity, Scores& now, Scores& next, Check& kcheck, Check& vcheck) __attribute__((always_inline)) {
        constexpr int P = decltype(parity)::value;
        // Page p + 1's keys and page p's values stand in LDS, and every wave is done with page p's keys and p - 1's
        // values. (__syncthreads would wait for the codes asked for, too.)
        ring_barrier();
        odd |= (!EXACT && is_odd(p + 2, kcheck)) | is_odd(p + 1, vcheck);
        if (__builtin_expect(odd, 0)) return;
        const int left = most - (p + 1) * kPage4;
        if (p * kPage4 < wmost) {
          float kc;
          const float ref = exponents(p, (unsigned)pages[0] >= (unsigned)a.pages, now, kc);
          both(now, next, kc, ref, keys[1 - P], vals[P], keys[P], vals[1 - P], left);
        } else {
          widen_keys(keys[P], T());
          widen_values(vals[1 - P], left, f16());
        }
        keys_at(3);
        values_at(2);
        if (!EXACT) ask(a.ks, place(pages[4]), kcheck);
        ask(a.vs, place(pages[3]), vcheck);
#pragma unroll
        for (int i = 0; i < 4; i++) pages[i] = pages[i + 1];
        p++;
        pages[4] = entry(p + 4);
      };
      while (p < p1 && !odd) {
        round(Const<0>(), s0, s1, kc0, vc0);
        if (p < p1 && !odd) round(Const<1>(), s1, s0, kc1, vc1);
      }
    }
    // From the first page that fp16 does not hold on (and the few before it that are on their way) a page at a time, nothing on
    // its way: 2,000 fp16 queries of 4 x 4 heads behind 8,000 tokens with such a block of values in none of the pages, the middle
    // one, the first and all at head width 32 100, 101, 101 and 128 us, at 64 119, 129, 150 and 210, at 128 179, 194, 232 and
    // 335, at 256 510, 617, 682 and 1,030; of keys the same, and 121, 192, 307 and 870 in all.
    for (; p < p1; p++) {
      pages[0] = entry(p);
      const int64_t at = place(pages[0]);
      keys_at(0);
      values_at(0);
      ask(a.ks, at, kc0);
      ask(a.vs, at, vc0);
      const bool kodd = !EXACT && is_odd(p, kc0), vodd = is_odd(p, vc0);
      const int left = most - p * kPage4;
      ring_barrier();
      if (kodd) widen_keys(keys[0], bf16());
      else widen_keys(keys[0], T());
      if (vodd) widen_values(vals[0], left, bf16());
      else widen_values(vals[0], left, f16());
      ring_barrier();
      if (p * kPage4 >= wmost) continue;
      if (kodd) product_odd(keys[0], s0);
      else product(keys[0], s0);
      float kc;
      const float ref = exponents(p, (unsigned)pages[0] >= (unsigned)a.pages, s0, kc);
      if (vodd) {
        add_odd(p, at, vals[0], s0, kc, ref);
      } else {
        f16x8 pr[4];
        probabilities(s0, kc, ref, pr);
        add_values(vals[0], pr);
      }
    }
  }

#pragma unroll
  for (int d = 0; d < NT; d++)
    if (poison >> d & 1)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[d][e] = __builtin_nanf("");
  const auto l32 = __builtin_amdgcn_permlane32_swap(__float_as_int(l), __float_as_int(l), false, false);
  l = __int_as_float(l32[0]) + __int_as_float(l32[1]);
  if (too_long) l = __builtin_nanf("");
  if (!real) return;
  const int64_t bh = (int64_t)b * a.H + h, place8 = (bh * a.rows + row) * a.splits + split;
  const int64_t all = (int64_t)gridDim.z * a.H * a.rows * a.splits;
  const float inv = a.splits > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
  T* op = (T*)a.o + b * a.os[0] + (int64_t)(row / a.G) * a.os[1] + (int64_t)(h * a.G + row % a.G) * a.os[2];
#pragma unroll
  for (int d = 0; d < NT; d++)
#pragma unroll
    for (int g = 0; g < 2; g++) {
      float f[8];
#pragma unroll
      for (int c = 0; c < 8; c++) f[c] = acc[d][8 * g + c] * inv;
      const int channel = 32 * d + 16 * g + 8 * hh;
      if (a.splits > 1) {
        float* to = a.part + place8 * D + channel;
        *reinterpret_cast<f32x4*>(to) = (f32x4){f[0], f[1], f[2], f[3]};
        *reinterpret_cast<f32x4*>(to + 4) = (f32x4){f[4], f[5], f[6], f[7]};
      } else {
        store8(op + channel, f);
      }
    }
  if (a.splits > 1 && hh == 0) {
    a.part[all * D + 2 * place8] = m == -__builtin_inff() ? 0.f : m;
    a.part[all * D + 2 * place8 + 1] = l;
  }
}

template <typename T, int D>
int launch_wide(const Attend4Args& a, dim3 grid, hipStream_t st) {
  constexpr int LDS = 2 * (WideLds<D>::KEYS + kPage4 * WideLds<D>::VROW);
  const auto kern = attend4_wide_kernel<T, D>;
  if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess)
    return check_launch("cache4_attention: set LDS size");
  hipLaunchKernelGGL(kern, grid, dim3(256), LDS, st, a);
  return LDX_OK;
}

template <typename T, int D>
int launch_d(const Attend4Args& a, int batch, hipStream_t st) {
  const dim3 grid((unsigned)a.splits * (unsigned)(a.H * ((a.rows + a.tile - 1) / a.tile)), 1, (unsigned)batch);
  if (a.tile == 16) {
    hipLaunchKernelGGL((attend4_kernel<T, D>), grid, dim3(64 * kWaves4), 0, st, a);
  } else if (int rc = launch_wide<T, D>(a, grid, st)) {
    return rc;
  }
  launch_join<T, D>(a, (int64_t)batch * a.H * a.rows, st);
  return check_launch("cache4_attention");
}

template <typename T>
int launch_t(const Attend4Args& a, int D, int batch, hipStream_t st) {
  if (D == 32) return launch_d<T, 32>(a, batch, st);
  if (D == 64) return launch_d<T, 64>(a, batch, st);
  if (D == 128) return launch_d<T, 128>(a, batch, st);
  return launch_d<T, 256>(a, batch, st);
}

int check_cache(const char* what, const ldx_cache4& c) {
  if (!c.k || !c.v || !c.k_scales || !c.v_scales) return fail("%s: null pointer", what);
  if (c.pages < 1 || c.heads < 1 || c.heads > 8192) return fail("%s: %d pages, %d heads", what, c.pages, c.heads);
  if (c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)
    return fail("%s: head_dim %d is not 32, 64, 128 or 256", what, c.head_dim);
  if ((uintptr_t)c.k % 16 || (uintptr_t)c.v % 16 || (uintptr_t)c.k_scales % 16 || (uintptr_t)c.v_scales % 16)
    return fail("%s: codes and scales must be aligned to 16 bytes", what);
  return LDX_OK;
}

int check_store(const char* what, const ldx_cache4& c, int batch, int tokens, int dtype, int64_t table_pitch, int width) {
  if (int rc = check_cache(what, c)) return rc;
  if (dtype != LDX_DTYPE_F16 && dtype != LDX_DTYPE_BF16 && dtype != LDX_DTYPE_F32)
    return fail("%s: dtype %d is not LDX_DTYPE_F16, LDX_DTYPE_BF16 or LDX_DTYPE_F32", what, dtype);
  if (batch < 1 || batch > 65535 || tokens < 1 || tokens > 1 << 28 || width < 1 || width > (1 << 24))
    return fail("%s: batch %d, %d tokens, %d pages a sequence", what, batch, tokens, width);
  if (table_pitch < width) return fail("%s: table pitch below %d", what, width);
  return LDX_OK;
}

// Pages that `tokens` tokens from any place on may touch, by a head's keys and values, by sequences.
dim3 store_grid(const ldx_cache4& c, int batch, int tokens) {
  return dim3((unsigned)((tokens + 2 * (int64_t)kPage4 - 2) / kPage4), 2 * (unsigned)c.heads, (unsigned)batch);
}

// How a call is laid out. The host knows only how many pages a table's row holds; the kernels divide the
// pages that a sequence has.
struct Plan {
  bool wide;    // pages shared through LDS by 128 rows of a cache head, or streamed by 16
  int splits;   // parts that a sequence's pages may be spread over
};

constexpr int kLeastChunk = 8;   // pages of a part at least: two for each wave

size_t split_bytes(const ldx_cache4_attention_args* p, int splits) {
  if (splits < 2) return 0;
  const size_t rows = (size_t)p->q_len * (p->q_heads / p->cache.heads);
  return (size_t)p->batch * p->cache.heads * rows * splits * (p->cache.head_dim + 2) * sizeof(float);
}

// What partial results may take at most. (It bounds the join's launch, too.)
constexpr size_t kMostPartBytes = (size_t)256 << 20;

Plan plan_of(const ldx_cache4_attention_args* p) {
  const int64_t heads = (int64_t)p->batch * p->cache.heads, rows = (int64_t)p->q_len * (p->q_heads / p->cache.heads);
  const int64_t most = (p->width + kLeastChunk - 1) / kLeastChunk;
  Plan plan;
  const int D = p->cache.head_dim;
  // A page of 16 rows is a unit of work. Sharing pages is ahead from about 40,000 of them on, at head width 256, where a page
  // costs more to widen, earlier the more groups of rows there are for the CUs. A causal call's us shared and streamed at head
  // widths 32, 64, 128 and 256: 8 heads of 512 rows behind 8,000 tokens (34,000 units, 32 groups) 31 32, 38 38, 51 51, 96 103;
  // 4 of 1,900 behind 2,000 (29,000, 60) 27 26, 31 30, 45 41, 84 89, behind 4,000 (44,000) 34 35, 41 43, 57 59, 109 124;
  // 15 of 1,024 behind 500 (23,000, 120) 22 22, 28 25, 39 37, 70 80; 1 of 1,900 behind 16,000 (33,000, 15) 45 34, 50 39,
  // 69 52, 140 109.
  const int64_t groups = heads * ((rows + kWideRows - 1) / kWideRows), work = heads * ((rows + 15) / 16) * p->width;
  plan.wide = rows >= kWideRows && work >= (D < 256 || groups < 32 ? 40000 : groups < 64 ? 28000 : 20000);
  int64_t s = 1;
  if (plan.wide) {
    // Rounds of workgroups on the CUs' places, the pages of a round, and what a part more costs: 3 pages of a round
    // to join, or what it writes and the join reads, at 4.5 TB/s and 2.2 us a page of a round.
    const int64_t places = D == 32 ? 768 : D <= 128 ? 512 : 256;
    const double traffic = 8e-7 * (double)(heads * rows) * (D + 2), part = traffic > 3.0 ? traffic : 3.0;
    double best = 1e30;
    for (int64_t i = 1; i <= kFewParts && i <= most; i++) {
      if (split_bytes(p, (int)i) > kMostPartBytes) break;
      const double cost = (double)((groups * i + places - 1) / places) * ((p->width + i - 1) / i) + part * i;
      if (cost < best) best = cost, s = i;
    }
  } else {
    // Two workgroups for each CU: a query of 8 x 4 heads for each of 32 sequences of up to 16,384 tokens 83 us with the join
    // at 128 and 56 at 64, with four 84 and 57, with eight 86 and 54, with one 97 and 73; 16 of 256 behind 8,192 55, 58, 67
    // and 86. Where that leaves one to some CUs and two to others, each in two parts, three to a CU: 300 heads behind up to
    // 5,000 tokens 45 and 40 us at 128, 31 and 30 at 64, 95 and 87 at 256, 400 52 and 50, 37 and 33, 106 and 100, 470 52 and 54,
    // 37 and 39, 118 and 125. Below 32 pages a join costs more than it saves: a query of 8 heads behind 2,040 tokens 10.5 us
    // at 64 and 12 at 128 in parts, 12.7 and 16 in one; behind 1,000 tokens 9.7 and 11.6, 8.8 and 10.7.
    const int64_t units = heads * ((rows + 15) / 16);
    s = units > 256 && units <= 400 ? 2 : 512 / units;
    if (s > most) s = most;
    if (p->width < 32) s = 1;
  }
  plan.splits = (int)(s < 1 ? 1 : s > kMostParts ? kMostParts : s);
  return plan;
}

int check_attention(const ldx_cache4_attention_args* p) {
  if (!p || !p->q || !p->o || !p->table || !p->lengths) return fail("cache4_attention: null pointer");
  if (int rc = check_cache("cache4_attention", p->cache)) return rc;
  if (p->dtype != LDX_DTYPE_F16 && p->dtype != LDX_DTYPE_BF16)
    return fail("cache4_attention: dtype %d is not LDX_DTYPE_F16 or LDX_DTYPE_BF16", p->dtype);
  if (p->batch < 1 || p->batch > 65535 || p->q_len < 1 || p->width < 1 || p->width > (1 << 24))
    return fail("cache4_attention: batch %d, %d queries, %d pages a sequence", p->batch, p->q_len, p->width);
  if (p->q_heads < 1 || p->q_heads % p->cache.heads)
    return fail("cache4_attention: %d query heads over %d cache heads", p->q_heads, p->cache.heads);
  const int64_t rows = (int64_t)p->q_len * (p->q_heads / p->cache.heads);
  if (rows * p->cache.heads * p->batch > 0x7fffffff || (rows + 15) / 16 * p->cache.heads > 1 << 23)   // 2^31 threads
    return fail("cache4_attention: %d x %d queries of %d heads are more than one launch takes", p->batch, p->q_len,
                p->q_heads);
  if (p->table_pitch < p->width) return fail("cache4_attention: table pitch below %d", p->width);
  if (!(p->scale > -1e30f && p->scale < 1e30f)) return fail("cache4_attention: scale %g", (double)p->scale);
  return LDX_OK;
}

}  // namespace
}  // namespace ldx

using namespace ldx;

extern "C" int ldx_cache4_append(const ldx_cache4_append_args* p, void* stream) {
  if (!p || !p->k || !p->v || !p->table || !p->starts) return fail("cache4_append: null pointer");
  if (int rc = check_store("cache4_append", p->cache, p->batch, p->tokens, p->dtype, p->table_pitch, p->width)) return rc;
  const ldx_cache4& c = p->cache;
  const Store4Args a = {{(uint8_t*)c.k, (uint8_t*)c.v}, {(uint8_t*)c.k_scales, (uint8_t*)c.v_scales},
                        {(void*)p->k, (void*)p->v},
                        {{p->k_stride[0], p->k_stride[1], p->k_stride[2]}, {p->v_stride[0], p->v_stride[1], p->v_stride[2]}},
                        c.pages, c.heads, p->tokens, p->table, p->table_pitch, p->width, p->starts, p->counts, nullptr, false};
  const dim3 grid = store_grid(c, p->batch, p->tokens);
  if (p->dtype == LDX_DTYPE_F16) launch_store<f16, false>(a, c.head_dim, grid, as_stream(stream));
  else if (p->dtype == LDX_DTYPE_BF16) launch_store<bf16, false>(a, c.head_dim, grid, as_stream(stream));
  else launch_store<float, false>(a, c.head_dim, grid, as_stream(stream));
  return check_launch("cache4_append");
}

extern "C" int ldx_cache4_read(const ldx_cache4_read_args* p, void* stream) {
  if (!p || !p->k || !p->v || !p->table || !p->lengths) return fail("cache4_read: null pointer");
  if (int rc = check_store("cache4_read", p->cache, p->batch, p->tokens, p->dtype, p->table_pitch, p->width)) return rc;
  const ldx_cache4& c = p->cache;
  const Store4Args a = {{(uint8_t*)c.k, (uint8_t*)c.v}, {(uint8_t*)c.k_scales, (uint8_t*)c.v_scales}, {p->k, p->v},
                        {{p->k_stride[0], p->k_stride[1], p->k_stride[2]}, {p->v_stride[0], p->v_stride[1], p->v_stride[2]}},
                        c.pages, c.heads, p->tokens, p->table, p->table_pitch, p->width, p->starts, nullptr, p->lengths,
                        p->fill != 0};
  const dim3 grid = store_grid(c, p->batch, p->tokens);
  if (p->dtype == LDX_DTYPE_F16) launch_store<f16, true>(a, c.head_dim, grid, as_stream(stream));
  else if (p->dtype == LDX_DTYPE_BF16) launch_store<bf16, true>(a, c.head_dim, grid, as_stream(stream));
  else launch_store<float, true>(a, c.head_dim, grid, as_stream(stream));
  return check_launch("cache4_read");
}

extern "C" size_t ldx_cache4_attention_workspace_bytes(const ldx_cache4_attention_args* p) {
  return check_attention(p) == LDX_OK ? split_bytes(p, plan_of(p).splits) : 0;
}

extern "C" int ldx_cache4_attention_rows(const ldx_cache4_attention_args* p) {
  if (int rc = check_attention(p)) return rc;
  return plan_of(p).wide ? kWideRows : 16;
}

extern "C" int ldx_cache4_attention(const ldx_cache4_attention_args* p, void* stream) {
  if (int rc = check_attention(p)) return rc;
  Plan plan = plan_of(p);
  if (plan.splits > 1 && (!p->workspace || p->workspace_bytes < split_bytes(p, plan.splits))) plan.splits = 1;
  if (plan.splits > 1 && (uintptr_t)p->workspace % 16) return fail("cache4_attention: workspace not aligned");
  const int G = p->q_heads / p->cache.heads;
  const Attend4Args a = {(const uint8_t*)p->cache.k, (const uint8_t*)p->cache.v, (const uint8_t*)p->cache.k_scales,
                         (const uint8_t*)p->cache.v_scales, p->cache.pages, p->cache.heads,
                         p->q, {p->q_stride[0], p->q_stride[1], p->q_stride[2]},
                         p->o, {p->o_stride[0], p->o_stride[1], p->o_stride[2]},
                         G, p->q_len, G * p->q_len, p->scale * 1.4426950408889634f,
                         p->table, p->table_pitch, p->width, p->lengths, p->starts, plan.splits, kLeastChunk,
                         plan.wide ? kWideRows : 16,
                         (float*)p->workspace};
  hipStream_t st = as_stream(stream);
  return p->dtype == LDX_DTYPE_F16 ? launch_t<f16>(a, p->cache.head_dim, p->batch, st)
                                   : launch_t<bf16>(a, p->cache.head_dim, p->batch, st);
}
