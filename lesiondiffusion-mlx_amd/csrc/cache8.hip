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
  int pages, H, tokens;
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
// codes. A thread keeps its D / 32 groups of eight channels of a token between the two. Values go through
// LDS, where they are turned channel by token (rows of 68 bytes: the groups of a token meet different banks).
// Bound by memory where there are many tokens: 8 sequences of 9,000 with 8 heads of 128 in fp16 85 us, 5.2 TB/s
// (read twice and turned in rows of 64 bytes 118); one token for each of 48 sequences 5.7 us, latency.
template <typename T, int D>
__global__ __launch_bounds__(256) void append8_kernel(AppendArgs a) {
  constexpr int UNITS = D / 8, MOST = D / 32, PITCH = kPage8 + 4;
  __shared__ float red[4];
  __shared__ __align__(16) uint8_t turned[D * PITCH];
  const int b = blockIdx.z, h = blockIdx.y >> 1, which = blockIdx.y & 1, tid = threadIdx.x;
  const int start = a.starts[b];
  const int n = a.counts ? min(a.counts[b], a.tokens) : a.tokens;
  if (start < 0 || n <= 0) return;
  const int64_t end = (int64_t)start + n;
  const int64_t slot = start / kPage8 + (int64_t)blockIdx.x, first = slot * kPage8;
  if (first >= end || slot >= a.width) return;
  const int page = a.table[b * a.tp + slot];
  if ((unsigned)page >= (unsigned)a.pages) return;
  uint8_t* scale = a.scales[which] + (int64_t)page * a.H + h;
  uint8_t* codes = a.codes[which] + ((int64_t)page * a.H + h) * D * kPage8;
  const int was = *scale;
  const int lo = (int)max(start - first, (int64_t)0), hi = (int)min(end - first, (int64_t)kPage8);
  const int chunks = (hi - lo) * UNITS;
  const int64_t tok = a.st[which][1];
  const T* src = (const T*)a.src[which] + b * a.st[which][0] + (first + lo - start) * tok + h * a.st[which][2];
  float f[MOST][8];
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < MOST; j++) {
    const int c = tid + 256 * j;
    if (c < chunks) {
      load8(src + c / UNITS * tok + c % UNITS * 8, f[j]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) f[j][i] = 0.f;
    }
  }
#pragma unroll
  for (int j = 0; j < MOST; j++)
#pragma unroll
    for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(f[j][i]));
  amax = wave_max(amax);
  if ((tid & 63) == 0) red[tid >> 6] = amax;
  __syncthreads();   // behind it every thread has read the old scale, too
  amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  int to = scale_byte(amax);
  const bool rises = lo > 0 && to > was;
  if (lo > 0 && to < was) to = was;
  // (254, which no append makes, may be an older page's: its inverse, 2^-127, is a subnormal number.)
  const float inv = to < 254 ? inverse_of(to) : __int_as_float(0x00400000);
  if (tid == 0) *scale = (uint8_t)to;
  if (which == 0) {
    if (rises)
      for (int c = tid; c < lo * D / 4; c += 256) {
        int* w = reinterpret_cast<int*>(codes) + c;
        *w = recode4(*w, was, to);
      }
#pragma unroll
    for (int j = 0; j < MOST; j++) {
      const int c = tid + 256 * j;
      if (c >= chunks) break;
      const i32x2 w = {encode4(f[j][0], f[j][1], f[j][2], f[j][3], inv), encode4(f[j][4], f[j][5], f[j][6], f[j][7], inv)};
      __builtin_nontemporal_store(w, reinterpret_cast<i32x2*>(codes + (lo + c / UNITS) * D + c % UNITS * 8));
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < MOST; j++) {
    const int c = tid + 256 * j;
    if (c >= chunks) break;
    const int w0 = encode4(f[j][0], f[j][1], f[j][2], f[j][3], inv), w1 = encode4(f[j][4], f[j][5], f[j][6], f[j][7], inv);
    uint8_t* t = turned + c % UNITS * 8 * PITCH + lo + c / UNITS;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      t[i * PITCH] = (uint8_t)(w0 >> (8 * i));
      t[(i + 4) * PITCH] = (uint8_t)(w1 >> (8 * i));
    }
  }
  __syncthreads();
  // Four tokens of a channel at a time: older ones (re-coded where the scale rises) below lo, new ones
  // up to hi, the rest as it is.
  const int g0 = rises ? 0 : lo / 4, g1 = (hi + 3) / 4, per = g1 - g0;
  for (int c = tid; c < D * per; c += 256) {
    const int d = c / per, t0 = (g0 + c % per) * 4, at = d * kPage8 + t0;
    int w = *reinterpret_cast<const int*>(turned + d * PITCH + t0);
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
    __builtin_nontemporal_store(w, reinterpret_cast<int*>(codes + at));
  }
}

template <typename T>
void launch_append(const AppendArgs& a, int D, dim3 grid, hipStream_t st) {
  if (D == 32) hipLaunchKernelGGL((append8_kernel<T, 32>), grid, dim3(256), 0, st, a);
  else if (D == 64) hipLaunchKernelGGL((append8_kernel<T, 64>), grid, dim3(256), 0, st, a);
  else if (D == 128) hipLaunchKernelGGL((append8_kernel<T, 128>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((append8_kernel<T, 256>), grid, dim3(256), 0, st, a);
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
  int splits, chunk;     // parts of a sequence; least pages of a part
  int tile;              // rows of a workgroup
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
// Eight codes times s, a power of two; as they stand, and within 2^-15 .. 2^7, e4m3's values fit fp16 and
// bf16 exactly.
__device__ __forceinline__ void codes_as(int lo, int hi, float s, f16x8& r) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, s, false);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, s, true);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, s, false);
  const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, s, true);
  r = (f16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ void codes_as(int lo, int hi, float s, bf16x8& r) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
  r = (bf16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The largest of three numbers, NaN ignored where there is another. (fmaxf of a product's results costs a
// second instruction for each, which would quiet a signalling NaN.)
__device__ __forceinline__ float max3_f(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Entry p of a page table by a scalar load, whose result is awaited where it is used. (As a vector load of
// one address its value is moved to a scalar, and so awaited, where it is loaded.)
typedef const __attribute__((address_space(4))) int32_t* scalar_ints;
__device__ __forceinline__ int table_entry(const int32_t* table, int p) { return ((scalar_ints)(uintptr_t)table)[p]; }

// A page's scale byte, loaded by every lane (none is 0 that the compiler does not know) for the same reason.
__device__ __forceinline__ int scale_entry(const uint8_t* scales, int64_t at, int none) { return scales[at + none]; }

// The keys that a query sees: limit = min(length, start + i + 1) with starts, the length without.
__device__ __forceinline__ int key_limit(const Attend8Args& a, int len, int64_t start, int row) {
  if (!a.starts) return len;
  const int64_t c = start + row / a.G + 1;
  return (int)(c < 0 ? 0 : c < len ? c : len);
}

// The softmax scale's size, in powers of two (1 for a scale of 0); its sign, or 0, is the queries'.
__device__ __forceinline__ float soft_scale(const Attend8Args& a) { return a.scale == 0.f ? 1.f : fabsf(a.scale); }

// A page's scale, any E8M0 byte (append makes 1 to 247); infinity for 255.
__device__ __forceinline__ float any_scale(int byte) { return byte ? scale_of(byte) : __int_as_float(0x00400000); }

// That and the keys' scale (c and a wave's byte) go onto the scores inside the exponential: an exponent more on c, in
// scalar arithmetic, but where it leaves the normal numbers. Kept a number larger than 0, so that a masked score stays
// minus infinity and a score of 0 stays 0; least scales make it a subnormal number, which the fused multiply-add takes
// as it is.
__device__ __forceinline__ float score_scale(int c, int byte) {
  const int e = (c >> 23) + byte - 127;
  if (c >= 0x00800000 && e >= 1 && e <= 253) return __int_as_float(c + (byte - 127) * (1 << 23));
  return fminf(fmaxf(__int_as_float(c) * any_scale(byte), 1.4e-45f), 3.0e38f);
}

// A query's reference for its exponentials is 2^kRaise below its maximum, and follows it only where that passes it by
// kSlack more (in powers of two): the sums are seldom multiplied then. Probabilities reach 2^15, and fp16 holds those
// from 2^-21 of the largest on to 2^-11 of themselves and smaller ones to 2^-32 of it, so that many small ones beside
// a dominant one keep their weight (with the maximum as the reference 2^-14 and 2^-25: 100,000 keys at 2^-23.6 of the
// first one weighed a quarter less). What is summed is kept kLower times as large, so that the values' range is fp32's.
constexpr float kSlack = 8.f, kRaise = 7.f, kLower = 0x1p-7f;

// A score times its scale goes into the exponential unrounded, its reference does not: what the reference's rounding
// left out, up to 2^-24 of it, moves all probabilities of a query by one factor, which beyond scores of 2^28 leaves
// fp16. Pages that may hold scores of 2^22 and more have them multiplied, and rounded, first, and have no slack (7 less
// is rounded, too: to 8 less, or to nothing from 2^27 on). This is the least scale byte of such a page, by the largest
// code and the sums of the wave's queries' magnitudes, of which a lane holds one of `lanes` parts.
__device__ __forceinline__ int far_byte(float sum, int lanes, float c) {
  const float most = wave_max(sum) * (448.f * lanes) * c;   // below 2^(e - 126)
  return 127 + 22 + 127 - (__builtin_amdgcn_readfirstlane(__float_as_int(most)) >> 23);
}

// l and eight probabilities: as the products take them, in fp16 (their sum in fp32), so that rounding moves
// both sides of the quotient alike. Two at a time: half the additions of fp32 numbers.
__device__ __forceinline__ float sum8(f16x8 p, float l) {
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    l = __builtin_amdgcn_fdot2((f16x2){p[i], p[i + 1]}, (f16x2){(f16)1.f, (f16)1.f}, l, false);
  return l;
}

// A value page's scale; 1 for 255, NaN, whose queries get NaN by their sum.
__device__ __forceinline__ float page_scale(int byte) { return byte == 255 ? 1.f : any_scale(byte); }

// Channels at .. at + 7 of a query, with the softmax scale's sign; their magnitudes are added to sum.
template <typename T>
__device__ __forceinline__ typename Vec8<T>::V query8(const Attend8Args& a, const T* q, int at, bool real, float& sum) {
  float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (real) load8(q + at, f);
  const float sign = a.scale > 0.f ? 1.f : a.scale < 0.f ? -1.f : 0.f;
  typename Vec8<T>::V v;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    v[e] = (T)(f[e] * sign);
    sum += fabsf(f[e]);
  }
  return v;
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
// sum as it is added to the running one, so that probabilities are what fp16 rounds.
//
// What bounds it while tokens are produced one by one is reading the cache. A wave holds one page's keys
// and one page's values and always has one of the two on its way: the next page's keys are asked for when
// the scores are done, the next values when the sums are. (Two whole pages in registers left one wave a
// SIMD at head width 128.) The loads go through buffer descriptors that end at the page, or at nothing
// behind the last page, so that every round issues the same loads and waits for the older half only. (One
// query of 8 x 4 heads of 128 for each of 32 sequences of up to 8,192 tokens 63 us and 5 to join the parts,
// 5.4 TB/s; with a page's loads issued where they are used 108.)
constexpr int kAttendWaves = 4;

template <typename T, int D>
__global__ __launch_bounds__(64 * kAttendWaves, D == 256 ? 1 : D == 128 ? 2 : 3) void attend8_kernel(Attend8Args a) {
  typedef typename Vec8<T>::V V8;
  constexpr int ND = D / 16;              // channel tiles
  constexpr int NK = D / 32;              // products per key tile
  __shared__ float sm[kAttendWaves][16], sl[kAttendWaves][16];
  __shared__ float sacc[kAttendWaves][16][D + 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int b = blockIdx.z, split = blockIdx.x % a.splits, tiles = (a.rows + 15) / 16, tile = blockIdx.x / a.splits;
  const int h = tile / tiles, row0 = tile % tiles * 16;
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
  const int chunk = max((npages + a.splits - 1) / a.splits, a.chunk);
  const int p0 = a.splits > 1 ? split * chunk : 0, p1 = a.splits > 1 ? min(p0 + chunk, npages) : npages;
  if (p0 >= p1 && split > 0) return;   // the join knows that there is no such part

  const float c = soft_scale(a);
  const int c_bits = __builtin_amdgcn_readfirstlane(__float_as_int(c));
  V8 q[NK];
  float q_sum = 0.f;
  {
    const T* qp = (const T*)a.q + b * a.qs[0] + (int64_t)(row / a.G) * a.qs[1] + (int64_t)(h * a.G + row % a.G) * a.qs[2];
    // D >= 64: the products 2 j and 2 j + 1 take channels 64 j + 16 g + 0..7 and + 8..15, so that a
    // key's bytes are read 16 at a time.
#pragma unroll
    for (int j = 0; j < NK; j++) q[j] = query8<T>(a, qp, D == 32 ? 8 * g : 64 * (j / 2) + 16 * g + 8 * (j % 2), real, q_sum);
  }

  float acc[ND][4];   // single numbers: as vectors, every branch that changes them copies them
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int i = 0; i < 4; i++) acc[d][i] = 0.f;
  float m = -__builtin_inff(), l = 0.f;
  uint64_t poison = 0;   // bit 4 d + i: acc[d][i] holds a NaN value that its query sees

  const int32_t* table = a.table + b * a.tp;
  const unsigned koff = (unsigned)(16 * (r >> 2) + (r & 3)) * D + (D == 32 ? 8 : 16) * g;
  const unsigned voff = (unsigned)r * kPage8 + 16 * g;
  i32x4 kc[D == 32 ? 2 : D / 16];   // a page's keys (head width 32: two tiles of 8 bytes in one)
  i32x4 vc[ND];
  int ks, vs;
  // Where page p of the sequence stands (its head's place in the cache), and whether the cache has it.
  struct Place {
    int64_t at;
    bool missing;
  };
  int none = 0;
  asm volatile("" : "+v"(none));
  const auto place = [&](int page) {
    const bool missing = (unsigned)page >= (unsigned)a.pages;
    return Place{(int64_t)(missing ? 0 : page) * a.H + h, missing};
  };
  const auto load_k = [&](Place t, int p) {
    const __amdgpu_buffer_rsrc_t kr = make_rsrc(a.k + t.at * (kPage8 * D), p < p1 ? (unsigned)(kPage8 * D) : 0u);
    ks = scale_entry(a.ks, t.at, none);
    if constexpr (D == 32) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const auto w = __builtin_amdgcn_raw_buffer_load_b64(kr, koff, 4 * i * D, 0);
        kc[i / 2][i % 2 * 2] = (int)w[0];
        kc[i / 2][i % 2 * 2 + 1] = (int)w[1];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < NK / 2; j++) kc[i * (NK / 2) + j] = buffer_load16<i32x4>(kr, koff, 4 * i * D + 64 * j);
    }
  };
  const auto load_v = [&](Place t, int p) {
    const __amdgpu_buffer_rsrc_t vr = make_rsrc(a.v + t.at * (kPage8 * D), p < p1 ? (unsigned)(kPage8 * D) : 0u);
    vs = scale_entry(a.vs, t.at, none);
#pragma unroll
    for (int d = 0; d < ND; d++) vc[d] = buffer_load16<i32x4>(vr, voff, d * 16 * kPage8);
  };

  // Page numbers are known two rounds ahead; behind the last page the last one's is read again.
  const int last = max(p1 - 1, 0);
  const auto entry = [&](int p) { return table_entry(table, min(p, last)); };
  int p = p0 + wave;
  Place now = place(entry(p)), next = place(entry(p + kAttendWaves));
  int after = entry(p + 2 * kAttendWaves);
  load_k(now, p);
  load_v(now, p);
  const int far_from = far_byte(q_sum, 4, c);
  for (; p < p1; p += kAttendWaves) {
    const int ksb = __builtin_amdgcn_readfirstlane(ks);
    const bool none_k = ksb == 255, far = ksb >= far_from;
    const float scale = score_scale(c_bits, ksb), grow = far ? 1.f : scale;
    const int base = p * kPage8 + 16 * g;   // the lane's first token
    float s[16];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
      V8 kv;
      if constexpr (D == 32) {
        codes_as(kc[t / 2][t % 2 * 2], kc[t / 2][t % 2 * 2 + 1], 1.f, kv);
        o = mfma_q(kv, q[0], o);
      } else {
#pragma unroll
        for (int j = 0; j < NK / 2; j++) {
          const i32x4 w = kc[t * (NK / 2) + j];
          codes_as(w[0], w[1], 1.f, kv);
          o = mfma_q(kv, q[2 * j], o);
          codes_as(w[2], w[3], 1.f, kv);
          o = mfma_q(kv, q[2 * j + 1], o);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; i++) s[4 * t + i] = o[i];
      __builtin_amdgcn_sched_barrier(0);   // one tile's widened codes at a time
    }
    load_k(next, p + kAttendWaves);
    __builtin_amdgcn_sched_barrier(0);
    const float vscale = page_scale(vs) * kLower;
    if ((now.missing || none_k || vs == 255) && p * kPage8 < limit) l = __builtin_nanf("");   // (page 0 was read in a missing one's place)
    const bool cut = p * kPage8 + kPage8 > least;   // some query does not see the whole page
    if (cut || far) {
      int left = limit - base;
      pin_value(left);
      const float first = far ? scale : 1.f;
#pragma unroll
      for (int i = 0; i < 16; i++) s[i] = i < left ? s[i] * first : -__builtin_inff();
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 15; i += 2) mx = max3_f(mx, s[i], s[i + 1]);
    mx = max3_f(mx, s[15], s[15]);
    const auto x16 = __builtin_amdgcn_permlane16_swap(__float_as_int(mx), __float_as_int(mx), false, false);
    mx = max3_f(__int_as_float(x16[0]), __int_as_float(x16[1]), __int_as_float(x16[1]));
    const auto x32 = __builtin_amdgcn_permlane32_swap(__float_as_int(mx), __float_as_int(mx), false, false);
    const float mn = max3_f(m, __builtin_fmaf(__int_as_float(x32[0]), grow, -kRaise),
                            __builtin_fmaf(__int_as_float(x32[1]), grow, -kRaise));
    float ref = m == -__builtin_inff() ? 0.f : m;
    if (__any(mn - m > (far ? 0.f : kSlack))) {
      ref = mn == -__builtin_inff() ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m - ref);
      l *= alpha;
#pragma unroll
      for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[d][i] *= alpha;
      m = mn;
    }
    f16x8 pr[2];
    float lp = 0.f;   // the page's own sum, so that small ones do not go one by one into a large one
#pragma unroll
    for (int u = 0; u < 2; u++) {   // eight at a time; left alone, the sums are made behind the products below
#pragma unroll
      for (int i = 0; i < 8; i++) pr[u][i] = (f16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * u + i], grow, -ref));
      lp = sum8(pr[u], lp);
      pin_value(lp);
      __builtin_amdgcn_sched_barrier(0);
    }
    l += lp;
    if (cut) {
      // Tokens behind the sequence are whatever was there: zero them. Tokens that only some of the queries
      // see may be NaN, and zero times NaN is not zero: their codes are zeroed too, and a product of their
      // places with 1 for each token seen says which sums they belong in (one bit each, applied last).
      const int left = len - base;
      unsigned nan = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int n = left - 4 * i;
        const int keep = n >= 4 ? -1 : n <= 0 ? 0 : (int)(0xffffffffu >> (32 - 8 * n));
#pragma unroll
        for (int d = 0; d < ND; d++) {
          vc[d][i] &= keep;
          nan |= nan_bytes(vc[d][i]);
        }
      }
      if (__any(nan != 0)) {
        f16x8 seen[2];
#pragma unroll
        for (int i = 0; i < 16; i++) seen[i / 8][i % 8] = base + i < limit ? (f16)1.f : (f16)0.f;
        const __amdgpu_buffer_rsrc_t vr = make_rsrc(a.v + now.at * (kPage8 * D), (unsigned)(kPage8 * D));
#pragma unroll 1
        for (int d = 0; d < ND; d++) {
          const i32x4 w = buffer_load16<i32x4>(vr, voff, d * 16 * kPage8);
          f16x8 mk[2];
#pragma unroll
          for (int i = 0; i < 16; i++)
            mk[i / 8][i % 8] = i < left && ((nan_bytes(w[i / 4]) >> (8 * (i % 4))) & 0x80) ? (f16)1.f : (f16)0.f;
          const f32x4 marks = mfma16(mk[1], seen[1], mfma16(mk[0], seen[0], (f32x4){0.f, 0.f, 0.f, 0.f}));
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (marks[i] > 0.f) poison |= 1ull << (4 * d + i);
        }
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            int w = vc[d][i];
            pin_value(w);   // computed anew: kept from above, the bytes' bits double the registers
            vc[d][i] = w & ~(int)((nan_bytes(w) >> 7) * 255u);
          }
      }
    }
#pragma unroll
    for (int d = 0; d < ND; d++) {
      f16x8 v0, v1;
      codes_as(vc[d][0], vc[d][1], 1.f, v0);
      codes_as(vc[d][2], vc[d][3], 1.f, v1);
      const f32x4 o = mfma16(v1, pr[1], mfma16(v0, pr[0], (f32x4){0.f, 0.f, 0.f, 0.f}));
#pragma unroll
      for (int i = 0; i < 4; i++) acc[d][i] += o[i] * vscale;
      if (d % 2) __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_sched_barrier(0);
    load_v(next, p + kAttendWaves);
    __builtin_amdgcn_sched_barrier(0);
    now = next;
    next = place(after);
    after = entry(p + 3 * kAttendWaves);
  }

  if (poison) {
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (poison >> (4 * d + i) & 1) acc[d][i] = __builtin_nanf("");
  }
  // l over the four lane groups of a query, then the waves' states through LDS.
  const auto l16 = __builtin_amdgcn_permlane16_swap(__float_as_int(l), __float_as_int(l), false, false);
  l = __int_as_float(l16[0]) + __int_as_float(l16[1]);
  const auto l32 = __builtin_amdgcn_permlane32_swap(__float_as_int(l), __float_as_int(l), false, false);
  l = (__int_as_float(l32[0]) + __int_as_float(l32[1])) * kLower;
  if (g == 0) {
    sm[wave][r] = m;
    sl[wave][r] = l;
  }
#pragma unroll
  for (int d = 0; d < ND; d++) *reinterpret_cast<f32x4*>(&sacc[wave][r][16 * d + 4 * g]) = (f32x4){acc[d][0], acc[d][1], acc[d][2], acc[d][3]};
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

// ------------------------------------------------------------------- many queries of a cache head
//
// A workgroup takes 128 rows (queries x grouped heads), a wave 32 of them, and shares each page through
// LDS as 16-bit operands, so that a code is widened once for all of them. S^T = K Q^T and O^T += V^T P^T
// on 32 x 32 x 16 products: lane l holds query column l % 32, h = l / 32. Row 8 q + 4 h + i of a 32-token
// key tile is its token 16 h + 4 q + i, so that the scores a lane receives are 16 tokens in a row and the
// probabilities go into the second product as they lie, against eight tokens side by side of the turned
// values.
//
// LDS holds the operands in fragment order (a lane's 16 bytes at its place), the fragments padded so that
// 16 widening lanes, which write to several fragments at once, meet all banks once; two page buffers, one
// barrier a page. The next page's codes are asked for before a page's products and widened behind them.
//
// The keys' scale goes with the softmax's into the exponential's argument (whose sign goes into the queries).
// The values' goes into their widening, exactly (see `unit` below), so that the products add to the running
// sums themselves. (Scaled and added behind each page's products: 2,048 causal queries of 8 x 4 heads of 128
// behind 8,192 tokens 396 us, so 345 to 360, 860 to 900 TF/s; 2,000 of 4 x 4 heads of 64 behind 8,000 140 and 129,
// 118 with the join now; of 256 510 and 580 TF/s.)
//
// What bounds it is issue: at head width 64 a page of 32 rows takes a SIMD 1,560 cycles, of which products 512
// and 32 exponentials, their arguments, maxima, sums and conversions 880, only 150 of them at once -- with two
// waves a SIMD as with three or four, with a raised priority around the products, and with 64 rows a wave
// whose products and exponentials alternate.
constexpr int kWideRows = 128;

__device__ __forceinline__ f32x16 mfma_w(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma_w(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
// 16 lanes widen the keys' pieces j of 256 / D tokens and the values' four pieces of four channels: a key
// fragment's pad moves its 16-byte places by 256 / D a piece, a value fragment's by 4, and its
// second half of tokens by 4 again.
template <int D>
struct WideLds {
  static constexpr int KF = 1024 + 4096 / D, VH = 512 + 64, VF = 2 * 512 + 64;
  static constexpr int KEYS = 2 * (D / 16) * KF, BUF = KEYS + 4 * (D / 32) * VF;
};

template <typename T, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : D == 128 ? 2 : 3) void attend8_wide_kernel(Attend8Args a) {
  typedef typename Vec8<T>::V V8;
  constexpr int NJ = D / 16;               // products per key tile
  constexpr int NT = D / 32;               // channel tiles
  constexpr int RAW = D / 64;              // 16-byte pieces of a page's keys (values) a thread widens
  typedef WideLds<D> L;
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ int flags[2];                 // the last page of each buffer that holds a NaN value code
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, hh = lane >> 5;
  const int b = blockIdx.z, split = blockIdx.x % a.splits, tiles = (a.rows + kWideRows - 1) / kWideRows;
  const int tile = blockIdx.x / a.splits;
  const int h = tile / tiles, row0 = (tiles - 1 - tile % tiles) * kWideRows;   // causal: longest first
  const int wrow = row0 + 32 * wave, row = wrow + r;
  const bool real = row < a.rows;
  const int raw = a.lengths[b];
  const bool too_long = raw > (int64_t)a.width * kPage8;
  const int len = too_long || raw < 0 ? 0 : raw;
  const int64_t start = a.starts ? a.starts[b] : 0;
  const int limit = real ? key_limit(a, len, start, row) : 0;
  const int least = wrow < a.rows ? key_limit(a, len, start, wrow) : 0;                             // of the wave
  const int wmost = wrow < a.rows ? key_limit(a, len, start, min(wrow + 31, a.rows - 1)) : 0;
  const int tleast = key_limit(a, len, start, row0);                                                // of the tile
  const int most = key_limit(a, len, start, min(row0 + kWideRows, a.rows) - 1);
  const int npages = (most + kPage8 - 1) / kPage8;
  const int chunk = max((npages + a.splits - 1) / a.splits, a.chunk);
  const int p0 = a.splits > 1 ? split * chunk : 0, p1 = a.splits > 1 ? min(p0 + chunk, npages) : npages;
  if (p0 >= p1 && split > 0) return;   // the join knows that there is no such part

  const float c = soft_scale(a);
  const int c_bits = __builtin_amdgcn_readfirstlane(__float_as_int(c));
  V8 q[NJ];
  float q_sum = 0.f;
  {
    const T* qp = (const T*)a.q + b * a.qs[0] + (int64_t)(row / a.G) * a.qs[1] + (int64_t)(h * a.G + row % a.G) * a.qs[2];
#pragma unroll
    for (int j = 0; j < NJ; j++) q[j] = query8<T>(a, qp, 16 * j + 8 * hh, real, q_sum);
  }
  int far_from = 0;
  f32x16 acc[NT];
#pragma unroll
  for (int d = 0; d < NT; d++)
#pragma unroll
    for (int e = 0; e < 16; e++) acc[d][e] = 0.f;
  float m = -__builtin_inff(), l = 0.f;
  uint64_t poison[(NT + 3) / 4] = {};   // 16 bits a channel tile: sums that hold a NaN value their query sees

  const int32_t* table = a.table + b * a.tp;
  int none = 0;
  asm volatile("" : "+v"(none));
  const auto entry = [&](int p) { return table_entry(table, min(p, p1 - 1)); };
  const auto place = [&](int page) { return (int64_t)((unsigned)page >= (unsigned)a.pages ? 0 : page) * a.H + h; };

  i32x4 kraw[RAW], vraw[RAW];
  int ks, vs;
  // A thread's pieces of a page: keys in rows of D bytes, values in rows of 64.
  const auto load = [&](int64_t at) {
    ks = scale_entry(a.ks, at, none);
    vs = scale_entry(a.vs, at, none);
    const i32x4* kp = reinterpret_cast<const i32x4*>(a.k + at * (kPage8 * D));
    const i32x4* vp = reinterpret_cast<const i32x4*>(a.v + at * (kPage8 * D));
#pragma unroll
    for (int i = 0; i < RAW; i++) {
      kraw[i] = kp[tid + 256 * i];
      vraw[i] = vp[tid + 256 * i];
    }
  };
  // Values are widened times 2^(scale - unit), exact in fp16 (codes are 2^-9 .. 448) where that is 2^-15 .. 2^7,
  // and summed in that unit, at first the first page's scale. A page further off makes its scale the unit,
  // but never one more than 2^63 below the largest so far: the sums (2^15 times 448 x 2^7 and up to 2^30 tokens)
  // would pass fp32.
  int unit = 0, top = 0;   // of the page widened last; the largest
  const auto unit_for = [&](int byte) {
    if (byte == 255 || (byte - unit >= -15 && byte - unit <= 7)) return;   // 255: its queries get NaN
    unit = max(max(byte, top - 63), 1);
    top = max(top, unit);
  };
  // What a page's values are widened by (1 for a scale of NaN: queries that do not see the page must not get
  // zero times infinity).
  const auto widen_by = [&](int byte) { return byte == 255 ? 1.f : scale_of(max(127 + byte - unit, 1)); };
  const auto times = [&](float f) {
#pragma unroll
    for (int d = 0; d < NT; d++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[d][e] *= f;
  };
  // Widen page p's pieces into buffer p & 1, the values times vf.
  const auto widen = [&](int p, float vf) {
    uint8_t* kb = lds + (p & 1) * L::BUF;
    uint8_t* vb = kb + L::KEYS;
    const bool cut = p * kPage8 + kPage8 > tleast;
#pragma unroll
    for (int i = 0; i < RAW; i++) {
      const int e = tid + 256 * i, key = e / (D / 16), j = e % (D / 16);
      const int t = key & 31, at = 8 * (t >> 2 & 3) + 4 * (t >> 4) + (t & 3);   // the token's row of its tile
      V8 w;
      uint8_t* f = kb + ((key >> 5) * NJ + j) * L::KF + at * 16;
      codes_as(kraw[i][0], kraw[i][1], 1.f, w);
      *reinterpret_cast<V8*>(f) = w;
      codes_as(kraw[i][2], kraw[i][3], 1.f, w);
      *reinterpret_cast<V8*>(f + 512) = w;
    }
#pragma unroll
    for (int i = 0; i < RAW; i++) {
      const int e = tid + 256 * i, d = e >> 2, part = e & 3;   // channel; 16 tokens from 16 part on
      if (cut) {   // tokens behind the sequence and NaN codes as zero; see the streaming kernel
        const int left = len - p * kPage8 - 16 * part;
        unsigned nan = 0;
#pragma unroll
        for (int x = 0; x < 4; x++) {
          const int n = left - 4 * x;
          int w = vraw[i][x] & (n >= 4 ? -1 : n <= 0 ? 0 : (int)(0xffffffffu >> (32 - 8 * n)));
          const unsigned nb = nan_bytes(w);
          nan |= nb;
          vraw[i][x] = w & ~(int)((nb >> 7) * 255u);
        }
        if (nan) flags[p & 1] = p;
      }
      f16x8 w;
      uint8_t* f = vb + ((d >> 5) * 4 + (part >> 1) * 2) * L::VF + (part & 1) * L::VH + (d & 31) * 16;
      codes_as(vraw[i][0], vraw[i][1], vf, w);
      *reinterpret_cast<f16x8*>(f) = w;
      codes_as(vraw[i][2], vraw[i][3], vf, w);
      *reinterpret_cast<f16x8*>(f + L::VF) = w;
    }
  };

  int sums = 0;   // the unit of the lane's sums: a page that its query does not see leaves them alone
  const auto attend = [&](int p, bool missing, int ksb, int punit, bool moved) {
    const uint8_t* kb = lds + (p & 1) * L::BUF + lane * 16;
    const uint8_t* vb = lds + (p & 1) * L::BUF + L::KEYS + hh * L::VH + r * 16;
    f32x16 sv[2];
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) sv[t][e] = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; j++) {
#pragma unroll
      for (int t = 0; t < 2; t++) sv[t] = mfma_w(*reinterpret_cast<const V8*>(kb + (t * NJ + j) * L::KF), q[j], sv[t]);
      if (j % 2) __builtin_amdgcn_sched_barrier(0);   // bounds the operands read ahead
    }
    float s[2][16];
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) s[t][e] = sv[t][e];
    const int base = p * kPage8 + 16 * hh;   // score e of tile t is token base + 32 t + e
    if (missing && p * kPage8 < limit) l = __builtin_nanf("");   // (page 0 was read in a missing one's place)
    const bool far = ksb >= far_from;
    const float scale = score_scale(c_bits, ksb), kc = far ? 1.f : scale;
    if (p * kPage8 + kPage8 > least || far) {
      int left = limit - base;
      pin_value(left);
      const float first = far ? scale : 1.f;
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) s[t][e] = 32 * t + e < left ? s[t][e] * first : -__builtin_inff();
    }
    float mx = max3_f(s[0][0], s[1][0], s[0][1]);
    mx = max3_f(mx, s[1][1], s[1][1]);
#pragma unroll
    for (int e = 2; e < 16; e++) mx = max3_f(mx, s[0][e], s[1][e]);
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_int(mx), __float_as_int(mx), false, false);
    const float mn = max3_f(m, __builtin_fmaf(__int_as_float(x[0]), kc, -kRaise),
                            __builtin_fmaf(__int_as_float(x[1]), kc, -kRaise));
    float ref = m == -__builtin_inff() ? 0.f : m;
    if (moved || __any(mn - m > (far ? 0.f : kSlack))) {
      ref = mn == -__builtin_inff() ? 0.f : mn;
      float alpha = __builtin_amdgcn_exp2f(m - ref);
      l *= alpha;
      if (p * kPage8 < limit) {
        alpha *= scale_of(max(127 + sums - punit, 0));
        sums = punit;
      }
      times(alpha);
      m = mn;
    }
    f16x8 pr[2][2];
    float lp = 0.f;
    // Eight at a time: left alone, all 32 probabilities stay in fp32 until the products below.
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int u = 0; u < 2; u++) {
#pragma unroll
        for (int e = 0; e < 8; e++) pr[t][u][e] = (f16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[t][8 * u + e], kc, -ref));
        lp = sum8(pr[t][u], lp);
        pin_value(lp);
        __builtin_amdgcn_sched_barrier(0);
      }
    l += lp;
#pragma unroll
    for (int d = 0; d < NT; d++) {
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int u = 0; u < 2; u++)
          acc[d] = mfma_w(*reinterpret_cast<const f16x8*>(vb + (d * 4 + t * 2 + u) * L::VF), pr[t][u], acc[d]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Which sums a page's NaN values belong in: their places times 1 for each token that a query sees.
  const auto mark = [&](int p, int64_t at) {
    const uint8_t* vp = a.v + at * (kPage8 * D) + r * kPage8 + 16 * hh;
#pragma unroll 1
    for (int d = 0; d < NT; d++) {
      f32x16 marks;
#pragma unroll
      for (int e = 0; e < 16; e++) marks[e] = 0.f;
#pragma unroll 1
      for (int tu = 0; tu < 4; tu++) {
        const i32x2 w = *reinterpret_cast<const i32x2*>(vp + d * 32 * kPage8 + 32 * (tu / 2) + 8 * (tu % 2));
        const int base = p * kPage8 + 16 * hh + 32 * (tu / 2) + 8 * (tu % 2);
        f16x8 mk, seen;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          mk[e] = base + e < len && ((nan_bytes(w[e / 4]) >> (8 * (e % 4))) & 0x80) ? (f16)1.f : (f16)0.f;
          seen[e] = base + e < limit ? (f16)1.f : (f16)0.f;
        }
        marks = mfma_w(mk, seen, marks);
      }
#pragma unroll
      for (int e = 0; e < 16; e++)
        if (marks[e] > 0.f) poison[d / 4] |= 1ull << (16 * (d % 4) + e);
    }
  };

  if (tid < 2) flags[tid] = -1;
  __syncthreads();
  if (p0 < p1) {
    int page = entry(p0), next = entry(p0 + 1);
    int64_t at = place(page);
    load(at);
    far_from = far_byte(q_sum, 2, c);
    const int first = __builtin_amdgcn_readfirstlane(vs);
    unit = top = max(first == 255 ? 127 : first, 1);
    sums = unit;
    widen(p0, widen_by(first));
    int was = unit;
    for (int p = p0; p < p1; p++) {
      const int ksb = __builtin_amdgcn_readfirstlane(ks), vsb = __builtin_amdgcn_readfirstlane(vs), punit = unit;
      const int64_t nat = place(next);
      const int after = entry(p + 2);
      if (p + 1 < p1) load(nat);
      // Page p stands in its buffer, and every wave is done with the other one. (__syncthreads would wait
      // for the codes asked for above.)
      ring_barrier();
      if (p * kPage8 < wmost) {
        attend(p, (unsigned)page >= (unsigned)a.pages || ksb == 255 || vsb == 255, ksb, punit, punit != was);
        if (p * kPage8 + kPage8 > tleast && flags[p & 1] == p) mark(p, at);
      }
      if (p + 1 < p1) {
        const int nvs = __builtin_amdgcn_readfirstlane(vs);
        unit_for(nvs);
        widen(p + 1, widen_by(nvs));
      }
      was = punit;
      page = next;
      next = after;
      at = nat;
    }
  }

#pragma unroll
  for (int d = 0; d < NT; d++)
    if (poison[d / 4])
#pragma unroll
      for (int e = 0; e < 16; e++)
        if (poison[d / 4] >> (16 * (d % 4) + e) & 1) acc[d][e] = __builtin_nanf("");
  times(scale_of(sums) * kLower);
  const auto l32 = __builtin_amdgcn_permlane32_swap(__float_as_int(l), __float_as_int(l), false, false);
  l = (__int_as_float(l32[0]) + __int_as_float(l32[1])) * kLower;
  if (too_long) l = __builtin_nanf("");
  if (!real) return;
  if (a.splits > 1) {
    const int64_t bh = (int64_t)b * a.H + h, place8 = (bh * a.rows + row) * a.splits + split;
    const int64_t all = (int64_t)gridDim.z * a.H * a.rows * a.splits;
#pragma unroll
    for (int d = 0; d < NT; d++)
#pragma unroll
      for (int g = 0; g < 4; g++)
        *reinterpret_cast<f32x4*>(a.part + place8 * D + 32 * d + 8 * g + 4 * hh) =
            (f32x4){acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
    if (hh == 0) {
      a.part[all * D + 2 * place8] = m == -__builtin_inff() ? 0.f : m;
      a.part[all * D + 2 * place8 + 1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* op = (T*)a.o + b * a.os[0] + (int64_t)(row / a.G) * a.os[1] + (int64_t)(h * a.G + row % a.G) * a.os[2];
#pragma unroll
  for (int d = 0; d < NT; d++)
#pragma unroll
    for (int g = 0; g < 2; g++) {   // halves exchanged between a row's two lanes: eight channels each
      float f[8];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const auto x = __builtin_amdgcn_permlane32_swap(__float_as_int(acc[d][8 * g + e]),
                                                        __float_as_int(acc[d][8 * g + 4 + e]), false, false);
        f[e] = __int_as_float(x[0]) * inv;
        f[4 + e] = __int_as_float(x[1]) * inv;
      }
      store8(op + 32 * d + 16 * g + 8 * hh, f);
    }
}

template <typename T, int D>
int launch_wide(const Attend8Args& a, dim3 grid, hipStream_t st) {
  constexpr int LDS = 2 * WideLds<D>::BUF;
  const auto kern = attend8_wide_kernel<T, D>;
  if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess)
    return check_launch("cache8_attention: set LDS size");
  hipLaunchKernelGGL(kern, grid, dim3(256), LDS, st, a);
  return LDX_OK;
}

// Parts that a sequence of npages has (of a.splits possible ones), at least one.
__device__ __forceinline__ int part_count(const Attend8Args& a, int npages) {
  const int chunk = max((npages + a.splits - 1) / a.splits, a.chunk);
  return max((npages + chunk - 1) / chunk, 1);
}

// The output of four channels of a row.
template <typename T>
__device__ __forceinline__ void put4(const Attend8Args& a, int b, int h, int row, int channel, f32x4 o, float l) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* op = (T*)a.o + b * a.os[0] + (int64_t)(row / a.G) * a.os[1] + (int64_t)(h * a.G + row % a.G) * a.os[2] + channel;
#pragma unroll
  for (int i = 0; i < 4; i++) op[i] = (T)(o[i] * inv);
}

// Parts that a row's sequence was given.
__device__ __forceinline__ int parts_of(const Attend8Args& a, int b, int row) {
  const int raw = a.lengths[b];
  const int len = raw < 0 || raw > (int64_t)a.width * kPage8 ? 0 : raw;
  // The last row of a workgroup's tile says how many pages it reads.
  const int most = key_limit(a, len, a.starts ? a.starts[b] : 0, min((row / a.tile + 1) * a.tile, a.rows) - 1);
  return part_count(a, (most + kPage8 - 1) / kPage8);
}

// Joins the parts of rows, few parts (at most kFewParts): a thread takes four channels of a row.
constexpr int kFewParts = 8;

template <typename T, int D>
__global__ __launch_bounds__(256) void attend8_join_kernel(Attend8Args a, int64_t total) {
  constexpr int PER = D / 4;
  const int64_t at = (int64_t)blockIdx.x * (256 / PER) + threadIdx.x / PER, bh = at / a.rows;
  if (at >= total) return;
  const int b = (int)(bh / a.H), h = (int)(bh % a.H), row = (int)(at % a.rows), c = threadIdx.x % PER;
  const int parts = parts_of(a, b, row);
  const f32x2* ml = reinterpret_cast<const f32x2*>(a.part + total * a.splits * D) + at * a.splits;
  float mt = -__builtin_inff();
  for (int s = 0; s < parts; s++)
    if (ml[s][1] != 0.f) mt = fmaxf(mt, ml[s][0]);   // a part without a token that the row sees has sum 0
  float lt = 0.f;
  f32x4 ot = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < parts; s++) {
    const float f = ml[s][1] != 0.f ? __builtin_amdgcn_exp2f(ml[s][0] - mt) : 0.f;
    lt += ml[s][1] * f;
    ot += *reinterpret_cast<const f32x4*>(a.part + (at * a.splits + s) * D + 4 * c) * f;
  }
  put4<T>(a, b, h, row, 4 * c, ot, lt);
}

// Joins the parts of a row, a workgroup each: the parts' weights side by side, then a thread takes four
// channels of every (1024 / D)-th part and the threads of a channel are joined through LDS.
constexpr int kMostParts = 1024;

template <typename T, int D>
__global__ __launch_bounds__(256) void attend8_merge_kernel(Attend8Args a) {
  constexpr int PER = D / 4, LANES = 256 / PER;
  __shared__ float weight[kMostParts];
  __shared__ f32x4 so[LANES][PER];
  __shared__ float red[8];
  const int64_t total = gridDim.x, at = blockIdx.x, bh = at / a.rows;
  const int b = (int)(bh / a.H), h = (int)(bh % a.H), row = (int)(at % a.rows), tid = threadIdx.x;
  const int parts = parts_of(a, b, row);
  const f32x2* ml = reinterpret_cast<const f32x2*>(a.part + total * a.splits * D) + at * a.splits;
  float mt = -__builtin_inff();
  for (int s = tid; s < parts; s += 256) {
    const f32x2 e = ml[s];
    if (e[1] != 0.f) mt = fmaxf(mt, e[0]);   // a part without a token that the row sees has sum 0
  }
  mt = wave_max(mt);
  if ((tid & 63) == 0) red[tid >> 6] = mt;
  __syncthreads();
  mt = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  float lt = 0.f;
  for (int s = tid; s < parts; s += 256) {
    const f32x2 e = ml[s];
    const float f = e[1] != 0.f ? __builtin_amdgcn_exp2f(e[0] - mt) : 0.f;
    weight[s] = f;
    lt += e[1] * f;
  }
  lt = wave_sum(lt);
  if ((tid & 63) == 0) red[4 + (tid >> 6)] = lt;
  __syncthreads();
  lt = red[4] + red[5] + red[6] + red[7];
  const int c = tid % PER, lane = tid / PER;
  f32x4 ot = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = lane; s < parts; s += LANES)
    ot += *reinterpret_cast<const f32x4*>(a.part + (at * a.splits + s) * D + 4 * c) * weight[s];
  so[lane][c] = ot;
  __syncthreads();
  if (lane) return;
#pragma unroll
  for (int s = 1; s < LANES; s++) ot += so[s][c];
  put4<T>(a, b, h, row, 4 * c, ot, lt);
}

template <typename T, int D>
int launch_d(const Attend8Args& a, int batch, hipStream_t st) {
  const dim3 grid((unsigned)a.splits * (unsigned)(a.H * ((a.rows + a.tile - 1) / a.tile)), 1, (unsigned)batch);
  if (a.tile == 16) {
    hipLaunchKernelGGL((attend8_kernel<T, D>), grid, dim3(64 * kAttendWaves), 0, st, a);
  } else if constexpr (D >= 64) {
    if (int rc = launch_wide<T, D>(a, grid, st)) return rc;
  }
  const int64_t total = (int64_t)batch * a.H * a.rows;
  constexpr int ROWS = 1024 / D;   // of a workgroup
  if (a.splits > kFewParts)
    hipLaunchKernelGGL((attend8_merge_kernel<T, D>), dim3((unsigned)total), dim3(256), 0, st, a);
  else if (a.splits > 1)
    hipLaunchKernelGGL((attend8_join_kernel<T, D>), dim3((unsigned)((total + ROWS - 1) / ROWS)), dim3(256), 0, st, a, total);
  return check_launch("cache8_attention");
}

template <typename T>
int launch_t(const Attend8Args& a, int D, int batch, hipStream_t st) {
  if (D == 32) return launch_d<T, 32>(a, batch, st);
  if (D == 64) return launch_d<T, 64>(a, batch, st);
  if (D == 128) return launch_d<T, 128>(a, batch, st);
  return launch_d<T, 256>(a, batch, st);
}

int check_cache(const char* what, const ldx_cache8& c) {
  if (!c.k || !c.v || !c.k_scales || !c.v_scales) return fail("%s: null pointer", what);
  if (c.pages < 1 || c.heads < 1 || c.heads > 8192) return fail("%s: %d pages, %d heads", what, c.pages, c.heads);
  if (c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)
    return fail("%s: head_dim %d is not 32, 64, 128 or 256", what, c.head_dim);
  if ((uintptr_t)c.k % 16 || (uintptr_t)c.v % 16) return fail("%s: codes not aligned", what);
  return LDX_OK;
}

// How a call is laid out. The host knows only how many pages a table's row holds; the kernels divide the
// pages that a sequence has.
struct Plan {
  bool wide;    // pages shared through LDS by 128 rows of a cache head, or streamed by 16
  int splits;   // parts that a sequence's pages may be spread over
};

constexpr int kLeastChunk = 8;   // pages of a part at least: two for each streaming wave. (8 and 16: 4 sequences
                                 // of 8,000 tokens 20 and 22 us, 8 of 5,000 at head width 256 22 and 28)

size_t split_bytes(const ldx_cache8_attention_args* p, int splits) {
  if (splits < 2) return 0;
  const size_t rows = (size_t)p->q_len * (p->q_heads / p->cache.heads);
  return (size_t)p->batch * p->cache.heads * rows * splits * (p->cache.head_dim + 2) * sizeof(float);
}

// What partial results may take at most. (It bounds the join's launch, too.)
constexpr size_t kMostPartBytes = (size_t)256 << 20;

Plan plan_of(const ldx_cache8_attention_args* p) {
  const int D = p->cache.head_dim;
  const int64_t heads = (int64_t)p->batch * p->cache.heads, rows = (int64_t)p->q_len * (p->q_heads / p->cache.heads);
  const int64_t most = (p->width + kLeastChunk - 1) / kLeastChunk;
  Plan plan;
  // A page of 16 rows costs a streaming wave about 0.6 / 1.5 / 3.0 us at head width 64 / 128 / 256 (0.38 at 32,
  // and as much shared, so that is not done), shared 0.5 / 0.9 / 2.3, and sharing 10 to 20 us more at the start and end. From these sums
  // of pages on it was ahead (4,096 queries of 4 heads behind 8,192 tokens 103 -> 84 / 262 -> 139 us at 64 /
  // 128, 512 queries of 16 heads 200 -> 151 at 256; below, 4,096 queries behind 256 tokens 35 and 41 at 64).
  const int64_t work = heads * ((rows + 15) / 16) * p->width;
  plan.wide = rows >= kWideRows && work >= (D == 32 ? INT64_MAX : D == 64 ? 100000 : D == 128 ? 18000 : 9000);
  int64_t s = 1;
  if (plan.wide) {
    // Rounds of workgroups on the CUs' places, the pages of a round, and what a part more costs: 3 pages of a round
    // to join, or what it writes and the join reads, at 4.5 TB/s and 2.2 us a page of a round. (With 3 pages for any
    // number of rows calls that fill the card anyway were split: of 40 random ones 35 are faster so, 0.85 of the time
    // on average, 16 x 1,769 queries of 12 x 8 heads of 128 4,039 -> 2,431 us without 4.2 GB; four are 4 to 9 % slower.)
    const int64_t groups = heads * ((rows + kWideRows - 1) / kWideRows), places = D == 64 ? 768 : D == 128 ? 512 : 256;
    const double traffic = 8e-7 * (double)(heads * rows) * (D + 2), part = traffic > 3.0 ? traffic : 3.0;
    double best = 1e30;
    for (int64_t i = 1; i <= kFewParts && i <= most; i++) {
      if (split_bytes(p, (int)i) > kMostPartBytes) break;
      const double cost = (double)((groups * i + places - 1) / places) * ((p->width + i - 1) / i) + part * i;
      if (cost < best) best = cost, s = i;
    }
  } else {
    // Two workgroups a CU (256 to 1,024 parts in all were within a tenth for most calls, more slower).
    s = 512 / (heads * ((rows + 15) / 16));
    if (s > most) s = most;
    // Parts cost a second launch to join, 3 us on the device and 4 on the host. A whole sequence's pages take a
    // workgroup 0.17 / 0.2 / 0.4 / 0.8 us each at head width 32 / 64 / 128 / 256: up to these many it is ahead or
    // near it (one token behind 1,500 at 64 10.0 us in parts, 9.5 whole, behind 2,000 10.5 and 10.9, 3,000 11.2
    // and 13.7; called one by one 19.4 and 15.4; behind 1,000 at 128 12.1 and 11.5, 2,000 13.0 and 17.0).
    if (p->width <= (D <= 64 ? 32 : D == 128 ? 20 : 10)) s = 1;
  }
  plan.splits = (int)(s < 1 ? 1 : s > kMostParts ? kMostParts : s);
  return plan;
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
  if (rows * p->cache.heads * p->batch > 0x7fffffff || (rows + 15) / 16 * p->cache.heads > 1 << 23)   // 2^31 threads
    return fail("cache8_attention: %d x %d queries of %d heads are more than one launch takes", p->batch, p->q_len,
                p->q_heads);
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
  if (p->batch < 1 || p->batch > 65535 || p->tokens < 1 || p->tokens > 1 << 28 || p->width < 1 || p->width > (1 << 24))
    return fail("cache8_append: batch %d, %d tokens, %d pages a sequence", p->batch, p->tokens, p->width);
  if (p->table_pitch < p->width) return fail("cache8_append: table pitch below %d", p->width);
  AppendArgs a = {{(uint8_t*)p->cache.k, (uint8_t*)p->cache.v},
                  {(uint8_t*)p->cache.k_scales, (uint8_t*)p->cache.v_scales},
                  {p->k, p->v},
                  {{p->k_stride[0], p->k_stride[1], p->k_stride[2]}, {p->v_stride[0], p->v_stride[1], p->v_stride[2]}},
                  p->cache.pages, p->cache.heads, p->tokens,
                  p->table, p->table_pitch, p->width, p->starts, p->counts};
  const unsigned slots = (unsigned)((p->tokens + 2 * (int64_t)kPage8 - 2) / kPage8);
  const dim3 grid(slots, 2 * (unsigned)p->cache.heads, (unsigned)p->batch);
  hipStream_t st = as_stream(stream);
  if (p->dtype == LDX_DTYPE_F16) launch_append<f16>(a, p->cache.head_dim, grid, st);
  else if (p->dtype == LDX_DTYPE_BF16) launch_append<bf16>(a, p->cache.head_dim, grid, st);
  else launch_append<float>(a, p->cache.head_dim, grid, st);
  return check_launch("cache8_append");
}

extern "C" size_t ldx_cache8_attention_workspace_bytes(const ldx_cache8_attention_args* p) {
  return check_attention(p) == LDX_OK ? split_bytes(p, plan_of(p).splits) : 0;
}

extern "C" int ldx_cache8_attention_rows(const ldx_cache8_attention_args* p) {
  if (int rc = check_attention(p)) return rc;
  return plan_of(p).wide ? kWideRows : 16;
}

extern "C" int ldx_cache8_attention(const ldx_cache8_attention_args* p, void* stream) {
  if (int rc = check_attention(p)) return rc;
  Plan plan = plan_of(p);
  if (plan.splits > 1 && (!p->workspace || p->workspace_bytes < split_bytes(p, plan.splits))) plan.splits = 1;
  if (plan.splits > 1 && (uintptr_t)p->workspace % 16) return fail("cache8_attention: workspace not aligned");
  const int G = p->q_heads / p->cache.heads;
  const Attend8Args a = {(const uint8_t*)p->cache.k, (const uint8_t*)p->cache.v, (const uint8_t*)p->cache.k_scales,
                         (const uint8_t*)p->cache.v_scales, p->cache.pages, p->cache.heads,
                         p->q, {p->q_stride[0], p->q_stride[1], p->q_stride[2]},
                         p->o, {p->o_stride[0], p->o_stride[1], p->o_stride[2]},
                         G, p->q_len, G * p->q_len, p->scale * 1.4426950408889634f,
                         p->table, p->table_pitch, p->width, p->lengths, p->starts, plan.splits, kLeastChunk,
                         plan.wide ? kWideRows : 16, (float*)p->workspace};
  hipStream_t st = as_stream(stream);
  return p->dtype == LDX_DTYPE_F16 ? launch_t<f16>(a, p->cache.head_dim, p->batch, st)
                                   : launch_t<bf16>(a, p->cache.head_dim, p->batch, st);
}
