// Norms of queries and keys for each head with the position rotation in the same pass.
//
//   f = x / sqrt(mean(x^2) + eps) * gamma       (over a head's channels; x itself without gamma)
//   for every pair (a, b) of channels of axis A:  t = position_A * turns,  (a cos 2 pi t - b sin 2 pi t,
//                                                                        b cos 2 pi t + a sin 2 pi t)
//
// Positions have one axis (text) or several (a volume's depth, height and width); an axis turns a section of the
// head's channels, whose pairs are its two halves' or neighbours. Channels behind the sections stay as they are.
//
// One pass. A workgroup takes the query or the key heads of a few tokens: its threads first make the tokens' cosines and
// sines, which the heads share, then a lane takes a part of a head, and the lanes of a head add their squares. Where pairs
// are neighbours, or the halves of all sections whole fours, a lane holds both ends of its pairs; else it takes channels
// as they lie, so that every access to memory is of whole lines, and gets the other ends through LDS.
//
// Bound by memory: 51,200 tokens of 16 query and 16 key heads of 32 in fp16, three axes, 45 us, 4.7 TB/s; 16,384 of 32 and 8
// heads of 128 in bf16 64, 5.3, in fp32 141, 4.8, with neighbours 64 and 131. Few heads are bound by the launch (a token's 3.3
// us). Queries and keys in the same workgroups, without the next head asked for ahead, took 104 and 78.
#include "quant8.h"

namespace ldx {
namespace {

constexpr int kAxes = LDX_ROTARY_AXES;
constexpr int kMostPairs = 1024;   // of the tokens of a workgroup
constexpr int kMostPlaces = 64;    // tokens of a workgroup

struct RotateArgs {
  const void* x[2]; int64_t xs[2][3];   // queries and keys: batch, token, head strides
  void* y[2]; int64_t ys[2][3];
  const float* gamma[2];
  int heads[2];
  int group[2];                   // tokens of a workgroup
  unsigned blocks;                // workgroups of the queries; the keys' follow
  float eps, per;                 // per: 1 / channels
  const int32_t* positions; int64_t ps[3];   // axis, batch, token strides
  const double* turns;
  int section[kAxes + 1];         // first pair of each axis and of the channels that stay
  int axes, pairs;                // pairs of a head
  int64_t places;                 // batch * tokens
  int L;                          // tokens of a sequence
  int lanes;                      // of a head, a power of two
  UDiv by_L, by_pairs, by_heads[2];
};

// cos and sin of t turns, |t| at most half a turn: the nearest quarter turn is taken off (exactly), the rest, at most
// pi / 4, goes into the Taylor sums, cut off below 2^-28 of the result's size.
__device__ __forceinline__ void turn(double t, float& cos, float& sin) {
  const double n = __builtin_rint(4.0 * t);
  const float x = (float)((t - 0.25 * n) * 6.283185307179586), z = x * x;
  float s = 2.7557319e-6f;   // 1 / 9!
  s = __builtin_fmaf(s, z, -1.9841270e-4f);
  s = __builtin_fmaf(s, z, 8.3333333e-3f);
  s = __builtin_fmaf(s, z, -1.6666667e-1f);
  s = __builtin_fmaf(s * z, x, x);
  float c = -2.7557319e-7f;   // 1 / 10!
  c = __builtin_fmaf(c, z, 2.4801587e-5f);
  c = __builtin_fmaf(c, z, -1.3888889e-3f);
  c = __builtin_fmaf(c, z, 4.1666667e-2f);
  c = __builtin_fmaf(c, z, -0.5f);
  c = __builtin_fmaf(c, z, 1.f);
  const int q = (int)n & 3;
  const float a = q & 1 ? s : c, b = q & 1 ? c : s;
  cos = q == 1 || q == 2 ? -a : a;
  sin = q >= 2 ? -b : b;
}

// Sum over the lanes (a power of two) that hold a head.
__device__ __forceinline__ float head_sum(float v, int lanes) {
  if (lanes > 1) v += dpp_f<0xB1>(v);    // quad_perm 1 0 3 2
  if (lanes > 2) v += dpp_f<0x4E>(v);    // quad_perm 2 3 0 1
  if (lanes > 4) v += dpp_f<0x141>(v);   // row_half_mirror
  if (lanes > 8) v += dpp_f<0x140>(v);   // row_mirror
  if (lanes > 16) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    v = __int_as_float(a[0]) + __int_as_float(a[1]);
  }
  if (lanes > 32) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    v = __int_as_float(a[0]) + __int_as_float(a[1]);
  }
  return v;
}

template <typename T, int N>
struct Run {
  T v[N];
  // To memory of any alignment, past the caches' retention.
  __device__ __forceinline__ void stream(T* p) const {
    if constexpr (N == 1) {
      __builtin_nontemporal_store(v[0], p);
    } else {
      typedef T V __attribute__((ext_vector_type(N)));
      typedef V Unaligned __attribute__((aligned(sizeof(T))));
      V w;
#pragma unroll
      for (int i = 0; i < N; i++) w[i] = v[i];
      __builtin_nontemporal_store(w, reinterpret_cast<Unaligned*>(p));
    }
  }
};
template <int N>
__device__ __forceinline__ void table_n(const float* p, float (&f)[N]) {
  Run<float, N> u;
  __builtin_memcpy(&u, __builtin_assume_aligned(p, N < 4 ? 4 * N : 16), sizeof(u));
#pragma unroll
  for (int i = 0; i < N; i++) f[i] = u.v[i];
}

// The two ends of V pairs as they lie in memory: runs of V, or neighbours.
template <typename T, int V, bool NEAR>
struct Ends {
  Run<T, V> a, b;
  __device__ __forceinline__ void load(const T* p, int at, int to) {
    if constexpr (NEAR) {
      Run<T, 2 * V> w;
      __builtin_memcpy(&w, p + at, sizeof(w));
#pragma unroll
      for (int v = 0; v < V; v++) a.v[v] = w.v[2 * v], b.v[v] = w.v[2 * v + 1];
    } else {
      __builtin_memcpy(&a, p + at, sizeof(a));
      __builtin_memcpy(&b, p + to, sizeof(b));
    }
  }
  __device__ __forceinline__ void store(T* p, int at, int to) const {
    if constexpr (NEAR) {
      Run<T, 2 * V> w;
#pragma unroll
      for (int v = 0; v < V; v++) w.v[2 * v] = a.v[v], w.v[2 * v + 1] = b.v[v];
      w.stream(p + at);
    } else {
      a.stream(p + at);
      b.stream(p + to);
    }
  }
};

// In a cosine's place for channels behind the sections. They are passed through: 0 times an infinity or a NaN of the channel
// that is paired with them is not 0, and zeros keep their sign.
constexpr float kStay = 2.f;

// What a workgroup is to do: a part of the tokens, all heads of the queries or of the keys.
struct Part {
  int which, heads, count;
  int64_t first;
  __device__ __forceinline__ Part(const RotateArgs& a) {
    which = blockIdx.x >= a.blocks ? 1 : 0;
    heads = a.heads[which];
    first = (int64_t)(blockIdx.x - (which ? a.blocks : 0)) * a.group[which];
    count = (int)min((int64_t)a.group[which], a.places - first);
  }
};

// Where the tokens' heads begin, of x and y, and put(token, pair, cos, sin) for each pair of each token.
template <typename F>
__device__ __forceinline__ void prepare(const RotateArgs& a, const Part& w, int64_t (&base)[2][kMostPlaces], F put) {
  for (int n = threadIdx.x; n < w.count; n += 256) {
    const int b = udiv((int)(w.first + n), a.by_L), l = (int)(w.first + n) - b * a.L;
    base[0][n] = b * a.xs[w.which][0] + l * a.xs[w.which][1];
    base[1][n] = b * a.ys[w.which][0] + l * a.ys[w.which][1];
  }
  for (int e = threadIdx.x; e < w.count * a.pairs; e += 256) {
    const int n = udiv(e, a.by_pairs), pair = e - n * a.pairs;
    const int b = udiv((int)(w.first + n), a.by_L), l = (int)(w.first + n) - b * a.L;
    float c = kStay, s = 0.f;
    if (pair < a.section[a.axes]) {
      int axis = 0;
#pragma unroll
      for (int i = 1; i < kAxes; i++) axis += i < a.axes && pair >= a.section[i] ? 1 : 0;
      const double t = (double)a.positions[axis * a.ps[0] + b * a.ps[1] + l * a.ps[2]] * a.turns[pair];
      turn(t - __builtin_rint(t), c, s);
    }
    put(n, pair, c, s);
  }
}

// The section that a pair is in: its first pair and its number of pairs.
__device__ __forceinline__ void section_of(const RotateArgs& a, int pair, int& low, int& size) {
  low = 0, size = a.section[1];
#pragma unroll
  for (int x = 1; x <= kAxes; x++)
    if (x <= a.axes && pair >= a.section[x]) {
      low = a.section[x];
      size = (x < a.axes ? a.section[x < kAxes ? x + 1 : x] : a.pairs) - low;
    }
}

// 1 / sqrt(mean(x^2) + eps) of a head whose N values a lane's f are a part of; it goes to the values before gamma does, since
// it may leave fp32 with gamma alone. Where the mean with eps passes fp32, values are squared at 2^-70 of themselves (512
// squares of fp32's largest number make 2^125; values, or the root of eps, are 2^59 or more, so what is lost below does not
// count), and the values, which the root goes to, are made 2^-16 of themselves, so that the root stays a normal number: it is
// at least 2^-128 of fp32's largest value, 2^-112 then.
template <int N>
__device__ __forceinline__ float root_of(const RotateArgs& a, float (&f)[N]) {
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; i++) sum = __builtin_fmaf(f[i], f[i], sum);
  const float mean = __builtin_fmaf(head_sum(sum, a.lanes), a.per, a.eps);
  if (mean < __builtin_inff()) return __builtin_amdgcn_rsqf(mean);
  sum = 0.f;   // (or NaN)
#pragma unroll
  for (int i = 0; i < N; i++) {
    const float x = f[i] * 0x1p-70f;
    sum = __builtin_fmaf(x, x, sum);
    f[i] *= 0x1p-16f;
  }
  return __builtin_amdgcn_rsqf(__builtin_fmaf(head_sum(sum, a.lanes), a.per, a.eps * 0x1p-70f * 0x1p-70f)) * 0x1p-54f;
}

// Pairs that lie well: lane u of a head takes pairs (u + i * lanes) V .., i < NU; neighbours (NEAR) or halves of a section.
template <typename T, int V, int NU, bool NEAR>
__global__ __launch_bounds__(256) void rotate_kernel(RotateArgs a) {
  __shared__ __align__(16) float table[2][kMostPairs];   // cosines, sines
  __shared__ int64_t base[2][kMostPlaces];
  const int tid = threadIdx.x, u = tid & (a.lanes - 1), step = 256 / a.lanes;
  const Part w(a);
  int at[NU], to[NU];   // a unit's channels: first ends from `at` on, second ends from `to` on
  bool in[NU];
#pragma unroll
  for (int i = 0; i < NU; i++) {
    const int pair = (u + i * a.lanes) * V;
    int low, size;
    section_of(a, pair, low, size);
    in[i] = pair < a.pairs;
    at[i] = !in[i] ? 0 : NEAR ? 2 * pair : low + pair;   // (a lane without pairs reads the head's first ones, and writes nothing)
    to[i] = !in[i] ? 0 : at[i] + size;
  }
  prepare(a, w, base, [&](int n, int pair, float c, float s) {
    table[0][n * a.pairs + pair] = c;
    table[1][n * a.pairs + pair] = s;
  });
  Ends<float, V, NEAR> gamma[NU];
  const bool norm = a.gamma[w.which] != nullptr, stay = a.section[a.axes] < a.pairs;
  if (norm)
#pragma unroll
    for (int i = 0; i < NU; i++) gamma[i].load(a.gamma[w.which], at[i], to[i]);
  __syncthreads();

  // A token's head at a time; the next one's values are asked for before this one's are worked on.
  const T* x = (const T*)a.x[w.which];
  T* y = (T*)a.y[w.which];
  const int item = tid / a.lanes, tokens = udiv(step, a.by_heads[w.which]), rest = step - tokens * w.heads;
  int n = udiv(item, a.by_heads[w.which]), h = item - n * w.heads;
  Ends<T, V, NEAR> now[NU], next[NU];
  const auto load = [&](Ends<T, V, NEAR> (&e)[NU], int n, int h) {
    const T* p = x + base[0][n] + h * a.xs[w.which][2];
#pragma unroll
    for (int i = 0; i < NU; i++) e[i].load(p, at[i], to[i]);
  };
  if (n < w.count) load(now, n, h);
  while (n < w.count) {
    int nn = n + tokens, nh = h + rest;
    if (nh >= w.heads) nn++, nh -= w.heads;
    if (nn < w.count) load(next, nn, nh);
    float f[2 * NU * V];   // a unit's first ends, then its second ones
#pragma unroll
    for (int i = 0; i < NU; i++)
#pragma unroll
      for (int v = 0; v < V; v++) {
        f[2 * i * V + v] = in[i] ? (float)now[i].a.v[v] : 0.f;
        f[(2 * i + 1) * V + v] = in[i] ? (float)now[i].b.v[v] : 0.f;
      }
    if (norm) {
      const float root = root_of(a, f);
#pragma unroll
      for (int i = 0; i < NU; i++)
#pragma unroll
        for (int v = 0; v < V; v++) {
          f[2 * i * V + v] = f[2 * i * V + v] * root * gamma[i].a.v[v];
          f[(2 * i + 1) * V + v] = f[(2 * i + 1) * V + v] * root * gamma[i].b.v[v];
        }
    }
    T* q = y + base[1][n] + h * a.ys[w.which][2];
#pragma unroll
    for (int i = 0; i < NU; i++) {
      if (!in[i]) continue;
      const int pair = n * a.pairs + (u + i * a.lanes) * V;
      float c[V], s[V];
      table_n<V>(&table[0][pair], c);
      table_n<V>(&table[1][pair], s);
      Ends<T, V, NEAR> o;
#pragma unroll
      for (int v = 0; v < V; v++) {
        const float p = f[2 * i * V + v], r = f[(2 * i + 1) * V + v];
        o.a.v[v] = (T)__builtin_fmaf(p, c[v], -(r * s[v]));
        o.b.v[v] = (T)__builtin_fmaf(r, c[v], p * s[v]);
      }
      if (__builtin_expect(stay, 0))
#pragma unroll
        for (int v = 0; v < V; v++)
          if (c[v] == kStay) o.a.v[v] = (T)f[2 * i * V + v], o.b.v[v] = (T)f[(2 * i + 1) * V + v];
      o.store(q, at[i], to[i]);
    }
#pragma unroll
    for (int i = 0; i < NU; i++) now[i] = next[i];
    n = nn;
    h = nh;
  }
}

// Halves that lie anyhow: lane u of a head takes channels (u + i * lanes) C .. as they lie in memory, and gets the other
// ends of their pairs from the lanes that hold them, through LDS (a wave's own part of it, a lane's values side by side
// over the lanes, so that lanes of a section meet different banks).
template <typename T, int C, int NU>
__global__ __launch_bounds__(256) void rotate_mixed_kernel(RotateArgs a) {
  constexpr int TABLE = 2 * kMostPairs, OWN = NU * C * 64;
  __shared__ __align__(16) float lds[2 * TABLE + 4 * OWN];   // cosines and sines by channel, the waves' values
  __shared__ int64_t base[2][kMostPlaces];
  __shared__ int16_t other[512];
  const int tid = threadIdx.x, lane = tid & 63, u = tid & (a.lanes - 1), step = 256 / a.lanes, D = 2 * a.pairs;
  const Part w(a);
  prepare(a, w, base, [&](int n, int pair, float c, float s) {
    int low, size;
    section_of(a, pair, low, size);
    const int at = low + pair;
    // A channel that stays is one time itself and its cosine, 1, times -0, which added leaves every number, -0 too, as it is.
    const bool stay = c == kStay;
    float* token = lds + n * D;
    token[at] = token[at + size] = stay ? 1.f : c;
    token[TABLE + at] = -s;
    token[TABLE + at + size] = stay ? -s : s;
    if (n == 0) other[at] = (int16_t)(stay ? -1 : at + size), other[at + size] = (int16_t)(stay ? -1 : at);
  });
  bool in[NU];
  int at[NU];
#pragma unroll
  for (int i = 0; i < NU; i++) {
    in[i] = (u + i * a.lanes) * C < D;
    at[i] = in[i] ? (u + i * a.lanes) * C : 0;
  }
  Run<float, C> gamma[NU];
  const bool norm = a.gamma[w.which] != nullptr;
  if (norm)
#pragma unroll
    for (int i = 0; i < NU; i++) __builtin_memcpy(&gamma[i], a.gamma[w.which] + at[i], sizeof(gamma[i]));
  __syncthreads();
  const int own = 2 * TABLE + (tid >> 6) * OWN;
  const int log = __builtin_ctz(a.lanes);
  int from[NU * C];   // where the other end of a channel stands
#pragma unroll
  for (int i = 0; i < NU * C; i++) {
    const int mine = at[i / C] + i % C, c = other[mine], unit = c / C;
    from[i] = c < 0 ? mine : own + ((unit >> log) * C + c % C) * 64 + (lane - u) + (unit & (a.lanes - 1));
  }

  const T* x = (const T*)a.x[w.which];
  T* y = (T*)a.y[w.which];
  const int item = tid / a.lanes, tokens = udiv(step, a.by_heads[w.which]), rest = step - tokens * w.heads;
  int n = udiv(item, a.by_heads[w.which]), h = item - n * w.heads;
  Run<T, C> now[NU], next[NU];
  const auto load = [&](Run<T, C> (&e)[NU], int n, int h) {
    const T* p = x + base[0][n] + h * a.xs[w.which][2];
#pragma unroll
    for (int i = 0; i < NU; i++) __builtin_memcpy(&e[i], p + at[i], sizeof(e[i]));
  };
  if (n < w.count) load(now, n, h);
  while (n < w.count) {
    int nn = n + tokens, nh = h + rest;
    if (nh >= w.heads) nn++, nh -= w.heads;
    if (nn < w.count) load(next, nn, nh);
    float f[NU * C];
#pragma unroll
    for (int i = 0; i < NU * C; i++) f[i] = in[i / C] ? (float)now[i / C].v[i % C] : 0.f;
    if (norm) {
      const float root = root_of(a, f);
#pragma unroll
      for (int i = 0; i < NU * C; i++) f[i] = f[i] * root * gamma[i / C].v[i % C];
    }
#pragma unroll
    for (int i = 0; i < NU * C; i++) lds[own + i * 64 + lane] = f[i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    T* q = y + base[1][n] + h * a.ys[w.which][2];
#pragma unroll
    for (int i = 0; i < NU; i++) {
      if (!in[i]) continue;
      float c[C], s[C];
      table_n<C>(lds + n * D + at[i], c);
      table_n<C>(lds + TABLE + n * D + at[i], s);
      Run<T, C> o;
#pragma unroll
      for (int v = 0; v < C; v++) o.v[v] = (T)__builtin_fmaf(f[i * C + v], c[v], lds[from[i * C + v]] * s[v]);
      o.stream(q + at[i]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int i = 0; i < NU; i++) now[i] = next[i];
    n = nn;
    h = nh;
  }
}

template <typename T>
int launch_rotate(RotateArgs& a, bool near, int run, hipStream_t st) {
  // A lane's channels: `run` pairs of two halves, or eight channels as they lie, and fewer where heads are not whole
  // eights; of heads of many such units a lane takes several. Pairs are taken from halves of whole eights and fours: 30,000
  // tokens of 20 heads of 64 in fp16 33 us, 20,000 of 72 in three sections of 24 28 us, as they lie 36; halves of 4, 6 and 6
  // the other way round, 52 and 45 for 51,200 tokens of 32 heads of 32.
  const int D = 2 * a.pairs, each = run > 0 ? 2 * run : D % 8 == 0 ? 8 : D % 4 == 0 ? 4 : 2, units = D / each;
  int lanes = 1;
  while (lanes < units && lanes < 64) lanes *= 2;
  a.lanes = lanes;
  const bool many = units > lanes;
  // About four rounds of the threads a workgroup, but a thousand workgroups first, and the table's size.
  int64_t blocks[2] = {0, 0};
  for (int i = 0; i < 2; i++) {
    if (!a.heads[i]) continue;
    int64_t group = 1024 / ((int64_t)a.heads[i] * lanes);
    if (group > a.places / 1024) group = a.places / 1024;
    if (group < a.places >> 22) group = a.places >> 22;
    if (group > kMostPairs / a.pairs) group = kMostPairs / a.pairs;
    if (group > kMostPlaces) group = kMostPlaces;
    a.group[i] = (int)(group < 1 ? 1 : group);
    blocks[i] = (a.places + a.group[i] - 1) / a.group[i];
  }
  if (blocks[0] + blocks[1] > 1 << 23)   // 2^31 threads
    return fail("rotate_heads: %lld tokens of %d heads of %d are more than one launch takes", (long long)a.places,
                a.heads[0] + a.heads[1], 2 * a.pairs);
  a.blocks = (unsigned)blocks[0];
  const dim3 grid((unsigned)(blocks[0] + blocks[1])), block(256);
  if (run == 8) hipLaunchKernelGGL((rotate_kernel<T, 8, 1, false>), grid, block, 0, st, a);
  else if (run == 4) hipLaunchKernelGGL((rotate_kernel<T, 4, 1, false>), grid, block, 0, st, a);
  else if (near && each == 8) hipLaunchKernelGGL((rotate_kernel<T, 4, 1, true>), grid, block, 0, st, a);
  else if (near && each == 4 && many) hipLaunchKernelGGL((rotate_kernel<T, 2, 2, true>), grid, block, 0, st, a);
  else if (near && each == 4) hipLaunchKernelGGL((rotate_kernel<T, 2, 1, true>), grid, block, 0, st, a);
  else if (near && many) hipLaunchKernelGGL((rotate_kernel<T, 1, 4, true>), grid, block, 0, st, a);
  else if (near) hipLaunchKernelGGL((rotate_kernel<T, 1, 1, true>), grid, block, 0, st, a);
  else if (each == 8) hipLaunchKernelGGL((rotate_mixed_kernel<T, 8, 1>), grid, block, 0, st, a);
  else if (each == 4 && many) hipLaunchKernelGGL((rotate_mixed_kernel<T, 4, 2>), grid, block, 0, st, a);
  else if (each == 4) hipLaunchKernelGGL((rotate_mixed_kernel<T, 4, 1>), grid, block, 0, st, a);
  else if (many) hipLaunchKernelGGL((rotate_mixed_kernel<T, 2, 4>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((rotate_mixed_kernel<T, 2, 1>), grid, block, 0, st, a);
  return LDX_OK;
}

}  // namespace
}  // namespace ldx

using namespace ldx;

extern "C" int ldx_rotate_heads(const ldx_rotate_heads_args* p, void* stream) {
  if (!p || !p->q || !p->q_out || !p->positions || !p->turns) return fail("rotate_heads: null pointer");
  if (p->k_heads < 0 || (p->k_heads > 0 && (!p->k || !p->k_out))) return fail("rotate_heads: null pointer");
  if (p->dtype != LDX_DTYPE_F16 && p->dtype != LDX_DTYPE_BF16 && p->dtype != LDX_DTYPE_F32)
    return fail("rotate_heads: dtype %d is not LDX_DTYPE_F16, LDX_DTYPE_BF16 or LDX_DTYPE_F32", p->dtype);
  if (p->head_dim < 2 || p->head_dim % 2 || p->head_dim > 512)
    return fail("rotate_heads: head_dim %d is not an even number from 2 to 512", p->head_dim);
  if (p->q_heads < 1 || p->q_heads > 65536 || p->k_heads > 65536)
    return fail("rotate_heads: %d query and %d key heads", p->q_heads, p->k_heads);
  const int64_t places = (int64_t)p->batch * p->tokens;
  if (p->batch < 1 || p->tokens < 1 || places > 0x7fffffff)
    return fail("rotate_heads: %d sequences of %d tokens", p->batch, p->tokens);
  if (p->axes < 1 || p->axes > kAxes) return fail("rotate_heads: %d axes", p->axes);
  if ((p->q_gamma || p->k_gamma) && !(p->eps >= 1e-30f)) return fail("rotate_heads: eps %g is below 1e-30", (double)p->eps);
  RotateArgs a = {};
  int at = 0;
  int run = p->interleaved ? 0 : 8;   // every section's halves are whole eights, fours, or neither (0)
  const auto narrow = [&run](int pairs) { run = pairs % 8 == 0 ? run : pairs % 4 == 0 && run ? 4 : 0; };
  for (int i = 0; i < p->axes; i++) {
    const int w = p->axis_dims[i];
    if (w < 2 || w % 2 || w > p->head_dim) return fail("rotate_heads: axis of %d channels", w);
    a.section[i] = at;
    at += w / 2;
    narrow(w / 2);
  }
  if (at > p->head_dim / 2) return fail("rotate_heads: axes of %d channels in a head of %d", 2 * at, p->head_dim);
  a.section[p->axes] = at;
  a.pairs = p->head_dim / 2;
  narrow(a.pairs - at);
  a.x[0] = p->q, a.x[1] = p->k;
  a.y[0] = p->q_out, a.y[1] = p->k_out;
  for (int i = 0; i < 3; i++) {
    a.xs[0][i] = p->q_stride[i], a.xs[1][i] = p->k_stride[i];
    a.ys[0][i] = p->q_out_stride[i], a.ys[1][i] = p->k_out_stride[i];
    a.ps[i] = p->position_stride[i];
  }
  a.gamma[0] = p->q_gamma, a.gamma[1] = p->k_gamma;
  a.heads[0] = p->q_heads, a.heads[1] = p->k_heads;
  a.eps = p->eps;
  a.per = 1.f / (float)p->head_dim;
  a.positions = p->positions;
  a.turns = p->turns;
  a.axes = p->axes;
  a.places = places;
  a.L = p->tokens;
  a.by_L = make_udiv((unsigned)p->tokens);
  for (int i = 0; i < 2; i++) a.by_heads[i] = make_udiv((unsigned)(a.heads[i] > 0 ? a.heads[i] : 1));
  a.by_pairs = make_udiv((unsigned)a.pairs);
  hipStream_t st = as_stream(stream);
  const bool near = p->interleaved != 0;
  if (int rc = p->dtype == LDX_DTYPE_F16    ? launch_rotate<f16>(a, near, run, st)
               : p->dtype == LDX_DTYPE_BF16 ? launch_rotate<bf16>(a, near, run, st)
                                            : launch_rotate<float>(a, near, run, st))
    return rc;
  return check_launch("rotate_heads");
}
