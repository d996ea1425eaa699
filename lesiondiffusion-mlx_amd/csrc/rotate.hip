// Norms of queries and keys for each head with the position rotation in the same pass.
//
//   f = x / sqrt(mean(x^2) + eps) * gamma       (over a head's channels; x itself without gamma)
//   for every pair (a, b) of channels of axis A:  t = position_A * turns,  (a cos 2 pi t - b sin 2 pi t,
//                                                                        b cos 2 pi t + a sin 2 pi t)
//
// Positions have one axis (text) or several (a volume's depth, height and width); an axis turns a section of the
// head's channels, whose pairs are its two halves' or neighbours. Channels behind the sections stay as they are.
//
// One pass. A workgroup takes all heads of a few tokens: its threads first make the tokens' cosines and sines, which
// the heads share, then a lane takes V pairs of a head, both ends of each, so that a pair never leaves its lane, and
// the lanes of a head add their squares. V is what divides every section's pairs (8 where it can: 16 bytes at a time).
#include "quant8.h"

namespace ldx {
namespace {

constexpr int kAxes = LDX_ROTARY_AXES;
constexpr int kMostPairs = 1024;   // of the tokens of a workgroup

struct RotateArgs {
  const void* x[2]; int64_t xs[2][3];   // queries and keys: batch, token, head strides
  void* y[2]; int64_t ys[2][3];
  const float* gamma[2];
  int heads[2];
  float eps, per;       // per: 1 / channels
  const int32_t* positions; int64_t ps[3];   // axis, batch, token strides
  const double* turns;
  int section[kAxes + 1], rest;   // first pair of each axis and of the channels that stay; pairs of those
  int axes, pairs;                // pairs of a head
  int64_t places;                 // batch * tokens
  int L, group;                   // tokens of a sequence; tokens of a workgroup
  int lanes;                      // of a head, a power of two
  UDiv by_L, by_heads, by_pairs;
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

template <int N, typename T>
__device__ __forceinline__ void load_n(const T* p, float* f) {
  struct { T v[N]; } u;
  __builtin_memcpy(&u, p, sizeof(u));
#pragma unroll
  for (int i = 0; i < N; i++) f[i] = (float)u.v[i];
}
template <int N, typename T>
__device__ __forceinline__ void store_n(T* p, const float* f) {
  struct { T v[N]; } u;
#pragma unroll
  for (int i = 0; i < N; i++) u.v[i] = (T)f[i];
  __builtin_memcpy(p, &u, sizeof(u));
}

// Lane u of a head takes pairs (u + i * lanes) V .., i < NU; neighbours (NEAR) or halves of a section.
template <typename T, int V, int NU, bool NEAR>
__global__ __launch_bounds__(256) void rotate_kernel(RotateArgs a) {
  __shared__ __align__(16) float table[2][kMostPairs];   // cosines, sines
  const int tid = threadIdx.x;
  const int64_t first = (int64_t)blockIdx.x * a.group;
  const int count = (int)min((int64_t)a.group, a.places - first);
  for (int e = tid; e < count * a.pairs; e += 256) {
    const int n = udiv(e, a.by_pairs), pair = e - n * a.pairs;
    const int64_t place = first + n;
    const int b = udiv((int)place, a.by_L), l = (int)place - b * a.L;
    float c = 1.f, s = 0.f;
    if (pair < a.section[a.axes]) {
      int axis = 0;
#pragma unroll
      for (int i = 1; i < kAxes; i++) axis += i < a.axes && pair >= a.section[i] ? 1 : 0;
      const double t = (double)a.positions[axis * a.ps[0] + b * a.ps[1] + l * a.ps[2]] * a.turns[pair];
      turn(t - __builtin_rint(t), c, s);
    }
    table[0][e] = c;
    table[1][e] = s;
  }
  __syncthreads();

  const int heads = a.heads[0] + a.heads[1], u = tid & (a.lanes - 1), per = 256 / a.lanes;
  int at[NU], to[NU];   // a unit's channels: first ends from `at` on, second ends from `to` on
#pragma unroll
  for (int i = 0; i < NU; i++) {
    const int pair = (u + i * a.lanes) * V;
    int low = 0, size = a.axes > 0 ? a.section[1] : a.rest;
#pragma unroll
    for (int x = 1; x <= kAxes; x++)
      if (x <= a.axes && pair >= a.section[x]) {
        low = a.section[x];
        size = (x < a.axes ? a.section[x + 1 > kAxes ? kAxes : x + 1] : a.pairs) - low;
      }
    at[i] = NEAR ? 2 * pair : low + pair;
    to[i] = at[i] + size;
  }
  for (int item = tid / a.lanes; item < count * heads; item += per) {
    const int n = udiv(item, a.by_heads), h = item - n * heads, which = h >= a.heads[0] ? 1 : 0;
    const int head = which ? h - a.heads[0] : h;
    const int64_t place = first + n;
    const int b = udiv((int)place, a.by_L), l = (int)place - b * a.L;
    const T* x = (const T*)a.x[which] + b * a.xs[which][0] + l * a.xs[which][1] + head * a.xs[which][2];
    T* y = (T*)a.y[which] + b * a.ys[which][0] + l * a.ys[which][1] + head * a.ys[which][2];
    const float* gamma = a.gamma[which];
    float f[NU][V], g[NU][V];   // first and second ends
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NU; i++) {
      const bool in = (u + i * a.lanes) * V < a.pairs;
#pragma unroll
      for (int v = 0; v < V; v++) f[i][v] = g[i][v] = 0.f;
      if (in) {
        if constexpr (NEAR) {
          float w[2 * V];
          load_n<2 * V>(x + at[i], w);
#pragma unroll
          for (int v = 0; v < V; v++) f[i][v] = w[2 * v], g[i][v] = w[2 * v + 1];
        } else {
          load_n<V>(x + at[i], f[i]);
          load_n<V>(x + to[i], g[i]);
        }
      }
#pragma unroll
      for (int v = 0; v < V; v++) sum = __builtin_fmaf(f[i][v], f[i][v], __builtin_fmaf(g[i][v], g[i][v], sum));
    }
    if (gamma) {
      sum = head_sum(sum, a.lanes);
      float root, pre = 1.f;
      if (sum <= 3.0e38f) {
        root = __builtin_amdgcn_rsqf(__builtin_fmaf(sum, a.per, a.eps));
      } else {   // squares past fp32 (or NaN): those of the values times 2^-66
        pre = 0x1p-66f;
        float small = 0.f;
#pragma unroll
        for (int i = 0; i < NU; i++)
#pragma unroll
          for (int v = 0; v < V; v++) {
            const float p = f[i][v] * pre, q = g[i][v] * pre;
            small = __builtin_fmaf(p, p, __builtin_fmaf(q, q, small));
          }
        small = head_sum(small, a.lanes);
        root = __builtin_amdgcn_rsqf(small * a.per);
      }
#pragma unroll
      for (int i = 0; i < NU; i++) {
        const bool in = (u + i * a.lanes) * V < a.pairs;
        if (!in) continue;
        float p[V], q[V];
        if constexpr (NEAR) {
          float w[2 * V];
          load_n<2 * V>(gamma + at[i], w);
#pragma unroll
          for (int v = 0; v < V; v++) p[v] = w[2 * v], q[v] = w[2 * v + 1];
        } else {
          load_n<V>(gamma + at[i], p);
          load_n<V>(gamma + to[i], q);
        }
#pragma unroll
        for (int v = 0; v < V; v++) {
          f[i][v] = f[i][v] * pre * root * p[v];
          g[i][v] = g[i][v] * pre * root * q[v];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NU; i++) {
      const int pair = (u + i * a.lanes) * V;
      if (pair >= a.pairs) continue;
      float c[V], s[V];
      load_n<V>(&table[0][n * a.pairs + pair], c);
      load_n<V>(&table[1][n * a.pairs + pair], s);
      float p[V], q[V];
#pragma unroll
      for (int v = 0; v < V; v++) {
        p[v] = __builtin_fmaf(f[i][v], c[v], -(g[i][v] * s[v]));
        q[v] = __builtin_fmaf(g[i][v], c[v], f[i][v] * s[v]);
      }
      if constexpr (NEAR) {
        float w[2 * V];
#pragma unroll
        for (int v = 0; v < V; v++) w[2 * v] = p[v], w[2 * v + 1] = q[v];
        store_n<2 * V>(y + at[i], w);
      } else {
        store_n<V>(y + at[i], p);
        store_n<V>(y + to[i], q);
      }
    }
  }
}

template <typename T, bool NEAR>
void launch_near(RotateArgs& a, int v, hipStream_t st) {
  const int units = a.pairs / v;
  int lanes = 1;
  while (lanes < units && lanes < 64) lanes *= 2;
  a.lanes = lanes;
  const int nu = (units + lanes - 1) / lanes;   // 1; up to 4 at one pair a lane
  const int heads = a.heads[0] + a.heads[1];
  // About four rounds of the threads a workgroup, but a thousand workgroups first, and the table's size.
  int64_t group = 1024 / ((int64_t)heads * lanes);
  if (group > a.places / 1024) group = a.places / 1024;
  if (group > kMostPairs / a.pairs) group = kMostPairs / a.pairs;
  a.group = (int)(group < 1 ? 1 : group);
  const dim3 grid((unsigned)((a.places + a.group - 1) / a.group)), block(256);
  if constexpr (!NEAR)
    if (v == 8) {
      hipLaunchKernelGGL((rotate_kernel<T, 8, 1, false>), grid, block, 0, st, a);
      return;
    }
  if (v == 4) hipLaunchKernelGGL((rotate_kernel<T, 4, 1, NEAR>), grid, block, 0, st, a);
  else if (v == 2 && nu == 1) hipLaunchKernelGGL((rotate_kernel<T, 2, 1, NEAR>), grid, block, 0, st, a);
  else if (v == 2) hipLaunchKernelGGL((rotate_kernel<T, 2, 2, NEAR>), grid, block, 0, st, a);
  else if (nu == 1) hipLaunchKernelGGL((rotate_kernel<T, 1, 1, NEAR>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((rotate_kernel<T, 1, 4, NEAR>), grid, block, 0, st, a);
}

template <typename T>
void launch_rotate(RotateArgs& a, bool near, int v, hipStream_t st) {
  if (near) launch_near<T, true>(a, v, st);
  else launch_near<T, false>(a, v, st);
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
  int at = 0, common = p->interleaved ? p->head_dim / 2 : 0;   // what V has to divide
  const auto gcd = [](int x, int y) {
    while (y) {
      const int r = x % y;
      x = y;
      y = r;
    }
    return x;
  };
  for (int i = 0; i < p->axes; i++) {
    const int w = p->axis_dims[i];
    if (w < 2 || w % 2 || w > p->head_dim) return fail("rotate_heads: axis of %d channels", w);
    a.section[i] = at;
    at += w / 2;
    if (!p->interleaved) common = gcd(common, w / 2);
  }
  if (at > p->head_dim / 2) return fail("rotate_heads: axes of %d channels in a head of %d", 2 * at, p->head_dim);
  a.section[p->axes] = at;
  a.pairs = p->head_dim / 2;
  a.rest = a.pairs - at;
  if (!p->interleaved) common = gcd(common, a.rest);
  const int v = common % 8 == 0 && !p->interleaved ? 8 : common % 4 == 0 ? 4 : common % 2 == 0 ? 2 : 1;
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
  a.by_heads = make_udiv((unsigned)(p->q_heads + p->k_heads));
  a.by_pairs = make_udiv((unsigned)a.pairs);
  hipStream_t st = as_stream(stream);
  if (p->dtype == LDX_DTYPE_F16) launch_rotate<f16>(a, p->interleaved != 0, v, st);
  else if (p->dtype == LDX_DTYPE_BF16) launch_rotate<bf16>(a, p->interleaved != 0, v, st);
  else launch_rotate<float>(a, p->interleaved != 0, v, st);
  return check_launch("rotate_heads");
}
