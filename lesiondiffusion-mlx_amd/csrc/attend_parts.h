// What the attention kernels over paged caches share: page tables, the tokens that a query sees, and the
// join of a sequence's parts where it is split over workgroups. A is a kernel's argument block with the
// fields used here: G (query heads of a cache head), H, lq, rows = G * lq, tile (rows of a workgroup), o and
// its strides, lengths, starts, width, splits (parts that a sequence may have), chunk (least pages of one)
// and part: [b][h][row][split] of D sums, then of (reference, sum of probabilities).
#pragma once

#include "quant8.h"

namespace ldx {

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

// The keys that a query sees: limit = min(length, start + i + 1) with starts, the length without.
template <typename A>
__device__ __forceinline__ int key_limit(const A& a, int len, int64_t start, int row) {
  if (!a.starts) return len;
  const int64_t c = start + row / a.G + 1;
  return (int)(c < 0 ? 0 : c < len ? c : len);
}

// Parts that a sequence of npages has (of a.splits possible ones), at least one.
template <typename A>
__device__ __forceinline__ int part_count(const A& a, int npages) {
  const int chunk = max((npages + a.splits - 1) / a.splits, a.chunk);
  return max((npages + chunk - 1) / chunk, 1);
}

// The output of four channels of a row.
template <typename T, typename A>
__device__ __forceinline__ void put4(const A& a, int b, int h, int row, int channel, f32x4 o, float l) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* op = (T*)a.o + b * a.os[0] + (int64_t)(row / a.G) * a.os[1] + (int64_t)(h * a.G + row % a.G) * a.os[2] + channel;
#pragma unroll
  for (int i = 0; i < 4; i++) op[i] = (T)(o[i] * inv);
}

// Parts that a row's sequence was given.
template <typename A>
__device__ __forceinline__ int parts_of(const A& a, int b, int row) {
  const int raw = a.lengths[b];
  const int len = raw < 0 || raw > (int64_t)a.width * kPage8 ? 0 : raw;
  // The last row of a workgroup's tile says how many pages it reads.
  const int most = key_limit(a, len, a.starts ? a.starts[b] : 0, min((row / a.tile + 1) * a.tile, a.rows) - 1);
  return part_count(a, (most + kPage8 - 1) / kPage8);
}

// Joins the parts of rows, few parts (at most kFewParts): a thread takes four channels of a row.
constexpr int kFewParts = 8;

template <typename T, int D, typename A>
__global__ __launch_bounds__(256) void attend_join_kernel(A a, int64_t total) {
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

template <typename T, int D, typename A>
__global__ __launch_bounds__(256) void attend_merge_kernel(A a) {
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

template <typename T, int D, typename A>
void launch_join(const A& a, int64_t total, hipStream_t st) {
  constexpr int ROWS = 1024 / D;   // of a workgroup
  if (a.splits > kFewParts)
    hipLaunchKernelGGL((attend_merge_kernel<T, D, A>), dim3((unsigned)total), dim3(256), 0, st, a);
  else if (a.splits > 1)
    hipLaunchKernelGGL((attend_join_kernel<T, D, A>), dim3((unsigned)((total + ROWS - 1) / ROWS)), dim3(256), 0, st, a, total);
}

}  // namespace ldx
