// sas_product.h - what the projection kernels share: matrix products of bf16
// operands, f32 values as bf16 pieces, and the last steps of a result.
#pragma once

#include <utility>

#include "sas_device.h"
#include "sas_launch.h"

namespace sas {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef u16x4 u16x4u __attribute__((aligned(2)));

constexpr int kSub = 16;  // rows, outputs or ranks of one matrix instruction

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// An f32 value as three bf16 pieces whose sum it is, but for bits below 2^-133,
// bf16's last, which are cut off (values under 2^-110 have such bits).  Not
// finite: the first piece alone.
__device__ __forceinline__ void pieces_of(float x, uint16_t (&p)[3]) {
  const uint32_t u = __float_as_uint(x);
  const bool finite = (u & 0x7F800000u) != 0x7F800000u;
  p[0] = (uint16_t)((u | (x != x ? 0x400000u : 0u)) >> 16);
  const float r1 = finite ? x - __uint_as_float(u & 0xFFFF0000u) : 0.0f;
  const uint32_t u1 = __float_as_uint(r1);
  p[1] = (uint16_t)(u1 >> 16);
  const float r2 = r1 - __uint_as_float(u1 & 0xFFFF0000u);
  p[2] = (uint16_t)(__float_as_uint(r2) >> 16);
}

__device__ __forceinline__ uint16_t bf16_of(float x) {
  uint32_t u = __float_as_uint(x);
  if (x != x) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

// 8 f32 values as three bf16 operands.
__device__ __forceinline__ void split_f32(const float (&v)[8], u32x4 (&p)[3]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint16_t a[3], b[3];
    pieces_of(v[2 * i], a);
    pieces_of(v[2 * i + 1], b);
#pragma unroll
    for (int k = 0; k < 3; ++k) p[k][i] = (uint32_t)a[k] | ((uint32_t)b[k] << 16);
  }
}
// The same of 8 consecutive ones in memory (4-byte aligned).
__device__ __forceinline__ void split8(const float *src, u32x4 (&p)[3]) {
  const f32x4 v0 = *reinterpret_cast<const f32x4u *>(src), v1 = *reinterpret_cast<const f32x4u *>(src + 4);
  const float v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
  split_f32(v, p);
}

// tanh within 3.2 ulp by its roundings (1 ulp of the instructions' exp2 and
// reciprocal), 1.58 at worst over half a million values (at 0.627); below the split
// 0.72.  The method is Cody and Waite's (Software Manual for the Elementary
// Functions, 1980): below a split, here 0.625, x + x^3 P(x^2), P fitted to the
// relative error (8.6e-9 at most), above it 1 - 2 / (e^2|x| + 1).  A third of
// tanhf's instructions: 34 million capped values took 30 us of a call's 440.
// The part below the split:
__device__ __forceinline__ float tanh_small(float x) {
  const float u = x * x;
  float p = -0.005704975221306086f;
  p = __builtin_fmaf(p, u, 0.020639074966311455f);
  p = __builtin_fmaf(p, u, -0.05373971164226532f);
  p = __builtin_fmaf(p, u, 0.13331441581249237f);
  p = __builtin_fmaf(p, u, -0.3333328068256378f);
  return __builtin_fmaf(x * u, p, x);
}
__device__ __forceinline__ float tanh_fast(float x) {
  const float ax = fabsf(x), small = tanh_small(x);
  const float e = __builtin_amdgcn_exp2f(fminf(ax, 16.0f) * 2.8853900817779268f);  // e^2|x|
  const float large = copysignf(__builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f), x);
  return x != x ? x : ax < 0.625f ? small : large;
}

// The last steps of four sums of row `row`, outputs n .. n + 3: added to what
// is there, capped, rounded, stored.  Nontemporal: the result is not read here
// (128 x 262,144 f32: 312 -> 281 us a call, 268 with whole lines a row).
template <typename Args>
__device__ __forceinline__ void finish4(const Args &a, int row, int n, f32x4 v) {
  if (n >= a.out_dim) return;
  const bool whole = n + 4 <= a.out_dim;
  const int64_t at = (int64_t)row * a.out_stride + n;
  float *of = static_cast<float *>(a.out) + at;
  uint16_t *ob = static_cast<uint16_t *>(a.out) + at;
  if (a.accumulate) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.out_dim) v[i] += a.out_bf16 ? __uint_as_float((uint32_t)ob[i] << 16) : of[i];
  }
  if (a.softcap > 0.0f) {
    const float inv = 1.0f / a.softcap;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a.softcap * tanh_fast(v[i] * inv);
  }
  if (a.out_bf16) {
    const u16x4 p = {bf16_of(v[0]), bf16_of(v[1]), bf16_of(v[2]), bf16_of(v[3])};
    if (whole) {
      __builtin_nontemporal_store(p, reinterpret_cast<u16x4u *>(ob));
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (n + i < a.out_dim) ob[i] = p[i];
    }
  } else if (whole) {
    __builtin_nontemporal_store(v, reinterpret_cast<f32x4u *>(of));
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (n + i < a.out_dim) of[i] = v[i];
  }
}

// Blocks in runs that one XCD's L2 serves: block i runs on XCD i % 8.
__device__ __forceinline__ int xcd_run(int i, int n) {
  const int per = n / 8, left = n % 8, x = i % 8;
  return x * per + min(x, left) + i / 8;
}

// f(integral_constant 0) .. f(integral_constant N - 1).
template <int N, typename F, int... I>
__device__ __forceinline__ void each_const_of(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each_const(F f) {
  each_const_of<N>(f, std::make_integer_sequence<int, N>{});
}

}  // namespace sas
