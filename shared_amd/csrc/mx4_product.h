// mx4_product.h - products with rows of MXFP4 values (gfx950): the kernels that
// sas_project_mx4 and the fused head share.
#pragma once

#include "sas_product.h"

namespace sas {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kBlock = SAS_MX4_BLOCK;
// The f32 scale of byte s as the conversions take it.
__device__ __forceinline__ float scale_of(uint32_t s) { return __uint_as_float(s << 23); }

// --------------------------------------------------------------- products --

constexpr int kRun = 4 * kBlock;  // values of dim a step: a block a lane

// The 32 values of a block as four bf16 operands of 8.
__device__ __forceinline__ void widen(u32x4 c, uint32_t s, u32x4 (&w)[4]) {
  const float by = scale_of(s);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[i], by, 0));
    w[i][1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[i], by, 1));
    w[i][2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[i], by, 2));
    w[i][3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[i], by, 3));
  }
}

__device__ __forceinline__ f32x4 mfma4(u32x4 w, uint32_t ws, u32x4 x, uint32_t xs, f32x4 c) {
  const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  const i32x8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, 0, (int)ws, 0, (int)xs);
}

// Eight waves split dim for the same 16 NT outputs of 16 MT rows; their sums
// meet in LDS in a fixed order.
constexpr int kSplitWaves = 8;

template <int MT, int NT, int kX>
__global__ __launch_bounds__(64 * kSplitWaves) void mx4_split_kernel(const Mx4ProjArgs a) {
  __shared__ f32x4 part[kSplitWaves][MT * NT][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int mtiles = (a.rows + 16 * MT - 1) / (16 * MT);
  const int pos = xcd_run((int)blockIdx.x, (int)gridDim.x);
  const int m0 = (pos % mtiles) * 16 * MT, n0 = (pos / mtiles) * 16 * NT;
  const u32x4 none = {0u, 0u, 0u, 0u};
  const int blocks = (a.dim + kBlock - 1) / kBlock, runs = (blocks + 3) / 4;
  const int g0 = runs * wave / kSplitWaves, g1 = runs * (wave + 1) / kSplitWaves;
  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int g = g0; g < g1; ++g) {
    const int b = 4 * g + q;
    const bool in = b < blocks;
    u32x4 w[NT];
    uint32_t ws[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int64_t row = min(n0 + 16 * t + r, a.out_dim - 1);
      w[t] = in ? *reinterpret_cast<const u32x4 *>(a.w + row * a.w_stride + 16 * b) : none;
      ws[t] = in ? a.w_scales[row * a.w_scales_stride + b] : 127u;
    }
    if constexpr (kX == SAS_TYPE_MX4) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int64_t row = min(m0 + 16 * m + r, a.rows - 1);
        const u32x4 x = in ? *reinterpret_cast<const u32x4 *>(static_cast<const uint8_t *>(a.x) + row * a.x_stride + 16 * b) : none;
        const uint32_t xs = in ? a.x_scales[row * a.x_scales_stride + b] : 127u;
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[m][t] = mfma4(w[t], ws[t], x, xs, acc[m][t]);
      }
    } else {
      u32x4 wide[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) widen(w[t], ws[t], wide[t]);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int64_t row = min(m0 + 16 * m + r, a.rows - 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = kBlock * b + 8 * i;
          if constexpr (kX == SAS_TYPE_F32) {
            u32x4 x[3] = {none, none, none};
            if (k < a.dim) split8(static_cast<const float *>(a.x) + row * a.x_stride + k, x);
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
              for (int t = 0; t < NT; ++t) acc[m][t] = mfma(wide[t][i], x[p], acc[m][t]);
          } else {
            const u32x4 x = k < a.dim ? *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(a.x) + row * a.x_stride + k) : none;
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[m][t] = mfma(wide[t][i], x, acc[m][t]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][m * NT + t][lane] = acc[m][t];
  __syncthreads();
  for (int i = wave; i < MT * NT; i += kSplitWaves) {
    f32x4 v = part[0][i][lane];
#pragma unroll
    for (int w = 1; w < kSplitWaves; ++w) v = v + part[w][i][lane];
    const int row = m0 + 16 * (i / NT) + r;
    if (row < a.rows) finish4(a, row, n0 + 16 * (i % NT) + 4 * q, v);
  }
}

template <int MT, int NT, int kX>
void launch_split(const Mx4ProjArgs &a, hipStream_t stream) {
  const int blocks = ((a.rows + 16 * MT - 1) / (16 * MT)) * ((a.out_dim + 16 * NT - 1) / (16 * NT));
  mx4_split_kernel<MT, NT, kX><<<blocks, 64 * kSplitWaves, 0, stream>>>(a);
}

}  // namespace
}  // namespace sas
