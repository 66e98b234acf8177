// mx4_kernel.hip - values in microscaled 4-bit floating point (MXFP4):
// quantisation, lookup of a table's rows, and products (gfx950).
//
// A row's values lie in blocks of 32: 16 bytes of elements (a sign, two bits of
// exponent, one of mantissa: 0 0.5 1 1.5 2 3 4 6; the first of a byte in its low
// half) and a byte s, the block's scale 2^(s - 127); 255 is NaN.  Quantisation
// rounds x / 2^(s - 127), which is exact, once.  The products are in
// mx4_product.h; here is which kernel takes a call.
#include <algorithm>

#include "mx4_product.h"

namespace sas {
namespace {

constexpr int kUnit = 4 * kBlock;  // values that 16 lanes handle, 8 each

// 8 consecutive values of a row as f32, those from `left` on zero.
template <int kType, bool kWide>
__device__ __forceinline__ void load8(const void *row, int64_t k, int left, float (&v)[8]) {
  if constexpr (kType == SAS_TYPE_F32) {
    const float *p = static_cast<const float *>(row) + k;
    if (kWide && left >= 8) {
      const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : 0.0f;
  } else {
    const uint16_t *p = static_cast<const uint16_t *>(row) + k;
    uint16_t h[8];
    if (kWide && left >= 8) {
      const u32x4 a = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) h[2 * i] = (uint16_t)a[i], h[2 * i + 1] = (uint16_t)(a[i] >> 16);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = i < left ? p[i] : (uint16_t)0;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = kType == SAS_TYPE_BF16 ? __uint_as_float((uint32_t)h[i] << 16) : (float)__builtin_bit_cast(_Float16, h[i]);
  }
}

// Units of 4 blocks, 16 lanes each, a lane 8 values: a block's largest magnitude
// is two exchanges among four lanes.  Bound by memory: 262,144 x 2,560 bf16 307 us
// (5.5 TB/s of what it reads and writes), 2,048 x 4,096 6.3 us.  Rows off 16 bytes
// load value by value: 262,144 x 2,559 746 us.
template <int kType, bool kWide>
__global__ __launch_bounds__(kThreads) void mx4_quantize_kernel(const Mx4QuantizeArgs a) {
  const int e = threadIdx.x & 15;
  const uint32_t units = (uint32_t)a.rows * (uint32_t)a.row_units;
  // (16 lanes together)
  for (uint32_t u = blockIdx.x * (kThreads / 16) + (threadIdx.x >> 4); u < units; u += gridDim.x * (kThreads / 16)) {
    const uint32_t row = u / (uint32_t)a.row_units, k = (u - row * (uint32_t)a.row_units) * kUnit + 8 * e;
    float v[8];
    const int left = a.dim - (int)k;
    const int64_t size = kType == SAS_TYPE_F32 ? 4 : 2;
    load8<kType, kWide>(static_cast<const char *>(a.x) + (int64_t)row * a.x_stride * size, k, left, v);
    // the largest magnitude's bits order as it does, NaN above infinity
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    top = max(top, dppx<kDppQuad1032>(top));
    top = max(top, dppx<kDppQuad2301>(top));
    const bool finite = top < 0x7F800000u;
    // 2^(s - 127) = 2^(floor(log2 top) - 2), at least 2^-127
    const uint32_t s = finite ? (uint32_t)max((int)(top >> 23) - 2, 0) : 255u;
    // x / 2^(s - 127) is exact, below 8; the conversion rounds it to the nearest
    // element, ties to the even one, and stops at 6
    const float by = __uint_as_float((254u - (finite ? s : 127u)) << 23);
    uint32_t c = 0;
    each_const<4>([&](auto it) __attribute__((always_inline)) {
      constexpr int i = decltype(it)::value;
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2 * i] * by, v[2 * i + 1] * by, 1.0f, i);
    });
    if (!finite) c = 0;
    // (a block that the row has no value of is left alone)
    const int b = (int)k / kBlock, blocks = (a.dim + kBlock - 1) / kBlock;
    if (b < blocks) *reinterpret_cast<uint32_t *>(a.codes + (int64_t)row * a.codes_stride + k / 2) = c;
    uint32_t four = (b < blocks ? s : 0u) << (8 * (e >> 2));
    four |= dppx<kDppRowRor4>(four);
    four |= dppx<kDppRowRor8>(four);
    if (e == 0) *reinterpret_cast<uint32_t *>(a.scales + (int64_t)row * a.scales_stride + k / kBlock) = four;
  }
}

// Units of 4 blocks, a lane 16 bytes of the result, so that a wave's store is whole
// lines: nontemporal then (8,192 x 4,096 to bf16 21.0 -> 14.9 us, 5.7 TB/s; f32
// in two stores of every second 16 bytes 18.2 -> 21.9 us).  Results off 16 bytes
// are stored value by value: 262,144 x 2,560 bf16 354 us, x 2,559 889.
template <int kType>
constexpr int kLookup = kType == SAS_TYPE_F32 ? 4 : 8;  // values of a lane
template <int kType, bool kWide>
__global__ __launch_bounds__(kThreads) void mx4_lookup_kernel(const Mx4LookupArgs a) {
  constexpr int V = kLookup<kType>, kLanes = kUnit / V;
  const int e = threadIdx.x % kLanes;
  const uint32_t units = (uint32_t)a.rows * (uint32_t)a.row_units;
  for (uint32_t u = blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes; u < units; u += gridDim.x * (kThreads / kLanes)) {
    const uint32_t row = u / (uint32_t)a.row_units, k = (u - row * (uint32_t)a.row_units) * kUnit + V * e;
    const int left = a.dim - (int)k;
    if (left <= 0) continue;
    const uint32_t id = a.ids ? a.ids[row] : row;
    const bool in = id < (uint32_t)a.table_rows;
    const uint8_t *at4 = a.codes + (int64_t)id * a.codes_stride + k / 2;
    uint32_t c = 0u;
    if (in) c = V == 8 ? *reinterpret_cast<const uint32_t *>(at4) : *reinterpret_cast<const uint16_t *>(at4);
    const float by = scale_of(in ? a.scales[(int64_t)id * a.scales_stride + k / kBlock] : 127u);
    float v[V];
    each_const<V / 2>([&](auto it) __attribute__((always_inline)) {
      constexpr int i = decltype(it)::value;
      const f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, by, i);
      v[2 * i] = p[0];
      v[2 * i + 1] = p[1];
    });
    const int64_t at = (int64_t)row * a.out_stride + k;
    if constexpr (kType == SAS_TYPE_F32) {
      float *o = static_cast<float *>(a.out) + at;
      if (kWide && left >= V) {
        __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4 *>(o));
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i < left) o[i] = v[i];
      }
    } else {
      uint16_t *o = static_cast<uint16_t *>(a.out) + at;
      uint16_t h[V];
#pragma unroll
      for (int i = 0; i < V; ++i) h[i] = kType == SAS_TYPE_BF16 ? bf16_of(v[i]) : __builtin_bit_cast(uint16_t, (_Float16)v[i]);
      if (kWide && left >= V) {
        u32x4 p;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = (uint32_t)h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
        __builtin_nontemporal_store(p, reinterpret_cast<u32x4 *>(o));
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i < left) o[i] = h[i];
      }
    }
  }
}

// The outputs a wave of the wide kernel takes, in 16s: the fewest rounds of blocks,
// a round counted as its products and half of 16 outputs more.  One / two of
// them, us: bf16, 64 rows x 4,096 x 32,768 (one round either way) 25 / 36; 32 x
// 4,096 x 65,536 (two rounds, one) 33 / 30; 128 x 2,560 x 262,144 191 / 161; f32,
// one / two / three, 16 x 2,560 x 32,000 17 / 24 / 31, x 128,256 52 / 47 / 63,
// x 151,936 63 / 65 / 63; 12 x 2,048 x 200,000 67 / 66 / 70.
int wide_nt(const Mx4ProjArgs &a, int mt, int most) {
  int best = 1;
  int64_t cost = INT64_MAX;
  for (int nt = 1; nt <= most; ++nt) {
    const int64_t blocks = (int64_t)((a.rows + 16 * mt - 1) / (16 * mt)) * ((a.out_dim + 128 * nt - 1) / (128 * nt));
    const int64_t c = (blocks + a.cus - 1) / a.cus * (2 * nt + 1);
    if (c <= cost) {
      cost = c;
      best = nt;
    }
  }
  return best;
}

template <int kX>
void launch_products(const Mx4ProjArgs &a, hipStream_t stream) {
  if (kX == SAS_TYPE_F32 && a.rows <= kMx4Few) return launch_mx4_few(a, stream);
  // (rows further apart than the other kernels' 32-bit offsets reach)
  const bool far = a.x_stride >= kMaxXStride || a.out_stride >= kMaxOutStride;
  if (a.rows <= 16) {
    if (far || split_fits<1, 1>(a)) return launch_split<1, 1, kX>(a, stream);
    if constexpr (kX != SAS_TYPE_F32)
      if (stream_fits<1, kX>(a)) return launch_stream<1, 1, kX>(a, stream);
    switch (wide_nt(a, 1, 3)) {
      case 1: return launch_wide<1, 1, kX>(a, stream);
      case 2: return launch_wide<1, 2, kX>(a, stream);
      default: return launch_wide<1, 3, kX>(a, stream);
    }
  }
  if (a.rows <= 32) {
    if (far || split_fits<2, 2>(a)) return launch_split<2, 2, kX>(a, stream);
    if constexpr (kX == SAS_TYPE_MX4)
      if (stream_fits<2, kX>(a)) return launch_stream<2, 1, kX>(a, stream);
    return wide_nt(a, 2, 2) == 1 ? launch_wide<2, 1, kX>(a, stream) : launch_wide<2, 2, kX>(a, stream);
  }
  if (far || split_fits<4, 2>(a)) return launch_split<4, 2, kX>(a, stream);
  if constexpr (kX == SAS_TYPE_MX4)
    if (a.rows <= 64 && stream_fits<4, kX>(a)) return launch_stream<4, 1, kX>(a, stream);
  // (128 rows of f32 pieces do not fit in LDS)
  if (a.rows <= 64 || kX == SAS_TYPE_F32)
    return wide_nt(a, 4, 2) == 1 ? launch_wide<4, 1, kX>(a, stream) : launch_wide<4, 2, kX>(a, stream);
  if constexpr (kX != SAS_TYPE_F32)
    return wide_nt(a, 8, 2) == 1 ? launch_wide<8, 1, kX>(a, stream) : launch_wide<8, 2, kX>(a, stream);
}

template <int kType>
void launch_quantize_of(const Mx4QuantizeArgs &a, bool wide, unsigned blocks, hipStream_t stream) {
  if (wide) mx4_quantize_kernel<kType, true><<<blocks, kThreads, 0, stream>>>(a);
  else mx4_quantize_kernel<kType, false><<<blocks, kThreads, 0, stream>>>(a);
}

template <int kType>
void launch_lookup_of(const Mx4LookupArgs &a, bool wide, unsigned blocks, hipStream_t stream) {
  if (wide) mx4_lookup_kernel<kType, true><<<blocks, kThreads, 0, stream>>>(a);
  else mx4_lookup_kernel<kType, false><<<blocks, kThreads, 0, stream>>>(a);
}

// Blocks for `units` of them, `per` a block: a launch holds fewer than 2^32
// threads, so that past 2^22 blocks they go round.
unsigned unit_blocks(int64_t units, int per) { return (unsigned)std::min<int64_t>((units + per - 1) / per, 1 << 22); }

// Whether rows may be read or written in 16-byte pieces.
bool in_pieces(const void *p, int64_t stride, int type) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % (type == SAS_TYPE_F32 ? 4 : 8) == 0;
}

}  // namespace

hipError_t launch_mx4_quantize(const Mx4QuantizeArgs &in, hipStream_t stream) {
  Mx4QuantizeArgs a = in;
  a.row_units = (a.dim + kUnit - 1) / kUnit;
  const unsigned blocks = unit_blocks((int64_t)a.rows * a.row_units, kThreads / 16);
  const bool wide = in_pieces(a.x, a.x_stride, a.x_type);
  if (a.x_type == SAS_TYPE_F32) launch_quantize_of<SAS_TYPE_F32>(a, wide, blocks, stream);
  else if (a.x_type == SAS_TYPE_BF16) launch_quantize_of<SAS_TYPE_BF16>(a, wide, blocks, stream);
  else launch_quantize_of<SAS_TYPE_F16>(a, wide, blocks, stream);
  return hipGetLastError();
}

hipError_t launch_mx4_lookup(const Mx4LookupArgs &in, hipStream_t stream) {
  Mx4LookupArgs a = in;
  a.row_units = (a.dim + kUnit - 1) / kUnit;
  const int per = kThreads / (a.out_type == SAS_TYPE_F32 ? kUnit / kLookup<SAS_TYPE_F32> : kUnit / kLookup<SAS_TYPE_BF16>);
  const unsigned blocks = unit_blocks((int64_t)a.rows * a.row_units, per);
  const bool wide = in_pieces(a.out, a.out_stride, a.out_type);
  if (a.out_type == SAS_TYPE_F32) launch_lookup_of<SAS_TYPE_F32>(a, wide, blocks, stream);
  else if (a.out_type == SAS_TYPE_BF16) launch_lookup_of<SAS_TYPE_BF16>(a, wide, blocks, stream);
  else launch_lookup_of<SAS_TYPE_F16>(a, wide, blocks, stream);
  return hipGetLastError();
}

hipError_t launch_mx4_project(const Mx4ProjArgs &a, hipStream_t stream) {
  if (a.x_type == SAS_TYPE_F32) launch_products<SAS_TYPE_F32>(a, stream);
  else if (a.x_type == SAS_TYPE_BF16) launch_products<SAS_TYPE_BF16>(a, stream);
  else launch_products<SAS_TYPE_MX4>(a, stream);
  return hipGetLastError();
}

}  // namespace sas
