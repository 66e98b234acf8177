// mx4_product.h - products with rows of MXFP4 values (gfx950): the kernels that
// sas_project_mx4 and the fused head share.
#pragma once

#include "sas_product.h"

namespace sas {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef u32x4 u32x4a4 __attribute__((aligned(4)));

constexpr int kBlock = SAS_MX4_BLOCK;
// The f32 scale of byte s as the conversions take it.
__device__ __forceinline__ float scale_of(uint32_t s) { return __uint_as_float(s << 23); }

// --------------------------------------------------------------- products --

constexpr int kRun = 4 * kBlock;   // values of dim a step: a block a lane
constexpr int kSuper = 4 * kRun;   // values whose scales are loaded together

// Element octet i of a block (16 bytes of codes) under scale byte j of `s4` as a
// bf16 operand; exact.
template <int kByte>
__device__ __forceinline__ float scale_byte(uint32_t s4) {
  if constexpr (kByte == 0) return scale_of(s4 & 255u);
  else return __uint_as_float((s4 >> (8 * kByte - 8) & 0xFF00u) << 15);
}
__device__ __forceinline__ u32x4 widen(uint32_t c, float by) {
  u32x4 w;
  w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, by, 0));
  w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, by, 1));
  w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, by, 2));
  w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, by, 3));
  return w;
}

// 16 outputs x 16 rows x 128 values of MXFP4: lane l holds block l / 16 of weight
// row and row l % 16, its scale in byte kByte of ws and xs.
template <int kByte>
__device__ __forceinline__ f32x4 mfma4(u32x4 w, uint32_t ws, u32x4 x, uint32_t xs, f32x4 c) {
  const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  const i32x8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, kByte, (int)ws, kByte, (int)xs);
}

// A lane's scales of a super-run: of the row's 16 bytes from block 16 s on, byte
// q of each dword (blocks q, 4 + q, 8 + q, 12 + q).
struct Scales {
  u32x4 d;
};
__device__ __forceinline__ Scales load_scales(const uint8_t *row, int s, int blocks) {
  Scales v;
  const int last = (blocks - 1) / 4;  // the dwords behind it are not the row's
  if (4 * s + 3 <= last) {
    v.d = *reinterpret_cast<const u32x4a4 *>(row + 16 * s);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v.d[i] = *reinterpret_cast<const uint32_t *>(row + 4 * min(4 * s + i, last));
  }
  return v;
}
// Bytes past the row's last block become 127 (1): what is there may be NaN.
__device__ __forceinline__ uint32_t pack_scales(const Scales &v, int q, int s, int blocks) {
  const uint32_t sel = 0x0C0C0400u + 0x0101u * (uint32_t)q;
  const uint32_t lo = __builtin_amdgcn_perm(v.d[1], v.d[0], sel), hi = __builtin_amdgcn_perm(v.d[3], v.d[2], sel);
  uint32_t p = lo | (hi << 16);
  if (16 * s + 16 > blocks) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (16 * s + 4 * j + q >= blocks) p = (p & ~(0xFFu << (8 * j))) | (0x7Fu << (8 * j));
  }
  return p;
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
        for (int t = 0; t < NT; ++t) acc[m][t] = mfma4<0>(w[t], ws[t], x, xs, acc[m][t]);
      }
    } else {
      u32x4 wide[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) wide[t][i] = widen(w[t][i], scale_of(ws[t]));
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

// ---- the hidden states in LDS ----
//
// An operand: 16 rows x 128 values of bf16 (4 KB) in two halves of 64 values,
// value octet o of row r in 16-byte slot 8 r + (o ^ r / 2) of its half; or 16 rows
// x 64 bytes of codes (1 KB), block c of row r in slot 4 r + (c ^ r / 4).  The
// lanes that write a row, and the 16 rows that read an octet or a block, meet
// every bank once.
template <int kX>
struct XOperand {
  static constexpr int kSlots = kX == SAS_TYPE_MX4 ? 64 : 256;
  static constexpr int kLoads = kX == SAS_TYPE_MX4 ? 1 : 4;  // a wave's loads of it: 8 rows x 64 values, or all codes
  static constexpr int kPieces = kX == SAS_TYPE_F32 ? 3 : 1;
};
// The slot of lane's read: octet 4 q + i of row r, or block q.
template <int kX>
__device__ __forceinline__ int x_get(int i) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  if constexpr (kX == SAS_TYPE_MX4) return 4 * r + (q ^ (r >> 2));
  return 128 * (q >> 1) + 8 * r + ((4 * (q & 1) + i) ^ (r >> 1));
}
// Load f of an operand: the lane's row, its first value (or byte) in the run, and
// the slot it goes to.
template <int kX>
__device__ __forceinline__ int x_row(int f) {
  const int lane = threadIdx.x & 63;
  return kX == SAS_TYPE_MX4 ? lane >> 2 : 8 * (f & 1) + (lane >> 3);
}
template <int kX>
__device__ __forceinline__ int x_at(int f) {
  const int lane = threadIdx.x & 63;
  return kX == SAS_TYPE_MX4 ? 16 * (lane & 3) : 64 * (f >> 1) + 8 * (lane & 7);
}
template <int kX>
__device__ __forceinline__ int x_put(int f, int r) {
  const int lane = threadIdx.x & 63;
  if constexpr (kX == SAS_TYPE_MX4) return 4 * r + ((lane & 3) ^ (r >> 2));
  return 128 * (f >> 1) + 8 * r + ((lane & 7) ^ (r >> 1));
}
template <int kX>
struct XPart {  // what a lane loads: an octet, or a block
  u32x4 v[kX == SAS_TYPE_F32 ? 2 : 1];
};
// From `at` on, of `size` values (bytes) a row has; zeros past them.
template <int kX>
__device__ __forceinline__ XPart<kX> x_load(const void *row, int at, int size) {
  XPart<kX> p;
  const u32x4 none = {0u, 0u, 0u, 0u};
  if constexpr (kX == SAS_TYPE_F32) {
    const u32x4a4 *src = reinterpret_cast<const u32x4a4 *>(static_cast<const float *>(row) + at);
    p.v[0] = at < size ? src[0] : none;
    p.v[1] = at < size ? src[1] : none;
  } else if constexpr (kX == SAS_TYPE_BF16) {
    p.v[0] = at < size ? *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(row) + at) : none;
  } else {
    p.v[0] = at < size ? *reinterpret_cast<const u32x4 *>(static_cast<const uint8_t *>(row) + at) : none;
  }
  return p;
}
// The bf16 operands of a part: itself, or its three pieces.
template <int kX>
__device__ __forceinline__ void x_pieces(const XPart<kX> &p, u32x4 (&o)[XOperand<kX>::kPieces]) {
  if constexpr (kX == SAS_TYPE_F32) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(p.v[i / 4][i % 4]);
    split_f32(v, o);
  } else {
    o[0] = p.v[0];
  }
}

// The sums of 16 rows x 16 NT outputs from the matrix layout to whole runs of a
// row's outputs, through LDS of the wave's own: f(row, column, 4 sums).
template <int NT>
constexpr int kStage = 16 * (16 * NT + 4);  // floats
template <int NT, typename F>
__device__ __forceinline__ void by_rows(float *stage, const f32x4 (&acc)[NT], F f) {
  const int lane = threadIdx.x & 63;
  constexpr int kPitch = 16 * NT + 4, kLanes = 4 * NT;
  wave_lds_sync();
#pragma unroll
  for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4 *>(stage + (lane & 15) * kPitch + 16 * t + 4 * (lane >> 4)) = acc[t];
  wave_lds_sync();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int i = 64 * n + lane, row = i / kLanes, col = 4 * (i % kLanes);
    f(row, col, *reinterpret_cast<const f32x4 *>(stage + row * kPitch + col));
  }
}

// Weight rows.  A super-run of 16 rows is 4 KB: loaded eight lanes a row, whole
// 128-byte lines (load k: rows 8 (k % 2) .., line k / 2 of the super-run), and
// turned into the matrix layout through LDS of the wave's own, laid out as a bf16
// operand's 16-byte slots are.
template <int NT>
struct WSuper {
  u32x4 c[4][NT];
  Scales s[NT];
};
template <int NT>
struct WRows {
  const uint8_t *codes[NT];   // of the tile's first row (uniform)
  const uint8_t *scales[NT];
  uint32_t at[NT][2];         // the lane's rows of a load, its chunk
  uint32_t scale_at[NT];      // the lane's row
  template <bool kDirect = false>
  __device__ __forceinline__ void set(const Mx4ProjArgs &a, int n0) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int n = n0 + 16 * t, first = min(n, a.out_dim - 1);
      codes[t] = a.w + (int64_t)first * a.w_stride;
      scales[t] = a.w_scales + (int64_t)first * a.w_scales_stride;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        at[t][h] = (uint32_t)(min(n + (kDirect ? lane & 15 : 8 * h + (lane >> 3)), a.out_dim - 1) - first) * (uint32_t)a.w_stride;
      scale_at[t] = (uint32_t)(min(n + (lane & 15), a.out_dim - 1) - first) * (uint32_t)a.w_scales_stride;
    }
  }
  // The same straight into the matrix layout: lane l block l / 16 of run k of row
  // l % 16 (half lines: for products that the matrix instructions bound).
  __device__ __forceinline__ void load_direct(WSuper<NT> &b, int s, int blocks) const {
#pragma unroll
    for (int t = 0; t < NT; ++t) b.s[t] = load_scales(scales[t] + scale_at[t], s, blocks);
#pragma unroll
    for (int k = 0; k < 4; ++k) load_direct_run(b, k, s, blocks);
  }
  __device__ __forceinline__ void load_direct_run(WSuper<NT> &b, int k, int s, int blocks) const {
    const uint32_t chunk = 16u * (uint32_t)min(16 * s + 4 * k + (int)((threadIdx.x & 63) >> 4), blocks - 1);
#pragma unroll
    for (int t = 0; t < NT; ++t) b.c[k][t] = *reinterpret_cast<const u32x4 *>(codes[t] + (at[t][0] + chunk));
  }
  // kOnce: no other wave reads these rows (nontemporal loads then)
  template <bool kOnce>
  __device__ __forceinline__ void load(WSuper<NT> &b, int s, int blocks) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int t = 0; t < NT; ++t) b.s[t] = load_scales(scales[t] + scale_at[t], s, blocks);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t chunk = 16u * (uint32_t)min(16 * s + 8 * (k >> 1) + (lane & 7), blocks - 1);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const u32x4 *src = reinterpret_cast<const u32x4 *>(codes[t] + (at[t][k & 1] + chunk));
        b.c[k][t] = kOnce ? __builtin_nontemporal_load(src) : *src;
      }
    }
  }
};
constexpr int kWSlots = 256;  // of a tile's super-run
template <int NT>
__device__ __forceinline__ void w_put(u32x4 *ws, const WSuper<NT> &b) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = 8 * (k & 1) + (lane >> 3);
#pragma unroll
    for (int t = 0; t < NT; ++t) ws[kWSlots * t + 128 * (k >> 1) + 8 * r + ((lane & 7) ^ (r >> 1))] = b.c[k][t];
  }
}
// Lane l: block l / 16 of run j of row l % 16.
__device__ __forceinline__ int w_get(int j) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  return 128 * (j >> 1) + 8 * r + ((4 * (j & 1) + q) ^ (r >> 1));
}

// Adds a run's products: c the tiles' blocks, ws their packed scales, x the run's
// operands in LDS, get the lane's slots in one, xscale the subtiles' scales.
template <int MT, int NT, int kX, int P, int kRunOf4>
__device__ __forceinline__ void add_run(const u32x4 (&c)[NT], const uint32_t (&ws)[NT], const u32x4 *x, const int (&get)[4],
                                        const uint32_t *xscale, f32x4 (&acc)[MT][NT]) {
  constexpr int kSlots = XOperand<kX>::kSlots;
  if constexpr (kX == SAS_TYPE_MX4) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const u32x4 xv = x[m * kSlots + get[0]];
      const uint32_t xs = xscale[64 * m];
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[m][t] = mfma4<kRunOf4>(c[t], ws[t], xv, xs, acc[m][t]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 wv[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) wv[t] = widen(c[t][i], scale_byte<kRunOf4>(ws[t]));
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int p = 0; p < P; ++p) {
          const u32x4 xv = x[(P * m + p) * kSlots + get[i]];
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[m][t] = mfma(wv[t], xv, acc[m][t]);
        }
    }
  }
}

// Few rows, hidden states that fit in LDS: every block holds all of them, and its
// waves take 16 NT outputs after another, their weight rows two super-runs
// ahead in registers; no barrier after the first.
// kPack: up to kMx4Few rows of f32, whose pieces are rows of one operand (row r's
// piece p is row kMx4Few p + r): a third of the products.
constexpr int kStreamWaves = 8;
constexpr int kStreamSlots = 128 * 1024 / 16;

template <int MT, int NT, int kX, bool kPack>
__global__ __launch_bounds__(64 * kStreamWaves, 2) void mx4_stream_kernel(const Mx4ProjArgs a) {
  using X = XOperand<kX>;
  constexpr int P = kPack ? 1 : X::kPieces, kSubs = MT * P;
  // the hidden states (MX4: then their scales, [super-run][subtile][lane])
  __shared__ u32x4 xs[kStreamSlots];
  __shared__ u32x4 wls[kStreamWaves][NT * kWSlots];
  static_assert(kStage<NT> * 4 <= NT * kWSlots * 16, "the sums fit where the weight rows were");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int blocks = (a.dim + kBlock - 1) / kBlock, supers = (blocks + 15) / 16, runs = 4 * supers;
  uint32_t *xsc = reinterpret_cast<uint32_t *>(xs + runs * kSubs * X::kSlots);
  const int waves = (int)gridDim.x * kStreamWaves, gw = wave * (int)gridDim.x + (int)blockIdx.x;
  const int groups = (a.out_dim + 16 * NT - 1) / (16 * NT);
  const int total = gw < groups ? (groups - gw + waves - 1) / waves * supers : 0;
  WRows<NT> w;
  int lg = gw, ls = 0;  // the next super-run to load
  w.set(a, 16 * NT * lg);
  // (past the last super-run the last again)
  auto load = [&](WSuper<NT> &b) __attribute__((always_inline)) {
    w.template load<true>(b, ls, blocks);
    if (++ls == supers) {
      if (lg + waves < groups) {
        lg += waves;
        ls = 0;
        w.set(a, 16 * NT * lg);
      } else {
        ls = supers - 1;
      }
    }
  };
  WSuper<NT> b0, b1;
  load(b0);
  load(b1);
  // the hidden states, zeros past dim and the last row
  {
    const int size = kX == SAS_TYPE_MX4 ? 16 * blocks : a.dim;
    const int64_t bytes = a.x_stride * (kX == SAS_TYPE_F32 ? 4 : kX == SAS_TYPE_BF16 ? 2 : 1);
    constexpr int kRunSize = kX == SAS_TYPE_MX4 ? 64 : kRun;
    for (int i = wave; i < MT * X::kLoads * runs; i += kStreamWaves) {
      const int f = i % X::kLoads, m = i / X::kLoads % MT, run = i / X::kLoads / MT;
      const int xr = x_row<kX>(f), row = 16 * m + xr;
      if (kPack && (f & 1)) continue;
      const XPart<kX> p = x_load<kX>(static_cast<const char *>(a.x) + (int64_t)min(row, a.rows - 1) * bytes, kRunSize * run + x_at<kX>(f),
                                     row < a.rows ? size : 0);
      u32x4 o[X::kPieces];
      x_pieces<kX>(p, o);
#pragma unroll
      for (int k = 0; k < X::kPieces; ++k) {
        if constexpr (kPack) {
          if (xr < kMx4Few) xs[run * X::kSlots + x_put<kX>(f, kMx4Few * k + xr)] = o[k];
        } else {
          xs[(run * kSubs + P * m + k) * X::kSlots + x_put<kX>(f, xr)] = o[k];
        }
      }
      if constexpr (kPack) {
        if (xr == kMx4Few) xs[run * X::kSlots + x_put<kX>(f, 15)] = u32x4{0u, 0u, 0u, 0u};
      }
    }
    if constexpr (kX == SAS_TYPE_MX4) {
      for (int i = wave; i < MT * supers; i += kStreamWaves) {
        const int m = i % MT, s = i / MT, row = min(16 * m + r, a.rows - 1);
        xsc[i * 64 + lane] = pack_scales(load_scales(a.x_scales + (int64_t)row * a.x_scales_stride, s, blocks), q, s, blocks);
      }
    }
  }
  int get[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) get[i] = x_get<kX>(i);
  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  lds_barrier();
  int g = gw, s = 0;
  u32x4 *wl = wls[wave];
  // a super-run out of b, which then takes the one two ahead
  auto compute = [&](WSuper<NT> &b) __attribute__((always_inline)) {
    uint32_t ws[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) ws[t] = pack_scales(b.s[t], q, s, blocks);
    wave_lds_sync();
    w_put<NT>(wl, b);
    __builtin_amdgcn_sched_barrier(0);
    load(b);
    wave_lds_sync();
    __builtin_amdgcn_sched_barrier(0);
    each_const<4>([&](auto jt) __attribute__((always_inline)) {
      constexpr int j = decltype(jt)::value;
      u32x4 c[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) c[t] = wl[kWSlots * t + w_get(j)];
      add_run<MT, NT, kX, P, j>(c, ws, xs + (4 * s + j) * kSubs * X::kSlots, get, xsc + s * MT * 64 + lane, acc);
    });
    if (++s == supers) {
      const int n0 = 16 * NT * g;
      float *stage = reinterpret_cast<float *>(wl);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        by_rows<NT>(stage, acc[m], [&](int row, int col, f32x4 v) __attribute__((always_inline)) {
          if constexpr (kPack) {
            if (row >= a.rows) return;
            const float *st = stage + row * (16 * NT + 4) + col;
            const f32x4 v1 = *reinterpret_cast<const f32x4 *>(st + kMx4Few * (16 * NT + 4));
            const f32x4 v2 = *reinterpret_cast<const f32x4 *>(st + 2 * kMx4Few * (16 * NT + 4));
            v = (v2 + v1) + v;
          }
          if (16 * m + row < a.rows) finish4(a, 16 * m + row, n0 + col, v);
        });
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
      s = 0;
      g += waves;
    }
  };
  int at = 0;
  for (; at + 2 <= total; at += 2) {
    compute(b0);
    compute(b1);
  }
  if (at < total) compute(b0);
}

// Whether the stream kernel's LDS holds the hidden states.
template <int MT, int kX, bool kPack>
bool stream_fits(const Mx4ProjArgs &a) {
  using X = XOperand<kX>;
  const int64_t supers = ((int64_t)a.dim + kSuper - 1) / kSuper;
  return supers * MT * (4 * (kPack ? 1 : X::kPieces) * X::kSlots + (kX == SAS_TYPE_MX4 ? 16 : 0)) <= kStreamSlots;
}

template <int MT, int NT, int kX, bool kPack>
void launch_stream(const Mx4ProjArgs &a, hipStream_t stream) {
  const int groups = (a.out_dim + 16 * NT - 1) / (16 * NT);
  const int blocks = groups < a.cus ? groups : a.cus;
  mx4_stream_kernel<MT, NT, kX, kPack><<<blocks, 64 * kStreamWaves, 0, stream>>>(a);
}

// Many outputs: WM x WN waves, a wave 16 MT rows x 16 NT outputs; the hidden
// states' chunks of kChunk runs in LDS, the next one on its way in registers,
// weight rows one super-run ahead in registers.
constexpr int kWideWaves = 8;
template <int MT, int WM, int NT, int kX>
struct Wide4 {
  static constexpr int kWN = kWideWaves / WM, kRows = 16 * MT * WM, kOuts = 16 * NT * kWN;
  static constexpr int S = MT * WM, P = XOperand<kX>::kPieces, kSubs = S * P;
  static constexpr int kChunk = kX == SAS_TYPE_MX4 ? 4 : kSubs <= 2 ? 4 : kSubs <= 4 ? 2 : 1;
  static constexpr int kXSlots = 2 * kChunk * kSubs * XOperand<kX>::kSlots;
  // Rows that bound the matrix instructions (WM > 1) take their weights straight.
  static constexpr bool kDirect = WM > 1;
  static constexpr int kWave = kDirect ? kStage<NT> / 4 : NT * kWSlots;  // 16-byte slots of a wave
  static constexpr int kLoads = S * XOperand<kX>::kLoads * kChunk;
  static constexpr int kMine = (kLoads + kWideWaves - 1) / kWideWaves;
};

template <int MT, int WM, int NT, int kX, bool kOnce>
__global__ __launch_bounds__(64 * kWideWaves, 2) void mx4_wide_kernel(const Mx4ProjArgs a) {
  using X = XOperand<kX>;
  using C = Wide4<MT, WM, NT, kX>;
  constexpr int P = C::P, S = C::S, kChunk = C::kChunk;
  __shared__ u32x4 xs[C::kXSlots];
  __shared__ u32x4 wls[kWideWaves][C::kWave];
  __shared__ uint32_t xsc[kX == SAS_TYPE_MX4 ? 2 * S * 64 : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4, wm = wave % WM, wn = wave / WM;
  const int mtiles = kOnce ? 1 : (a.rows + C::kRows - 1) / C::kRows;
  const int pos = xcd_run((int)blockIdx.x, (int)gridDim.x);
  const int m0 = (pos % mtiles) * C::kRows, n0 = (pos / mtiles) * C::kOuts + wn * 16 * NT;
  const int blocks = (a.dim + kBlock - 1) / kBlock, supers = (blocks + 15) / 16, chunks = supers * (4 / kChunk);
  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  WRows<NT> w;
  w.template set<C::kDirect>(a, n0);
  // This wave's loads of a chunk: load i = wave + 8 n is load f of operand (run,
  // subtile), in the order f, subtile, run (a subtile's f and, where a run has
  // as many loads as there are waves, its subtile are the wave's).
  static_assert(S == 1 || S == 2 || S == 4 || S == 8, "a power of two");
  constexpr int kFirst = X::kLoads == 4 ? 2 : 8;  // subtiles that the waves take together
  const int size = kX == SAS_TYPE_MX4 ? 16 * blocks : a.dim;
  constexpr int kSize = kX == SAS_TYPE_F32 ? 4 : kX == SAS_TYPE_BF16 ? 2 : 1, kRunSize = kX == SAS_TYPE_MX4 ? 64 : kRun;
  const int f = wave % X::kLoads, i0 = wave / X::kLoads;
  auto sub_of = [&](int n) { return (i0 + kFirst * n) % S; };
  auto run_of = [&](int n) { return (i0 + kFirst * n) / S; };
  constexpr int kXRows = S <= kFirst ? 1 : S / kFirst;  // different subtiles of a wave
  const char *xbase = static_cast<const char *>(a.x) + (int64_t)m0 * a.x_stride * kSize;
  uint32_t xrow[kXRows];
#pragma unroll
  for (int n = 0; n < kXRows; ++n)
    xrow[n] = (uint32_t)min(16 * sub_of(n) + x_row<kX>(f), a.rows - 1 - m0) * ((uint32_t)a.x_stride * kSize);
  const int xput = x_put<kX>(f, x_row<kX>(f));
  XPart<kX> x[C::kMine];
  Scales xsv;
  const uint8_t *xscale_row = kX == SAS_TYPE_MX4 ? a.x_scales + (int64_t)min(m0 + 16 * (wave % S) + r, a.rows - 1) * a.x_scales_stride : nullptr;
  auto load_x = [&](int chunk) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < C::kMine; ++n)
      x[n] = x_load<kX>(xbase + xrow[n % kXRows], kRunSize * (chunk * kChunk + run_of(n)) + x_at<kX>(f), size);
    if constexpr (kX == SAS_TYPE_MX4) {
      if (wave < S) xsv = load_scales(xscale_row, chunk, blocks);
    }
  };
  auto store_x = [&](int buf, int chunk) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < C::kMine; ++n) {
      if (C::kLoads % kWideWaves != 0 && wave + kWideWaves * n >= C::kLoads) continue;
      u32x4 o[X::kPieces];
      x_pieces<kX>(x[n], o);
#pragma unroll
      for (int p = 0; p < P; ++p) xs[((buf * kChunk + run_of(n)) * C::kSubs + P * sub_of(n) + p) * X::kSlots + xput] = o[p];
    }
    if constexpr (kX == SAS_TYPE_MX4) {
      if (wave < S) xsc[(buf * S + wave) * 64 + lane] = pack_scales(xsv, q, chunk, blocks);
    }
  };
  int get[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) get[i] = x_get<kX>(i);
  WSuper<NT> b;
  load_x(0);
  if constexpr (C::kDirect) w.load_direct(b, 0, blocks);
  else w.template load<kOnce>(b, 0, blocks);
  store_x(0, 0);
  lds_barrier();
  u32x4 *wl = wls[wave];
  for (int s = 0; s < supers; ++s) {
    uint32_t ws[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) ws[t] = pack_scales(b.s[t], q, s, blocks);
    const int ns = min(s + 1, supers - 1);
    if constexpr (C::kDirect) {
#pragma unroll
      for (int t = 0; t < NT; ++t) b.s[t] = load_scales(w.scales[t] + w.scale_at[t], ns, blocks);
    } else {
      wave_lds_sync();
      w_put<NT>(wl, b);
      __builtin_amdgcn_sched_barrier(0);
      load_x(min(s * (4 / kChunk) + 1, chunks - 1));
      w.template load<kOnce>(b, ns, blocks);
      wave_lds_sync();
      __builtin_amdgcn_sched_barrier(0);
    }
    each_const<4>([&](auto jt) __attribute__((always_inline)) {
      constexpr int j = decltype(jt)::value;
      const int chunk = s * (4 / kChunk) + j / kChunk, buf = chunk & 1;
      if constexpr ((C::kDirect || j != 0) && j % kChunk == 0) load_x(min(chunk + 1, chunks - 1));
      u32x4 c[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) c[t] = C::kDirect ? b.c[j][t] : wl[kWSlots * t + w_get(j)];
      if constexpr (C::kDirect) w.load_direct_run(b, j, ns, blocks);
      add_run<MT, NT, kX, P, j>(c, ws, xs + ((buf * kChunk + j % kChunk) * C::kSubs + P * MT * wm) * X::kSlots, get,
                                xsc + (buf * S + MT * wm) * 64 + lane, acc);
      if constexpr (j % kChunk == kChunk - 1) {
        __builtin_amdgcn_sched_barrier(0);
        store_x(buf ^ 1, min(chunk + 1, chunks - 1));
        lds_barrier();
      }
    });
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
    by_rows<NT>(reinterpret_cast<float *>(wl), acc[m], [&](int row, int col, f32x4 v) __attribute__((always_inline)) {
      const int at = m0 + 16 * (MT * wm + m) + row;
      if (at < a.rows) finish4(a, at, n0 + col, v);
    });
}

template <int MT, int WM, int NT, int kX>
void launch_wide(const Mx4ProjArgs &a, hipStream_t stream) {
  using C = Wide4<MT, WM, NT, kX>;
  const int mtiles = (a.rows + C::kRows - 1) / C::kRows, blocks = mtiles * ((a.out_dim + C::kOuts - 1) / C::kOuts);
  if (mtiles == 1) mx4_wide_kernel<MT, WM, NT, kX, true><<<blocks, 64 * kWideWaves, 0, stream>>>(a);
  else mx4_wide_kernel<MT, WM, NT, kX, false><<<blocks, 64 * kWideWaves, 0, stream>>>(a);
}

}  // namespace
}  // namespace sas
