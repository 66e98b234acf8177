// mx4_product.h - products with rows of MXFP4 values (gfx950): the kernels that
// sas_project_mx4 and the fused head share.
//
//   y[r][n] = cap(sum over k of x[r][k] w[n][k] (+ y[r][n]))
//
// A weight is element x scale, exact in bf16 (v_cvt_scalef32_pk_bf16_fp4 makes
// two of them), so its product with a bf16 value is exact in the matrix
// instructions' f32 sums; f32 hidden states are three bf16 pieces, 24 bits,
// three products.  Hidden states of MXFP4 take the scaled 4-bit matrix
// instruction: 128 values at the cost of bf16's 32, no conversions.
//
// Three kernels:
//   - mx4_split_kernel: few outputs.  Eight waves split dim, every load of a
//     call in flight together (1 x 2,560 x 2,560 4.8 us).  Also up to five f32 rows
//     of more than 4,096 values over wide outputs, far from their floor: one row x
//     5,120 x 151,936 270 us (413 MB, 1.5 TB/s), x 8,192 288, x 12,288 427.  And rows
//     further apart than the others' 32-bit offsets reach.
//   - mx4_stream_kernel: few rows, hidden states that fit in LDS.  Bound by the
//     weights' stream: one f32 row x 2,560 x 262,144 60 us (357 MB, 6.0 TB/s), 16
//     bf16 rows x 151,936 42, 16 MXFP4 rows 39, 61 MXFP4 rows x 4,096 x 11,007 12.7.
//   - mx4_wide_kernel: the rest.  2,048 x 4,096 x 4,096 bf16 56 us (1.23 PFLOP/s),
//     8,192 x 4,096 x 11,008 587 (1.26), the same of MXFP4 285 (2.6): a wave reads
//     all of a tile's hidden states from LDS, and waits for what it read; f32, three
//     products each, 2,048 x 4,096 x 4,096 161, 8,192 x 4,096 x 11,008 1,785; 128
//     bf16 rows x 2,560 x 262,144, capped, 160 us (1.07 PFLOP/s; 129 without loads
//     and results), 16 f32 rows x 151,936 63 (52).
// (Calls queued one behind another; a launch alone under the profiler takes about
// a tenth more, 61 MXFP4 rows 14.2 us.)
// What carried them: weight rows in whole 128-byte lines, nontemporal (half lines
// in the matrix layout: nontemporal 469 MB fetched for 357, 84 us for a head's
// row; cached 66; whole lines through LDS 60); one tile of 16 rows at a time, so
// that what a wave asks for lies together (two tiles 77 us, four 88); operands read
// a step ahead; one block of code a loop; bands of tiles for the L2.
#pragma once

#include "sas_product.h"

namespace sas {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef u32x4 u32x4a4 __attribute__((aligned(4)));

constexpr int kBlock = SAS_MX4_BLOCK;

// The f32 scale of byte s as the conversions take it.
__device__ __forceinline__ float scale_of(uint32_t s) { return __uint_as_float(s << 23); }

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

// A lane's scales of a super-run (blocks 16 s ..): lane l loads the l / 16-th of
// its row's four dwords; exchanged among the row's four lanes, each keeps byte
// l / 16 of every one, in the order of the runs.  No branches: the loops that
// use them stay one block, or the compiler moves all products behind the loads.
// (run: the first of the four)
__device__ __forceinline__ uint32_t load_scales_of(const uint8_t *row, int run, int blocks) {
  // (the dwords behind the last block's are not the row's)
  return *reinterpret_cast<const uint32_t *>(row + 4 * min(run + (int)((threadIdx.x & 63) >> 4), (blocks - 1) / 4));
}
template <bool kTail = true>
__device__ __forceinline__ uint32_t load_scales(const uint8_t *row, int s, int blocks) {
  if constexpr (!kTail) return *reinterpret_cast<const uint32_t *>(row + 16 * s + ((threadIdx.x & 63) >> 4 << 2));
  return load_scales_of(row, 4 * s, blocks);
}
// The bytes of a lane's runs that the row has blocks for.
__device__ __forceinline__ uint32_t scale_mask_of(int run, int blocks) {
  const int q = (threadIdx.x & 63) >> 4, n = min(max((blocks - 4 * run - q + 3) >> 2, 0), 4);
  return n == 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1u;
}
__device__ __forceinline__ uint32_t scale_mask(int s, int blocks) { return scale_mask_of(4 * s, blocks); }
// The others become 127 (1): what is there may be NaN.
template <bool kTail = true>
__device__ __forceinline__ uint32_t pack_scales(uint32_t mine, uint32_t mask) {
  const uint32_t q = (threadIdx.x & 63) >> 4, sel = 0x0C0C0400u + 0x0101u * q;
  const auto half = __builtin_amdgcn_permlane32_swap(mine, mine, false, false);
  const auto lo = __builtin_amdgcn_permlane16_swap(half[0], half[0], false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(half[1], half[1], false, false);
  const uint32_t a = __builtin_amdgcn_perm(lo[1], lo[0], sel), b = __builtin_amdgcn_perm(hi[1], hi[0], sel);
  const uint32_t p = __builtin_amdgcn_perm(b, a, 0x05040100u);
  return kTail ? (p & mask) | (0x7F7F7F7Fu & ~mask) : p;
}

// ---- the hidden states in LDS ----
//
// An operand: 16 rows x 128 values of bf16 (4 KB) in two halves of 64 values, a
// row's octets in the eight 16-byte slots from 8 r of its half on; or 16 rows x 64
// bytes of codes (1 KB), a row's blocks in the four slots from 4 r on.  LDS serves
// a 16-byte read 16 lanes at a time: lanes 0 .. 3, 12 .. 15, 20 .. 23 and 24 .. 27
// together, then the other 16 of the first 32, the upper half alike.  In these
// orders each such set meets every bank once.  (With octet o at o ^ r / 2, right
// for 16 lanes after another, SQ_LDS_BANK_CONFLICT was 40 % of the LDS's cycles.)
__device__ __forceinline__ int octet_slot(int o, int r) { return 8 * r + (((o & 3) << 1 | o >> 2) ^ (r >> 1)); }
__device__ __forceinline__ int block_slot(int c, int r) {
  const int t = r >> 2;  // 0 2 3 1
  return 4 * r + (c ^ ((t & 1) << 1) ^ (t >> 1) * 3);
}
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
  if constexpr (kX == SAS_TYPE_MX4) return block_slot(q, r);
  return 128 * (q >> 1) + octet_slot(4 * (q & 1) + i, r);
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
  if constexpr (kX == SAS_TYPE_MX4) return block_slot(lane & 3, r);
  return 128 * (f >> 1) + octet_slot(lane & 7, r);
}
template <int kX>
struct XPart {  // what a lane loads: an octet, or a block
  u32x4 v[kX == SAS_TYPE_F32 ? 2 : 1];
};
// A part, at p.
template <int kX>
__device__ __forceinline__ XPart<kX> x_load(const char *p) {
  XPart<kX> v;
  const u32x4a4 *src = reinterpret_cast<const u32x4a4 *>(p);
  if constexpr (kX == SAS_TYPE_F32) {
    v.v[0] = src[0];
    v.v[1] = src[1];
  } else {
    v.v[0] = *reinterpret_cast<const u32x4 *>(p);
  }
  return v;
}
template <int kX>
constexpr int kXSize = kX == SAS_TYPE_F32 ? 4 : kX == SAS_TYPE_BF16 ? 2 : 1;  // bytes
// Of `size` values (bytes) a row has, the part from `at` on is read here: its last
// one past them (no branch; x_pieces makes zeros of it).
template <int kX>
__device__ __forceinline__ int x_within(int at, int size) {
  return min(at, size - (kX == SAS_TYPE_MX4 ? 16 : 8));
}
// The operands of a part: itself, or its three pieces; zeros from `size` on.
template <int kX>
__device__ __forceinline__ void x_pieces(const XPart<kX> &p, int at, int size, u32x4 (&o)[XOperand<kX>::kPieces]) {
  const u32x4 none = {0u, 0u, 0u, 0u};
  if constexpr (kX == SAS_TYPE_F32) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(at < size ? p.v[i / 4][i % 4] : 0u);
    split_f32(v, o);
  } else {
    o[0] = at < size ? p.v[0] : none;
  }
}

// The sums of 16 rows x 16 NT outputs go out as whole runs of a row's outputs:
// from the matrix layout through LDS of the wave's own (kStage<NT> floats), 4 NT
// lanes a row.  n0: the first output; row0: the first row; value(row, col): the
// four sums.  (Addresses are a uniform base and 32 bits a lane: what is spent on
// them here is as much as on the products of 512 values.)
template <int NT>
constexpr int kStage = 16 * (16 * NT + 4);
constexpr int64_t kMaxOutStride = 1 << 25;  // elements: 16 rows of 4 bytes within 32 bits
constexpr int64_t kMaxXStride = 1 << 23;    // elements (MXFP4: bytes): 128 rows of 2 bytes, or 64 of 4
template <int NT, typename F>
__device__ __forceinline__ void put_rows(const Mx4ProjArgs &a, int row0, int n0, F value) {
  const int lane = threadIdx.x & 63;
  constexpr int kLanes = 4 * NT;
  const uint32_t size = a.out_bf16 ? 2u : 4u;
  char *base = static_cast<char *>(a.out) + ((int64_t)row0 * a.out_stride + n0) * size;
  const float inv = a.softcap > 0.0f ? 1.0f / a.softcap : 0.0f;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int i = 64 * n + lane, row = i / kLanes, col = 4 * (i % kLanes), left = a.out_dim - n0 - col;
    if (row0 + row >= a.rows || left <= 0) continue;
    f32x4 v = value(row, col);
    char *at = base + ((uint32_t)row * (uint32_t)a.out_stride + (uint32_t)col) * size;
    float *of = reinterpret_cast<float *>(at);
    uint16_t *ob = reinterpret_cast<uint16_t *>(at);
    if (a.accumulate) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < left) v[k] += a.out_bf16 ? __uint_as_float((uint32_t)ob[k] << 16) : of[k];
    }
    if (a.softcap > 0.0f) {
      const f32x4 u = v * inv;
      // (logits lie far below the cap as a rule: then half of tanh is all of it)
      // (of NaN it is NaN)
      if (__any(fmaxf(fmaxf(fabsf(u[0]), fabsf(u[1])), fmaxf(fabsf(u[2]), fabsf(u[3]))) >= 0.625f)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = a.softcap * tanh_fast(u[k]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = a.softcap * tanh_small(u[k]);
      }
    }
    // (nontemporal: the result is not read here)
    if (a.out_bf16) {
      const u16x4 p = __builtin_bit_cast(u16x4, __builtin_convertvector(v, bf16x4));
      if (left >= 4) {
        __builtin_nontemporal_store(p, reinterpret_cast<u16x4u *>(ob));
      } else {
#pragma unroll
        for (int k = 0; k < 3; ++k)
          if (k < left) ob[k] = p[k];
      }
    } else if (left >= 4) {
      __builtin_nontemporal_store(v, reinterpret_cast<f32x4u *>(of));
    } else {
#pragma unroll
      for (int k = 0; k < 3; ++k)
        if (k < left) of[k] = v[k];
    }
  }
}
template <int NT>
__device__ __forceinline__ void stage_rows(float *stage, const f32x4 (&acc)[NT]) {
  const int lane = threadIdx.x & 63;
  wave_lds_sync();
#pragma unroll
  for (int t = 0; t < NT; ++t)
    *reinterpret_cast<f32x4 *>(stage + (lane & 15) * (16 * NT + 4) + 16 * t + 4 * (lane >> 4)) = acc[t];
  wave_lds_sync();
}
template <int NT>
__device__ __forceinline__ f32x4 staged(const float *stage, int row, int col) {
  return *reinterpret_cast<const f32x4 *>(stage + row * (16 * NT + 4) + col);
}

// Weight rows.  A super-run of 16 rows is 4 KB: loaded eight lanes a row, whole
// 128-byte lines (load k: rows 8 (k % 2) .., line k / 2 of the super-run), and
// turned into the matrix layout, a line of each row at a time, through LDS of the
// wave's own, laid out as a bf16 operand's 16-byte slots are.
template <int NT>
struct WSuper {
  u32x4 c[4][NT];
  uint32_t s[NT];
};
template <int NT>
struct WRows {
  const uint8_t *codes[NT];   // of the tile's first row (uniform)
  const uint8_t *scales[NT];
  uint32_t at[NT][2];         // the lane's rows of a load, its chunk
  uint32_t scale_at[NT];      // the lane's row
  __device__ __forceinline__ void set(const Mx4ProjArgs &a, int n0) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int n = n0 + 16 * t, first = min(n, a.out_dim - 1);
      codes[t] = a.w + (int64_t)first * a.w_stride;
      scales[t] = a.w_scales + (int64_t)first * a.w_scales_stride;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        at[t][h] = (uint32_t)(min(n + 8 * h + (lane >> 3), a.out_dim - 1) - first) * (uint32_t)a.w_stride;
      scale_at[t] = (uint32_t)(min(n + (lane & 15), a.out_dim - 1) - first) * (uint32_t)a.w_scales_stride;
    }
  }
  // kOnce: no other wave reads these rows (nontemporal loads then)
  template <bool kOnce, bool kTail = true>
  __device__ __forceinline__ void load(WSuper<NT> &b, int s, int blocks) const {
    const uint32_t lane = threadIdx.x & 63;
    load_s<kTail>(b.s, s, blocks);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint8_t *p = kTail ? codes[t] + (at[t][k & 1] + 16u * (uint32_t)min(16 * s + 8 * (k >> 1) + (int)(lane & 7), blocks - 1))
                                 : codes[t] + 256 * s + (at[t][k & 1] + 16u * (lane & 7)) + 128 * (k >> 1);
        const u32x4 *src = reinterpret_cast<const u32x4 *>(p);
        b.c[k][t] = kOnce ? __builtin_nontemporal_load(src) : *src;
      }
    }
  }
  template <bool kTail>
  __device__ __forceinline__ void load_s(uint32_t (&v)[NT], int s, int blocks) const {
#pragma unroll
    for (int t = 0; t < NT; ++t) v[t] = load_scales<kTail>(scales[t] + scale_at[t], s, blocks);
  }
};
constexpr int kWSlots = 128;  // of a tile's line
template <int NT>
__device__ __forceinline__ void w_put(u32x4 *ws, const WSuper<NT> &b, int line) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = 8 * h + (lane >> 3);
#pragma unroll
    for (int t = 0; t < NT; ++t) ws[kWSlots * t + 8 * r + ((lane & 7) ^ (r >> 1))] = b.c[2 * line + h][t];
  }
}
// Lane l: block l / 16 of run j of row l % 16.
__device__ __forceinline__ int w_get(int j) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  return 8 * r + ((4 * (j & 1) + q) ^ (r >> 1));
}

// Adds a run's products: c the tiles' blocks, ws their packed scales, x the run's
// operands in LDS, get the lane's slots in one, xscale the subtiles' scales.
template <int MT, int NT, int kX, int kRunOf4>
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
      for (int m = 0; m < MT; ++m) {
        const u32x4 xv = x[m * kSlots + get[i]];
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[m][t] = mfma(wv[t], xv, acc[m][t]);
      }
    }
  }
}

// Few outputs: eight waves split dim for the same 16 NT outputs of 16 MT rows, all
// operands straight from memory, kFlight runs' loads together; their sums meet in
// LDS in a fixed order.
constexpr int kSplitWaves = 8;

template <int MT, int NT, int kX>
__global__ __launch_bounds__(64 * kSplitWaves, 2) void mx4_split_kernel(const Mx4ProjArgs a) {
  using X = XOperand<kX>;
  constexpr int P = X::kPieces, kOctets = kX == SAS_TYPE_MX4 ? 1 : 4;
  constexpr int kFlight = kX == SAS_TYPE_MX4 ? 4 : MT == 1 && kX == SAS_TYPE_BF16 ? 4 : MT == 1 ? 2 : 1;
  __shared__ f32x4 part[kSplitWaves][MT * NT][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int mtiles = (a.rows + 16 * MT - 1) / (16 * MT);
  const int pos = xcd_run((int)blockIdx.x, (int)gridDim.x);
  const int m0 = (pos % mtiles) * 16 * MT, n0 = (pos / mtiles) * 16 * NT;
  const int blocks = (a.dim + kBlock - 1) / kBlock, runs = (blocks + 3) / 4;
  const int g0 = runs * wave / kSplitWaves, g1 = runs * (wave + 1) / kSplitWaves;
  const int size = kX == SAS_TYPE_MX4 ? 16 * blocks : a.dim;
  const uint8_t *wr[NT], *wsr[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t row = min(n0 + 16 * t + r, a.out_dim - 1);
    wr[t] = a.w + row * a.w_stride;
    wsr[t] = a.w_scales + row * a.w_scales_stride;
  }
  const char *xr[MT];
  const uint8_t *xsr[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t row = min(m0 + 16 * m + r, a.rows - 1);
    xr[m] = static_cast<const char *>(a.x) + row * a.x_stride * kXSize<kX>;
    xsr[m] = kX == SAS_TYPE_MX4 ? a.x_scales + row * a.x_scales_stride : nullptr;
  }
  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int g4 = g0; g4 < g1; g4 += 4) {
    uint32_t ws[NT], xs[MT];
#pragma unroll
    for (int t = 0; t < NT; ++t) ws[t] = load_scales_of(wsr[t], g4, blocks);
#pragma unroll
    for (int m = 0; m < MT; ++m)
      if constexpr (kX == SAS_TYPE_MX4) xs[m] = load_scales_of(xsr[m], g4, blocks);
    each_const<4 / kFlight>([&](auto part_of) __attribute__((always_inline)) {
      const int g = g4 + kFlight * decltype(part_of)::value;
      u32x4 w[kFlight][NT];
      XPart<kX> x[kFlight][MT][kOctets];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        // (past the wave's last run, and the row's last block, what is there again:
        // x_pieces makes zeros of the hidden states)
        const int b = min(4 * min(g + u, g1 - 1) + q, blocks - 1);
#pragma unroll
        for (int t = 0; t < NT; ++t) w[u][t] = *reinterpret_cast<const u32x4 *>(wr[t] + 16 * b);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
          for (int i = 0; i < kOctets; ++i) {
            const int at = kX == SAS_TYPE_MX4 ? 16 * b : kBlock * b + 8 * i;
            x[u][m][i] = x_load<kX>(xr[m] + (int64_t)x_within<kX>(at, size) * kXSize<kX>);
          }
        }
      }
      if constexpr (decltype(part_of)::value == 0) {
        // (of the wave's own runs: behind them are the last one's codes again, and
        // under another block's scale they may pass bf16's range, times 0 NaN)
        const uint32_t mask = scale_mask_of(g4, min(blocks, 4 * g1));
#pragma unroll
        for (int t = 0; t < NT; ++t) ws[t] = pack_scales(ws[t], mask);
#pragma unroll
        for (int m = 0; m < MT; ++m)
          if constexpr (kX == SAS_TYPE_MX4) xs[m] = pack_scales(xs[m], mask);
      }
      each_const<kFlight>([&](auto ut) __attribute__((always_inline)) {
        constexpr int u = decltype(ut)::value, j = kFlight * decltype(part_of)::value + u;
        const int b = 4 * (g + u) + q;
        const bool in = g + u < g1 && b < blocks;
#pragma unroll
        for (int i = 0; i < kOctets; ++i) {
          u32x4 wv[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if constexpr (kX == SAS_TYPE_MX4) wv[t] = w[u][t];
            else wv[t] = widen(w[u][t][i], scale_byte<j>(ws[t]));
          }
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            u32x4 o[P];
            x_pieces<kX>(x[u][m][i], in ? (kX == SAS_TYPE_MX4 ? 16 * b : kBlock * b + 8 * i) : size, size, o);
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                if constexpr (kX == SAS_TYPE_MX4) acc[m][t] = mfma4<j>(wv[t], ws[t], o[p], xs[m], acc[m][t]);
                else acc[m][t] = mfma(wv[t], o[p], acc[m][t]);
              }
          }
        }
      });
    });
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][m * NT + t][lane] = acc[m][t];
  __syncthreads();
  for (int i = wave; i < MT * NT; i += kSplitWaves) {
    f32x4 v = part[0][i][lane];
#pragma unroll
    for (int k = 1; k < kSplitWaves; ++k) v = v + part[k][i][lane];
    const int row = m0 + 16 * (i / NT) + r;
    if (row < a.rows) finish4(a, row, n0 + 16 * (i % NT) + 4 * q, v);
  }
}

// Few outputs: the split kernel, where it fills the chip once at most and dim is
// more than two super-runs; then the waves of a block share dim, and all of a
// call's loads are one latency.  The wide kernel's blocks walk along dim.  Over
// 440 shapes (8 to 2,048 rows, 256 to 32,768 outputs of 512 to 8,192 values; up to
// five f32 rows, which follow the same rule, were not among them), split / wide, us: bf16, 16 rows x 2,560 x 4,096 7 / 8, x 16,384 15 / 10; 128 x
// 2,560 x 4,096 23 / 27, x 8,192 43 / 27; 128 x 8,192 x 4,096 41 / 76; 64 x 512 x
// 4,096 11 / 7; MXFP4, 64 x 8,192 x 4,096 17 / 23, x 16,384 34 / 30.
template <int MT, int NT>
inline bool split_fits(const Mx4ProjArgs &a) {
  return a.dim > 2 * kSuper && (int64_t)((a.rows + 16 * MT - 1) / (16 * MT)) * (((int64_t)a.out_dim + 16 * NT - 1) / (16 * NT)) <= a.cus;
}

// A launch holds fewer than 2^32 threads, 512 a block here: launch(part, groups)
// for parts of the outputs that take 2^22 blocks of `outs` of them at most.
template <typename F>
void in_parts(const Mx4ProjArgs &a, int mtiles, int outs, F launch) {
  static_assert((SAS_MAX_PROJECT_ROWS + 15) / 16 <= 1 << 22, "a part of one block's outputs at least");
  const int64_t most = (int64_t)((1 << 22) / mtiles) * outs;
  for (int64_t n = 0; n < a.out_dim; n += most) {
    Mx4ProjArgs part = a;
    part.w += n * a.w_stride;
    part.w_scales += n * a.w_scales_stride;
    part.out = static_cast<char *>(a.out) + n * (a.out_bf16 ? 2 : 4);
    part.out_dim = (int32_t)(a.out_dim - n < most ? a.out_dim - n : most);
    launch(part, (part.out_dim + outs - 1) / outs);
  }
}

template <int MT, int NT, int kX>
void launch_split(const Mx4ProjArgs &a, hipStream_t stream) {
  const int mtiles = (a.rows + 16 * MT - 1) / (16 * MT);
  in_parts(a, mtiles, 16 * NT, [&](const Mx4ProjArgs &part, int groups) {
    mx4_split_kernel<MT, NT, kX><<<mtiles * groups, 64 * kSplitWaves, 0, stream>>>(part);
  });
}

// Few rows, hidden states that fit in LDS: every block holds all of them, and its
// waves take 16 NT outputs after another, their weight rows two super-runs
// ahead in registers; no barrier after the first.
// f32 hidden states are packed: up to kMx4Few rows, whose pieces are rows of one
// operand (row r's piece p is row kMx4Few p + r): a third of the products.
// (Twelve waves against eight: 16 bf16 rows x 2,560 x 151,936 42.9 / 44.8 us, a
// head's row 59.8 / 60.6.)
constexpr int kStreamWaves = 12;
constexpr int kStreamSlots = 136 * 1024 / 16;

template <int MT, int NT, int kX>
__global__ __launch_bounds__(64 * kStreamWaves, 3) void mx4_stream_kernel(const Mx4ProjArgs a) {
  using X = XOperand<kX>;
  constexpr bool kPack = kX == SAS_TYPE_F32;
  static_assert(!kPack || MT == 1, "packed rows are one operand");
  // the hidden states (MX4: then their scales, [super-run][subtile][lane])
  __shared__ u32x4 xs[kStreamSlots];
  __shared__ u32x4 wls[kStreamWaves][NT * kWSlots];
  static_assert(kStage<NT> * 4 <= NT * kWSlots * 16, "the sums fit where the weight rows were");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15;
  const int blocks = (a.dim + kBlock - 1) / kBlock, supers = (blocks + 15) / 16, runs = 4 * supers;
  uint32_t *xsc = reinterpret_cast<uint32_t *>(xs + runs * MT * X::kSlots);
  const int waves = (int)gridDim.x * kStreamWaves, gw = wave * (int)gridDim.x + (int)blockIdx.x;
  const int groups = (a.out_dim + 16 * NT - 1) / (16 * NT);
  const int total = gw < groups ? (groups - gw + waves - 1) / waves * supers : 0;
  WRows<NT> w;
  int lg = gw, ls = 0;  // the super-run to load
  w.set(a, 16 * NT * lg);
  // (past the last super-run the last again)
  auto advance = [&] {
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
  w.template load<true>(b0, ls, blocks);
  advance();
  w.template load<true>(b1, ls, blocks);
  // the hidden states, zeros past dim (rows past the last: the last again)
  {
    const int size = kX == SAS_TYPE_MX4 ? 16 * blocks : a.dim;
    const int64_t bytes = a.x_stride * kXSize<kX>;
    constexpr int kRunSize = kX == SAS_TYPE_MX4 ? 64 : kRun;
    for (int i = wave; i < MT * X::kLoads * runs; i += kStreamWaves) {
      const int f = i % X::kLoads, m = i / X::kLoads % MT, run = i / X::kLoads / MT;
      const int xr = x_row<kX>(f), row = 16 * m + xr;
      if (kPack && (f & 1)) continue;
      const int at = kRunSize * run + x_at<kX>(f);
      const XPart<kX> p = x_load<kX>(static_cast<const char *>(a.x) + (int64_t)min(row, a.rows - 1) * bytes +
                                     (int64_t)x_within<kX>(at, size) * kXSize<kX>);
      u32x4 o[X::kPieces];
      x_pieces<kX>(p, at, size, o);
      if constexpr (kPack) {
#pragma unroll
        for (int k = 0; k < X::kPieces; ++k)
          if (xr < kMx4Few) xs[run * X::kSlots + x_put<kX>(f, kMx4Few * k + xr)] = o[k];
        if (xr == kMx4Few) xs[run * X::kSlots + x_put<kX>(f, 15)] = u32x4{0u, 0u, 0u, 0u};
      } else {
        xs[(run * MT + m) * X::kSlots + x_put<kX>(f, xr)] = o[0];
      }
    }
    if constexpr (kX == SAS_TYPE_MX4) {
      for (int i = wave; i < MT * supers; i += kStreamWaves) {
        const int m = i % MT, s = i / MT, row = min(16 * m + r, a.rows - 1);
        xsc[i * 64 + lane] = pack_scales(load_scales(a.x_scales + (int64_t)row * a.x_scales_stride, s, blocks), scale_mask(s, blocks));
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
    advance();  // (not behind a product: see the wide kernel)
    uint32_t ws[NT];
    const uint32_t mask = scale_mask(s, blocks);
#pragma unroll
    for (int t = 0; t < NT; ++t) ws[t] = pack_scales(b.s[t], mask);
    each_const<4>([&](auto jt) __attribute__((always_inline)) {
      constexpr int j = decltype(jt)::value;
      if constexpr (j % 2 == 0) {
        wave_lds_sync();
        w_put<NT>(wl, b, j / 2);
        if constexpr (j == 2) {
          __builtin_amdgcn_sched_barrier(0);
          w.template load<true>(b, ls, blocks);
        }
        wave_lds_sync();
        __builtin_amdgcn_sched_barrier(0);
      }
      u32x4 c[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) c[t] = wl[kWSlots * t + w_get(j)];
      add_run<MT, NT, kX, j>(c, ws, xs + (4 * s + j) * MT * X::kSlots, get, xsc + s * MT * 64 + lane, acc);
    });
    if (++s == supers) {
      const int n0 = 16 * NT * g;
      float *stage = reinterpret_cast<float *>(wl);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        stage_rows<NT>(stage, acc[m]);
        put_rows<NT>(a, 16 * m, n0, [&](int row, int col) __attribute__((always_inline)) {
          f32x4 v = staged<NT>(stage, row, col);
          if constexpr (kPack) v = (staged<NT>(stage, row + 2 * kMx4Few, col) + staged<NT>(stage, row + kMx4Few, col)) + v;
          return v;
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
template <int MT, int kX>
bool stream_fits(const Mx4ProjArgs &a) {
  const int64_t supers = ((int64_t)a.dim + kSuper - 1) / kSuper;
  return supers * MT * (4 * XOperand<kX>::kSlots + (kX == SAS_TYPE_MX4 ? 16 : 0)) <= kStreamSlots;
}

template <int MT, int NT, int kX>
void launch_stream(const Mx4ProjArgs &a, hipStream_t stream) {
  const int groups = (a.out_dim + 16 * NT - 1) / (16 * NT);
  const int blocks = groups < a.cus ? groups : a.cus;
  mx4_stream_kernel<MT, NT, kX><<<blocks, 64 * kStreamWaves, 0, stream>>>(a);
}

// Many outputs: eight waves share the hidden states of 16 MT rows and take 16 NT
// outputs each; the hidden states' chunks of kChunk runs in LDS, the next one on
// its way in registers, weight rows one super-run ahead in registers.  kOnce: one
// tile has all rows, and a block takes one group of outputs after another, its
// loads going on across them.
// A step is one operand of each subtile: its products come with the reads of the
// next step's operands, so that no product waits for LDS; the next chunk is
// stored half-way, and the barrier that shows it stands before the last step
// (2,048 x 4,096 x 4,096 bf16 67 -> 59 us, with the loop free of branches, cheap
// addresses and bands of tiles; MXFP4 115 -> 27).  A matrix instruction leaves room
// for two others beside it (16 cycles, or 8 and 4 for each of them): the
// conversions are one, what goes beyond costs.
constexpr int kWideWaves = 8;
template <int MT, int NT, int kX>
struct Mx4Wide {
  static constexpr int kRows = 16 * MT, kOuts = 16 * NT * kWideWaves;
  static constexpr int P = XOperand<kX>::kPieces, kSubs = MT * P;
  static constexpr int kChunk = kX == SAS_TYPE_MX4 ? 4 : kSubs <= 2 ? 4 : kSubs <= 4 ? 2 : 1;
  static constexpr int kXSlots = 2 * kChunk * kSubs * XOperand<kX>::kSlots;
  static constexpr int kWave = NT * kWSlots + kStage<NT> / 4;  // 16-byte slots of a wave: weight rows, sums
  static constexpr int kLoads = MT * XOperand<kX>::kLoads * kChunk;
  static constexpr int kMine = (kLoads + kWideWaves - 1) / kWideWaves;
  static constexpr int kRunSteps = kX == SAS_TYPE_MX4 ? 1 : 4;   // operands of a run
  static constexpr int kChunkSteps = kChunk * kRunSteps;
};

// (8,192 x 4,096 x 11,008, MXFP4: bands of 4 tiles 283 us, 8 301, all rows 313;
// bf16: 4 613, 8 623, all rows 680)
constexpr int kTileRows = 4;

template <int MT, int NT, int kX, bool kOnce, bool kTail>
__global__ __launch_bounds__(64 * kWideWaves, 2) void mx4_wide_kernel(const Mx4ProjArgs a) {
  using X = XOperand<kX>;
  using C = Mx4Wide<MT, NT, kX>;
  constexpr int P = C::P, kChunk = C::kChunk, kRunSteps = C::kRunSteps, kChunkSteps = C::kChunkSteps;
  __shared__ u32x4 xs[C::kXSlots];
  __shared__ u32x4 wls[kWideWaves][C::kWave];
  __shared__ uint32_t xsc[kX == SAS_TYPE_MX4 ? 2 * MT * 64 : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15;
  const int groups = (a.out_dim + C::kOuts - 1) / C::kOuts;
  const int mtiles = kOnce ? 1 : (a.rows + C::kRows - 1) / C::kRows;
  const int pos = kOnce ? (int)blockIdx.x : xcd_run((int)blockIdx.x, (int)gridDim.x);
  // tiles in the order of kTileRows of them by all groups: the 32 blocks that an
  // XCD runs at a time share rows and weights out of its L2
  int mt = 0, g = pos;
  if constexpr (!kOnce) {
    const int band = pos / (kTileRows * groups), at = pos % (kTileRows * groups);
    const int rows = min(mtiles - kTileRows * band, kTileRows);
    mt = kTileRows * band + at % rows;
    g = at / rows;
  }
  const int m0 = mt * C::kRows, gstep = kOnce ? (int)gridDim.x : groups;
  const int blocks = (a.dim + kBlock - 1) / kBlock, supers = (blocks + 15) / 16, chunks = supers * (4 / kChunk);
  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  WRows<NT> w;
  int lg = g, ls = 0;  // the super-run to load
  w.set(a, lg * C::kOuts + wave * 16 * NT);
  // (past the last one the last group's first again)
  auto advance = [&] {
    if (++ls == supers) {
      ls = 0;
      if (lg + gstep < groups) {
        lg += gstep;
        w.set(a, lg * C::kOuts + wave * 16 * NT);
      }
    }
  };
  // This wave's loads of a chunk: load i = wave + 8 n is load f of operand (run,
  // subtile), in the order f, subtile, run (a subtile's f and, where a run has
  // as many loads as there are waves, its subtile are the wave's).
  static_assert(MT == 1 || MT == 2 || MT == 4 || MT == 8, "a power of two");
  constexpr int kFirst = X::kLoads == 4 ? 2 : 8;  // subtiles that the waves take together
  const int size = kX == SAS_TYPE_MX4 ? 16 * blocks : a.dim;
  constexpr int kSize = kXSize<kX>, kRunSize = kX == SAS_TYPE_MX4 ? 64 : kRun;
  // (fewer loads than waves: the same again)
  const int f = wave % X::kLoads, i0 = wave % C::kLoads / X::kLoads;
  auto sub_of = [&](int n) { return (i0 + kFirst * n) % MT; };
  auto run_of = [&](int n) { return (i0 + kFirst * n) / MT; };
  constexpr int kXRows = MT <= kFirst ? 1 : MT / kFirst;  // different subtiles of a wave
  const char *xbase = static_cast<const char *>(a.x) + (int64_t)m0 * a.x_stride * kSize;
  uint32_t xrow[kXRows];
#pragma unroll
  for (int n = 0; n < kXRows; ++n)
    xrow[n] = (uint32_t)min(16 * sub_of(n) + x_row<kX>(f), a.rows - 1 - m0) * ((uint32_t)a.x_stride * kSize);
  const int xput = x_put<kX>(f, x_row<kX>(f));
  XPart<kX> x[C::kMine];
  uint32_t xsv = 0;
  const uint8_t *xscale_row = kX == SAS_TYPE_MX4 ? a.x_scales + (int64_t)min(m0 + 16 * (wave % MT) + r, a.rows - 1) * a.x_scales_stride : nullptr;
  auto x_first = [&](int chunk, int n) { return kRunSize * (chunk * kChunk + run_of(n)) + x_at<kX>(f); };
  auto load_x = [&](int chunk) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < C::kMine; ++n)
      x[n] = kTail ? x_load<kX>(xbase + (xrow[n % kXRows] + (uint32_t)(x_within<kX>(x_first(chunk, n), size) * kSize)))
                   : x_load<kX>(xbase + (int64_t)chunk * (kRunSize * kChunk * kSize) + (xrow[n % kXRows] + (uint32_t)(x_first(0, n) * kSize)));
    if constexpr (kX == SAS_TYPE_MX4) xsv = load_scales<kTail>(xscale_row, chunk, blocks);
  };
  auto store_x = [&](int buf, int chunk) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < C::kMine; ++n) {
      u32x4 o[X::kPieces];
      x_pieces<kX>(x[n], kTail ? x_first(chunk, n) : 0, kTail ? size : 1, o);
#pragma unroll
      for (int p = 0; p < P; ++p) xs[((buf * kChunk + run_of(n)) * C::kSubs + P * sub_of(n) + p) * X::kSlots + xput] = o[p];
    }
    if constexpr (kX == SAS_TYPE_MX4) xsc[(buf * MT + wave % MT) * 64 + lane] = pack_scales<kTail>(xsv, scale_mask(chunk, blocks));
  };
  auto after = [&](int chunk) { return chunk + 1 == chunks ? 0 : chunk + 1; };
  int get[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) get[i] = x_get<kX>(i);
  u32x4 *wl = wls[wave];
  // the operands of the next step, as they are read: hidden states, a run's
  // weights, MX4: a super-run's scales of the hidden states
  u32x4 xf[P * MT], c[NT];
  uint32_t xscale[MT];
  auto read_x = [&](int buf, int run, int i, int n) __attribute__((always_inline)) {
    xf[n] = xs[((buf * kChunk + run) * C::kSubs + n) * X::kSlots + get[i]];
  };
  auto read_c = [&](int j) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < NT; ++t) c[t] = wl[kWSlots * t + w_get(j)];
  };
  // A line of the weight rows into LDS, and the next super-run's loads once the
  // second one is there.
  WSuper<NT> b;
  auto line = [&](int l) __attribute__((always_inline)) {
    wave_lds_sync();
    w_put<NT>(wl, b, l);
    if (l == 1) w.template load<kOnce, kTail>(b, ls, blocks);
    wave_lds_sync();
  };
  load_x(0);
  w.template load<kOnce, kTail>(b, ls, blocks);
  store_x(0, 0);
  load_x(after(0));
  lds_barrier();
#pragma unroll
  for (int n = 0; n < P * MT; ++n) read_x(0, 0, 0, n);
  if constexpr (kX == SAS_TYPE_MX4) {
#pragma unroll
    for (int m = 0; m < MT; ++m) xscale[m] = xsc[m * 64 + lane];
  }
  line(0);
  read_c(0);
  int first = 0;  // the buffer of the super-run's first chunk
  for (; g < groups; g += gstep) {
    for (int s = 0; s < supers; ++s) {
      // (here: behind the products, its branch would have the compiler move them
      // past it, and all their operands would have to wait in registers)
      advance();
      uint32_t ws[NT];
      const uint32_t mask = scale_mask(s, blocks);
#pragma unroll
      for (int t = 0; t < NT; ++t) ws[t] = pack_scales<kTail>(b.s[t], mask);
      each_const<4 * kRunSteps>([&](auto st) __attribute__((always_inline)) {
        // step i of run j, the e-th of its chunk; the next one: step i2 of run j2
        constexpr int step = decltype(st)::value, j = step / kRunSteps, i = step % kRunSteps, e = step % kChunkSteps;
        constexpr int j2 = (step + 1) / kRunSteps % 4, i2 = (step + 1) % kRunSteps;
        const int buf = (first + j / kChunk) & 1, chunk = s * (4 / kChunk) + j / kChunk;
        // the chunk after this one is in registers: into the other buffer, whose
        // last reads lie before the barrier of the chunk before
        if constexpr (e == kChunkSteps / 2 - 1) {
          const int next = after(chunk);
          store_x(buf ^ 1, next);
          load_x(after(next));
        }
        u32x4 wv[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if constexpr (kX == SAS_TYPE_MX4) wv[t] = c[t];
          else wv[t] = widen(c[t][i], scale_byte<j>(ws[t]));
        }
        if constexpr (i2 == 0) {
          if constexpr (j2 % 2 == 0) line(j2 / 2);
          read_c(j2);
        }
        const int buf2 = e == kChunkSteps - 1 ? buf ^ 1 : buf;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          uint32_t xv = 0;
          if constexpr (kX == SAS_TYPE_MX4) {
            xv = xscale[m];
            if constexpr (step == 3) xscale[m] = xsc[(buf2 * MT + m) * 64 + lane];
          }
#pragma unroll
          for (int p = 0; p < P; ++p) {
            const u32x4 o = xf[P * m + p];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              if constexpr (kX == SAS_TYPE_MX4) acc[m][t] = mfma4<j>(wv[t], ws[t], o, xv, acc[m][t]);
              else acc[m][t] = mfma(wv[t], o, acc[m][t]);
            }
            read_x(buf2, j2 % kChunk, i2, P * m + p);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (e == kChunkSteps - 2) lds_barrier();
      });
      first = (first + 4 / kChunk) & 1;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float *stage = reinterpret_cast<float *>(wl + NT * kWSlots);
      stage_rows<NT>(stage, acc[m]);
      put_rows<NT>(a, m0 + 16 * m, g * C::kOuts + wave * 16 * NT,
                   [&](int row, int col) __attribute__((always_inline)) { return staged<NT>(stage, row, col); });
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
}

// Whether calls with more rows than one tile's come here (launch_products).
template <int MT, int kX>
constexpr bool kManyTiles = MT == 8 || (MT == 4 && kX == SAS_TYPE_F32);

template <int MT, int NT, int kX>
void launch_wide(const Mx4ProjArgs &a, hipStream_t stream) {
  using C = Mx4Wide<MT, NT, kX>;
  const int mtiles = (a.rows + C::kRows - 1) / C::kRows;
  in_parts(a, mtiles, C::kOuts, [&](const Mx4ProjArgs &part, int groups) {
    // whole super-runs have no blocks to mask
    const bool whole = a.dim % kSuper == 0;
    if constexpr (kManyTiles<MT, kX>) {
      if (mtiles > 1) {
        if (whole) mx4_wide_kernel<MT, NT, kX, false, false><<<mtiles * groups, 64 * kWideWaves, 0, stream>>>(part);
        else mx4_wide_kernel<MT, NT, kX, false, true><<<mtiles * groups, 64 * kWideWaves, 0, stream>>>(part);
        return;
      }
    }
    const int blocks = groups < a.cus ? groups : a.cus;
    if (whole) mx4_wide_kernel<MT, NT, kX, true, false><<<blocks, 64 * kWideWaves, 0, stream>>>(part);
    else mx4_wide_kernel<MT, NT, kX, true, true><<<blocks, 64 * kWideWaves, 0, stream>>>(part);
  });
}

}  // namespace
}  // namespace sas
