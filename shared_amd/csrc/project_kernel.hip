// project_kernel.hip - a shared projection with the low-rank adapters of many
// requests beside it (gfx950).
//
//   y[r] = cap(W x[r] + s[a] B[a] (A[a] x[r])),  a = row_adapter[r]
//
// Two launches:
//   1. proj_inner_kernel: h[r] = s[a] A[a] x[r], f32, stored as three bf16
//      pieces (8 + 8 + 8 bits of the f32 significand, cut, not rounded: their
//      sum is the f32 value); f32 hidden states are stored as three pieces
//      too.  Products of bf16 pieces are exact in the f32 sums of the matrix
//      instructions, so f32 inputs keep all their bits.
//   2. proj_rows_kernel: the rows' products with W, then with B of each
//      adapter among a subtile's 16 rows, each adapter in sums of its own that
//      only its rows add: a value that is not finite stays with its adapter.
#include "sas_device.h"
#include "sas_launch.h"

namespace sas {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef u16x4 u16x4u __attribute__((aligned(2)));

constexpr int kSub = 16;  // rows, outputs or ranks of one matrix instruction

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// An f32 value as three bf16 pieces whose sum it is (values below 2^-110
// lose bits that no product of theirs keeps).  Not finite: the first piece
// alone.
__device__ __forceinline__ void pieces_of(float x, uint16_t (&p)[3]) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7F800000u) == 0x7F800000u) {
    p[0] = (uint16_t)((u >> 16) | ((u & 0x7FFFFFu) ? 0x40u : 0u));
    p[1] = p[2] = 0;
    return;
  }
  p[0] = (uint16_t)(u >> 16);
  const float r1 = x - __uint_as_float(u & 0xFFFF0000u);
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

// 8 consecutive f32 values as three bf16 operands.
__device__ __forceinline__ void split8(const float *src, u32x4 (&p)[3]) {
  const f32x4 v0 = *reinterpret_cast<const f32x4 *>(src), v1 = *reinterpret_cast<const f32x4 *>(src + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint16_t a[3], b[3];
    pieces_of(i < 2 ? v0[2 * i] : v1[2 * i - 4], a);
    pieces_of(i < 2 ? v0[2 * i + 1] : v1[2 * i - 3], b);
#pragma unroll
    for (int k = 0; k < 3; ++k) p[k][i] = (uint32_t)a[k] | ((uint32_t)b[k] << 16);
  }
}

// The adapter of row `row`, -1 for none.
__device__ __forceinline__ int adapter_of(const ProjArgs &a, int row) {
  if (row >= a.rows || a.adapters == 0) return -1;
  const int n = a.row_adapter[row];
  return n >= 0 && n < a.adapters ? n : -1;
}

__device__ __forceinline__ int rank_of(const ProjArgs &a, int n) {
  return a.ranks ? min(max(a.ranks[n], 0), a.rank) : a.rank;
}

// Calls f(adapter) for each adapter among the 16 rows whose adapters lanes
// l & 15 hold in `mine`, in the order of their first rows.
template <typename F>
__device__ __forceinline__ void each_adapter(int mine, F f) {
  uint32_t left = (uint32_t)__ballot(mine >= 0) & 0xFFFFu;
  while (left) {
    const int cur = __builtin_amdgcn_readlane(mine, __builtin_ctz(left));
    left &= ~(uint32_t)__ballot(mine == cur);
    f(cur);
  }
}

// Block (subtile, slot): the slot-th adapter of the subtile's rows; its waves
// split dim, their sums meet in LDS.  Blocks past the subtiles write the
// pieces of f32 hidden states.
__global__ __launch_bounds__(kThreads) void proj_inner_kernel(const ProjArgs a) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int subs = (a.rows + kSub - 1) / kSub;
  if ((int)blockIdx.x >= subs) {
    if (!a.xp) return;
    // 8 values a thread
    const int per = a.dim / 8;
    const int64_t n = (int64_t)a.rows * per;
    const int64_t step = (int64_t)(gridDim.x - subs) * gridDim.y * kThreads;
    for (int64_t i = ((int64_t)(blockIdx.x - subs) * gridDim.y + blockIdx.y) * kThreads + tid; i < n; i += step) {
      const int64_t row = i / per, c = i - row * per;
      u32x4 p[3];
      split8(static_cast<const float *>(a.x) + row * a.x_stride + 8 * c, p);
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x4 *>(a.xp + ((int64_t)k * a.rows + row) * a.dim + 8 * c) = p[k];
    }
    return;
  }
  __shared__ f32x4 part[kWaves][64];
  const int row = (int)blockIdx.x * kSub + (lane & 15);
  const int mine = adapter_of(a, row);
  int cur = -1, at = 0;
  each_adapter(mine, [&](int n) {
    if (at++ == (int)blockIdx.y) cur = n;
  });
  if (cur < 0) return;
  const int used = rank_of(a, cur);
  const float scale = a.scales ? a.scales[cur] : 1.0f;
  const int xrow = min(row, a.rows - 1);
  const int kc = 8 * (lane >> 4);
  // dim in runs of 32 for the waves to share
  const int steps = (a.dim + 31) / 32, k0 = 32 * (steps * wave / kWaves), k1 = min(a.dim, 32 * (steps * (wave + 1) / kWaves));
  const uint16_t *A = static_cast<const uint16_t *>(a.a) + (int64_t)cur * a.a_adapter_stride;
  for (int t = 0; t < a.rank; t += kSub) {
    const uint16_t *ar = A + (int64_t)min(t + (lane & 15), a.rank - 1) * a.a_stride;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = k0 + kc; k - kc < k1; k += 32) {
      const bool in = k < k1;
      const u32x4 none = {0u, 0u, 0u, 0u};
      const u32x4 w = in ? *reinterpret_cast<const u32x4 *>(ar + k) : none;
      if (a.x_f32) {
        u32x4 p[3] = {none, none, none};
        if (in) split8(static_cast<const float *>(a.x) + (int64_t)xrow * a.x_stride + k, p);
#pragma unroll
        for (int i = 0; i < 3; ++i) acc = mfma(w, p[i], acc);
      } else {
        const uint16_t *xr = static_cast<const uint16_t *>(a.x) + (int64_t)xrow * a.x_stride;
        acc = mfma(w, in ? *reinterpret_cast<const u32x4 *>(xr + k) : none, acc);
      }
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave == 0) {
      // lane: row lane & 15, ranks t + 4 (lane / 16) ..
      f32x4 h = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
      const int r0 = t + 4 * (lane >> 4);
      if (mine == cur && r0 < a.rank) {
        u16x4 p[3];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint16_t q[3];
          pieces_of(r0 + i < used ? h[i] * scale : 0.0f, q);
#pragma unroll
          for (int k = 0; k < 3; ++k) p[k][i] = q[k];
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<u16x4 *>(a.hp + ((int64_t)row * 3 + k) * a.rank + r0) = p[k];
      }
    }
    __syncthreads();
  }
}

// A row of B from column r on: 8 ranks, those from `used` on zero.
__device__ __forceinline__ u32x4 b_ranks(const uint16_t *row, int r, int used) {
  u32x4 w = {0u, 0u, 0u, 0u};
  if (r >= used) return w;
  w = *reinterpret_cast<const u32x4 *>(row + r);
  if (r + 8 > used) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int left = used - r - 2 * i;
      w[i] = left <= 0 ? 0u : left == 1 ? w[i] & 0xFFFFu : w[i];
    }
  }
  return w;
}

// Four outputs from column n on of one row: added to, capped, rounded, stored.
__device__ __forceinline__ void store4(const ProjArgs &a, int row, int n, f32x4 v) {
  if (row >= a.rows || n >= a.out_dim) return;
  const int left = min(a.out_dim - n, 4);
  const int64_t at = (int64_t)row * a.out_stride + n;
  float *of = static_cast<float *>(a.out) + at;
  uint16_t *ob = static_cast<uint16_t *>(a.out) + at;
  if (a.accumulate) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) v[i] += a.out_bf16 ? __uint_as_float((uint32_t)ob[i] << 16) : of[i];
  }
  if (a.softcap > 0.0f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a.softcap * tanhf(v[i] / a.softcap);
  }
  if (a.out_bf16) {
    const u16x4 p = {bf16_of(v[0]), bf16_of(v[1]), bf16_of(v[2]), bf16_of(v[3])};
    if (left == 4) {
      *reinterpret_cast<u16x4u *>(ob) = p;
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (i < left) ob[i] = p[i];
    }
  } else if (left == 4) {
    *reinterpret_cast<f32x4u *>(of) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < left) of[i] = v[i];
  }
}

// Block (n, m): 64 outputs (16 a wave) of 16 rows.
template <int P>
__global__ __launch_bounds__(kThreads) void proj_rows_kernel(const ProjArgs a) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = (int)blockIdx.y * kSub + (lane & 15);
  const int xrow = min(row, a.rows - 1);
  const int kc = 8 * (lane >> 4);
  const int n0 = ((int)blockIdx.x * kWaves + wave) * kSub;
  if (n0 >= a.out_dim) return;
  const int wrow = min(n0 + (lane & 15), a.out_dim - 1);
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  if (a.weight) {
    const uint16_t *w = static_cast<const uint16_t *>(a.weight) + (int64_t)wrow * a.weight_stride;
    const uint16_t *x[P];
#pragma unroll
    for (int p = 0; p < P; ++p)
      x[p] = P == 1 ? static_cast<const uint16_t *>(a.x) + (int64_t)xrow * a.x_stride
                    : a.xp + ((int64_t)p * a.rows + xrow) * a.dim;
    for (int k = kc; k - kc < a.dim; k += 32) {
      const bool in = k < a.dim;
      const u32x4 none = {0u, 0u, 0u, 0u};
      const u32x4 wv = in ? *reinterpret_cast<const u32x4 *>(w + k) : none;
#pragma unroll
      for (int p = 0; p < P; ++p) acc = mfma(wv, in ? *reinterpret_cast<const u32x4 *>(x[p] + k) : none, acc);
    }
  }
  const int mine = adapter_of(a, row);
  each_adapter(mine, [&](int cur) {
    const int used = rank_of(a, cur);
    const uint16_t *b = static_cast<const uint16_t *>(a.b) + (int64_t)cur * a.b_adapter_stride + (int64_t)wrow * a.b_stride;
    const uint16_t *h = a.hp + (int64_t)xrow * 3 * a.rank;
    f32x4 ext = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int e = kc; e - kc < 3 * a.rank; e += 32) {
      const u32x4 none = {0u, 0u, 0u, 0u};
      const bool in = e < 3 * a.rank;
      const int r = e < a.rank ? e : e < 2 * a.rank ? e - a.rank : e - 2 * a.rank;
      const u32x4 bv = in ? b_ranks(b, r, used) : none;
      ext = mfma(bv, in ? *reinterpret_cast<const u32x4 *>(h + e) : none, ext);
    }
    if (mine == cur) acc = acc + ext;
  });
  store4(a, row, n0 + 4 * (lane >> 4), acc);
}

}  // namespace

size_t proj_scratch_bytes(int rows, int dim, int rank, bool x_f32) {
  const size_t h = ((size_t)rows * 3 * rank * 2 + 255) & ~size_t(255);
  return h + (x_f32 ? (size_t)rows * 3 * dim * 2 : 0);
}

hipError_t launch_project(const ProjArgs &a, hipStream_t stream) {
  const int subs = (a.rows + kSub - 1) / kSub;
  if (a.adapters > 0 || a.xp) {
    const int split = a.xp ? (int)(((int64_t)a.rows * (a.dim / 8) + kSub * kThreads - 1) / (kSub * kThreads)) : 0;
    proj_inner_kernel<<<dim3(subs + (split > 1024 ? 1024 : split), kSub), kThreads, 0, stream>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  const dim3 grid((a.out_dim + kWaves * kSub - 1) / (kWaves * kSub), subs);
  if (a.xp) proj_rows_kernel<3><<<grid, kThreads, 0, stream>>>(a);
  else proj_rows_kernel<1><<<grid, kThreads, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace sas
