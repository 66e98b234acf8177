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
//      instructions, so f32 inputs keep all their bits (two pieces would be
//      2e-6 off, one 2e-3).  One block puts the rows in the order of their
//      adapters, so that a tile of rows meets few of them.
//   2. proj_wide_kernel or proj_split_kernel: the rows' products with W, then
//      with B of each adapter among a tile's rows, each adapter in sums of its
//      own that only its rows add: a value that is not finite stays with its
//      adapter.
//
// What bounds it, and what it measured (MI355X, a call):
//   - up to about 128 rows W's stream from memory: 16 f32 rows x 2,560 x
//     151,936 160 us (5.0 TB/s), 128 rows x 2,560 x 262,144, capped, 16
//     adapters, 355 to 368 us (4.4 TB/s; 320 without adapters, 235 of it without the
//     134 MB of results).  What carried it: weight rows in whole lines,
//     nontemporal; loads kept several runs ahead of their use against the
//     compiler's order; results in whole lines past the caches.
//   - more rows the matrix instructions' operands in LDS, each wave reading all
//     of a tile's hidden states: 2,048 x 4,096 x 4,096 98 us (0.71 PFLOP/s, the
//     product 89 us of it; a library's 60), 200 f32 rows x 2,048 x 50,257 209
//     us (three products each: 0.6 PFLOP/s).
//   - an adapter a row (61 rows, ranks up to 64, 4,096 x 11,007: 115 us) the
//     addresses of B's and h's loads, 16 bytes a lane.
#include "sas_product.h"

namespace sas {
namespace {

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

// Block (subtile, slot, tile): 16 ranks of the slot-th adapter of the
// subtile's rows.  Its waves share out the runs of 32 of dim; their parts meet
// in LDS in a fixed order.  Of the blocks past the
// subtiles the first puts the rows in order, the others write the pieces of
// f32 hidden states.
constexpr int kInnerWaves = 16;
constexpr int kInnerThreads = 64 * kInnerWaves;
constexpr int kInnerDeep = 4;  // runs whose loads are in flight together

// The rows in the order of their adapters (rows without one last), so that a
// tile holds few adapters: a counting sort by one block.  Adapters past the
// bins share them, and rows of one bin come in any order; a row's result does
// not depend on its place.
constexpr int kOrderBins = 1024;
__device__ void order_rows(const ProjArgs &a) {
  __shared__ uint32_t bin[kOrderBins];
  __shared__ uint32_t wsum[kInnerWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  bin[tid] = 0u;
  __syncthreads();
  auto bin_of = [&](int row) {
    const int n = adapter_of(a, row);
    return n < 0 ? kOrderBins - 1 : n % (kOrderBins - 1);
  };
  for (int r = tid; r < a.rows; r += kInnerThreads) atomicAdd(&bin[bin_of(r)], 1u);
  __syncthreads();
  const uint32_t n = bin[tid];
  uint32_t x = n;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const uint32_t y = (uint32_t)__shfl_up((int)x, s, 64);
    if (lane >= s) x += y;
  }
  if (lane == 63) wsum[tid >> 6] = x;
  __syncthreads();
  for (int w = 0; w < (tid >> 6); ++w) x += wsum[w];
  bin[tid] = x - n;
  __syncthreads();
  for (int r = tid; r < a.rows; r += kInnerThreads) a.perm[atomicAdd(&bin[bin_of(r)], 1u)] = r;
}
static_assert(kOrderBins == kInnerThreads, "a thread a bin");

template <bool kF32>
__global__ __launch_bounds__(kInnerThreads) void proj_inner_kernel(const ProjArgs a) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int subs = (a.rows + kSub - 1) / kSub;
  if ((int)blockIdx.x >= subs && blockIdx.z > 0) return;
  if ((int)blockIdx.x == subs) {
    if (a.perm && blockIdx.y == 0) order_rows(a);
    return;
  }
  if ((int)blockIdx.x > subs) {
    if constexpr (kF32) {
      // 8 values a thread
      const int per = a.dim / 8;
      const int64_t n = (int64_t)a.rows * per;
      const int64_t step = (int64_t)(gridDim.x - subs - 1) * gridDim.y * kInnerThreads;
      for (int64_t i = ((int64_t)(blockIdx.x - subs - 1) * gridDim.y + blockIdx.y) * kInnerThreads + tid; i < n; i += step) {
        const int64_t row = i / per, c = i - row * per;
        u32x4 p[3];
        split8(static_cast<const float *>(a.x) + row * a.x_stride + 8 * c, p);
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x4 *>(a.xp + ((int64_t)k * a.rows + row) * a.dim + 8 * c) = p[k];
      }
    }
    return;
  }
  __shared__ f32x4 part[kInnerWaves][64];
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
  const int t = kSub * (int)blockIdx.z;
  const int steps = (a.dim + 31) / 32, g0 = steps * wave / kInnerWaves, g1 = steps * (wave + 1) / kInnerWaves;
  const uint16_t *A = static_cast<const uint16_t *>(a.a) + (int64_t)cur * a.a_adapter_stride;
  const u32x4 none = {0u, 0u, 0u, 0u};
  const uint16_t *ar = A + (int64_t)min(t + (lane & 15), a.rank - 1) * a.a_stride + kc;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int g = g0; g < g1; g += kInnerDeep) {
    u32x4 w[kInnerDeep], x[kInnerDeep][kF32 ? 3 : 1];
#pragma unroll
    for (int d = 0; d < kInnerDeep; ++d) {
      const int k = 32 * (g + d);
      const bool in = g + d < g1 && k + kc < a.dim;
      w[d] = in ? *reinterpret_cast<const u32x4 *>(ar + k) : none;
      if constexpr (kF32) {
        if (in) split8(static_cast<const float *>(a.x) + (int64_t)xrow * a.x_stride + k + kc, x[d]);
        else x[d][0] = x[d][1] = x[d][2] = none;
      } else {
        x[d][0] = in ? *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(a.x) + (int64_t)xrow * a.x_stride + k + kc) : none;
      }
    }
#pragma unroll
    for (int d = 0; d < kInnerDeep; ++d)
#pragma unroll
      for (int i = 0; i < (kF32 ? 3 : 1); ++i) acc = mfma(w[d], x[d][i], acc);
  }
  part[wave][lane] = acc;
  __syncthreads();
  if (wave == 0) {
    // lane: row lane & 15, ranks t + 4 (lane / 16) ..
    f32x4 h = part[0][lane];
#pragma unroll
    for (int i = 1; i < kInnerWaves; ++i) h = h + part[i][lane];
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

// A tile of 16 MT rows (positions tile0 .. of the order in a.perm): its rows,
// and its pairs (subtile, adapter) with the subtile's rows that use it.
template <int MT>
struct Tile {
  int row[16 * MT];       // the row at a position; past the last row: the last row
  int adapter[16 * MT];   // -1: none, or past the last row
  int pairs;
  int pair_adapter[16 * MT];
  uint32_t pair_users[16 * MT];  // rank in use << 20 | subtile << 16 | rows as bits
};

// Fills l (the block's threads; a barrier before it is read).
template <int MT>
__device__ __forceinline__ void tile_rows(const ProjArgs &a, int tile0, Tile<MT> &l) {
  for (int i = threadIdx.x; i < 16 * MT; i += blockDim.x) {
    const int at = tile0 + i, row = a.perm ? a.perm[min(at, a.rows - 1)] : min(at, a.rows - 1);
    l.row[i] = row;
    l.adapter[i] = at < a.rows ? adapter_of(a, row) : -1;
  }
}
template <int MT>
__device__ __forceinline__ void tile_pairs(const ProjArgs &a, Tile<MT> &l) {
  if (threadIdx.x >= 64 || a.adapters == 0) return;
  const int lane = threadIdx.x;
  int n = 0;
  for (int m = 0; m < MT; ++m) {
    const int mine = l.adapter[16 * m + (lane & 15)];
    each_adapter(mine, [&](int cur) {
      const uint32_t users = (uint32_t)__ballot(mine == cur) & 0xFFFFu;
      const int used = rank_of(a, cur);
      if (lane == 0) {
        l.pair_adapter[n] = cur;
        l.pair_users[n] = (uint32_t)used << 20 | (uint32_t)m << 16 | users;
      }
      ++n;
    });
  }
  if (lane == 0) l.pairs = n;
}

// Adds the tile's adapters' terms, B times the pieces of h, 32 ranks an item,
// an item's loads two ahead of its products.  An item's sums are its own and
// only the adapter's rows add them.  mine(adapter): whether this wave takes it.
template <int MT, int NT, typename F>
__device__ __forceinline__ void add_adapters(const ProjArgs &a, const Tile<MT> &l, int n0, F takes, f32x4 (&acc)[MT][NT]) {
  const int lane = threadIdx.x & 63, q = lane >> 4;
  const u32x4 none = {0u, 0u, 0u, 0u};
  const int blocks = (a.rank + 31) / 32, pairs = l.pairs;
  struct Item {
    int m;          // subtile, -1: no item
    uint32_t users;
    int products;
    u32x4 b[NT], h[3];
  };
  int at = -1, rb = blocks - 1, cur = 0, used = 0;
  uint32_t mu = 0;
  // the next item's loads
  auto next = [&](Item &it) __attribute__((always_inline)) {
    if (++rb == blocks) {
      rb = 0;
      do ++at;
      while (at < pairs && !takes(l.pair_adapter[at]));
      if (at < pairs) {
        cur = __builtin_amdgcn_readfirstlane(l.pair_adapter[at]);
        mu = __builtin_amdgcn_readfirstlane(l.pair_users[at]);
        used = (int)(mu >> 20);
      }
    }
    it.m = -1;
    if (at >= pairs) {
      rb = blocks - 1;  // (stays past the end)
      return;
    }
    it.m = (int)(mu >> 16) & 15;
    it.users = mu & 0xFFFFu;
    const int r0 = 32 * rb, n = a.rank - r0;  // ranks from r0 on
    // The four octets of an operand: of up to 8 ranks the three pieces (one
    // product), of up to 16 two pieces and then the third (two), of more one
    // piece after another (three).  B's octets repeat under them.
    const int oct = n <= 8 ? 0 : n <= 16 ? q & 1 : q;
    it.products = n <= 8 ? 1 : n <= 16 ? 2 : 3;
    const uint16_t *b = static_cast<const uint16_t *>(a.b) + (int64_t)cur * a.b_adapter_stride;
#pragma unroll
    for (int t = 0; t < NT; ++t)
      it.b[t] = b_ranks(b + (int64_t)min(n0 + 16 * t + (lane & 15), a.out_dim - 1) * a.b_stride, r0 + 8 * oct, used);
    // (rows of other adapters are left out: an address a lane is what a load costs)
    const uint16_t *h = a.hp + (int64_t)l.row[16 * it.m + (lane & 15)] * 3 * a.rank + r0 + 8 * oct;
    const bool user = (it.users >> (lane & 15)) & 1u;
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const int piece = n <= 8 ? q : n <= 16 ? 2 * j + (q >> 1) : j;
      it.h[j] = user && j < it.products && piece < 3 && r0 + 8 * oct < used ? *reinterpret_cast<const u32x4 *>(h + piece * a.rank) : none;
    }
  };
  auto add = [&](const Item &it, f32x4 (&sum)[NT]) __attribute__((always_inline)) {
    f32x4 ext[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) ext[t] = mfma(it.b[t], it.h[0], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
    // (operands past `products` are zero, but B's may hold what is not finite)
    if (it.products > 1) {
#pragma unroll
      for (int t = 0; t < NT; ++t) ext[t] = mfma(it.b[t], it.h[1], ext[t]);
    }
    if (it.products > 2) {
#pragma unroll
      for (int t = 0; t < NT; ++t) ext[t] = mfma(it.b[t], it.h[2], ext[t]);
    }
    const bool mine = (it.users >> (lane & 15)) & 1u;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[t][i] += mine ? ext[t][i] : 0.0f;
  };
  // the pairs come subtile by subtile: the sums of each have a loop of their
  // own (selecting them by a variable doubles the kernel's registers)
  Item x, y;
  next(x);
  next(y);
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    while (x.m == m) {
      Item z;
      next(z);
      add(x, acc[m]);
      x = y;
      y = z;
    }
  }
}

// An operand of 16 rows x 64 values (2 KB): loaded eight lanes a row, whole
// 128-byte lines (memory serves lines 10 % faster than the matrix layout's 64
// bytes a row), and turned into the matrix layout through LDS, where value
// octet o of row r sits in 16-byte slot 8 r + (o ^ r / 2): the eight lanes
// that write a row, and the 16 rows that read an octet, meet every bank once.
constexpr int kRun = 64;          // values of dim in an operand
constexpr int kSlots = 128;       // 16-byte slots of an operand
__device__ __forceinline__ int put_slot(int j) {  // of lane's load j (rows 8 j ..)
  const int lane = threadIdx.x & 63, r = 8 * j + (lane >> 3);
  return 8 * r + ((lane & 7) ^ (r >> 1));
}
__device__ __forceinline__ int get_slot(int h) {  // half h: values 32 h ..
  const int lane = threadIdx.x & 63, r = lane & 15;
  return 8 * r + ((4 * h + (lane >> 4)) ^ (r >> 1));
}

// Many outputs: eight waves share a tile's rows (16 MT) and take 16 NT outputs
// each.  A wave's weight rows go through LDS of its own, kDeep runs ahead in
// registers, so that a block alone keeps enough of memory in flight; the hidden
// states' chunks of kSteps runs are staged for all waves.
constexpr int kWideWaves = 8;
constexpr int kWideThreads = 64 * kWideWaves;
template <int MT, int NT, int P>
struct Wide {
  static constexpr int kBlockOut = kWideWaves * 16 * NT;
  static constexpr int kSteps = MT * P >= 5 ? 1 : MT * P >= 2 ? 2 : 4;  // runs a chunk
  static constexpr int kDeep = NT == 1 || (MT >= 7 && P == 1) ? 4 : 2;  // runs of the weight rows in registers
  // Chunks of the hidden states in registers: as far ahead as the weight rows.
  // Loads end in the order they began, so waiting for a younger chunk would
  // wait for every weight row behind it (128 rows: 4 runs ahead were no
  // faster than 2 until the hidden states were too).
  static constexpr int kAhead = kDeep / kSteps > 2 ? kDeep / kSteps : 2;
  static constexpr int kUnroll = kAhead;  // chunks a turn of the loop
  static constexpr int kTiles = kSteps * P * MT;                        // operands of a chunk
  static constexpr int kMine = (2 * kTiles + kWideWaves - 1) / kWideWaves;  // a wave's loads of them
};

// kOnce: one tile holds all rows, so that no other block reads a weight row
// again (nontemporal loads then: 6.2 -> 6.9 TB/s in a bare stream of a head).
template <int MT, int NT, int P, bool kOnce>
__global__ __launch_bounds__(kWideThreads, P == 1 && MT <= 6 ? 4 : 2) void proj_wide_kernel(const ProjArgs a) {
  using C = Wide<MT, NT, P>;
  __shared__ u32x4 xs[2][C::kTiles][kSlots];
  __shared__ u32x4 ws[kWideWaves][NT][kSlots];
  __shared__ Tile<MT> tile;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int mtiles = kOnce ? 1 : (a.rows + 16 * MT - 1) / (16 * MT);
  const int pos = xcd_run((int)blockIdx.x, (int)gridDim.x);
  const int tile0 = (pos % mtiles) * 16 * MT, n0 = (pos / mtiles) * C::kBlockOut + wave * 16 * NT;
  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  tile_rows<MT>(a, tile0, tile);
  __syncthreads();
  tile_pairs<MT>(a, tile);
  // piece p of the hidden state at a position
  auto x_row = [&](int p, int at) {
    const int64_t row = tile.row[at];
    return P == 1 ? static_cast<const uint16_t *>(a.x) + row * a.x_stride : a.xp + ((int64_t)p * a.rows + row) * a.dim;
  };
  if (a.weight) {
    const int chunks = a.dim / (kRun * C::kSteps), runs = chunks * C::kSteps;  // whole ones
    const int w0 = min(n0, a.out_dim - 1);
    if (chunks > 0) {
      // byte offsets from the wave's first weight row
      const char *wbase = static_cast<const char *>(a.weight) + (int64_t)w0 * a.weight_stride * 2;
      uint32_t wr[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          wr[t][j] = ((uint32_t)(min(n0 + 16 * t + 8 * j + (lane >> 3), a.out_dim - 1) - w0) * (uint32_t)a.weight_stride + 8 * (lane & 7)) * 2u;
      // run g of the weight rows (past the last: the last again)
      auto load_w = [&](int g, u32x4 (&w)[NT][2]) __attribute__((always_inline)) {
        const char *wk = wbase + 2 * kRun * (int64_t)min(g, runs - 1);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const u32x4 *src = reinterpret_cast<const u32x4 *>(wk + wr[t][j]);
            w[t][j] = kOnce ? __builtin_nontemporal_load(src) : *src;
          }
      };
      // this wave's loads of chunk c: load f is half f % 2 of operand f / 2 =
      // (step, piece, subtile)
      const uint16_t *xr[C::kMine];
#pragma unroll
      for (int i = 0; i < C::kMine; ++i) {
        const int f = min(wave + kWideWaves * i, 2 * C::kTiles - 1);
        xr[i] = x_row((f / 2 / MT) % P, 16 * ((f / 2) % MT) + 8 * (f & 1) + (lane >> 3)) + kRun * (f / 2 / MT / P) + 8 * (lane & 7);
      }
      auto load_x = [&](int c, u32x4 (&x)[C::kMine]) __attribute__((always_inline)) {
        const int64_t k = kRun * C::kSteps * (int64_t)min(c, chunks - 1);
#pragma unroll
        for (int i = 0; i < C::kMine; ++i) x[i] = *reinterpret_cast<const u32x4 *>(xr[i] + k);
      };
      auto store_x = [&](int buf, const u32x4 (&x)[C::kMine]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < C::kMine; ++i) {
          const int f = wave + kWideWaves * i;
          if (2 * C::kTiles % kWideWaves == 0 || f < 2 * C::kTiles) xs[buf][f / 2][put_slot(f & 1)] = x[i];
        }
      };
      u32x4 w[C::kDeep][NT][2], x[C::kAhead][C::kMine];
      // in the order of their use (a wait in the loop covers the loop's first
      // turn too)
#pragma unroll
      for (int d = 0; d < C::kAhead; ++d) {
        load_x(d, x[d]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < C::kDeep; ++e)
          if (e / C::kSteps == d || (d == C::kAhead - 1 && e / C::kSteps > d)) {
            load_w(e, w[e]);
            __builtin_amdgcn_sched_barrier(0);
          }
      }
      store_x(0, x[0]);
      lds_barrier();
      // chunk c, the v-th of its turn, then the next one's hidden states (past
      // the last the last again)
      auto chunk = [&](int c, auto vt) __attribute__((always_inline)) {
        constexpr int v = decltype(vt)::value;
#pragma unroll
        for (int s = 0; s < C::kSteps; ++s) {
          constexpr int D = C::kDeep;
          const int slot = (v * C::kSteps + s) % D;
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) ws[wave][t][put_slot(j)] = w[slot][t][j];
          // the loads stay here: left to itself the compiler moves them down to
          // where they are used, and every run waits for memory
          if (s == 0) load_x(c + C::kAhead, x[v]);
          load_w(c * C::kSteps + s + D, w[slot]);
          wave_lds_sync();
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            u32x4 wv[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) wv[t] = ws[wave][t][get_slot(h)];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int p = 0; p < P; ++p) {
                const u32x4 xv = xs[v & 1][(s * P + p) * MT + m][get_slot(h)];
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[m][t] = mfma(wv[t], xv, acc[m][t]);
              }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        store_x((v + 1) & 1, x[(v + 1) % C::kAhead]);
        __builtin_amdgcn_sched_barrier(0);
        lds_barrier();
      };
      // Whole turns first: the loop has no way out but its end (a way from its
      // middle back to its head, even one never taken, would make the waits at
      // the head cover the loads just begun).
      int c = 0;
      for (; c + C::kUnroll <= chunks; c += C::kUnroll) each_const<C::kUnroll>([&](auto v) { chunk(c + decltype(v)::value, v); });
      each_const<C::kUnroll - 1>([&](auto v) {
        if (c + decltype(v)::value < chunks) chunk(c + decltype(v)::value, v);
      });
    }
    if (chunks == 0) __syncthreads();
    // what is left of dim, straight to registers
    const u32x4 none = {0u, 0u, 0u, 0u};
    for (int k0 = runs * kRun; k0 < a.dim; k0 += 32) {
      const int k = k0 + 8 * (lane >> 4);
      const bool in = k < a.dim;
      u32x4 wv[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t)
        wv[t] = in ? *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(a.weight) +
                                                      (int64_t)min(n0 + 16 * t + (lane & 15), a.out_dim - 1) * a.weight_stride + k)
                   : none;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int p = 0; p < P; ++p) {
          const u32x4 xv = in ? *reinterpret_cast<const u32x4 *>(x_row(p, 16 * m + (lane & 15)) + k) : none;
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[m][t] = mfma(wv[t], xv, acc[m][t]);
        }
    }
  } else {
    __syncthreads();
  }
  if (a.adapters > 0 && n0 < a.out_dim) add_adapters<MT, NT>(a, tile, n0, [](int) { return true; }, acc);
  // A subtile's rows at a time through LDS, so that a row's outputs go out in
  // whole lines (lane: outputs 4 l .. of a row).
  constexpr int kPitch = C::kBlockOut + 4, kLanes = C::kBlockOut / 4, kRows = 64 / kLanes;
  static_assert(16 * kPitch * 4 <= (int)sizeof(xs), "a subtile's sums fit");
  float *stage = reinterpret_cast<float *>(&xs[0][0][0]);
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    lds_barrier();
#pragma unroll
    for (int t = 0; t < NT; ++t)
      *reinterpret_cast<f32x4 *>(stage + (lane & 15) * kPitch + wave * 16 * NT + 16 * t + 4 * (lane >> 4)) = acc[m][t];
    lds_barrier();
#pragma unroll
    for (int r = wave * kRows; r < 16; r += kWideWaves * kRows) {
      const int at = 16 * m + r + lane / kLanes, col = 4 * (lane % kLanes);
      const f32x4 v = *reinterpret_cast<const f32x4 *>(stage + (r + lane / kLanes) * kPitch + col);
      if (tile0 + at < a.rows) finish4(a, tile.row[at], (pos / mtiles) * C::kBlockOut + col, v);
    }
  }
}

// Few outputs: eight waves split dim (and the tile's adapters) for the same
// 16 NT outputs of 16 MT rows; their sums meet in LDS in a fixed order.  No
// two waves need the same operand, so all go straight to registers.
constexpr int kSplitWaves = 8;

template <int MT, int NT, int P>
__global__ __launch_bounds__(64 * kSplitWaves) void proj_split_kernel(const ProjArgs a) {
  __shared__ f32x4 part[kSplitWaves][MT * NT][64];
  __shared__ Tile<MT> tile;
  constexpr int U = MT * P >= 8 ? 1 : MT * P >= 4 ? 2 : 4;  // runs of 32 whose loads are in flight together
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int mtiles = (a.rows + 16 * MT - 1) / (16 * MT);
  const int pos = xcd_run((int)blockIdx.x, (int)gridDim.x);
  const int tile0 = (pos % mtiles) * 16 * MT, n0 = (pos / mtiles) * 16 * NT;
  const int kc = 8 * (lane >> 4);
  const u32x4 none = {0u, 0u, 0u, 0u};
  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  tile_rows<MT>(a, tile0, tile);
  __syncthreads();
  tile_pairs<MT>(a, tile);
  __syncthreads();
  if (a.weight) {
    const int steps = (a.dim + 31) / 32, g0 = steps * wave / kSplitWaves, g1 = steps * (wave + 1) / kSplitWaves;
    const uint16_t *wr[NT], *xr[MT][P];
#pragma unroll
    for (int t = 0; t < NT; ++t)
      wr[t] = static_cast<const uint16_t *>(a.weight) + (int64_t)min(n0 + 16 * t + (lane & 15), a.out_dim - 1) * a.weight_stride + kc;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int64_t row = tile.row[16 * m + (lane & 15)];
#pragma unroll
      for (int p = 0; p < P; ++p)
        xr[m][p] = (P == 1 ? static_cast<const uint16_t *>(a.x) + row * a.x_stride : a.xp + ((int64_t)p * a.rows + row) * a.dim) + kc;
    }
    for (int g = g0; g < g1; g += U) {
      u32x4 w[U][NT], x[U][MT][P];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = 32 * (g + u);
        const bool in = g + u < g1 && k + kc < a.dim;
#pragma unroll
        for (int t = 0; t < NT; ++t) w[u][t] = in ? *reinterpret_cast<const u32x4 *>(wr[t] + k) : none;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int p = 0; p < P; ++p) x[u][m][p] = in ? *reinterpret_cast<const u32x4 *>(xr[m][p] + k) : none;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int p = 0; p < P; ++p)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[m][t] = mfma(w[u][t], x[u][m][p], acc[m][t]);
    }
  }
  // (by the adapter, not its place in the tile: a row's sums then do not
  // depend on the order of the rows)
  if (a.adapters > 0) add_adapters<MT, NT>(a, tile, n0, [&](int cur) { return cur % kSplitWaves == wave; }, acc);
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][m * NT + t][lane] = acc[m][t];
  __syncthreads();
  for (int i = wave; i < MT * NT; i += kSplitWaves) {
    f32x4 v = part[0][i][lane];
#pragma unroll
    for (int w = 1; w < kSplitWaves; ++w) v = v + part[w][i][lane];
    const int at = 16 * (i / NT) + (lane & 15);
    if (tile0 + at < a.rows) finish4(a, tile.row[at], n0 + 16 * (i % NT) + 4 * (lane >> 4), v);
  }
}

template <int MT, int NT, int P>
void launch_wide(const ProjArgs &a, hipStream_t stream) {
  using C = Wide<MT, NT, P>;
  const int blocks = ((a.rows + 16 * MT - 1) / (16 * MT)) * ((a.out_dim + C::kBlockOut - 1) / C::kBlockOut);
  // a tile of up to four subtiles has all rows (launch_rows)
  if (MT <= 4 || a.rows <= 16 * MT) proj_wide_kernel<MT, NT, P, true><<<blocks, kWideThreads, 0, stream>>>(a);
  else proj_wide_kernel<MT, NT, P, MT <= 4><<<blocks, kWideThreads, 0, stream>>>(a);
}

template <int MT, int NT, int P>
void launch_split(const ProjArgs &a, hipStream_t stream) {
  const int blocks = ((a.rows + 16 * MT - 1) / (16 * MT)) * ((a.out_dim + 16 * NT - 1) / (16 * NT));
  proj_split_kernel<MT, NT, P><<<blocks, 64 * kSplitWaves, 0, stream>>>(a);
}

template <int P>
void launch_rows(const ProjArgs &a, hipStream_t stream) {
  const int subs = (a.rows + kSub - 1) / kSub;
  // subtiles a tile of the wide kernel: as few tiles as 8 allow, evenly
  const int tiles = (subs + 7) / 8, mt = (subs + tiles - 1) / tiles;
  // The wide kernel takes few, long blocks: from 3/8 of a tile of 256 outputs a CU
  // on (up to 32 bf16 rows: from one).  Over 1,826 shapes (1 to 4,096 rows, 512 to
  // 80,000 outputs of 512 to 8,192 values) that is 2 % off the faster kernel in the
  // mean, 2.1 times at worst; one tile a CU for all was 8 %, and 9.4 times at worst.
  // bf16 rows x 4,096 values, wide / split: 64 rows x 11,007 (43 tiles) 55 / 47 us,
  // 512 x 4,096 (64) 67 / 88, 512 x 8,192 (128) 68 / 170, 1,920 x 4,096 (240) 76 / 334;
  // 16 x 32,768 (128) 52 / 49, 16 x 65,536 (256) 96 / 130.
  const bool few = P == 1 && subs <= 2;
  if ((int64_t)tiles * ((a.out_dim + 255) / 256) * 8 >= (int64_t)a.cus * (few ? 8 : 3)) {
    switch (mt) {
      case 1: return launch_wide<1, 1, P>(a, stream);
      case 2: return launch_wide<2, 1, P>(a, stream);
      case 3: return launch_wide<3, 2, P>(a, stream);
      case 4: return launch_wide<4, 2, P>(a, stream);
      case 5: return launch_wide<5, 2, P>(a, stream);
      case 6: return launch_wide<6, 2, P>(a, stream);
      case 7: return launch_wide<7, 2, P>(a, stream);
      default: return launch_wide<8, 2, P>(a, stream);
    }
  }
  if (subs == 1) {
    if (a.out_dim <= 32 * a.cus) return launch_split<1, 1, P>(a, stream);
    return launch_split<1, 2, P>(a, stream);
  }
  if (subs <= 2) return launch_split<2, 2, P>(a, stream);
  launch_split<4, 2, P>(a, stream);
}

}  // namespace

// The order of the rows, h, then the pieces of x.
ProjScratch proj_scratch(int rows, int dim, int rank, bool x_f32) {
  auto up = [](size_t n) { return (n + 255) & ~size_t(255); };
  ProjScratch p;
  p.hp = rank > 0 ? up((size_t)rows * 4) : 0;
  p.xp = p.hp + up((size_t)rows * 3 * rank * 2);
  p.bytes = p.xp + (x_f32 ? (size_t)rows * 3 * dim * 2 : 0);
  return p;
}

hipError_t launch_project(const ProjArgs &a, hipStream_t stream) {
  const int subs = (a.rows + kSub - 1) / kSub;
  if (a.adapters > 0 || a.xp) {
    const int slots = a.adapters < 1 ? 1 : a.adapters < kSub ? a.adapters : kSub;
    const int64_t split = a.xp ? ((int64_t)a.rows * (a.dim / 8) + slots * kInnerThreads - 1) / (slots * kInnerThreads) : 0;
    const dim3 grid(subs + 1 + (unsigned)(split > 1024 ? 1024 : split), slots, a.rank > 0 ? (a.rank + kSub - 1) / kSub : 1);
    if (a.x_f32) proj_inner_kernel<true><<<grid, kInnerThreads, 0, stream>>>(a);
    else proj_inner_kernel<false><<<grid, kInnerThreads, 0, stream>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  if (a.xp) launch_rows<3>(a, stream);
  else launch_rows<1>(a, stream);
  return hipGetLastError();
}

}  // namespace sas
