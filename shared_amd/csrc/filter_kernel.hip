// filter_kernel.hip - sampling over the whole vocabulary with temperature,
// top-k of any size, top-p and min-p (gfx950).
//
// A row's candidates in the order (value descending, id ascending) are cut to
// a prefix, and the draw walks the kept ids in ascending order.  No ids are
// sorted: where the prefix ends is found from the counts and masses of value
// ranges, then among the ids of one range.
//
// Masses exp((v - m) / T) are summed in doubles in a fixed order, or as 64-bit
// integers of 2^-shift, whose sums of any order, atomic ones too, are the same
// bits.  2^shift * vocab <= 2^62, so no sum overflows; rounding one mass is off
// by 2^-(shift + 1) of the largest at most (2^-45 for 262,144 ids).
//
// Four launches:
//   1. filter_parts_kernel, a block a part (8,192 ids, fewer in small batches):
//      reads the logits once; leaves the part's largest value, its mass, the
//      masses and counts of 128 ranges below its largest value, and its best
//      ids.  Bound by the issue of vector instructions: 256 rows x 262,144 f32,
//      nothing cut, 78 us (3.4 TB/s), 41 an id, 13 of them double, 88 % of what
//      the units issue (the LDS that holds the exponential's table is busy 18 %
//      of the time, half of it conflicts); 128 rows under a grammar 67 us, 69 an
//      id, 83 %; 64 bf16 rows x 151,936 with min-p 26 us, 71 an id, 57 %, the
//      rest waits of 4.75 blocks a CU.
//   2. filter_merge_kernel, four waves a row: the ends of the prefixes among
//      the lists' ids, kept in registers, and the draw; 10 to 30 us, a chain of
//      dependent steps.  (One kernel of 1,024 threads for every row: 24 to 30.)
//   3. filter_gather_kernel, the whole chip: the ids of the ranges in which the
//      ends lie, for rows whose lists do not reach them (wide nuclei).
//   4. filter_rest_kernel, a block a row left: the ends among those ids, 34 to
//      54 us; or by rereading the row, where a value is out of the ranges' scope,
//      an end lies below the 128 ranges (8 to 16 T) or its ranges hold more than
//      4,096 ids: 0.5 ms at 151,936 ids, 0.95 at 262,144, 1.5 with two ends.
//      Launches 3 and 4 end at once where no row was left (4 to 9 us together).
#include <algorithm>

#include "sas_device.h"
#include "sas_launch.h"

namespace sas {
namespace {

typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef u16x4 u16x4u __attribute__((aligned(2)));

constexpr int kRowThreads = 512;  // (1,024 would leave 128 registers a thread, and spill)
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kSpan = 16384;                      // ids a block of the rest kernel holds at once
constexpr int kQuads = kSpan / (4 * kRowThreads); // quads of ids per thread
constexpr int kMaxFilterParts = 2048;             // 2,048 ids a part: batches of up to 512 parts of 8,192
constexpr int kEntries = 4096;                    // listed ids the merge takes
constexpr int kBins = 512;                        // value ranges of (m - v) / T, 1/8 each; the last takes the rest
constexpr uint32_t kNegInf = 0x007FFFFFu;         // okey(-inf): candidates lie above

__device__ __forceinline__ sas_filter_params load_filter_params(const FilterArgs &a, int row) {
  if (!a.row_params) return a.params;
  static_assert(sizeof(sas_filter_params) % 4 == 0, "whole words");
  union {
    sas_filter_params p;
    uint32_t w[sizeof(sas_filter_params) / 4];
  } u;
  const uint32_t *src = reinterpret_cast<const uint32_t *>(a.row_params + row);
#pragma unroll
  for (int i = 0; i < (int)(sizeof(sas_filter_params) / 4); ++i) u.w[i] = __builtin_nontemporal_load(src + i);
  return u.p;
}

// Four logits from id `id` on (NaN past the row's end), as f32.
template <int kType>
__device__ __forceinline__ f32x4 load_logits(const FilterArgs &a, int64_t row0, int id) {
  const float nan = qnan();
  f32x4 v = {nan, nan, nan, nan};
  const int left = a.vocab - id;
  if (left <= 0) return v;
  if constexpr (kType == SAS_TYPE_F32) {
    const float *p = static_cast<const float *>(a.logits) + row0 + id;
    if (left >= 4) return *reinterpret_cast<const f32x4u *>(p);
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < left) v[i] = p[i];
    return v;
  }
  const uint16_t *p = static_cast<const uint16_t *>(a.logits) + row0 + id;
  u16x4 h = {0, 0, 0, 0};
  if (left >= 4) {
    h = *reinterpret_cast<const u16x4u *>(p);
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < left) h[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float f = kType == SAS_TYPE_BF16 ? __uint_as_float((uint32_t)h[i] << 16)
                                            : (float)__builtin_bit_cast(_Float16, (uint16_t)h[i]);
    v[i] = i < left ? f : nan;
  }
  return v;
}

// A row's history: its ids and how often each of a span's ids occurs.
struct History {
  const uint32_t *ids;
  int n;
};
__device__ __forceinline__ History history_of(const FilterArgs &a, int row) {
  History h{nullptr, 0};
  if (!a.hist_ids) return h;
  const int64_t lo = min(max((int64_t)a.hist_offsets[row], (int64_t)0), a.hist_count);
  const int64_t hi = min(max((int64_t)a.hist_offsets[row + 1], lo), a.hist_count);
  h.ids = a.hist_ids + lo;
  h.n = (int)min(hi - lo, (int64_t)SAS_MAX_HISTORY);
  return h;
}

__device__ __forceinline__ float penalized(float v, uint32_t count, const sas_filter_params &p) {
  double d = (double)v;
  d = d > 0.0 ? d / p.repetition_penalty : d * p.repetition_penalty;
  d = d - p.frequency_penalty * (double)count;
  d = d - p.presence_penalty;
  return (float)d;
}

// ---------------------------------------------------------------- parts --
// A part's values on one grid of ranges of width 2^e, e = floor(log2(T / 8)):
// 1/16 to 1/8 of (v - m) / T.  The grid is the same for every part of a row,
// so their ranges add up, and scaling by a power of two is exact.
struct Grid {
  float inv_width;   // 2^-e
  double per;        // 256 / (T ln 2): 256ths of an octave a unit of value
  bool plain;        // T is in the grid's scope
};
__device__ __forceinline__ Grid grid_of(double temperature) {
  Grid g;
  const int e = (int)(((uint64_t)__double_as_longlong(temperature) >> 52) & 0x7FF) - 1023 - 3;
  g.plain = temperature > 0.0 && e >= -24 && e <= 24;
  g.inv_width = __uint_as_float((uint32_t)(127 - (g.plain ? e : 0)) << 23);
  g.per = 369.3299304675746 / temperature;
  return g;
}
// A value's range; exact below 2^22 ranges from zero (kFar otherwise).
__device__ __forceinline__ float range_of(float v, const Grid &g) { return __builtin_floorf(v * g.inv_width); }
constexpr float kFar = 4194304.0f;
// A part's ranges are kept where its largest value lies within kFar.  A part below
// that counts for nothing in its row, so a row's largest value has to lie 2,048
// ranges above: 128 T at least, masses below 2^-184.
constexpr float kNear = 2048.0f - kFar;
// A part's ranges sum masses as integers of 2^-kFilterShift: 8,192 of at most 1
// stay below 2^64.
constexpr double kUnit = (double)(1ull << kFilterShift);

// Masses are powers of two counted in 256ths of an octave.  2^(j / 256), j = 0
// .. 255, within 1 ulp, computed once a block, a thread an entry (its first 256).
constexpr int kTab = 256;
__device__ __forceinline__ void fill_tab(double *tab) {
  if (threadIdx.x < kTab) tab[threadIdx.x] = exp2((double)threadIdx.x * (1.0 / 256.0));
}
// 2^(y / 256), -32768 <= y <= 0: the table's 2^(k / 256) times a Taylor series
// in |r| <= 1/2 (2^(r / 256) to degree 4, 4e-17 short), the exponent added as
// an integer; within 3 ulp of y's.  14 instructions a value, a third of what the
// parts kernel issues where nothing is cut.
__device__ __forceinline__ double exp256(double y, const double *tab) {
  const double magic = 6755399441055744.0;
  const double kf = y + magic;
  const int k = (int)(uint32_t)(uint64_t)__double_as_longlong(kf);
  const double r = y - (kf - magic);
  const double t = tab[k & (kTab - 1)];
  const double c1 = 0.0027076061740622863, c2 = 3.665565596910106e-06, c3 = 3.308302680541371e-09, c4 = 2.239395190875157e-12;
  const double x = t * fma(fma(fma(fma(r, c4, c3), r, c2), r, c1), r, 1.0);
  return __hiloint2double(__double2hiint(x) + ((k >> 8) << 20), __double2loint(x));
}
constexpr double kLeast = -32768.0;  // (2^-128: nothing)

__device__ __forceinline__ bool filters(const sas_filter_params &p) {
  return p.top_k > 0 || p.top_p < 1.0 || p.min_p > 0.0;
}
__device__ __forceinline__ bool greedy_row(const sas_filter_params &p) { return !(p.temperature > 0.0) || p.top_k == 1; }

// The values of a span of ids as the operator takes them, -inf for what is no
// candidate: quad j of thread t of kT holds ids id0 + 4 (j kT + t) ..
template <int kT, int kType, bool kSoft, int Q>
__device__ __forceinline__ void span_values(const FilterArgs &a, const sas_filter_params &p, int64_t row0, const uint32_t *mask,
                                            const History &h, uint32_t *count, int id0, float (&v)[Q][4]) {
  const float neg = -__builtin_inff();
  uint32_t bits[Q];
#pragma unroll
  for (int j = 0; j < Q; ++j) {
    const int id = id0 + 4 * (j * kT + (int)threadIdx.x);
    const f32x4 x = load_logits<kType>(a, row0, id);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[j][i] = x[i];
    bits[j] = !mask ? 0xFu : id < a.vocab ? mask[id >> 5] >> (id & 31) : 0u;
  }
  if (h.n) {
    constexpr int kIds = 4 * kT * Q;
    __syncthreads();
    for (int i = threadIdx.x; i < kIds / 2; i += kT) count[i] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < h.n; i += kT) {
      const uint32_t at = h.ids[i] - (uint32_t)id0;
      if (at < (uint32_t)kIds) atomicAdd(&count[at >> 1], 1u << (16 * (at & 1)));
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < Q; ++j) {
    // two counts a word; most quads have none
    const int at = 4 * (j * kT + (int)threadIdx.x);
    const uint32_t c0 = h.n ? count[at >> 1] : 0u, c1 = h.n ? count[(at >> 1) + 1] : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = v[j][i];
      if (kSoft && p.softcap > 0.0f) x = softcap_f32(x, p.softcap);
      if (c0 | c1) {
        const uint32_t c = ((i < 2 ? c0 : c1) >> (16 * (i & 1))) & 0xFFFFu;
        if (c) x = penalized(x, c, p);
      }
      v[j][i] = ((bits[j] >> i) & 1u) && x > neg ? x : neg;
    }
  }
}

template <int kType, bool kSoft, int kT, int Q>
__global__ __launch_bounds__(kT) void filter_parts_kernel(const FilterArgs a) {
  constexpr int kIds = 4 * Q * kT, kW = kT / 64;
  const int kList = 1 << a.log_list;
  __shared__ double tab[kTab];
  __shared__ uint32_t count[kIds / 2];
  __shared__ unsigned long long mass[kFilterRanges];
  __shared__ uint32_t cnt[kFilterRanges];
  __shared__ float wmax[kW];
  __shared__ double wsum[kW];
  __shared__ uint32_t wn[kW];
  __shared__ uint32_t first, listed, reach[kW], deep[2];
  __shared__ int lowest;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
  fill_tab(tab);
  if (blockIdx.x == 0 && tid == 0) *a.nleft = 0u;
  const sas_filter_params p = load_filter_params(a, row);
  const int64_t row0 = (int64_t)row * a.logits_stride;
  float v[Q][4];
  span_values<kT, kType, kSoft, Q>(a, p, row0, a.mask ? a.mask + (int64_t)row * a.mask_stride : nullptr, history_of(a, row), count,
                                         part * kIds, v);
  if (tid < kFilterRanges) {
    mass[tid] = 0ull;
    cnt[tid] = 0u;
  }
  if (tid == 0) {
    first = ~0u;
    listed = 0u;
    deep[0] = deep[1] = 0u;
  }
  const float neg = -__builtin_inff();
  float m = neg;
#pragma unroll
  for (int j = 0; j < Q; ++j) m = fmaxf(m, fmaxf(fmaxf(v[j][0], v[j][1]), fmaxf(v[j][2], v[j][3])));
  m = wave_max(m);
  if (lane == 0) wmax[wave] = m;
  __syncthreads();
  m = wmax[0];
#pragma unroll
  for (int w = 1; w < kW; ++w) m = fmaxf(m, wmax[w]);
  const int64_t at = (int64_t)row * a.parts + part;
  FilterPart *out = a.part + at;
  const Grid g = grid_of(p.temperature);
  const float top = range_of(m, g);
  const bool greedy = greedy_row(p), ranged = !greedy && g.plain && fabsf(top) < kFar && m > neg;
  const bool list = ranged && filters(p);
  // Masses are relative to the part's largest value: the difference is exact, so
  // equal values weigh exactly 1, and n of them exactly n.
  const double md = (double)m;
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
  uint32_t n = 0, best = ~0u;
#pragma unroll
  for (int j = 0; j < Q; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) n += v[j][i] > neg ? 1u : 0u;
  if (greedy) {
#pragma unroll
    for (int j = 0; j < Q; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (v[j][i] == m) best = min(best, (uint32_t)(part * kIds + 4 * (j * kT + tid) + i));
  }
  if (ranged) {
    const float hot = list ? (top - (float)(kFilterRanges - 1)) / g.inv_width : __uint_as_float(0x7F800000u);
#pragma unroll
    for (int j = 0; j < Q; ++j) {
      double u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u[i] = exp256(fmax(((double)v[j][i] - md) * g.per, kLeast), tab);
        sum[i] += u[i];
      }
      if (fmaxf(fmaxf(v[j][0], v[j][1]), fmaxf(v[j][2], v[j][3])) >= hot) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (v[j][i] >= hot) {
            const int d = (int)(top - range_of(v[j][i], g));
            // (a number below 2^51 in the low bits of its sum with 2^52)
            const uint64_t whole = (uint64_t)__double_as_longlong(fma(u[i], kUnit, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
            atomicAdd(&mass[d], (unsigned long long)whole);
            atomicAdd(&cnt[d], 1u);
          }
      }
    }
  }
  if (best != ~0u && m > neg) atomicMin(&first, best);
  const double s = wave_sum_d((sum[0] + sum[1]) + (sum[2] + sum[3]));
  n = wave_reduce(n, [](uint32_t x, uint32_t y) { return x + y; });
  if (lane == 0) {
    wsum[wave] = s;
    wn[wave] = n;
  }
  __syncthreads();
  // the list takes whole ranges, the largest values first
  if (list && wave == 0) {
    const uint32_t c0 = cnt[2 * lane], c1 = cnt[2 * lane + 1];
    uint32_t x = c0 + c1;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const uint32_t y = (uint32_t)__shfl_up((int)x, k, 64);
      if (lane >= k) x += y;
    }
    const uint64_t odd = __ballot(x <= (uint32_t)kList), even = __ballot(x - c1 <= (uint32_t)kList);
    const int no = odd == ~0ull ? 64 : __builtin_ctzll(~odd), ne = even == ~0ull ? 64 : __builtin_ctzll(~even);
    if (lane == 0) lowest = no + ne - 1;  // the last range whose running count fits, -1: none
  }
  if (list) {
    __syncthreads();
    for (int i = tid; i < kFilterRanges; i += kT) {
      a.range_mass[at * kFilterRanges + i] = mass[i];
      a.range_count[at * kFilterRanges + i] = cnt[i];
    }
  }
  float edge = list && lowest >= 0 ? (top - (float)lowest) / g.inv_width : __uint_as_float(0x7F800000u);
  if (list && p.top_k > 0 && lowest == kFilterRanges - 1) {
    // The ranges leave room in the list and top-k may reach below them: down to
    // a value that half a list of ids reaches, the smallest of the waves' J-th
    // largest of their lanes' maxima; or to the largest, if that is too far.
    const int J = kList / 2 / kW;
    float mine = neg;
#pragma unroll
    for (int j = 0; j < Q; ++j) mine = fmaxf(mine, fmaxf(fmaxf(v[j][0], v[j][1]), fmaxf(v[j][2], v[j][3])));
    const uint32_t key = wave_jth_largest_key(mine > neg ? okey(mine) : 0u, J);
    if (lane == 0) reach[wave] = key;
    __syncthreads();
    uint32_t t[2] = {~0u, 0u};
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      t[0] = min(t[0], reach[w]);
      t[1] = max(t[1], reach[w]);
    }
    if (t[0] == 0u) t[0] = kNegInf + 1u;  // few candidates: all of them
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t c = 0;
      const float least = fkey(t[k]);
#pragma unroll
      for (int j = 0; j < Q; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) c += t[k] && v[j][i] >= least ? 1u : 0u;
      c = wave_reduce(c, [](uint32_t x, uint32_t y) { return x + y; });
      if (lane == 0) atomicAdd(&deep[k], c);
    }
    __syncthreads();
    const int k = deep[0] <= (uint32_t)kList ? 0 : 1;
    if (t[k] && deep[k] <= (uint32_t)kList) edge = fminf(edge, fkey(t[k]));
  }
  if (list && lowest >= 0) {
#pragma unroll
    for (int j = 0; j < Q; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (v[j][i] >= edge) {
          const uint32_t to = atomicAdd(&listed, 1u);
          a.list[at * kList + to] =
              (uint64_t)okey(v[j][i]) << 32 | (uint32_t) ~(uint32_t)(part * kIds + 4 * (j * kT + tid) + i);
        }
  }
  __syncthreads();
  if (tid == 0) {
    FilterPart f;
    f.max = m;
    f.id = first;
    f.count = 0;
    f.mass = 0.0;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      f.count += (int32_t)wn[w];
      f.mass += wsum[w];
    }
    if (!ranged) f.mass = 0.0;
    f.listed = ranged ? (int32_t)listed : -1;
    f.edge = edge;
    f.top = ranged ? (int32_t)top : 0;
    *out = f;
  }
}

// (value range) of a key: 0 for m itself, kBins - 1 for the rest.
struct Scale {
  double m, inv_t, per_bin;
  int shift;
};
__device__ __forceinline__ int bin_of(uint32_t key, const Scale &s) {
  const double d = s.m - (double)fkey(key);
  const double t = d * s.per_bin;
  return key == okey((float)s.m) ? 0 : t < (double)(kBins - 1) ? (int)t : kBins - 1;  // (NaN: the rest)
}
// e^x, x <= 0; of -inf and NaN: 0.
__device__ __forceinline__ double mass_exp(double x) { return exp(fmax(x, -1100.0)); }
__device__ __forceinline__ double mass_of(uint32_t key, const Scale &s) {
  const float v = fkey(key);
  return v == (float)s.m ? 1.0 : mass_exp(((double)v - s.m) * s.inv_t);
}
__device__ __forceinline__ uint64_t units_of(double mass, const Scale &s) {
  return (uint64_t)__builtin_rint(__builtin_amdgcn_ldexp(mass, s.shift));
}

// The smallest key whose mass reaches min_p (the mass falls with the key).
__device__ __forceinline__ uint32_t least_key(double min_p, uint32_t top, const Scale &s) {
  const double least = fmin(min_p, 1.0);
  uint32_t lo = kNegInf, hi = top;  // hi reaches it, lo does not (or is no candidate's)
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (mass_of(mid, s) >= least) hi = mid;
    else lo = mid;
  }
  return hi;
}

// Every id of a larger key than `key`, and the first `take` of its own.
struct Edge {
  uint32_t key;
  uint32_t take;
};

struct RowShared {
  uint32_t count[kSpan / 2];  // history counts of a span's ids, 16 bits each
  unsigned long long mass[kBins];
  uint32_t cnt[kBins];
  unsigned long long red[kRowWaves][2];
  unsigned long long sel[4];
  unsigned long long part[kMaxFilterParts];
  unsigned long long ent[kEntries];   // listed ids: key << 32 | ~id
  unsigned long long entm[kEntries];  // and their masses
};

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t x, int s) { return (uint64_t)__shfl_xor((unsigned long long)x, s, 64); }

// Block-wide sums of two integers, on every thread.
__device__ __forceinline__ void block_sum2(RowShared &l, uint64_t &x, uint64_t &y) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) {
    x += shfl_xor64(x, s);
    y += shfl_xor64(y, s);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    l.red[threadIdx.x >> 6][0] = x;
    l.red[threadIdx.x >> 6][1] = y;
  }
  __syncthreads();
  x = y = 0;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) {
    x += l.red[w][0];
    y += l.red[w][1];
  }
}

// Inclusive block-wide prefix sum in thread order.
__device__ __forceinline__ uint64_t block_scan(RowShared &l, uint64_t x, uint64_t *total) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const uint64_t y = (uint64_t)__shfl_up((unsigned long long)x, s, 64);
    if (lane >= s) x += y;
  }
  __syncthreads();
  if (lane == 63) l.red[threadIdx.x >> 6][0] = x;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) {
    if (w < (int)(threadIdx.x >> 6)) before += l.red[w][0];
    all += l.red[w][0];
  }
  *total = all;
  return before + x;
}

// One row, one block.
template <int kType, bool kSoft>
struct Row {
  const FilterArgs &a;
  RowShared &l;
  const sas_filter_params &p;
  int64_t row0;
  const uint32_t *mask;
  History h;
  Scale s;

  // The keys of the thread's ids of span `q` (0: no candidate): quad j holds
  // ids q * kSpan + (j * kRowThreads + threadIdx.x) * 4 ..
  __device__ __forceinline__ int id0(int q, int j) const { return q * kSpan + (j * kRowThreads + (int)threadIdx.x) * 4; }
  __device__ __forceinline__ void keys(int q, uint32_t (&key)[kQuads][4]) const {
    float v[kQuads][4];
    span_values<kRowThreads, kType, kSoft, kQuads>(a, p, row0, mask, h, l.count, q * kSpan, v);
#pragma unroll
    for (int j = 0; j < kQuads; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) key[j][i] = v[j][i] > -__builtin_inff() ? okey(v[j][i]) : 0u;
  }
  __device__ __forceinline__ int spans() const { return (a.vocab + kSpan - 1) / kSpan; }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int q = 0; q < spans(); ++q) {
      uint32_t key[kQuads][4];
      keys(q, key);
#pragma unroll
      for (int j = 0; j < kQuads; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) f(key[j][i]);
    }
  }

  // The first bin b (of n in l.mass / l.cnt) at which the running mass (or,
  // with by_count, count) reaches need; before: what lies above it.  Bins
  // rise from the largest keys on.
  __device__ __forceinline__ int find(int n, bool by_count, uint64_t need, uint64_t *mass, uint64_t *count, int base = 0) const {
    __syncthreads();
    if (threadIdx.x < 64) {
      const int lane = threadIdx.x, per = n / 64;
      uint64_t m = 0, c = 0;
      for (int i = 0; i < per; ++i) {
        m += l.mass[base + lane * per + i];
        c += l.cnt[base + lane * per + i];
      }
      uint64_t mi = m, ci = c;
#pragma unroll
      for (int st = 1; st < 64; st <<= 1) {
        const uint64_t mu = (uint64_t)__shfl_up((unsigned long long)mi, st, 64), cu = (uint64_t)__shfl_up((unsigned long long)ci, st, 64);
        if (lane >= st) {
          mi += mu;
          ci += cu;
        }
      }
      const uint64_t upto = by_count ? ci : mi, own = by_count ? c : m;
      if (upto >= need && upto - own < need) {
        uint64_t mm = mi - m, cc = ci - c;
        int i = 0;
        for (; i < per - 1; ++i) {
          const uint64_t m1 = mm + l.mass[base + lane * per + i], c1 = cc + l.cnt[base + lane * per + i];
          if ((by_count ? c1 : m1) >= need) break;
          mm = m1;
          cc = c1;
        }
        l.sel[0] = (unsigned long long)(lane * per + i);
        l.sel[1] = mm;
        l.sel[2] = cc;
      }
    }
    __syncthreads();
    *mass = l.sel[1];
    *count = l.sel[2];
    return (int)l.sel[0];
  }

  // The edge at which the running mass (count) of the order reaches need,
  // from the histogram over bins in l.mass / l.cnt, which does not outlive it.
  // *mass (not by_count), *count: of the prefix up to the edge, its `take` in.
  __device__ __forceinline__ Edge edge(bool by_count, uint64_t need, uint64_t *mass, uint64_t *count) {
    uint64_t m0, c0;
    const int bin = find(kBins, by_count, need, &m0, &c0);
    // radix over the bin's keys, 8 bits a pass from the top
    uint32_t top = 0u;
    for (int sh = 24; sh >= 0; sh -= 8) {
      __syncthreads();
      for (int i = threadIdx.x; i < 256; i += kRowThreads) {
        l.mass[i] = 0ull;
        l.cnt[i] = 0u;
      }
      __syncthreads();
      const uint32_t above = sh == 24 ? 0u : ~0u << (sh + 8);
      each([&](uint32_t k) {
        if (k && (k & above) == top && bin_of(k, s) == bin) {
          const int d = 255 - (int)((k >> sh) & 0xFFu);
          atomicAdd(&l.mass[d], (unsigned long long)units_of(mass_of(k, s), s));
          atomicAdd(&l.cnt[d], 1u);
        }
      });
      uint64_t m1, c1;
      const int d = find(256, by_count, by_count ? need - c0 : need - m0, &m1, &c1);
      m0 += m1;
      c0 += c1;
      top |= (uint32_t)(255 - d) << sh;
    }
    const uint64_t unit = units_of(mass_of(top, s), s);
    const uint32_t n = l.cnt[255 - (top & 0xFFu)];
    uint64_t take = by_count ? need - c0 : unit ? (need - m0 + unit - 1) / unit : 1;
    take = min(max(take, (uint64_t)1), (uint64_t)n);
    *mass = m0 + take * unit;
    *count = c0 + take;
    return Edge{top, (uint32_t)take};
  }

  // The histogram over the bins of the row's candidates that rank up to `end`
  // (key 0: all); by_count: without masses.
  __device__ __forceinline__ void histogram(bool by_count, Edge end) {
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kRowThreads) {
      l.mass[i] = 0ull;
      l.cnt[i] = 0u;
    }
    __syncthreads();
    uint64_t rest = 0, nrest = 0;
    each([&](uint32_t k) {
      if (!k || k <= end.key) return;
      const int b = bin_of(k, s);
      const uint64_t u = by_count ? 0ull : units_of(mass_of(k, s), s);
      if (b == kBins - 1) {
        rest += u;
        ++nrest;
      } else {
        if (!by_count) atomicAdd(&l.mass[b], (unsigned long long)u);
        atomicAdd(&l.cnt[b], 1u);
      }
    });
    block_sum2(l, rest, nrest);
    if (threadIdx.x == 0) {
      l.mass[kBins - 1] = rest;
      l.cnt[kBins - 1] = (uint32_t)nrest;
      if (end.key) {
        const int b = bin_of(end.key, s);
        l.mass[b] += end.take * units_of(mass_of(end.key, s), s);
        l.cnt[b] += end.take;
      }
    }
    __syncthreads();
  }
};

// What a row's token is: written by one thread.
struct Result {
  const FilterArgs &a;
  int row;
  __device__ __forceinline__ void operator()(uint32_t id, double prob, uint64_t count) const {
    a.out_ids[row] = id;
    if (a.out_probs) a.out_probs[row] = prob;
    if (a.out_counts) a.out_counts[row] = (int32_t)count;
    if (a.out_flags) a.out_flags[row] = count ? 0u : SAS_FLAG_EMPTY_ROW;
  }
};

// The part of a row (of n, their kept masses in l.part) in which the running
// mass exceeds goal; before: what lies before it.
__device__ __forceinline__ int part_of(RowShared &l, int n, uint64_t goal, uint64_t *before) {
  const int per = (n + kRowThreads - 1) / kRowThreads, first = (int)threadIdx.x * per;
  uint64_t mine = 0, all;
  for (int i = first; i < min(first + per, n); ++i) mine += l.part[i];
  uint64_t run = block_scan(l, mine, &all) - mine;
  for (int i = first; i < min(first + per, n); ++i) {
    if (run <= goal && goal < run + l.part[i]) {
      l.sel[0] = (unsigned long long)i;
      l.sel[1] = run;
    }
    run += l.part[i];
  }
  __syncthreads();
  *before = l.sel[1];
  return (int)l.sel[0];
}

// The row by its values alone, read as often as it takes: right for every
// temperature, value and cut, and what the others fall back on.
template <int kType, bool kSoft>
__device__ __forceinline__ void row_by_values(Row<kType, kSoft> &R, const FilterArgs &a, RowShared &l, const sas_filter_params &p, int row,
                                           uint32_t top, uint64_t n, const Result &done) {
  const int tid = threadIdx.x;
  uint64_t zero = 0;
  Edge e{0u, 0u};  // no edge: every candidate
  uint64_t mass = 0, count = 0;
  if (p.top_k > 0 && (uint64_t)p.top_k < n) {
    R.histogram(true, e);
    e = R.edge(true, (uint64_t)p.top_k, &mass, &count);
  }
  if (p.top_p < 1.0) {
    R.histogram(false, e);
    mass = zero = 0;
    for (int i = tid; i < kBins; i += kRowThreads) mass += l.mass[i];
    block_sum2(l, mass, zero);
    const double need = ceil(fmax(p.top_p, 0.0) * (double)mass);
    const Edge f = R.edge(false, min(max((uint64_t)need, (uint64_t)1), mass), &mass, &count);
    if (!e.key || f.key > e.key || (f.key == e.key && f.take < e.take)) e = f;
  }
  if (p.min_p > 0.0) {
    const uint32_t hi = least_key(p.min_p, top, R.s);
    if (hi > e.key) e = Edge{hi, ~0u};
  }
  // what is kept of each span; the edge's ids count in ascending order
  uint64_t total = 0, kept = 0, ties = 0;
  const uint64_t unit = e.key ? units_of(mass_of(e.key, R.s), R.s) : 0;
  for (int q = 0; q < R.spans(); ++q) {
    uint32_t key[kQuads][4];
    R.keys(q, key);
    uint64_t m = 0, c = 0;
#pragma unroll
    for (int j = 0; j < kQuads; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t k = key[j][i];
        if (k > e.key) {
          m += units_of(mass_of(k, R.s), R.s);
          c += 1;
        } else if (k && k == e.key) {
          c += 1ull << 32;
        }
      }
    block_sum2(l, m, c);
    const uint64_t here = min(c >> 32, (uint64_t)e.take - ties);
    ties += here;
    kept += (c & 0xFFFFFFFFull) + here;
    m += here * unit;
    total += m;
    if (tid == 0) l.part[q] = m;
  }
  __syncthreads();
  // the draw: the first kept id whose running mass exceeds u * total
  const double u = a.uniforms[row];
  uint64_t goal = (uint64_t)fmax(u * (double)total, 0.0);
  goal = min(goal, total - 1);
  int q = 0;
  uint64_t before = 0;
  while (q < R.spans() - 1 && before + l.part[q] <= goal) before += l.part[q++];
  // the edge's ids in the spans before
  uint64_t tie0 = 0;
  if (e.key && e.take != ~0u) {
    for (int s = 0; s < q; ++s) {
      uint32_t key[kQuads][4];
      R.keys(s, key);
#pragma unroll
      for (int j = 0; j < kQuads; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) tie0 += key[j][i] == e.key ? 1 : 0;
    }
    zero = 0;
    block_sum2(l, tie0, zero);
  }
  uint32_t key[kQuads][4];
  R.keys(q, key);
  for (int j = 0; j < kQuads; ++j) {
    uint64_t t = 0, all = 0;
    uint64_t mine[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) t += key[j][i] && key[j][i] == e.key ? 1 : 0;
    uint64_t tie = tie0 + block_scan(l, t, &all) - t;
    tie0 += all;
    uint64_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t k = key[j][i];
      bool in = k > e.key;
      if (k && k == e.key) in = tie++ < e.take;
      mine[i] = in ? units_of(mass_of(k, R.s), R.s) : 0;
      m += mine[i];
    }
    uint64_t run = before + block_scan(l, m, &all) - m;
    if (run <= goal && goal < run + m) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (run <= goal && goal < run + mine[i])
          done((uint32_t)(R.id0(q, j) + i), mass_of(key[j][i], R.s) / __builtin_amdgcn_ldexp((double)total, -a.shift), kept);
        run += mine[i];
      }
    }
    before += all;
  }
}

// The entry that ends a prefix of those of the first c entries of l.ent that
// are `in`, ranked by (key, id): the one of rank need (by_count), else the first at which the
// running mass reaches need.  Radix passes of 8 bits from the highest in which
// the entries differ.  *mass, *count: of the entries up to it.
template <typename R, typename In>
__device__ __forceinline__ uint64_t end_of(const R &row, RowShared &l, int c, In in, bool by_count, uint64_t need, uint64_t *mass, uint64_t *count) {
  constexpr int kBase = 256;
  const int tid = threadIdx.x;
  uint64_t all = ~0ull, any = 0;
  for (int i = tid; i < c; i += kRowThreads)
    if (in(l.ent[i])) {
      all &= l.ent[i];
      any |= l.ent[i];
    }
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) {
    all &= shfl_xor64(all, s);
    any |= shfl_xor64(any, s);
  }
  __syncthreads();
  if ((tid & 63) == 0) {
    l.red[tid >> 6][0] = all;
    l.red[tid >> 6][1] = any;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) {
    all &= l.red[w][0];
    any |= l.red[w][1];
  }
  int sh = all == any ? 0 : max(63 - __builtin_clzll(all ^ any) - 7, 0);
  uint64_t high = sh + 8 >= 64 ? 0ull : ~0ull << (sh + 8), at = all & high, m0 = 0, c0 = 0;
  for (;;) {
    __syncthreads();
    if (tid < 256) {
      l.mass[kBase + tid] = 0ull;
      l.cnt[kBase + tid] = 0u;
    }
    __syncthreads();
    for (int i = tid; i < c; i += kRowThreads) {
      const uint64_t e = l.ent[i];
      if ((e & high) != at || !in(e)) continue;
      const int d = 255 - (int)((e >> sh) & 0xFFu);
      atomicAdd(&l.mass[kBase + d], l.entm[i]);
      atomicAdd(&l.cnt[kBase + d], 1u);
    }
    uint64_t m1, c1;
    const int d = row.find(256, by_count, by_count ? need - c0 : need - m0, &m1, &c1, kBase);
    m0 += m1;
    c0 += c1;
    at |= (uint64_t)(255 - d) << sh;
    if (l.cnt[kBase + d] == 1u || sh == 0) {
      // one entry (they differ): its low bits
      const uint64_t low = ~0ull << sh;
      __syncthreads();
      for (int i = tid; i < c; i += kRowThreads)
        if ((l.ent[i] & low) == at && in(l.ent[i])) {
          l.sel[0] = l.ent[i];
          l.sel[1] = l.entm[i];
        }
      __syncthreads();
      *mass = m0 + l.sel[1];
      *count = c0 + 1;
      return l.sel[0];
    }
    const int down = min(sh, 8);
    high = ~0ull << sh;
    sh -= down;
  }
}

// The row's largest key, from its parts' maxima; *candidates: how many there are.
__device__ __forceinline__ uint32_t row_top(const FilterArgs &a, RowShared &l, int row, uint64_t *candidates) {
  const FilterPart *parts = a.part + (int64_t)row * a.parts;
  uint64_t best = 0, n = 0;
  for (int i = threadIdx.x; i < a.parts; i += kRowThreads) {
    const FilterPart f = parts[i];
    if (f.max > -__builtin_inff()) {
      best = max(best, (uint64_t)okey(f.max));
      n += (uint64_t)f.count;
    }
  }
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) {
    best = max(best, shfl_xor64(best, s));
    n += shfl_xor64(n, s);
  }
  if ((threadIdx.x & 63) == 0) {
    l.red[threadIdx.x >> 6][0] = best;
    l.red[threadIdx.x >> 6][1] = n;
  }
  __syncthreads();
  n = 0;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) {
    best = max(best, (uint64_t)l.red[w][0]);
    n += l.red[w][1];
  }
  *candidates = n;
  return (uint32_t)best;
}

// A cut row by what its parts left, where the merge planned its ranges (x.planned)
// and `n` candidates reach down from key `top`; false where that does not tell.
template <int kType, bool kSoft>
__device__ __forceinline__ bool row_by_parts(Row<kType, kSoft> &R, const FilterArgs &a, RowShared &l, const sas_filter_params &p, const FilterLeft &x, int row,
                                             uint32_t top, uint64_t n, const Result &done) {
  const int tid = threadIdx.x;
  const FilterPart *parts = a.part + (int64_t)row * a.parts;
  uint64_t zero = 0;
  const Grid g = grid_of(p.temperature);
  const float mrange = range_of(fkey(top), g);
  const bool by_k = p.top_k > 0 && (uint64_t)p.top_k < n, by_p = p.top_p < 1.0, by_min = p.min_p > 0.0;
  // a part's factor to the row's units
  auto scale_of = [&](const FilterPart &f) { return mass_of(okey(f.max), R.s); };
  uint64_t all = 0;
  for (int i = tid; i < a.parts; i += kRowThreads) {
    const FilterPart f = parts[i];
    if (f.listed >= 0) all += (uint64_t)__builtin_rint(__builtin_amdgcn_ldexp(f.mass * scale_of(f), a.shift));
  }
  block_sum2(l, all, zero);
  uint64_t last = 0;      // every id whose (key, ~id) reaches it is kept
  const int log_span = 31 - __builtin_clz(a.span);
  // the ranges of all parts, in the row's units
  for (int i = tid; i < kFilterRanges; i += kRowThreads) {
    l.mass[i] = 0ull;
    l.cnt[i] = 0u;
  }
  __syncthreads();
  // fn(part, range, count, mass in the row's units) of every range that has ids, four
  // ranges' loads in flight together
  auto each_range = [&](auto fn) {
    for (int i0 = tid; i0 < a.parts * kFilterRanges; i0 += 4 * kRowThreads) {
      uint32_t c[4];
      uint64_t w[4];
      FilterPart f[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = min(i0 + k * kRowThreads, a.parts * kFilterRanges - 1);
        const int64_t at = (int64_t)row * a.parts * kFilterRanges + i;
        c[k] = a.range_count[at];
        w[k] = a.range_mass[at];
        f[k] = parts[i / kFilterRanges];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + k * kRowThreads;
        const int d = (int)mrange - f[k].top + i % kFilterRanges;
        if (i >= a.parts * kFilterRanges || f[k].listed < 0 || !(f[k].max > -__builtin_inff()) || c[k] == 0u || d >= kFilterRanges) continue;
        fn(i / kFilterRanges, d, c[k],
           (uint64_t)__builtin_rint(__builtin_amdgcn_ldexp((double)w[k] * scale_of(f[k]), a.shift - kFilterShift)));
      }
    }
  };
  each_range([&](int, int d, uint32_t c, uint64_t u) {
    atomicAdd(&l.cnt[d], c);
    atomicAdd(&l.mass[d], (unsigned long long)u);
  });
  __syncthreads();
  uint64_t have = 0, havem = 0;
  for (int i = tid; i < kFilterRanges; i += kRowThreads) {
    have += l.cnt[i];
    havem += l.mass[i];
  }
  block_sum2(l, have, havem);
  const uint32_t least = by_min ? least_key(p.min_p, top, R.s) : 0u;
  // the ids of the planned ranges
  const int entries = (int)a.found[row];
  if (entries > kEntries) return false;
  for (int i = tid; i < entries; i += kRowThreads) {
    const uint64_t e = a.ids[(int64_t)row * kEntries + i];
    l.ent[i] = e;
    l.entm[i] = units_of(mass_of((uint32_t)(e >> 32), R.s), R.s);
  }
  __syncthreads();
  auto planned = [&](int bin) { return bin < kFilterRanges && ((x.ranges[bin >> 5] >> (bin & 31)) & 1u) != 0u; };
  auto bin_of_entry = [&](uint64_t e) { return (int)(mrange - range_of(fkey((uint32_t)(e >> 32)), g)); };
  // the ends of the prefixes of top-k and top-p
  bool known = true;
  auto prefix = [&](bool by_count, uint64_t need, uint64_t *mass) {
    if (need > (by_count ? have : havem)) {
      known = false;
      return;
    }
    uint64_t m0, c0, m1, c1;
    const int bin = R.find(kFilterRanges, by_count, need, &m0, &c0);
    known = planned(bin);
    if (!known) return;
    // (the range's mass was rounded as a whole, its ids' one by one)
    uint64_t sum = 0;
    zero = 0;
    for (int i = tid; i < entries; i += kRowThreads) sum += bin_of_entry(l.ent[i]) == bin ? l.entm[i] : 0ull;
    block_sum2(l, sum, zero);
    known = sum > 0;
    if (!known) return;
    last = max(last, end_of(R, l, entries, [&](uint64_t e) { return bin_of_entry(e) == bin; }, by_count,
                            by_count ? need - c0 : min(need - m0, sum), &m1, &c1));
    *mass = m0 + m1;
  };
  uint64_t mass = all;
  if (by_k) prefix(true, (uint64_t)p.top_k, &mass);
  if (known && by_p) {
    const uint64_t need = (uint64_t)ceil(fmax(p.top_p, 0.0) * (double)mass);
    prefix(false, min(max(need, (uint64_t)1), mass), &mass);
  }
  if (known && by_min && (uint64_t)least << 32 > last) {
    last = (uint64_t)least << 32;
    known = mrange - range_of(fkey(least), g) < (float)kFilterRanges;
  }
  if (!known) return false;
  // what is kept of each part: of the ranges above the end's all, of its own
  // by its ids
  const int bin = (int)(mrange - range_of(fkey((uint32_t)(last >> 32)), g));
  if (!planned(bin)) return false;
  uint64_t total = 0, kept = 0;
  for (int i = tid; i < a.parts; i += kRowThreads) l.part[i] = 0ull;
  __syncthreads();
  each_range([&](int part, int d, uint32_t c, uint64_t u) {
    if (d >= bin) return;
    total += u;
    kept += c;
    atomicAdd(&l.part[part], (unsigned long long)u);
  });
  __syncthreads();
  for (int i = tid; i < entries; i += kRowThreads)
    if (l.ent[i] >= last && bin_of_entry(l.ent[i]) == bin) {
      total += l.entm[i];
      ++kept;
      atomicAdd(&l.part[~(uint32_t)l.ent[i] >> log_span], l.entm[i]);
    }
  block_sum2(l, total, kept);
  // the draw: the part, then the id
  uint64_t goal = (uint64_t)fmax(a.uniforms[row] * (double)total, 0.0), before;
  goal = min(goal, total - 1);
  const int q = part_of(l, a.parts, goal, &before);
  const double whole = __builtin_amdgcn_ldexp((double)total, -a.shift);
  // the part's values again: its kept ids' masses, and the goal as a share of them
  constexpr int kDraw = 8192 / (4 * kRowThreads);  // quads of the longest part
  float v[kDraw][4];
  const int id0 = q * a.span;
  span_values<kRowThreads, kType, kSoft, kDraw>(a, p, R.row0, R.mask, R.h, l.count, id0, v);
  uint64_t u[kDraw][4], run[kDraw], sums = 0;
#pragma unroll
  for (int j = 0; j < kDraw; ++j) {
    uint64_t sum = 0, of_all;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = 4 * (j * kRowThreads + tid) + i;
      const uint32_t key = okey(v[j][i]);
      const bool in = at < a.span && v[j][i] > -__builtin_inff() && ((uint64_t)key << 32 | (uint32_t) ~(uint32_t)(id0 + at)) >= last;
      u[j][i] = in ? units_of(mass_of(key, R.s), R.s) : 0ull;
      sum += u[j][i];
    }
    run[j] = sums + block_scan(l, sum, &of_all) - sum;
    sums += of_all;
  }
  uint64_t target = (uint64_t)((double)(goal - before) * ((double)sums / (double)l.part[q]));
  target = min(target, sums - 1);
#pragma unroll
  for (int j = 0; j < kDraw; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (run[j] <= target && target < run[j] + u[j][i])
        done((uint32_t)(id0 + 4 * (j * kRowThreads + tid) + i), mass_of(okey(v[j][i]), R.s) / whole, kept);
      run[j] += u[j][i];
    }
  return true;
}

// The rows that the merge left: each has a candidate, and none is greedy.
template <int kType, bool kSoft>
__global__ __launch_bounds__(kRowThreads) void filter_rest_kernel(const FilterArgs a) {
  __shared__ RowShared l;
  if (blockIdx.x >= *a.nleft) return;
  const FilterLeft x = a.left[blockIdx.x];
  const int row = x.row;
  const sas_filter_params p = load_filter_params(a, row);
  Row<kType, kSoft> R{a, l, p, (int64_t)row * a.logits_stride, a.mask ? a.mask + (int64_t)row * a.mask_stride : nullptr,
                      history_of(a, row), Scale{}};
  const Result done{a, row};
  uint64_t n;
  const uint32_t top = row_top(a, l, row, &n);
  R.s = Scale{(double)fkey(top), 1.0 / p.temperature, 8.0 / p.temperature, a.shift};
  if (!x.planned || !row_by_parts<kType, kSoft>(R, a, l, p, x, row, top, n, done))
    row_by_values<kType, kSoft>(R, a, l, p, row, top, n, done);
}

// ----------------------------------------------------------------- merge --
// One row, four waves.  The lists' entries stay in registers; every wave
// finds the same ends of the prefixes from the ranges' sums in LDS, so that
// few barriers are left.  Rows whose ends the lists do not hold, or whose
// values are out of the ranges' scope, are left to the rest kernel.
constexpr int kMergeEntries = 16;                          // a thread's
constexpr int kMergeMost = kMergeEntries * kThreads;       // entries of a row
constexpr int kMergeSome = 512;                            // ids of one range, or of one part

struct MergeShared {
  double tab[kTab];
  uint64_t red[kWaves][3];
  unsigned long long mass[kFilterRanges];
  uint32_t cnt[kFilterRanges];
  unsigned long long part[kMaxFilterParts];
  unsigned long long ent[kMergeSome], entm[kMergeSome];
  uint64_t end[2];
  uint32_t nsome;
};

template <typename Op>
__device__ __forceinline__ uint64_t wave_reduce64(uint64_t x, Op op) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) x = op(x, shfl_xor64(x, s));
  return x;
}
__device__ __forceinline__ uint64_t wave_scan64(uint64_t x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const uint64_t y = (uint64_t)__shfl_up((unsigned long long)x, s, 64);
    if (lane >= s) x += y;
  }
  return x;
}
__device__ __forceinline__ uint64_t lane64(uint64_t x, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}

// The merge's bins: 96 ranges, then 32 of 16 ranges each, the last without end.
__device__ __forceinline__ int merge_bin(float d) {
  return d < 96.0f ? (int)d : d < 592.0f ? 96 + ((int)d - 96) / 16 : kFilterRanges - 1;
}

template <int kType, bool kSoft, int Q>
__global__ __launch_bounds__(kThreads) void filter_merge_kernel(const FilterArgs a) {
  constexpr int kIds = 4 * Q * kThreads;
  const int kList = 1 << a.log_list;
  constexpr int kLogIds = Q == 8 ? 13 : Q == 4 ? 12 : 11;
  static_assert(kIds == 1 << kLogIds, "a power of two");
  __shared__ MergeShared l;
  __shared__ uint32_t hcount[kIds / 2];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const FilterPart *parts = a.part + (int64_t)row * a.parts;
  const uint64_t *lists = a.list + (int64_t)row * a.parts * kList;
  const int slots = a.parts * kList;
  // what the parts left: their entries (read before it is known how many hold)
  uint64_t e[kMergeEntries];
#pragma unroll
  for (int i = 0; i < kMergeEntries; ++i) e[i] = i * kThreads + tid < slots ? lists[i * kThreads + tid] : 0ull;
  const sas_filter_params p = load_filter_params(a, row);
  fill_tab(l.tab);
  if (tid < kFilterRanges) {
    l.mass[tid] = 0ull;
    l.cnt[tid] = 0u;
  }
  uint64_t best = 0, n = 0;
  uint32_t edge = 0;
  for (int i = tid; i < a.parts; i += kThreads) {
    const FilterPart f = parts[i];
    if (f.max > -__builtin_inff()) {
      best = max(best, (uint64_t)okey(f.max) << 32 | (uint32_t)~f.id);
      n += (uint64_t)f.count;
      edge = max(edge, f.listed < 0 ? okey(f.max) + 1u : okey(f.edge));
    }
  }
  auto more = [](uint64_t x, uint64_t y) { return x > y ? x : y; };
  auto plus = [](uint64_t x, uint64_t y) { return x + y; };
  best = wave_reduce64(best, more);
  n = wave_reduce64(n, plus);
  edge = wave_max_u32(edge);
  if (lane == 0) {
    l.red[wave][0] = best;
    l.red[wave][1] = n;
    l.red[wave][2] = edge;
  }
  __syncthreads();
  best = n = 0;
  edge = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    best = more(best, l.red[w][0]);
    n += l.red[w][1];
    edge = max(edge, (uint32_t)l.red[w][2]);
  }
  const Result done{a, row};
  if (best == 0 || greedy_row(p)) {
    if (tid == 0) done(best ? ~(uint32_t)best : SAS_NO_TOKEN, best ? 1.0 : 0.0, best ? 1 : 0);
    return;
  }
  // leaves the row to the rest kernel, by its values alone
  auto leave = [&]() {
    if (tid == 0) a.left[atomicAdd(a.nleft, 1u)] = FilterLeft{row, 0u, {0u, 0u, 0u, 0u}};
  };
  const uint32_t top = (uint32_t)(best >> 32);
  const Grid g = grid_of(p.temperature);
  const float mrange = range_of(fkey(top), g);
  if (!g.plain || !(mrange >= kNear && mrange < kFar)) return leave();
  // the mass of a value (of a part's largest: what its own masses count in)
  const double m = (double)fkey(top);
  auto mass_at = [&](double v) { return exp256(fmax((v - m) * g.per, kLeast), l.tab); };
  auto units = [&](double mass) { return (uint64_t)__builtin_rint(__builtin_amdgcn_ldexp(mass, a.shift)); };
  const bool by_k = p.top_k > 0 && (uint64_t)p.top_k < n, by_p = p.top_p < 1.0, by_min = p.min_p > 0.0;
  const bool cut = by_k || by_p || by_min;
  // The parts' masses in the row's units.  Where nothing is cut the draw goes by
  // them, then by the units of the chosen part's ids: a part whose largest value
  // rounds to none has no id to draw, though its sum may round to many.
  uint64_t all = 0;
  for (int i = tid; i < a.parts; i += kThreads) {
    const FilterPart f = parts[i];
    const bool none = f.listed < 0 || (!cut && units(mass_at((double)f.max)) == 0ull);
    const uint64_t u = none ? 0ull : units(f.mass * mass_at((double)f.max));
    l.part[i] = cut ? 0ull : u;
    all += u;
  }
  // the entries that count: all there are from `edge` on
  uint64_t u[kMergeEntries];
  bool known = slots <= kMergeMost;
  if (cut && known) {
#pragma unroll
    for (int i = 0; i < kMergeEntries; ++i) {
      const int at = i * kThreads + tid;
      u[i] = 0ull;
      if (at >= slots) continue;
      const float v = fkey((uint32_t)(e[i] >> 32)), d = mrange - range_of(v, g);
      const bool in = (at & (kList - 1)) < max(parts[at >> a.log_list].listed, 0) && (uint32_t)(e[i] >> 32) >= edge;
      e[i] = in ? e[i] : 0ull;
      if (!in) continue;
      u[i] = units(mass_at((double)v));
      atomicAdd(&l.mass[merge_bin(d)], (unsigned long long)u[i]);
      atomicAdd(&l.cnt[merge_bin(d)], 1u);
    }
  }
  all = wave_reduce64(all, plus);
  __syncthreads();  // (red is read above)
  if (lane == 0) l.red[wave][0] = all;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all += l.red[w][0];
  uint64_t last = 0, total = all, kept = n;
  if (cut) {
    // the running sums over the ranges, two a lane
    const uint64_t m0 = l.mass[2 * lane], m1 = l.mass[2 * lane + 1], c0 = l.cnt[2 * lane], c1 = l.cnt[2 * lane + 1];
    const uint64_t mrun = wave_scan64(m0 + m1), crun = wave_scan64(c0 + c1);
    const uint64_t havem = lane64(mrun, 63), have = lane64(crun, 63);
    uint64_t mass = all;
    // the entry that ends a prefix: its range, then its place among the range's
    auto prefix = [&](bool by_count, uint64_t need) {
      if (need > (by_count ? have : havem)) {
        known = false;
        return;
      }
      const uint64_t run = by_count ? crun : mrun, second = by_count ? c1 : m1;
      const int at = __builtin_ctzll(__ballot(run >= need));
      const bool late = lane64(run, at) - lane64(second, at) < need;
      const int bin = 2 * at + (late ? 1 : 0);
      const uint64_t mb = lane64(mrun, at) - lane64(m1, at) - (late ? 0ull : lane64(m0, at));
      const uint64_t cb = lane64(crun, at) - lane64(c1, at) - (late ? 0ull : lane64(c0, at));
      if (l.cnt[bin] > (uint32_t)kMergeSome) {
        known = false;
        return;
      }
      __syncthreads();
      if (tid == 0) l.nsome = 0u;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kMergeEntries; ++i)
        if (e[i] && merge_bin(mrange - range_of(fkey((uint32_t)(e[i] >> 32)), g)) == bin) {
          const uint32_t to = atomicAdd(&l.nsome, 1u);
          l.ent[to] = e[i];
          l.entm[to] = u[i];
        }
      __syncthreads();
      const int c = (int)l.nsome;
      const uint64_t rest = need - (by_count ? cb : mb);
      for (int t = tid; t < c; t += kThreads) {
        const uint64_t mine = l.ent[t], own = l.entm[t];
        uint64_t before = 0, rank = 0;
#pragma unroll 4
        for (int i = 0; i < c; ++i) {
          const bool first = l.ent[i] > mine;
          before += first ? l.entm[i] : 0ull;
          rank += first ? 1 : 0;
        }
        if (by_count ? rank + 1 == rest : before < rest && rest <= before + own) {
          l.end[0] = mine;
          l.end[1] = before + own;
        }
      }
      __syncthreads();
      last = more(last, l.end[0]);
      mass = mb + l.end[1];
    };
    if (known && by_k) prefix(true, (uint64_t)p.top_k);
    if (known && by_p) {
      const uint64_t need = (uint64_t)ceil(fmax(p.top_p, 0.0) * (double)mass);
      prefix(false, min(max(need, (uint64_t)1), mass));
    }
    uint32_t hi = top;
    if (by_min) {
      // the smallest key whose mass reaches min_p, 64 at a time
      const double least = fmin(p.min_p, 1.0);
      uint32_t lo = kNegInf;
      while (hi - lo > 1) {
        const uint32_t step = max((hi - lo) / 65u, 1u), key = lo + step * (uint32_t)(lane + 1);
        const uint64_t reach = __ballot(key >= hi || key < lo || mass_at((double)fkey(key)) >= least);
        const int k = reach ? __builtin_ctzll(reach) : 64;
        const uint32_t to = lo + step * (uint32_t)(k + 1);
        if (k < 64 && to < hi && to > lo) hi = to;
        lo = lo + step * (uint32_t)k;
      }
      if (known && (uint64_t)hi << 32 > last) {
        last = (uint64_t)hi << 32;
        known = hi >= edge;
      }
    }
    if (!known) {
      // the ranges that the ends lie in, from the ranges of all parts
      __syncthreads();
      if (tid < kFilterRanges) {
        l.mass[tid] = 0ull;
        l.cnt[tid] = 0u;
      }
      __syncthreads();
      for (int i = tid; i < a.parts * kFilterRanges; i += kThreads) {
        const FilterPart f = parts[i / kFilterRanges];
        const int64_t at = (int64_t)row * a.parts * kFilterRanges + i;
        const uint32_t c = a.range_count[at];
        const uint64_t w = a.range_mass[at];
        const int d = (int)mrange - f.top + i % kFilterRanges;
        if (f.listed < 0 || !(f.max > -__builtin_inff()) || c == 0u || d >= kFilterRanges) continue;
        atomicAdd(&l.cnt[d], c);
        atomicAdd(&l.mass[d], (unsigned long long)__builtin_rint(__builtin_amdgcn_ldexp((double)w * mass_at((double)f.max), a.shift - kFilterShift)));
      }
      __syncthreads();
      if (wave > 0) return;
      const uint64_t rm0 = l.mass[2 * lane], rm1 = l.mass[2 * lane + 1], rc0 = l.cnt[2 * lane], rc1 = l.cnt[2 * lane + 1];
      const uint64_t mr = wave_scan64(rm0 + rm1), cr = wave_scan64(rc0 + rc1);
      // the range in which a running sum reaches need (kFilterRanges: none)
      auto range_at = [&](uint64_t run, uint64_t second, uint64_t need) {
        const uint64_t hit = __ballot(run >= need);
        if (!hit) return (int)kFilterRanges;
        const int at = __builtin_ctzll(hit);
        return 2 * at + (lane64(run, at) - lane64(second, at) < need ? 1 : 0);
      };
      FilterLeft x{row, 0u, {0u, 0u, 0u, 0u}};
      bool sure = true;
      uint64_t ids = 0, low = all, high = all;
      auto plan = [&](int bin) {
        if (bin >= kFilterRanges) {
          sure = false;
          return;
        }
        if (!((x.ranges[bin >> 5] >> (bin & 31)) & 1u)) ids += l.cnt[bin];
        x.ranges[bin >> 5] |= 1u << (bin & 31);
      };
      if (by_k) {
        const int bin = range_at(cr, rc1, (uint64_t)p.top_k);
        plan(bin);
        if (sure) {
          // top-p's share is of a mass between the ranges' above the end and with it
          high = lane64(mr, bin >> 1) - (bin & 1 ? 0ull : lane64(rm1, bin >> 1));
          low = high - l.mass[bin];
        }
      }
      if (by_p && sure) {
        auto share = [&](uint64_t of) { return max((uint64_t)ceil(fmax(p.top_p, 0.0) * (double)of), (uint64_t)1); };
        const int from = range_at(mr, rm1, share(low)), to = range_at(mr, rm1, min(share(high), lane64(mr, 63)));
        for (int bin = from; bin <= to && sure; ++bin) plan(bin);
      }
      if (by_min) plan((int)fminf(mrange - range_of(fkey(hi), g), (float)kFilterRanges));
      if (sure && ids <= (uint64_t)kEntries) x.planned = 1u;
      if (lane == 0) {
        a.found[row] = 0u;
        a.left[atomicAdd(a.nleft, 1u)] = x;
      }
      return;
    }
    total = kept = 0;
#pragma unroll
    for (int i = 0; i < kMergeEntries; ++i)
      if (e[i] && e[i] >= last) {
        total += u[i];
        ++kept;
        atomicAdd(&l.part[~(uint32_t)e[i] >> kLogIds], (unsigned long long)u[i]);
      }
    total = wave_reduce64(total, plus);
    kept = wave_reduce64(kept, plus);
    __syncthreads();
    if (lane == 0) {
      l.red[wave][0] = total;
      l.red[wave][1] = kept;
    }
    if (tid == 0) l.nsome = 0u;
    __syncthreads();
    total = kept = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      total += l.red[w][0];
      kept += l.red[w][1];
    }
  }
  // the draw: the part (every wave finds it), then the id
  const double whole = __builtin_amdgcn_ldexp((double)total, -a.shift);
  const uint64_t goal = min((uint64_t)fmax(a.uniforms[row] * (double)total, 0.0), total - 1);
  uint64_t before = 0;
  int q = a.parts - 1;
  for (int i0 = 0; i0 < a.parts; i0 += 64) {
    const uint64_t mine = i0 + lane < a.parts ? l.part[i0 + lane] : 0ull, run = before + wave_scan64(mine);
    const uint64_t hit = __ballot(goal < run);
    if (hit) {
      const int w = __builtin_ctzll(hit);
      q = i0 + w;
      before = lane64(run, w) - lane64(mine, w);
      break;
    }
    before = lane64(run, 63);
  }
  if (cut) {
#pragma unroll
    for (int i = 0; i < kMergeEntries; ++i)
      if (e[i] && e[i] >= last && (int)(~(uint32_t)e[i] >> kLogIds) == q) {
        const uint32_t to = atomicAdd(&l.nsome, 1u);  // (<= kList)
        l.ent[to] = e[i];
        l.entm[to] = u[i];
      }
    __syncthreads();
    if (tid < (int)l.nsome) {
      const uint32_t mine = ~(uint32_t)l.ent[tid];
      uint64_t run = before;
      for (int i = 0; i < (int)l.nsome; ++i) run += ~(uint32_t)l.ent[i] < mine ? l.entm[i] : 0ull;
      if (run <= goal && goal < run + l.entm[tid]) done(mine, mass_at((double)fkey((uint32_t)(l.ent[tid] >> 32))) / whole, kept);
    }
    return;
  }
  // nothing is cut: the part's values again, the goal as a share of their masses
  float v[Q][4];
  span_values<kThreads, kType, kSoft, Q>(a, p, (int64_t)row * a.logits_stride, a.mask ? a.mask + (int64_t)row * a.mask_stride : nullptr,
                                         history_of(a, row), hcount, q * kIds, v);
  uint64_t sums = 0;
  // (ids rise with the quad, then the thread: a quad's sums over the block first)
  uint64_t quad[Q];
#pragma unroll
  for (int j = 0; j < Q; ++j) {
    uint64_t s = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) s += v[j][i] > -__builtin_inff() ? units(mass_at((double)v[j][i])) : 0ull;
    quad[j] = wave_scan64(s);
    if (lane == 63) l.mass[j * kWaves + wave] = quad[j];
    quad[j] -= s;
  }
  __syncthreads();
  for (int i = 0; i < Q * kWaves; ++i) sums += l.mass[i];
  const uint64_t target = min((uint64_t)((double)(goal - before) * ((double)sums / (double)l.part[q])), sums - 1);
  uint64_t base = 0;
#pragma unroll
  for (int j = 0; j < Q; ++j) {
    for (int w = 0; w < wave; ++w) base += l.mass[j * kWaves + w];
    uint64_t run = base + quad[j];
    for (int w = wave; w < kWaves; ++w) base += l.mass[j * kWaves + w];
    if (target < run) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t x = v[j][i] > -__builtin_inff() ? units(mass_at((double)v[j][i])) : 0ull;
      if (run <= target && target < run + x) done((uint32_t)(q * kIds + 4 * (j * kThreads + tid) + i), mass_at((double)v[j][i]) / whole, kept);
      run += x;
    }
  }
}

// The ids of the planned ranges of the rows left: a part at a time, on the
// whole chip (one block a row read 16,384 ids in 5 us).
template <int kType, bool kSoft, int Q>
__global__ __launch_bounds__(kThreads) void filter_gather_kernel(const FilterArgs a) {
  constexpr int kIds = 4 * Q * kThreads;
  __shared__ uint32_t count[kIds / 2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int items = (int)*a.nleft * a.parts;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const FilterLeft x = a.left[item / a.parts];
    const int part = item % a.parts;
    if (!x.planned) continue;
    const FilterPart *parts = a.part + (int64_t)x.row * a.parts;
    // the row's first range, as the merge has it
    float m = -__builtin_inff();
    for (int i = lane; i < a.parts; i += 64) m = fmaxf(m, parts[i].max);
    m = wave_max(m);
    const sas_filter_params p = load_filter_params(a, x.row);
    const Grid g = grid_of(p.temperature);
    const float mrange = range_of(m, g);
    const FilterPart f = parts[part];
    if (f.listed < 0 || !(f.max > -__builtin_inff())) continue;
    bool any = false;
    for (int d = lane; d < kFilterRanges; d += 64) {
      const int i = d - (int)mrange + f.top;
      any = any || ((x.ranges[d >> 5] >> (d & 31)) & 1u && i >= 0 && i < kFilterRanges &&
                    a.range_count[((int64_t)x.row * a.parts + part) * kFilterRanges + i] > 0u);
    }
    if (!__ballot(any)) continue;  // (the same in every wave)
    float v[Q][4];
    __syncthreads();
    span_values<kThreads, kType, kSoft, Q>(a, p, (int64_t)x.row * a.logits_stride,
                                           a.mask ? a.mask + (int64_t)x.row * a.mask_stride : nullptr, history_of(a, x.row), count,
                                           part * kIds, v);
    uint32_t hits = 0;
#pragma unroll
    for (int j = 0; j < Q; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float d = mrange - range_of(v[j][i], g);
        const int bin = d < (float)kFilterRanges ? (int)d : 0;
        const uint32_t word = bin < 64 ? (bin < 32 ? x.ranges[0] : x.ranges[1]) : (bin < 96 ? x.ranges[2] : x.ranges[3]);
        hits |= (d < (float)kFilterRanges ? (word >> (bin & 31)) & 1u : 0u) << (4 * j + i);
      }
    const uint32_t mine = __popc(hits);
    uint32_t upto = mine;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const uint32_t y = (uint32_t)__shfl_up((int)upto, s, 64);
      if (lane >= s) upto += y;
    }
    uint32_t base = 0;
    if (lane == 63 && upto) base = atomicAdd(&a.found[x.row], upto);
    uint32_t to = (uint32_t)__builtin_amdgcn_readlane((int)base, 63) + upto - mine;
#pragma unroll
    for (int j = 0; j < Q; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if ((hits >> (4 * j + i)) & 1u) {
          if (to < (uint32_t)kEntries)
            a.ids[(int64_t)x.row * kEntries + to] =
                (uint64_t)okey(v[j][i]) << 32 | (uint32_t) ~(uint32_t)(part * kIds + 4 * (j * kThreads + tid) + i);
          ++to;
        }
  }
}

template <int kType, bool kSoft>
hipError_t launch(const FilterArgs &a, hipStream_t stream) {
  const int blocks = a.rows * a.parts;
  auto three = [&](auto parts_kernel, int threads, auto merge_kernel, auto gather_kernel) {
    parts_kernel<<<blocks, threads, 0, stream>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    merge_kernel<<<a.rows, kThreads, 0, stream>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    gather_kernel<<<blocks < 1024 ? blocks : 1024, kThreads, 0, stream>>>(a);
    return hipGetLastError();
  };
  hipError_t e;
  switch (a.span) {
    case 2048: e = three(filter_parts_kernel<kType, kSoft, 256, 2>, 256, filter_merge_kernel<kType, kSoft, 2>,
                               filter_gather_kernel<kType, kSoft, 2>); break;
    case 4096: e = three(filter_parts_kernel<kType, kSoft, 256, 4>, 256, filter_merge_kernel<kType, kSoft, 4>,
                               filter_gather_kernel<kType, kSoft, 4>); break;
    default: e = three(filter_parts_kernel<kType, kSoft, 512, 4>, 512, filter_merge_kernel<kType, kSoft, 8>,
                               filter_gather_kernel<kType, kSoft, 8>); break;
  }
  if (e != hipSuccess) return e;
  filter_rest_kernel<kType, kSoft><<<a.rows, kRowThreads, 0, stream>>>(a);
  return hipGetLastError();
}
template <int kType>
hipError_t launch(const FilterArgs &a, bool soft, hipStream_t stream) {
  return soft ? launch<kType, true>(a, stream) : launch<kType, false>(a, stream);
}

}  // namespace

int filter_span(int rows, int vocab, int min_blocks) {
  int span = 8192;
  while (span > 2048 && (int64_t)rows * ((vocab + span - 1) / span) < min_blocks) span /= 2;
  return span;
}

// The most parts that a row of at most `vocab` ids may have in a batch of `rows`:
// a length of part has the most at the largest vocabulary that is cut so.  2,048
// and 4,096 ids are for rows of fewer than min_blocks / rows parts of twice that.
int filter_most_parts(int rows, int vocab, int min_blocks) {
  int64_t most = ((int64_t)vocab + 8191) / 8192;
  for (int64_t span = 4096; span >= 2048; span /= 2) {
    const int64_t v = std::min((int64_t)vocab, 2 * span * ((min_blocks - 1) / rows));
    most = std::max(most, (v + span - 1) / span);
  }
  return (int)most;
}

// The parts, their lists, the masses and counts of their ranges.
size_t filter_scratch_bytes(int rows, int parts) {
  const size_t n = (size_t)rows * parts;
  return n * (sizeof(FilterPart) + kFilterList * 8 + kFilterRanges * 12) + (size_t)rows * (kEntries * 8 + sizeof(FilterLeft) + 4) + 8;
}
void filter_scratch(void *base, FilterArgs *a) {
  const size_t n = (size_t)a->rows * a->parts;
  static_assert(sizeof(FilterPart) % 8 == 0, "whole words");
  char *at = static_cast<char *>(base);
  a->part = reinterpret_cast<FilterPart *>(at);
  a->list = reinterpret_cast<uint64_t *>(at += n * sizeof(FilterPart));
  a->range_mass = reinterpret_cast<uint64_t *>(at += n * kFilterList * 8);
  a->range_count = reinterpret_cast<uint32_t *>(at += n * kFilterRanges * 8);
  a->ids = reinterpret_cast<uint64_t *>(at += n * kFilterRanges * 4);
  a->left = reinterpret_cast<FilterLeft *>(at += (size_t)a->rows * kEntries * 8);
  a->found = reinterpret_cast<uint32_t *>(at += (size_t)a->rows * sizeof(FilterLeft));
  a->nleft = reinterpret_cast<uint32_t *>(at + (size_t)a->rows * 4);
}

// Ids a part lists: as many as keep a row's within what the merge takes, at
// most kFilterList (at 25 parts of 2,048 ids 32 a part left top-k 200 short).
int filter_log_list(int parts) {
  int log = 7;
  while (log > 5 && (parts << log) > kMergeMost) --log;
  return log;
}

hipError_t launch_filter(const FilterArgs &a, hipStream_t stream) {
  const bool soft = a.row_params || a.params.softcap > 0.0f;
  switch (a.type) {
    case SAS_TYPE_F32: return launch<SAS_TYPE_F32>(a, soft, stream);
    case SAS_TYPE_BF16: return launch<SAS_TYPE_BF16>(a, soft, stream);
    default: return launch<SAS_TYPE_F16>(a, soft, stream);
  }
}

}  // namespace sas
