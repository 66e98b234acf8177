// filter_kernel.hip - sampling over the whole vocabulary with temperature,
// top-k of any size, top-p and min-p (gfx950).
//
// A row's candidates in the order (value descending, id ascending) are cut to
// a prefix; the prefix ends inside the ids that share one value, the edge:
// every id of a larger value is kept, and of the edge's the first `take` in
// ascending order.  No ids are sorted: the edge is found by counts and masses
// of value ranges, and the draw walks the kept ids in ascending order.
//
// Masses exp((v - m) / T) are summed as 64-bit integers of 2^-shift: sums of
// any order, atomic ones too, are the same bits.  2^shift * vocab <= 2^62, so
// no sum overflows; rounding one mass is off by 2^-(shift + 1) of the largest
// at most (2^-45 for 262,144 ids).
#include "sas_device.h"
#include "sas_exp.h"
#include "sas_launch.h"

namespace sas {
namespace {

typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef u16x4 u16x4u __attribute__((aligned(2)));

constexpr int kRowThreads = 1024;
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kSpan = 8192;                       // ids a block holds at once
constexpr int kQuads = kSpan / (4 * kRowThreads); // quads of ids per thread
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
__device__ __forceinline__ f32x4 load_logits(const FilterArgs &a, int64_t row0, int id) {
  const float nan = qnan();
  f32x4 v = {nan, nan, nan, nan};
  const int left = a.vocab - id;
  if (left <= 0) return v;
  if (a.type == SAS_TYPE_F32) {
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
    const float f = a.type == SAS_TYPE_BF16 ? __uint_as_float((uint32_t)h[i] << 16)
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
__device__ __forceinline__ double mass_of(uint32_t key, const Scale &s, const ExpTab &tab) {
  const float v = fkey(key);
  return v == (float)s.m ? 1.0 : exp_sum(((double)v - s.m) * s.inv_t, tab);
}
__device__ __forceinline__ uint64_t units_of(double mass, const Scale &s) {
  return (uint64_t)__builtin_rint(__builtin_amdgcn_ldexp(mass, s.shift));
}

// Every id of a larger key than `key`, and the first `take` of its own.
struct Edge {
  uint32_t key;
  uint32_t take;
};

struct RowShared {
  ExpTab tab;
  uint32_t count[kSpan / 2];  // history counts of a span's ids, 16 bits each
  unsigned long long mass[kBins];
  uint32_t cnt[kBins];
  unsigned long long red[kRowWaves][2];
  unsigned long long sel[4];
  unsigned long long part[(SAS_MAX_VOCAB + kSpan - 1) / kSpan];
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
    if (h.n) {
      __syncthreads();
      for (int i = threadIdx.x; i < kSpan / 2; i += kRowThreads) l.count[i] = 0u;
      __syncthreads();
      for (int i = threadIdx.x; i < h.n; i += kRowThreads) {
        const uint32_t at = h.ids[i] - (uint32_t)(q * kSpan);
        if (at < (uint32_t)kSpan) atomicAdd(&l.count[at >> 1], 1u << (16 * (at & 1)));
      }
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < kQuads; ++j) {
      const int id = id0(q, j);
      const f32x4 v = load_logits(a, row0, id);
      const uint32_t bits = !mask ? 0xFu : id < a.vocab ? mask[id >> 5] >> (id & 31) : 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = v[i];
        if (p.softcap > 0.0f) x = softcap_f32(x, p.softcap);
        if (h.n) {
          const uint32_t at = (uint32_t)(id + i - q * kSpan);
          const uint32_t c = (l.count[at >> 1] >> (16 * (at & 1))) & 0xFFFFu;
          if (c) x = penalized(x, c, p);
        }
        const uint32_t k = okey(x);
        key[j][i] = ((bits >> i) & 1u) && k > kNegInf ? k : 0u;
      }
    }
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
  __device__ __forceinline__ int find(int n, bool by_count, uint64_t need, uint64_t *mass, uint64_t *count) const {
    __syncthreads();
    if (threadIdx.x < 64) {
      const int lane = threadIdx.x, per = n / 64;
      uint64_t m = 0, c = 0;
      for (int i = 0; i < per; ++i) {
        m += l.mass[lane * per + i];
        c += l.cnt[lane * per + i];
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
          const uint64_t m1 = mm + l.mass[lane * per + i], c1 = cc + l.cnt[lane * per + i];
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
  // from the histogram over bins in l.mass / l.cnt, which stays as it is only
  // if `keep`.  *mass, *count: of the prefix up to the edge, its `take` in.
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
          atomicAdd(&l.mass[d], (unsigned long long)units_of(mass_of(k, s, l.tab), s));
          atomicAdd(&l.cnt[d], 1u);
        }
      });
      uint64_t m1, c1;
      const int d = find(256, by_count, by_count ? need - c0 : need - m0, &m1, &c1);
      m0 += m1;
      c0 += c1;
      top |= (uint32_t)(255 - d) << sh;
    }
    const uint64_t unit = units_of(mass_of(top, s, l.tab), s);
    const uint32_t n = l.cnt[255 - (top & 0xFFu)];
    uint64_t take = by_count ? need - c0 : unit ? (need - m0 + unit - 1) / unit : 1;
    take = min(max(take, (uint64_t)1), (uint64_t)n);
    *mass = m0 + take * unit;
    *count = c0 + take;
    return Edge{top, (uint32_t)take};
  }

  // The histogram of the row's candidates over the bins.
  __device__ __forceinline__ void histogram() {
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kRowThreads) {
      l.mass[i] = 0ull;
      l.cnt[i] = 0u;
    }
    __syncthreads();
    uint64_t rest = 0, nrest = 0;
    each([&](uint32_t k) {
      if (!k) return;
      const int b = bin_of(k, s);
      const uint64_t u = units_of(mass_of(k, s, l.tab), s);
      if (b == kBins - 1) {
        rest += u;
        ++nrest;
      } else {
        atomicAdd(&l.mass[b], (unsigned long long)u);
        atomicAdd(&l.cnt[b], 1u);
      }
    });
    block_sum2(l, rest, nrest);
    if (threadIdx.x == 0) {
      l.mass[kBins - 1] = rest;
      l.cnt[kBins - 1] = (uint32_t)nrest;
    }
    __syncthreads();
  }
};

__global__ __launch_bounds__(kRowThreads) void filter_row_kernel(const FilterArgs a) {
  __shared__ RowShared l;
  const int row = blockIdx.x, tid = threadIdx.x;
  l.tab.fill(exp_tab_entry());
  __syncthreads();
  const sas_filter_params p = load_filter_params(a, row);
  Row r{a, l, p, (int64_t)row * a.logits_stride, a.mask ? a.mask + (int64_t)row * a.mask_stride : nullptr,
        history_of(a, row), Scale{}};
  // the best candidate, and how many there are
  uint64_t best = 0, n = 0;
  for (int q = 0; q < r.spans(); ++q) {
    uint32_t key[kQuads][4];
    r.keys(q, key);
#pragma unroll
    for (int j = 0; j < kQuads; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t k = key[j][i] ? ((uint64_t)key[j][i] << 32) | (uint32_t)~(r.id0(q, j) + i) : 0ull;
        best = max(best, k);
        n += k ? 1 : 0;
      }
  }
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) best = max(best, shfl_xor64(best, s));
  __syncthreads();
  if ((tid & 63) == 0) l.red[tid >> 6][0] = best;
  __syncthreads();
  for (int w = 0; w < kRowWaves; ++w) best = max(best, (uint64_t)l.red[w][0]);
  uint64_t zero = 0;
  block_sum2(l, n, zero);
  auto done = [&](uint32_t id, double prob, uint64_t count) {
    a.out_ids[row] = id;
    if (a.out_probs) a.out_probs[row] = prob;
    if (a.out_counts) a.out_counts[row] = (int32_t)count;
    if (a.out_flags) a.out_flags[row] = best ? 0u : SAS_FLAG_EMPTY_ROW;
  };
  const bool greedy = !(p.temperature > 0.0) || p.top_k == 1;
  if (best == 0 || greedy) {
    if (tid == 0) done(best ? ~(uint32_t)best : SAS_NO_TOKEN, best ? 1.0 : 0.0, best ? 1 : 0);
    return;
  }
  const uint32_t top = (uint32_t)(best >> 32);
  r.s = Scale{(double)fkey(top), 1.0 / p.temperature, 8.0 / p.temperature, a.shift};

  Edge e{0u, 0u};  // no edge: every candidate
  uint64_t mass = 0, count = 0;
  if (p.top_k > 0 && (uint64_t)p.top_k < n) {
    r.histogram();
    e = r.edge(true, (uint64_t)p.top_k, &mass, &count);
  }
  if (p.top_p < 1.0) {
    r.histogram();
    if (!e.key) {
      uint64_t all = 0;
      zero = 0;
      for (int i = tid; i < kBins; i += kRowThreads) all += l.mass[i];
      block_sum2(l, all, zero);
      mass = all;
    }
    const double need = ceil(fmax(p.top_p, 0.0) * (double)mass);
    const Edge f = r.edge(false, min(max((uint64_t)need, (uint64_t)1), mass), &mass, &count);
    if (!e.key || f.key > e.key || (f.key == e.key && f.take < e.take)) e = f;
  }
  if (p.min_p > 0.0) {
    // the smallest key whose mass reaches min_p (the mass falls with the key)
    const double least = fmin(p.min_p, 1.0);
    uint32_t lo = kNegInf, hi = top;  // hi reaches it, lo does not (or is no candidate's)
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (mass_of(mid, r.s, l.tab) >= least) hi = mid;
      else lo = mid;
    }
    if (hi > e.key) e = Edge{hi, ~0u};
  }
  // what is kept of each span; the edge's ids count in ascending order
  uint64_t total = 0, kept = 0, ties = 0;
  const uint64_t unit = e.key ? units_of(mass_of(e.key, r.s, l.tab), r.s) : 0;
  for (int q = 0; q < r.spans(); ++q) {
    uint32_t key[kQuads][4];
    r.keys(q, key);
    uint64_t m = 0, c = 0;
#pragma unroll
    for (int j = 0; j < kQuads; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t k = key[j][i];
        if (k > e.key) {
          m += units_of(mass_of(k, r.s, l.tab), r.s);
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
  while (q < r.spans() - 1 && before + l.part[q] <= goal) before += l.part[q++];
  // the edge's ids in the spans before
  uint64_t tie0 = 0;
  if (e.key && e.take != ~0u) {
    for (int s = 0; s < q; ++s) {
      uint32_t key[kQuads][4];
      r.keys(s, key);
#pragma unroll
      for (int j = 0; j < kQuads; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) tie0 += key[j][i] == e.key ? 1 : 0;
    }
    zero = 0;
    block_sum2(l, tie0, zero);
  }
  uint32_t key[kQuads][4];
  r.keys(q, key);
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
      mine[i] = in ? units_of(mass_of(k, r.s, l.tab), r.s) : 0;
      m += mine[i];
    }
    uint64_t run = before + block_scan(l, m, &all) - m;
    if (run <= goal && goal < run + m) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (run <= goal && goal < run + mine[i])
          done((uint32_t)(r.id0(q, j) + i), mass_of(key[j][i], r.s, l.tab) / __builtin_amdgcn_ldexp((double)total, -a.shift), kept);
        run += mine[i];
      }
    }
    before += all;
  }
}

}  // namespace

hipError_t launch_filter(const FilterArgs &a, hipStream_t stream) {
  filter_row_kernel<<<a.rows, kRowThreads, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace sas
