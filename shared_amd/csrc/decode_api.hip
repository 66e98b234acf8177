// decode_api.hip - the C ABI of the multi-adapter decode head: sas_project
// and sas_sample_filtered.  Validation, scratch and launches only.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <limits>
#include <string>

#include "sas_handle.h"
#include "sas_launch.h"
#include "shared_amd_sampler.h"

using namespace sas;

namespace {

const char *check_projection(const sas_projection *p) {
  if (!p) return "descriptor is NULL";
  if (p->rows < 0 || p->rows > SAS_MAX_PROJECT_ROWS) return "rows must be in [0, SAS_MAX_PROJECT_ROWS]";
  if (p->dim < 8 || p->dim % 8 != 0) return "dim must be a positive multiple of 8";
  if (p->out_dim < 1) return "out_dim must be >= 1";
  if (p->x_type != SAS_TYPE_F32 && p->x_type != SAS_TYPE_BF16) return "x_type must be SAS_TYPE_F32 or SAS_TYPE_BF16";
  if (p->out_type != SAS_TYPE_F32 && p->out_type != SAS_TYPE_BF16)
    return "out_type must be SAS_TYPE_F32 or SAS_TYPE_BF16";
  if (p->adapters < 0) return "adapters must be >= 0";
  if (!p->weight && !p->accumulate) return "weight may be NULL only with accumulate";
  if (p->softcap < 0.0f || !std::isfinite(p->softcap)) return "softcap must be finite and >= 0";
  // (its reciprocal has to be finite)
  if (p->softcap > 0.0f && p->softcap < std::numeric_limits<float>::min()) return "softcap must be 0 or a normal number";
  if (p->adapters > 0 && (p->rank < 8 || p->rank > SAS_MAX_RANK || p->rank % 8 != 0))
    return "rank must be a multiple of 8 in [8, SAS_MAX_RANK]";
  // (a block an output tile of 16 x 16 at most)
  if ((((int64_t)p->rows + 15) / 16) * (((int64_t)p->out_dim + 15) / 16) > INT32_MAX) return "rows * out_dim is too large";
  if (p->rows == 0) return nullptr;
  if (!p->x || !p->out) return "x and out are required";
  if (p->x_stride < p->dim || p->x_stride % (p->x_type == SAS_TYPE_F32 ? 4 : 8) != 0)
    return "x_stride must be >= dim and a multiple of 8 (f32: of 4)";
  if (!aligned(p->x, 16)) return "x must be 16-byte aligned";
  if (p->out_stride < p->out_dim) return "out_stride < out_dim";
  if (!aligned(p->out, p->out_type == SAS_TYPE_F32 ? 4 : 2)) return "out must be aligned to its elements";
  if (p->weight) {
    // (a wave's rows are addressed by 32-bit offsets from its first)
    if (p->weight_stride < p->dim || p->weight_stride % 8 != 0 || p->weight_stride > SAS_MAX_PROJECT_STRIDE)
      return "weight_stride must be >= dim, a multiple of 8 and <= SAS_MAX_PROJECT_STRIDE";
    if (!aligned(p->weight, 16)) return "weight must be 16-byte aligned";
  }
  if (p->adapters > 0) {
    if (!p->a || !p->b || !p->row_adapter) return "a, b and row_adapter are required with adapters";
    if (p->a_stride < p->dim || p->a_stride % 8 != 0 || p->a_adapter_stride < 0 || p->a_adapter_stride % 8 != 0)
      return "a_stride must be >= dim, and it and a_adapter_stride multiples of 8";
    if (p->b_stride < p->rank || p->b_stride % 8 != 0 || p->b_adapter_stride < 0 || p->b_adapter_stride % 8 != 0)
      return "b_stride must be >= rank, and it and b_adapter_stride multiples of 8";
    if (!aligned(p->a, 16) || !aligned(p->b, 16)) return "a and b must be 16-byte aligned";
  }
  return nullptr;
}

const char *check_filter_rows(const sas_filter_rows *r) {
  if (!r) return "rows descriptor is NULL";
  if (r->rows < 0) return "rows must be >= 0";
  if (r->vocab < 1 || r->vocab > SAS_MAX_VOCAB) return "vocab must be in [1, SAS_MAX_VOCAB]";
  if (r->logits_type < SAS_TYPE_F32 || r->logits_type > SAS_TYPE_F16) return "logits_type must be one of SAS_TYPE_*";
  // (a block 2,048 ids at least)
  if ((int64_t)r->rows * (((int64_t)r->vocab + 2047) / 2048) > INT32_MAX) return "rows * vocab is too large";
  if (r->rows == 0) return nullptr;
  if (!r->logits || !r->out_ids) return "logits and out_ids are required";
  if (r->logits_stride < r->vocab) return "logits_stride < vocab";
  if (!aligned(r->logits, r->logits_type == SAS_TYPE_F32 ? 4 : 2)) return "logits must be aligned to their elements";
  if (r->mask && r->mask_stride != 0 && r->mask_stride < ((int64_t)r->vocab + 31) / 32)
    return "mask_stride must be 0 or >= ceil(vocab / 32)";
  if (r->hist_ids && !r->hist_offsets) return "hist_ids requires hist_offsets";
  if (r->hist_ids && r->hist_count < 1) return "hist_count must be >= 1 with hist_ids";
  const bool all_greedy = !r->row_params && !(r->params.temperature > 0.0);
  if (!r->uniforms && !all_greedy) return "uniforms are required unless every row is greedy";
  return nullptr;
}

int log2_ceil(int n) {
  int b = 0;
  while ((int64_t(1) << b) < n) ++b;
  return b;
}

}  // namespace

extern "C" {

int sas_project(sas_sampler *s, const sas_projection *p, void *stream) {
  return guarded(s, [&]() -> int {
    const char *who = "sas_project";
    if (!s) return fail(nullptr, SAS_ERR_INVALID, "sas_project: handle is NULL");
    if (const char *m = check_projection(p)) return fail(s, SAS_ERR_INVALID, std::string("sas_project: ") + m);
    if (p->rows == 0) return SAS_OK;
    if (int rc = set_device(s)) return rc;
    // the pieces of f32 hidden states serve the product with the weight
    const bool pieces = p->x_type == SAS_TYPE_F32 && p->weight;
    const int rank = p->adapters > 0 ? p->rank : 0;
    const ProjScratch at = proj_scratch(p->rows, p->dim, rank, pieces);
    if (int rc = grow(s, &s->proj, &s->proj_cap, at.bytes, stream, who, "sas_reserve_project")) return rc;
    char *scratch = static_cast<char *>(s->proj);
    ProjArgs a{};
    a.x = p->x;
    a.x_stride = p->x_stride;
    a.weight = p->weight;
    a.weight_stride = p->weight_stride;
    a.a = p->a;
    a.a_stride = p->a_stride;
    a.a_adapter_stride = p->a_adapter_stride;
    a.b = p->b;
    a.b_stride = p->b_stride;
    a.b_adapter_stride = p->b_adapter_stride;
    a.scales = p->scales;
    a.ranks = p->ranks;
    a.row_adapter = p->row_adapter;
    a.out = p->out;
    a.out_stride = p->out_stride;
    // rows of one subtile, or of one adapter, need no order
    a.perm = p->rows > 16 && p->adapters > 1 ? reinterpret_cast<int32_t *>(scratch) : nullptr;
    a.hp = reinterpret_cast<uint16_t *>(scratch + at.hp);
    a.xp = pieces ? reinterpret_cast<uint16_t *>(scratch + at.xp) : nullptr;
    a.rows = p->rows;
    a.dim = p->dim;
    a.out_dim = p->out_dim;
    a.adapters = p->adapters;
    a.rank = rank;
    a.softcap = p->softcap;
    a.x_f32 = p->x_type == SAS_TYPE_F32;
    a.out_bf16 = p->out_type == SAS_TYPE_BF16;
    a.accumulate = p->accumulate != 0;
    a.cus = s->cus;
    hipError_t e = launch_project(a, pick_stream(s, stream));
    return e == hipSuccess ? SAS_OK : hip_fail(s, e, "sas_project launch");
  });
}

int sas_reserve_project(sas_sampler *s, int32_t rows, int32_t dim, int32_t rank) {
  return guarded(s, [&]() -> int {
    if (!s) return fail(nullptr, SAS_ERR_INVALID, "sas_reserve_project: handle is NULL");
    if (rows < 0 || rows > SAS_MAX_PROJECT_ROWS || dim < 8 || dim % 8 != 0 || rank < 0 || rank > SAS_MAX_RANK || rank % 8 != 0)
      return fail(s, SAS_ERR_INVALID,
                  "sas_reserve_project: rows must be in [0, SAS_MAX_PROJECT_ROWS], dim a positive multiple of 8, rank a "
                  "multiple of 8 in [0, SAS_MAX_RANK]");
    if (int rc = set_device(s)) return rc;
    return grow(s, &s->proj, &s->proj_cap, proj_scratch(rows, dim, rank, true).bytes, nullptr, "sas_reserve_project");
  });
}

int sas_sample_filtered(sas_sampler *s, const sas_filter_rows *r, void *stream) {
  return guarded(s, [&]() -> int {
    if (!s) return fail(nullptr, SAS_ERR_INVALID, "sas_sample_filtered: handle is NULL");
    if (const char *m = check_filter_rows(r)) return fail(s, SAS_ERR_INVALID, std::string("sas_sample_filtered: ") + m);
    if (r->rows == 0) return SAS_OK;
    if (int rc = set_device(s)) return rc;
    FilterArgs a{};
    a.logits = r->logits;
    a.logits_stride = r->logits_stride;
    a.mask = r->mask;
    a.mask_stride = r->mask_stride;
    a.hist_ids = r->hist_ids;
    a.hist_offsets = r->hist_ids ? r->hist_offsets : nullptr;
    a.hist_count = r->hist_ids ? r->hist_count : 0;
    a.uniforms = r->uniforms;
    a.row_params = r->row_params;
    a.params = r->params;
    a.out_ids = r->out_ids;
    a.out_probs = r->out_probs;
    a.out_counts = r->out_counts;
    a.out_flags = r->out_flags;
    a.type = r->logits_type;
    a.vocab = r->vocab;
    a.rows = r->rows;
    a.shift = 62 - log2_ceil(r->vocab);
    a.span = filter_span(r->rows, r->vocab, 2 * s->cus);
    a.parts = (r->vocab + a.span - 1) / a.span;
    a.log_list = filter_log_list(a.parts);
    if (int rc = grow(s, &s->filt, &s->filt_cap, filter_scratch_bytes(r->rows, a.parts), stream, "sas_sample_filtered",
                      "sas_reserve_filtered"))
      return rc;
    filter_scratch(s->filt, &a);
    hipError_t e = launch_filter(a, pick_stream(s, stream));
    return e == hipSuccess ? SAS_OK : hip_fail(s, e, "sas_sample_filtered launch");
  });
}

int sas_reserve_filtered(sas_sampler *s, int32_t rows, int32_t vocab) {
  return guarded(s, [&]() -> int {
    if (!s) return fail(nullptr, SAS_ERR_INVALID, "sas_reserve_filtered: handle is NULL");
    if (rows < 0 || vocab < 1 || vocab > SAS_MAX_VOCAB || (int64_t)rows * (((int64_t)vocab + 2047) / 2048) > INT32_MAX)
      return fail(s, SAS_ERR_INVALID, "sas_reserve_filtered: rows must be >= 0, vocab in [1, SAS_MAX_VOCAB], rows * vocab below 2^42");
    if (int rc = set_device(s)) return rc;
    // fewer rows, and smaller vocabularies, may be cut into more parts (from
    // 2 cus rows on no longer)
    size_t bytes = 0;
    auto most = [&](int n) {
      bytes = std::max(bytes, filter_scratch_bytes(n, filter_most_parts(n, vocab, 2 * s->cus)));
    };
    for (int n = 1; n <= std::min(rows, 2 * s->cus); ++n) most(n);
    if (rows > 0) most(rows);
    return grow(s, &s->filt, &s->filt_cap, bytes, nullptr, "sas_reserve_filtered");
  });
}

}  // extern "C"
