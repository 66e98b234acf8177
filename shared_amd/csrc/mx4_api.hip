// mx4_api.hip - the C ABI of the MXFP4 tables: sas_quantize_mx4, sas_lookup_mx4
// and sas_project_mx4.  Validation and launches only.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <limits>
#include <string>

#include "sas_handle.h"
#include "sas_launch.h"
#include "shared_amd_sampler.h"

using namespace sas;

namespace {

bool bad_type(int32_t t) { return t != SAS_TYPE_F32 && t != SAS_TYPE_BF16 && t != SAS_TYPE_F16; }

bool aligned_to(const void *p, int32_t type) { return aligned(p, type == SAS_TYPE_F32 ? 4 : 2); }

// (the kernels address a row's blocks by 32-bit offsets)
bool too_many_units(int32_t rows, int32_t dim) { return (int64_t)rows * ((mx4_blocks(dim) + 3) / 4) > INT32_MAX; }

const char *check_quantization(const sas_mx4_quantization *q) {
  if (!q) return "descriptor is NULL";
  if (q->rows < 0) return "rows must be >= 0";
  if (q->dim < 1) return "dim must be >= 1";
  if (bad_type(q->x_type)) return "x_type must be SAS_TYPE_F32, SAS_TYPE_BF16 or SAS_TYPE_F16";
  if (too_many_units(q->rows, q->dim)) return "rows * dim is too large";
  if (q->rows == 0) return nullptr;
  if (!q->x) return "x is required";
  if (q->x_stride < q->dim) return "x_stride < dim";
  if (!aligned_to(q->x, q->x_type)) return "x must be aligned to its elements";
  return check_mx4(q->out.codes, q->out.codes_stride, q->out.scales, q->out.scales_stride, q->dim);
}

const char *check_lookup(const sas_mx4_lookup *l) {
  if (!l) return "descriptor is NULL";
  if (l->rows < 0 || l->table_rows < 0) return "rows and table_rows must be >= 0";
  if (l->dim < 1) return "dim must be >= 1";
  if (bad_type(l->out_type)) return "out_type must be SAS_TYPE_F32, SAS_TYPE_BF16 or SAS_TYPE_F16";
  if (too_many_units(l->rows, l->dim)) return "rows * dim is too large";
  if (!l->ids && l->rows > l->table_rows) return "rows must be <= table_rows without ids";
  if (l->rows == 0) return nullptr;
  if (!l->out) return "out is required";
  if (l->out_stride < l->dim) return "out_stride < dim";
  if (!aligned_to(l->out, l->out_type)) return "out must be aligned to its elements";
  // (a table of no rows is never read: it may lie nowhere)
  if (l->table_rows == 0) return nullptr;
  return check_mx4(l->table.codes, l->table.codes_stride, l->table.scales, l->table.scales_stride, l->dim);
}

const char *check_mx4_projection(const sas_mx4_projection *p) {
  if (!p) return "descriptor is NULL";
  if (p->rows < 0 || p->rows > SAS_MAX_PROJECT_ROWS) return "rows must be in [0, SAS_MAX_PROJECT_ROWS]";
  if (p->x_type != SAS_TYPE_F32 && p->x_type != SAS_TYPE_BF16 && p->x_type != SAS_TYPE_MX4)
    return "x_type must be SAS_TYPE_F32, SAS_TYPE_BF16 or SAS_TYPE_MX4";
  if (p->dim < 1 || (p->x_type != SAS_TYPE_MX4 && p->dim % 8 != 0)) return "dim must be positive, and a multiple of 8 but with MX4 hidden states";
  if (p->out_dim < 1) return "out_dim must be >= 1";
  if (p->out_type != SAS_TYPE_F32 && p->out_type != SAS_TYPE_BF16)
    return "out_type must be SAS_TYPE_F32 or SAS_TYPE_BF16";
  if (p->softcap < 0.0f || !std::isfinite(p->softcap)) return "softcap must be finite and >= 0";
  // (its reciprocal has to be finite)
  if (p->softcap > 0.0f && p->softcap < std::numeric_limits<float>::min()) return "softcap must be 0 or a normal number";
  // (2^39 outputs are more than memory holds)
  if ((((int64_t)p->rows + 15) / 16) * (((int64_t)p->out_dim + 15) / 16) > INT32_MAX) return "rows * out_dim is too large";
  if (p->rows == 0) return nullptr;
  if (!p->out) return "out is required";
  if (p->out_stride < p->out_dim) return "out_stride < out_dim";
  if (!aligned_to(p->out, p->out_type)) return "out must be aligned to its elements";
  if (p->x_type == SAS_TYPE_MX4) {
    if (const char *m = check_mx4(p->x4.codes, p->x4.codes_stride, p->x4.scales, p->x4.scales_stride, p->dim)) return m;
  } else {
    if (!p->x) return "x is required";
    if (p->x_stride < p->dim || p->x_stride % (p->x_type == SAS_TYPE_F32 ? 4 : 8) != 0)
      return "x_stride must be >= dim and a multiple of 8 (f32: of 4)";
    if (!aligned(p->x, 16)) return "x must be 16-byte aligned";
  }
  return check_mx4(p->weight.codes, p->weight.codes_stride, p->weight.scales, p->weight.scales_stride, p->dim);
}

}  // namespace

extern "C" {

int sas_quantize_mx4(sas_sampler *s, const sas_mx4_quantization *q, void *stream) {
  return guarded(s, [&]() -> int {
    if (!s) return fail(nullptr, SAS_ERR_INVALID, "sas_quantize_mx4: handle is NULL");
    if (const char *m = check_quantization(q)) return fail(s, SAS_ERR_INVALID, std::string("sas_quantize_mx4: ") + m);
    if (q->rows == 0) return SAS_OK;
    if (int rc = set_device(s)) return rc;
    Mx4QuantizeArgs a{};
    a.x = q->x;
    a.x_stride = q->x_stride;
    a.codes = static_cast<uint8_t *>(q->out.codes);
    a.codes_stride = q->out.codes_stride;
    a.scales = static_cast<uint8_t *>(q->out.scales);
    a.scales_stride = q->out.scales_stride;
    a.x_type = q->x_type;
    a.rows = q->rows;
    a.dim = q->dim;
    hipError_t e = launch_mx4_quantize(a, pick_stream(s, stream));
    return e == hipSuccess ? SAS_OK : hip_fail(s, e, "sas_quantize_mx4 launch");
  });
}

int sas_lookup_mx4(sas_sampler *s, const sas_mx4_lookup *l, void *stream) {
  return guarded(s, [&]() -> int {
    if (!s) return fail(nullptr, SAS_ERR_INVALID, "sas_lookup_mx4: handle is NULL");
    if (const char *m = check_lookup(l)) return fail(s, SAS_ERR_INVALID, std::string("sas_lookup_mx4: ") + m);
    if (l->rows == 0) return SAS_OK;
    if (int rc = set_device(s)) return rc;
    Mx4LookupArgs a{};
    a.codes = static_cast<const uint8_t *>(l->table.codes);
    a.codes_stride = l->table.codes_stride;
    a.scales = static_cast<const uint8_t *>(l->table.scales);
    a.scales_stride = l->table.scales_stride;
    a.ids = l->ids;
    a.out = l->out;
    a.out_stride = l->out_stride;
    a.out_type = l->out_type;
    a.table_rows = l->table_rows;
    a.rows = l->rows;
    a.dim = l->dim;
    hipError_t e = launch_mx4_lookup(a, pick_stream(s, stream));
    return e == hipSuccess ? SAS_OK : hip_fail(s, e, "sas_lookup_mx4 launch");
  });
}

int sas_project_mx4(sas_sampler *s, const sas_mx4_projection *p, void *stream) {
  return guarded(s, [&]() -> int {
    if (!s) return fail(nullptr, SAS_ERR_INVALID, "sas_project_mx4: handle is NULL");
    if (const char *m = check_mx4_projection(p)) return fail(s, SAS_ERR_INVALID, std::string("sas_project_mx4: ") + m);
    if (p->rows == 0) return SAS_OK;
    if (int rc = set_device(s)) return rc;
    const bool four = p->x_type == SAS_TYPE_MX4;
    Mx4ProjArgs a{};
    a.x = four ? p->x4.codes : p->x;
    a.x_stride = four ? p->x4.codes_stride : p->x_stride;
    a.x_scales = four ? static_cast<const uint8_t *>(p->x4.scales) : nullptr;
    a.x_scales_stride = four ? p->x4.scales_stride : 0;
    a.w = static_cast<const uint8_t *>(p->weight.codes);
    a.w_stride = p->weight.codes_stride;
    a.w_scales = static_cast<const uint8_t *>(p->weight.scales);
    a.w_scales_stride = p->weight.scales_stride;
    a.out = p->out;
    a.out_stride = p->out_stride;
    a.x_type = p->x_type;
    a.rows = p->rows;
    a.dim = p->dim;
    a.out_dim = p->out_dim;
    a.softcap = p->softcap;
    a.out_bf16 = p->out_type == SAS_TYPE_BF16;
    a.accumulate = p->accumulate != 0;
    a.cus = s->cus;
    hipError_t e = launch_mx4_project(a, pick_stream(s, stream));
    return e == hipSuccess ? SAS_OK : hip_fail(s, e, "sas_project_mx4 launch");
  });
}

}  // extern "C"
