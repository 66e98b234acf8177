// sas_handle.h - the handle behind the C ABI: its scratch, its errors.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <string>
#include <vector>

#include "shared_amd_sampler.h"

struct sas_sampler {
  int device = 0;
  hipStream_t stream = nullptr;
  std::string err;
  void *recs = nullptr;        // candidate record slots of every (row, part)
  size_t recs_cap = 0;
  void *vscratch = nullptr;   // sas_verify partials
  size_t vscratch_cap = 0;
  void *pad = nullptr;        // rows of fewer than 4 logits, padded to 4
  size_t pad_cap = 0;
  void *logits = nullptr;     // the LM head's logits (its calls without out_logits)
  size_t logits_cap = 0;
  void *hb = nullptr;         // long histories bucketed by part
  size_t hb_cap = 0;
  void *proj = nullptr;       // sas_project: the rows' inner products and pieces
  size_t proj_cap = 0;
  void *filt = nullptr;       // sas_sample_filtered: what its parts kernel leaves
  size_t filt_cap = 0;
  int cus = 0;                 // compute units of the device
  // Buffers a growth replaced.  Work already queued (or recorded into a
  // HIP graph) may still use them, so they are freed by sas_destroy only.
  std::vector<void *> retired;
};

namespace sas {

inline thread_local std::string g_err;

inline int fail(sas_sampler *s, int code, const std::string &msg) {
  if (s) s->err = msg;
  else g_err = msg;
  return code;
}

inline int hip_fail(sas_sampler *s, hipError_t e, const char *what) {
  return fail(s, SAS_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

inline hipStream_t pick_stream(sas_sampler *, void *stream) { return reinterpret_cast<hipStream_t>(stream); }

// Whether work on `stream` is being recorded into a graph.
inline bool capturing(void *stream) {
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(reinterpret_cast<hipStream_t>(stream), &cs) == hipSuccess &&
         cs != hipStreamCaptureStatusNone;
}

// Grow a scratch buffer to at least `need` bytes.  The buffer it replaces
// is retired, not freed: launches queued on any stream, and graphs that
// recorded them, keep a valid address; sas_destroy frees it.  Capacities
// at least double, so retired buffers hold less than the live one.  Under
// stream capture nothing is allocated: the call fails and names the fix,
// `reserve` (the entry that sizes this buffer) or an eager call.
inline int grow(sas_sampler *s, void **buf, size_t *cap, size_t need, void *stream, const char *who,
                const char *reserve = "sas_reserve_for") {
  if (need <= *cap) return SAS_OK;
  if (capturing(stream))
    return fail(s, SAS_ERR_INVALID,
                std::string(who) + ": the handle's scratch is too small for this call and the stream is being "
                                   "captured: size it before the capture (" + reserve + ", or one eager call of "
                                   "this shape)");
  size_t bytes = (need + 255) & ~size_t(255);
  if (*cap && bytes < 2 * *cap) bytes = 2 * *cap;
  void *fresh = nullptr;
  hipError_t e = hipMalloc(&fresh, bytes);
  if (e != hipSuccess) return fail(s, SAS_ERR_NOMEM, std::string(who) + ": hipMalloc scratch: " + hipGetErrorString(e));
  if (*buf) s->retired.push_back(*buf);
  *buf = fresh;
  *cap = bytes;
  return SAS_OK;
}

inline int set_device(sas_sampler *s) {
  hipError_t e = hipSetDevice(s->device);
  return e == hipSuccess ? SAS_OK : hip_fail(s, e, "hipSetDevice");
}

}  // namespace sas
