// extern "C" boundary of the operators beside the hot path that preference and
// policy training adds: host-side validation and launches, as in capi.cpp.
#include <hip/hip_runtime.h>

#include "../../include/siq_kernels.h"
#include "capi_internal.h"
#include "pack8.h"

using namespace siq_capi;

namespace {

// Elements per call: two vectors of eight a thread, and fewer than 2^32 threads.
constexpr int64_t kMaxNumel = int64_t(1) << 35;

int check_format(int dtype, int format) {
  if (dtype != SIQ_DTYPE_BF16 && dtype != SIQ_DTYPE_FP32)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "dtype must be SIQ_DTYPE_BF16 or SIQ_DTYPE_FP32");
  if (format != SIQ_FORMAT_INT8 && format != SIQ_FORMAT_E4M3)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "format must be SIQ_FORMAT_INT8 or SIQ_FORMAT_E4M3");
  return SIQ_OK;
}

int check_ptr(const void* p, const char* name) {
  if (p == nullptr) return fail(SIQ_ERR_INVALID_ARGUMENT, "%s must not be NULL", name);
  if (!aligned16(p)) return fail(SIQ_ERR_ALIGNMENT, "%s is not 16-byte aligned", name);
  return SIQ_OK;
}

int check_numel(int64_t numel) {
  if (numel < 0 || numel > kMaxNumel)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "the number of elements must be in [0, 2^35] (got %lld)", (long long)numel);
  return SIQ_OK;
}

// rows x cols elements at row stride ld (elements) of tensors whose rows are
// either contiguous or start at 16-byte boundaries.
int check_rows(int64_t rows, int64_t cols, int64_t ld0, int64_t ld1, int dtype, const char* names) {
  if (rows < 0 || cols < 0) return fail(SIQ_ERR_INVALID_ARGUMENT, "rows and cols must be >= 0");
  if (cols > 0 && rows > kMaxNumel / cols)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "rows * cols must be at most 2^35 (%lld x %lld)", (long long)rows,
                (long long)cols);
  const int64_t ld[2] = {ld0, ld1}, step = dtype == SIQ_DTYPE_FP32 ? 4 : 8;
  if (ld0 == cols && ld1 == cols) return SIQ_OK;
  for (int i = 0; i < 2; ++i)
    if (ld[i] < cols || ld[i] > kMaxNumel || ld[i] % step != 0)
      return fail(SIQ_ERR_ALIGNMENT, "row strides of %s must be at least cols and multiples of 16 bytes (got %lld)", names,
                  (long long)ld[i]);
  if (cols % 8 != 0)
    return fail(SIQ_ERR_UNSUPPORTED, "cols (%lld) must be a multiple of 8 where rows are not contiguous", (long long)cols);
  return SIQ_OK;
}

int launched(hipError_t e, const char* what) {
  return e == hipSuccess ? ok() : fail(SIQ_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
}

}  // namespace

extern "C" {

int siq_pack8(const void* x, int64_t numel, int dtype, int format, void* codes, void* scales, void* stream) {
  int rc;
  if ((rc = check_format(dtype, format)) || (rc = check_numel(numel))) return rc;
  if (numel == 0) return ok();
  if ((rc = check_ptr(x, "x")) || (rc = check_ptr(codes, "codes")) || (rc = check_ptr(scales, "scales"))) return rc;
  return launched(siq::launch_pack8(x, numel, dtype == SIQ_DTYPE_FP32, format == SIQ_FORMAT_E4M3,
                                    static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales),
                                    static_cast<hipStream_t>(stream)),
                  "pack8");
}

int siq_unpack8(const void* codes, const void* scales, int64_t numel, int dtype, int format, void* x, void* stream) {
  int rc;
  if ((rc = check_format(dtype, format)) || (rc = check_numel(numel))) return rc;
  if (numel == 0) return ok();
  if ((rc = check_ptr(x, "x")) || (rc = check_ptr(codes, "codes")) || (rc = check_ptr(scales, "scales"))) return rc;
  return launched(siq::launch_unpack8(static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), numel,
                                      dtype == SIQ_DTYPE_FP32, format == SIQ_FORMAT_E4M3, x,
                                      static_cast<hipStream_t>(stream)),
                  "unpack8");
}

int siq_swiglu8_fwd(const void* gate, const void* up, int64_t rows, int64_t cols, int64_t gate_stride,
                    int64_t up_stride, int dtype, int format, void* h, void* gate_codes, void* gate_scales,
                    void* up_codes, void* up_scales, void* stream) {
  int rc;
  if ((rc = check_format(dtype, format)) || (rc = check_rows(rows, cols, gate_stride, up_stride, dtype, "gate / up")))
    return rc;
  if (rows * cols == 0) return ok();
  if ((rc = check_ptr(gate, "gate")) || (rc = check_ptr(up, "up")) || (rc = check_ptr(h, "h"))) return rc;
  if (gate_codes != nullptr || gate_scales != nullptr || up_codes != nullptr || up_scales != nullptr)
    if ((rc = check_ptr(gate_codes, "gate_codes")) || (rc = check_ptr(gate_scales, "gate_scales")) ||
        (rc = check_ptr(up_codes, "up_codes")) || (rc = check_ptr(up_scales, "up_scales")))
      return rc;
  siq::SwigluArgs a{};
  a.gate = gate;
  a.up = up;
  a.h = h;
  a.gcodes = static_cast<uint8_t*>(gate_codes);
  a.gscales = static_cast<uint8_t*>(gate_scales);
  a.ucodes = static_cast<uint8_t*>(up_codes);
  a.uscales = static_cast<uint8_t*>(up_scales);
  a.rows = rows;
  a.cols = cols;
  a.ld0 = gate_stride;
  a.ld1 = up_stride;
  a.f32 = dtype == SIQ_DTYPE_FP32;
  a.e4m3 = format == SIQ_FORMAT_E4M3;
  return launched(siq::launch_swiglu8_fwd(a, static_cast<hipStream_t>(stream)), "swiglu8 forward");
}

int siq_swiglu8_bwd(const void* dh, const void* gate_codes, const void* gate_scales, const void* up_codes,
                    const void* up_scales, int64_t rows, int64_t cols, int64_t dgate_stride, int64_t dup_stride,
                    int dtype, int format, void* dgate, void* dup, void* h, void* stream) {
  int rc;
  if ((rc = check_format(dtype, format)) ||
      (rc = check_rows(rows, cols, dgate_stride, dup_stride, dtype, "dgate / dup")))
    return rc;
  if (rows * cols == 0) return ok();
  if ((rc = check_ptr(dh, "dh")) || (rc = check_ptr(dgate, "dgate")) || (rc = check_ptr(dup, "dup")) ||
      (rc = check_ptr(gate_codes, "gate_codes")) || (rc = check_ptr(gate_scales, "gate_scales")) ||
      (rc = check_ptr(up_codes, "up_codes")) || (rc = check_ptr(up_scales, "up_scales")))
    return rc;
  if (h != nullptr && (rc = check_ptr(h, "h"))) return rc;
  siq::SwigluArgs a{};
  a.dh = dh;
  a.h = h;
  a.dgate = dgate;
  a.dup = dup;
  a.gcodes = static_cast<uint8_t*>(const_cast<void*>(gate_codes));
  a.gscales = static_cast<uint8_t*>(const_cast<void*>(gate_scales));
  a.ucodes = static_cast<uint8_t*>(const_cast<void*>(up_codes));
  a.uscales = static_cast<uint8_t*>(const_cast<void*>(up_scales));
  a.rows = rows;
  a.cols = cols;
  a.ld0 = dgate_stride;
  a.ld1 = dup_stride;
  a.f32 = dtype == SIQ_DTYPE_FP32;
  a.e4m3 = format == SIQ_FORMAT_E4M3;
  return launched(siq::launch_swiglu8_bwd(a, static_cast<hipStream_t>(stream)), "swiglu8 backward");
}

}  // extern "C"
