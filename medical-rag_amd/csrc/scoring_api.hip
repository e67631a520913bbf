// C ABI of the scoring head's operators (declared in include/medtutor_retrieval.h):
// argument checks and launches.  The kernels are in mx_rows.hip, mx_matmul.hip and
// token_logprobs.hip.
#include <hip/hip_runtime.h>

#include "../../include/medtutor_retrieval.h"
#include "mx_format.h"

namespace mtr {
int set_error(int code, const char* fmt, ...);  // mtr_api.hip: thread-local message behind mtr_last_error()
}

namespace {

using mtr::set_error;

struct DeviceGuard {
    int prev = -1;
    bool ok = false;
    explicit DeviceGuard(int dev) {
        if (hipGetDevice(&prev) != hipSuccess) prev = -1;
        ok = prev == dev || hipSetDevice(dev) == hipSuccess;
        if (prev == dev) prev = -1;     // nothing to put back
    }
    ~DeviceGuard() {
        if (prev >= 0) (void)hipSetDevice(prev);
    }
};

int launched(const char* what, hipError_t e) {
    if (e == hipSuccess) return MTR_OK;
    return set_error(e == hipErrorOutOfMemory ? MTR_ERR_OOM : MTR_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

bool is_float(int32_t dtype) { return dtype == MTR_F32 || dtype == MTR_BF16 || dtype == MTR_F16; }
bool is_mx(int32_t format) { return format == MTR_MX_FP4 || format == MTR_MX_FP8; }
bool off(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }
uintptr_t size_of(int32_t dtype) { return dtype == MTR_F32 ? 4 : 2; }

constexpr int64_t kMost = 0x7fffffff;       // rows, row groups and workgroups are numbered in 31 bits
constexpr int64_t kMostProduct = MTR_MX_MATMUL_MAX_ROWS;    // a launch counts its threads in 32 bits, four a row

int check_rows(const char* what, int64_t n, int32_t d, const void* values, const void* scales, int32_t format) {
    if (!is_mx(format)) return set_error(MTR_ERR_INVALID, "%s: bad format %d", what, format);
    if (n < 0 || n > kMost || d < 1 || d > kMost - MTR_MX_PAD || n * (mtr::mx_padded(d) / MTR_MX_PAD) > kMost)
        return set_error(MTR_ERR_INVALID, "%s: bad shape (n=%lld, d=%d)", what, (long long)n, d);
    if (n == 0) return MTR_OK;
    if (!values || !scales) return set_error(MTR_ERR_INVALID, "%s: NULL argument", what);
    if (off(values, 16) || off(scales, 4))
        return set_error(MTR_ERR_INVALID, "%s: element bytes must start on 16 bytes, scale bytes on 4", what);
    return MTR_OK;
}

}  // namespace

extern "C" {

int mtr_mx_quantize(const void* dev_x, int32_t dtype, int64_t n, int32_t d, int64_t ld, int32_t format, void* dev_values,
                    void* dev_scales, int32_t device_id, void* stream) {
    if (!is_float(dtype)) return set_error(MTR_ERR_INVALID, "bad dtype %d", dtype);
    if (int rc = check_rows("mtr_mx_quantize", n, d, dev_values, dev_scales, format)) return rc;
    if (n == 0) return MTR_OK;
    if (!dev_x) return set_error(MTR_ERR_INVALID, "NULL argument");
    if (off(dev_x, size_of(dtype)) || ld < 0) return set_error(MTR_ERR_INVALID, "bad row stride %lld or address", (long long)ld);
    DeviceGuard guard(device_id);
    if (!guard.ok) return set_error(MTR_ERR_HIP, "hipSetDevice(%d) failed", device_id);
    return launched("mtr_mx_quantize", mtr::launch_mx_quantize(dev_x, dtype, n, d, ld, format, dev_values, dev_scales,
                                                               static_cast<hipStream_t>(stream)));
}

int mtr_mx_dequantize(const void* dev_values, const void* dev_scales, int32_t format, int64_t n, int32_t d, void* dev_out,
                      int32_t dtype, int64_t ld, int32_t device_id, void* stream) {
    if (!is_float(dtype)) return set_error(MTR_ERR_INVALID, "bad dtype %d", dtype);
    if (int rc = check_rows("mtr_mx_dequantize", n, d, dev_values, dev_scales, format)) return rc;
    if (n == 0) return MTR_OK;
    if (!dev_out) return set_error(MTR_ERR_INVALID, "NULL argument");
    if (off(dev_out, size_of(dtype)) || (n > 1 && ld < d)) return set_error(MTR_ERR_INVALID, "bad row stride %lld or address", (long long)ld);
    DeviceGuard guard(device_id);
    if (!guard.ok) return set_error(MTR_ERR_HIP, "hipSetDevice(%d) failed", device_id);
    return launched("mtr_mx_dequantize", mtr::launch_mx_dequantize(dev_values, dev_scales, format, n, d, dev_out, dtype, ld,
                                                                   static_cast<hipStream_t>(stream)));
}

int mtr_rms_norm_mx(const void* dev_x, const void* dev_residual, const void* dev_weight, int32_t dtype, int32_t weight_dtype,
                    int64_t n, int32_t d, int64_t ld_x, int64_t ld_residual, float eps, int32_t format, void* dev_residual_out,
                    void* dev_values, void* dev_scales, int32_t device_id, void* stream) {
    if (!is_float(dtype)) return set_error(MTR_ERR_INVALID, "bad dtype %d", dtype);
    if (weight_dtype != dtype && weight_dtype != MTR_F32)
        return set_error(MTR_ERR_INVALID, "the weight must have the rows' dtype or be fp32, got %d", weight_dtype);
    if (int rc = check_rows("mtr_rms_norm_mx", n, d, dev_values, dev_scales, format)) return rc;
    if (d > MTR_RMS_NORM_MAX_WIDTH) return set_error(MTR_ERR_INVALID, "d=%d: at most %d", d, MTR_RMS_NORM_MAX_WIDTH);
    if (!(eps >= 0.f)) return set_error(MTR_ERR_INVALID, "eps must not be negative");
    if (n == 0) return MTR_OK;
    if (!dev_x || !dev_weight) return set_error(MTR_ERR_INVALID, "NULL argument");
    if (!dev_residual != !dev_residual_out)
        return set_error(MTR_ERR_INVALID, "a residual and the place for the updated one come together");
    if (dev_residual && (dev_residual_out == dev_residual || dev_residual_out == dev_x))
        return set_error(MTR_ERR_INVALID, "the updated residual wants memory of its own");
    const uintptr_t size = size_of(dtype);
    if (off(dev_x, size) || off(dev_weight, size_of(weight_dtype)) || off(dev_residual, size) || off(dev_residual_out, size) ||
        ld_x < 0 || ld_residual < 0)
        return set_error(MTR_ERR_INVALID, "bad row stride or address");
    DeviceGuard guard(device_id);
    if (!guard.ok) return set_error(MTR_ERR_HIP, "hipSetDevice(%d) failed", device_id);
    return launched("mtr_rms_norm_mx",
                    mtr::launch_rms_norm_mx(dev_x, dev_residual, dev_weight, dtype, weight_dtype, n, d, ld_x, ld_residual, eps, format,
                                            dev_residual_out, dev_values, dev_scales, static_cast<hipStream_t>(stream)));
}

int64_t mtr_mx_matmul_workspace(int64_t m, int64_t n, int32_t d) {
    if (m < 1 || n < 1 || d < 1 || d > kMost - MTR_MX_PAD || m > kMostProduct || n > kMostProduct) return 0;
    return mtr::mx_matmul_workspace(m, n, d);
}

int mtr_mx_matmul(const void* dev_a_values, const void* dev_a_scales, int32_t a_format, int64_t m, const void* dev_b_values,
                  const void* dev_b_scales, int64_t n, int32_t d, void* dev_out, int32_t out_dtype, int64_t ld_out,
                  void* dev_workspace, int64_t workspace_bytes, int32_t device_id, void* stream) {
    if (out_dtype != MTR_F32 && out_dtype != MTR_BF16) return set_error(MTR_ERR_INVALID, "bad output dtype %d", out_dtype);
    if (int rc = check_rows("mtr_mx_matmul", m, d, dev_a_values, dev_a_scales, a_format)) return rc;
    if (int rc = check_rows("mtr_mx_matmul", n, d, dev_b_values, dev_b_scales, MTR_MX_FP4)) return rc;
    if (m > kMostProduct || n > kMostProduct) return set_error(MTR_ERR_INVALID, "bad shape (m=%lld, n=%lld)", (long long)m, (long long)n);
    if (m == 0 || n == 0) return MTR_OK;
    if (!dev_out) return set_error(MTR_ERR_INVALID, "NULL argument");
    if (off(dev_out, size_of(out_dtype)) || (m > 1 && ld_out < n))
        return set_error(MTR_ERR_INVALID, "bad row stride %lld or address", (long long)ld_out);
    const int64_t need = mtr::mx_matmul_workspace(m, n, d);
    if (workspace_bytes < need || (need && (!dev_workspace || off(dev_workspace, 4))))
        return set_error(MTR_ERR_INVALID, "the workspace needs %lld bytes on 4, got %lld", (long long)need, (long long)workspace_bytes);
    DeviceGuard guard(device_id);
    if (!guard.ok) return set_error(MTR_ERR_HIP, "hipSetDevice(%d) failed", device_id);
    return launched("mtr_mx_matmul", mtr::launch_mx_matmul(dev_a_values, dev_a_scales, a_format, m, dev_b_values, dev_b_scales, n, d,
                                                           dev_out, out_dtype, ld_out, dev_workspace, static_cast<hipStream_t>(stream)));
}

int64_t mtr_token_logprobs_workspace(int64_t n, int64_t v, int32_t top_k) {
    if (n < 0 || v < 1 || v > kMost || n > kMost / 1024 || top_k < 0 || top_k > MTR_MAX_ALTERNATIVES) return 0;
    return mtr::token_logprobs_workspace(n, v, top_k);
}

int mtr_token_logprobs(const void* dev_logits, int32_t dtype, int64_t n, int64_t v, int64_t ld, const int64_t* dev_tokens,
                       int32_t n_tokens, int32_t top_k, float* dev_logprobs, float* dev_entropy, int64_t* dev_top_ids,
                       float* dev_top_logprobs, void* dev_workspace, int64_t workspace_bytes, int32_t device_id, void* stream) {
    if (!is_float(dtype)) return set_error(MTR_ERR_INVALID, "bad dtype %d", dtype);
    // rows are multiplied with up to 1024 parts of a row in the grid
    if (n < 0 || n > kMost / 1024 || v < 1 || v > kMost || ld < 0)
        return set_error(MTR_ERR_INVALID, "bad shape (n=%lld, v=%lld, row stride %lld)", (long long)n, (long long)v, (long long)ld);
    if (n_tokens < 0 || top_k < 0 || top_k > MTR_MAX_ALTERNATIVES)
        return set_error(MTR_ERR_INVALID, "n_tokens=%d must not be negative, top_k=%d in [0, %d]", n_tokens, top_k, MTR_MAX_ALTERNATIVES);
    if (n == 0) return MTR_OK;
    if (!dev_logits || !dev_entropy || (n_tokens && (!dev_tokens || !dev_logprobs)) || (top_k && (!dev_top_ids || !dev_top_logprobs)))
        return set_error(MTR_ERR_INVALID, "NULL argument");
    if (off(dev_logits, size_of(dtype)) || off(dev_tokens, 8) || off(dev_logprobs, 4) || off(dev_entropy, 4) || off(dev_top_ids, 8) ||
        off(dev_top_logprobs, 4))
        return set_error(MTR_ERR_INVALID, "bad address");
    const int64_t need = mtr::token_logprobs_workspace(n, v, top_k);
    if (workspace_bytes < need || (need && (!dev_workspace || off(dev_workspace, 8))))
        return set_error(MTR_ERR_INVALID, "the workspace needs %lld bytes on 8, got %lld", (long long)need, (long long)workspace_bytes);
    DeviceGuard guard(device_id);
    if (!guard.ok) return set_error(MTR_ERR_HIP, "hipSetDevice(%d) failed", device_id);
    return launched("mtr_token_logprobs",
                    mtr::launch_token_logprobs(dev_logits, dtype, n, v, ld, reinterpret_cast<const long long*>(dev_tokens), n_tokens, top_k,
                                               dev_logprobs, dev_entropy, reinterpret_cast<long long*>(dev_top_ids), dev_top_logprobs,
                                               dev_workspace, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
