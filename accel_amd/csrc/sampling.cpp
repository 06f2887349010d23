// The operator layer's sampling: argument checks and the launch (sample.hip).  A
// row's settings are on the device; what is out of range there has a meaning of its
// own instead of a refusal.
#include <hip/hip_runtime.h>

#include "checks.hpp"
#include "internal.hpp"

using namespace accel;

#define ACCEL_API extern "C" __attribute__((visibility("default")))

namespace {

// A vector of one setting a row, or none.
int check_setting(const char* op, const char* what, const accel_tensor_t* t, int32_t dtype,
                  int64_t rows, const void** data) {
    char buf[256];
    *data = nullptr;
    if (!t) return ACCEL_OK;
    if (!valid_tensor(t) || t->rank != 1 || t->dtype != dtype || t->shape[0] != rows) {
        snprintf(buf, sizeof buf, "%s must be a %s vector of %lld, one a row", what,
                 dtype_name(dtype), (long long)rows);
        return refuse(op, buf);
    }
    if (rows && !t->data) {
        snprintf(buf, sizeof buf, "%s is missing", what);
        return refuse(op, buf);
    }
    *data = t->data;
    return ACCEL_OK;
}

}  // namespace

ACCEL_API int accel_sample(int dev, void* stream, const accel_tensor_t* logits,
                           const accel_tensor_t* u, const accel_sampling_t* opt,
                           accel_tensor_t* tokens, accel_tensor_t* logprobs) {
    clear_error();
    const char* op = "Sample";
    char buf[256];
    if (!valid_tensor(logits) || (logits->rank != 1 && logits->rank != 2))
        return refuse(op, "the logits must be [rows, width] or [width]");
    if (logits->dtype != ACCEL_F32 && logits->dtype != ACCEL_F16 && logits->dtype != ACCEL_BF16) {
        snprintf(buf, sizeof buf, "the logits are %s; f32, f16 and bf16 are served",
                 dtype_name(logits->dtype));
        return refuse(op, buf);
    }
    const int64_t rows = logits->rank == 2 ? logits->shape[0] : 1;
    const int64_t width = logits->shape[logits->rank - 1];
    if (rows < 0 || rows > INT32_MAX || width < 1 || width > ACCEL_SAMPLE_WIDTH) {
        snprintf(buf, sizeof buf, "logits %s; up to 2^31 - 1 rows of 1 to %d are served",
                 shape_str(logits).c_str(), ACCEL_SAMPLE_WIDTH);
        return refuse(op, buf);
    }
    Sampling s{};
    const void* p[7];
    int rc;
    if (!u || !tokens) return refuse(op, "the random numbers or the tokens are missing");
    if ((rc = check_setting(op, "the random numbers", u, ACCEL_F32, rows, &p[0])) != ACCEL_OK ||
        (rc = check_setting(op, "the tokens", tokens, ACCEL_U32, rows, &p[1])) != ACCEL_OK ||
        (rc = check_setting(op, "the logarithms", logprobs, ACCEL_F32, rows, &p[2])) != ACCEL_OK)
        return rc;
    p[3] = p[4] = p[5] = p[6] = nullptr;
    if (opt) {
        if ((rc = check_setting(op, "temperature", opt->temperature, ACCEL_F32, rows, &p[3])) !=
                ACCEL_OK ||
            (rc = check_setting(op, "top_k", opt->top_k, ACCEL_U32, rows, &p[4])) != ACCEL_OK ||
            (rc = check_setting(op, "top_p", opt->top_p, ACCEL_F32, rows, &p[5])) != ACCEL_OK ||
            (rc = check_setting(op, "min_p", opt->min_p, ACCEL_F32, rows, &p[6])) != ACCEL_OK)
            return rc;
    }
    if (rows && !logits->data) return refuse(op, "the logits are missing");
    // rows are read in blocks of 16 bytes, from whichever of a block's numbers they begin at
    if ((uintptr_t)logits->data % (logits->dtype == ACCEL_F32 ? 4 : 2))
        return refuse(op, "the logits must start at an address aligned to their type");
    Device* d = device(dev);
    if (!d) return ACCEL_E_NO_DEVICE;
    if ((rc = begin_submission(d)) != ACCEL_OK || rows == 0) return rc;
    s.logits = logits->data;
    s.dtype = logits->dtype;
    s.rows = (uint32_t)rows;
    s.width = (uint32_t)width;
    s.u = static_cast<const float*>(p[0]);
    s.tokens = static_cast<uint32_t*>(const_cast<void*>(p[1]));
    s.logprobs = static_cast<float*>(const_cast<void*>(p[2]));
    s.temperature = static_cast<const float*>(p[3]);
    s.top_k = static_cast<const uint32_t*>(p[4]);
    s.top_p = static_cast<const float*>(p[5]);
    s.min_p = static_cast<const float*>(p[6]);
    int status = ACCEL_OK;
    const hipError_t e = launch_sample(d, (hipStream_t)stream, s, &status);
    return status != ACCEL_OK ? status : classify(d, e, "Sample launch");
}
