// rt_capi_util.hpp -- error-reporting helpers shared by the C ABI sources.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/rt_hip.h"

namespace rt {

// Record a printf-style message for rt_last_error() and return `code`.
rt_status set_error(rt_status code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
// RT_OK for hipSuccess, otherwise RT_ENOMEM / RT_EHIP with the HIP message.
rt_status hip_error(hipError_t e, const char *what);
bool aligned16(const void *p);
// The calling thread's GEMM workspace for `stream` on the current device, of at
// least `bytes`; RT_ESTATE if it would have to grow while the stream is captured.
rt_status gemm_workspace(size_t bytes, hipStream_t stream, void **out);

// c = a . W^T (+ bias) on an MXFP4 weight, arguments checked here; act is an MxAct.
rt_status mx_product(const char *who, int act, const void *a, const void *w, const float *bias, void *c, bool c_bf16,
                     int64_t m, int64_t n, int64_t k, hipStream_t s);

}  // namespace rt
