// capi_common.h -- what the extern "C" entry points share (capi.hip,
// paged_capi.hip): the thread's error message and the kernel timer.
#pragma once
#include <hip/hip_runtime.h>

#include "mugen_attn.h"
#include "kernels.h"

namespace mugen_attn {

// sets mugen_attn_last_error() and returns `code`
__attribute__((format(printf, 2, 3))) int fail(int code, const char* fmt, ...);
int hip_status(hipError_t e, const char* what);
KernelTimer* active_timer();

}  // namespace mugen_attn
