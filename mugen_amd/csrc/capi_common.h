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

// mugen_attn_gqa_prefill, and the same for a caller that has V in fp16 already:
// whether the call would copy it (BF16), and the workspace it then needs with the
// key splits' partials in fp32 (part32)
int prefill_run(const mugen_attn_gqa_prefill_args* a, bool v16, void* stream, bool part32 = false);
bool prefill_takes_v16(const mugen_attn_gqa_prefill_args* a);
size_t prefill_split_workspace(const mugen_attn_gqa_prefill_args* a);

}  // namespace mugen_attn
