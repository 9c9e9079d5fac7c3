// paged_decode8.hip -- paged attention over E4M3 pages (the kernel:
// paged_decode.h).
#include "paged_decode.h"

namespace mugen_attn {

hipError_t launch_paged_decode8(const PagedDecodeParams& p, int nwg, int D, int dt, int wr, hipStream_t st,
                                KernelTimer* t) {
    return paged::launch_decode<true>(p, nwg, D, dt, wr, st, t);
}

}  // namespace mugen_attn
