// paged_decode16.hip -- paged attention over 16-bit pages, and the merge of
// the split partials (the kernel: paged_decode.h).
#include "paged_decode.h"

namespace mugen_attn {

// Log-sum-exp merge of the split partials of one output row, 64 dims a wave:
// lane s holds split s's (m, l), the first partials are in flight meanwhile
template <int D, bool LIST>
__global__ __launch_bounds__(64) void paged_combine_kernel(PagedDecodeParams p) {
    constexpr int kPre = 32;
    __shared__ float f_lds[64];
    // grid (H, q_len, B * D / 64): no division before the loads
    const int h = blockIdx.x, i = blockIdx.y, b = (int)blockIdx.z / (D / 64), lane = threadIdx.x;
    const int d = (int)blockIdx.z % (D / 64) * 64 + lane;
    const int planned = *p.plan;
    const paged::Lens len = paged::seq_lens_of(p, b);
    if (i >= len.n) return;  // no such token: its row stays as it was
    const int units = (p.chunk ? p.chunk : planned) >> 5;
    const int range = LIST ? paged::list_len(p, len.T - len.n + i + 1) << p.st.p_shift : len.T;
    const int nact = min(p.num_splits, paged::splits_of(range, units, plan_rcp(units)));
    if (nact <= 1) return;  // one split: the result is there
    const int64_t row = ((int64_t)b * p.q_len + i) * p.H + h;
    const float* ml = p.ws_ml + row * p.num_splits * 2;
    const float* os = p.ws_o + row * p.num_splits * D + d;
    float M = kNegInf, L = 0.f, O = 0.f;
    for (int s0 = 0; s0 < nact; s0 += 64) {
        const int ns = min(64, nact - s0);
        const float m = lane < ns ? ml[2 * (s0 + lane)] : kNegInf, l = lane < ns ? ml[2 * (s0 + lane) + 1] : 0.f;
        float v[kPre];
#pragma unroll
        for (int k = 0; k < kPre; k++) v[k] = os[(int64_t)(s0 + min(k, ns - 1)) * D];
        const float M2 = fmaxf(M, wave_max(m));
        const float old = M == kNegInf ? 0.f : fast_exp2(M - M2);
        const float f = m == kNegInf ? 0.f : fast_exp2(m - M2);
        L = L * old + wave_sum(f * l);
        O *= old;
        M = M2;
        f_lds[lane] = f;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        // (a weight of 0, also that of lanes past the splits, keeps out what its
        // partial may be; no branch, so the weights' LDS reads overlap)
        float acc[4] = {O, 0.f, 0.f, 0.f};
        auto add = [&](int k, float weight, float x) { acc[k & 3] = fmaf(weight, weight != 0.f ? x : 0.f, acc[k & 3]); };
#pragma unroll
        for (int k = 0; k < kPre; k++) add(k, f_lds[k], v[k]);
        for (int s = kPre; s < ns; s += 16) {
            float u[16];
#pragma unroll
            for (int k = 0; k < 16; k++) u[k] = os[(int64_t)(s0 + min(s + k, ns - 1)) * D];
#pragma unroll
            for (int k = 0; k < 16; k++) add(k, f_lds[s + k], u[k]);
        }
        O = (acc[0] + acc[1]) + (acc[2] + acc[3]);
        __builtin_amdgcn_wave_barrier();
    }
    O = L > 0.f ? O / L : L == L ? 0.f : L;
    if (p.out_dt == DT_F32) store_out<DT_F32>(p.out, row * D + d, O);
    else if (p.out_dt == DT_F16) store_out<DT_F16>(p.out, row * D + d, O);
    else store_out<DT_BF16>(p.out, row * D + d, O);
}

template <int D>
static hipError_t launch_combine_d(const PagedDecodeParams& p, hipStream_t st, KernelTimer* t) {
    const dim3 grid(p.H, p.q_len, (p.sel ? p.B / p.q_len : p.B) * (D / 64));
    if (p.sel) return launch_k(t, "gqa_decode_paged_combine", paged_combine_kernel<D, true>, grid, dim3(64), st, p);
    return launch_k(t, "gqa_decode_paged_combine", paged_combine_kernel<D, false>, grid, dim3(64), st, p);
}
hipError_t launch_paged_combine(const PagedDecodeParams& p, int D, hipStream_t st, KernelTimer* t) {
    if (D == 256) return launch_combine_d<256>(p, st, t);
    if (D == 128) return launch_combine_d<128>(p, st, t);
    return launch_combine_d<64>(p, st, t);
}

hipError_t launch_paged_decode16(const PagedDecodeParams& p, int nwg, int D, int dt, int wr, hipStream_t st,
                                 KernelTimer* t) {
    return paged::launch_decode<false>(p, nwg, D, dt, wr, st, t);
}

}  // namespace mugen_attn
