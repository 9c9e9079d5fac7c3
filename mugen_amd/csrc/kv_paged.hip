// kv_paged.hip -- append to the paged K/V cache with the rotation on the way,
// and the gather of one sequence's pages into contiguous 16-bit rows.
//
// Rows.  One thread rotates 2 x 8 values: dims 8u .. 8u+7 and their partners
// rope_dim/2 further on (16 adjacent dims past rope_dim, copied), of
// heads_per_thread heads of one token, so that the sine and cosine of a pair
// are formed once for all of them.  With turns = position * f / (2 pi) in 64 bits
// only the fraction of a turn goes to 32 bits: the phase of position 10^6 is as
// exact as that of position 1, where a float angle would be off by 10^6 * 2^-24
// radians.
//
// Pages (8-bit stores, and the key ranges of 16-bit ones).  One workgroup per
// (sequence, touched page, kv head, tensor) forms a page that these tokens
// fill from the rows that were there (ring or page) and the new ones, all in
// registers: magnitude, exponent, codes in one pass.  It rotates the new rows
// itself, so it need not wait for the row threads.  The ring slots of the open page's
// held rows, which the page job reads, are its own to write too: where a long prompt's
// newest tokens wrap around to them, the row threads leave those slots alone and the job
// writes them once it holds the old rows.
//
// Bound: the launch and two dependent reads (length, page table) for a few tokens: one
// token of 28 / 4 heads 3.1 us, of 64 sequences of 32 / 8 heads with 8-bit pages 4.0,
// and 1.5 more where one of them fills a page (one job's loads, reduction and codes).
// A prompt moves each row once and reads K and V once more for the pages: 2047 tokens
// of 28 / 4 heads, 40 MB, 11.4 us a call (3.5 TB/s): one wave of workgroups whose loads, sines
// and stores follow one another.
// The least e with amax <= 448 * 2^e: amax = m 2^x, 0.5 <= m < 1, is
// m * 2^(x-9) * 512, so e = x - 9 where m <= 448/512, else x - 8: no division.
#include "paged.h"

namespace mugen_attn {
namespace {

// the rotation of pairs 8u .. 8u+7 at a position
struct Turn8 {
    float c[8], s[8];
};
template <int N>
__device__ __forceinline__ Turn8 turn8(const RopeTurns<N>& t, int u, int pos) {
    Turn8 r;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const double a = (double)pos * t.f[8 * u + e];
        sincospif(2.0f * (float)(a - rint(a)), &r.s[e], &r.c[e]);
    }
    return r;
}
// (fused explicitly: the row threads and the page jobs round alike)
template <int DT>
__device__ __forceinline__ void rotate8(const Turn8& t, u32x4_t& a, u32x4_t& b) {
#pragma clang fp contract(off)
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float a0 = lo_f32<DT>(a[e]), a1 = hi_f32<DT>(a[e]), b0 = lo_f32<DT>(b[e]), b1 = hi_f32<DT>(b[e]);
        const float c0 = t.c[2 * e], c1 = t.c[2 * e + 1], s0 = t.s[2 * e], s1 = t.s[2 * e + 1];
        a[e] = pack2<DT>(fmaf(a0, c0, -(b0 * s0)), fmaf(a1, c1, -(b1 * s1)));
        b[e] = pack2<DT>(fmaf(b0, c0, a0 * s0), fmaf(b1, c1, a1 * s1));
    }
}
// first dims of a unit's two runs of 8
__device__ __forceinline__ void unit_dims(int u, int rope_dim, int& d0, int& d1) {
    const bool rot = 16 * u < rope_dim;
    d0 = rot ? 8 * u : 16 * u;
    d1 = rot ? 8 * u + rope_dim / 2 : 16 * u + 8;
}

// tokens that sequence b gets, and holds before
__device__ __forceinline__ void append_lens(const PagedAppendParams& p, int b, int& T, int& T_out) {
    T = clamp_len(p.seq_lens[b], p.st.max_T);
    const int n = p.new_lens ? min(max(p.new_lens[b], 0), p.n_new) : p.n_new;
    T_out = n < p.st.max_T - T ? T + n : p.st.max_T;
}

// 8-bit: new token `pos` goes to a ring slot that holds a row of the open page while
// a page job fills that page
__device__ __forceinline__ bool page_jobs_slot(const PagedAppendParams& p, int T, int T_out, int pos) {
    const int P = 1 << p.st.p_shift, open = T & -P;  // first token of the open page
    return T_out >= open + P && ((pos - open) & (p.st.ring - 1)) < T - open;
}

template <int D, int DT, bool BITS8>
__device__ __forceinline__ void append_rows(const PagedAppendParams& p, const RopeTurns<D / 2>& turns, uint32_t thread) {
    constexpr uint32_t U = D / 16;
    const int hpt = p.heads_per_thread, heads = p.H + 2 * p.st.Hk;
    const uint32_t groups = (uint32_t)(heads + hpt - 1) / (uint32_t)hpt;
    const int u = (int)(thread % U);
    const uint32_t token = thread / U / groups;  // b * n_new + j
    const int hg = (int)(thread / U - token * groups);
    if (token >= (uint32_t)p.n_seq * (uint32_t)p.n_new) return;
    const int b = (int)(token / (uint32_t)p.n_new), j = (int)token - b * p.n_new;
    const int64_t id = token;
    int T, T_out;
    append_lens(p, b, T, T_out);
    if (p.seq_lens_out && j == 0 && hg == 0 && u == 0) p.seq_lens_out[b] = T_out;
    const int pos = T + j;
    if (pos >= T_out) return;
    int d0, d1;
    unit_dims(u, p.rope_dim, d0, d1);
    const bool rot = 16 * u < p.rope_dim;
    const int h_end = min((hg + 1) * hpt, heads);
    // where the token's K and V rows go (heads kv_head elements apart; -1: nowhere)
    int64_t kv_at = -1, kv_head = D;
    uint16_t *k_to, *v_to;
    if constexpr (BITS8) {
        k_to = p.st.tail_k;
        v_to = p.st.tail_v;
        // (not if this call's own tokens push it out of the ring)
        if (pos >= T_out - p.st.ring && !page_jobs_slot(p, T, T_out, pos))
            kv_at = b * p.st.tail_stride + (int64_t)(pos & (p.st.ring - 1)) * p.st.Hk * D;
    } else {
        k_to = reinterpret_cast<uint16_t*>(p.st.k);
        v_to = reinterpret_cast<uint16_t*>(p.st.v);
        const int page = checked_page(p.st.table[b * p.st.table_stride + (pos >> p.st.p_shift)], p.st.n_pages);
        kv_head = (int64_t)D << p.st.p_shift;
        if (page >= 0) kv_at = (int64_t)page * p.st.Hk * kv_head + (pos & ((1 << p.st.p_shift) - 1)) * D;
    }
    Turn8 turn{};
    if (rot && hg * hpt < p.H + p.st.Hk) turn = turn8(turns, u, pos);  // (V heads come last)
    // four heads at a time: their rows are all on the way before the first is turned
    for (int h0 = hg * hpt; h0 < h_end; h0 += 4) {
        u32x4_t x[4], y[4];
        uint16_t* to[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int h = h0 + e;
            const uint16_t* src;
            to[e] = nullptr;
            if (h >= h_end) continue;
            if (h < p.H) {
                src = p.q + id * p.q_stride + (int64_t)h * D;
                to[e] = p.q_out + (id * p.H + h) * D;
            } else {
                const bool is_v = h >= p.H + p.st.Hk;
                const int kvh = h - p.H - (is_v ? p.st.Hk : 0);
                src = (is_v ? p.v_new + id * p.v_stride : p.k_new + id * p.k_stride) + (int64_t)kvh * D;
                if (kv_at >= 0) to[e] = (is_v ? v_to : k_to) + kv_at + (int64_t)kvh * kv_head;
            }
            if (!to[e]) continue;
            x[e] = load16(src + d0);
            y[e] = load16(src + d1);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (!to[e]) continue;
            if (rot && h0 + e < p.H + p.st.Hk) rotate8<DT>(turn, x[e], y[e]);
            *reinterpret_cast<u32x4_t*>(to[e] + d0) = x[e];
            *reinterpret_cast<u32x4_t*>(to[e] + d1) = y[e];
        }
    }
}

// Two 16-bit floats as unsigned numbers of the same order, `lo` from below and `hi`
// from above, so that the least of either is the minimum and the maximum; a NaN is the
// least of both.  Packed 16-bit integers: 12 instructions for a pair and its two minima.
using u16x2_t = unsigned short __attribute__((ext_vector_type(2)));
using s16x2_t = short __attribute__((ext_vector_type(2)));
template <int DT>
__device__ __forceinline__ void range_keys(uint32_t x, uint32_t& lo, uint32_t& hi) {
    const u16x2_t v = __builtin_bit_cast(u16x2_t, x), one = {1, 1};
    const u16x2_t inf = DT == DT_F16 ? u16x2_t{0x7c00, 0x7c00} : u16x2_t{0x7f80, 0x7f80};
    const u16x2_t sign = __builtin_bit_cast(u16x2_t, __builtin_bit_cast(s16x2_t, v) >> 15);
    const u16x2_t key = v ^ (sign | u16x2_t{0x8000, 0x8000});
    const u16x2_t nan = __builtin_elementwise_min(__builtin_elementwise_sub_sat(v & u16x2_t{0x7fff, 0x7fff}, inf), one);
    const u16x2_t keep = nan - one;  // (0 for a NaN, else all ones)
    lo = __builtin_bit_cast(uint32_t, key & keep);
    hi = __builtin_bit_cast(uint32_t, ~key & keep);
}
__device__ __forceinline__ uint32_t least2(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}
// the floats again (is_hi: from a `hi`)
__device__ __forceinline__ uint32_t range_values(uint32_t k, bool is_hi) {
    const u16x2_t key = __builtin_bit_cast(u16x2_t, is_hi ? ~k : k);
    const u16x2_t pos = __builtin_bit_cast(u16x2_t, __builtin_bit_cast(s16x2_t, key) >> 15);
    return __builtin_bit_cast(uint32_t, key ^ (~pos | u16x2_t{0x8000, 0x8000}));
}

// the page that job `id` is about, where this call fills it
template <int D, int P, int DT, bool BITS8>
__device__ __forceinline__ void append_page(const PagedAppendParams& p, const RopeTurns<D / 2>& turns, int id, char* lds) {
    constexpr int U = D / 16, UNITS = P * U, UPT = (UNITS + 255) / 256;
    // job = ((b * pages + c) * tensors + tensor) * Hk + kvh
    const int Hk = p.st.Hk;
    const int kvh = id % Hk;
    id /= Hk;
    bool is_v = false;
    if constexpr (BITS8) {
        is_v = id & 1;
        id >>= 1;
    }
    const int b = id / p.pages, c = id - b * p.pages;
    int T, T_out;
    append_lens(p, b, T, T_out);
    const int page = T / P + c;
    if (page >= T_out / P) return;  // not filled by this call
    const int phys = checked_page(p.st.table[b * p.st.table_stride + page], p.st.n_pages);
    if (phys < 0 && !(BITS8 && c == 0)) return;  // (its ring slots are still this job's)
    const int64_t ph = (int64_t)phys * Hk + kvh;
    const bool ranged = !is_v && p.st.k_range;
    // (+: a choice of two values, where the choice of the two members copies the struct to scratch)
    uint16_t* const tail = is_v ? +p.st.tail_v : +p.st.tail_k;
    u32x4_t xa[UPT], xb[UPT];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < UPT; i++) {
        const int unit = threadIdx.x + 256 * i;
        xa[i] = xb[i] = u32x4_t{0, 0, 0, 0};
        if (unit >= UNITS) continue;
        const int r = unit / U, u = unit % U, t = page * P + r;
        int d0, d1;
        unit_dims(u, p.rope_dim, d0, d1);
        if (t >= T) {
            const int64_t row = (int64_t)b * p.n_new + (t - T);
            const uint16_t* src = (is_v ? p.v_new + row * p.v_stride : p.k_new + row * p.k_stride) + (int64_t)kvh * D;
            xa[i] = load16(src + d0);
            xb[i] = load16(src + d1);
            if (!is_v && 16 * u < p.rope_dim) rotate8<DT>(turn8(turns, u, t), xa[i], xb[i]);
        } else {
            const uint16_t* src;
            if constexpr (BITS8)
                src = tail + b * p.st.tail_stride + ((int64_t)(t & (p.st.ring - 1)) * Hk + kvh) * D;
            else src = reinterpret_cast<const uint16_t*>(p.st.k) + (ph * P + r) * D;
            xa[i] = load16(src + d0);
            xb[i] = load16(src + d1);
        }
        if constexpr (BITS8) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float v[4] = {lo_f32<DT>(xa[i][e]), hi_f32<DT>(xa[i][e]), lo_f32<DT>(xb[i][e]), hi_f32<DT>(xb[i][e])};
#pragma unroll
                for (int k = 0; k < 4; k++) amax = fmaxf(amax, fabsf(v[k]) < -kNegInf ? fabsf(v[k]) : 0.f);
            }
        }
    }
    int byte = 127;
    uint32_t code[UPT][4];
    if constexpr (BITS8) {
        float* red = reinterpret_cast<float*>(lds);
        amax = wave_max(amax);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = amax;
        __syncthreads();  // (and every old row of the page is in registers)
        amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        __syncthreads();
        if (c == 0) {
            // the newest tokens whose slots those rows had
            const int held = T - page * P;
            for (int unit = threadIdx.x; unit < held * U; unit += 256) {
                const int r = unit / U, u = unit % U, slot = (page * P + r) & (p.st.ring - 1);
                // the last token before T_out at this slot
                const int t = T_out - 1 - ((T_out - 1 - slot) & (p.st.ring - 1));
                if (t < T) continue;
                int d0, d1;
                unit_dims(u, p.rope_dim, d0, d1);
                const int64_t row = (int64_t)b * p.n_new + (t - T);
                const uint16_t* src = (is_v ? p.v_new + row * p.v_stride : p.k_new + row * p.k_stride) + (int64_t)kvh * D;
                u32x4_t x = load16(src + d0), y = load16(src + d1);
                if (!is_v && 16 * u < p.rope_dim) rotate8<DT>(turn8(turns, u, t), x, y);
                uint16_t* dst = tail + b * p.st.tail_stride + ((int64_t)slot * Hk + kvh) * D;
                *reinterpret_cast<u32x4_t*>(dst + d0) = x;
                *reinterpret_cast<u32x4_t*>(dst + d1) = y;
            }
        }
        if (phys < 0) return;
        byte = 1;
        if (amax > 0.f) {
            int x;
            const float m = frexpf(amax, &x);
            byte = min(max(x - (m <= 0.875f ? 9 : 8) + 127, 1), 254);
        }
        const float inv = ldexpf(1.f, 127 - byte);
        auto enc = [&](float a, float c2, uint32_t old, auto hi) -> uint32_t {
            // E4M3 rounds to nearest even; in range by the choice of the exponent
            uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a * inv, c2 * inv, (int)old, decltype(hi)::value);
            constexpr int sh = decltype(hi)::value ? 16 : 0;
            if (!(fabsf(a) < -kNegInf)) w = (w & ~(0xffu << sh)) | (0x7fu << sh);
            if (!(fabsf(c2) < -kNegInf)) w = (w & ~(0xff00u << sh)) | (0x7f00u << sh);
            return w;
        };
#pragma unroll
        for (int i = 0; i < UPT; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const u32x4_t& x = e < 2 ? xa[i] : xb[i];
                const int k = 2 * (e & 1);
                uint32_t w = enc(lo_f32<DT>(x[k]), hi_f32<DT>(x[k]), 0u, std::false_type{});
                code[i][e] = enc(lo_f32<DT>(x[k + 1]), hi_f32<DT>(x[k + 1]), w, std::true_type{});
            }
        if (threadIdx.x == 0) (is_v ? +p.st.v_exp : +p.st.k_exp)[ph] = (uint8_t)byte;
#pragma unroll
        for (int i = 0; i < UPT; i++) {
            const int unit = threadIdx.x + 256 * i;
            if (unit >= UNITS) continue;
            const int r = unit / U, u = unit % U;
            int d0, d1;
            unit_dims(u, p.rope_dim, d0, d1);
            uint8_t* dst = is_v ? reinterpret_cast<uint8_t*>(lds) + r * D : p.st.k + (ph * P + r) * D;
            *reinterpret_cast<u32x2_t*>(dst + d0) = u32x2_t{code[i][0], code[i][1]};
            *reinterpret_cast<u32x2_t*>(dst + d1) = u32x2_t{code[i][2], code[i][3]};
        }
        if (is_v) {  // [P][D] in LDS -> [P/32][D][32]: 16 tokens of a dim a thread
            __syncthreads();
            const uint8_t* rows = reinterpret_cast<const uint8_t*>(lds);
            for (int i = threadIdx.x; i < P * D / 16; i += 256) {
                const int d = (i >> 1) % D, t0 = 32 * ((i >> 1) / D) + 16 * (i & 1);
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const uint32_t x = rows[(t0 + e) * D + d];
                    w[e >> 2] = (e & 3) ? w[e >> 2] | (x << (8 * (e & 3))) : x;
                }
                *reinterpret_cast<u32x4_t*>(p.st.v + ph * P * D + 16 * (int64_t)i) = u32x4_t{w[0], w[1], w[2], w[3]};
            }
            return;
        }
    }
    if (!ranged) return;
    // minimum and maximum of each dim: a thread's own rows, then over the lanes of the same
    // dims (each exchange leaves a lane half of the words: the minima or the maxima, then
    // the first or the second eight dims), then over the waves through LDS: 0.8 us of a step
    // in which a page of 64 fills (all threads' values through LDS, twice: 2.6)
    uint32_t m[16];
#pragma unroll
    for (int e = 0; e < 16; e++) m[e] = 0xffffffffu;
    const float scale = exp_scale((uint32_t)byte);
#pragma unroll
    for (int i = 0; i < UPT; i++) {
        if (threadIdx.x + 256 * i >= UNITS) continue;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            uint32_t w, lo, hi;
            if constexpr (BITS8)
                w = (e & 1) ? cvt2_fp8<DT, true>(code[i][e >> 1], scale) : cvt2_fp8<DT, false>(code[i][e >> 1], scale);
            else w = e < 4 ? xa[i][e] : xb[i][e - 4];
            range_keys<DT>(w, lo, hi);
            m[e] = least2(m[e], lo);
            m[8 + e] = least2(m[8 + e], hi);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const auto r = __builtin_amdgcn_permlane32_swap(m[e], m[8 + e], false, false);
        m[e] = least2(r[0], r[1]);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const auto r = __builtin_amdgcn_permlane16_swap(m[e], m[4 + e], false, false);
        m[e] = least2(r[0], r[1]);
        if constexpr (U <= 8) m[e] = least2(m[e], __float_as_uint(dpp_xor<8>(__uint_as_float(m[e]))));
        if constexpr (U <= 4) m[e] = least2(m[e], __float_as_uint(dpp_xor<4>(__uint_as_float(m[e]))));
    }
    u32x4_t* part = reinterpret_cast<u32x4_t*>(lds);  // [wave][minimum, maximum][d0, d1][U]
    const int lane = threadIdx.x & 63, l16 = lane & 15;
    if (l16 < U) part[(threadIdx.x >> 6) * 4 * U + (lane >> 4) * U + l16] = u32x4_t{m[0], m[1], m[2], m[3]};
    __syncthreads();
    if (threadIdx.x < 4 * U) {
        const int u = threadIdx.x % U, which = threadIdx.x / U;
        u32x4_t r = part[threadIdx.x];
#pragma unroll
        for (int w = 1; w < 4; w++) {
            const u32x4_t x = part[w * 4 * U + threadIdx.x];
#pragma unroll
            for (int e = 0; e < 4; e++) r[e] = least2(r[e], x[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) r[e] = range_values(r[e], which >= 2);
        int d0, d1;
        unit_dims(u, p.rope_dim, d0, d1);
        *reinterpret_cast<u32x4_t*>(p.st.k_range + (ph * 2 + (which >> 1)) * D + ((which & 1) ? d1 : d0)) = r;
    }
}

template <int D, int DT, bool BITS8>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendParams p, RopeTurns<D / 2> turns) {
    if ((int)blockIdx.x < p.row_blocks) {
        append_rows<D, DT, BITS8>(p, turns, blockIdx.x * 256u + threadIdx.x);
        return;
    }
    // a page's V codes; the ranges' partials of 4 waves, at most 4 KiB
    __shared__ __attribute__((aligned(16))) char lds[BITS8 ? 128 * D : 4096];
    const int id = (int)blockIdx.x - p.row_blocks;
    if (p.st.p_shift == 5) append_page<D, 32, DT, BITS8>(p, turns, id, lds);
    else if (p.st.p_shift == 6) append_page<D, 64, DT, BITS8>(p, turns, id, lds);
    else append_page<D, 128, DT, BITS8>(p, turns, id, lds);
}

// 32 tokens of one kv head: pages (or ring) -> [T][Hk * D] rows.  V codes, [dim][32
// tokens], turn through LDS in rows of D + 8 values (16 bytes off the banks of the row
// before).  8184 tokens of 4 kv heads d128, 25 MB: 4.5 us (5.6 TB/s, the writes held by
// the cache that the prefill then reads)
template <int D, int DT, bool BITS8>
__global__ __launch_bounds__(256) void paged_gather_kernel(PagedGatherParams p) {
    __shared__ __attribute__((aligned(16))) uint16_t tile[BITS8 ? 32 * (D + 8) : 8];
    const int t0 = 32 * (int)blockIdx.x, kvh = blockIdx.y, Hk = p.st.Hk;
    const int ps = p.st.p_shift, P = 1 << ps, lp = t0 >> ps;
    const int n = min(32, p.T - t0);
    const int64_t row = (int64_t)Hk * D;
    uint16_t* ko = p.k_out + t0 * row + (int64_t)kvh * D;
    uint16_t* vo = p.v_out + t0 * row + (int64_t)kvh * D;
    const uint16_t *ks = nullptr, *vs = nullptr;
    int64_t srow = D;
    int phys = -1;
    if (BITS8 && (lp + 1) * P > p.T) {
        const int64_t o = p.seq * p.st.tail_stride + ((int64_t)(t0 & (p.st.ring - 1)) * Hk + kvh) * D;
        ks = p.st.tail_k + o;
        vs = p.st.tail_v + o;
        srow = row;
    } else {
        phys = checked_page(p.st.table[p.seq * p.st.table_stride + lp], p.st.n_pages);
        if (!BITS8 && phys >= 0) {
            const int64_t o = ((((int64_t)phys * Hk + kvh) << ps) + (t0 & (P - 1))) * D;
            ks = reinterpret_cast<const uint16_t*>(p.st.k) + o;
            vs = reinterpret_cast<const uint16_t*>(p.st.v) + o;
        }
    }
    if (ks || phys < 0) {  // 16-bit rows, or none: zeros
        for (int i = threadIdx.x; i < n * (D / 8); i += 256) {
            const int r = i / (D / 8), d = 8 * (i % (D / 8));
            *reinterpret_cast<u32x4_t*>(ko + r * row + d) = ks ? load16(ks + r * srow + d) : u32x4_t{0, 0, 0, 0};
            u32x4_t v = ks ? load16(vs + r * srow + d) : u32x4_t{0, 0, 0, 0};
            if (DT == DT_BF16 && p.v16) {
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = pack2<DT_F16>(lo_f32<DT>(v[e]), hi_f32<DT>(v[e]));
            }
            *reinterpret_cast<u32x4_t*>(vo + r * row + d) = v;
        }
        return;
    }
    if constexpr (BITS8) {
        const int64_t ph = (int64_t)phys * Hk + kvh;
        const float sk = exp_scale(p.st.k_exp[ph]), sv = exp_scale(p.st.v_exp[ph]);
        const uint8_t* k8 = p.st.k + ((ph << ps) + (t0 & (P - 1))) * D;
        const uint8_t* v8 = p.st.v + ((ph << ps) + (t0 & (P - 1))) * D;  // tile (t0 % P) / 32 of 32 * D bytes
        for (int i = threadIdx.x; i < 32 * D / 16; i += 256) {
            const u32x4_t w = load16(k8 + 16 * i);
            uint16_t* dst = ko + (i / (D / 16)) * row + 16 * (i % (D / 16));
            *reinterpret_cast<u32x4_t*>(dst) = cvt8_fp8<DT>(w[0], w[1], sk);
            *reinterpret_cast<u32x4_t*>(dst + 8) = cvt8_fp8<DT>(w[2], w[3], sk);
            const u32x4_t x = load16(v8 + 16 * i);
            const int d = i >> 1, r = 16 * (i & 1);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const u32x4_t y = DT == DT_F16 || p.v16 ? cvt8_fp8<DT_F16>(x[2 * h], x[2 * h + 1], sv)
                                                        : cvt8_fp8<DT>(x[2 * h], x[2 * h + 1], sv);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    tile[(r + 8 * h + 2 * e) * (D + 8) + d] = (uint16_t)y[e];
                    tile[(r + 8 * h + 2 * e + 1) * (D + 8) + d] = (uint16_t)(y[e] >> 16);
                }
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n * (D / 8); i += 256) {  // (a whole page: n = 32)
            const int r = i / (D / 8), d = 8 * (i % (D / 8));
            *reinterpret_cast<u32x4_t*>(vo + r * row + d) = load16(&tile[r * (D + 8) + d]);
        }
    }
}

template <typename F>
hipError_t by_shape(int D, int dt, bool bits8, F f) {
    auto by_dt = [&](auto d) {
        auto by_bits = [&](auto t) {
            return bits8 ? f(d, t, std::true_type{}) : f(d, t, std::false_type{});
        };
        return dt == DT_F16 ? by_bits(std::integral_constant<int, DT_F16>{}) : by_bits(std::integral_constant<int, DT_BF16>{});
    };
    if (D == 256) return by_dt(std::integral_constant<int, 256>{});
    if (D == 128) return by_dt(std::integral_constant<int, 128>{});
    return by_dt(std::integral_constant<int, 64>{});
}

}  // namespace

hipError_t launch_paged_append(PagedAppendParams p, const RopeTurns<128>& turns, int D, int dt, bool bits8, hipStream_t st, KernelTimer* t) {
    const int heads = p.H + 2 * p.st.Hk, groups = (heads + p.heads_per_thread - 1) / p.heads_per_thread;
    const int64_t threads = (int64_t)p.n_seq * p.n_new * groups * (D / 16);
    p.row_blocks = (int)((threads + 255) / 256);
    const int jobs = bits8 || p.st.k_range ? p.n_seq * p.pages * p.st.Hk * (bits8 ? 2 : 1) : 0;
    return by_shape(D, dt, bits8, [&](auto d, auto e, auto b8) {
        constexpr int DD = decltype(d)::value;
        RopeTurns<DD / 2> f;
        for (int i = 0; i < DD / 2; i++) f.f[i] = turns.f[i];
        return launch_k(t, "kv_paged_append", paged_append_kernel<DD, decltype(e)::value, decltype(b8)::value>,
                        dim3(p.row_blocks + jobs), dim3(256), st, p, f);
    });
}

hipError_t launch_paged_gather(const PagedGatherParams& p, int D, int dt, bool bits8, hipStream_t st, KernelTimer* t) {
    return by_shape(D, dt, bits8, [&](auto d, auto e, auto b8) {
        return launch_k(t, "paged_gather", paged_gather_kernel<decltype(d)::value, decltype(e)::value, decltype(b8)::value>,
                        dim3((p.T + 31) / 32, p.st.Hk), dim3(256), st, p);
    });
}

}  // namespace mugen_attn
