// page_select.hip -- the choice of the pages a query reads
// (mugen_attn_page_select): a score kernel over the page ranges, then a top-k per
// (query, kv head).
//
// Score.  sum over heads and dims of max(q min, q max) = Q-.min + Q+.max with
// Q-, Q+ the sums over the group's heads of the negative and the positive parts
// of q: one product of 2 * head_dim terms per page whatever the group's size.
// In 64 bits: 16-bit factors make 22-bit products, so the sums come out the same in
// any order but for terms 2^30 apart, and a page next to the border does not change
// sides with the kernel's tiling.  16 lanes take a page (2 * head_dim contiguous values), 4 pages
// a wave instruction; every query of a sequence is scored from one read.
// Bound: HBM (4 * head_dim bytes a page and kv head) past some ten MB, latency below:
// the launch and four dependent reads (lengths, table, ranges, queries).  4.2 MB of
// one sequence of 131k tokens 4.3 us, 17.7 MB of 16 sequences 8.7 (2 TB/s).  (The
// queries' loads ahead of the table's: no gain, 4.3 and 9.0.)
//
// Choice.  Scores become 64-bit integers of the same order, held in registers.  One
// histogram over 1024 equal bins between the least and the largest score finds the bin
// of the border; the few keys in it are ranked by one wave.  Where more than 64
// share the bin (equal or very uneven scores), a radix select takes over: 8 bits a
// pass from the highest bit in which any two candidates differ, then, among equal
// keys, over the page number (the lowest pages win).  Either way the choice is a
// border (key, page), and a ballot with one scan places the ascending list.
// Bound: latency, a chain of 8 barriers (radix passes alone: 20, 2048 pages 7.7 us;
// now 5.8, and 4.7 to 5.6 up to 1024 pages).
#include <algorithm>

#include "paged.h"

namespace mugen_attn {
namespace {

__device__ __forceinline__ double row_sum16(double v) {  // over the 16 lanes of a row, in every lane
    auto step = [&](auto ctrl) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)u, decltype(ctrl)::value, 0xF, 0xF, false);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), decltype(ctrl)::value, 0xF, 0xF, false);
        v += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
    };
    step(std::integral_constant<int, 0x128>{});  // row rotations by 8, 4, 2, 1
    step(std::integral_constant<int, 0x124>{});
    step(std::integral_constant<int, 0x122>{});
    step(std::integral_constant<int, 0x121>{});
    return v;
}

// what query i of sequence b sees
struct Seen {
    int n;      // new tokens of the sequence
    int pages;  // pages that query i sees
};
__device__ __forceinline__ int select_len(const PageSelectParams& p, int b) { return clamp_len(p.seq_lens[b], p.st.max_T); }
__device__ __forceinline__ int select_new(const PageSelectParams& p, int b) {
    return p.q_lens ? min(max(p.q_lens[b], 0), p.q_len) : p.q_len;
}
__device__ __forceinline__ int pages_seen(const PageSelectParams& p, int T, int n, int i) {
    return (max(T - n + i + 1, 0) + (1 << p.st.p_shift) - 1) >> p.st.p_shift;
}

// pages of a score item, 16 a step: all their ranges are in flight at once, and the
// group's queries are summed meanwhile
template <int D>
constexpr int score_pages() { return D == 64 ? 64 : D == 128 ? 32 : 16; }
constexpr int kScoreQueries = 4;  // queries whose Q-, Q+ are held at a time

// candidates of sequence b's last query, the one that sees most, and whether any
// query leaves pages out
__device__ __forceinline__ int score_end(const PageSelectParams& p, int b) {
    const int n = select_new(p, b);
    const int pages = n > 0 ? pages_seen(p, select_len(p, b), n, n - 1) : 0;
    return pages > p.n_select ? pages - p.n_last : 0;
}

// The items (sequence, kv head, score_pages pages) are a compact list, walked by as
// many workgroups as the card holds: one workgroup for each item of the longest
// sequence allowed left most of them to find out that there was nothing to do
// (16 sequences of 1k..32k tokens, 8 kv heads, d64: 13.4 -> 9.8 us)
using f64x2_t = double __attribute__((ext_vector_type(2)));
template <int D, int DT>
__global__ __launch_bounds__(256) void page_score_kernel(PageSelectParams p) {
    constexpr int C = 2 * D / 128;  // 16-byte loads of a lane per page
    constexpr int PAGES = score_pages<D>(), STEPS = PAGES / 16;
    // [16 dims][pair of dims][lane]: the 16 lanes' pairs lie side by side (each lane's 8
    // dims in a row put every fourth lane on the same banks)
    __shared__ __attribute__((aligned(16))) double Q[kScoreQueries][2 * D];
    auto at = [](int d) { return (d / 128 * 4 + d % 8 / 2) * 32 + d / 8 % 16 * 2 + d % 2; };
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l16 = lane & 15;
    for (int item = blockIdx.x;; item += gridDim.x) {
    int b, r;
    if (!find_sequence(p.B, item, [&](int j) { return (score_end(p, j) + PAGES - 1) / PAGES * p.st.Hk; }, b, r)) return;
    const int kvh = r % p.st.Hk, page0 = r / p.st.Hk * PAGES;
    const int n = select_new(p, b), end = score_end(p, b);
    // this wave's pages: page0 + 16 * step + 4 * wave + lane / 16
    u32x4_t raw[STEPS][C];
    int phys[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; s++)
        phys[s] = p.st.table[b * p.st.table_stride + min(page0 + 16 * s + 4 * wave + (lane >> 4), end - 1)];
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
        phys[s] = checked_page(phys[s], p.st.n_pages);
        const uint16_t* src = p.st.k_range + ((int64_t)max(phys[s], 0) * p.st.Hk + kvh) * 2 * D;
#pragma unroll
        for (int c = 0; c < C; c++) raw[s][c] = load16(src + 8 * (16 * c + l16));
    }
    for (int i0 = 0; i0 < n; i0 += kScoreQueries) {
        const int ni = min(kScoreQueries, n - i0);
        __syncthreads();  // (the sums before are read)
        for (int x = threadIdx.x; x < ni * (D / 2); x += 256) {  // two dims a thread
            const int i = x / (D / 2), d = 2 * (x - i * (D / 2));
            const uint16_t* q = p.q + (((int64_t)b * p.q_len + i0 + i) * p.H + (int64_t)kvh * p.G) * D + d;
            uint32_t w[16];
#pragma unroll
            for (int h = 0; h < 16; h++) w[h] = *reinterpret_cast<const uint32_t*>(q + min(h, p.G - 1) * D);
            double neg0 = 0.0, pos0 = 0.0, neg1 = 0.0, pos1 = 0.0;
#pragma unroll
            for (int h = 0; h < 16; h++) {
                if (h >= p.G) break;
                const double v0 = (double)lo_f32<DT>(w[h]), v1 = (double)hi_f32<DT>(w[h]);
                neg0 += v0 < 0.0 ? v0 : 0.0;
                pos0 += v0 < 0.0 ? 0.0 : v0;  // (a NaN too)
                neg1 += v1 < 0.0 ? v1 : 0.0;
                pos1 += v1 < 0.0 ? 0.0 : v1;
            }
            *reinterpret_cast<f64x2_t*>(&Q[i][at(d)]) = f64x2_t{neg0, neg1};
            *reinterpret_cast<f64x2_t*>(&Q[i][at(D + d)]) = f64x2_t{pos0, pos1};
        }
        __syncthreads();
        double x[STEPS][8 * C];
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[s][8 * c + 2 * e] = (double)lo_f32<DT>(raw[s][c][e]);
                    x[s][8 * c + 2 * e + 1] = (double)hi_f32<DT>(raw[s][c][e]);
                }
        for (int i = 0; i < ni; i++) {
            double part[STEPS][2] = {};  // (two chains a page: an fma takes 8 cycles to come back)
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const f64x2_t w = *reinterpret_cast<const f64x2_t*>(&Q[i][at(8 * (16 * c + l16) + e)]);
#pragma unroll
                    for (int s = 0; s < STEPS; s++) {
                        part[s][0] = fma(w[0], x[s][8 * c + e], part[s][0]);
                        part[s][1] = fma(w[1], x[s][8 * c + e + 1], part[s][1]);
                    }
                }
#pragma unroll
            for (int s = 0; s < STEPS; s++) {
                const int page = page0 + 16 * s + 4 * wave + (lane >> 4);
                double sum = row_sum16(part[s][0] + part[s][1]) + 0.0;  // (-0 counts as 0)
                uint64_t key = __builtin_bit_cast(uint64_t, sum);
                key = sum != sum ? ~0ull : (key >> 63) ? ~key : key | (1ull << 63);
                if (phys[s] < 0) key = 0;
                if (l16 == 0 && page < end)
                    p.keys[(((int64_t)b * p.q_len + i0 + i) * p.st.Hk + kvh) * p.max_pages + page] = key;
            }
        }
    }
    }
}

// minimum (MAX: maximum) over the wave, in every lane
template <bool MAX>
__device__ __forceinline__ float wave_least(float v) { return MAX ? wave_max(v) : -wave_max(-v); }

// the bin, counted from the top one, that holds the need-th key: hist[n_bins],
// n_bins a multiple of 64; leaves (bin, keys wanted in it, keys in it) in `pick`
__device__ __forceinline__ void find_bin(const uint32_t* hist, int n_bins, int need, int lane, int* pick) {
    const int per = n_bins / 64, top = n_bins - 1 - per * lane;
    uint32_t sum = 0;
    for (int e = 0; e < per; e++) sum += hist[top - e];
    const int incl = wave_scan_i32((int)sum);
    if (lane == __builtin_ctzll(__ballot(incl >= need))) {
        int above = incl - (int)sum, e = 0;
        while (e < per - 1 && above + (int)hist[top - e] < need) above += (int)hist[top - e++];
        pick[0] = top - e;
        pick[1] = need - above;
        pick[2] = (int)hist[top - e];
    }
}

template <int WAVES, int KPT>
__global__ __launch_bounds__(64 * WAVES) void page_select_kernel(PageSelectParams p) {
    constexpr int NT = 64 * WAVES, BINS = 1024;
    __shared__ uint32_t hist[BINS];
    __shared__ uint32_t counts[KPT * WAVES];
    __shared__ float red[2 * WAVES];
    __shared__ uint64_t list_key[64];
    __shared__ int list_page[64];
    __shared__ uint32_t list_n;
    __shared__ int pick[3];
    __shared__ uint64_t border_key;
    __shared__ int border_page;
    const int kvh = blockIdx.x, i = blockIdx.y, b = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int T = select_len(p, b), n = select_new(p, b);
    if (i >= n) return;
    int32_t* out = p.pages + (((int64_t)b * p.q_len + i) * p.st.Hk + kvh) * p.n_select;
    const int pages = pages_seen(p, T, n, i);
    if (pages <= p.n_select) {  // all of them
        for (int x = tid; x < p.n_select; x += NT) out[x] = x < pages ? x : -1;
        return;
    }
    const int first = p.n_first, end = pages - p.n_last;  // candidates [first, end)
    int need = p.n_select - p.n_first - p.n_last;
    const uint64_t* keys = p.keys + (((int64_t)b * p.q_len + i) * p.st.Hk + kvh) * p.max_pages;
    uint64_t key[KPT];
    float val[KPT];  // the score in fp32: of the same order, but for equal roundings
    float lo = -kNegInf, hi = kNegInf;
    auto cand = [&](int m) { return m * NT + tid >= first && m * NT + tid < end; };
#pragma unroll
    for (int m = 0; m < KPT; m++) {
        key[m] = cand(m) ? keys[m * NT + tid] : 0;
        const uint64_t bits = (key[m] >> 63) ? key[m] & ~(1ull << 63) : ~key[m];
        val[m] = key[m] == ~0ull ? -kNegInf : key[m] == 0 ? kNegInf : (float)__builtin_bit_cast(double, bits);
        if (cand(m) && fabsf(val[m]) < -kNegInf) {
            lo = fminf(lo, val[m]);
            hi = fmaxf(hi, val[m]);
        }
    }
    for (int x = tid; x < BINS; x += NT) hist[x] = 0;
    if (tid == 0) list_n = 0;
    lo = wave_least<false>(lo);
    hi = wave_least<true>(hi);
    if (lane == 0) {
        red[2 * w] = lo;
        red[2 * w + 1] = hi;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < WAVES; x++) {
        lo = fminf(lo, red[2 * x]);
        hi = fmaxf(hi, red[2 * x + 1]);
    }
    // taken: candidates whose key is above the border's, or equal with a page up to its
    bool done = need == 0;
    if (need == 0) {  // first and last fill the list
        if (tid == 0) {
            border_key = ~0ull;
            border_page = -1;
        }
    } else if (hi > lo && hi - lo < -kNegInf) {
        const float per = (float)BINS / (hi - lo);
        // (monotonic; infinities and NaN keys go to the ends)
        auto bin_of = [&](int m) { return val[m] >= hi ? BINS - 1 : val[m] <= lo ? 0 : (int)fminf((val[m] - lo) * per, BINS - 1.f); };
#pragma unroll
        for (int m = 0; m < KPT; m++)
            if (cand(m)) atomicAdd(&hist[bin_of(m)], 1u);
        __syncthreads();
        if (w == 0) find_bin(hist, BINS, need, lane, pick);
        __syncthreads();
        const int bin = pick[0], wanted = pick[1], held = pick[2];
        if (held <= 64) {  // (uniform)
#pragma unroll
            for (int m = 0; m < KPT; m++)
                if (cand(m) && bin_of(m) == bin) {
                    const uint32_t at = atomicAdd(&list_n, 1u);
                    list_key[at] = key[m];
                    list_page[at] = m * NT + tid;
                }
            __syncthreads();
            if (w == 0) {  // lane l's rank among them: the `wanted`-th is the border
                const uint64_t mine = lane < held ? list_key[lane] : 0;
                const int page = lane < held ? list_page[lane] : INT32_MAX;
                int rank = 0;
                for (int x = 0; x < held; x++) {
                    const uint64_t k = list_key[x];
                    rank += k > mine || (k == mine && list_page[x] < page);
                }
                if (lane < held && rank == wanted - 1) {
                    border_key = mine;
                    border_page = page;
                }
            }
            done = true;
        }
    }
    if (!done) {
        // radix: the key from the highest bit that differs, then the page downwards
        uint64_t all = ~0ull, any = 0;
#pragma unroll
        for (int m = 0; m < KPT; m++)
            if (cand(m)) {
                all &= key[m];
                any |= key[m];
            }
        for (int d = 32; d; d >>= 1) {
            all &= __shfl_xor(all, d, 64);
            any |= __shfl_xor(any, d, 64);
        }
        __syncthreads();
        if (lane == 0) {
            list_key[2 * w] = all;
            list_key[2 * w + 1] = any;
        }
        __syncthreads();
        all = ~0ull, any = 0;
#pragma unroll
        for (int x = 0; x < WAVES; x++) {
            all &= list_key[2 * x];
            any |= list_key[2 * x + 1];
        }
        const uint64_t differ = all ^ any;
        int shift = differ ? 64 - __builtin_clzll(differ) : 0;
        uint64_t top = shift < 64 ? any >> shift : 0;  // the border's bits so far
        int page_shift = 14, page_top = 0;             // (pages < 2^14; inverted: the lowest is the largest)
        bool whole = false;
        auto tail = [&](int m) { return 16383 - (m * NT + tid); };
        while (!whole && (shift > 0 || page_shift > 0)) {
            const bool by_key = shift > 0;
            const int bits = by_key ? min(8, shift) : 7;
            __syncthreads();
            for (int x = tid; x < 256; x += NT) hist[x] = 0;
            __syncthreads();
#pragma unroll
            for (int m = 0; m < KPT; m++) {
                const bool in = cand(m) && (by_key ? (shift == 64 || key[m] >> shift == top)
                                                   : key[m] == top && tail(m) >> page_shift == page_top);
                const uint32_t digit = by_key ? (uint32_t)(key[m] >> (shift - bits)) : (uint32_t)tail(m) >> (page_shift - bits);
                if (in) atomicAdd(&hist[digit & ((1u << bits) - 1)], 1u);
            }
            __syncthreads();
            if (w == 0) find_bin(hist, 256, need, lane, pick);
            __syncthreads();
            need = pick[1];
            whole = pick[2] == need;  // everything below this digit is taken
            if (by_key) {
                top = (shift == 64 ? 0 : top << bits) | (uint64_t)pick[0];
                shift -= bits;
            } else {
                page_top = page_top << bits | pick[0];
                page_shift -= bits;
            }
        }
        if (tid == 0) {
            border_key = shift < 64 ? top << shift : 0;
            border_page = 16383 - (page_top << page_shift);
        }
    }
    __syncthreads();
    const uint64_t bk = border_key;
    const int bp = border_page;
    auto taken = [&](int m) {
        const int x = m * NT + tid;
        if (x < first || (x >= end && x < pages)) return true;
        return cand(m) && (key[m] > bk || (key[m] == bk && x <= bp));
    };
    // places: a ballot per 64 pages, their counts scanned in page order
    uint64_t bal[KPT];
#pragma unroll
    for (int m = 0; m < KPT; m++) {
        bal[m] = __ballot(taken(m));
        if (lane == 0) counts[m * WAVES + w] = (uint32_t)__popcll(bal[m]);
    }
    __syncthreads();
    if (w == 0) {
        int carry = 0;
        for (int x0 = 0; x0 < KPT * WAVES; x0 += 64) {
            const int c = x0 + lane < KPT * WAVES ? (int)counts[x0 + lane] : 0;
            const int incl = wave_scan_i32(c);
            if (x0 + lane < KPT * WAVES) counts[x0 + lane] = (uint32_t)(carry + incl - c);
            carry += __builtin_amdgcn_readlane(incl, 63);
        }
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < KPT; m++) {
        const uint32_t at = counts[m * WAVES + w] + (uint32_t)__popcll(bal[m] & ((1ull << lane) - 1));
        if (taken(m) && at < (uint32_t)p.n_select) out[at] = m * NT + tid;
    }
}

template <int D>
hipError_t launch_score_d(const PageSelectParams& p, int dt, hipStream_t st, KernelTimer* t) {
    const int64_t items = (int64_t)((p.max_pages + score_pages<D>() - 1) / score_pages<D>()) * p.st.Hk * p.B;
    const dim3 grid((unsigned)std::min<int64_t>(items, 1024));
    if (dt == DT_F16) return launch_k(t, "page_score", page_score_kernel<D, DT_F16>, grid, dim3(256), st, p);
    return launch_k(t, "page_score", page_score_kernel<D, DT_BF16>, grid, dim3(256), st, p);
}

}  // namespace

hipError_t launch_page_score(const PageSelectParams& p, int D, int dt, hipStream_t st, KernelTimer* t) {
    if (D == 256) return launch_score_d<256>(p, dt, st, t);
    if (D == 128) return launch_score_d<128>(p, dt, st, t);
    return launch_score_d<64>(p, dt, st, t);
}

hipError_t launch_page_select(const PageSelectParams& p, hipStream_t st, KernelTimer* t) {
    const dim3 grid(p.st.Hk, p.q_len, p.B);
    if (p.max_pages <= 1024) return launch_k(t, "page_select", page_select_kernel<4, 4>, grid, dim3(256), st, p);
    if (p.max_pages <= 4096) return launch_k(t, "page_select", page_select_kernel<16, 4>, grid, dim3(1024), st, p);
    return launch_k(t, "page_select", page_select_kernel<16, 16>, grid, dim3(1024), st, p);
}

}  // namespace mugen_attn
