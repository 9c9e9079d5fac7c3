// paged_decode.h -- split-K GQA attention over the paged K/V cache, the kernel
// behind paged_decode16.hip (16-bit pages) and paged_decode8.hip (E4M3 pages).
//
// Semantics: softmax(q.K^T * scale) V with fp32 accumulation, kv head = h /
// (H / Hk), for 1..n new tokens per sequence, causal among them, over the pages
// of the sequence or over a page list per query (LIST).
//
// Design (HBM-bound: each K and V byte is read once):
//  * one workgroup = (context split, kv head, sequence, row block); its rows
//    are (token, head of the group) pairs, 16 to a wave.  WR waves side by side
//    take WR * 16 rows of the same tiles (a verify step's tokens share one read of
//    K and V from HBM, the others hit L1), WT of them the 32-token tiles t, t + WT,
//    ... of the split; each loads the next tile while computing the current one.
//    (One wave with up to 4 row blocks needs over 600 registers at head_dim 128
//    and spilled: 5 tokens of 28 / 4 heads over 4 x 31k tokens took 160 us.)
//    A page holds whole
//    tiles, so a tile's address is one page id away: the ids (and the 8-bit
//    scales) of 64 pages sit in one register across the lanes, read with
//    v_readlane, the next 64 loaded ahead;
//  * S^T[32 tokens x 16 rows] = K.Q^T and O^T[D x 16 rows] += V^T.P^T on MFMA
//    16x16x32.  K rows are the A operand straight from memory, in the token order
//    that leaves each lane 8 consecutive tokens of its row (A row m of block nb
//    is token 8*(m/4) + 4*nb + m%4) and in the dim order that makes a lane's
//    8-bit loads 16 bytes wide (k-step 2j+h, lane group g: dims 64j + 16g + 8h
//    .. +7); q is loaded in the same order;
//  * 8-bit V pages are stored [dim][32 tokens], so V^T is an A operand straight
//    from memory too: no LDS in the main loop.  Codes are expanded in registers
//    (v_cvt_scalef32_pk), V's scale in that conversion, K's with the softmax scale;
//  * 16-bit V rows (16-bit pages, and the ring behind the last whole 8-bit page)
//    go through a per-wave LDS buffer and ds_read_b64_tr_b16;
//  * online softmax in the exp2 domain with a lazy max (a row is re-based only
//    when a weight would exceed 2^8); P is fp16, or bf16 hi + lo;
//  * a V row that a query does not see is zeroed before its product, not only
//    weighted 0: 0 * inf is NaN.  Tiles that reach past the first query's last token
//    are checked for values that are not finite; where one is met, each token's
//    rows get their own product with the later rows zeroed;
//  Bound: HBM for a batch (64 sequences of 512..8191 tokens, 32 / 8 heads, 8-bit: 570 MB
//  read, no byte twice, in 111 us, 5.1 TB/s of a copy's 5.2; MFMA busy a tenth of the
//  time); 5 tokens of 4 x 31k 129 MB of codes in 31 us, 4.1 TB/s,
//  beside the softmax of 48 rows (MFMA busy 15%); one sequence of 4096 latency, 5.6 us for 8.4 MB: the launch, four
//  dependent reads and the merge of the waves;
//  * the WT waves of a row block merge (m, l, o) through LDS.  A range in one split
//    stores its result; otherwise fp32 partials go to the workspace and the combine
//    merges them.  (Merging in the workgroup that counts itself last instead saves
//    the launch, 3.7 us of host time, but the written-through partials, the count and
//    the merge follow one another at the end of the longest chain: 5 drafted tokens over
//    4 x 31k 50 -> 63 us, one sequence of 4096 8.8 -> 11.4, and the workspace would have
//    to be cleared once.)
#pragma once
#include "paged.h"

namespace mugen_attn {
namespace paged {

// 16-byte chunk c of staged V row r sits at chunk c ^ swz(r): the transpose
// reads of lane groups g, g+1 (rows 8g + r', r' < 4, chunks 2d, 2d + 1) then
// hit distinct banks (rows of 128 B at D = 64, 256 B or more above)
template <int D>
__device__ constexpr int swz(int r) {
    if constexpr (D == 64) return (((r >> 1) & 1) * 2) ^ (((r >> 3) & 1) * 4) ^ ((r >> 4) & 1);
    else return ((r & 1) * 2) ^ (((r >> 1) & 1) * 4) ^ (((r >> 3) & 1) * 8) ^ ((r >> 4) & 1);
}

// any 16-bit element (inf, NaN) / E4M3 code (NaN) of w that is not finite
template <int DT>
__device__ __forceinline__ bool bad16(uint32_t w) {
    if constexpr (DT == DT_F16) return (((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u) != 0;
    else return (((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u) != 0;
}
__device__ __forceinline__ bool bad8(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; }

// tokens the new tokens' queries see: sequence length and count
struct Lens {
    int T, n;
};
// (loads without branches, so that they leave together: what is not given is read
// from the table, which always is there)
__device__ __forceinline__ Lens seq_lens_of(const PagedDecodeParams& p, int b) {
    const int T = *(p.seq_lens ? p.seq_lens + b : p.st.table), n = *(p.q_lens ? p.q_lens + b : p.st.table);
    return Lens{p.seq_lens ? clamp_len(T, p.st.max_T) : p.fixed_T, p.q_lens ? clamp_len(n, p.q_len) : p.q_len};
}

// list entries a query that sees `limit` tokens may use
__device__ __forceinline__ int list_len(const PagedDecodeParams& p, int limit) {
    return min(p.n_sel, (max(limit, 0) + (1 << p.st.p_shift) - 1) >> p.st.p_shift);
}

// tokens in sequence (LIST: query) j's key range
template <bool LIST>
__device__ __forceinline__ int range_of(const PagedDecodeParams& p, int j) {
    if constexpr (LIST) {
        const int b = div_f(j, p.q_len, p.r_q_len), i = j - b * p.q_len;
        const Lens s = seq_lens_of(p, b);
        return i < s.n ? list_len(p, s.T - s.n + i + 1) << p.st.p_shift : 0;
    } else {
        const Lens s = seq_lens_of(p, j);
        return s.n > 0 ? s.T : 0;
    }
}

// splits of a key range of `len` tokens, chunks of `units` 32-token tiles
__device__ __forceinline__ int splits_of(int len, int units, float r_units) {
    return ceil_div_f((len + 31) >> 5, units, r_units);
}

template <bool LIST>
__device__ __forceinline__ int plan(const PagedDecodeParams& p) {
    auto units = [&](int j) { return (range_of<LIST>(p, j) + 31) >> 5; };
    return plan_chunk_device<1>(
        p.B, p.st.Hk * p.nrb, p.budget, [](int) { return 2; }, p.num_splits, units,
        [&](int j, int c, float rc) { return max(1, ceil_div_f(units(j), c, rc)); });
}

template <int D, int DT, bool BITS8, int WR, bool LIST>
__global__ __launch_bounds__(64 * WR * paged_tiles(D, BITS8, WR))
    __attribute__((amdgpu_waves_per_eu(paged_waves_per_simd(D, BITS8)))) void paged_decode_kernel(PagedDecodeParams p) {
    constexpr int WT = paged_tiles(D, BITS8, WR), NW = WR * WT, STEP = 32 * WT;
    constexpr int KK = D / 32;          // MFMA k-steps of S
    constexpr int KJ = D / 64;          // 16-byte loads of an 8-bit K row per lane
    constexpr int DB = D / 16;          // 16-dim blocks of O^T
    constexpr int RB = 2 * D;           // bytes of a staged V row
    constexpr int VL = 32 * RB / 1024;  // 16-byte V loads per lane per 16-bit tile
    constexpr int RPL = 1024 / RB;      // V rows per load instruction
    constexpr int NP = p_terms<DT>();
    constexpr float kHeadroom = 8.f;
    constexpr int kNever = 0x3fffffff;  // a tile that no row sees
    constexpr int STAGE = NW * 32 * RB;
    constexpr int PARTS = 2 * KJ + DB / 2;                              // 16-byte parts of an 8-bit tile per lane
    constexpr int PASS = BITS8 && WR > 1 ? NW * PARTS * 1024 + NW * 16 : 0;  // (8-bit row blocks side by side)
    constexpr int OROW = D + 4;
    constexpr int MERGE = NW * 16 * OROW * 4 + 3 * NW * 16 * 4 + WR * 2 * 16 * 4;
    __shared__ __attribute__((aligned(16))) char lds[PASS > STAGE ? (PASS > MERGE ? PASS : MERGE) : (STAGE > MERGE ? STAGE : MERGE)];

    const int Hk = p.st.Hk, ps = p.st.p_shift, P = 1 << ps;
    // one sequence, planned by the host: the split's place is known without the length,
    // so its page ids are on their way meanwhile
    const bool early = !LIST && p.B == 1 && p.chunk;
    int early_id = -1;
    if (early) {
        const int page = (div_f((int)blockIdx.x, Hk * p.nrb, p.r_mult) * p.chunk >> ps) + (int)(threadIdx.x & 63);
        early_id = p.st.table[min(page, (p.st.max_T - 1) >> ps)];
    }
    const int chunk = p.chunk ? p.chunk : plan<LIST>(p);
    int j = -1, r = 0;
    const int mult = Hk * p.nrb;
    const float r_units = plan_rcp(chunk >> 5);
    auto items = [&](int x) { return max(1, splits_of(range_of<LIST>(p, x), chunk >> 5, r_units)) * mult; };
    if (!find_sequence(p.B, (int)blockIdx.x, items, j, r)) return;  // grid padding
    const int s = div_f(r, mult, p.r_mult), kr = r - s * mult, kvh = div_f(kr, p.nrb, p.r_nrb), rb = kr - kvh * p.nrb;
    if (p.num_splits > 1 && s >= p.num_splits) return;  // past the workspace's stride
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int b = LIST ? div_f(j, p.q_len, p.r_q_len) : j, i0 = LIST ? j - b * p.q_len : 0;
    const Lens len = seq_lens_of(p, b);
    const int T = len.T;
    const int range = range_of<LIST>(p, j);
    const int t_begin = s * chunk, t_end = min(t_begin + chunk, range);
    if (p.chunk == 0 && blockIdx.x == 0 && threadIdx.x == 0) *p.plan = chunk;  // for the merge
    const int n_act = min(p.num_splits, max(1, splits_of(range, chunk >> 5, r_units)));  // splits of this range
    const int G = p.G, wg_row = rb * WR * 16, n_rows = (LIST ? 1 : len.n) * G;
    if (wg_row >= n_rows) return;  // rows of tokens that are not there
    const int wr = w % WR, wt = w / WR, first_row = wg_row + 16 * wr;

    // the lane's row first_row + n: its query, and how many tokens that sees
    const int row = first_row + n;
    const bool live = row < n_rows;
    const int tok = LIST ? i0 : div_f(row, G, p.r_G);
    const int limit = live ? max(T - len.n + tok + 1, 0) : 0;
    u32x4_t qf[KK];
    {
        const uint16_t* qp = p.q + (((int64_t)b * p.q_len + tok) * p.H + kvh * G + (LIST ? row : row - tok * G)) * D;
#pragma unroll
        for (int kk = 0; kk < KK; kk++)
            qf[kk] = live ? load16(qp + 64 * (kk >> 1) + 16 * g + 8 * (kk & 1)) : u32x4_t{0, 0, 0, 0};
    }
    // the wave's first and last token; tiles below `low` are seen by all its rows
    const int tok_first = LIST ? i0 : div_f(first_row, G, p.r_G),
              tok_last = LIST ? i0 : div_f(min(first_row + 16, n_rows) - 1, G, p.r_G);
    const int low = first_row < n_rows ? max(T - len.n + tok_first + 1, 0) : 0;
    const int t_first = first_row < n_rows ? t_begin + 32 * wt : t_end;  // (a wave without rows has no tiles)

    f32x4_t o[DB];  // lane (g, n): O[row n][16d + 4g + i]
    float m_run = kNegInf, l_part = 0.f;
#pragma unroll
    for (int d = 0; d < DB; d++) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    // ---- page ids: lane l holds page first_page + l of the split, physical
    // (-1: not there), logical (LIST), and the two exponents
    const int first_page = t_begin >> ps, end_page = (t_end + P - 1) >> ps;
    const int32_t* table = p.st.table + b * p.st.table_stride;
    const int whole = T >> ps;  // 8-bit: pages before it are whole, page `whole` is in the ring
    const int my_limit = LIST ? max(T - len.n + i0 + 1, 0) : T;
    const int32_t* list = LIST ? p.sel + (((int64_t)b * p.q_len + i0) * Hk + kvh) * p.n_sel : nullptr;
    struct Ids {
        int phys, lp;
        uint32_t exps;
    };
    auto load_ids = [&](int page0) {
        Ids x{-1, -1, 0x0101};  // (exponents of a page that is not there: any that are finite)
        const int k = page0 + lane;
        if (k < end_page) {
            int lp = k;
            if constexpr (LIST) {
                lp = list[k];
                const int before = k > 0 ? list[k - 1] : -1;
                if (lp <= before || lp >= (my_limit + P - 1) >> ps) lp = -1;
            }
            if (lp >= 0) {
                if (!BITS8 || lp < whole)
                    x.phys = checked_page(early && page0 == first_page ? early_id : table[lp], p.st.n_pages);
                x.lp = lp;
            }
        }
        if constexpr (BITS8) {
            if (x.phys >= 0) {
                const int64_t e = (int64_t)x.phys * Hk + kvh;
                x.exps = (uint32_t)p.st.k_exp[e] | ((uint32_t)p.st.v_exp[e] << 8);
            }
        }
        return x;
    };
    Ids ids = load_ids(first_page), ids_next = ids;
    int ids_at = first_page;
    if (ids_at + 64 < end_page) ids_next = load_ids(ids_at + 64);

    // a tile's place: its page, where it starts in it, its first token
    struct Tile {
        int phys, off, t0;
        uint32_t exps;
    };
    auto find_tile = [&](int t) {  // t: wave-uniform, ascending over the calls
        const int k = t >> ps;
        while (k >= ids_at + 64) {
            ids = ids_next;
            ids_at += 64;
            if (ids_at + 64 < end_page) ids_next = load_ids(ids_at + 64);
        }
        Tile x;
        x.phys = __builtin_amdgcn_readlane(ids.phys, k - ids_at);
        x.off = t & (P - 1);
        const int lp = LIST ? __builtin_amdgcn_readlane(ids.lp, k - ids_at) : k;
        x.t0 = x.phys >= 0 ? (lp << ps) + x.off : kNever;
        x.exps = BITS8 ? (uint32_t)__builtin_amdgcn_readlane((int)ids.exps, k - ids_at) : 0u;
        return x;
    };

    // ---- softmax of one tile's scores (lane: 8 consecutive tokens of its
    // rows), P as the B operand.  The maximum is taken of the raw scores (scale > 0)
    // and the scale goes into the exponent's fma; only edge tiles are masked
    auto softmax_tile = [&](f32x4_t (&sacc)[2], int t0, auto edge, float scale, u32x4_t (&pf)[NP]) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = sacc[e >> 2][e & 3];
        if constexpr (decltype(edge)::value) {
            const int seen = limit - t0 - 8 * g;
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = e < seen ? x[e] : kNegInf;
        }
        float smax = x[0];
#pragma unroll
        for (int e = 1; e < 8; e++) smax = fmaxf(smax, x[e]);
        smax *= scale;
        if (__any(smax > m_run + kHeadroom)) {  // re-base the rows (wave-uniform branch)
            const float m_new = fmaxf(m_run, max_x32(max_x16(smax)));
            if (m_new > m_run) {
                const float alpha = fast_exp2(m_run - m_new);  // 0 while m_run = -inf
                l_part *= alpha;
#pragma unroll
                for (int d = 0; d < DB; d++) o[d] *= alpha;
                m_run = m_new;
            }
        }
        const float nm = m_run == kNegInf ? 0.f : -m_run;
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            x[e] = fast_exp2(fmaf(x[e], scale, nm));
            sum += x[e];
        }
        l_part += sum;
        split_p<DT, NP>(x, pf);
    };
    // O^T += V^T.P^T, V^T blocks from vt(d)
    auto product = [&](auto vt, u32x4_t (&pf)[NP]) {
#pragma unroll
        for (int d = 0; d < DB; d++) {
            const u32x4_t a = vt(d);
#pragma unroll
            for (int t = 0; t < NP; t++) o[d] = mfma16x16x32<DT>(a, pf[t], o[d]);
        }
    };
    // the same for the rows of token i alone (a lane holds one row of O; the
    // others' weights are no zeros that would keep a NaN out)
    auto product_of = [&](int i, auto vt, u32x4_t (&pf)[NP]) {
#pragma unroll
        for (int d = 0; d < DB; d++) {
            const u32x4_t a = vt(d);
            f32x4_t x = o[d];
#pragma unroll
            for (int t = 0; t < NP; t++) x = mfma16x16x32<DT>(a, pf[t], x);
            if (tok == i) o[d] = x;
        }
    };

    // ---- a tile of 16-bit rows: K [32][D] and V [32][D], rows `stride` apart
    const int kr0 = 8 * (n >> 2) + (n & 3);  // + 4nb
    auto load16_tile = [&](const uint16_t* kb, const uint16_t* vb, int stride, int last, u32x4_t (&kq)[2][KK],
                           u32x4_t (&vq)[VL]) {
#pragma unroll
        for (int nb = 0; nb < 2; nb++) {
            const int row = min(kr0 + 4 * nb, last) * stride;
#pragma unroll
            for (int kk = 0; kk < KK; kk++) kq[nb][kk] = load16(kb + row + 64 * (kk >> 1) + 16 * g + 8 * (kk & 1));
        }
#pragma unroll
        for (int x = 0; x < VL; x++)
            vq[x] = load16(vb + min(x * RPL + lane / (RB / 16), last) * stride + 8 * (lane % (RB / 16)));
    };
    char* stage = &lds[w * 32 * RB];
    // (opaque in the open page's loop, where these offsets had better be formed again than
    // held in registers over the main loop: 64 sequences of 512..8191 tokens 125.9 -> 114.8 us)
    int st_lane = lane;
    auto st_off = [&](int x) {
        const int row = x * RPL + st_lane / (RB / 16), c = st_lane % (RB / 16);
        return row * RB + ((c ^ swz<D>(row)) * 16);
    };
    auto t_off = [&](int d) {
        const int sn = st_lane & 15, tr = 8 * (st_lane >> 4) + (sn >> 2);
        return tr * RB + (((2 * d + ((sn & 3) >> 1)) ^ swz<D>(tr)) * 16) + 8 * (sn & 1);
    };
    auto wave_sync = [] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    auto staged = [&](int d) {
        const u32x2_t lo = lds_read_tr16(reinterpret_cast<const uint16_t*>(stage + t_off(d)));
        const u32x2_t hi = lds_read_tr16(reinterpret_cast<const uint16_t*>(stage + t_off(d) + 4 * RB));
        return u32x4_t{lo[0], lo[1], hi[0], hi[1]};
    };
    // V rows from `seen` on zeroed
    auto stage_rows = [&](u32x4_t (&vq)[VL], int seen) {
#pragma unroll
        for (int x = 0; x < VL; x++) {
            const bool in = x * RPL + lane / (RB / 16) < seen;
            *reinterpret_cast<u32x4_t*>(stage + st_off(x)) = in ? vq[x] : u32x4_t{0, 0, 0, 0};
        }
    };
    auto compute16 = [&](u32x4_t (&kq)[2][KK], u32x4_t (&vq)[VL], int t0, auto edge) {
        constexpr bool EDGE = decltype(edge)::value;
        if constexpr (!EDGE) {
#pragma unroll
            for (int x = 0; x < VL; x++) *reinterpret_cast<u32x4_t*>(stage + st_off(x)) = vq[x];
        }
        f32x4_t sacc[2];
#pragma unroll
        for (int nb = 0; nb < 2; nb++) {
            f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < KK; kk++) acc = mfma16x16x32<DT>(kq[nb][kk], qf[kk], acc);
            sacc[nb] = acc;
        }
        u32x4_t pf[NP];
        softmax_tile(sacc, t0, edge, p.scale_log2, pf);
        if constexpr (EDGE) {
            bool bad = false;
#pragma unroll
            for (int x = 0; x < VL; x++)
#pragma unroll
                for (int e = 0; e < 4; e++) bad |= bad16<DT>(vq[x][e]);
            if (tok_first != tok_last && __any(bad)) {
                for (int i = tok_first; i <= tok_last; i++) {
                    stage_rows(vq, T - len.n + i + 1 - t0);
                    wave_sync();
                    product_of(i, staged, pf);
                    wave_sync();
                }
                return;
            }
            stage_rows(vq, T - len.n + tok_last + 1 - t0);
        }
        wave_sync();
        product(staged, pf);
        wave_sync();
    };

    // ---- The tiles: first those that every row sees whole, the next one loading
    // meanwhile (tiles of a page that is not there are passed over), then the last
    // few, which some row sees in part: the range ascends, so they come last.
    if constexpr (!BITS8) {
        u32x4_t kf[2][KK], kn[2][KK], vf[VL], vn[VL];
        auto load = [&](const Tile& x, u32x4_t (&kq)[2][KK], u32x4_t (&vq)[VL]) {
            const int64_t at = ((((int64_t)max(x.phys, 0) * Hk + kvh) << ps) + x.off) * D;
            // tokens past the sequence are not read: the last one instead
            load16_tile(reinterpret_cast<const uint16_t*>(p.st.k) + at, reinterpret_cast<const uint16_t*>(p.st.v) + at, D,
                        min(31, max(T - 1 - x.t0, 0)), kq, vq);
        };
        int t = t_first;
        Tile at{-1, 0, kNever, 0}, at_next = at;
        if (t < t_end) {
            at = find_tile(t);
            load(at, kf, vf);
        }
        for (; t < t_end; t += STEP) {
            if (at.phys >= 0 && at.t0 + 32 > low) break;
            const bool more = t + STEP < t_end;
            if (more) {
                at_next = find_tile(t + STEP);
                load(at_next, kn, vn);
            }
            if (at.phys >= 0) compute16(kf, vf, at.t0, std::false_type{});
            if (more) {
                at = at_next;
#pragma unroll
                for (int nb = 0; nb < 2; nb++)
#pragma unroll
                    for (int kk = 0; kk < KK; kk++) kf[nb][kk] = kn[nb][kk];
#pragma unroll
                for (int x = 0; x < VL; x++) vf[x] = vn[x];
            }
        }
        for (; t < t_end; t += STEP) {
            if (at.phys >= 0) compute16(kf, vf, at.t0, std::true_type{});
            if (t + STEP < t_end) {
                at = find_tile(t + STEP);
                load(at, kf, vf);
            }
        }
    } else {
        struct Raw {
            u32x4_t k[2][KJ];
            u32x2_t v[DB];
        };
        auto load = [&](const Tile& at, Raw& x) {
            const int64_t base = ((((int64_t)max(at.phys, 0) * Hk + kvh) << ps) + at.off) * D;
            const uint8_t* kb = p.st.k + base;
            const uint8_t* vb = p.st.v + base;
#pragma unroll
            for (int nb = 0; nb < 2; nb++)
#pragma unroll
                for (int c = 0; c < KJ; c++) x.k[nb][c] = load16(kb + (kr0 + 4 * nb) * D + 64 * c + 16 * g);
#pragma unroll
            for (int d = 0; d < DB; d++) x.v[d] = load8(vb + (16 * d + n) * 32 + 8 * g);
        };
        // V codes of tokens from `seen` on zeroed (the lane's tokens 8g .. 8g+7)
        auto keep = [&](u32x2_t v, int seen) {
            const int k = min(max(seen - 8 * g, 0), 8);
            const uint64_t mask = k >= 8 ? ~0ull : (1ull << (8 * k)) - 1;
            return u32x2_t{v[0] & (uint32_t)mask, v[1] & (uint32_t)(mask >> 32)};
        };
        auto compute8 = [&](Raw& x, const Tile& at, auto edge) {
            const float ks = exp_scale(at.exps & 0xffu) * p.scale_log2, vs = exp_scale((at.exps >> 8) & 0xffu);
            f32x4_t sacc[2];
#pragma unroll
            for (int nb = 0; nb < 2; nb++) {
                u32x4_t kf[KK];
#pragma unroll
                for (int c = 0; c < KJ; c++) {
                    kf[2 * c] = cvt8_fp8<DT>(x.k[nb][c][0], x.k[nb][c][1], 1.0f);
                    kf[2 * c + 1] = cvt8_fp8<DT>(x.k[nb][c][2], x.k[nb][c][3], 1.0f);
                }
                f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < KK; kk++) acc = mfma16x16x32<DT>(kf[kk], qf[kk], acc);
                sacc[nb] = acc;
            }
            u32x4_t pf[NP];
            softmax_tile(sacc, at.t0, edge, ks, pf);
            if constexpr (decltype(edge)::value) {
                bool bad = false;
#pragma unroll
                for (int d = 0; d < DB; d++) bad |= bad8(x.v[d][0]) | bad8(x.v[d][1]);
                if (__any(bad)) {
                    for (int i = tok_first; i <= tok_last; i++) {
                        const int seen = T - len.n + i + 1 - at.t0;
                        product_of(i, [&](int d) {
                            const u32x2_t v = keep(x.v[d], seen);
                            return cvt8_fp8<DT>(v[0], v[1], vs);
                        }, pf);
                    }
                    return;
                }
            }
            product([&](int d) { return cvt8_fp8<DT>(x.v[d][0], x.v[d][1], vs); }, pf);
        };
        // tiles in whole pages; the open page's, in the ring (dense: from token
        // whole * P on; LIST: the last valid entry, here a page that is not there) after them
        const int end8 = LIST ? t_end : min(t_end, whole << ps);
        if constexpr (WR > 1) {
            // Row blocks side by side would each load every tile, and have only WT of
            // them under way in a CU.  Instead every wave loads a tile of its own, a
            // step's NW tiles are passed through LDS as they are (a lane's part is the
            // same in every wave), and each wave takes WR of them, the next step's
            // tiles loading meanwhile (5 drafted tokens, 28 / 4 heads, over 4 x 31k tokens
            // 37.3 -> 33.0 us)
            u32x4_t* pass = reinterpret_cast<u32x4_t*>(&lds[0]);  // [NW][PARTS][64]
            int4* place = reinterpret_cast<int4*>(&lds[NW * PARTS * 1024]);  // [NW]
            // (tiles that the workgroup's first token sees whole; the last few after them)
            const int seen = min(end8, max(T - len.n + div_f(wg_row, G, p.r_G) + 1, 0));
            const int full = t_begin + max(seen - t_begin, 0) / 32 * 32;
            Raw raw;
            Tile at{-1, 0, kNever, 0x0101};
            auto fetch = [&](int t) {
                at.phys = -1;
                if (t < full) {
                    at = find_tile(t);
                    load(at, raw);
                }
            };
            fetch(t_begin + 32 * w);
            for (int t = t_begin; t < full; t += 32 * NW) {
#pragma unroll
                for (int x = 0; x < 2 * KJ; x++) pass[(w * PARTS + x) * 64 + lane] = raw.k[x / KJ][x % KJ];
#pragma unroll
                for (int x = 0; x < DB / 2; x++)
                    pass[(w * PARTS + 2 * KJ + x) * 64 + lane] =
                        u32x4_t{raw.v[2 * x][0], raw.v[2 * x][1], raw.v[2 * x + 1][0], raw.v[2 * x + 1][1]};
                if (lane == 0) place[w] = int4{at.phys, at.t0, (int)at.exps, 0};
                __syncthreads();
                fetch(t + 32 * (NW + w));
                for (int y = 0; y < WR; y++) {
                    const int slot = wt * WR + y;
                    const int4 pl = place[slot];
                    const Tile here{__builtin_amdgcn_readfirstlane(pl.x), 0, __builtin_amdgcn_readfirstlane(pl.y),
                                    (uint32_t)__builtin_amdgcn_readfirstlane(pl.z)};
                    if (here.phys < 0 || first_row >= n_rows) continue;
                    Raw x;
#pragma unroll
                    for (int i = 0; i < 2 * KJ; i++) x.k[i / KJ][i % KJ] = pass[(slot * PARTS + i) * 64 + lane];
#pragma unroll
                    for (int i = 0; i < DB / 2; i++) {
                        const u32x4_t v = pass[(slot * PARTS + 2 * KJ + i) * 64 + lane];
                        x.v[2 * i] = u32x2_t{v[0], v[1]};
                        x.v[2 * i + 1] = u32x2_t{v[2], v[3]};
                    }
                    compute8(x, here, std::false_type{});
                }
                __syncthreads();
            }
            if (first_row < n_rows) {
                for (int t = full + 32 * wt; t < end8; t += STEP) {
                    at = find_tile(t);
                    load(at, raw);
                    if (at.phys >= 0) compute8(raw, at, std::true_type{});
                }
            }
        } else {
        int t = t_first;
        Raw cur, nxt;
        Tile at{-1, 0, kNever, 0x0101}, at_next = at;
        if (t < end8) {
            at = find_tile(t);
            load(at, cur);
        }
        for (; t < end8; t += STEP) {
            if (at.phys >= 0 && at.t0 + 32 > low) break;
            const bool more = t + STEP < end8;
            if (more) {
                at_next = find_tile(t + STEP);
                load(at_next, nxt);
            }
            if (at.phys >= 0) compute8(cur, at, std::false_type{});
            if (more) {
                cur = nxt;
                at = at_next;
            }
        }
        for (; t < end8; t += STEP) {
            if (at.phys >= 0) compute8(cur, at, std::true_type{});
            if (t + STEP < end8) {
                at = find_tile(t + STEP);
                load(at, cur);
            }
        }
        }
        // ---- the open page
        int open = LIST ? -1 : whole;  // its place in the range, in pages
        if constexpr (LIST) {
            // the lists ascend, so the open page can only be the last entry that counts
            for (int k = first_page + lane; k < end_page; k += 64) {
                const int lp = list[k], before = k > 0 ? list[k - 1] : -1;
                if (lp == whole && lp > before && lp < (my_limit + P - 1) >> ps) open = k;
            }
            open = -wave_min_i32(-open);
        }
        open = __builtin_amdgcn_readfirstlane(open);
        if (open >= first_page && open < end_page) {
            // this wave's tiles of the page inside the split
            const int lo = max(open << ps, t_begin), hi = min((open + 1) << ps, t_end);
            int tt = t_first;
            if (tt < lo) tt += (lo - tt + STEP - 1) / STEP * STEP;
            for (; tt < hi; tt += STEP) {
                const int t0 = (whole << ps) + (tt & (P - 1));  // its first token
                if (t0 >= T) break;
                asm volatile("" : "+v"(st_lane));
                const int64_t ring_at = b * p.st.tail_stride + ((int64_t)(t0 & (p.st.ring - 1)) * Hk + kvh) * D;
                u32x4_t kq[2][KK], vq[VL];
                load16_tile(p.st.tail_k + ring_at, p.st.tail_v + ring_at, Hk * D, min(31, T - 1 - t0), kq, vq);
                compute16(kq, vq, t0, std::true_type{});
            }
        }
    }

    // ---- merge the WT waves' (m, l, O) of each row through LDS
    float* o_lds = reinterpret_cast<float*>(&lds[0]);  // [NW][16][OROW]
    float* m_lds = o_lds + NW * 16 * OROW;             // [NW][16]
    float* l_lds = m_lds + NW * 16;
    float* f_lds = l_lds + NW * 16;                    // [NW][16]: the waves' factors
    float* ml_out = f_lds + NW * 16;                   // [WR][16][2]: the row's (M, L)
    const float l = sum_x32(sum_x16(l_part));
    __syncthreads();
#pragma unroll
    for (int d = 0; d < DB; d++) *reinterpret_cast<f32x4_t*>(&o_lds[(w * 16 + n) * OROW + 16 * d + 4 * g]) = o[d];
    if (g == 0) {
        // (a NaN sum behind a maximum that no number set still counts)
        m_lds[w * 16 + n] = l != l && m_run == kNegInf ? 0.f : m_run;
        l_lds[w * 16 + n] = l;
    }
    __syncthreads();
    if (threadIdx.x < 16 * WR) {
        const int h = threadIdx.x;  // row of the workgroup: wave x * WR + h / 16, its row h % 16
        auto at = [&](int x) { return (x * WR + (h >> 4)) * 16 + (h & 15); };
        float M = kNegInf;
#pragma unroll
        for (int x = 0; x < WT; x++) M = fmaxf(M, m_lds[at(x)]);
        float f[WT], L = 0.f;
#pragma unroll
        for (int x = 0; x < WT; x++) {
            const float mw = m_lds[at(x)];
            f[x] = mw == kNegInf ? 0.f : fast_exp2(mw - M);
            L += f[x] * l_lds[at(x)];
        }
        const float c = n_act == 1 ? (L > 0.f ? 1.f / L : L == L ? 0.f : L) : 1.f;
#pragma unroll
        for (int x = 0; x < WT; x++) f_lds[at(x)] = f[x] * c;
        ml_out[2 * h] = M;
        ml_out[2 * h + 1] = L;
    }
    __syncthreads();
    const int rows_here = min(WR * 16, n_rows - wg_row);
    // row r of the workgroup in q and out
    auto out_row = [&](int r2) {
        const int i = LIST ? i0 : div_f(wg_row + r2, G, p.r_G);
        return ((int64_t)b * p.q_len + i) * p.H + kvh * G + (LIST ? r2 : wg_row + r2 - i * G);
    };
    auto store4 = [&](int64_t orow, int d, f32x4_t v) {
        if (p.out_dt == DT_F32) {
            *reinterpret_cast<f32x4_t*>(static_cast<float*>(p.out) + orow * D + d) = v;
        } else {
            const u32x2_t x = p.out_dt == DT_F16 ? u32x2_t{pack2<DT_F16>(v[0], v[1]), pack2<DT_F16>(v[2], v[3])}
                                                 : u32x2_t{pack2<DT_BF16>(v[0], v[1]), pack2<DT_BF16>(v[2], v[3])};
            *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(p.out) + orow * D + d) = x;
        }
    };
    for (int idx = threadIdx.x; idx < rows_here * (D / 4); idx += 64 * NW) {
        const int h = idx / (D / 4), d = 4 * (idx % (D / 4));
        f32x4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < WT; x++) {
            const int at = (x * WR + (h >> 4)) * 16 + (h & 15);
            const float f = f_lds[at];
            const f32x4_t v = *reinterpret_cast<const f32x4_t*>(&o_lds[at * OROW + d]);
            O += f * (f != 0.f ? v : f32x4_t{0.f, 0.f, 0.f, 0.f});
        }
        const int64_t orow = out_row(h);
        if (n_act == 1) {
            store4(orow, d, O);
        } else {
            const int64_t slot = orow * p.num_splits + s;
            *reinterpret_cast<f32x4_t*>(p.ws_o + slot * D + d) = O;
            if (d == 0) *reinterpret_cast<float2*>(p.ws_ml + slot * 2) = float2{ml_out[2 * h], ml_out[2 * h + 1]};
        }
    }
}

template <int D, int DT, bool BITS8>
hipError_t launch_rows(const PagedDecodeParams& p, int nwg, int wr, hipStream_t st, KernelTimer* t) {
    auto go = [&](auto r, auto list) {
        constexpr int WR = decltype(r)::value;
        return launch_k(t, "gqa_decode_paged", paged_decode_kernel<D, DT, BITS8, WR, decltype(list)::value>, dim3(nwg),
                        dim3(64 * WR * paged_tiles(D, BITS8, WR)), st, p);
    };
    if (p.sel) return go(std::integral_constant<int, 1>{}, std::true_type{});
    if (wr == 1) return go(std::integral_constant<int, 1>{}, std::false_type{});
    if (wr == 2) return go(std::integral_constant<int, 2>{}, std::false_type{});
    if constexpr (D < 256) {  // (3 does not divide a CU's 4 waves there)
        if (wr == 3) return go(std::integral_constant<int, 3>{}, std::false_type{});
    }
    return go(std::integral_constant<int, 4>{}, std::false_type{});
}

template <bool BITS8>
hipError_t launch_decode(const PagedDecodeParams& p, int nwg, int D, int dt, int wr, hipStream_t st, KernelTimer* t) {
    auto by_dt = [&](auto d) {
        constexpr int DD = decltype(d)::value;
        return dt == DT_F16 ? launch_rows<DD, DT_F16, BITS8>(p, nwg, wr, st, t)
                            : launch_rows<DD, DT_BF16, BITS8>(p, nwg, wr, st, t);
    };
    if (D == 256) return by_dt(std::integral_constant<int, 256>{});
    if (D == 128) return by_dt(std::integral_constant<int, 128>{});
    return by_dt(std::integral_constant<int, 64>{});
}

}  // namespace paged
}  // namespace mugen_attn
