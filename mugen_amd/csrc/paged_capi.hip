// paged_capi.hip -- extern "C" entry points of the paged K/V cache (see
// include/mugen_attn_paged.h): validation, split plans, workspace carving.
// Nothing here allocates device memory or synchronises the host.
#include <math.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "capi_common.h"
#include "paged.h"

namespace mugen_attn {
namespace {

bool is16(int dt) { return dt == DT_F16 || dt == DT_BF16; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

constexpr int kMaxTokens = 1 << 27;  // split plans count 32-token units in 23 bits

int store_validate(const mugen_attn_kv_pages& s, const char* who, bool tensors = true) {
    if (s.n_seq <= 0 || s.n_pages <= 0 || s.n_kv_heads <= 0 || s.max_seq_len <= 0)
        return fail(MUGEN_ATTN_E_INVALID, "%s: n_seq, n_pages, n_kv_heads and max_seq_len must be > 0", who);
    if (s.head_dim != 64 && s.head_dim != 128 && s.head_dim != 256)
        return fail(MUGEN_ATTN_E_UNSUPPORTED, "%s: head_dim %d (supported: 64, 128, 256)", who, s.head_dim);
    if (s.page_tokens != 32 && s.page_tokens != 64 && s.page_tokens != 128)
        return fail(MUGEN_ATTN_E_UNSUPPORTED, "%s: page_tokens %d (supported: 32, 64, 128)", who, s.page_tokens);
    if (s.page_bits != 16 && s.page_bits != 8)
        return fail(MUGEN_ATTN_E_UNSUPPORTED, "%s: page_bits %d (supported: 16, 8)", who, s.page_bits);
    if (!is16(s.dtype)) return fail(MUGEN_ATTN_E_UNSUPPORTED, "%s: dtype must be F16 or BF16", who);
    if (s.max_seq_len > kMaxTokens || s.n_kv_heads > 1024 || s.n_seq > 65535)
        return fail(MUGEN_ATTN_E_UNSUPPORTED, "%s: max_seq_len > 2^27, n_kv_heads > 1024 or n_seq > 65535", who);
    if (!s.page_table) return fail(MUGEN_ATTN_E_INVALID, "%s: null page_table", who);
    if (s.table_stride < ceil_div(s.max_seq_len, s.page_tokens))
        return fail(MUGEN_ATTN_E_INVALID, "%s: table_stride %lld < max_seq_len / page_tokens", who, (long long)s.table_stride);
    if (!aligned16(s.k_range)) return fail(MUGEN_ATTN_E_INVALID, "%s: k_range must be 16-byte aligned", who);
    if (!tensors) return MUGEN_ATTN_OK;
    if (!s.k_pages || !s.v_pages) return fail(MUGEN_ATTN_E_INVALID, "%s: null page pointer", who);
    if (!aligned16(s.k_pages) || !aligned16(s.v_pages))
        return fail(MUGEN_ATTN_E_INVALID, "%s: pages must be 16-byte aligned", who);
    if (s.page_bits == 16) return MUGEN_ATTN_OK;
    if (!s.k_exp || !s.v_exp || !s.tail_k || !s.tail_v)
        return fail(MUGEN_ATTN_E_INVALID, "%s: 8-bit pages need k_exp, v_exp, tail_k and tail_v", who);
    if (!aligned16(s.tail_k) || !aligned16(s.tail_v) || s.tail_seq_stride % 8)
        return fail(MUGEN_ATTN_E_INVALID, "%s: tails must be 16-byte aligned, tail_seq_stride a multiple of 8", who);
    if (s.ring <= s.page_tokens || (s.ring & (s.ring - 1)))
        return fail(MUGEN_ATTN_E_INVALID, "%s: ring %d must be a power of two > page_tokens", who, s.ring);
    if (s.n_seq > 1 && s.tail_seq_stride < (int64_t)s.ring * s.n_kv_heads * s.head_dim)
        return fail(MUGEN_ATTN_E_INVALID, "%s: tail_seq_stride smaller than one ring", who);
    return MUGEN_ATTN_OK;
}

int heads_validate(const mugen_attn_kv_pages& s, int n_heads, const char* who) {
    if (n_heads <= 0 || n_heads % s.n_kv_heads)
        return fail(MUGEN_ATTN_E_INVALID, "%s: n_heads %d not a multiple of n_kv_heads %d", who, n_heads, s.n_kv_heads);
    if (n_heads / s.n_kv_heads > 16)
        return fail(MUGEN_ATTN_E_UNSUPPORTED, "%s: n_heads / n_kv_heads = %d > 16", who, n_heads / s.n_kv_heads);
    return MUGEN_ATTN_OK;
}

PagedStore store_params(const mugen_attn_kv_pages& s) {
    PagedStore p{};
    p.k = static_cast<uint8_t*>(s.k_pages);
    p.v = static_cast<uint8_t*>(s.v_pages);
    p.k_exp = static_cast<uint8_t*>(s.k_exp);
    p.v_exp = static_cast<uint8_t*>(s.v_exp);
    p.tail_k = static_cast<uint16_t*>(s.tail_k);
    p.tail_v = static_cast<uint16_t*>(s.tail_v);
    p.k_range = static_cast<uint16_t*>(s.k_range);
    p.table = s.page_table;
    p.table_stride = s.table_stride;
    p.tail_stride = s.tail_seq_stride;
    p.n_pages = s.n_pages;
    p.p_shift = s.page_tokens == 32 ? 5 : s.page_tokens == 64 ? 6 : 7;
    p.ring = s.page_bits == 8 ? s.ring : 0;
    p.Hk = s.n_kv_heads;
    p.max_T = s.max_seq_len;
    return p;
}

float* align256(void* p) { return reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(p) + 255) & ~uintptr_t(255)); }

// ------------------------------------------------------------------ append

// turns per position of rope_dim / 2 pairs: theta^(-2i/rope_dim) / (2 pi), for
// factor > 1 with the YaRN correction of yarn_rope_freq (transformer.cpp:41-70;
// beta_fast 32, beta_slow 1), in 64 bits (the powers by repeated products in extended
// precision: a pow() a pair took 3 us of a call)
RopeTurns<128> rope_turns(const mugen_attn_rope_params& r, int rope_dim) {
    RopeTurns<128> out{};
    const double two_pi = 6.283185307179586476925286766559;
    const double theta = r.theta, dim = rope_dim;
    const bool yarn = r.factor > 1.f;
    const double span = yarn ? 2.0 * std::log(theta) : 1.0;
    const double low = yarn ? std::max(0.0, std::floor(dim * std::log(r.original_ctx / (32.0 * two_pi)) / span)) : 0.0;
    const double high = yarn ? std::min(dim / 2 - 1, std::ceil(dim * std::log(r.original_ctx / two_pi) / span)) : 0.0;
    const long double step = powl((long double)theta, -2.0L / rope_dim);
    long double power = 1.0L;
    for (int i = 0; i < rope_dim / 2; i++, power *= step) {
        double f = (double)power;
        if (yarn) {
            const double ramp = i < low ? 0.0 : i > high ? 1.0 : (i - low) / std::max(0.001, high - low);
            f = f * (1.0 - std::min(1.0, ramp)) + f / r.factor * std::min(1.0, ramp);
        }
        out.f[i] = f / two_pi;
    }
    return out;
}

}  // namespace
}  // namespace mugen_attn

using namespace mugen_attn;

extern "C" int mugen_attn_kv_paged_append(const mugen_attn_kv_paged_append_args* a, void* stream) {
    const char* who = "kv_paged_append";
    if (!a) return fail(MUGEN_ATTN_E_INVALID, "%s: null args", who);
    const mugen_attn_kv_pages& s = a->store;
    if (int rc = store_validate(s, who)) return rc;
    if (a->n_new < 0) return fail(MUGEN_ATTN_E_INVALID, "%s: n_new < 0", who);
    if (a->rope_dim < 0 || a->rope_dim > s.head_dim || a->rope_dim % 16)
        return fail(MUGEN_ATTN_E_UNSUPPORTED, "%s: rope_dim %d (supported: multiples of 16 up to head_dim)", who, a->rope_dim);
    const mugen_attn_rope_params& r = a->rope;
    if (a->rope_dim && (!std::isfinite(r.theta) || !(r.theta > 0.f) || !std::isfinite(r.factor) ||
                        (r.factor > 1.f && (r.original_ctx <= 0 || !(r.theta > 1.f)))))
        return fail(MUGEN_ATTN_E_INVALID, "%s: bad rope parameters", who);
    if (a->n_new == 0 && !a->seq_lens_out) return MUGEN_ATTN_OK;
    if (!a->seq_lens) return fail(MUGEN_ATTN_E_INVALID, "%s: null seq_lens", who);
    if (a->seq_lens_out == a->seq_lens) return fail(MUGEN_ATTN_E_INVALID, "%s: seq_lens_out aliases seq_lens", who);
    if (a->n_new == 0)
        return fail(MUGEN_ATTN_E_INVALID, "%s: n_new must be > 0 where seq_lens_out is asked for", who);
    if (!a->k_new || !a->v_new) return fail(MUGEN_ATTN_E_INVALID, "%s: null k_new / v_new", who);
    const int64_t row = (int64_t)s.n_kv_heads * s.head_dim;
    if (!aligned16(a->k_new) || !aligned16(a->v_new) || a->k_stride % 8 || a->v_stride % 8)
        return fail(MUGEN_ATTN_E_INVALID, "%s: k_new / v_new must be 16-byte aligned, strides multiples of 8", who);
    if (a->k_stride < row || a->v_stride < row)
        return fail(MUGEN_ATTN_E_INVALID, "%s: k_stride / v_stride smaller than n_kv_heads * head_dim", who);
    if (a->q) {
        if (int rc = heads_validate(s, a->n_heads, who)) return rc;
        if (!a->q_out) return fail(MUGEN_ATTN_E_INVALID, "%s: q without q_out", who);
        if (!aligned16(a->q) || !aligned16(a->q_out) || a->q_stride % 8 || a->q_stride < (int64_t)a->n_heads * s.head_dim)
            return fail(MUGEN_ATTN_E_INVALID, "%s: q / q_out must be 16-byte aligned, q_stride a multiple of 8 and a row", who);
    }
    PagedAppendParams p{};
    p.st = store_params(s);
    p.k_new = static_cast<const uint16_t*>(a->k_new);
    p.v_new = static_cast<const uint16_t*>(a->v_new);
    p.q = static_cast<const uint16_t*>(a->q);
    p.q_out = static_cast<uint16_t*>(a->q_out);
    p.seq_lens = a->seq_lens;
    p.new_lens = a->new_lens;
    p.seq_lens_out = a->seq_lens_out;
    p.k_stride = a->k_stride;
    p.v_stride = a->v_stride;
    p.q_stride = a->q_stride;
    p.n_seq = s.n_seq;
    p.n_new = a->n_new;
    p.H = a->q ? a->n_heads : 0;
    p.rope_dim = a->rope_dim;
    RopeTurns<128> turns{};
    if (a->rope_dim) turns = rope_turns(r, a->rope_dim);
    const int heads = p.H + 2 * s.n_kv_heads;
    const int64_t tokens = (int64_t)s.n_seq * a->n_new;
    // one head a thread where the tokens are few (latency), up to 8 where their
    // threads fill the card anyway (the sines are shared)
    p.heads_per_thread = (int)std::min<int64_t>(8, std::max<int64_t>(1, tokens * heads * (s.head_dim / 16) / (64 * 1024)));
    p.pages = (a->n_new + s.page_tokens - 1) / s.page_tokens;  // that n_new tokens can fill
    const int64_t jobs = (int64_t)s.n_seq * p.pages * s.n_kv_heads * 2;
    // (a launch takes less than 2^32 threads: 2^24 workgroups, at most half of them rows)
    if (tokens * heads * (s.head_dim / 16) > INT32_MAX || jobs >= 1 << 23)
        return fail(MUGEN_ATTN_E_UNSUPPORTED, "%s: too many tokens in one call", who);
    return hip_status(launch_paged_append(p, turns, s.head_dim, s.dtype, s.page_bits == 8, static_cast<hipStream_t>(stream),
                                          active_timer()),
                      "kv_paged_append launch");
}

// ------------------------------------------------------------------ decode

namespace {

struct DecodePlan {
    int chunk = 0;   // 0: planned by the kernels
    int splits = 1;  // the partials' stride
    int wr = 1, nrb = 1;  // row blocks of a workgroup, workgroups of a (range, kv head)
    int budget = 0;
    int64_t nwg = 0;
    size_t bytes = 0;
};

// the key ranges the plan cuts: sequences, or (with page lists) queries, whose lists
// are as long as the last query's at most
int ranges_of(const mugen_attn_gqa_decode_paged_args* a) { return a->store.n_seq * (a->pages ? a->q_len : 1); }
int64_t range_of_len(const mugen_attn_gqa_decode_paged_args* a, int T) {
    if (!a->pages) return T;
    const int P = a->store.page_tokens;
    return (int64_t)std::min((uint32_t)a->n_select, ((uint32_t)T + P - 1) / P) * P;
}
int64_t longest_range(const mugen_attn_gqa_decode_paged_args* a) { return range_of_len(a, a->store.max_seq_len); }
// of sequence b
int64_t range_len(const mugen_attn_gqa_decode_paged_args* a, int b) {
    if (!a->seq_lens_host) return longest_range(a);
    return range_of_len(a, std::min(std::max(a->seq_lens_host[b], 0), a->store.max_seq_len));
}

// most splits of a range: 32, more only in pieces of 512 tokens and up
constexpr int kCap = 32, kCapLong = kPagedMaxSplits, kCapTokens = 512, kChunkMin = 64;
int split_cap(int64_t len) { return (int)std::max<int64_t>(kCap, std::min<int64_t>(kCapLong, len / kCapTokens)); }
int split_bound(int64_t len) { return (int)std::min<int64_t>(split_cap(len), ceil_div(len, kChunkMin)); }

// work items of a chunk size; counting ends past `most` (the search asks no more)
int64_t decode_items(const mugen_attn_gqa_decode_paged_args* a, int chunk, int64_t mult, int64_t most = INT64_MAX) {
    if (!a->seq_lens_host) return ranges_of(a) * std::max<int64_t>(1, ceil_div(longest_range(a), chunk)) * mult;
    const int64_t each = mult * (a->pages ? a->q_len : 1);
    int64_t n = 0;
    for (int b = 0; b < a->store.n_seq && n * each <= most; b++)
        n += std::max(1u, ((uint32_t)range_len(a, b) + chunk - 1) / (uint32_t)chunk);
    return n * each;
}

// Whether one split a range (no partials, no merge launch) is as fast as the cut into
// `chunk`: a model in us of what was measured, kernel and merge, in captured steps.  A
// workgroup takes 128 tokens in `step` us while it waits for nothing but its own
// chain, all together stream at most 4.8 TB/s, and the two overlap by half; ragged
// ranges end in a tail of the longest; the merge costs its launch and the partials'
// way.  (28 / 4 heads d128, 8-bit, us
// unsplit / cut: 1 x 512 7.7 / 7.4, 1 x 1024 10.4 / 7.5, 32 x 512 9.3 / 12.8, 32 x 1024 13.0
// / 15.7; 16-bit 1 x 256 7.1 / 7.4, 8 x 384 9.1 / 8.1, 32 x 512 11.9 / 13.8; 32 / 8 d64 8-bit
// 32 x 1024 10.9 / 14.0; 16 / 8 d256 8-bit 8 x 256 8.7 / 9.0, 8 x 768 15.9 / 13.6)
bool one_split_pays(const mugen_attn_gqa_decode_paged_args* a, int wr, int nrb, int64_t len, int chunk) {
    const mugen_attn_kv_pages& s = a->store;
    const bool b8 = s.page_bits == 8;
    const double step = (s.head_dim == 64 ? (b8 ? 0.5 : 0.7) : s.head_dim == 128 ? (b8 ? 0.65 : 1.7) : b8 ? 1.45 : 3.6) *
                        (wr == 1 || wr == 3 ? 1.0 : wr == 2 ? 1.6 : 3.0);
    double sum = 0;
    for (int b = 0; b < s.n_seq; b++) sum += (double)range_len(a, b);
    const double tail = 0.25 * ((double)len - sum / s.n_seq) / 128 * step;
    if (a->pages) sum *= a->q_len;
    constexpr double kRate = 4.8e6;  // bytes a us
    const double stream = sum * s.n_kv_heads * nrb * 2 * s.head_dim * s.page_bits / 8 / kRate;
    const double splits = (double)ceil_div(len, chunk);
    const double partials = (double)s.n_seq * a->q_len * a->n_heads * splits * s.head_dim * 8 / kRate;
    auto time = [&](int64_t tokens) {
        const double chain = (double)tokens / 128 * step;
        return std::max(chain, stream) + 0.5 * std::min(chain, stream);
    };
    return time(len) + tail <= time(chunk) + 2.6 + partials;
}

size_t decode_bytes(const mugen_attn_gqa_decode_paged_args* a, int splits) {
    if (splits <= 1) return 0;
    const size_t rows = (size_t)a->store.n_seq * a->q_len * a->n_heads;
    return 512 + rows * splits * ((size_t)a->store.head_dim * 4 + 8);  // (512: alignment, and the planned chunk)
}

DecodePlan decode_plan(const mugen_attn_gqa_decode_paged_args* a, bool for_size) {
    DecodePlan r;
    const mugen_attn_kv_pages& s = a->store;
    const int G = a->n_heads / s.n_kv_heads, rows = (a->pages ? 1 : a->q_len) * G;
    r.wr = rows <= 16 ? 1 : rows <= 32 ? 2 : rows <= 48 && s.head_dim < 256 ? 3 : 4;
    r.nrb = (int)ceil_div(rows, 16 * r.wr);
    const int64_t mult = (int64_t)s.n_kv_heads * r.nrb;
    r.budget = 256 * paged_groups_per_cu(s.head_dim, s.page_bits == 8, r.wr);
    const int64_t longest = longest_range(a);
    int64_t len = 1;
    for (int b = 0, B = a->seq_lens_host ? s.n_seq : 1; b < B; b++) len = std::max(len, range_len(a, b));
    if (a->num_splits > 0) {
        r.chunk = (int)ceil_div(ceil_div(longest, a->num_splits), 32) * 32;
    } else {
        const int64_t most = ceil_div(len, 32) * 32;
        int64_t lo = std::max<int64_t>(ceil_div(ceil_div(len, split_cap(len)), 32) * 32, kChunkMin), hi = std::max(most, lo);
        if (decode_items(a, (int)hi, mult, r.budget) > r.budget) lo = hi;  // a range each already fills the round
        while (lo < hi) {                                        // items fall as the chunk grows
            const int64_t mid = (lo + hi) / 2 / 32 * 32;
            if (mid < lo) break;
            if (decode_items(a, (int)mid, mult, r.budget) <= r.budget) hi = mid;
            else lo = mid + 32;
        }
        r.chunk = (int)hi;
        if ((a->seq_lens_host || a->pages) && r.chunk < most && one_split_pays(a, r.wr, r.nrb, len, r.chunk)) r.chunk = (int)most;
        // large ragged batches: even items of 1024 tokens over several rounds, where
        // the longest range would run on alone
        else if (a->seq_lens_host && r.chunk > 1024) {
            int64_t sum = 0;
            for (int b = 0; b < s.n_seq; b++) sum += range_len(a, b) * (a->pages ? a->q_len : 1);
            if ((double)std::min<int64_t>(r.chunk, len) * r.budget > 1.35 * (double)(sum * mult))
                r.chunk = (int)std::max<int64_t>(1024, ceil_div(ceil_div(len, kCap), 32) * 32);
        }
    }
    r.splits = (int)std::max<int64_t>(1, ceil_div(a->seq_lens_host ? len : longest, r.chunk));
    if (!a->seq_lens_host && a->num_splits <= 0) {
        const int bound = split_bound(longest);
        // without host lengths the kernels cut the lengths they find, where the
        // ranges alone leave at least half the round free
        if (!a->pages && bound > 1 && ranges_of(a) * mult * 2 <= r.budget) {
            r.chunk = 0;
            r.splits = bound;
        } else if (for_size) {
            r.splits = std::max(r.splits, bound);  // covers every later host copy
        }
    }
    r.nwg = r.chunk ? decode_items(a, r.chunk, mult)
                    : std::min<int64_t>(r.budget, ranges_of(a) * mult * r.splits);
    r.bytes = decode_bytes(a, r.splits);
    return r;
}

int decode_validate(const mugen_attn_gqa_decode_paged_args* a) {
    const char* who = "gqa_decode_paged";
    if (!a) return fail(MUGEN_ATTN_E_INVALID, "%s: null args", who);
    if (int rc = store_validate(a->store, who)) return rc;
    if (int rc = heads_validate(a->store, a->n_heads, who)) return rc;
    if (!a->q || !a->out || !a->seq_lens) return fail(MUGEN_ATTN_E_INVALID, "%s: null tensor pointer", who);
    if (!aligned16(a->q) || !aligned16(a->out))
        return fail(MUGEN_ATTN_E_INVALID, "%s: q and out must be 16-byte aligned", who);
    if (a->q_len <= 0 || a->q_len > MUGEN_ATTN_PAGED_MAX_Q)
        return fail(MUGEN_ATTN_E_UNSUPPORTED, "%s: q_len %d (supported: 1 .. %d)", who, a->q_len, MUGEN_ATTN_PAGED_MAX_Q);
    if (a->num_splits < 0 || a->num_splits > kPagedMaxSplits)
        return fail(MUGEN_ATTN_E_INVALID, "%s: num_splits %d (0 .. %d)", who, a->num_splits, kPagedMaxSplits);
    if (a->out_dtype != DT_F32 && !is16(a->out_dtype)) return fail(MUGEN_ATTN_E_UNSUPPORTED, "%s: bad out_dtype", who);
    if (a->pages && a->n_select <= 0) return fail(MUGEN_ATTN_E_INVALID, "%s: page lists need n_select > 0", who);
    if (!(a->scale == a->scale) || std::isinf(a->scale)) return fail(MUGEN_ATTN_E_INVALID, "%s: scale is not finite", who);
    return MUGEN_ATTN_OK;
}

}  // namespace

extern "C" size_t mugen_attn_gqa_decode_paged_workspace_size(const mugen_attn_gqa_decode_paged_args* a) {
    return decode_validate(a) == MUGEN_ATTN_OK ? decode_plan(a, true).bytes : 0;
}

namespace {
// fixed_T >= 0: one sequence of fixed_T tokens (a prompt chunk's few rows)
int decode_run(const mugen_attn_gqa_decode_paged_args* a, const DecodePlan& plan, int fixed_T, void* ws, hipStream_t st) {
    const mugen_attn_kv_pages& s = a->store;
    PagedDecodeParams p{};
    p.st = store_params(s);
    p.q = static_cast<const uint16_t*>(a->q);
    p.out = a->out;
    p.seq_lens = fixed_T >= 0 ? nullptr : a->seq_lens;
    p.q_lens = a->q_lens;
    p.sel = a->pages;
    p.n_sel = a->n_select;
    p.fixed_T = fixed_T;
    p.B = ranges_of(a);
    p.q_len = a->q_len;
    p.H = a->n_heads;
    p.G = a->n_heads / s.n_kv_heads;
    p.nrb = plan.nrb;
    p.out_dt = a->out_dtype;
    p.chunk = plan.chunk;
    p.num_splits = plan.splits;
    p.budget = plan.budget;
    p.r_mult = 1.f / (float)(s.n_kv_heads * plan.nrb);
    p.r_nrb = 1.f / (float)plan.nrb;
    p.r_G = 1.f / (float)p.G;
    p.r_q_len = 1.f / (float)a->q_len;
    p.scale_log2 = (a->scale > 0.f ? a->scale : 1.f / sqrtf((float)s.head_dim)) * kLog2e;
    if (plan.splits > 1) {
        const size_t slots = (size_t)s.n_seq * a->q_len * a->n_heads * plan.splits;
        p.ws_o = align256(ws);
        p.ws_ml = p.ws_o + slots * s.head_dim;
        p.plan = reinterpret_cast<int*>(p.ws_ml + slots * 2);
    }
    // (work items are counted in 23 bits, their launch, of up to 768 threads each, takes
    // less than 2^32; the merge's grid in 16 bits)
    if (plan.nwg >= 1 << 22 || (int64_t)s.n_seq * (s.head_dim / 64) > 65535)
        return fail(MUGEN_ATTN_E_UNSUPPORTED, "gqa_decode_paged: too many sequences or work items");
    hipError_t e = s.page_bits == 8
                       ? launch_paged_decode8(p, (int)plan.nwg, s.head_dim, s.dtype, plan.wr, st, active_timer())
                       : launch_paged_decode16(p, (int)plan.nwg, s.head_dim, s.dtype, plan.wr, st, active_timer());
    if (e == hipSuccess && plan.splits > 1) e = launch_paged_combine(p, s.head_dim, st, active_timer());
    return hip_status(e, "gqa_decode_paged launch");
}
}  // namespace

extern "C" int mugen_attn_gqa_decode_paged(const mugen_attn_gqa_decode_paged_args* a, void* ws, size_t ws_bytes,
                                           void* stream) {
    if (int rc = decode_validate(a)) return rc;
    const DecodePlan plan = decode_plan(a, false);
    if (plan.bytes && (!ws || ws_bytes < plan.bytes))
        return fail(MUGEN_ATTN_E_WORKSPACE, "gqa_decode_paged: workspace of %zu bytes required, %zu given", plan.bytes,
                    ws_bytes);
    return decode_run(a, plan, -1, ws, static_cast<hipStream_t>(stream));
}

// ------------------------------------------------------------------ selection

static int select_validate(const mugen_attn_page_select_args* a) {
    const char* who = "page_select";
    if (!a) return fail(MUGEN_ATTN_E_INVALID, "%s: null args", who);
    if (int rc = store_validate(a->store, who, false)) return rc;
    if (int rc = heads_validate(a->store, a->n_heads, who)) return rc;
    if (!a->store.k_range) return fail(MUGEN_ATTN_E_INVALID, "%s: the store has no k_range", who);
    if (!a->q || !a->pages || !a->seq_lens) return fail(MUGEN_ATTN_E_INVALID, "%s: null tensor pointer", who);
    if (a->q_len <= 0 || a->q_len > MUGEN_ATTN_PAGED_MAX_Q)
        return fail(MUGEN_ATTN_E_UNSUPPORTED, "%s: q_len %d (supported: 1 .. %d)", who, a->q_len, MUGEN_ATTN_PAGED_MAX_Q);
    if (a->n_first < 0 || a->n_last < 1 || a->n_select <= 0 || (int64_t)a->n_first + a->n_last > a->n_select)
        return fail(MUGEN_ATTN_E_INVALID, "%s: n_first >= 0, n_last >= 1 and n_first + n_last <= n_select are needed", who);
    if (ceil_div(a->store.max_seq_len, a->store.page_tokens) > 16384)
        return fail(MUGEN_ATTN_E_UNSUPPORTED, "%s: max_seq_len is more than 16384 pages", who);
    return MUGEN_ATTN_OK;
}

static int select_pages_of(const mugen_attn_page_select_args* a) {
    return (int)ceil_div(a->store.max_seq_len, a->store.page_tokens);
}

extern "C" size_t mugen_attn_page_select_workspace_size(const mugen_attn_page_select_args* a) {
    if (select_validate(a) != MUGEN_ATTN_OK || select_pages_of(a) <= a->n_select) return 0;
    return (size_t)a->store.n_seq * a->q_len * a->store.n_kv_heads * select_pages_of(a) * 8 + 256;
}

extern "C" int mugen_attn_page_select(const mugen_attn_page_select_args* a, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = select_validate(a)) return rc;
    const size_t need = mugen_attn_page_select_workspace_size(a);
    if (need && (!ws || ws_bytes < need))
        return fail(MUGEN_ATTN_E_WORKSPACE, "page_select: workspace of %zu bytes required, %zu given", need, ws_bytes);
    PageSelectParams p{};
    p.st = store_params(a->store);
    p.q = static_cast<const uint16_t*>(a->q);
    p.pages = a->pages;
    p.seq_lens = a->seq_lens;
    p.q_lens = a->q_lens;
    p.B = a->store.n_seq;
    p.q_len = a->q_len;
    p.H = a->n_heads;
    p.G = a->n_heads / a->store.n_kv_heads;
    p.n_select = a->n_select;
    p.n_first = a->n_first;
    p.n_last = a->n_last;
    p.max_pages = select_pages_of(a);
    hipStream_t st = static_cast<hipStream_t>(stream);
    hipError_t e = hipSuccess;
    if (need) {  // (else every page is taken, no score needed)
        p.keys = reinterpret_cast<uint64_t*>(align256(ws));
        e = launch_page_score(p, a->store.head_dim, a->store.dtype, st, active_timer());
    }
    if (e == hipSuccess) e = launch_page_select(p, st, active_timer());
    return hip_status(e, "page_select launch");
}

// ------------------------------------------------------------------ prefill

namespace {

int prefill_validate(const mugen_attn_gqa_prefill_paged_args* a) {
    const char* who = "gqa_prefill_paged";
    if (!a) return fail(MUGEN_ATTN_E_INVALID, "%s: null args", who);
    if (int rc = store_validate(a->store, who)) return rc;
    if (int rc = heads_validate(a->store, a->n_heads, who)) return rc;
    if (!a->q || !a->out) return fail(MUGEN_ATTN_E_INVALID, "%s: null tensor pointer", who);
    if (!aligned16(a->q) || !aligned16(a->out)) return fail(MUGEN_ATTN_E_INVALID, "%s: q / out must be 16-byte aligned", who);
    if (a->seq < 0 || a->seq >= a->store.n_seq) return fail(MUGEN_ATTN_E_INVALID, "%s: seq %d of %d", who, a->seq, a->store.n_seq);
    if (a->n_tokens < 0 || a->start_pos < 0 || (int64_t)a->start_pos + a->n_tokens > a->store.max_seq_len)
        return fail(MUGEN_ATTN_E_INVALID, "%s: start_pos + n_tokens outside [0, max_seq_len]", who);
    if (a->out_dtype != DT_F32 && !is16(a->out_dtype)) return fail(MUGEN_ATTN_E_UNSUPPORTED, "%s: bad out_dtype", who);
    if (!(a->scale == a->scale) || std::isinf(a->scale)) return fail(MUGEN_ATTN_E_INVALID, "%s: scale is not finite", who);
    if (((int64_t)a->start_pos + a->n_tokens) * a->store.n_kv_heads * a->store.head_dim * 2 > INT32_MAX)
        return fail(MUGEN_ATTN_E_UNSUPPORTED, "%s: K/V of the sequence larger than 2 GiB per tensor", who);
    return MUGEN_ATTN_OK;
}

// the gathered rows of one tensor, 256-byte steps
size_t gather_bytes(const mugen_attn_gqa_prefill_paged_args* a) {
    const size_t n = ((size_t)a->start_pos + a->n_tokens) * a->store.n_kv_heads * a->store.head_dim * 2;
    return (n + 255) / 256 * 256;
}

// the call over the gathered rows (k, v: any non-null pointers for its size)
mugen_attn_gqa_prefill_args gathered(const mugen_attn_gqa_prefill_paged_args* a, void* k, void* v) {
    mugen_attn_gqa_prefill_args g{};
    g.q = a->q;
    g.k = k;
    g.v = v;
    g.out = a->out;
    g.n_tokens = a->n_tokens;
    g.n_heads = a->n_heads;
    g.n_kv_heads = a->store.n_kv_heads;
    g.head_dim = a->store.head_dim;
    g.kv_len = a->start_pos + a->n_tokens;
    g.start_pos = a->start_pos;
    g.causal = 1;
    g.scale = a->scale;
    g.dtype = a->store.dtype;
    g.out_dtype = a->out_dtype;
    return g;
}

// Few tokens go through the decode kernel, which reads the pages as they are; more
// of them through the gathered rows, which cost their copy but feed the prompt
// kernels (us rows / gathered, 8-bit pages; 28 / 4 heads d128, 168 / 224 / 336 rows a kv
// head: after 1k 12.9 / 14.7, 14.0 / 15.0, 18.8 / 15.1, after 8k 22.8 / 22.4, 24.1 / 22.9,
// 29.5 / 33.4, after 32k 38 / 48, 45 / 49, 57 / 79; 32 / 8 d64, 256 rows: 12.8 / 11.8,
// 23.3 / 24.1, 44 / 58; 16 / 8 d256, 128 rows: 21.0 / 26.1, 36 / 61, 89 / 155)
constexpr int kRowsMost = 224, kRowsMostOther = 256;  // head_dim 128; 64 and 256
bool prefill_by_rows(const mugen_attn_gqa_prefill_paged_args* a) {
    return a->n_tokens <= MUGEN_ATTN_PAGED_MAX_Q &&
           a->n_tokens * (a->n_heads / a->store.n_kv_heads) <= (a->store.head_dim == 128 ? kRowsMost : kRowsMostOther);
}
mugen_attn_gqa_decode_paged_args as_decode(const mugen_attn_gqa_prefill_paged_args* a, int32_t* len) {
    mugen_attn_gqa_decode_paged_args d{};
    d.store = a->store;
    d.store.n_seq = 1;
    d.store.page_table += a->seq * a->store.table_stride;
    if (a->store.page_bits == 8) {
        d.store.tail_k = static_cast<uint16_t*>(a->store.tail_k) + a->seq * a->store.tail_seq_stride;
        d.store.tail_v = static_cast<uint16_t*>(a->store.tail_v) + a->seq * a->store.tail_seq_stride;
    }
    d.q = a->q;
    d.out = a->out;
    d.q_len = a->n_tokens;
    d.n_heads = a->n_heads;
    d.scale = a->scale;
    d.out_dtype = a->out_dtype;
    *len = a->start_pos + a->n_tokens;
    d.seq_lens_host = len;
    return d;
}

}  // namespace

extern "C" size_t mugen_attn_gqa_prefill_paged_workspace_size(const mugen_attn_gqa_prefill_paged_args* a) {
    if (prefill_validate(a) != MUGEN_ATTN_OK || a->n_tokens == 0) return 0;
    if (prefill_by_rows(a)) {
        int32_t len;
        const mugen_attn_gqa_decode_paged_args d = as_decode(a, &len);
        return decode_plan(&d, true).bytes;
    }
    const mugen_attn_gqa_prefill_args g = gathered(a, a->store.k_pages, a->store.v_pages);
    return 256 + 2 * gather_bytes(a) + prefill_split_workspace(&g);
}

extern "C" int mugen_attn_gqa_prefill_paged(const mugen_attn_gqa_prefill_paged_args* a, void* ws, size_t ws_bytes,
                                            void* stream) {
    if (int rc = prefill_validate(a)) return rc;
    if (a->n_tokens == 0) return MUGEN_ATTN_OK;
    const size_t need = mugen_attn_gqa_prefill_paged_workspace_size(a);
    if (need && (!ws || ws_bytes < need))
        return fail(MUGEN_ATTN_E_WORKSPACE, "gqa_prefill_paged: workspace of %zu bytes required, %zu given", need, ws_bytes);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (prefill_by_rows(a)) {
        int32_t len;
        const mugen_attn_gqa_decode_paged_args d = as_decode(a, &len);
        return decode_run(&d, decode_plan(&d, false), len, ws, st);
    }
    char* base = reinterpret_cast<char*>(align256(ws));
    PagedGatherParams p{};
    p.st = store_params(a->store);
    p.k_out = reinterpret_cast<uint16_t*>(base);
    p.v_out = reinterpret_cast<uint16_t*>(base + gather_bytes(a));
    p.seq = a->seq;
    p.T = a->start_pos + a->n_tokens;
    mugen_attn_gqa_prefill_args g = gathered(a, p.k_out, p.v_out);
    p.v16 = prefill_takes_v16(&g);
    if (int rc = hip_status(launch_paged_gather(p, a->store.head_dim, a->store.dtype, a->store.page_bits == 8, st, active_timer()),
                            "gqa_prefill_paged launch"))
        return rc;
    const size_t more = prefill_split_workspace(&g);
    if (more) {
        g.workspace = base + 2 * gather_bytes(a);
        g.workspace_bytes = more;
    }
    return prefill_run(&g, p.v16, stream, true);
}
