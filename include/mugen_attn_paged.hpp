// mugen_attn_paged.hpp -- C++ adapter and attention provider over the paged K/V
// cache (mugen_attn_paged.h), in the style of mugen_attn.hpp and
// mugen_attn_engine.hpp: Status returns, memory allocated once at create(), every
// per-step value in device memory so that a step's calls can be captured into a
// StepGraph and replayed.
//
// GqaAttentionPaged keeps a model's caches in pages that its sequences share: a
// sequence takes pages as it grows (reserve) and gives them back (release), so
// the memory follows the tokens held, not batch * max_seq_len as in
// GqaAttention.  A slot of the batch without pages is idle: a step's rows for it go
// nowhere, its outputs mean nothing and its length is 0 again when it is next reserved.
// Positions, lengths and the page table live on the device; a captured step replays
// for as long as the reserved pages last (steps_left(); past them a step's tokens are
// dropped, nothing else is written).
#pragma once

#include <algorithm>
#include <memory>
#include <string>
#include <vector>

#include "mugen_attn_engine.hpp"
#include "mugen_attn_paged.h"

namespace mugen_attn {

inline Status kv_paged_append(const mugen_attn_kv_paged_append_args& a, void* stream) {
    return check(mugen_attn_kv_paged_append(&a, stream));
}
inline size_t gqa_decode_paged_workspace_size(const mugen_attn_gqa_decode_paged_args& a) {
    return mugen_attn_gqa_decode_paged_workspace_size(&a);
}
inline Status gqa_decode_paged(const mugen_attn_gqa_decode_paged_args& a, void* ws, size_t ws_bytes, void* stream) {
    return check(mugen_attn_gqa_decode_paged(&a, ws, ws_bytes, stream));
}
inline size_t page_select_workspace_size(const mugen_attn_page_select_args& a) {
    return mugen_attn_page_select_workspace_size(&a);
}
inline Status page_select(const mugen_attn_page_select_args& a, void* ws, size_t ws_bytes, void* stream) {
    return check(mugen_attn_page_select(&a, ws, ws_bytes, stream));
}
inline size_t gqa_prefill_paged_workspace_size(const mugen_attn_gqa_prefill_paged_args& a) {
    return mugen_attn_gqa_prefill_paged_workspace_size(&a);
}
inline Status gqa_prefill_paged(const mugen_attn_gqa_prefill_paged_args& a, void* ws, size_t ws_bytes, void* stream) {
    return check(mugen_attn_gqa_prefill_paged(&a, ws, ws_bytes, stream));
}

struct GqaPagedShape {
    int n_layers = 0;
    int batch = 1;  // sequences
    int n_heads = 0;
    int n_kv_heads = 0;
    int head_dim = 0;     // 64, 128 or 256
    int max_seq_len = 0;  // of one sequence
    int n_pages = 0;      // per layer; 0: enough for every sequence at max_seq_len
    int page_tokens = 64;
    int page_bits = 8;    // 8: E4M3 pages with a scale per page and kv head; 16
    int max_new = 8;      // most tokens a decode_layer call adds per sequence (and take_back may undo)
    int max_prefill = 2048;  // most tokens of one prefill_layer call
    int kv_dtype = MUGEN_ATTN_F16;
    int out_dtype = MUGEN_ATTN_F16;
    float scale = 0.f;    // 0: 1/sqrt(head_dim)
    int rope_dim = 0;     // 0: queries and keys come rotated
    mugen_attn_rope_params rope{10000.f, 1.f, 0};
    int n_select = 0;     // > 0: decode reads the n_select pages that score highest, per query and kv head
    int n_first = 1, n_last = 2;
};

class GqaAttentionPaged {
public:
    static Status create(const GqaPagedShape& shape, std::unique_ptr<GqaAttentionPaged>* out) {
        GqaPagedShape s = shape;
        if (s.n_layers <= 0 || s.batch <= 0 || s.max_seq_len <= 0 || s.max_new <= 0 || s.page_tokens <= 0 ||
            s.max_prefill <= 0 || s.n_pages < 0 || s.n_heads <= 0 || s.n_kv_heads <= 0 || s.head_dim <= 0)
            return fail("GqaAttentionPaged: n_layers, batch, heads, max_seq_len, page_tokens, max_new and max_prefill must be > 0");
        if (s.max_new > MUGEN_ATTN_PAGED_MAX_Q) return fail("GqaAttentionPaged: max_new above MUGEN_ATTN_PAGED_MAX_Q");
        if (s.page_tokens != 32 && s.page_tokens != 64 && s.page_tokens != 128)
            return fail("GqaAttentionPaged: page_tokens must be 32, 64 or 128");
        const int per_seq = (s.max_seq_len + s.page_tokens - 1) / s.page_tokens;
        if (s.n_pages == 0) s.n_pages = s.batch * per_seq;
        std::unique_ptr<GqaAttentionPaged> a(new GqaAttentionPaged(s, per_seq));
        const size_t row = (size_t)s.n_kv_heads * s.head_dim, page = row * s.page_tokens;
        a->layers_.resize(s.n_layers);
        for (Layer& L : a->layers_) {
            const size_t pool = (size_t)s.n_pages * page * (s.page_bits == 8 ? 1 : 2);
            if (auto r = L.k.alloc(pool, "GqaAttentionPaged K pages"); !r) return r;
            if (auto r = L.v.alloc(pool, "GqaAttentionPaged V pages"); !r) return r;
            if (s.page_bits == 8) {
                const size_t tail = (size_t)s.batch * a->ring_ * row * 2, exps = (size_t)s.n_pages * s.n_kv_heads;
                if (auto r = L.k_exp.alloc(exps, "GqaAttentionPaged scales"); !r) return r;
                if (auto r = L.v_exp.alloc(exps, "GqaAttentionPaged scales"); !r) return r;
                if (auto r = L.tail_k.alloc(tail, "GqaAttentionPaged tail"); !r) return r;
                if (auto r = L.tail_v.alloc(tail, "GqaAttentionPaged tail"); !r) return r;
            }
            if (s.n_select > 0)
                if (auto r = L.range.alloc((size_t)s.n_pages * 2 * row * 2, "GqaAttentionPaged key ranges"); !r) return r;
        }
        if (auto r = a->table_.alloc(sizeof(int32_t) * s.batch * per_seq, "GqaAttentionPaged page table"); !r) return r;
        if (auto r = a->lens_.alloc(sizeof(int32_t) * 2 * s.batch, "GqaAttentionPaged lengths"); !r) return r;
        if (s.rope_dim > 0) {
            const size_t tokens = std::max<size_t>((size_t)s.batch * s.max_new, (size_t)s.max_prefill);
            if (auto r = a->q_.alloc(tokens * s.n_heads * s.head_dim * 2, "GqaAttentionPaged queries"); !r) return r;
        }
        // what the kernels do not take is refused here: calls without a token, and the
        // selection's size, check everything and launch nothing
        void* any = a->layers_[0].k.ptr;
        mugen_attn_kv_paged_append_args none = a->append_args(a->store(0), any, any, any, 0);
        none.seq_lens = a->before();
        if (auto r = kv_paged_append(none, nullptr); !r) return r;
        if (auto r = gqa_prefill_paged(a->prefill_args(0, 0, 0, 0, any, any), nullptr, 0, nullptr); !r) return r;
        if (s.n_select > 0 && page_select_workspace_size(a->select_args(0, 1, any)) == 0)
            return fail(std::string("GqaAttentionPaged: ") + mugen_attn_last_error());
        size_t ws = 0;
        for (int q_len = 1; q_len <= s.max_new; q_len++) {
            mugen_attn_gqa_decode_paged_args d = a->decode_args(0, q_len, any, any);
            ws = std::max(ws, gqa_decode_paged_workspace_size(d));
            if (s.n_select > 0) {
                d.pages = static_cast<const int32_t*>(any);  // (a placeholder: only the shape matters)
                ws = std::max({ws, gqa_decode_paged_workspace_size(d),
                               page_select_workspace_size(a->select_args(0, q_len, any))});
            }
        }
        for (int n = std::min(s.max_prefill, s.max_seq_len); n > 0; n--) {
            // a chunk needs most at the end of the cache; a short one, whose rows are one
            // sequence's verify rows, what covers every length of it
            ws = std::max(ws, gqa_prefill_paged_workspace_size(a->prefill_args(0, 0, n, s.max_seq_len - n, any, any)));
            if (n > MUGEN_ATTN_PAGED_MAX_Q) continue;
            mugen_attn_gqa_decode_paged_args d = a->decode_args(0, n, any, any);
            d.store.n_seq = 1;
            ws = std::max(ws, gqa_decode_paged_workspace_size(d));
        }
        if (auto r = a->ws_.alloc(ws, "GqaAttentionPaged workspace"); !r) return r;
        if (s.n_select > 0)
            if (auto r = a->pages_.alloc(sizeof(int32_t) * s.batch * s.max_new * s.n_kv_heads * s.n_select,
                                         "GqaAttentionPaged page lists");
                !r)
                return r;
        // no slot has a page yet (the zeroed table would name page 0)
        if (auto r = detail::hip_ok(hipMemcpy(a->table_.ptr, a->host_table_.data(), a->table_.bytes, hipMemcpyHostToDevice),
                                    "GqaAttentionPaged page table");
            !r)
            return r;
        for (int i = s.n_pages - 1; i >= 0; i--) a->free_.push_back(i);
        *out = std::move(a);
        return Status{};
    }

    // Pages for `tokens` tokens of sequence `seq` in all (outside a captured
    // step; waits for the copy of its table row).
    Status reserve(int seq, int tokens, hipStream_t st) {
        if (seq < 0 || seq >= s_.batch) return fail("GqaAttentionPaged::reserve: bad sequence");
        if (tokens < 0 || tokens > s_.max_seq_len) return fail("GqaAttentionPaged::reserve: past max_seq_len");
        const int need = (tokens + s_.page_tokens - 1) / s_.page_tokens;
        if (need <= held_[seq]) return Status{};
        if (need - held_[seq] > (int)free_.size()) return fail("GqaAttentionPaged::reserve: out of pages");
        if (held_[seq] == 0)  // (idle until now: steps in between moved its length)
            if (auto r = set_length(seq, 0, st); !r) return r;
        while (held_[seq] < need) {
            host_table_[(size_t)seq * per_seq_ + held_[seq]++] = free_.back();
            free_.pop_back();
        }
        return put_row(seq, st);
    }
    // Sequence `seq` ends: its length is 0, its table row names no page (a step
    // replayed later writes to none of them) and its pages are free.
    Status release(int seq, hipStream_t st) {
        if (seq < 0 || seq >= s_.batch) return fail("GqaAttentionPaged::release: bad sequence");
        const std::vector<int32_t> was(&host_table_[(size_t)seq * per_seq_], &host_table_[(size_t)seq * per_seq_] + held_[seq]);
        std::fill_n(&host_table_[(size_t)seq * per_seq_], per_seq_, -1);
        if (auto r = put_row(seq, st); !r) {
            std::copy(was.begin(), was.end(), &host_table_[(size_t)seq * per_seq_]);
            return r;
        }
        free_.insert(free_.end(), was.rbegin(), was.rend());
        held_[seq] = 0;
        return set_length(seq, 0, st);
    }
    // Sequence `seq` goes back to `tokens` tokens (drafts that were rejected).
    // Reads the lengths back first: replayed steps have moved them.
    Status take_back(int seq, int tokens, hipStream_t st) {
        if (seq < 0 || seq >= s_.batch) return fail("GqaAttentionPaged::take_back: bad sequence");
        if (auto r = sync_lengths(st); !r) return r;
        if (tokens < 0 || tokens > host_lens_[seq]) return fail("GqaAttentionPaged::take_back: not that long");
        const int open = tokens / s_.page_tokens * s_.page_tokens;
        if (s_.page_bits == 8 && tokens != open && open < low_[seq])
            return fail("GqaAttentionPaged::take_back: the ring no longer holds that page's rows");
        const int low = std::min(low_[seq], tokens);
        auto r = set_length(seq, tokens, st);
        low_[seq] = low;
        return r;
    }

    // One layer of a decode or verify step: q [batch][n_new][H][d], k_new / v_new
    // [batch][n_new][Hk*d], out like q.  Every sequence that is not idle needs its
    // pages reserved.
    Status decode_layer(int L, const void* q, const void* k_new, const void* v_new, void* out, hipStream_t st, int n_new = 1) {
        if (L < 0 || L >= s_.n_layers) return fail("GqaAttentionPaged::decode_layer: bad layer");
        if (n_new < 1 || n_new > s_.max_new) return fail("GqaAttentionPaged::decode_layer: n_new outside [1, max_new]");
        if (std::all_of(held_.begin(), held_.end(), [](int h) { return h == 0; }))
            return fail("GqaAttentionPaged::decode_layer: no sequence has pages (reserve)");
        for (int b = 0; b < s_.batch; b++)
            if (held_[b] > 0 && host_lens_[b] + n_new > room(b))
                return fail("GqaAttentionPaged::decode_layer: sequence " + std::to_string(b) + " has no page for the step (reserve)");
        mugen_attn_kv_paged_append_args ap = append_args(store(L), q, k_new, v_new, n_new);
        ap.seq_lens = before();
        ap.seq_lens_out = after();
        if (auto r = kv_paged_append(ap, st); !r) return r;
        const void* rq = s_.rope_dim > 0 ? q_.ptr : q;
        mugen_attn_gqa_decode_paged_args d = decode_args(L, n_new, rq, out);
        if (s_.n_select > 0) {
            if (auto r = page_select(select_args(L, n_new, rq), ws_.ptr, ws_.bytes, st); !r) return r;
            d.pages = static_cast<const int32_t*>(pages_.ptr);
        }
        return gqa_decode_paged(d, ws_.ptr, ws_.bytes, st);
    }

    // Prompt chunk of n_tokens for sequence `seq`, one layer: q [n_tokens][H][d],
    // k_new / v_new [n_tokens][Hk*d], out like q; attends over every token held.
    // Reads the host copy of the length, so it is not for captured steps;
    // advance_sequence(seq, n_tokens) after the last layer.
    Status prefill_layer(int L, int seq, const void* q, const void* k_new, const void* v_new, void* out, int n_tokens,
                         hipStream_t st) {
        if (L < 0 || L >= s_.n_layers) return fail("GqaAttentionPaged::prefill_layer: bad layer");
        if (seq < 0 || seq >= s_.batch) return fail("GqaAttentionPaged::prefill_layer: bad sequence");
        if (n_tokens < 1 || n_tokens > s_.max_prefill)
            return fail("GqaAttentionPaged::prefill_layer: n_tokens outside [1, max_prefill]");
        const int start = host_lens_[seq];
        if (held_[seq] == 0 || start + n_tokens > room(seq))
            return fail("GqaAttentionPaged::prefill_layer: no page for the prompt (reserve)");
        mugen_attn_kv_pages one = store(L);  // the sequence alone
        one.n_seq = 1;
        one.page_table += (int64_t)seq * one.table_stride;
        if (s_.page_bits == 8) {
            one.tail_k = static_cast<uint16_t*>(one.tail_k) + seq * one.tail_seq_stride;
            one.tail_v = static_cast<uint16_t*>(one.tail_v) + seq * one.tail_seq_stride;
        }
        mugen_attn_kv_paged_append_args ap = append_args(one, q, k_new, v_new, n_tokens);
        ap.seq_lens = before() + seq;
        if (auto r = kv_paged_append(ap, st); !r) return r;
        return gqa_prefill_paged(prefill_args(L, seq, n_tokens, start, s_.rope_dim > 0 ? q_.ptr : q, out), ws_.ptr, ws_.bytes, st);
    }

    // End of a step: every length += n (device side, capturable; the host
    // mirror follows).
    Status advance(hipStream_t st, int n = 1) {
        for (int b = 0; b < s_.batch; b++)
            if (held_[b] > 0 && host_lens_[b] + n > s_.max_seq_len)
                return fail("GqaAttentionPaged::advance: past max_seq_len");
        for (int b = 0; b < s_.batch; b++) grow(b, n);
        return seq_advance(before(), n, s_.batch, s_.max_seq_len, st);
    }
    Status advance_sequence(int seq, int n, hipStream_t st) {
        if (seq < 0 || seq >= s_.batch) return fail("GqaAttentionPaged::advance_sequence: bad sequence");
        if (host_lens_[seq] + n > s_.max_seq_len) return fail("GqaAttentionPaged::advance_sequence: past max_seq_len");
        grow(seq, n);
        return seq_advance(before() + seq, n, 1, s_.max_seq_len, st);
    }
    // Host mirror <- device lengths (after StepGraph replays); waits.
    Status sync_lengths(hipStream_t st) {
        if (auto r = detail::read_ints(lens_.ptr, host_lens_, s_.batch, st, "GqaAttentionPaged::sync_lengths"); !r) return r;
        for (int b = 0; b < s_.batch; b++) grow(b, 0);
        return Status{};
    }
    // Steps of n tokens that the reserved pages still hold for every sequence that
    // is not idle (from the host's lengths: sync_lengths() after replays).
    int steps_left(int n = 1) const {
        int m = s_.max_seq_len;
        for (int b = 0; b < s_.batch; b++)
            if (held_[b] > 0) m = std::min(m, (room(b) - host_lens_[b]) / std::max(n, 1));
        return m;
    }

    mugen_attn_kv_pages store(int L) const {
        const Layer& y = layers_[L];
        mugen_attn_kv_pages p{};
        p.k_pages = y.k.ptr;
        p.v_pages = y.v.ptr;
        p.k_exp = y.k_exp.ptr;
        p.v_exp = y.v_exp.ptr;
        p.tail_k = y.tail_k.ptr;
        p.tail_v = y.tail_v.ptr;
        p.k_range = y.range.ptr;
        p.page_table = static_cast<const int32_t*>(table_.ptr);
        p.table_stride = per_seq_;
        p.tail_seq_stride = (int64_t)ring_ * s_.n_kv_heads * s_.head_dim;
        p.n_seq = s_.batch;
        p.n_pages = s_.n_pages;
        p.page_tokens = s_.page_tokens;
        p.page_bits = s_.page_bits;
        p.ring = ring_;
        p.n_kv_heads = s_.n_kv_heads;
        p.head_dim = s_.head_dim;
        p.max_seq_len = s_.max_seq_len;
        p.dtype = s_.kv_dtype;
        return p;
    }
    int free_pages() const { return (int)free_.size(); }
    const std::vector<int32_t>& host_lengths() const { return host_lens_; }
    const GqaPagedShape& shape() const { return s_; }

private:
    struct Layer {
        detail::DeviceBuffer k, v, k_exp, v_exp, tail_k, tail_v, range;
    };
    GqaAttentionPaged(const GqaPagedShape& s, int per_seq)
        : s_(s), per_seq_(per_seq), host_table_((size_t)s.batch * per_seq, -1), held_(s.batch, 0), host_lens_(s.batch, 0),
          low_(s.batch, 0) {
        for (ring_ = 1; ring_ < s.page_tokens + s.max_new; ring_ *= 2) {}
    }
    int32_t* before() const { return static_cast<int32_t*>(lens_.ptr); }
    int32_t* after() const { return before() + s_.batch; }
    int room(int b) const { return std::min(s_.max_seq_len, held_[b] * s_.page_tokens); }
    void grow(int b, int n) {
        host_lens_[b] = held_[b] > 0 ? host_lens_[b] + n : 0;
        low_[b] = std::max(low_[b], host_lens_[b] - ring_);
    }
    Status put_row(int seq, hipStream_t st) {
        const size_t at = (size_t)seq * per_seq_;
        if (auto r = detail::hip_ok(hipMemcpyAsync(static_cast<int32_t*>(table_.ptr) + at, &host_table_[at],
                                                   sizeof(int32_t) * per_seq_, hipMemcpyHostToDevice, st),
                                    "GqaAttentionPaged page table");
            !r)
            return r;
        return detail::hip_ok(hipStreamSynchronize(st), "GqaAttentionPaged page table");
    }
    Status set_length(int seq, int32_t tokens, hipStream_t st) {
        host_lens_[seq] = tokens;
        low_[seq] = 0;
        if (auto r = detail::hip_ok(hipMemcpyAsync(before() + seq, &host_lens_[seq], sizeof(int32_t), hipMemcpyHostToDevice, st),
                                    "GqaAttentionPaged length");
            !r)
            return r;
        return detail::hip_ok(hipStreamSynchronize(st), "GqaAttentionPaged length");
    }
    mugen_attn_kv_paged_append_args append_args(const mugen_attn_kv_pages& at, const void* q, const void* k_new,
                                                const void* v_new, int n_new) const {
        mugen_attn_kv_paged_append_args a{};
        a.store = at;
        a.k_new = k_new;
        a.v_new = v_new;
        a.k_stride = a.v_stride = (int64_t)s_.n_kv_heads * s_.head_dim;
        a.n_new = n_new;
        a.rope_dim = s_.rope_dim;
        a.rope = s_.rope;
        if (s_.rope_dim > 0) {
            a.q = q;
            a.q_out = q_.ptr;
            a.q_stride = (int64_t)s_.n_heads * s_.head_dim;
            a.n_heads = s_.n_heads;
        }
        return a;
    }
    mugen_attn_gqa_decode_paged_args decode_args(int L, int q_len, const void* q, void* out) const {
        mugen_attn_gqa_decode_paged_args d{};
        d.store = store(L);
        d.q = q;
        d.out = out;
        d.seq_lens = after();
        d.n_select = s_.n_select;
        d.q_len = q_len;
        d.n_heads = s_.n_heads;
        d.scale = s_.scale;
        d.out_dtype = s_.out_dtype;
        return d;  // (planned on the device from its lengths: one call serves every step)
    }
    mugen_attn_page_select_args select_args(int L, int q_len, const void* q) const {
        mugen_attn_page_select_args a{};
        a.store = store(L);
        a.q = q;
        a.pages = static_cast<int32_t*>(pages_.ptr ? pages_.ptr : layers_[0].k.ptr);  // (for the size: any)
        a.seq_lens = after();
        a.q_len = q_len;
        a.n_heads = s_.n_heads;
        a.n_select = s_.n_select;
        a.n_first = s_.n_first;
        a.n_last = s_.n_last;
        return a;
    }
    mugen_attn_gqa_prefill_paged_args prefill_args(int L, int seq, int n, int start, const void* q, void* out) const {
        mugen_attn_gqa_prefill_paged_args a{};
        a.store = store(L);
        a.q = q;
        a.out = out;
        a.seq = seq;
        a.n_tokens = n;
        a.start_pos = start;
        a.n_heads = s_.n_heads;
        a.scale = s_.scale;
        a.out_dtype = s_.out_dtype;
        return a;
    }

    GqaPagedShape s_;
    int per_seq_;  // table entries of a sequence
    int ring_ = 1;
    std::vector<Layer> layers_;
    detail::DeviceBuffer table_, lens_, q_, ws_, pages_;
    std::vector<int32_t> host_table_, free_;
    std::vector<int> held_;  // pages of each sequence
    std::vector<int32_t> host_lens_, low_;  // low_: from there on the rows are in the ring (8-bit)
};

}  // namespace mugen_attn
