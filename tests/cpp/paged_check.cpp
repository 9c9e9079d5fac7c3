// paged_check.cpp -- GqaAttentionPaged (include/mugen_attn_paged.hpp) over several
// layers, 16- and 8-bit pages, with and without page selection: prompts in
// chunks, then a step captured once and replayed as the sequences grow; every
// output equals that of a second provider driven eagerly.  Pages run out, come
// back and are taken again; drafts are taken back; what does not fit is refused.
// Exit status 0 and a last line "PASS" when all of it holds.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstring>
#include <memory>
#include <string>
#include <vector>

#include "mugen_attn_paged.hpp"

using mugen_attn::GqaAttentionPaged;
using mugen_attn::GqaPagedShape;
using mugen_attn::Status;

namespace {

bool failed = false;
void expect(bool ok, const std::string& what) {
    if (ok) return;
    std::printf("FAIL %s\n", what.c_str());
    std::fflush(stdout);
    failed = true;
}
void expect(const Status& r, const std::string& what) { expect(bool(r), what + (r ? "" : ": " + r.error())); }
void hip(hipError_t e) { expect(e == hipSuccess, std::string("hip: ") + hipGetErrorString(e)); }

struct Dev {
    void* p = nullptr;
    size_t n;
    explicit Dev(size_t bytes) : n(bytes) { hip(hipMalloc(&p, bytes)); }
    ~Dev() { (void)hipFree(p); }
    void put(const std::vector<_Float16>& h) { hip(hipMemcpy(p, h.data(), h.size() * 2, hipMemcpyHostToDevice)); }
    std::vector<uint16_t> get() const {
        std::vector<uint16_t> h(n / 2);
        hip(hipMemcpy(h.data(), p, n, hipMemcpyDeviceToHost));
        return h;
    }
};

uint64_t seed = 1;
std::vector<_Float16> draw(size_t n) {
    std::vector<_Float16> v(n);
    for (auto& x : v) {
        seed = seed * 6364136223846793005ull + 1442695040888963407ull;
        x = (_Float16)((float)(seed >> 40) / 8388608.0f - 1.0f);
    }
    return v;
}

void run(int bits, int n_select) {
    const std::string name = "bits " + std::to_string(bits) + " select " + std::to_string(n_select);
    GqaPagedShape s;
    s.n_layers = 2;
    s.batch = 3;
    s.n_heads = 8;
    s.n_kv_heads = 2;
    s.head_dim = 64;
    s.max_seq_len = 400;
    s.n_pages = 30;
    s.page_tokens = 32;
    s.page_bits = bits;
    s.max_new = 4;
    s.max_prefill = 96;
    s.rope_dim = 64;
    s.rope = {500000.f, 1.f, 0};
    s.n_select = n_select;
    s.n_first = s.n_last = 1;
    std::unique_ptr<GqaAttentionPaged> a, b;
    expect(GqaAttentionPaged::create(s, &a), name + " create");
    expect(GqaAttentionPaged::create(s, &b), name + " create");
    if (failed) return;
    auto refused = [&](GqaPagedShape bad, const char* why) {
        std::unique_ptr<GqaAttentionPaged> c;
        expect(!GqaAttentionPaged::create(bad, &c) && !c, name + " create: " + why);
    };
    GqaPagedShape bad = s;
    bad.head_dim = 96, refused(bad, "head_dim 96"), bad = s;
    bad.n_heads = 9, refused(bad, "9 heads over 2"), bad = s;
    bad.page_tokens = 48, refused(bad, "page_tokens 48"), bad = s;
    bad.page_bits = 4, refused(bad, "page_bits 4"), bad = s;
    bad.rope_dim = 66, refused(bad, "rope_dim past head_dim"), bad = s;
    bad.max_new = 65, refused(bad, "max_new 65"), bad = s;
    if (n_select) bad.n_select = 1 << 20, refused(bad, "n_select 2^20");
    hipStream_t st;
    hip(hipStreamCreate(&st));
    const size_t qn = (size_t)s.n_heads * s.head_dim, kn = (size_t)s.n_kv_heads * s.head_dim;
    const size_t rows = 96;
    Dev q(rows * qn * 2), k(rows * kn * 2), v(rows * kn * 2), o0(rows * qn * 2), o1(rows * qn * 2);
    std::vector<std::unique_ptr<Dev>> out;  // the captured step's outputs, a layer each
    for (int L = 0; L < s.n_layers; L++) out.emplace_back(new Dev(s.batch * qn * 2));
    auto inputs = [&](size_t n) {
        q.put(draw(n * qn));
        k.put(draw(n * kn));
        v.put(draw(n * kn));
    };
    auto same = [&](const Dev& x, const Dev& y, size_t n) {
        hip(hipStreamSynchronize(st));
        const auto g = x.get(), w = y.get();
        return std::memcmp(g.data(), w.data(), n * qn * 2) == 0;
    };

    // refusals: no page reserved, bad sequence, too many tokens
    inputs(1);
    expect(!a->decode_layer(0, q.p, k.p, v.p, o0.p, st), name + ": a step without pages is refused");
    expect(!a->prefill_layer(0, 0, q.p, k.p, v.p, o0.p, 1, st), name + ": a prompt without pages is refused");
    expect(!a->reserve(3, 1, st), name + ": bad sequence");
    expect(!a->reserve(0, 401, st), name + ": past max_seq_len");
    expect(!a->decode_layer(0, q.p, k.p, v.p, o0.p, st, 5), name + ": more than max_new");

    // prompts in chunks
    const int prompt[3] = {150, 33, 64};
    for (int i = 0; i < 3; i++) {
        expect(a->reserve(i, 250, st), name + " reserve");
        expect(b->reserve(i, 250, st), name + " reserve");
        for (int at = 0; at < prompt[i];) {
            const int n = std::min(prompt[i] - at, i == 0 ? 61 : 96);
            for (int L = 0; L < s.n_layers; L++) {
                inputs(n);
                expect(a->prefill_layer(L, i, q.p, k.p, v.p, o0.p, n, st), name + " prefill");
                expect(b->prefill_layer(L, i, q.p, k.p, v.p, o1.p, n, st), name + " prefill");
                expect(same(o0, o1, n), name + " prefill: the same from both providers");
            }
            expect(a->advance_sequence(i, n, st), name + " advance_sequence");
            expect(b->advance_sequence(i, n, st), name + " advance_sequence");
            at += n;
        }
    }
    // 24 of 30 pages are taken: 5 more for one sequence, then 1 is left
    expect(a->reserve(0, 400, st), name + ": five more pages");
    expect(!a->reserve(1, 400, st), name + ": out of pages");

    // a step captured once, replayed over page ends, against eager calls
    std::vector<std::unique_ptr<Dev>> in;  // q, k, v of every layer
    for (int L = 0; L < s.n_layers; L++) {
        in.emplace_back(new Dev(s.batch * qn * 2));
        in.emplace_back(new Dev(s.batch * kn * 2));
        in.emplace_back(new Dev(s.batch * kn * 2));
    }
    mugen_attn::StepGraph step;
    const int left = a->steps_left();
    expect(left == 256 - 64, name + " steps_left");
    expect(step.capture(st, [&](hipStream_t cs) -> Status {
               for (int L = 0; L < s.n_layers; L++)
                   if (auto r = a->decode_layer(L, in[3 * L]->p, in[3 * L + 1]->p, in[3 * L + 2]->p, out[L]->p, cs); !r) return r;
               return a->advance(cs);
           }),
           name + " capture");
    for (int t = 0; t < 70 && !failed; t++) {
        for (auto& x : in) x->put(draw(x->n / 2));
        expect(step.replay(st), name + " replay");
        for (int L = 0; L < s.n_layers; L++) {
            expect(b->decode_layer(L, in[3 * L]->p, in[3 * L + 1]->p, in[3 * L + 2]->p, o1.p, st), name + " decode");
            expect(same(*out[L], o1, s.batch), name + " replay " + std::to_string(t) + " layer " + std::to_string(L));
        }
        expect(b->advance(st), name + " advance");
    }
    expect(a->sync_lengths(st), name + " sync_lengths");
    expect(a->host_lengths() == b->host_lengths(), name + ": the same lengths");

    // drafts: four tokens, two of them taken back, the next step over them; against the
    // provider that never saw them
    std::vector<_Float16> hq = draw(s.batch * 4 * qn), hk = draw(s.batch * 4 * kn), hv = draw(s.batch * 4 * kn);
    for (int L = 0; L < s.n_layers; L++) {
        q.put(hq), k.put(hk), v.put(hv);
        expect(a->decode_layer(L, q.p, k.p, v.p, o0.p, st, 4), name + " verify");
        // the first two tokens of each sequence, as a step of two
        auto two = [&](const std::vector<_Float16>& x, size_t w) {
            std::vector<_Float16> r;
            for (int i = 0; i < s.batch; i++) r.insert(r.end(), x.begin() + i * 4 * w, x.begin() + (i * 4 + 2) * w);
            return r;
        };
        q.put(two(hq, qn)), k.put(two(hk, kn)), v.put(two(hv, kn));
        hip(hipStreamSynchronize(st));
        expect(b->decode_layer(L, q.p, k.p, v.p, o1.p, st, 2), name + " two tokens");
        hip(hipStreamSynchronize(st));
    }
    expect(a->advance(st, 4), name + " advance 4");
    expect(b->advance(st, 2), name + " advance 2");
    for (int i = 0; i < s.batch; i++) expect(a->take_back(i, a->host_lengths()[i] - 2, st), name + " take_back");
    for (int t = 0; t < 3; t++) {
        for (int L = 0; L < s.n_layers; L++) {
            inputs(s.batch);
            expect(a->decode_layer(L, q.p, k.p, v.p, o0.p, st), name + " after drafts");
            expect(b->decode_layer(L, q.p, k.p, v.p, o1.p, st), name + " after drafts");
            expect(same(o0, o1, s.batch), name + " after drafts: step " + std::to_string(t));
        }
        expect(a->advance(st), name + " advance");
        expect(b->advance(st), name + " advance");
    }
    if (bits == 8) expect(!a->take_back(0, 130, st), name + ": the ring does not reach that far back");

    // a sequence leaves, its pages serve another while the captured step goes on: the
    // others' outputs are the eager ones, whose provider still has its pages
    const int free = a->free_pages();
    expect(a->release(1, st), name + " release");
    expect(a->free_pages() == free + 8, name + ": its pages are free");
    expect(a->host_lengths()[1] == 0, name + ": length 0");
    expect(a->reserve(2, 400, st), name + ": and taken");
    const int n2 = a->host_lengths()[2];
    for (int t = 0; t < 20 && !failed; t++) {
        for (auto& x : in) x->put(draw(x->n / 2));
        expect(step.replay(st), name + " replay");
        for (int L = 0; L < s.n_layers; L++) {
            expect(b->decode_layer(L, in[3 * L]->p, in[3 * L + 1]->p, in[3 * L + 2]->p, o1.p, st), name + " decode");
            hip(hipStreamSynchronize(st));
            const auto g = out[L]->get(), w = o1.get();
            for (int i : {0, 2})
                expect(std::memcmp(&g[i * qn], &w[i * qn], qn * 2) == 0,
                       name + " beside an idle slot: step " + std::to_string(t) + " sequence " + std::to_string(i));
        }
        expect(b->advance(st), name + " advance");
    }
    expect(a->sync_lengths(st), name + " sync_lengths");
    expect(a->host_lengths()[1] == 0 && a->host_lengths()[2] == n2 + 20, name + ": lengths beside an idle slot");

    // and the slot serves a new sequence, from its first token on
    expect(a->release(2, st), name + " release");
    expect(a->reserve(1, 40, st), name + " reserve again");
    expect(b->release(1, st), name + " release");
    expect(b->reserve(1, 40, st), name + " reserve again");
    for (int n : {33, 5}) {
        for (int L = 0; L < s.n_layers; L++) {
            inputs(n);
            expect(a->prefill_layer(L, 1, q.p, k.p, v.p, o0.p, n, st), name + " second prompt");
            expect(b->prefill_layer(L, 1, q.p, k.p, v.p, o1.p, n, st), name + " second prompt");
            expect(same(o0, o1, n), name + " second prompt: the same from both providers");
        }
        expect(a->advance_sequence(1, n, st), name + " advance_sequence");
        expect(b->advance_sequence(1, n, st), name + " advance_sequence");
    }
    hip(hipStreamDestroy(st));
    std::printf("%s done\n", name.c_str());
    std::fflush(stdout);
}

}  // namespace

int main() {
    for (int bits : {16, 8})
        for (int n_select : {0, 3}) run(bits, n_select);
    std::printf(failed ? "FAILED\n" : "PASS\n");
    return failed ? 1 : 0;
}
