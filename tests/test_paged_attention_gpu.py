"""Attention over the paged cache (decode, verify, page lists, prefill) against
a plain 64-bit implementation."""
import math

import pytest
import torch

from tests import paged_cases as P

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def reference(q, K, V, lens, q_lens, dtype, **kw):
    """q [B, L, H, D] -> output, bound; rows that are not there NaN."""
    B, L, H, D = q.shape
    out = torch.full((B, L, H, D), math.nan, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(B):
        n = L if q_lens is None else q_lens[b]
        for i in range(n):
            t = max(lens[b] - n + i + 1, 0)
            out[b, i], tol[b, i] = P.attend(q[b, i], K[b][:t], V[b][:t], tol_dtype=dtype, **kw)
    return out, tol


def run(store, q, lens, q_lens=None, out_dtype=None, host=True, **kw):
    """The call into a buffer of NaN, so that a row left alone shows."""
    out = torch.full(q.shape, math.nan, dtype=out_dtype or q.dtype, device=q.device)
    dev = [torch.tensor(x, dtype=torch.int32, device=q.device) if x is not None else None for x in (lens, q_lens)]
    store.attention(q, dev[0], q_lens=dev[1], out=out, seq_lens_host=lens if host else None, **kw)
    torch.cuda.synchronize()
    return out


def compare(out, want, tol, what):
    there = ~want.isnan()
    assert torch.equal(out.cpu().isnan(), ~there), f"{what}: rows written that should not be, or the reverse"
    P.check(out.cpu()[there], want[there], tol[there], out.dtype, what)


# lengths around nothing, a token, a tile, a page, a wave round
LENS = [1, 0, 31, 32, 33, 64, 65, 127, 129, 300]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,Hk,D,page", [(8, 2, 64, 32), (7, 1, 128, 64), (4, 4, 128, 128), (32, 2, 64, 128), (3, 1, 256, 32)])
def test_decode(device, bits, dtype, H, Hk, D, page):
    P.say(f"decode bits={bits} {dtype} H={H}/{Hk} D={D} page={page}")
    store, K, V = P.make_store(11, LENS, Hk, D, page, bits, dtype)
    q = P.randn(12, len(LENS), 1, H, D, dtype=dtype)
    want, tol = reference(q.cpu(), K, V, LENS, None, dtype)
    for host in (True, False):
        compare(run(store, q, LENS, host=host), want, tol, f"host={host}")
    for splits in (1, 3):
        compare(run(store, q, LENS, num_splits=splits, out_dtype=torch.float32), want, tol, f"splits={splits}")


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("H,Hk,D,L", [(8, 2, 64, 3), (7, 1, 128, 5), (16, 1, 128, 8), (2, 2, 64, 40), (6, 2, 256, 9)])
def test_verify(device, bits, H, Hk, D, L):
    """Several new tokens, causal among them; ragged counts, a sequence shorter than its new tokens."""
    lens = [200, 64 + L, L, 97, 33, max(1, L - 2)]
    q_lens = [L, max(1, L - 1), L, 0, 2, L]
    for dtype in (F16, BF16):
        P.say(f"verify bits={bits} {dtype} H={H}/{Hk} D={D} L={L}")
        store, K, V = P.make_store(21, lens, Hk, D, 32, bits, dtype)
        q = P.randn(22, len(lens), L, H, D, dtype=dtype)
        for ql in (q_lens, None):
            want, tol = reference(q.cpu(), K, V, lens, ql, dtype)
            for kw in (dict(), dict(host=False), dict(num_splits=2)):
                compare(run(store, q, lens, ql, **kw), want, tol, f"q_lens={ql} {kw}")


@pytest.mark.parametrize("bits", [16, 8])
def test_long_ragged_splits(device, bits):
    """Contexts that take many splits, more than 64 pages a split, both planners."""
    lens = [5000, 17, 2300, 4097, 640, 1]
    P.say(f"long bits={bits}")
    store, K, V = P.make_store(31, lens, 1, 64, 32, bits, F16)
    q = P.randn(32, len(lens), 1, 4, 64)
    want, tol = reference(q.cpu(), K, V, lens, None, F16)
    for kw in (dict(), dict(host=False), dict(num_splits=1), dict(num_splits=70)):
        compare(run(store, q, lens, **kw), want, tol, str(kw))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_what_a_query_does_not_see(device, bits, dtype):
    """V of later new tokens that is not finite reaches no earlier query; K either."""
    L, T = 6, 70 if bits == 8 else 61
    store, K, V = P.make_store(41, [T], 1, 128, 32, bits, dtype)
    q = P.randn(42, 1, L, 7, 128, dtype=dtype)
    t = T - 3  # seen by the last 3 queries only
    if bits == 8:  # two of the tokens in question are in a whole page's codes
        page = int(store.page_table[0, 1])
        T = 64
        L = 3
        q = q[:, :L].contiguous()
        t = 62
        store.v_pages[page, 0, 0, :, t - 32] = 0x7f
        store.k_pages[page, 0, t - 32, 5] = 0x7f
    else:
        page = int(store.page_table[0, t // 32])
        store.v_pages[page, 0, t % 32, 3:9] = math.inf
        store.k_pages[page, 0, t % 32, 5] = math.nan
    V[0] = V[0].clone()
    want, tol = reference(q.cpu(), [K[0][:T]], [V[0][:T]], [T], None, dtype)
    out = run(store, q, [T]).cpu()
    blind = [i for i in range(L) if T - L + i + 1 <= t]
    assert blind
    P.check(out[0, blind], want[0, blind], tol[0, blind], dtype, "queries before the token")
    assert out[0, max(blind) + 1:].isnan().all(), "a NaN that a query sees has to show"


@pytest.mark.parametrize("bits", [16, 8])
def test_page_lists(device, bits):
    H, Hk, D, page, L = 6, 2, 128, 32, 2
    lens = [400, 33, 64, 96]
    store, K, V = P.make_store(51, lens, Hk, D, page, bits, F16)
    q = P.randn(52, len(lens), L, H, D)
    lists = torch.full((len(lens), L, Hk, 7), -1, dtype=torch.int32)
    # ascending; repeated and unordered entries; past the end; empty; the open page alone
    lists[0, 0, 0] = torch.tensor([0, 3, 4, 9, 11, 12, -1])
    lists[0, 0, 1] = torch.tensor([5, 5, 6, 2, 11, 11, 12])
    lists[0, 1, 0] = torch.tensor([12, 13, 500, 2 ** 31 - 1, -1, -1, -1])
    lists[0, 1, 1] = torch.tensor([-5, -3, 0, 1, -1, 2, 3])
    lists[1, :, :, 0] = 1
    lists[2, :, :, :2] = torch.tensor([0, 1])
    lists[3, :, 0, 0] = 0
    lists[3, :, 1, :3] = torch.tensor([1, 2, 3])

    def kept(seen, row, t):
        """The rule: an entry above the one before it, of a page that is seen."""
        n = -(-t // page)
        ok = [p for k, p in enumerate(row[:min(len(row), n)]) if p > (row[k - 1] if k else -1) and 0 <= p < n]
        m = torch.zeros(seen, dtype=torch.bool)
        for p in ok:
            m[p * page:(p + 1) * page] = True
        return m[:t]

    want = torch.zeros((len(lens), L, H, D), dtype=torch.float64)
    tol = torch.zeros_like(want)
    for b, T in enumerate(lens):
        for i in range(L):
            t = T - L + i + 1
            keep = [kept(T + 32, lists[b, i, j].tolist(), t) for j in range(Hk)]
            want[b, i], tol[b, i] = P.attend(q[b, i].cpu(), K[b][:t], V[b][:t], keep=keep, tol_dtype=F16)
    for kw in (dict(), dict(host=False), dict(num_splits=1), dict(num_splits=3)):
        compare(run(store, q, lens, pages=lists.cuda(), **kw), want, tol, str(kw))


@pytest.mark.parametrize("bits", [16, 8])
def test_pages_that_are_not_there(device, bits):
    """A table entry outside the pool leaves its tokens out."""
    lens = [200, 96]
    store, K, V = P.make_store(61, lens, 1, 64, 32, bits, F16)
    store.page_table[0, 1], store.page_table[0, 4], store.page_table[1, 0] = -1, 10 ** 6, -2 ** 31
    q = P.randn(62, 2, 1, 3, 64)
    keep = [torch.ones(T, dtype=torch.bool) for T in lens]
    keep[0][32:64] = keep[0][128:160] = keep[1][:32] = False
    ref = [P.attend(q[b, 0].cpu(), K[b], V[b], keep=[keep[b]], tol_dtype=F16) for b in range(2)]
    want, tol = (torch.stack([r[x] for r in ref])[:, None] for x in (0, 1))
    for kw in (dict(), dict(host=False)):
        compare(run(store, q, lens, **kw), want, tol, str(kw))


def test_empty_and_clamped_lengths(device):
    store, K, V = P.make_store(71, [40, 64], 1, 64, 32, 16, F16, max_seq=64)
    q = P.randn(72, 2, 1, 2, 64)
    out = run(store, q, [0, -3], host=False)
    assert (out == 0).all()
    # a device length past max_seq_len is the cache's end
    want, tol = reference(q.cpu(), [K[0], K[1]], [V[0], V[1]], [40, 64], None, F16)
    compare(run(store, q, [40, 9999], host=False), want, tol, "clamped")


@pytest.mark.parametrize("bits", [16, 8])
def test_far_pages(device, bits):
    """A pool of more than 2^32 bytes: the pages at its end."""
    Hk, D, page = 8, 128, 128
    n = (1 << 32) // (Hk * page * D * bits // 8) + 70
    small, K, V = P.make_store(81, [300], Hk, D, page, bits, F16, junk=False)
    import mugen_amd
    shape = {n_: (n, *getattr(small, n_).shape[1:]) for n_ in ("k_pages", "v_pages")}
    big = {n_: torch.empty(s, dtype=small.k_pages.dtype, device=device) for n_, s in shape.items()}
    kw = {}
    m = small.k_pages.shape[0]
    for n_ in big:
        big[n_][n - m:] = getattr(small, n_)
    if bits == 8:
        for n_ in ("k_exp", "v_exp"):
            kw[n_] = torch.ones((n, Hk), dtype=torch.uint8, device=device)
            kw[n_][n - m:] = getattr(small, n_)
        kw["tail_k"], kw["tail_v"] = small.tail_k, small.tail_v
    table = torch.where(small.page_table >= 0, small.page_table + (n - m), small.page_table)
    store = mugen_amd.PagedStore(big["k_pages"], big["v_pages"], table, 384, **kw)
    q = P.randn(82, 1, 1, 8, D)
    want, tol = reference(q.cpu(), K, V, [300], None, F16)
    compare(run(store, q, [300]), want, tol, "far pages")


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("H,Hk,D,page,n,start", [(4, 2, 64, 32, 1, 0), (7, 1, 128, 64, 9, 100), (7, 1, 128, 64, 77, 0),
                                                 (4, 2, 64, 128, 130, 333), (2, 1, 256, 32, 65, 31), (28, 4, 128, 64, 253, 700)])
def test_prefill(device, bits, H, Hk, D, page, n, start):
    for dtype in (F16, BF16):
        P.say(f"prefill bits={bits} {dtype} H={H}/{Hk} D={D} n={n} start={start}")
        T = start + n
        store, K, V = P.make_store(91, [40, T], Hk, D, page, bits, dtype, junk=False)
        q = P.randn(92, n, H, D, dtype=dtype)
        rows = sorted({0, 1, n // 2, n - 2, n - 1} & set(range(n)))
        out = store.prefill(q, 1, start).cpu()
        for i in rows:
            # (the prompt kernels weight bf16 V in fp16 too)
            want, tol = P.attend(q[i].cpu(), K[1][:start + i + 1], V[1][:start + i + 1], tol_dtype=F16)
            P.check(out[i], want, tol * 2, dtype, f"token {i}")


@pytest.mark.parametrize("H,Hk,D,n,start", [(28, 4, 128, 100, 3000), (32, 8, 64, 80, 2500)])
def test_prefill_split_partials_keep_small_values(device, H, Hk, D, n, start):
    """Key ranges that are merged keep 32 bits: V of 1 .. 4 times the least
    fp16 number, whose means fp16 cannot hold."""
    P.say(f"prefill of least values H={H}/{Hk} D={D} n={n} start={start}")
    T = start + n
    store, K, _ = P.make_store(93, [40, T], Hk, D, 64, 16, F16, junk=False)
    g = torch.Generator().manual_seed(94)
    v = torch.randint(1, 5, store.v_pages.shape, generator=g).to(torch.float64) * 2.0 ** -24
    store.v_pages.copy_(v.to(F16))
    pages = store.page_table[1, :-(-T // 64)].long().cpu()
    V = v[pages].transpose(1, 2).reshape(-1, Hk, D)[:T]
    q = P.randn(95, n, H, D)
    out = store.prefill(q, 1, start, out_dtype=torch.float32).cpu()
    for i in (0, n // 2, n - 1):
        want, tol = P.attend(q[i].cpu(), K[1][:start + i + 1], V[:start + i + 1], tol_dtype=F16)
        P.check(out[i], want, tol, torch.float32, f"token {i}")
