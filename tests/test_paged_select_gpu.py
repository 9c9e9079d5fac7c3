"""The choice of pages against the definition in 64 bits: exact, ties included."""
import math

import pytest
import torch

from tests import paged_cases as P

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def ranges_store(seed, lens, Hk, D, page, dtype, max_seq=None, values=None):
    """A store whose ranges are random (the selection reads nothing else)."""
    import mugen_amd
    g = torch.Generator().manual_seed(seed)
    width = -(-(max_seq or max(lens) + 1) // page)
    count = [-(-t // page) for t in lens]
    n = sum(count) + 2
    table = torch.full((len(lens), width), -9, dtype=torch.int32)
    ids, at = torch.randperm(n, generator=g).to(torch.int32), 0
    for b, c in enumerate(count):
        table[b, :c] = ids[at:at + c]
        at += c
    r = values(n) if values else torch.randn((n, Hk, 2, D), generator=g).sort(2).values
    r = r.to(dtype)
    z = torch.zeros((n, Hk, page, D), dtype=dtype, device="cuda")
    return mugen_amd.PagedStore(z, z, table.cuda(), width * page, k_range=r.cuda()), r.double(), table


def expect(store, r, table, q, lens, q_lens, n_select, first, last, old):
    page, Hk = store.k_pages.shape[2], store.n_kv_heads
    out = old.clone()
    for b, T in enumerate(lens):
        n = q.shape[1] if q_lens is None else q_lens[b]
        for i in range(n):
            pages = -(-max(T - n + i + 1, 0) // page)
            rows = r[table[b, :pages].long()]
            for j in range(Hk):
                G = q.shape[2] // Hk
                got = P.choose(q[b, i, j * G:(j + 1) * G].cpu(), rows[:, j, 0], rows[:, j, 1], pages, n_select, first, last)
                out[b, i, j] = torch.tensor(got + [-1] * (n_select - len(got)))
    return out


def run(store, q, lens, n_select, first, last, q_lens=None):
    dev = [torch.tensor(x, dtype=torch.int32, device="cuda") if x is not None else None for x in (lens, q_lens)]
    out = torch.full((*q.shape[:2], store.n_kv_heads, n_select), -77, dtype=torch.int32, device="cuda")
    store.select_pages(q, dev[0], n_select, first=first, last=last, q_lens=dev[1], out=out)
    torch.cuda.synchronize()
    return out.cpu()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,Hk,D,page,L,lens,pick", [
    (8, 2, 64, 32, 1, [3000, 1, 0, 64, 65, 32 * 9, 32 * 9 + 1], (9, 1, 2)),
    (7, 1, 128, 64, 3, [5000, 700, 2, 64 * 20], (8, 0, 1)),
    (16, 1, 128, 32, 11, [4000, 333], (20, 3, 4)),
    (6, 2, 256, 128, 2, [9000, 128 * 30 + 5], (7, 2, 5)),
])
def test_selection(device, dtype, H, Hk, D, page, L, lens, pick):
    P.say(f"select {dtype} H={H}/{Hk} D={D} page={page} L={L}")
    store, r, table = ranges_store(7, lens, Hk, D, page, dtype)
    q = P.randn(8, len(lens), L, H, D, dtype=dtype)
    old = torch.full((len(lens), L, Hk, pick[0]), -77, dtype=torch.int32)
    for ql in (None, [max(0, L - b) for b in range(len(lens))]):
        want = expect(store, r, table, q, lens, ql, *pick, old)
        assert torch.equal(run(store, q, lens, *pick, q_lens=ql), want)


# rows of the select kernel's three widths, and its longest
@pytest.mark.parametrize("pages", [1000, 1025, 4096, 4097, 16384])
def test_many_pages(device, pages):
    T = pages * 32
    store, r, table = ranges_store(9, [T, T // 3], 1, 64, 32, F16, max_seq=T)
    q = P.randn(10, 2, 1, 2, 64)
    for pick in ((64, 1, 2), (pages // 2, 0, 1), (pages - 1, 0, 1), (3, 1, 2)):
        want = expect(store, r, table, q, [T, T // 3], None, *pick, torch.zeros((2, 1, 1, pick[0]), dtype=torch.int32))
        assert torch.equal(run(store, q, [T, T // 3], *pick), want), pick


def test_ties_take_the_lowest_pages(device):
    """Equal scores, whole runs of them around the border, zeros of both signs."""
    T = 200 * 32

    def values(n):
        v = torch.zeros((n, 1, 2, 64))
        v[:, 0, :, 0] = (torch.arange(n) % 3)[:, None].float()
        v[::7, 0, :, 1] = -0.0
        return v

    store, r, table = ranges_store(13, [T], 1, 64, 32, F16, values=values)
    q = torch.zeros((1, 1, 1, 64), dtype=F16, device="cuda")
    for q0 in (1.0, 0.0, -1.0):
        q[..., 0] = q0
        for n in (3, 10, 70, 150, 199):
            want = expect(store, r, table, q, [T], None, n, 1, 2, torch.zeros((1, 1, 1, n), dtype=torch.int32))
            assert torch.equal(run(store, q, [T], n, 1, 2), want), (q0, n)


def test_values_that_are_not_finite(device):
    """NaN scores come first (an infinite range makes one too: 0 * inf, no query
    here has a negative part); a page that is not there last."""
    T = 64 * 32
    store, r, table = ranges_store(17, [T], 1, 64, 32, F16)
    q = torch.ones((1, 1, 1, 64), dtype=F16, device="cuda")
    for page, v in ((5, math.nan), (50, math.nan), (30, math.inf), (20, -math.inf)):
        r[table[0, page].long(), 0, :, 3] = v
    store.k_range.copy_(r.to(F16))
    assert run(store, q, [T], 3, 1, 1)[0, 0, 0].tolist() == [0, 5, 63]
    assert run(store, q, [T], 6, 1, 1)[0, 0, 0].tolist() == [0, 5, 20, 30, 50, 63]
    # with both parts in the query infinities count as such: +inf first, -inf last
    q = torch.ones((1, 1, 2, 64), dtype=F16, device="cuda")
    q[0, 0, 1] = -2.0
    for page, lo, hi in ((5, 0.0, 1.0), (50, 0.0, 1.0), (30, 0.0, math.inf), (20, math.inf, -math.inf)):
        r[table[0, page].long(), 0, 0, 3], r[table[0, page].long(), 0, 1, 3] = lo, hi
    store.k_range.copy_(r.to(F16))
    assert run(store, q, [T], 3, 1, 1)[0, 0, 0].tolist() == [0, 30, 63]
    assert 20 not in run(store, q, [T], 63, 1, 1)[0, 0, 0].tolist()
    store.page_table[0, 40] = -1
    got = run(store, q, [T], 62, 1, 1)[0, 0, 0].tolist()
    assert 40 not in got and 20 not in got


def test_far_apart_scores_are_summed_exactly(device):
    """Terms that cancel: 32-bit sums would lose the small ones that decide."""
    T = 40 * 32
    store, r, table = ranges_store(19, [T], 1, 64, 32, F16)
    r[:] = 0
    r[..., 0], r[..., 1] = 60000.0, -60000.0
    for page in range(40):
        r[table[0, page].long(), 0, :, 2] = (page * 7 % 40) * 2.0 ** -20
    store.k_range.copy_(r.to(F16))
    q = torch.zeros((1, 1, 1, 64), dtype=F16, device="cuda")
    q[..., 0] = q[..., 1] = 1000.0
    q[..., 2] = 1.0
    want = sorted([39] + sorted(range(39), key=lambda p: -(p * 7 % 40))[:9])
    assert run(store, q, [T], 10, 0, 1)[0, 0, 0].tolist() == want
