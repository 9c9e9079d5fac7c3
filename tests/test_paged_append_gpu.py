"""Appending to the paged cache: the rotation against 64 bits, the 8-bit pages bit
for bit, what is left alone, and the operators together as a serving loop uses them."""
import math

import numpy as np
import pytest
import torch

import mugen_amd
from tests import paged_cases as P

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def empty_store(B, width, Hk, D, page, bits, dtype, ring=None, ranges=True, fill=0x55):
    n = B * width + 2
    table = torch.randperm(n, generator=torch.Generator().manual_seed(5))[:B * width].to(torch.int32).view(B, width)
    kw = {}
    if bits == 8:
        k = torch.full((n, Hk, page, D), fill, dtype=torch.uint8, device="cuda")
        v = torch.full((n, Hk, page // 32, D, 32), fill, dtype=torch.uint8, device="cuda")
        for x in ("k_exp", "v_exp"):
            kw[x] = torch.full((n, Hk), fill, dtype=torch.uint8, device="cuda")
        for x in ("tail_k", "tail_v"):
            kw[x] = torch.full((B, ring or 2 * page, Hk, D), 3.0, dtype=dtype, device="cuda")
    else:
        k, v = (torch.full((n, Hk, page, D), 3.0, dtype=dtype, device="cuda") for _ in range(2))
    if ranges:
        kw["k_range"] = torch.full((n, Hk, 2, D), 3.0, dtype=dtype, device="cuda")
    return mugen_amd.PagedStore(k, v, table.cuda(), width * page, **kw)


def tensors(store):
    return {n: getattr(store, n) for n in ("k_pages", "v_pages", "k_exp", "v_exp", "tail_k", "tail_v", "k_range")
            if getattr(store, n) is not None}


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def rotation_bound(x, pos, rope, dim, dtype):
    """Half a step of the result; sine and cosine (2^-22) and the two products and
    their sum in fp32 (2^-24 each) relative to the pair's magnitudes; the angle in 64
    bits adds pos * f * 2^-52 turns."""
    want = P.rotated(x, pos, rope, dim)
    x = x.double().cpu().abs()
    pair = torch.cat((x[..., :dim // 2] + x[..., dim // 2:dim],) * 2 + (x[..., dim:],), -1)
    return want, pair * (2.0 ** -21 + pos.abs().max().item() * 2.0 ** -50)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,rope_dim,rope,start", [
    (128, 128, (1e6, 1.0, 0), 0), (64, 64, (5e5, 1.0, 0), 40), (256, 256, (1e4, 1.0, 0), 7),
    (128, 64, (1e4, 40.0, 4096), 1000), (64, 16, (1e4, 1.0, 0), 3), (128, 0, (1e4, 1.0, 0), 3),
    (128, 128, (1e4, 8.0, 8192), 2 ** 20)])
def test_rotation(device, dtype, D, rope_dim, rope, start):
    """Queries and keys, slices of one fused projection; ragged counts; rows that are not there."""
    B, n, H, Hk, page = 3, 5, 6, 2, 32
    width = -(-(start + 64) // page)
    store = empty_store(B, width, Hk, D, page, 16, dtype, ranges=False)
    qkv = P.randn(3, B, n, H + 2 * Hk, D, dtype=dtype)
    q, k, v = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
    T, new = [start, start + 31, start + 1], [5, 3, 0]
    q_out = torch.full((B, n, H, D), 9.0, dtype=dtype, device=device)
    lens = torch.full((B,), -1, dtype=torch.int32, device=device)
    before = {x: t.clone() for x, t in tensors(store).items()}
    kw = dict(rope=rope, rope_dim=rope_dim) if rope_dim else {}
    store.append(k, v, i32(T), new_lens=i32(new), seq_lens_out=lens, q=q, q_out=q_out, **kw)
    torch.cuda.synchronize()
    assert lens.tolist() == [t + c for t, c in zip(T, new)]
    for b in range(B):
        pos = torch.arange(T[b], T[b] + n)
        for x, got in ((q[b], q_out[b]), (k[b], None)):
            want, tol = rotation_bound(x, pos, rope, rope_dim, dtype) if rope_dim else (x.double().cpu(), torch.zeros(x.shape))
            if got is None:
                got = torch.stack([store.k_pages[int(store.page_table[b, t // page]), :, t % page] for t in pos.tolist()])
            for j in range(new[b]):
                P.check(got[j], want[j], tol[j].double(), dtype, f"seq {b} token {j}")
        for j in range(new[b], n):
            assert (q_out[b, j] == 9.0).all()
        for j in range(new[b]):
            t = T[b] + j
            at = int(store.page_table[b, t // page])
            assert torch.equal(store.v_pages[at, :, t % page], v[b, j])
            before["k_pages"][at, :, t % page] = store.k_pages[at, :, t % page]
            before["v_pages"][at, :, t % page] = v[b, j]
    for x, t in tensors(store).items():
        assert torch.equal(t, before[x]), f"{x}: written beyond the new rows"


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Hk,D,page,ring", [(2, 64, 32, 64), (1, 128, 64, 128), (1, 256, 128, 256), (3, 128, 32, 256)])
def test_pages_are_a_function_of_their_tokens(device, dtype, Hk, D, page, ring):
    """However the tokens come in (one by one, drafts, one long prompt): the same
    pages, and those bit for bit the codes of the rotated 16-bit rows."""
    B, width, total = 2, 5, 4 * page + 11
    k, v = P.randn(13, B, total, Hk, D, dtype=dtype), P.randn(14, B, total, Hk, D, dtype=dtype)
    k[:, page:2 * page] *= 1e-4  # small pages, a zero one, one with a lone large value
    v[:, page:2 * page] = 0
    v[:, 2 * page] *= 500
    rows = empty_store(B, width, Hk, D, page, 16, dtype)
    rows.append(k, v, i32([0] * B), rope=P.ROPE)
    stores = []
    for steps in ([total], [1] * total, [page - 1, 1, 1, 2 * page + 3, 7, page - 8, total], [3] * total):
        s = empty_store(B, width, Hk, D, page, 8, dtype, ring=ring)
        at = 0
        for n in steps:
            n = min(n, total - at)
            if n > 0:
                s.append(k[:, at:at + n].contiguous(), v[:, at:at + n].contiguous(), i32([at] * B), rope=P.ROPE)
            at += n
        stores.append(s)
    torch.cuda.synchronize()
    first = tensors(stores[0])
    for s in stores[1:]:
        for x, t in tensors(s).items():
            if x.startswith("tail"):  # the newest rows; what older slots hold depends on the steps
                at = [t_ % ring for t_ in range(4 * page, total)]
                assert torch.equal(t[:, at], first[x][:, at]), x
            else:
                assert torch.equal(t.view(torch.uint8), first[x].view(torch.uint8)), x
    s = stores[0]
    for b in range(B):
        for p in range(width):
            i, ri = int(s.page_table[b, p]), int(rows.page_table[b, p])
            for h in range(Hk):
                if p >= total // page:
                    assert (s.k_pages[i, h] == 0x55).all() and int(s.k_exp[i, h]) == 0x55
                    continue
                kc, ke, kv = P.quantised(rows.k_pages[ri, h])
                vc, ve, _ = P.quantised(rows.v_pages[ri, h])
                assert int(s.k_exp[i, h]) == ke and int(s.v_exp[i, h]) == ve
                assert torch.equal(s.k_pages[i, h].cpu(), kc)
                assert torch.equal(s.v_pages[i, h].cpu(), vc.view(page // 32, 32, D).transpose(1, 2))
                assert torch.equal(s.k_range[i, h].cpu(), torch.stack((kv.amin(0), kv.amax(0))).to(dtype))
                r = rows.k_pages[ri, h].cpu()
                assert torch.equal(rows.k_range[ri, h].cpu(), torch.stack((r.amin(0), r.amax(0))))
    tail = torch.stack([rows.k_pages[rows.page_table[:, t // page].long(), :, t % page] for t in range(4 * page, total)], 1)
    assert torch.equal(s.tail_k[:, [t % ring for t in range(4 * page, total)]], tail)


def test_values_at_the_edge(device):
    """Not finite -> NaN codes (the page's exponent from its finite values), the
    largest and the smallest magnitudes of each type, borders of the exponent."""
    for dtype in (F16, BF16):
        fin = torch.finfo(dtype)
        k = P.randn(23, 1, 64, 1, 64, dtype=dtype)
        v = P.randn(24, 1, 64, 1, 64, dtype=dtype)
        k[0, 3, 0, 5], k[0, 4, 0, 6], k[0, 40, 0, 7] = math.inf, -math.inf, math.nan
        v[0, :32], v[0, 32:] = fin.tiny, fin.max
        v[0, 1, 0, 0] = fin.smallest_normal / 2
        k[0, 32:] = (k[0, 32:] * 0.01).clamp(-0.875, 0.875)
        k[0, 33, 0, 0] = -0.875  # 448 / 512: the last value of its exponent
        s = empty_store(1, 2, 1, 64, 32, 8, dtype)
        s.append(k, v, i32([0]))
        torch.cuda.synchronize()
        for p in range(2):
            i = int(s.page_table[0, p])
            for x, pool, exp in ((k, s.k_pages, s.k_exp), (v, s.v_pages, s.v_exp)):
                codes, byte, val = P.quantised(x[0, 32 * p:32 * p + 32, 0])
                got = pool[i, 0].cpu()
                got = got if x is k else got[0].T
                assert int(exp[i, 0]) == byte
                assert torch.equal(got, codes)
            lo = s.k_range[i, 0, 0].cpu()
            assert lo.isnan().any() and not lo.isnan().all()


def test_drafts_taken_back(device):
    """A step's rejected tokens: the length goes back over a filled page, the next
    tokens overwrite it."""
    page, D = 32, 64
    k, v = P.randn(33, 1, 100, 2, D), P.randn(34, 1, 100, 2, D)
    s = empty_store(1, 4, 2, D, page, 8, F16, ring=64)
    s.append(k[:, :29].contiguous(), v[:, :29].contiguous(), i32([0]), rope=P.ROPE)
    s.append(k[:, 60:68].contiguous(), v[:, 60:68].contiguous(), i32([29]), rope=P.ROPE)  # drafts: page 0 fills
    s.append(k[:, 30:36].contiguous(), v[:, 30:36].contiguous(), i32([30]), rope=P.ROPE)  # one was right
    kk = torch.cat((k[:, :29], k[:, 60:61], k[:, 30:36]), 1)
    vv = torch.cat((v[:, :29], v[:, 60:61], v[:, 30:36]), 1)
    r = empty_store(1, 4, 2, D, page, 8, F16, ring=64)
    r.append(kk, vv, i32([0]), rope=P.ROPE)
    torch.cuda.synchronize()
    i, j = int(s.page_table[0, 0]), int(r.page_table[0, 0])
    for x in ("k_pages", "v_pages", "k_exp", "v_exp", "k_range"):
        assert torch.equal(getattr(s, x)[i], getattr(r, x)[j]), x
    assert torch.equal(s.tail_k[:, 32:36], r.tail_k[:, 32:36])


def test_how_far_a_sequence_goes_back(device):
    """KVCachePaged.truncate: as far as the ring still holds the open page's rows, counted
    from the longest the sequence has been; a page's end needs none."""
    kv = mugen_amd.KVCachePaged(1, 1, 1, 64, 512, page_tokens=32, max_new=32, device=device)  # ring 64
    k = P.randn(37, 1, 200, 1, 64)
    kv.append(0, k, k)
    with pytest.raises(RuntimeError):
        kv.truncate(0, 100)
    with pytest.raises(RuntimeError):
        kv.release(0)
    kv.advance()
    kv.truncate(0, 170)  # open page 160: the ring holds 136 .. 199
    with pytest.raises(ValueError):
        kv.truncate(0, 150)  # open page 128
    kv.truncate(0, 128)
    kv.append(0, k[:, :7].contiguous(), k[:, :7].contiguous())
    kv.advance()
    with pytest.raises(ValueError):
        kv.truncate(0, 140)  # longer than it is
    kv.truncate(0, 130)  # its open page 128 is behind the ring of 200, but was written again ...
    kv.release(0)
    assert kv.free_pages == 16 and kv.seq_lens.tolist() == [0]


@pytest.mark.parametrize("bits", [16, 8])
def test_dropped_rows(device, bits):
    """Past max_seq_len, and in pages that are not there: nothing is written."""
    s = empty_store(2, 2, 1, 64, 32, bits, F16)
    s.page_table[1, 0] = -1
    before = {x: t.clone() for x, t in tensors(s).items()}
    n = 20
    k, v, q = (P.randn(43 + i, 2, n, h, 64) for i, h in enumerate((1, 1, 2)))
    q_out = torch.full((2, n, 2, 64), 9.0, dtype=F16, device=device)
    lens = i32([0, 0])
    s.append(k, v, i32([60, 3]), q=q, q_out=q_out, seq_lens_out=lens)
    torch.cuda.synchronize()
    assert lens.tolist() == [64, 23]
    assert torch.equal(q_out[0, :4], q[0, :4]) and (q_out[0, 4:] == 9.0).all() and torch.equal(q_out[1], q[1])
    if bits == 16:
        i = int(s.page_table[0, 1])
        before["k_pages"][i, :, 28:], before["v_pages"][i, :, 28:] = k[0, :4].transpose(0, 1), v[0, :4].transpose(0, 1)
        before["k_range"][i] = s.k_range[i]
        for x in ("k_pages", "v_pages", "k_range"):
            assert torch.equal(getattr(s, x), before[x]), x


# ---------------------------------------------------------------- together

def model_step(kv, layers, qkv, H, Hk, rope, pick=None):
    """One step of a model's attention calls; returns each layer's output."""
    out = []
    for x in range(layers):
        q, k, v = qkv[x][:, :, :H], qkv[x][:, :, H:H + Hk], qkv[x][:, :, H + Hk:]
        q = kv.append(x, k, v, q=q, rope=rope)
        pages = kv.select_pages(x, q, pick[0], first=pick[1], last=pick[2]) if pick else None
        out.append((q, kv.attention(x, q, pages=pages), pages))
    kv.advance()
    return out


@pytest.mark.parametrize("bits,dtype", [(16, BF16), (8, F16)])
def test_a_serving_loop(device, bits, dtype):
    """Prompts of two lengths, decode steps, a verify step that is taken back, a sequence
    that leaves and one that comes: every step against 64 bits over the rows appended."""
    layers, B, H, Hk, D = 2, 2, 6, 2, 64
    kv = mugen_amd.KVCachePaged(layers, B, Hk, D, 512, n_pages=20, page_tokens=32, page_bits=bits, dtype=dtype, max_new=8,
                                k_range=True, device=device)
    held = [[[torch.zeros(0, Hk, D, dtype=torch.float64)] * 2 for _ in range(B)] for _ in range(layers)]

    def values(x, b, T):
        """K, V that a query attends to: what the store holds (codes checked elsewhere)."""
        s, ks, vs = kv.layers[x], [], []
        for p in range(-(-T // 32)):
            i = int(kv.page_table[b, p])
            if bits == 8 and (p + 1) * 32 > T:
                at = torch.arange(p * 32, p * 32 + 32) % s.tail_k.shape[1]
                ks.append(s.tail_k[b, at].double().cpu())
                vs.append(s.tail_v[b, at].double().cpu())
                continue
            k, v = s.k_pages[i], s.v_pages[i]
            if bits == 8:
                k = k.view(P.E4M3).double() * 2.0 ** (s.k_exp[i].double() - 127)[:, None, None]
                v = v[:, 0].transpose(1, 2).contiguous().view(P.E4M3).double() * 2.0 ** (s.v_exp[i].double() - 127)[:, None, None]
            ks.append(k.double().cpu().transpose(0, 1))
            vs.append(v.double().cpu().transpose(0, 1))
        return torch.cat(ks)[:T], torch.cat(vs)[:T]

    def verify(step, lens, n):
        for x, (q, out, pages) in enumerate(step):
            for b in range(B):
                K, V = values(x, b, lens[b])
                # the rows are the appended ones, to an E4M3 step of the page's largest value
                for i in range(n):
                    t = lens[b] - n + i + 1
                    keep = None
                    if pages is not None:
                        keep = [torch.zeros(t, dtype=torch.bool) for _ in range(Hk)]
                        for j in range(Hk):
                            for p in pages[b, i, j].tolist():
                                if p >= 0:
                                    keep[j][32 * p:32 * p + 32] = True
                        assert all(m[-1] and m[0] for m in keep)
                    want, tol = P.attend(q[b, i], K[:t], V[:t], keep=keep, tol_dtype=dtype)
                    P.check(out[b, i], want, tol, dtype, f"layer {x} seq {b} token {i}")

    def rows(seed, n):
        return [P.randn(seed + x, B, n, H + 2 * Hk, D, dtype=dtype) for x in range(layers)]

    # prompts: 70 tokens for both, then 100 more for sequence 0
    qkv = rows(100, 70)
    for x in range(layers):
        q = kv.append(x, qkv[x][:, :, H:H + Hk], qkv[x][:, :, H + Hk:], q=qkv[x][:, :, :H], rope=P.ROPE)
        for b in range(B):
            out = kv.prefill(x, b, q[b])
            K, V = values(x, b, 70)
            for i in (0, 33, 69):
                want, tol = P.attend(q[b, i], K[:i + 1], V[:i + 1], tol_dtype=F16)
                P.check(out[i], want, 2 * tol, dtype, f"prompt {b} token {i}")
    kv.advance()
    qkv = rows(110, 100)
    for x in range(layers):
        q = kv.append(x, qkv[x][:, :, H:H + Hk], qkv[x][:, :, H + Hk:], q=qkv[x][:, :, :H], rope=P.ROPE, new_lens=[100, 0])
        kv.prefill(x, 0, q[0])
    kv.advance()
    lens = [170, 70]
    assert kv.seq_lens.tolist() == lens
    for s in range(24):
        step = model_step(kv, layers, rows(200 + 10 * s, 1), H, Hk, P.ROPE, pick=(3, 1, 1) if s % 2 else None)
        lens = [t + 1 for t in lens]
        verify(step, lens, 1)
    step = model_step(kv, layers, rows(500, 4), H, Hk, P.ROPE)
    verify(step, [t + 4 for t in lens], 4)
    kv.truncate(0, lens[0] + 1)
    kv.truncate(1, lens[1] + 3)
    lens = [lens[0] + 1, lens[1] + 3]
    free = kv.free_pages
    kv.release(1)
    assert kv.free_pages > free
    lens[1] = 0
    for s in range(3):
        step = model_step(kv, layers, rows(600 + 10 * s, 1), H, Hk, P.ROPE)
        lens = [t + 1 for t in lens]
        verify(step, lens, 1)
    with pytest.raises(RuntimeError):
        kv.reserve(1, 512)


@pytest.mark.parametrize("bits", [16, 8])
def test_a_captured_step(device, bits):
    """Append, selection and attention captured once, replayed over growing lengths with
    eager work between, each replay equal to the eager calls; two graphs share a workspace."""
    B, H, Hk, D, page = 3, 4, 1, 128, 32
    steps = 40
    inputs = [P.randn(700 + s, B, 1, H + 2 * Hk, D) for s in range(steps)]

    def fresh():
        s = empty_store(B, 12, Hk, D, page, bits, F16)
        prompt = P.randn(77, B, 250, 2 * Hk, D)
        s.append(prompt[:, :, :Hk], prompt[:, :, Hk:], i32([0] * B), rope=P.ROPE)
        return s, i32([250, 17, 96])

    def calls(s, lens, after, x, ws, pages, qr, out):
        q = s.append(x[:, :, H:H + Hk], x[:, :, H + Hk:], lens, q=x[:, :, :H], q_out=qr, rope=P.ROPE, seq_lens_out=after)
        s.select_pages(q, after, 4, first=1, last=1, out=pages, workspace=ws)
        s.attention(q, after, pages=pages, out=out[0], workspace=ws)
        s.attention(q, after, out=out[1], workspace=ws)
        mugen_amd.seq_advance(lens, 1, 12 * page)

    def buffers(s):
        return (s.attention_workspace(1, H, n_select=4), torch.zeros((B, 1, Hk, 4), dtype=torch.int32, device=device),
                torch.zeros((B, 1, H, D), dtype=F16, device=device), torch.zeros((2, B, 1, H, D), dtype=F16, device=device))

    s0, lens0 = fresh()
    s1, lens1 = fresh()
    ws, pages, qr, out = buffers(s1)
    after = i32([0] * B)
    x = inputs[0].clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # warm up outside the capture, on copies of the state
        s2, lens2 = fresh()
        calls(s2, lens2, after.clone(), x, *buffers(s2))
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g in graphs:
        with torch.cuda.graph(g):
            calls(s1, lens1, after, x, ws, pages, qr, out)
    for s in range(steps):
        x.copy_(inputs[s])
        graphs[s % 2].replay()
        b = buffers(s0)
        b[0].fill_(0xff)  # (whatever the workspace holds)
        calls(s0, lens0, i32([0] * B), inputs[s], *b)
        torch.cuda.synchronize()
        assert torch.equal(lens0, lens1)
        for got, want in ((pages, b[1]), (qr, b[2]), (out, b[3])):
            assert torch.equal(got, want), f"step {s}"
    for n, t in tensors(s0).items():
        assert torch.equal(t.view(torch.uint8), tensors(s1)[n].view(torch.uint8)), n


def test_another_stream(device):
    """Calls go to torch's current stream."""
    s, K, V = P.make_store(91, [300, 40], 1, 64, 32, 8, F16)
    q = P.randn(92, 2, 1, 4, 64)
    want = s.attention(q, i32([300, 40]))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device=device)
        for _ in range(10):
            big = big @ big * 1e-2
        q2 = q + 0 * big[0, 0].half()  # ready only when the products are
        q2 = torch.where(q2.isnan(), q, q2)
        got = s.attention(q2, i32([300, 40]))
    side.synchronize()
    assert torch.equal(got, want)


def test_a_refused_append_starts_no_step(device):
    """A first append that is refused leaves the lengths alone: advance() has nothing to commit;
    no step is without tokens, and no page list without entries."""
    kv = mugen_amd.KVCachePaged(1, 2, 1, 64, 256, page_tokens=32, max_new=32, device=device)
    k = P.randn(38, 2, 5, 1, 64)
    kv.append(0, k, k)
    kv.advance()
    for bad in (k.to(BF16), k[:, :3], k[..., :32].contiguous()):
        with pytest.raises(ValueError):
            kv.append(0, k, bad)
        kv.advance()
        assert kv.seq_lens.tolist() == [5, 5] and kv.seq_lens_host.tolist() == [5, 5]
    with pytest.raises(ValueError):
        kv.append(0, k[:, :0], k[:, :0])
    s = kv.layers[0]
    with pytest.raises(ValueError):
        s.append(k[:, :0], k[:, :0], kv.seq_lens, seq_lens_out=torch.zeros_like(kv.seq_lens))
    with pytest.raises(ValueError):
        s.attention(k[:, :1].contiguous(), kv.seq_lens, pages=torch.zeros((2, 1, 1, 0), dtype=torch.int32, device=device))
    kv.append(0, k, k)
    kv.advance()
    assert kv.seq_lens.tolist() == [10, 10]


def test_a_cache_under_capture(device):
    """KVCachePaged: a step is not captured; attention captured alone follows the device's
    lengths on every replay."""
    kv = mugen_amd.KVCachePaged(1, 2, 2, 64, 1024, page_tokens=32, max_new=32, device=device)
    q = P.randn(40, 2, 1, 4, 64)
    x = P.randn(41, 2, 40, 2, 64)
    kv.append(0, x, x)
    kv.advance()
    ws = kv.layers[0].attention_workspace(1, 4)
    out = torch.zeros_like(q)
    kv.attention(0, q, out=out, workspace=ws)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kv.attention(0, q, out=out, workspace=ws)
        with pytest.raises(RuntimeError):
            kv.append(0, x, x)
    for s in range(3):
        y = P.randn(42 + s, 2, 300, 2, 64)
        kv.append(0, y, y, new_lens=[300, 7 + s])
        kv.advance()
        out.zero_()
        g.replay()
        want = kv.layers[0].attention(q, kv.seq_lens)
        torch.cuda.synchronize()
        assert torch.equal(out, want), f"replay {s}"
