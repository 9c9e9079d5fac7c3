"""The paged K/V cache operators over the range a user meets, for timing:

  append   rotate and append a step's (or a prompt's) K and V, rotate its queries
  decode   attention of one or a few new tokens per sequence over the pages
  sparse   page selection by a cheap score, then attention over the chosen pages
  prefill  attention of one sequence's prompt chunk over its pages

Layout of one layer (n_pages pages of P tokens, Hk kv heads, head_dim D):
  16-bit pages  k, v [n_pages][Hk][P][D]
  8-bit pages   k [n_pages][Hk][P][D], v [n_pages][Hk][P/32][D][32] in e4m3, and one power-of-two
                scale per (page, kv head), kept as its exponent + 127; only whole pages are held in
                8 bits, the tokens behind a sequence's last whole page in a 16-bit ring
                [n_seq][ring][Hk][D] (token t at slot t % ring)
  k_range       [n_pages][Hk][2][D]: minimum and maximum of each dim over a whole page's keys

`own` False computes them in elementary torch operations, True through mugen_amd.
"""
import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"
DT = {"f16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn
THETA = 1000000.0


def listed():
    return [
        # the smallest call: one token of one sequence
        dict(name="append_b1", op="append", bits=16, dtype="f16", page=64, heads=28, kv_heads=4, dim=128, batch=1,
             new=1, lo=700, hi=700, ranges=False, pad=False),
        # a serving step: 64 sequences, a few of them filling a page
        dict(name="append_b64_8bit", op="append", bits=8, dtype="bf16", page=64, heads=32, kv_heads=8, dim=128,
             batch=64, new=1, lo=512, hi=4095, ranges=True, pad=False),
        # a prompt chunk of odd length into 8-bit pages
        dict(name="append_prompt_n2047_8bit", op="append", bits=8, dtype="f16", page=64, heads=28, kv_heads=4, dim=128,
             batch=1, new=2047, lo=1001, hi=1001, ranges=True, pad=False),
        # single-sequence decode at a medium context
        dict(name="decode_b1_t4096", op="decode", bits=16, dtype="f16", page=64, heads=28, kv_heads=4, dim=128,
             batch=1, new=1, lo=4096, hi=4096, pad=False),
        # the ordinary serving step: 16 ragged sequences
        dict(name="decode_b16_ragged_8bit", op="decode", bits=8, dtype="f16", page=64, heads=28, kv_heads=4, dim=128,
             batch=16, new=1, lo=256, hi=8192, pad=False),
        # a large serving batch, small pages
        dict(name="decode_b64_ragged_8bit_bf16", op="decode", bits=8, dtype="bf16", page=32, heads=32, kv_heads=8,
             dim=128, batch=64, new=1, lo=512, hi=8191, pad=False),
        # speculative verify: five drafted tokens behind long contexts
        dict(name="verify_b4_q5_t32768_8bit", op="decode", bits=8, dtype="bf16", page=64, heads=28, kv_heads=4,
             dim=128, batch=4, new=5, lo=30000, hi=32768, pad=True),
        # one very long context, 64 of its 2048 pages per query
        dict(name="sparse_b1_t131072_8bit", op="sparse", bits=8, dtype="f16", page=64, heads=28, kv_heads=4, dim=128,
             batch=1, new=1, lo=131000, hi=131072, chosen=64, first=1, last=2, pad=False),
        # ragged serving batch with small heads and small pages, 16-bit
        dict(name="sparse_b16_d64", op="sparse", bits=16, dtype="bf16", page=32, heads=32, kv_heads=8, dim=64,
             batch=16, new=1, lo=1024, hi=32768, chosen=64, first=1, last=2, pad=False),
        # verify with selection: every drafted token picks its own pages
        dict(name="sparse_verify_b4_q4_8bit", op="sparse", bits=8, dtype="bf16", page=32, heads=32, kv_heads=8,
             dim=128, batch=4, new=4, lo=8000, hi=16384, chosen=100, first=1, last=4, pad=True),
        # a prompt chunk that continues a long context, 8-bit
        dict(name="prefill_n253_at7931_8bit", op="prefill", bits=8, dtype="f16", page=64, heads=28, kv_heads=4,
             dim=128, batch=3, new=253, lo=7931, hi=7931),
        # a prompt from its start, small heads (odd length), 16-bit
        dict(name="prefill_n2045_d64", op="prefill", bits=16, dtype="bf16", page=32, heads=32, kv_heads=8, dim=64,
             batch=2, new=2045, lo=0, hi=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "sparse", "prefill"])
    heads, kv_heads, dim = rng.choice([(28, 4, 128), (32, 8, 64), (32, 8, 128), (16, 8, 256), (14, 2, 64), (8, 8, 128),
                                       (32, 2, 128), (12, 4, 256)])
    c = dict(op=op, bits=rng.choice([8, 8, 16]), dtype=rng.choice(["f16", "bf16"]), page=rng.choice([32, 64, 128]),
             heads=heads, kv_heads=kv_heads, dim=dim)
    if op == "prefill":
        new = _log(rng, 17, 2048)
        start = rng.choice([0, _log(rng, 1, 8192 - new)])
        return dict(c, batch=rng.randint(1, 3), new=new, lo=start, hi=start)
    batch = _log(rng, 1, 64)
    new = rng.choice([1, 1, rng.randint(2, 8)])
    if op == "append" and rng.random() < 0.3:
        new = _log(rng, 9, max(9, 4096 // batch))
    rows = 64 * 8192 // (batch * kv_heads)  # tokens a sequence may hold: no pool above the largest listed one
    hi = _log(rng, new + 1, max(new + 1, min(rows, 131072)))
    lo = _log(rng, new, hi)
    c = dict(c, batch=batch, new=new, lo=lo, hi=hi, pad=batch > 1 and rng.random() < 0.3)
    if op == "append":
        c["ranges"] = rng.random() < 0.5
    if op == "sparse":
        c["first"], c["last"] = rng.randint(0, 2), rng.randint(1, 4)
        c["chosen"] = c["first"] + c["last"] + _log(rng, 1, 120)
    return c


def _exponent(amax):
    """The least e with amax <= 448 * 2^e, as the stored byte e + 127 (at least 1)."""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, (x - torch.where(m <= 0.875, 9, 8) + 127).clamp(1, 254), 1).to(torch.int32)


def _pow2(byte):
    return torch.ldexp(torch.ones((), device=byte.device), byte.to(torch.int32) - 127)


def _v_in(v):  # [.., P, D] -> [.., P/32, D, 32]
    return v.unflatten(-2, (-1, 32)).transpose(-1, -2)


def _v_out(v):  # [.., P/32, D, 32] -> [.., P, D]
    return v.transpose(-1, -2).flatten(-3, -2)


def _to8(x):
    """x [.., P, D] in e4m3 with one exponent for the last two axes."""
    byte = _exponent(x.abs().amax((-1, -2)).float())
    return (x.float() / _pow2(byte)[..., None, None]).to(E4M3), byte.to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)
    op, bits, dt, P = case["op"], case["bits"], DT[case["dtype"]], case["page"]
    B, L, H, Hk, D = case["batch"], case["new"], case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=dt)

    before = [rng.randint(case["lo"], case["hi"]) for _ in range(B)]
    if op in ("decode", "sparse"):  # lo..hi count the new tokens too
        before = [max(0, t - L) for t in before]
    new = [L] * B
    if case.get("pad"):
        new = [rng.randint(1, L) for _ in range(B)]
        if B > 2:
            new[rng.randrange(B)] = 0  # a slot without a token in this step
    room = max(before) + L
    max_seq = -(-room // P) * P
    count = [-(-(t + L) // P) for t in before]
    # an append returns its pools whole: the same size whatever the seed's lengths
    n_pages = (B * -(-(case["hi"] + L) // P) if op == "append" else sum(count)) + 2
    table = torch.full((B, max_seq // P), -1, dtype=torch.int32)
    ids, at = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32), 0
    for b, c in enumerate(count):
        table[b, :c] = ids[at:at + c]
        at += c
    s = dict(case=case, table=table.to(DEV), max_seq=max_seq)
    s["before"] = torch.tensor(before, dtype=torch.int32, device=DEV)
    s["after_host"] = np.array([t + n for t, n in zip(before, new)], np.int32)
    s["after"] = torch.from_numpy(s["after_host"]).to(DEV)
    s["new"] = torch.tensor(new, dtype=torch.int32, device=DEV) if case.get("pad") else None
    # keys of one page resemble each other, as a passage's keys do
    k = normal(n_pages, Hk, P, D).mul_(0.8).add_(normal(n_pages, Hk, 1, D), alpha=0.6)
    v = normal(n_pages, Hk, P, D)
    s["k_exp"] = s["v_exp"] = s["tail_k"] = s["tail_v"] = s["ranges"] = None
    if bits == 8:
        k8, s["k_exp"] = _to8(k)
        v8, s["v_exp"] = _to8(v)
        k = (k8.float() * _pow2(s["k_exp"])[..., None, None]).to(dt)
        s["k"], s["v"] = k8.view(torch.uint8), _v_in(v8.view(torch.uint8)).contiguous()
        ring = 1 << (P + min(L, 64) - 1).bit_length()
        s["tail_k"], s["tail_v"] = normal(B, ring, Hk, D), normal(B, ring, Hk, D)
    else:
        s["k"], s["v"] = k, v
    if op == "sparse" or case.get("ranges"):
        s["ranges"] = torch.stack((k.amin(2), k.amax(2)), 2)
    if op == "append":
        qkv = normal(B, L, H + 2 * Hk, D)  # the fused projection's output
        s["q"], s["k_new"], s["v_new"] = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
        s["q_out"] = torch.zeros((B, L, H, D), dtype=dt, device=DEV)
    elif op == "prefill":
        s["seq"] = rng.randrange(B)
        s["start"], s["q"] = before[s["seq"]], normal(L, H, D)
    else:
        s["q"] = normal(B, L, H, D)
        s["out"] = torch.zeros((B, L, H, D), dtype=dt, device=DEV)
    if op == "sparse":
        s["pages"] = torch.full((B, L, Hk, case["chosen"]), -1, dtype=torch.int32, device=DEV)
    if own:
        import mugen_amd
        s["store"] = mugen_amd.PagedStore(s["k"], s["v"], s["table"], max_seq, k_exp=s["k_exp"], v_exp=s["v_exp"],
                                          tail_k=s["tail_k"], tail_v=s["tail_v"], k_range=s["ranges"])
        if op in ("decode", "sparse"):
            s["ws"] = s["store"].attention_workspace(L, H, n_select=case.get("chosen", 0))
        elif op == "prefill":
            s["ws"] = s["store"].prefill_workspace(L, H, s["start"])
    return s


def run(s):
    return {"append": _append, "decode": _decode, "sparse": _sparse, "prefill": _prefill}[s["case"]["op"]](s)


# ------------------------------------------------------------------ append

def _rotate(x, pos):
    """x [B, L, heads, D], pairs (i, i + D/2), rotated by pos [B, L] * THETA^(-2i/D)."""
    half = x.shape[-1] // 2
    freq = THETA ** (torch.arange(half, dtype=torch.float64, device=DEV) / -half)
    a = pos.double()[:, :, None, None] * freq
    cos, sin = a.cos().float(), a.sin().float()
    x0, x1 = x[..., :half].float(), x[..., half:].float()
    return torch.cat((x0 * cos - x1 * sin, x1 * cos + x0 * sin), -1).to(x.dtype)


def _append(s):
    c = s["case"]
    if own:
        s["store"].append(s["k_new"], s["v_new"], s["before"], new_lens=s["new"], q=s["q"], q_out=s["q_out"],
                          rope=(THETA, 1.0, 0))
    else:
        _append_plain(s)
    out = {"q": s["q_out"], "ranges": s["ranges"], "tail_k": s["tail_k"], "tail_v": s["tail_v"], "k_exp": s["k_exp"],
           "v_exp": s["v_exp"], "k": s["k"], "v": s["v"]}
    if c["bits"] == 8:
        out["k"], out["v"] = s["k"].view(E4M3), s["v"].view(E4M3)
    return {n: x for n, x in out.items() if x is not None}


def _append_plain(s):
    c = s["case"]
    B, L, P, bits = c["batch"], c["new"], c["page"], c["bits"]
    T = s["before"].long()
    n = s["new"].long() if s["new"] is not None else torch.full_like(T, L)
    pos = T[:, None] + torch.arange(L, device=DEV)
    live = (pos < (T + n)[:, None]) & (pos < s["max_seq"])
    k, v = _rotate(s["k_new"], pos), s["v_new"]
    s["q_out"].copy_(torch.where(live[:, :, None, None], _rotate(s["q"], pos), s["q_out"]))
    b = torch.arange(B, device=DEV)[:, None]
    table = s["table"].long()
    if bits == 16:
        phys, slot = table[b, (pos // P).clamp(max=table.shape[1] - 1)][live], (pos % P)[live]
        s["k"][phys, :, slot], s["v"][phys, :, slot] = k[live], v[live]
        if s["ranges"] is None:
            return
    # the pages that these tokens fill: [B, J]
    page = T[:, None] // P + torch.arange((P - 1 + L) // P, device=DEV)
    full = (page + 1) * P <= (T + n)[:, None]
    full &= page * P + P > T[:, None]
    phys = table[b, page.clamp(max=table.shape[1] - 1)]
    if bits == 16:
        rows = s["k"][phys[full]]
    else:
        t = (page[..., None] * P + torch.arange(P, device=DEV))  # [B, J, P]
        b3, ring = b[..., None], s["tail_k"].shape[1]
        held, at = (t < T[:, None, None])[..., None, None], (t - T[:, None, None]).clamp(0, L - 1)
        for fresh, tail, pool, exp in ((k, "tail_k", "k", "k_exp"), (v, "tail_v", "v", "v_exp")):
            x = torch.where(held, s[tail][b3, t % ring], fresh[b3, at]).transpose(2, 3)[full]  # [F, Hk, P, D]
            x8, byte = _to8(x)
            if pool == "k":
                rows = (x8.float() * _pow2(byte)[..., None, None]).to(x.dtype)
            x8 = x8.view(torch.uint8)
            s[pool][phys[full]] = x8 if pool == "k" else _v_in(x8)
            s[exp][phys[full]] = byte
        last = live & (pos >= (T + n)[:, None] - ring)
        at = (torch.where(last)[0], (pos % ring)[last])
        s["tail_k"][at], s["tail_v"][at] = k[last], v[last]
    if s["ranges"] is not None:
        s["ranges"][phys[full]] = torch.stack((rows.amin(2), rows.amax(2)), 2)


# ------------------------------------------------------------------ attention

def _held(s, phys, lp, b):
    """K and V (float) of physical pages `phys` [.., Hk] (logical pages lp, sequences b, heads the last
    axis): [.., Hk, P, D] each, the page behind the last whole one from the 16-bit ring."""
    c = s["case"]
    P, h = c["page"], torch.arange(c["kv_heads"], device=DEV)
    k, v = s["k"][phys, h], s["v"][phys, h]
    if c["bits"] == 16:
        return k.float(), v.float()
    k = k.view(E4M3).float() * _pow2(s["k_exp"][phys, h])[..., None, None]
    v = _v_out(v.view(E4M3).float()) * _pow2(s["v_exp"][phys, h])[..., None, None]
    open_ = (lp == (s["after"].long() // P)[b])[..., None, None]
    b, ring = torch.as_tensor(b, device=DEV), s["tail_k"].shape[1]
    slot = (s["after"].long() // P * P)[b][..., None] % ring + torch.arange(P, device=DEV)  # ring % P == 0
    tk, tv = s["tail_k"][b[..., None], slot % ring, h[:, None]], s["tail_v"][b[..., None], slot % ring, h[:, None]]
    return torch.where(open_, tk.float(), k), torch.where(open_, tv.float(), v)


def _softmax_v(x, seen, v):
    """softmax over the last axis of x where seen, times v; rows that see nothing are zero."""
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, 1.0)


def _limits(s):
    """How many tokens each query sees [B, L], and which queries there are."""
    c = s["case"]
    i = torch.arange(c["new"], device=DEV)
    n = s["new"].long() if s["new"] is not None else torch.full_like(s["after"], c["new"]).long()
    return (s["after"].long() - n)[:, None] + i + 1, i < n[:, None]


def _decode(s):
    c = s["case"]
    if own:
        return s["store"].attention(s["q"], s["after"], q_lens=s["new"], out=s["out"], workspace=s["ws"],
                                    seq_lens_host=s["after_host"])
    B, L, H, Hk, D, P = c["batch"], c["new"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    N = s["table"].shape[1]
    lp = torch.arange(N, device=DEV)[None, :, None].expand(B, N, Hk)
    b = torch.arange(B, device=DEV)[:, None, None].expand(B, N, Hk)
    k, v = _held(s, s["table"].long().clamp(min=0)[:, :, None].expand(B, N, Hk), lp, b)
    k, v = k.transpose(1, 2).reshape(B, Hk, N * P, D), v.transpose(1, 2).reshape(B, Hk, N * P, D)
    q = s["q"].float().view(B, L, Hk, H // Hk, D).transpose(1, 2).reshape(B, Hk, -1, D)
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(1 / math.sqrt(D))
    limit, live = _limits(s)
    t = torch.arange(N * P, device=DEV)
    v = torch.where((t < s["after"][:, None])[:, None, :, None], v, 0.0)
    o = _softmax_v(x.view(B, Hk, L, H // Hk, -1), (t < limit[..., None])[:, None, :, None], v[:, :, None])
    o = o.permute(0, 2, 1, 3, 4).reshape(B, L, H, D)
    s["out"].copy_(torch.where(live[..., None, None], o.to(s["out"].dtype), s["out"]))
    return s["out"]


def _sparse(s):
    c = s["case"]
    if own:
        s["store"].select_pages(s["q"], s["after"], c["chosen"], first=c["first"], last=c["last"], q_lens=s["new"],
                                out=s["pages"], workspace=s["ws"])
        o = s["store"].attention(s["q"], s["after"], q_lens=s["new"], pages=s["pages"], out=s["out"], workspace=s["ws"])
        return {"pages": s["pages"], "out": o}
    B, L, H, Hk, D, P = c["batch"], c["new"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    N = s["table"].shape[1]
    limit, live = _limits(s)
    # the score, in 64 bits: values next to the border decide which page is read
    q = s["q"].double().view(B, L, Hk, H // Hk, D)
    q = torch.cat((q.clamp(max=0).sum(3), q.clamp(min=0).sum(3)), -1)  # meets (minimum, maximum)
    r = s["ranges"][s["table"].long().clamp(min=0)].double().flatten(-2)  # [B, N, Hk, 2D]
    score = torch.matmul(q.transpose(1, 2), r.permute(0, 2, 3, 1)).transpose(1, 2)  # [B, L, Hk, N]
    pages = ((limit + P - 1) // P)[..., None, None]
    lp = torch.arange(N, device=DEV)
    score = torch.where((lp < c["first"]) | (lp >= pages - c["last"]), math.inf, score)
    score = torch.where(lp < pages, score, -math.inf)
    pick = min(c["chosen"], N)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :pick]
    order = torch.where(torch.arange(pick, device=DEV) < pages, order, N).sort(-1).values
    chosen = torch.full_like(s["pages"], -1)
    chosen[..., :pick] = torch.where(order < N, order, -1).to(torch.int32)
    s["pages"].copy_(torch.where(live[..., None, None], chosen, s["pages"]))
    # attention over the chosen pages [B, L, C, Hk]
    lp = order.transpose(2, 3)
    b = torch.arange(B, device=DEV)[:, None, None, None].expand(lp.shape)
    phys = s["table"].long()[b, lp.clamp(max=N - 1)].clamp(min=0)
    k, v = _held(s, phys, lp, b)
    k, v = k.transpose(2, 3).reshape(B, L, Hk, pick * P, D), v.transpose(2, 3).reshape(B, L, Hk, pick * P, D)
    t = (order[..., None] * P + torch.arange(P, device=DEV)).flatten(-2)  # [B, L, Hk, C * P]
    seen = (t < limit[..., None, None]) & (order < N).repeat_interleave(P, -1)
    v = torch.where(seen[..., None], v, 0.0)
    x = torch.matmul(s["q"].float().view(B, L, Hk, H // Hk, D), k.transpose(-1, -2)).mul_(1 / math.sqrt(D))
    o = _softmax_v(x, seen[..., None, :], v).reshape(B, L, H, D)
    s["out"].copy_(torch.where(live[..., None, None], o.to(s["out"].dtype), s["out"]))
    return {"pages": s["pages"], "out": s["out"]}


def _prefill(s):
    c = s["case"]
    if own:
        return s["store"].prefill(s["q"], s["seq"], s["start"], workspace=s["ws"])
    L, H, Hk, D, P = c["new"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    T = s["start"] + L
    N = -(-T // P)
    lp = torch.arange(N, device=DEV)[:, None].expand(N, Hk)
    k, v = _held(s, s["table"][s["seq"], :N].long()[:, None].expand(N, Hk), lp, torch.full_like(lp, s["seq"]))
    k, v = k.transpose(0, 1).reshape(Hk, N * P, D)[:, :T], v.transpose(0, 1).reshape(Hk, N * P, D)[:, :T]
    q = s["q"].float().view(L, Hk, H // Hk, D).permute(1, 2, 0, 3)
    x = torch.matmul(q, k.transpose(-1, -2)[:, None]).mul_(1 / math.sqrt(D))  # [Hk, G, L, T]
    seen = torch.arange(T, device=DEV) <= s["start"] + torch.arange(L, device=DEV)[:, None]
    o = _softmax_v(x, seen, v[:, None])
    return o.permute(2, 0, 1, 3).reshape(L, H, D).to(s["q"].dtype)


# ------------------------------------------------------------------ definition

def _sequence(s, b, T):
    """Sequence b's keys and values [T, Hk, D] in 64 bits."""
    c = s["case"]
    P, Hk, D = c["page"], c["kv_heads"], c["dim"]
    ks, vs = [], []
    for p in range(-(-T // P)):
        if c["bits"] == 8 and (p + 1) * P > int(s["after"][b]):
            ring = s["tail_k"].shape[1]
            at = (p * P + torch.arange(P, device=DEV)) % ring
            ks.append(s["tail_k"][b, at].double())
            vs.append(s["tail_v"][b, at].double())
            continue
        i = int(s["table"][b, p])
        k, v = s["k"][i], s["v"][i]
        if c["bits"] == 8:
            v = v.view(Hk, P // 32, D, 32).permute(0, 1, 3, 2).reshape(Hk, P, D)
            k = k.view(E4M3).double() * 2.0 ** (s["k_exp"][i].double() - 127)[:, None, None]
            v = v.contiguous().view(E4M3).double() * 2.0 ** (s["v_exp"][i].double() - 127)[:, None, None]
        ks.append(k.double().transpose(0, 1))
        vs.append(v.double().transpose(0, 1))
    return torch.cat(ks)[:T], torch.cat(vs)[:T]


def _attend(q, k, v, keep=None):
    """q [H, D] over k, v [T, Hk, D]; keep [Hk, T]: the tokens that are read."""
    H, D = q.shape
    G = H // k.shape[1]
    x = (k.transpose(0, 1) @ q.double().view(-1, G, D).transpose(1, 2)) / math.sqrt(D)  # [Hk, T, G]
    if keep is not None:
        x = x.masked_fill(~keep[..., None], -math.inf)
    w = torch.softmax(x, 1)
    return (w.transpose(1, 2) @ v.transpose(0, 1)).reshape(H, D)


def _exact_append(s):
    c = s["case"]
    P, D = c["page"], c["dim"]
    half = D // 2
    freq = torch.tensor([THETA ** (-i / half) for i in range(half)], dtype=torch.float64, device=DEV)

    def turn(x, t):
        z = torch.complex(x[..., :half].double(), x[..., half:].double()) * torch.polar(torch.ones_like(freq), t * freq)
        return torch.cat((z.real, z.imag), -1)

    q = s["q_out"].double()
    tails = {"k": s["tail_k"], "v": s["tail_v"]}
    # 8-bit pages and the ranges hold values that were rounded on their way: no exact value
    pools = {"k": None, "v": None}
    if c["bits"] == 16:
        pools = {"k": s["k"].double(), "v": s["v"].double()}
    else:
        tails = {n: x.double() for n, x in tails.items()}
    for b in range(c["batch"]):
        T = int(s["before"][b])
        n = int(s["new"][b]) if s["new"] is not None else c["new"]
        for j in range(n):
            t = T + j
            q[b, j] = turn(s["q"][b, j], t)
            for m, x in (("k", turn(s["k_new"][b, j], t)), ("v", s["v_new"][b, j].double())):
                if c["bits"] == 16:
                    pools[m][int(s["table"][b, t // P]), :, t % P] = x
                elif t >= T + n - tails[m].shape[1]:
                    tails[m][b, t % tails[m].shape[1]] = x
    out = {"q": q, "k": pools["k"], "v": pools["v"]}
    for name, x in (("ranges", s["ranges"]), ("k_exp", s["k_exp"]), ("v_exp", s["v_exp"])):
        if x is not None:
            out[name] = None
    if c["bits"] == 8:
        out["tail_k"], out["tail_v"] = tails["k"], tails["v"]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op, B, L, P = case["op"], case["batch"], case["new"], case["page"]
    if op == "append":
        return _exact_append(s)
    if op == "prefill":
        T = s["start"] + L
        k, v = _sequence(s, s["seq"], T)
        return torch.stack([_attend(s["q"][i], k[:s["start"] + i + 1], v[:s["start"] + i + 1]) for i in range(L)])
    out = s["out"].double()
    for b in range(B):
        T = int(s["after_host"][b])
        n = int(s["new"][b]) if s["new"] is not None else L
        if n == 0:
            continue
        k, v = _sequence(s, b, T)
        for i in range(n):
            t = T - n + i + 1
            keep = None
            if op == "sparse":
                N, Hk, D = -(-t // P), case["kv_heads"], case["dim"]
                r = s["ranges"][s["table"][b, :N].long()].double()  # [N, Hk, 2, D]
                q = s["q"][b, i].double().view(Hk, -1, D)
                bound = torch.maximum(q[None] * r[:, :, 0, None], q[None] * r[:, :, 1, None]).sum((-1, -2))  # [N, Hk]
                must = torch.arange(N, device=DEV)
                bound[(must < case["first"]) | (must >= N - case["last"])] = math.inf
                rank = torch.argsort(bound, dim=0, descending=True, stable=True)[:case["chosen"]]
                keep = torch.zeros((N, Hk), dtype=torch.bool, device=DEV).scatter_(0, rank, True)
                keep = keep.repeat_interleave(P, 0)[:t].T
            out[b, i] = _attend(s["q"][b, i], k[:t], v[:t], keep)
    return {"pages": None, "out": out} if op == "sparse" else out


def work(case):
    """Bytes and operations of one pass, from the mean length."""
    op, bits, P = case["op"], case["bits"], case["page"]
    B, L, H, Hk, D = case["batch"], case["new"], case["heads"], case["kv_heads"], case["dim"]
    T = (case["lo"] + case["hi"]) / 2
    token = 2 * Hk * D * bits / 8 + (2 * Hk / P if bits == 8 else 0)  # K and V of one token
    if op == "append":
        move = B * L * (2 * H * D * 2 + 2 * Hk * D * 2 + 2 * Hk * D * 2)  # q, k, v in; q and the 16-bit rows out
        if bits == 8:
            move += B * L * token
        return {"bytes": move, "flops": B * L * (H + Hk) * D * 3}
    if op == "prefill":
        return {"bytes": (T + L) * token + 4 * L * H * D, "flops": 4 * H * D * (L * T + L * (L + 1) / 2)}
    if op == "decode":
        return {"bytes": B * T * token + 4 * B * L * H * D, "flops": 4 * B * L * H * D * T}
    N = T / P
    read = min(case["chosen"], N) * P
    return {"bytes": B * (N * Hk * 2 * D * 2 + L * read * token + 4 * L * H * D + 4 * L * Hk * case["chosen"]),
            "flops": B * L * (Hk * N * 4 * D + 4 * H * D * read)}
