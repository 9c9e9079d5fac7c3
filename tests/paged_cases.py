"""Inputs and plain 64-bit implementations for the paged cache's tests."""
import math

import torch

E4M3 = torch.float8_e4m3fn
STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step, relative
ROPE = (500000.0, 1.0, 0)


def say(*a):
    print(*a, flush=True)


def randn(seed, *shape, dtype=torch.float16, dev="cuda"):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


def freqs(rope, dim):
    """Rotation per position of each pair, YaRN for factor > 1 (64 bits)."""
    theta, factor, ctx = rope
    out = []
    for i in range(dim // 2):
        f = theta ** (-2.0 * i / dim)
        if factor > 1:
            span = 2 * math.log(theta)
            low = max(0.0, math.floor(dim * math.log(ctx / (32 * 2 * math.pi)) / span))
            high = min(dim / 2 - 1, math.ceil(dim * math.log(ctx / (2 * math.pi)) / span))
            ramp = 0.0 if i < low else 1.0 if i > high else min(1.0, (i - low) / max(0.001, high - low))
            f = f * (1 - ramp) + f / factor * ramp
        out.append(f)
    return torch.tensor(out, dtype=torch.float64)


def rotated(x, pos, rope, dim):
    """x [.., heads, D] at positions pos [..], in 64 bits on the CPU."""
    x = x.double().cpu()
    a = pos.double().cpu()[..., None, None] * freqs(rope, dim)
    x0, x1 = x[..., :dim // 2], x[..., dim // 2:dim]
    return torch.cat((x0 * a.cos() - x1 * a.sin(), x1 * a.cos() + x0 * a.sin(), x[..., dim:]), -1)


def quantised(rows):
    """rows [P, D] (16-bit): E4M3 codes (uint8), exponent byte, and the values the
    codes stand for (64 bits); not finite -> NaN."""
    x = rows.double().cpu()
    amax = torch.where(x.isfinite(), x.abs(), 0.0).max().item()
    byte = 1
    if amax > 0:
        e = math.ceil(math.log2(amax / 448)) - 1
        while amax > 448 * 2.0 ** e:
            e += 1
        byte = min(max(e + 127, 1), 254)
    scale = 2.0 ** (byte - 127)
    y = torch.where(x.isfinite(), x / scale, math.nan).float()
    c = y.to(E4M3)
    codes = torch.where(y.isnan(), 0x7f, c.view(torch.uint8))
    return codes, byte, codes.view(E4M3).double() * scale


def make_store(seed, lens, Hk, D, P, bits, dtype, *, ring=None, max_seq=None, spare=3, junk=True, ranges=False,
               dev="cuda"):
    """A store holding random K / V of `lens` tokens per sequence, pages scattered;
    whatever no token owns is NaN (junk).  Returns (PagedStore, K, V): the
    values a query attends to, [T, Hk, D] in 64 bits per sequence."""
    import mugen_amd
    B = len(lens)
    max_seq = max_seq or max(1, -(-(max(lens) + 1) // P) * P)
    width = -(-max_seq // P)
    count = [-(-t // P) for t in lens]
    n_pages = sum(count) + spare
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(n_pages, generator=g).to(torch.int32)
    table = torch.full((B, width), -7, dtype=torch.int32)
    nan = math.nan if junk else 0.0
    k16, v16 = (torch.full((n_pages, Hk, P, D), nan, dtype=dtype) for _ in range(2))
    k8 = torch.full((n_pages, Hk, P, D), 0x7f if junk else 0, dtype=torch.uint8)
    v8 = torch.full((n_pages, Hk, P // 32, D, 32), 0x7f if junk else 0, dtype=torch.uint8)
    ke, ve = (torch.full((n_pages, Hk), 254 if junk else 1, dtype=torch.uint8) for _ in range(2))
    ring = ring or 2 * P
    tk, tv = (torch.full((B, ring, Hk, D), nan, dtype=dtype) for _ in range(2))
    kr = torch.full((n_pages, Hk, 2, D), nan, dtype=dtype)
    K, V, at = [], [], 0
    for b, T in enumerate(lens):
        k = (torch.randn((T, Hk, D), generator=g) * 0.8).to(dtype)
        v = torch.randn((T, Hk, D), generator=g).to(dtype)
        kd, vd = k.double(), v.double()
        for p in range(count[b]):
            i = int(ids[at])
            at += 1
            table[b, p] = i
            n = min(P, T - p * P)
            sl = slice(p * P, p * P + n)
            k16[i, :, :n], v16[i, :, :n] = k[sl].transpose(0, 1), v[sl].transpose(0, 1)
            if n < P:
                at_ring = torch.arange(p * P, p * P + n) % ring
                tk[b, at_ring], tv[b, at_ring] = k[sl], v[sl]
                continue
            for h in range(Hk):
                if bits == 8:
                    c, ke[i, h], kd[sl, h] = quantised(k[sl, h])
                    k8[i, h] = c
                    c, ve[i, h], vd[sl, h] = quantised(v[sl, h])
                    v8[i, h] = c.view(P // 32, 32, D).transpose(1, 2)
                kr[i, h, 0], kr[i, h, 1] = kd[sl, h].amin(0).to(dtype), kd[sl, h].amax(0).to(dtype)
        K.append(kd)
        V.append(vd)
    up = [t.to(dev) for t in (k8, v8, table, ke, ve, tk, tv)] if bits == 8 else [t.to(dev) for t in (k16, v16, table)]
    kw = dict(zip(("k_exp", "v_exp", "tail_k", "tail_v"), up[3:]))
    if ranges:
        kw["k_range"] = kr.to(dev)
    return mugen_amd.PagedStore(up[0], up[1], up[2], max_seq, **kw), K, V


def attend(q, K, V, scale=None, keep=None, tol_dtype=None):
    """One query q [H, D] over K, V [T, Hk, D] (64 bits): (output, bound of the
    kernel's error).  The bound: weights rounded to tol_dtype's product terms
    (fp16 2^-11, and 2^-25 absolute below its normal range; bf16 in two terms
    2^-16), scores summed in fp32 over D terms (each product and sum 2^-24, of
    the sum of magnitudes) plus 2^-20 for exp2 and the sums, the merge of the splits
    in fp32; and the output's own rounding."""
    H, D = q.shape
    T, Hk = K.shape[0], K.shape[1] if K.dim() > 1 else 1
    scale = scale or 1 / math.sqrt(D)
    G = H // Hk
    out, tol = torch.zeros(H, D, dtype=torch.float64), torch.zeros(H, D, dtype=torch.float64)
    q = q.double().cpu()
    for h in range(H):
        j = h // G
        k, v = K[:, j], V[:, j]
        if keep is not None:
            k, v = k[keep[j]], v[keep[j]]
        if k.shape[0] == 0:
            continue
        w = torch.softmax(k @ q[h] * scale, 0)
        out[h] = w @ v
        ds = ((k.abs() @ q[h].abs()).max() * scale * (D + 4) * 2.0 ** -24).item()
        p, tiny = (2.0 ** -11, 2.0 ** -25) if tol_dtype == torch.float16 else (2.0 ** -16, 0.0)
        tol[h] = (w @ v.abs()) * (p + 2 * ds + 2.0 ** -20) + v.abs().sum(0) * tiny
    return out, tol


def check(got, want, tol, dtype, what):
    """|got - want| <= tol + half a step of dtype (and of its smallest number)."""
    got = got.double().cpu()
    bound = tol * (1 + STEP[dtype]) + want.abs() * STEP[dtype] + torch.finfo(dtype).smallest_normal * STEP[dtype]
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, worst "
                           f"{((got - want).abs() - bound)[bad].max().item():.3g} over, first {bad.nonzero()[0].tolist()}")


def choose(q, lo, hi, pages, n_select, first, last):
    """Pages for one query q [G, D] of a kv head, from lo, hi [N, D] (64 bits):
    the ascending list."""
    if pages <= n_select:
        return list(range(pages))
    q = q.double()
    s = torch.maximum(q[None] * lo[:, None], q[None] * hi[:, None]).sum((-1, -2))
    cand = list(range(first, pages - last))
    key = [math.inf if math.isnan(s[p].item()) else s[p].item() for p in range(pages)]
    nan = [math.isnan(s[p].item()) for p in range(pages)]
    cand.sort(key=lambda p: (not nan[p], -key[p], p))
    return sorted(list(range(first)) + list(range(pages - last, pages)) + cand[:n_select - first - last])
