"""64-bit restatements of the attention-half operators (momij_b200/attn.py), from
their formulas, and the inputs the tests share."""
from __future__ import annotations

import math

import torch

PAGE = 64
TD = {"bf16": torch.bfloat16, "f16": torch.float16}
HALF_ULP = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}  # of a value's leading bit


def pages_of(lens):
    return [max(1, -(-l // PAGE)) for l in lens]


def block_tables(lens, seed=0, spare=0, cols=None):
    """Scattered pages for these lengths: (table int32 [B, cols], number of pages)."""
    cols = cols or max(pages_of(lens)) + spare
    n = len(lens) * cols
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(n, generator=g).to(torch.int32).view(len(lens), cols), n


def random_pool(pages, H, D, seed=0):
    """Codes and scales as an append leaves them, and every page's values in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        x = torch.randn(pages, H, PAGE, D, generator=g) * (0.5 + torch.rand(pages, H, 1, 1, generator=g))
        s = x.abs().amax(dim=(2, 3)) / 127
        out += [(torch.round(x / s[:, :, None, None]) + 128).to(torch.uint8), s]
    return out[0], out[2].transpose(2, 3).contiguous(), out[1], out[3]


def values(k, v, ks, vs):
    """K and V of all pages in 64 bits, [pages, H, PAGE, D] both."""
    kk = (k.double() - 128) * ks.double()[:, :, None, None]
    vv = ((v.double() - 128) * vs.double()[:, :, None, None]).transpose(2, 3)
    return kk, vv


def attention(q, k, v, ks, vs, table, lens, cu, window=0, scale=None):
    """(out, bound of |v| weights, largest sum |q||k| scale) in 64 bits, [T, Hq, D]."""
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(T, Hq, D, dtype=torch.float64)
    mag = torch.zeros(T, Hq, D, dtype=torch.float64)
    big = 0.0
    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if n == 0 or length == 0:
            continue
        ids = table[b, :-(-length // PAGE)].long()
        kk, vv = values(k[ids], v[ids], ks[ids], vs[ids])
        kk = kk.permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :length]
        vv = vv.permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :length]
        for i in range(n):
            p = length - n + i
            lo = max(0, p - window + 1) if window else 0
            if p < 0:
                continue
            for h in range(Hq):
                x = q[cu[b] + i, h].double()
                key, val = kk[h // G, lo:p + 1], vv[h // G, lo:p + 1]
                w = torch.softmax(key @ x * scale, dim=0)
                out[cu[b] + i, h] = w @ val
                mag[cu[b] + i, h] = w @ val.abs()
                big = max(big, float((key.abs() @ x.abs()).max()) * abs(scale))
    return out, mag, big


def attention_bound(ref, mag, big, D, dtype):
    """|kernel - ref| by element: one rounding of the output; weights rounded to
    fp16 (2^-11 each, the sum's other side exact to fp32); scores as fp32 sums of D
    products of exact factors, four times for the codes' offset, twice for the exponent."""
    return HALF_ULP[dtype] * 2 * ref.abs() + (2.0 ** -11 + 8 * (D + 8) * 2.0 ** -24 * big + 2.0 ** -18) * mag + 1e-12


def rotate(y, cos, sin, interleaved):
    half = cos.shape[-1]
    if half == 0:
        return y
    a, b = (y[..., :2 * half:2], y[..., 1:2 * half:2]) if interleaved else (y[..., :half], y[..., half:2 * half])
    u, w = a * cos - b * sin, a * sin + b * cos
    t = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([t, y[..., 2 * half:]], -1)


def append(qkv, pool, table, lens, cu, Hq, qw, kw, eps, rope, interleaved):
    """The append in 64 bits on copies of ``pool`` (k, v, ks, vs): queries, and the
    pool with K and V as [pages, H, PAGE, D] values and scales.  Rows of a written
    page past the sequence's end hold nothing that may be read: NaN here."""
    k, v, ks, vs = pool
    Hkv, D = k.shape[1], k.shape[3]
    kk, vv = values(k, v, ks, vs)
    ks, vs = ks.double().clone(), vs.double().clone()
    x = qkv.double().view(qkv.shape[0], Hq + 2 * Hkv, D)
    q = torch.zeros(qkv.shape[0], Hq, D, dtype=torch.float64)

    def turned(y, w, pos):
        if w is not None:
            y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * w.double()
        if rope is None:
            return y
        half = rope.shape[1] // 2
        row = rope[pos].double()[:, None]
        return rotate(y, row[..., :half], row[..., half:], interleaved)

    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        past, rows = length - n, slice(cu[b], cu[b + 1])
        pos = torch.arange(past, length)
        q[rows] = turned(x[rows, :Hq], qw, pos)
        for new, store, scales in ((turned(x[rows, Hq:Hq + Hkv], kw, pos), kk, ks), (x[rows, Hq + Hkv:], vv, vs)):
            for blk in range(past // PAGE, -(-length // PAGE)):
                lo, hi = max(past, blk * PAGE), min(length, (blk + 1) * PAGE)
                page, off = int(table[b, blk]), lo - blk * PAGE
                part = new[lo - past:hi - past].transpose(0, 1)  # [Hkv, rows, D]
                s = part.abs().amax(dim=(1, 2)) / 127
                s = torch.where(s < 2.0 ** -64, torch.zeros_like(s), s)
                if off:
                    s = torch.maximum(s, scales[page])
                    held = torch.where(scales[page] > 0, 1.0, 0.0)[:, None, None] * store[page][:, :off]
                    d = torch.where(s > 0, s, torch.ones_like(s))[:, None, None]
                    store[page][:, :off] = torch.round(held / d) * s[:, None, None]
                d = torch.where(s > 0, s, torch.ones_like(s))[:, None, None]
                store[page][:, off:off + hi - lo] = torch.round(part / d) * s[:, None, None] * (s > 0)[:, None, None]
                store[page][:, off + hi - lo:] = math.nan
                scales[page] = s
    return q, kk, vv, ks, vs


def rope_table(n, rot, theta=10000.0):
    half = rot // 2
    a = torch.arange(n, dtype=torch.float64)[:, None] * theta ** (-torch.arange(half, dtype=torch.float64) / half)
    return torch.cat([a.cos(), a.sin()], 1).float()


def offsets(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def qmm4(x, w, s, b, gs):
    """(product, sum of magnitudes) in 64 bits."""
    code = torch.stack([(w.long() >> (4 * i)) & 15 for i in range(8)], dim=-1).view(w.shape[0], -1).double()
    sd, bd = s.double().repeat_interleave(gs, 1), b.double().repeat_interleave(gs, 1)
    xd = x.double()
    return xd @ (sd * code + bd).T, xd.abs() @ ((sd * code).abs() + bd.abs()).T


def logits(l, hist, cu, rep, pres, freq, ids, bias, cub, allowed):
    out, size = l.double().clone(), l.double().abs().clone()
    B, V = out.shape
    for r in range(B):
        count = torch.zeros(V, dtype=torch.float64)
        for t in hist[cu[r]:cu[r + 1]].tolist() if hist is not None else []:
            if 0 <= t < V:
                count[t] += 1
        said = count > 0
        if hist is not None:
            x = out[r]
            x = torch.where(said, torch.where(x > 0, x / float(rep[r]), x * float(rep[r])), x)
            size[r] = torch.maximum(size[r], x.abs()) + said * (float(freq[r]) * count + float(pres[r])).abs()
            out[r] = x - said * (float(freq[r]) * count + float(pres[r]))
        if ids is not None:
            last = {}
            for i in range(cub[r], cub[r + 1]):
                if 0 <= int(ids[i]) < V:
                    last[int(ids[i])] = float(bias[i])
            for t, v in last.items():
                out[r, t] += v
                size[r, t] += abs(v)
        if allowed is not None:
            bits = torch.stack([(allowed[r].long() >> i) & 1 for i in range(32)], 1).view(-1)[:V]
            out[r][bits == 0] = -math.inf
    return out, size
