"""Cases of the attention-half and output-head operators, for timing and for comparison.

Four operators of a decode or prefill step are covered:

* ``append``  -- head-wise RMS norm of queries and keys, rotation by position, and the
  append of keys and values to the 8-bit paged cache (one scale per page and head);
* ``attend``  -- causal attention of new tokens over that cache (grouped heads, sliding window);
* ``qmm4``    -- product of a few tokens with a 4-bit weight matrix with group scales;
* ``logits``  -- repetition, presence and frequency penalties, biases and grammar masks.

``run`` computes a case in its plain form (elementary torch operations in 32 bits), or, where
``own`` is true, with the calls of :mod:`momij_b200.attn` and :mod:`momij_b200.head`.
``exact`` computes the same outputs in 64 bits from the operator's definition.
"""
from __future__ import annotations

import math

import torch

own = False

PAGE = 64  # tokens of a cache page, which shares one scale per head for K and one for V
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---- cases ---------------------------------------------------------------------

def listed():
    return [
        # one sequence, one token: a layer's append in interactive decoding
        dict(name="append decode 1", op="append", B=1, n=1, Hq=16, Hkv=4, D=128, rot=64, past=700, dtype="bf16", interleaved=False),
        # verification of 7 drafted tokens for 24 sequences, pages entered in their middle
        dict(name="append verify 24x8", op="append", B=24, n=8, Hq=16, Hkv=4, D=128, rot=128, past=5000, dtype="f16", interleaved=False),
        # a prompt's chunk, starting inside a page
        dict(name="append prefill 4099", op="append", B=1, n=4099, Hq=16, Hkv=4, D=128, rot=64, past=1001, dtype="bf16", interleaved=True),
        # one sequence with a short context: latency
        dict(name="attend decode 1x701", op="attend", B=1, n=1, Hq=16, Hkv=4, D=128, len=701, window=0, dtype="bf16"),
        # a batch of ragged long contexts, one token each: the cache's bandwidth
        dict(name="attend decode 32x16384", op="attend", B=32, n=1, Hq=16, Hkv=4, D=128, len=16384, window=0, dtype="bf16"),
        # verification over a sliding window, heads of 64
        dict(name="attend verify 24x8 window", op="attend", B=24, n=8, Hq=32, Hkv=4, D=64, len=5003, window=512, dtype="f16"),
        # a prompt's chunk behind a context
        dict(name="attend prefill 2048 of 8192", op="attend", B=1, n=2048, Hq=16, Hkv=4, D=128, len=8192, window=0, dtype="bf16"),
        # a square projection for one token
        dict(name="qmm4 1x2048x2048", op="qmm4", M=1, N=2048, K=2048, gs=64, dtype="bf16"),
        # the vocabulary's projection for one token
        dict(name="qmm4 1x151936x2048", op="qmm4", M=1, N=151936, K=2048, gs=64, dtype="bf16"),
        # the vocabulary's projection for a verified draft
        dict(name="qmm4 9x151936x2048", op="qmm4", M=9, N=151936, K=2048, gs=128, dtype="f16"),
        # one sequence's logits with penalties over its history and a grammar mask
        dict(name="logits 1x151936", op="logits", B=1, V=151936, history=700, biases=16, mask=True, dtype="bf16"),
        # a batch of sequences with longer histories and many biases
        dict(name="logits 48x151936", op="logits", B=48, V=151936, history=6000, biases=300, mask=True, dtype="f16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges, no larger than the largest of its operator."""
    op = rng.choice(("append", "attend", "attend", "qmm4", "logits"))
    top = [work(c) for c in listed() if c["op"] == op]
    most = {k: max(w[k] for w in top) for k in ("bytes", "flops")}
    while True:
        dtype = rng.choice(("bf16", "f16"))
        if op == "append":
            Hkv = rng.choice((1, 2, 4, 8))
            D = rng.choice((64, 128))
            n = rng.choice((1, rng.randint(2, 9), _log_int(rng, 10, 4099)))
            c = dict(op=op, B=_log_int(rng, 1, 64), n=n, Hq=Hkv * rng.choice((1, 2, 3, 4, 7, 8)), Hkv=Hkv, D=D,
                     rot=rng.choice((D, D // 2, 32)), past=rng.choice((0, _log_int(rng, 1, 16000))), dtype=dtype,
                     interleaved=rng.choice((False, True)))
        elif op == "attend":
            Hkv = rng.choice((1, 2, 4, 8))
            n = rng.choice((1, 1, rng.randint(2, 9), _log_int(rng, 10, 2048)))
            c = dict(op=op, B=_log_int(rng, 1, 64), n=n, Hq=Hkv * rng.choice((1, 2, 3, 4, 7, 8)), Hkv=Hkv,
                     D=rng.choice((64, 128)), len=max(n, _log_int(rng, 1, 32768)),
                     window=rng.choice((0, 0, 512, _log_int(rng, 1, 4096))), dtype=dtype)
            if c["B"] * c["len"] * c["Hq"] * c["n"] > 1 << 30:  # the plain form's scores
                continue
        elif op == "qmm4":
            c = dict(op=op, M=rng.choice((1, rng.randint(2, 9), rng.randint(10, 40))), N=_log_int(rng, 100, 151936),
                     K=128 * _log_int(rng, 1, 64), gs=rng.choice((64, 128)), dtype=dtype)
        else:
            c = dict(op=op, B=_log_int(rng, 1, 64), V=_log_int(rng, 1000, 300000), history=_log_int(rng, 1, 20000),
                     biases=rng.choice((0, _log_int(rng, 1, 300))), mask=rng.choice((False, True)), dtype=dtype)
        if 3072 in c.values():  # a size kept out of the measurements
            continue
        w = work(c)
        if w["bytes"] <= most["bytes"] and w["flops"] <= max(most["flops"], 1):
            return c


def _spread(top, low, count):
    """``count`` lengths between ``low`` and ``top``, the first of them ``top``: a ragged batch."""
    return [top - (b * 2654435761 % (1 << 32)) * (top - low) // (1 << 32) if b else top for b in range(count)]


def _past(case):
    """Tokens already in the cache before an append, per sequence."""
    return _spread(case["past"], case["past"] // 2, case["B"])


def _lens(case):
    """Tokens in the cache, the new ones among them, per sequence."""
    return _spread(case["len"], max(case["n"], case["len"] // 4), case["B"])


def _touched(n):
    """Pages that n consecutive tokens can touch."""
    return (n + PAGE - 2) // PAGE + 1


def _keys_seen(length, n, window):
    """Sum over the n last positions of a sequence of the keys that each of them sees."""
    first = length - n  # position p sees min(p + 1, window) keys
    def total(p):  # over positions 0 .. p-1
        if window == 0 or p <= window:
            return p * (p + 1) // 2
        return window * (window + 1) // 2 + (p - window) * window
    return total(length) - total(first)


def work(case):
    op = case["op"]
    if op == "append":
        T, D, Hq, Hkv = case["B"] * case["n"], case["D"], case["Hq"], case["Hkv"]
        pages = case["B"] * _touched(case["n"])
        reads = T * (Hq + 2 * Hkv) * D * 2 + case["n"] * case["B"] * case["rot"] * 4
        writes = T * Hq * D * 2 + T * 2 * Hkv * D
        values = pages * PAGE * Hkv * D * 2 * 2  # the touched pages as 16-bit values
        return {"bytes": reads + writes + values, "flops": T * (Hq + Hkv) * D * 8 + T * Hkv * D * 4}
    if op == "attend":
        D, Hq, Hkv, n, w = case["D"], case["Hq"], case["Hkv"], case["n"], case["window"]
        lens = _lens(case)
        keys = sum(l if w == 0 else min(l, w + n - 1) for l in lens)
        pairs = sum(_keys_seen(l, n, w) for l in lens)
        return {"bytes": 2 * keys * Hkv * D + 2 * (keys // PAGE + 1) * Hkv * 4 + 2 * case["B"] * n * Hq * D * 2,
                "flops": 4 * D * Hq * pairs}
    if op == "qmm4":
        M, N, K, gs = case["M"], case["N"], case["K"], case["gs"]
        return {"bytes": N * K // 2 + 2 * N * (K // gs) * 2 + M * K * 2 + M * N * 2, "flops": 2 * M * N * K}
    B, V = case["B"], case["V"]
    return {"bytes": B * (V * (2 + 4) + (V // 8 if case["mask"] else 0) + case["history"] * 4 + case["biases"] * 8),
            "flops": 6 * B * V}


# ---- inputs --------------------------------------------------------------------

def _tables(lens, extra, g):
    """A block table of scattered pages for these lengths (``extra`` spare columns), and the number of pages."""
    cols = max(-(-l // PAGE) for l in lens) + extra
    pages = len(lens) * cols
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    return order.view(len(lens), cols).contiguous(), pages


def _quantised(x):
    """Codes (128 + the rounded multiple of the scale) and scales of pages [P, H, PAGE, D]."""
    scale = x.abs().amax(dim=(2, 3)) / 127.0
    return (torch.round(x / scale[:, :, None, None]) + 128.0).to(torch.uint8), scale


def _pool(pages, H, D, g):
    """K [P, H, PAGE, D] and V [P, H, D, PAGE] codes and their scales: normal values, some pages larger than others."""
    out = []
    for _ in range(2):
        codes = torch.empty(pages, H, PAGE, D, dtype=torch.uint8, device="cuda")
        scales = torch.empty(pages, H, device="cuda")
        for p in range(0, pages, 1024):  # in parts: a pool in 32 bits would be large
            q = min(pages, p + 1024)
            x = torch.randn(q - p, H, PAGE, D, generator=g, device="cuda")
            x *= 0.5 + torch.rand(q - p, H, 1, 1, generator=g, device="cuda")
            codes[p:q], scales[p:q] = _quantised(x)
        out += [codes, scales]
    return out[0], out[2].transpose(2, 3).contiguous(), out[1], out[3]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    dev = dict(device="cuda", generator=g)
    if case["op"] == "append":
        B, n, Hq, Hkv, D = (case[k] for k in ("B", "n", "Hq", "Hkv", "D"))
        past = _past(case)
        table, pages = _tables([p + n for p in past], 1, g)
        k, v, ks, vs = _pool(pages, Hkv, D, g)
        qkv = torch.randn(B * n, (Hq + 2 * Hkv) * D, **dev)
        qkv *= torch.exp(0.4 * torch.randn(B * n, 1, **dev))
        half = case["rot"] // 2
        freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
        angle = torch.arange(max(past) + n, dtype=torch.float64)[:, None] * freq
        rope = torch.cat([angle.cos(), angle.sin()], dim=1).float().cuda()
        return dict(case=case, qkv=qkv.to(dt), k=k, v=v, ks=ks, vs=vs, table=table, rope=rope,
                    lens=torch.tensor([p + n for p in past], dtype=torch.int32).cuda(),
                    first=torch.tensor([p // PAGE * PAGE for p in past], dtype=torch.int32).cuda(),
                    qw=(1 + 0.2 * torch.randn(D, **dev)).to(dt), kw=(1 + 0.2 * torch.randn(D, **dev)).to(dt))
    if case["op"] == "attend":
        lens = _lens(case)
        table, pages = _tables(lens, 0, g)
        k, v, ks, vs = _pool(pages, case["Hkv"], case["D"], g)
        q = torch.randn(case["B"] * case["n"], case["Hq"], case["D"], **dev) * 1.5
        return dict(case=case, q=q.to(dt), k=k, v=v, ks=ks, vs=vs, table=table,
                    lens=torch.tensor(lens, dtype=torch.int32).cuda())
    if case["op"] == "qmm4":
        M, N, K, gs = (case[k] for k in ("M", "N", "K", "gs"))
        w = torch.randint(-2 ** 31, 2 ** 31, (N, K // 8), dtype=torch.int64, **dev).to(torch.int32)
        s = (0.002 + 0.004 * torch.rand(N, K // gs, **dev)).to(dt)
        b = (-7.5 * s.float() * (1 + 0.1 * torch.randn(N, K // gs, **dev))).to(dt)
        return dict(case=case, x=torch.randn(M, K, **dev).to(dt), w=w, s=s, b=b)
    B, V, nh, nb = (case[k] for k in ("B", "V", "history", "biases"))
    counts = _spread(nh, nh // 2, B)
    hist = (torch.rand(sum(counts), **dev) ** 3 * V).to(torch.int32)  # common tokens come back often
    bias_ids = torch.rand(B, max(nb, 1), **dev).argsort(dim=1)[:, :nb] * (V // max(nb, 1))
    allowed = None
    if case["mask"]:
        allowed = torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32), dtype=torch.int64, **dev).to(torch.int32)
    return dict(case=case, logits=(3 * torch.randn(B, V, **dev)).to(dt), hist=hist,
                cu_hist=torch.tensor([sum(counts[:b]) for b in range(B + 1)], dtype=torch.int32).cuda(),
                rows=torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(counts, device="cuda")),
                rep=1.0 + 0.3 * torch.rand(B, **dev), pres=0.5 * torch.rand(B, **dev), freq=0.2 * torch.rand(B, **dev),
                bias_ids=bias_ids.reshape(-1).to(torch.int32), bias=(4 * torch.randn(B * nb, **dev)),
                cu_bias=torch.arange(0, B * nb + 1, max(nb, 1), dtype=torch.int32).cuda() if nb else
                torch.zeros(B + 1, dtype=torch.int32).cuda(), allowed=allowed)


# ---- the plain forms -----------------------------------------------------------

def _heads_norm(x, w, eps):
    return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + eps) * w


def _rotated(x, cos, sin, interleaved):
    """x [..., D] with its first 2 * cos.shape[-1] elements rotated."""
    half = cos.shape[-1]
    a, b = (x[..., :2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, v], dim=-1).flatten(-2) if interleaved else torch.cat([u, v], dim=-1)
    return torch.cat([turned, x[..., 2 * half:]], dim=-1)


def _plain_append(s):
    c = s["case"]
    B, n, Hq, Hkv, D = (c[k] for k in ("B", "n", "Hq", "Hkv", "D"))
    dt = s["qkv"].dtype
    x = s["qkv"].float().view(B, n, Hq + 2 * Hkv, D)
    past = s["lens"].long() - n
    pos = past[:, None] + torch.arange(n, device="cuda")
    half = c["rot"] // 2
    cos, sin = s["rope"][pos][:, :, None, :half], s["rope"][pos][:, :, None, half:]
    q = _rotated(_heads_norm(x[:, :, :Hq], s["qw"].float(), 1e-6), cos, sin, c["interleaved"])
    k = _rotated(_heads_norm(x[:, :, Hq:Hq + Hkv], s["kw"].float(), 1e-6), cos, sin, c["interleaved"])
    v = x[:, :, Hq + Hkv:]

    blocks = _touched(n)
    off = past % PAGE
    col = past[:, None] // PAGE + torch.arange(blocks, device="cuda")
    page = torch.gather(s["table"].long(), 1, col.clamp(max=s["table"].shape[1] - 1))
    row = torch.arange(blocks * PAGE, device="cuda")
    fresh = (row >= off[:, None]) & (row < off[:, None] + n)                   # rows written now
    kept = row < off[:, None]                                                    # rows of the first page that stay
    source = (row - off[:, None]).clamp(0, n - 1)
    used = fresh.view(B, blocks, PAGE).any(dim=2)
    outs = []
    for new, pool, scales, turn in ((k, s["k"], s["ks"], False), (v, s["v"], s["vs"], True)):
        new = torch.gather(new, 1, source[:, :, None, None].expand(-1, -1, Hkv, D)) * fresh[:, :, None, None]
        need = new.view(B, blocks, PAGE, Hkv, D).abs().amax(dim=(2, 4)) * (1.0 / 127.0)
        before = scales[page]
        had = torch.where(kept.view(B, blocks, PAGE).any(dim=2)[:, :, None], before, torch.zeros_like(before))
        scale = torch.maximum(need, had)
        inv = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
        old = pool[page]                                                         # [B, blocks, Hkv, PAGE, D] or V's turned
        old = (old.transpose(3, 4) if turn else old).permute(0, 1, 3, 2, 4)
        shrunk = torch.round((old.float() - 128.0) * (had * inv)[:, :, None, :, None])
        fine = torch.round(new.view(B, blocks, PAGE, Hkv, D) * inv[:, :, None, :, None]).clamp(-127, 127)
        codes = torch.where(fresh.view(B, blocks, PAGE, 1, 1), (fine + 128.0).to(torch.uint8),
                            torch.where(kept.view(B, blocks, PAGE, 1, 1), (shrunk + 128.0).to(torch.uint8), old))
        codes = torch.where(used[:, :, None, None, None], codes, old).permute(0, 1, 3, 2, 4)
        scale = torch.where(used[:, :, None], scale, before)
        pool[page] = codes.transpose(3, 4) if turn else codes
        scales[page] = scale
        values = (codes.float() - 128.0) * scale[:, :, :, None, None]
        live = (fresh | kept).view(B, blocks, 1, PAGE, 1)
        outs.append((values * live).permute(0, 1, 3, 2, 4).reshape(B, blocks * PAGE, Hkv, D).to(dt))
    return {"q": q.reshape(B * n, Hq, D).to(dt), "k": outs[0], "v": outs[1], "k_scale": s["ks"], "v_scale": s["vs"]}


def _plain_attend(s):
    c = s["case"]
    B, n, Hq, Hkv, D = (c[k] for k in ("B", "n", "Hq", "Hkv", "D"))
    G = Hq // Hkv
    page = s["table"].long()
    L = page.shape[1] * PAGE
    k = (s["k"][page].float() - 128.0) * s["ks"][page][..., None, None]          # [B, pages, Hkv, PAGE, D]
    v = (s["v"][page].float() - 128.0) * s["vs"][page][..., None, None]          # [B, pages, Hkv, D, PAGE]
    k = k.permute(0, 2, 1, 3, 4).reshape(B, Hkv, L, D)
    v = v.permute(0, 2, 1, 4, 3).reshape(B, Hkv, L, D)
    q = s["q"].float().view(B, n, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * n, D)
    score = torch.matmul(q, k.transpose(2, 3)).view(B, Hkv, G, n, L) * D ** -0.5
    pos = s["lens"][:, None] - n + torch.arange(n, device="cuda")
    key = torch.arange(L, device="cuda")
    seen = key <= pos[:, :, None]
    if c["window"]:
        seen &= key > pos[:, :, None] - c["window"]
    score = score.masked_fill(~seen[:, None, None], float("-inf"))
    e = torch.exp(score - score.amax(dim=-1, keepdim=True))
    p = (e / e.sum(dim=-1, keepdim=True)).view(B, Hkv, G * n, L)
    out = torch.matmul(p, v).view(B, Hkv, G, n, D).permute(0, 3, 1, 2, 4).reshape(B * n, Hq, D)
    return out.to(s["q"].dtype)


def _plain_qmm4(s):
    c = s["case"]
    shift = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    code = ((s["w"][:, :, None] >> shift) & 15).float().view(c["N"], c["K"] // c["gs"], c["gs"])
    w = code * s["s"].float()[:, :, None] + s["b"].float()[:, :, None]
    return torch.matmul(s["x"].float(), w.view(c["N"], c["K"]).T).to(s["x"].dtype)


def _plain_logits(s):
    c = s["case"]
    B, V = c["B"], c["V"]
    l = s["logits"].float()
    count = torch.zeros(B * V, device="cuda").index_add_(0, s["rows"] * V + s["hist"].long(),
                                                         torch.ones(s["hist"].numel(), device="cuda")).view(B, V)
    rep = s["rep"][:, None]
    l = torch.where(count > 0, torch.where(l > 0, l / rep, l * rep), l)
    l = l - (s["freq"][:, None] * count + s["pres"][:, None] * (count > 0).float())
    if c["biases"]:
        at = torch.arange(B, device="cuda").repeat_interleave(c["biases"]) * V + s["bias_ids"].long()
        l = l.view(-1).index_add(0, at, s["bias"]).view(B, V)
    if s["allowed"] is not None:
        token = torch.arange(V, device="cuda")
        bit = (s["allowed"][:, token // 32] >> (token % 32)) & 1
        l = torch.where(bit.bool(), l, torch.full_like(l, float("-inf")))
    return l


# ---- one pass ------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "qmm4": _plain_qmm4, "logits": _plain_logits}[op](state)
    from momij_b200 import attn, head
    c = state["case"]
    if op == "qmm4":
        return head.qmm4(state["x"], state["w"], state["s"], state["b"], gs=c["gs"])
    if op == "logits":
        return head.process_logits(state["logits"], history=state["hist"], cu_history=state["cu_hist"],
                                   repetition=state["rep"], presence=state["pres"], frequency=state["freq"],
                                   bias_ids=state["bias_ids"], bias=state["bias"], cu_bias=state["cu_bias"],
                                   allowed=state["allowed"])
    if "cache" not in state:  # what a program keeps from call to call
        state["cache"] = attn.KVCache(state["k"], state["v"], state["ks"], state["vs"])
        state["ws"] = attn.new_workspace(c["B"] * c["n"], c["Hq"], c["D"])
    if op == "attend":
        return attn.attention(state["q"], state["cache"], state["table"], state["lens"], window=c["window"],
                              workspace=state["ws"])
    q = attn.qk_norm_rope_append(state["qkv"], state["cache"], state["table"], state["lens"], n_heads=c["Hq"],
                                 q_weight=state["qw"], k_weight=state["kw"], eps=1e-6, rope=state["rope"],
                                 interleaved=c["interleaved"], workspace=state["ws"])
    k, v = attn.cache_read(state["cache"], state["table"], state["lens"], first=state["first"],
                           count=_touched(c["n"]) * PAGE, dtype=state["qkv"].dtype, workspace=state["ws"])
    return {"q": q, "k": k, "v": v, "k_scale": state["ks"], "v_scale": state["vs"]}


# ---- the definitions in 64 bits --------------------------------------------------

def _exact_append(s):
    c = s["case"]
    B, n, Hq, Hkv, D = (c[k] for k in ("B", "n", "Hq", "Hkv", "D"))
    half, blocks = c["rot"] // 2, _touched(n)
    ks, vs = s["ks"].double().clone(), s["vs"].double().clone()
    q_out = torch.empty(B, n, Hq, D, dtype=torch.float64, device="cuda")
    k_out = torch.zeros(B, blocks * PAGE, Hkv, D, dtype=torch.float64, device="cuda")
    v_out = torch.zeros_like(k_out)
    for b, past in enumerate(_past(c)):
        x = s["qkv"][b * n:(b + 1) * n].double().view(n, Hq + 2 * Hkv, D)
        table = s["rope"][past:past + n].double()
        turn = torch.complex(table[:, :half], table[:, half:])[:, None]

        def turned(y, w):
            y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / D + 1e-6) * w.double()
            if c["interleaved"]:
                z = torch.view_as_complex(y[..., :2 * half].reshape(n, -1, half, 2).contiguous()) * turn
                return torch.cat([torch.view_as_real(z).reshape(n, -1, 2 * half), y[..., 2 * half:]], dim=-1)
            z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn
            return torch.cat([z.real, z.imag, y[..., 2 * half:]], dim=-1)

        q_out[b] = turned(x[:, :Hq], s["qw"])
        for new, pool, scales, out, t in ((turned(x[:, Hq:Hq + Hkv], s["kw"]), s["k"], ks, k_out, False),
                                          (x[:, Hq + Hkv:], s["v"], vs, v_out, True)):
            for j in range(blocks):
                lo, hi = past // PAGE * PAGE + j * PAGE, past // PAGE * PAGE + (j + 1) * PAGE
                a, z = max(lo, past), min(hi, past + n)
                if a >= z:
                    continue
                page = int(s["table"][b, lo // PAGE])
                part = new[a - past:z - past]
                scale = part.abs().amax(dim=(0, 2)) / 127
                if a > lo:
                    held = pool[page].double()
                    held = (held.transpose(1, 2) if t else held)[:, :a - lo] - 128
                    was = scales[page].clone()
                    scale = torch.maximum(scale, was)
                    ratio = (was / scale)[:, None, None]
                    out[b, j * PAGE:j * PAGE + a - lo] = (torch.round(held * ratio) * scale[:, None, None]).transpose(0, 1)
                out[b, j * PAGE + a - lo:j * PAGE + z - lo] = torch.round(part / scale[:, None]) * scale[:, None]
                scales[page] = scale
    return {"q": q_out.view(B * n, Hq, D), "k": k_out, "v": v_out, "k_scale": ks, "v_scale": vs}


def _exact_attend(s):
    c = s["case"]
    n, Hq, Hkv, D, w = (c[k] for k in ("n", "Hq", "Hkv", "D", "window"))
    G = Hq // Hkv
    out = torch.empty(c["B"], n, Hq, D, dtype=torch.float64, device="cuda")
    for b, length in enumerate(_lens(c)):
        lo = 0 if w == 0 else max(0, length - n - w + 1) // PAGE * PAGE  # no key before it is seen
        page = s["table"][b, lo // PAGE:-(-length // PAGE)].long()
        for h in range(Hkv):
            k = ((s["k"][page, h].double() - 128) * s["ks"][page, h].double()[:, None, None]).reshape(-1, D)
            v = ((s["v"][page, h].double() - 128) * s["vs"][page, h].double()[:, None, None]).transpose(1, 2).reshape(-1, D)
            k, v = k[:length - lo], v[:length - lo]
            at = torch.arange(lo, length, device="cuda")
            for t in range(0, n, 1024):
                u = min(n, t + 1024)
                q = s["q"][b * n + t:b * n + u, h * G:(h + 1) * G].double()
                score = torch.einsum("tgd,ld->tgl", q, k) / math.sqrt(D)
                p = torch.arange(length - n + t, length - n + u, device="cuda")[:, None]
                hidden = (at > p) | ((at <= p - w) if w else torch.zeros_like(at > p))
                score[hidden[:, None].expand(-1, G, -1)] = -math.inf
                out[b, t:u, h * G:(h + 1) * G] = torch.einsum("tgl,ld->tgd", torch.softmax(score, dim=-1), v)
    return out.view(-1, Hq, D)


def _exact_qmm4(s):
    c = s["case"]
    x, parts = s["x"].double(), []
    for r in range(0, c["N"], 8192):
        w = s["w"][r:r + 8192].long()
        code = torch.stack([(w >> (4 * i)) & 15 for i in range(8)], dim=-1).view(w.shape[0], -1).double()
        scale = s["s"][r:r + 8192].double().repeat_interleave(c["gs"], dim=1)
        bias = s["b"][r:r + 8192].double().repeat_interleave(c["gs"], dim=1)
        parts.append(x @ (scale * code + bias).T)
    return torch.cat(parts, dim=1)


def _exact_logits(s):
    c = s["case"]
    rows = []
    cu, bu = s["cu_hist"].tolist(), s["cu_bias"].tolist()
    for b in range(c["B"]):
        l = s["logits"][b].double()
        count = torch.bincount(s["hist"][cu[b]:cu[b + 1]].long(), minlength=c["V"]).double()
        rep, pres, freq = (float(s[k][b]) for k in ("rep", "pres", "freq"))
        said = count > 0
        l[said] = torch.where(l[said] > 0, l[said] / rep, l[said] * rep)
        l = l - freq * count - pres * said
        l[s["bias_ids"][bu[b]:bu[b + 1]].long()] += s["bias"][bu[b]:bu[b + 1]].double()
        if s["allowed"] is not None:
            word = s["allowed"][b].long() & 0xFFFFFFFF
            bits = torch.stack([(word >> i) & 1 for i in range(32)], dim=1).view(-1)[:c["V"]]
            l[bits == 0] = -math.inf
        rows.append(l)
    return torch.stack(rows)


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "qmm4": _exact_qmm4, "logits": _exact_logits}[case["op"]](s)
