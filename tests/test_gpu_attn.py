"""GPU tests of the attention half (momij_b200/attn.py) against 64-bit restatements
(tests/attn_ref.py): head norms with rotation and append, the cache's values,
attention over it, their refusals, and what must not matter (strides, streams,
scheduling, what lies beyond a sequence's end)."""
from __future__ import annotations

import math

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from momij_b200 import attn, moe


def cuda(*ts):
    return tuple(None if t is None else t.cuda() for t in ts)


def make_attend(B, counts, lens, Hq, Hkv, D, dtype, seed=0, spare=0):
    table, pages = R.block_tables(lens, seed, spare)
    pool = R.random_pool(pages, Hkv, D, seed + 1)
    g = torch.Generator().manual_seed(seed + 2)
    q = (torch.randn(sum(counts), Hq, D, generator=g) * 1.5).to(R.TD[dtype])
    return q, pool, table, lens, R.offsets(counts)


def run_attend(q, pool, table, lens, cu, ragged=False, **kw):
    cache = attn.KVCache(*cuda(*pool))
    lens_t = torch.tensor(lens, dtype=torch.int32).cuda()
    if ragged:
        kw.update(cu_q=torch.tensor(cu, dtype=torch.int32).cuda(), max_q=max(b - a for a, b in zip(cu, cu[1:])))
    ws = kw.pop("workspace", None)
    ws = attn.new_workspace(max(1, q.shape[0]), q.shape[1]) if ws is None else ws
    out = attn.attention(q.cuda(), cache, table.cuda(), lens_t, workspace=ws, **kw)
    moe.synchronize(workspace=ws)
    return out


def check_attend(q, pool, table, lens, cu, out, window=0, scale=None):
    ref, mag, big = R.attention(q, *pool, table, lens, cu, window, scale)
    bound = R.attention_bound(ref, mag, big, q.shape[2], q.dtype)
    err = (out.cpu().double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    return ref


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("B,n,length,Hq,Hkv,D,window", [
    (1, 1, 1, 4, 1, 64, 0),            # one token in the cache
    (3, 1, 64, 8, 8, 128, 0),          # exactly one page, one row a head
    (2, 1, 65, 16, 2, 128, 0),         # a page and a token
    (5, 1, 1500, 6, 2, 64, 0),         # groups of three
    (2, 3, 700, 14, 2, 64, 100),       # 21 rows: the tensor-memory kernel, window
    (4, 2, 300, 16, 2, 128, 1),        # a window of one: each token sees itself
    (3, 5, 333, 3, 1, 128, 40),        # 15 rows, a window inside a page or two
    (1, 1, 3000, 16, 1, 64, 0),        # 16 rows, many pages: shared by many blocks
    (2, 17, 17, 4, 4, 64, 0),          # prompt from nothing
    (2, 70, 130, 4, 2, 128, 0),        # 140 rows: two row tiles
    (1, 130, 400, 7, 1, 64, 90),       # 910 rows of groups of seven
])
def test_attention_matches_64_bits(B, n, length, Hq, Hkv, D, window, dtype):
    lens = [max(n, length - 37 * b) for b in range(B)]
    args = make_attend(B, [n] * B, lens, Hq, Hkv, D, dtype)
    out = run_attend(*args, window=window)
    check_attend(*args, out, window)


@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 64), (16, 2, 128)])
@pytest.mark.parametrize("most", [3, 40])
def test_attention_ragged_and_empty(Hq, Hkv, D, most):
    """Sequences of their own numbers of queries, none among them; a cache shorter
    than the queries (the first see nothing) and an empty one: zeros."""
    counts = [1, 0, most, 2, 3, 0, 2]
    lens = [200, 0, 90, 1, 0, 500, 2]
    args = make_attend(len(lens), counts, lens, Hq, Hkv, D, "f16", seed=5)
    out = run_attend(*args, ragged=True)
    ref = check_attend(*args, out)
    cu = args[-1]
    assert (out[cu[3]] == 0).all() and (ref[cu[3]] == 0).all()  # position -1 of a length of 1
    assert (out[cu[4]:cu[5]] == 0).all()


@pytest.mark.parametrize("n,Hq", [(1, 8), (40, 8)])
def test_attention_ignores_what_it_does_not_see(n, Hq):
    """Codes past the end, pages outside the window (NaN scales) and unused pages."""
    lens, Hkv, D, window = [300, 421], 2, 64, 70
    q, pool, table, lens, cu = make_attend(2, [n] * 2, lens, Hq, Hkv, D, "bf16", seed=3, spare=2)
    ref = run_attend(q, pool, table, lens, cu, window=window)
    k, v, ks, vs = (t.clone() for t in pool)
    for b, length in enumerate(lens):
        lo = max(0, length - n - window + 1)
        for i in range(table.shape[1]):
            p = int(table[b, i])
            if (i + 1) * 64 <= lo or i * 64 >= length:
                ks[p], vs[p] = math.nan, math.inf
            elif (i + 1) * 64 > length:  # the last page: rows past the end
                k[p, :, length - i * 64:] = 255
                v[p, :, :, length - i * 64:] = 1
    out = run_attend(q, (k, v, ks, vs), table, lens, cu, window=window)
    assert torch.equal(out, ref)


@pytest.mark.parametrize("n,Hq", [(1, 8), (40, 8)])
def test_attention_special_pages(n, Hq):
    """Pages of zeros keep their weight; a NaN page shows in the rows that see it
    and in no other head."""
    lens = [400]
    q, (k, v, ks, vs), table, lens, cu = make_attend(1, [n], lens, Hq, 2, 64, "bf16", seed=9)
    zero = int(table[0, 2])
    k[zero], v[zero], ks[zero], vs[zero] = 128, 128, 0.0, 0.0
    out = run_attend(q, (k, v, ks, vs), table, lens, cu)
    check_attend(q, (k, v, ks, vs), table, lens, cu, out)
    for which in (ks, vs):
        bad = which.clone()
        bad[int(table[0, 1]), 1] = math.nan
        args = (k, v, bad, vs) if which is ks else (k, v, ks, bad)
        got = run_attend(q, args, table, lens, cu)
        assert torch.equal(got[:, :Hq // 2], out[:, :Hq // 2])
        assert torch.isnan(got[:, Hq // 2:]).all()


def test_attention_page_scales_far_apart():
    """V pages whose scales differ by 2^40 and a K page that dominates: weights stay
    exact where a common scale would lose them."""
    lens = [256]
    q, (k, v, ks, vs), table, lens, cu = make_attend(1, [1], lens, 8, 1, 128, "bf16", seed=11)
    vs[int(table[0, 0])] *= 2.0 ** 20
    vs[int(table[0, 3])] *= 2.0 ** -20
    ks[int(table[0, 3])] *= 40  # nearly all weight on the page of small values
    out = run_attend(q, (k, v, ks, vs), table, lens, cu)
    check_attend(q, (k, v, ks, vs), table, lens, cu, out)


@pytest.mark.parametrize("scale", [0.3, -0.05, 0.0])
@pytest.mark.parametrize("n", [1, 30])
def test_attention_scale(scale, n):
    args = make_attend(2, [n] * 2, [150, 150], 4, 1, 64, "f16", seed=13)
    out = run_attend(*args, scale=scale)
    check_attend(*args, out, scale=scale)


@pytest.mark.parametrize("mult", [2.0 ** -60, 2.0 ** 60])
def test_attention_large_and_small_queries(mult):
    """Queries far from one, with a scale that brings the scores back."""
    q, pool, table, lens, cu = make_attend(1, [2], [130], 4, 2, 64, "bf16", seed=17)
    q = (q.double() * mult).to(q.dtype)
    out = run_attend(q, pool, table, lens, cu, scale=0.125 / mult)
    check_attend(q, pool, table, lens, cu, out, scale=0.125 / mult)


@pytest.mark.parametrize("n", [1, 2, 33])
def test_attention_strides_and_alignment(n):
    """Queries inside a wider projection, from an odd element on; a strided output."""
    q, pool, table, lens, cu = make_attend(3, [n] * 3, [100, 200, 300], 8, 2, 64, "bf16", seed=19)
    ref = run_attend(q, pool, table, lens, cu)
    T = q.shape[0]
    for off in (0, 64, 1):
        wide = torch.zeros(T * 900 + 8, dtype=q.dtype, device="cuda")
        view = wide[off:off + T * 900].view(T, 900)[:, :512].view(T, 8, 64) if off == 0 else \
            torch.as_strided(wide, (T, 8, 64), (900, 64, 1), off)
        view.copy_(q)
        out = torch.full((T, 10, 64), 7.0, dtype=q.dtype, device="cuda")
        cache = attn.KVCache(*cuda(*pool))
        ws = attn.new_workspace(T, 8)
        attn.attention(view, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), out=out[:, :8], workspace=ws)
        moe.synchronize(workspace=ws)
        assert torch.equal(out[:, :8], ref) and (out[:, 8:] == 7).all()


@pytest.mark.parametrize("n", [1, 40])
def test_attention_repeats_bit_for_bit_on_streams_and_graphs(n):
    q, pool, table, lens, cu = make_attend(9, [n] * 9, [900 - 90 * b for b in range(9)], 8, 2, 128, "f16", seed=23)
    ref = run_attend(q, pool, table, lens, cu)
    cache = attn.KVCache(*cuda(*pool))
    qd, td, ld = q.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    ws = attn.new_workspace(q.shape[0], 8)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    out = attn.attention(qd, cache, td, ld, workspace=ws, stream=side)
    moe.synchronize(stream=side, workspace=ws)
    assert torch.equal(out, ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a = attn.attention(qd, cache, td, ld, workspace=ws)
        b = attn.attention(qd, cache, td, ld, workspace=ws)
    for _ in range(3):
        g.replay()
    moe.synchronize(workspace=ws)
    assert torch.equal(a, ref) and torch.equal(b, ref)


def test_attention_workspace_serves_calls_of_any_size():
    ws = attn.new_workspace(64, 16)
    for n, B, length in ((1, 1, 2000), (32, 2, 500), (1, 30, 70), (16, 3, 3000), (1, 1, 2000)):
        args = make_attend(B, [n] * B, [length] * B, 4, 2, 64, "bf16", seed=n + B)
        out = run_attend(*args, workspace=ws)
        check_attend(*args, out)


def test_attention_cache_offsets_past_32_bits():
    """A pool of 4.6 GB of codes, pages from both ends of it."""
    pages, H, D = 70_000, 8, 128
    k = torch.full((pages, H, 64, D), 128, dtype=torch.uint8, device="cuda")
    v = torch.full((pages, H, D, 64), 128, dtype=torch.uint8, device="cuda")
    ks, vs = torch.zeros(pages, H, device="cuda"), torch.zeros(pages, H, device="cuda")
    ids = [0, 69_999, 35_000, 69_998]
    pool = R.random_pool(4, H, D, 1)
    for i, p in enumerate(ids):
        k[p], v[p], ks[p], vs[p] = (t[i].cuda() for t in pool)
    table = torch.tensor([ids], dtype=torch.int32)
    for n in (1, 40):
        q = torch.randn(n, 16, D, generator=torch.Generator().manual_seed(n)).bfloat16()
        ws = attn.new_workspace(n, 16)
        lens = torch.tensor([250], dtype=torch.int32).cuda()
        out = attn.attention(q.cuda(), attn.KVCache(k, v, ks, vs), table.cuda(), lens, workspace=ws)
        moe.synchronize(workspace=ws)
        check_attend(q, pool, torch.tensor([[0, 1, 2, 3]]), [250], [0, n], out)
        kv = attn.cache_read(attn.KVCache(k, v, ks, vs), table.cuda(), lens, count=256, workspace=ws)
        moe.synchronize(workspace=ws)
        ref = R.values(*pool)[1].permute(0, 2, 1, 3).reshape(256, H, D)[:250].bfloat16()
        assert torch.equal(kv[1][0, :250].cpu(), ref) and (kv[1][0, 250:] == 0).all()


# ---- append and cache values ------------------------------------------------------

def make_append(counts, lens, Hq, Hkv, D, rot, dtype, seed=0):
    table, pages = R.block_tables(lens, seed, 1)
    pool = R.random_pool(pages, Hkv, D, seed + 1)
    g = torch.Generator().manual_seed(seed + 2)
    dt = R.TD[dtype]
    qkv = (torch.randn(sum(counts), (Hq + 2 * Hkv) * D, generator=g)).to(dt)
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g)).to(dt) for _ in range(2))
    rope = R.rope_table(max(lens) + 1, rot) if rot else None
    return qkv, pool, table, lens, R.offsets(counts), qw, kw, rope


def run_append(qkv, pool, table, lens, cu, qw, kw, rope, Hq, interleaved=False, ragged=False, eps=1e-6, check=True):
    cache = attn.KVCache(*(t.clone().cuda() for t in pool))
    kw_ = dict(cu_q=torch.tensor(cu, dtype=torch.int32).cuda(), max_q=max(b - a for a, b in zip(cu, cu[1:]))) if ragged else {}
    ws = attn.new_workspace(1, 1)
    qwd, kwd, rd = cuda(qw, kw, rope)
    q = attn.qk_norm_rope_append(qkv.cuda(), cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), n_heads=Hq,
                                 q_weight=qwd, k_weight=kwd, eps=eps, rope=rd, interleaved=interleaved, workspace=ws, **kw_)
    if check:
        moe.synchronize(workspace=ws)
    return q, cache, ws


def check_append(q, cache, ref):
    """Queries: one rounding and fp32 steps.  Scales: fp32 steps.  Codes: at most one
    apart, and only where the fp32 steps (relative 2^-20 of up to 127 codes, twice)
    cross a rounding boundary."""
    rq, kk, vv, ks, vs = ref
    err = (q.cpu().double() - rq).abs()
    assert bool((err <= 2 * R.HALF_ULP[q.dtype] * rq.abs() + 2.0 ** -19 * rq.abs().amax(-1, keepdim=True)).all())
    for codes, scale, want, ws in ((cache.k.cpu().double() - 128, cache.k_scale, kk, ks),
                                   ((cache.v.cpu().double() - 128).transpose(2, 3), cache.v_scale, vv, vs)):
        s = scale.cpu().double()
        assert bool(((s - ws).abs() <= 2.0 ** -20 * ws).all())
        d = torch.where(ws > 0, ws, torch.ones_like(ws))[:, :, None, None]
        off = (codes * (ws > 0)[:, :, None, None] - want / d).abs()
        off = off[~torch.isnan(want)]  # (rows past the end)
        assert float(off.max()) <= 1 + 1e-6 and float((off > 0.5).double().mean()) <= 1e-3, (float(off.max()), float((off > 0.5).double().mean()))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("counts,lens,Hq,Hkv,D,rot,interleaved", [
    ([1], [1], 4, 1, 64, 64, False),              # the first token
    ([1, 1, 1], [64, 65, 700], 16, 4, 128, 64, False),  # a page's last row, its first, its middle
    ([9, 9], [130, 69], 6, 2, 64, 32, True),      # across a page's end
    ([200], [263], 8, 2, 128, 128, False),        # several pages from the middle of one
    ([64], [64], 3, 3, 64, 16, True),             # one whole page
    ([70, 70], [70, 198], 14, 2, 128, 0, False),  # without rotation
])
def test_append_matches_64_bits(counts, lens, Hq, Hkv, D, rot, interleaved, dtype):
    args = make_append(counts, lens, Hq, Hkv, D, rot, dtype)
    q, cache, _ = run_append(*args, Hq, interleaved)
    qkv, pool, table, lens, cu, qw, kw, rope = args
    check_append(q, cache, R.append(qkv, pool, table, lens, cu, Hq, qw, kw, 1e-6, rope, interleaved))


def test_append_without_norms_and_ragged():
    counts, lens = [0, 3, 1, 100, 0], [40, 3, 129, 150, 0]
    qkv, pool, table, lens, cu, _, _, rope = make_append(counts, lens, 8, 2, 64, 32, "bf16", seed=4)
    args = (qkv, pool, table, lens, cu, None, None, rope)
    q, cache, _ = run_append(*args, 8, ragged=True)
    check_append(q, cache, R.append(qkv, pool, table, lens, cu, 8, None, None, 1e-6, rope, False))


def test_append_one_token_at_a_time_and_values():
    """A page filled token by token, its scale growing: values stay within one and a
    half codes of the true ones (each growth rounds once more), the newest within half."""
    H, D, n = 2, 64, 100
    g = torch.Generator().manual_seed(1)
    x = torch.randn(n, (2 + 2 * H) * D, generator=g) * torch.linspace(0.2, 3, n)[:, None]
    x = x.bfloat16()
    cache = attn.new_kv_cache(4, H, D)
    table = torch.tensor([[2, 0]], dtype=torch.int32).cuda()
    ws = attn.new_workspace(1, 2)
    for i in range(n):
        attn.qk_norm_rope_append(x[i:i + 1].cuda(), cache, table, torch.tensor([i + 1], dtype=torch.int32).cuda(), n_heads=2, workspace=ws)
    k, v = attn.cache_read(cache, table, torch.tensor([n], dtype=torch.int32).cuda(), count=128, dtype=torch.float16, workspace=ws)
    moe.synchronize(workspace=ws)
    want = x.double().view(n, 2 + 2 * H, D)
    for got, true, scale in ((k, want[:, 2:2 + H], cache.k_scale), (v, want[:, 2 + H:], cache.v_scale)):
        assert (got[0, n:] == 0).all()
        s = torch.stack([scale[2], scale[0]]).cpu().double().repeat_interleave(64, 0)[:n, :, None]
        err = (got[0, :n].cpu().double() - true).abs() / s
        growths = 12  # records among 64 growing values: each adds at most half a code, smaller ones less
        assert float(err.max()) <= 0.5 * growths and float((err ** 2).mean().sqrt()) <= 1.5
        assert float(err[-1].max()) <= 0.51 + 127 * 2.0 ** -11  # (and fp16's rounding)
        assert bool((torch.stack([scale[2], scale[0]]).cpu() * 127 >= true.abs().amax((0, 2)).float() * 0.3).all())


def test_append_rolled_back_tokens_are_overwritten():
    H, D = 1, 64
    g = torch.Generator().manual_seed(2)
    x = torch.randn(12, 3 * D, generator=g).half()
    x[8:] *= 0.25
    cache, ws = attn.new_kv_cache(2, H, D), attn.new_workspace(1, 1)
    table = torch.tensor([[1]], dtype=torch.int32).cuda()

    def add(rows, length):
        attn.qk_norm_rope_append(rows.contiguous().cuda(), cache, table, torch.tensor([length], dtype=torch.int32).cuda(), n_heads=1, workspace=ws)

    add(x[:8], 8)
    add(x[8:11], 6)  # five kept, three new ones in place of the others
    k, _ = attn.cache_read(cache, table, torch.tensor([6], dtype=torch.int32).cuda(), count=8, dtype=torch.float16, workspace=ws)
    moe.synchronize(workspace=ws)
    # lens 6 with three new tokens: positions 3, 4, 5
    want = torch.cat([x[:3], x[8:11]])[:, D:2 * D].double()
    s = float(cache.k_scale[1, 0])
    assert float((k[0, :6, 0].cpu().double() - want).abs().max()) <= 0.5 * s + 127 * s * 2.0 ** -11 + 1e-9
    assert (k[0, 6:] == 0).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_append_non_finite_values_poison_their_page_only(bad):
    qkv, pool, table, lens, cu, qw, kw, rope = make_append([100], [100], 2, 2, 64, 0, "bf16", seed=6)
    clean, cache0, _ = run_append(qkv, pool, table, lens, cu, None, None, None, 2)
    x = qkv.clone()
    x.view(100, 6, 64)[70, 2, 5] = bad   # a key of head 0, second page
    x.view(100, 6, 64)[10, 5, 1] = bad   # a value of head 1, first page
    _, cache, ws = run_append(x, pool, table, lens, cu, None, None, None, 2)
    p = [int(i) for i in table[0, :2]]
    for got, ref, at in ((cache.k_scale, cache0.k_scale, (p[1], 0)), (cache.v_scale, cache0.v_scale, (p[0], 1))):
        assert torch.isnan(got[at])
        same = torch.ones_like(got, dtype=torch.bool)
        same[at] = False
        assert torch.equal(got[same], ref[same])
    k, v = attn.cache_read(cache, table.cuda(), torch.tensor([100], dtype=torch.int32).cuda(), count=100, workspace=ws)
    assert torch.isnan(k[0, 64:, 0]).all() and not torch.isnan(k[0, :64]).any() and not torch.isnan(k[0, :, 1]).any()
    # the page heals when its first row is written again
    again = run_append(qkv, tuple(t.cpu() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)), table, lens, cu, None, None, None, 2)[1]
    assert torch.equal(again.k_scale, cache0.k_scale) and torch.equal(again.v, cache0.v)


@pytest.mark.parametrize("mult", [0.0, 2.0 ** -100, 2.0 ** -40, 2.0 ** 90])
def test_append_small_and_large_values(mult):
    qkv, pool, table, lens, cu, _, _, _ = make_append([70], [70], 2, 1, 64, 0, "bf16", seed=7)
    qkv = (qkv.double() * mult).bfloat16()
    q, cache, _ = run_append(qkv, pool, table, lens, cu, None, None, None, 2)
    check_append(q, cache, R.append(qkv, pool, table, lens, cu, 2, None, None, 1e-6, None, False))


def test_append_strided_rows():
    qkv, pool, table, lens, cu, qw, kw, rope = make_append([20], [50], 4, 2, 64, 64, "bf16", seed=8)
    q, cache, _ = run_append(qkv, pool, table, lens, cu, qw, kw, rope, 4)
    wide = torch.zeros(20, 8 * 64 + 128, dtype=qkv.dtype)
    wide[:, 128:] = qkv
    cache2 = attn.KVCache(*(t.clone().cuda() for t in pool))
    qd = attn.qk_norm_rope_append(wide.cuda()[:, 128:], cache2, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), n_heads=4,
                                  q_weight=qw.cuda(), k_weight=kw.cuda(), rope=rope.cuda())
    assert torch.equal(qd, q) and all(torch.equal(a, b) for a, b in zip((cache.k, cache.v, cache.k_scale, cache.v_scale),
                                                                         (cache2.k, cache2.v, cache2.k_scale, cache2.v_scale)))


@pytest.mark.parametrize("first,count", [([0, 0], 30), ([5, 100], 130), ([64, 127], 1), ([500, 0], 10)])
def test_cache_read_any_stretch(first, count):
    lens = [150, 300]
    table, pages = R.block_tables(lens, 3)
    pool = R.random_pool(pages, 3, 64, 4)
    k, v = attn.cache_read(attn.KVCache(*cuda(*pool)), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), count=count,
                           first=torch.tensor(first, dtype=torch.int32).cuda(), dtype=torch.float16)
    kk, vv = R.values(*pool)
    for got, val in ((k, kk), (v, vv)):
        for b in range(2):
            seq = torch.cat([val[int(p)].transpose(0, 1) for p in table[b]])[:lens[b]]
            want = torch.zeros(count, 3, 64, dtype=torch.float16)
            part = seq[first[b]:first[b] + count]
            want[:part.shape[0]] = part.half()
            assert float((got[b].cpu().double() - want.double()).abs().max()) <= 2.0 ** -10 * float(want.abs().max() + 1e-6)


# ---- refusals ------------------------------------------------------------------------

def small(n=1, Hq=4, Hkv=2, D=64, dtype=torch.bfloat16):
    cache = attn.new_kv_cache(8, Hkv, D)
    table = torch.arange(8, dtype=torch.int32).view(2, 4).cuda()
    lens = torch.tensor([70, 70], dtype=torch.int32).cuda()
    q = torch.zeros(2 * n, Hq, D, dtype=dtype, device="cuda")
    return q, cache, table, lens


def test_bad_pages_and_lengths_are_reported_and_skipped():
    for n in (1, 20):
        q, cache, table, lens = small(n)
        ws = attn.new_workspace(2 * n, 4)
        bad = table.clone()
        bad[1, 1] = 8
        for t, l in ((bad, lens), (table, torch.tensor([70, 257], dtype=torch.int32).cuda()),
                     (table, torch.tensor([-1, 70], dtype=torch.int32).cuda())):
            attn.attention(q, cache, t, l, workspace=ws)
            with pytest.raises(moe.SeedlessError) as e:
                moe.synchronize(workspace=ws)
            assert e.value.status == 11
        attn.attention(q, cache, table, lens, workspace=ws)
        moe.synchronize(workspace=ws)  # reported once, usable again
    x = torch.zeros(2, 8 * 64, dtype=torch.bfloat16, device="cuda")
    rope = attn.rope_table(69, 64)
    for kw, l in ((dict(rope=rope), lens), ({}, torch.tensor([70, 300], dtype=torch.int32).cuda()),
                  ({}, torch.tensor([70, 0], dtype=torch.int32).cuda())):
        attn.qk_norm_rope_append(x, cache, table, l, n_heads=4, workspace=ws, **kw)
        with pytest.raises(moe.SeedlessError):
            moe.synchronize(workspace=ws)
    # more queries in a sequence than max_q says
    cu = torch.tensor([0, 2, 2], dtype=torch.int32).cuda()
    q, cache, table, lens = small(1)
    attn.attention(q, cache, table, lens, cu_q=cu, max_q=1, workspace=ws)
    with pytest.raises(moe.SeedlessError):
        moe.synchronize(workspace=ws)


def test_argument_refusals():
    q, cache, table, lens = small()
    ws = attn.new_workspace(2, 4)
    with pytest.raises(TypeError):
        attn.attention(q.float(), cache, table, lens, workspace=ws)
    with pytest.raises(TypeError):
        attn.attention(q, cache, table.long(), lens, workspace=ws)
    with pytest.raises(ValueError):
        attn.attention(q, cache, table, lens[:1], workspace=ws)
    with pytest.raises(ValueError):
        attn.attention(q.cpu(), cache, table, lens, workspace=ws)
    with pytest.raises(ValueError):
        attn.attention(q.transpose(0, 1), cache, table, lens, workspace=ws)
    wide = attn.new_kv_cache(2, 2, 128)  # (at 64 dimensions k and v have one shape)
    with pytest.raises(ValueError):
        attn.KVCache(wide.k, wide.k, wide.k_scale, wide.v_scale)
    with pytest.raises(moe.SeedlessError) as e:  # five query heads over two
        attn.attention(torch.zeros(2, 5, 64, dtype=q.dtype, device="cuda"), cache, table, lens, workspace=ws)
    assert e.value.status == moe.UNSUPPORTED_SHAPE
    with pytest.raises(moe.SeedlessError) as e:
        attn.attention(q, cache, table, lens, workspace=ws[:1000])
    assert e.value.status == moe.WORKSPACE
    with pytest.raises(moe.SeedlessError) as e:
        attn.attention(q, cache, table, lens, window=-1, workspace=ws)
    assert e.value.status == moe.INVALID_ARGUMENT
    c96 = attn.KVCache(torch.zeros(2, 1, 64, 96, dtype=torch.uint8, device="cuda"), torch.zeros(2, 1, 96, 64, dtype=torch.uint8, device="cuda"),
                       torch.zeros(2, 1, device="cuda"), torch.zeros(2, 1, device="cuda"))
    with pytest.raises(moe.SeedlessError) as e:
        attn.attention(torch.zeros(2, 1, 96, dtype=q.dtype, device="cuda"), c96, table, lens, workspace=ws)
    assert e.value.status == moe.UNSUPPORTED_SHAPE
    x = torch.zeros(2, 8 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        attn.qk_norm_rope_append(x, cache, table, lens, n_heads=4)
    with pytest.raises(moe.SeedlessError) as e:  # rows from an odd element on
        attn.qk_norm_rope_append(x[:, 1:513], cache, table, lens, n_heads=4)
    assert e.value.status == moe.INVALID_ARGUMENT
    with pytest.raises(moe.SeedlessError) as e:
        attn.qk_norm_rope_append(x[:, :512].contiguous(), cache, table, lens, n_heads=4, rope=attn.rope_table(100, 24))
    assert e.value.status == moe.UNSUPPORTED_SHAPE
    assert attn.attention(q[:0], cache, table[:0], lens[:0], workspace=ws).shape == (0, 4, 64)


def test_stop_flag_and_wait_limit():
    """A raised stop flag skips the call; waits that give up at once are reported,
    and the workspace serves the next call."""
    args = make_attend(2, [40] * 2, [900, 700], 8, 2, 64, "bf16", seed=31)
    ws = attn.new_workspace(80, 8)
    ref = run_attend(*args, workspace=ws)
    flag = torch.ones(1, dtype=torch.int32, device="cuda")
    q, pool, table, lens, cu = args
    dev = (q.cuda(), attn.KVCache(*cuda(*pool)), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    moe.set_stop_flag(flag)
    try:
        attn.attention(*dev, workspace=ws)
        with pytest.raises(moe.SeedlessError) as e:
            moe.synchronize(workspace=ws)
        assert e.value.status == moe.STOPPED
    finally:
        moe.set_stop_flag(None)
    moe.set_spin_limit(-1)
    try:
        attn.attention(*dev, workspace=ws)
        with pytest.raises(moe.SeedlessError) as e:
            moe.synchronize(workspace=ws)
        assert e.value.status == moe.TIMEOUT
    finally:
        moe.set_spin_limit(0)
    for _ in range(2):
        assert torch.equal(run_attend(*args, workspace=ws), ref)
