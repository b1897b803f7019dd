"""GPU tests of what the attention half must survive: a stop flag that the blocks of
one launch see differently, streams of the caller's, blocks that walk several pieces,
and arguments at the edges of their ranges."""
from __future__ import annotations

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from momij_b200 import attn, moe


def device_args(B, n, length, Hq, Hkv, D, dtype, seed=0):
    """(q, cache, table, lens) on the device, all sequences of one length."""
    table, pages = R.block_tables([length] * B, seed)
    cache = attn.KVCache(*(t.cuda() for t in R.random_pool(pages, Hkv, D, seed + 1)))
    q = (torch.randn(B * n, Hq, D, generator=torch.Generator().manual_seed(seed + 2)) * 1.5).to(R.TD[dtype]).cuda()
    return q, cache, table.cuda(), torch.full((B,), length, dtype=torch.int32, device="cuda")


# Rows of at most 16 a head (a join within the launch), more with few heads (a join
# launch of its own) and with many (joins within the launch).
STOPPED = [(1, 1, 3000, 8, 2, 128), (1, 40, 3000, 8, 2, 64), (6, 40, 3000, 32, 8, 64)]


@pytest.mark.parametrize("B,n,length,Hq,Hkv,D", STOPPED)
def test_stop_flag_seen_by_some_blocks(B, n, length, Hq, Hkv, D):
    """Some blocks of a launch see the flag, others do not, block 0 among either: the call
    is reported as stopped, what is written is what a whole call writes, and the
    workspace serves the next calls."""
    args = device_args(B, n, length, Hq, Hkv, D, "bf16")
    ws = attn.new_workspace(B * n, Hq)
    ref = attn.attention(*args, workspace=ws)
    moe.synchronize(workspace=ws)
    g = torch.Generator().manual_seed(4)
    blocks = moe.lib.momij_device_sm_count()
    for raised in (1, blocks // 2, blocks - 1, None):
        flag = torch.zeros(4096, dtype=torch.int32)
        flag[torch.randperm(blocks - 1, generator=g)[:raised] + 1 if raised else [0]] = 1  # (None: block 0 alone)
        out = torch.full_like(ref, 77.0)
        flag = flag.cuda()
        moe.set_stop_flag(flag)
        moe.set_stop_step(1)
        try:
            attn.attention(*args, out=out, workspace=ws)
            torch.cuda.synchronize()
        finally:
            moe.set_stop_step(0)
            moe.set_stop_flag(None)
        # (what blocks share is written by whoever joins it, or left)
        assert bool(((out == ref) | (out == 77)).all())
        if raised != 1:  # (a single block may have had nothing to do)
            assert bool((out == 77).any())
        attn.attention(*args, workspace=ws)  # a later call's own word does not hide it
        with pytest.raises(moe.SeedlessError) as e:
            moe.synchronize(workspace=ws)
        assert e.value.status == moe.STOPPED
        for _ in range(2):
            assert torch.equal(attn.attention(*args, workspace=ws), ref)
            moe.synchronize(workspace=ws)


def test_stop_flag_seen_by_some_blocks_of_an_append():
    _, cache, table, lens = device_args(2, 1, 300, 4, 2, 64, "bf16")
    x = torch.randn(2 * 200, 8 * 64, device="cuda").bfloat16()
    ws = attn.new_workspace(1, 1)
    flag = torch.zeros(4096, dtype=torch.int32, device="cuda")
    flag[3] = 1
    for call in (lambda: attn.qk_norm_rope_append(x, cache, table, lens, n_heads=4, workspace=ws),
                 lambda: attn.cache_read(cache, table, lens, count=300, workspace=ws)):
        moe.set_stop_flag(flag)
        moe.set_stop_step(1)
        try:
            call()
            torch.cuda.synchronize()
        finally:
            moe.set_stop_step(0)
            moe.set_stop_flag(None)
        with pytest.raises(moe.SeedlessError) as e:
            moe.synchronize(workspace=ws)
        assert e.value.status == moe.STOPPED
        call()
        moe.synchronize(workspace=ws)


@pytest.mark.parametrize("B,n,length,Hq,Hkv,D", STOPPED[1:])
def test_waits_that_give_up_leave_nothing_behind(B, n, length, Hq, Hkv, D):
    """Outputs are a whole call's or as they were, not joined from what is missing."""
    args = device_args(B, n, length, Hq, Hkv, D, "f16")
    ws = attn.new_workspace(B * n, Hq)
    ref = attn.attention(*args, workspace=ws)
    moe.synchronize(workspace=ws)
    out = torch.full_like(ref, 77.0)
    moe.set_spin_limit(-1)
    try:
        attn.attention(*args, out=out, workspace=ws)
        with pytest.raises(moe.SeedlessError) as e:
            moe.synchronize(workspace=ws)
        assert e.value.status == moe.TIMEOUT
    finally:
        moe.set_spin_limit(0)
    assert bool(((out == ref) | (out == 77)).all())
    for _ in range(2):
        assert torch.equal(attn.attention(*args, workspace=ws), ref)
        moe.synchronize(workspace=ws)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("B,n,Hq,Hkv,D,window", [(24, 40, 32, 8, 64, 0), (20, 50, 24, 8, 128, 100), (3, 700, 16, 4, 64, 300)])
def test_blocks_that_walk_several_pieces(B, n, Hq, Hkv, D, window, dtype):
    """More (row tile, head)s than SMs, of unequal lengths: a block carries its stages,
    phases and shared arrays from one piece to the next."""
    lens = [n + (b * 97) % 400 for b in range(B)]
    table, pages = R.block_tables(lens, 1)
    pool = R.random_pool(pages, Hkv, D, 2)
    q = (torch.randn(B * n, Hq, D, generator=torch.Generator().manual_seed(3)) * 1.5).to(R.TD[dtype])
    ws = attn.new_workspace(B * n, Hq)
    args = (q.cuda(), attn.KVCache(*(t.cuda() for t in pool)), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    out = attn.attention(*args, window=window, workspace=ws)
    moe.synchronize(workspace=ws)
    rows = torch.arange(0, B * n, 7)  # (every seventh token in 64 bits; the others by repetition)
    for b in range(B):
        at = rows[(rows >= b * n) & (rows < (b + 1) * n)]
        for t in at.tolist():
            length = lens[b] - n + (t - b * n) + 1
            ref, mag, big = R.attention(q[t:t + 1], *pool, table[b:b + 1], [length], [0, 1], window)
            err = (out[t:t + 1].cpu().double() - ref).abs()
            assert bool((err <= R.attention_bound(ref, mag, big, D, q.dtype)).all()), (b, t)
    for _ in range(20):
        assert torch.equal(attn.attention(*args, window=window, workspace=ws), out)
    moe.synchronize(workspace=ws)


@pytest.mark.parametrize("handle", [False, True])
@pytest.mark.parametrize("n", [1, 40])
def test_a_stream_of_the_callers_beside_a_busy_one(n, handle):
    """The current stream is busy, the call's stream is not: nothing that the call needs
    (a workspace of its own, filled with zeros) may wait for the busy one, and what it
    allocates is not memory that the busy one still uses."""
    from momij_b200 import head
    args = device_args(2, n, 2000, 8, 2, 64, "bf16")
    ref = attn.attention(*args)
    w, s, b = torch.randint(0, 1 << 30, (64, 32), dtype=torch.int32, device="cuda"), *(torch.rand(64, 4, device="cuda").bfloat16() for _ in range(2))
    x = torch.randn(2, 256, device="cuda").bfloat16()
    qkv = torch.randn(2 * n, 12 * 64, device="cuda").bfloat16()
    y, kv = head.qmm4(x, w, s, b), attn.cache_read(*args[1:], count=70)
    cache = attn.KVCache(*(t.clone() for t in (args[1].k, args[1].v, args[1].k_scale, args[1].v_scale)))
    q = attn.qk_norm_rope_append(qkv, cache, *args[2:], n_heads=8)
    logits = torch.randn(2, 500, device="cuda")
    side = torch.cuda.Stream()
    given = side.cuda_stream if handle else side
    size = attn.workspace_size(2 * n, 8)
    torch.cuda.synchronize()
    for _ in range(3):
        busy = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]  # freed memory full of ones
        busy += [torch.full((ref.numel(),), 1.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        torch.cuda._sleep(200_000_000)  # about a tenth of a second
        for t in busy:
            t.fill_(1)  # enqueued behind it, and then freed
        del t, busy
        out = attn.attention(*args, stream=given)
        y2, kv2 = head.qmm4(x, w, s, b, stream=given), attn.cache_read(*args[1:], count=70, stream=given)
        q2 = attn.qk_norm_rope_append(qkv, cache, *args[2:], n_heads=8, stream=given)
        l2 = head.process_logits(logits, stream=given)
        side.synchronize()
        torch.cuda.synchronize()
        for a, r in ((out, ref), (y2, y), (kv2[0], kv[0]), (kv2[1], kv[1]), (q2, q), (l2, logits)):
            assert torch.equal(a, r)


@pytest.mark.parametrize("length", [30, 400])
def test_attention_with_nothing_to_join_is_over_before_the_next_operator(length):
    """Few heads and 17 rows or more bring a joining launch, which a short context leaves
    nothing to do; what comes next reads the main kernel's results all the same."""
    from momij_b200 import head
    q, *rest = device_args(1, 20, length, 4, 1, 64, "bf16")
    w = torch.randint(-2 ** 31, 2 ** 31, (300, 32), dtype=torch.int64, device="cuda").to(torch.int32)
    s, b = (torch.rand(300, 4, device="cuda").bfloat16() - 0.5 for _ in range(2))
    ws, out = attn.new_workspace(20, 4), torch.empty_like(q)
    wants, gots = [], []
    qs = [torch.randn_like(q) for _ in range(40)]
    for x in qs:
        o = attn.attention(x, *rest, workspace=ws)
        torch.cuda.synchronize()
        wants.append(head.qmm4(o.flatten(1), w, s, b))
    torch.cuda.synchronize()
    for x in qs:
        gots.append(head.qmm4(attn.attention(x, *rest, out=out, workspace=ws).flatten(1), w, s, b))
    moe.synchronize(workspace=ws)
    for a, r in zip(gots, wants):
        assert torch.equal(a, r)


@pytest.mark.parametrize("n", [5, 40])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 30, 512, 511])
def test_windows_wider_than_the_cache(n, window):
    """Wider than anything, with caches shorter than the queries (positions below zero)."""
    lens = [2, 500, 0, n, 130]
    table, pages = R.block_tables(lens, 6)
    cache = attn.KVCache(*(t.cuda() for t in R.random_pool(pages, 2, 64, 7)))
    q = torch.randn(5 * n, 8, 64, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    ws = attn.new_workspace(5 * n, 8)
    args = (q, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    assert table.shape[1] * 64 == 512
    out = [attn.attention(*args, window=w, workspace=ws) for w in (0, window)]
    moe.synchronize(workspace=ws)
    assert torch.equal(*out)
    assert (out[0][:n - 2] == 0).all() and not (out[0][n - 2:n] == 0).all()


@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize("bad", [-2 ** 31, -2 ** 31 + 1, -1, 257, 2 ** 31 - 1, 2 ** 31 - 64])
def test_append_skips_and_reports_lengths_out_of_range(n, bad):
    """With and without a table of angles: lengths that positions computed from them would
    wrap at are skipped like any other, and the sequence beside them is served."""
    for rope in (None, attn.rope_table(256, 64)):
        _, cache, table, lens = device_args(2, 1, 256, 4, 2, 64, "bf16")  # (four columns)
        x = torch.randn(2 * n, 8 * 64, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
        ws = attn.new_workspace(1, 1)
        tensors = (cache.k, cache.v, cache.k_scale, cache.v_scale)
        good = attn.KVCache(*(t.clone() for t in tensors))
        ref = attn.qk_norm_rope_append(x[:n], good, table[:1], lens[:1], n_heads=4, rope=rope, workspace=ws)
        moe.synchronize(workspace=ws)
        lens[1] = bad
        q = attn.qk_norm_rope_append(x, cache, table, lens, n_heads=4, rope=rope, workspace=ws)
        with pytest.raises(moe.SeedlessError) as e:
            moe.synchronize(workspace=ws)
        assert e.value.status == 11
        assert torch.equal(q[:n], ref) and all(torch.equal(a, getattr(good, f)) for a, f in zip(tensors, ("k", "v", "k_scale", "v_scale")))


def test_tables_wider_than_positions_can_count_are_refused():
    q, cache, _, lens = device_args(1, 1, 64, 4, 2, 64, "bf16")
    table = torch.zeros(1, 2 ** 24 + 1, dtype=torch.int32, device="cuda")
    ws = attn.new_workspace(1, 4)
    for call in (lambda: attn.attention(q, cache, table, lens, workspace=ws),
                 lambda: attn.qk_norm_rope_append(torch.zeros(1, 8 * 64, dtype=q.dtype, device="cuda"), cache, table, lens, n_heads=4)):
        with pytest.raises(moe.SeedlessError) as e:
            call()
        assert e.value.status == moe.UNSUPPORTED_SHAPE


@pytest.mark.parametrize("n", [1, 17])
def test_the_longest_context(n):
    """2^30 tokens, all of them one page: with queries of zeros, the mean of its values.
    Bound: every sum in the order of the tokens, 2^-23 for each of a block's additions
    (its tiles, or its warps' half pages, and the products' steps of 16 tokens)."""
    table = torch.zeros(1, 2 ** 24, dtype=torch.int32, device="cuda")
    pool = R.random_pool(1, 1, 64, 5)
    cache = attn.KVCache(*(t.cuda() for t in pool))
    lens = torch.tensor([2 ** 30], dtype=torch.int32, device="cuda")
    ws = attn.new_workspace(n, 1)
    out = attn.attention(torch.zeros(n, 1, 64, dtype=torch.bfloat16, device="cuda"), cache, table, lens, workspace=ws)
    moe.synchronize(workspace=ws)
    v = R.values(*pool)[1][0, 0]
    want, mag = v.mean(0), v.abs().mean(0)  # (the last queries miss up to 16 of 2^30 tokens)
    steps = 2 ** 30 / 16 / moe.lib.momij_device_sm_count()
    err = (out[:, 0].cpu().double() - want).abs()
    assert bool((err <= 2 ** -8 * want.abs() + 2 * steps * 2 ** -23 * mag).all()), float((err / mag).max())


def test_workspaces_that_do_not_lie_where_their_bytes_say_are_refused():
    q, cache, table, lens = device_args(1, 1, 64, 4, 2, 64, "bf16")
    x = torch.zeros(1, 8 * 64, dtype=q.dtype, device="cuda")
    n = attn.workspace_size(1, 4)
    calls = (lambda ws: attn.attention(q, cache, table, lens, workspace=ws),
             lambda ws: attn.qk_norm_rope_append(x, cache, table, lens, n_heads=4, workspace=ws),
             lambda ws: attn.cache_read(cache, table, lens, count=4, workspace=ws))
    for call in calls:
        for bad in (torch.zeros(1, dtype=torch.uint8, device="cuda").expand(n), torch.zeros(2 * n, dtype=torch.uint8, device="cuda")[::2]):
            with pytest.raises(ValueError):
                call(bad)
        for off in (1, 2, 4):
            with pytest.raises(moe.SeedlessError) as e:
                call(torch.zeros(n + 16, dtype=torch.uint8, device="cuda")[off:off + n])
            assert e.value.status == moe.INVALID_ARGUMENT
        call(torch.zeros(n + 16, dtype=torch.uint8, device="cuda")[16:])
    torch.cuda.synchronize()


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("mult", [2.0 ** -45, 2.0 ** -20, 2.0 ** 30])
def test_pages_of_zeros_beside_small_and_large_values(mult, n):
    """Values scaled down or up, two pages of zeros (one of each parity, one of them the
    first) among them: the others keep their bits, the zeros their weight."""
    lens, Hkv, D = [400], 2, 64
    table, pages = R.block_tables(lens, 9)
    k, v, ks, vs = R.random_pool(pages, Hkv, D, 10)
    vs *= mult
    for i in (0, 3):
        p = int(table[0, i])
        v[p], vs[p] = 128, 0.0
    q = torch.randn(n, 8, D, generator=torch.Generator().manual_seed(11)).bfloat16()
    ws = attn.new_workspace(n, 8)
    out = attn.attention(q.cuda(), attn.KVCache(k.cuda(), v.cuda(), ks.cuda(), vs.cuda()), table.cuda(),
                         torch.tensor(lens, dtype=torch.int32).cuda(), workspace=ws)
    moe.synchronize(workspace=ws)
    ref, mag, big = R.attention(q, k, v, ks, vs, table, lens, [0, n])
    bound = R.attention_bound(ref / mult, mag / mult, big, D, q.dtype) * mult  # (its last term is for values near one)
    err = (out.cpu().double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("bad", [-1, -2 ** 31, 257, 2 ** 31 - 1])
def test_cache_read_reports_lengths_out_of_range(bad):
    _, cache, table, lens = device_args(2, 1, 256, 4, 2, 64, "bf16")  # (four columns)
    ws = attn.new_workspace(1, 1)
    want = attn.cache_read(cache, table, lens, count=100, workspace=ws)
    moe.synchronize(workspace=ws)
    lens[0] = bad
    got = attn.cache_read(cache, table, lens, count=100, workspace=ws)
    with pytest.raises(moe.SeedlessError) as e:
        moe.synchronize(workspace=ws)
    assert e.value.status == 11
    for a, r in zip(got, want):
        assert torch.equal(a[1], r[1])
        assert torch.equal(a[0], torch.zeros_like(r[0]) if bad < 0 else r[0])  # (the pages that are there)


def test_refusals_of_odd_arguments():
    q, cache, table, lens = device_args(1, 2, 64, 4, 2, 64, "bf16")
    x = torch.zeros(2, 8 * 64, dtype=q.dtype, device="cuda")
    ws = attn.new_workspace(2, 4)
    for bad, err in ((None, TypeError), (3, TypeError), (q[0], ValueError), (q.cpu(), ValueError)):
        for kw in ({}, dict(workspace=ws)):
            with pytest.raises(err):
                attn.attention(bad, cache, table, lens, **kw)
    with pytest.raises(RuntimeError):  # a truth value that there is not
        attn.qk_norm_rope_append(x, cache, table, lens, n_heads=4, interleaved=torch.zeros(2, device="cuda"))
    for call in (lambda: attn.attention(q, cache, table[:0], lens[:0], workspace=ws),  # rows of no sequence
                 lambda: attn.qk_norm_rope_append(x, cache, table[:0], lens[:0], n_heads=4)):
        with pytest.raises(moe.SeedlessError) as e:
            call()
        assert e.value.status == moe.INVALID_ARGUMENT


def shared_pages(B, cols, Hkv, D, seed=0):
    """Sequences that read pages of one small pool: (pool, table)."""
    pool = R.random_pool(50, Hkv, D, seed)
    return pool, torch.randint(0, 50, (B, cols), generator=torch.Generator().manual_seed(seed + 1), dtype=torch.int32)


def test_more_sequences_than_a_launch_takes():
    B, Hq, D = 4_100, 4, 64
    pool, table = shared_pages(B, 2, 1, D)
    lens = [1 + (b * 37) % 128 for b in range(B)]
    q = torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(2)).bfloat16()
    ws = attn.new_workspace(B, Hq)
    out = attn.attention(q.cuda(), attn.KVCache(*(t.cuda() for t in pool)), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), workspace=ws)
    moe.synchronize(workspace=ws)
    ref, mag, big = R.attention(q, *pool, table, lens, list(range(B + 1)))
    assert bool(((out.cpu().double() - ref).abs() <= R.attention_bound(ref, mag, big, D, q.dtype)).all())


def test_more_row_tiles_than_a_launch_takes():
    """34 sequences of 128 row tiles (32 a launch); a window of one: each token's output is
    its own value.  And a sequence of more tiles than a launch takes is refused."""
    B, n, Hq, D = 34, 2048, 8, 64
    pool, table = shared_pages(B, n // 64, 1, D)
    q = torch.randn(B * n, Hq, D, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    cache = attn.KVCache(*(t.cuda() for t in pool))
    ws = attn.new_workspace(B * n, Hq)
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    out = attn.attention(q, cache, table.cuda(), lens, window=1, workspace=ws)
    moe.synchronize(workspace=ws)
    want = R.values(*pool)[1].cuda()[table.long().cuda()][:, :, 0].reshape(B * n, 1, D)
    err = (out.double() - want).abs()
    assert bool((err <= R.attention_bound(want, want.abs(), 0.0, D, q.dtype)).all())
    # 65,537 tokens of eight heads to a kv head: 4,097 tiles
    big = torch.zeros(65_537, 8, D, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(moe.SeedlessError) as e:
        attn.attention(big, cache, torch.zeros(1, 1025, dtype=torch.int32, device="cuda"),
                       torch.tensor([65_537], dtype=torch.int32, device="cuda"), workspace=ws)
    assert e.value.status == moe.UNSUPPORTED_SHAPE
