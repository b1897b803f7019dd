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
