"""GPU tests of the codes that an append writes for values of 16 bits: the quotient by
the page's scale rounded once, ties to even."""
from __future__ import annotations

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from momij_b200 import attn, moe


def append_values(v, past=0, cache=None):
    """Appends v [n, H, D] (keys the same, without norm or rotation) at position `past`."""
    n, H, D = v.shape
    cache = cache or attn.new_kv_cache(-(-(past + n) // 64), H, D)
    table = torch.arange(cache.k.shape[0], dtype=torch.int32, device="cuda")[None]
    ws = attn.new_workspace(1, H)
    qkv = torch.cat([v, v, v], dim=1).flatten(1).cuda()
    attn.qk_norm_rope_append(qkv, cache, table, torch.tensor([past + n], dtype=torch.int32, device="cuda"), n_heads=H, workspace=ws)
    moe.synchronize(workspace=ws)
    return cache


def codes(cache):
    """K and V codes as [positions, H, D]."""
    k = cache.k.permute(0, 2, 1, 3).flatten(0, 1)
    v = cache.v.permute(0, 3, 1, 2).flatten(0, 1)
    return k.cpu().long() - 128, v.cpu().long() - 128


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("unit", [1.0, 2.0 ** -10, 3.0, 2.0 ** 5])
def test_halves_of_a_code_go_to_the_even_one(unit, D, dtype):
    """amax = 127 units: the values k + 1/2 lie in the middle of two codes (where the type
    holds 127 units; bf16 rounds 381, and the codes go by what it holds)."""
    dt = R.TD[dtype]
    half = torch.arange(-127, 127, dtype=torch.float64) + 0.5
    x = (torch.cat([half, torch.tensor([127.0])]) * unit).repeat(40)[:64 * D].view(64, 1, D)
    ok = x.to(dt).double() == x  # (three units times an odd number of halves may not fit 8 bits)
    x = torch.where(ok, x, torch.zeros_like(x))
    x[0, 0, 0] = 127 * unit
    want = torch.round(x.to(dt).double() * 127 / x.to(dt).double().abs().max()).long()
    for got in codes(append_values(x.to(dt))):
        assert torch.equal(got[:64], want)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n,past", [(64, 0), (130, 0), (40, 24)])
def test_codes_are_the_quotients_rounded_once(n, past, dtype):
    """Random values: every code is the 64-bit quotient by amax / 127 rounded, ties to even
    (a quotient in 32 bits may only differ within 2^-24 of a tie that is none)."""
    H, D = 3, 64
    g = torch.Generator().manual_seed(n)
    dt = R.TD[dtype]
    first = (0.01 * torch.randn(max(past, 1), H, D, generator=g)).to(dt)
    v = torch.randn(n, H, D, generator=g).to(dt)
    cache = attn.new_kv_cache(-(-(past + n) // 64), H, D)
    if past:
        append_values(first, 0, cache)  # smaller: the scale of the page grows to the new rows'
    append_values(v, past, cache)
    for got in codes(cache):
        for page in range(cache.k.shape[0]):
            a, z = max(past, 64 * page), min(past + n, 64 * page + 64)
            x = v[a - past:z - past].double()
            q = x * 127 / x.abs().amax(dim=(0, 2), keepdim=True)
            off = got[a:z] != torch.round(q).long()
            near = (q - torch.floor(q) - 0.5).abs() * 2 ** 24 <= q.abs()
            assert not bool((off & ~(near & (q - torch.floor(q) != 0.5))).any())
