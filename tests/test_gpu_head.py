"""GPU tests of the 4-bit product and the logit processing (momij_b200/head.py)
against 64-bit restatements (tests/attn_ref.py), and of their refusals."""
from __future__ import annotations

import math

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from momij_b200 import head, moe


def weights(N, K, gs, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(-2 ** 31, 2 ** 31, (N, K // 8), generator=g, dtype=torch.int64).to(torch.int32)
    s = (0.002 + 0.004 * torch.rand(N, K // gs, generator=g)).to(R.TD[dtype])
    b = (-7.5 * s.double() * (1 + 0.1 * torch.randn(N, K // gs, generator=g))).to(R.TD[dtype])
    return w, s, b


def check_qmm4(y, x, w, s, b, gs):
    """One rounding of the output; fp32 steps: gs/16 accumulations of 16 products per
    group, one or two per group, the warps' sums."""
    ref, mag = R.qmm4(x, w, s, b, gs)
    K = x.shape[1]
    steps = gs / 16 + 2 * K / gs + 16
    err = (y.cpu().double() - ref).abs()
    bound = 2 * R.HALF_ULP[y.dtype] * ref.abs() + steps * 2.0 ** -23 * mag + 1e-30
    if y.dtype == torch.float16:
        bound = bound + 2.0 ** -25
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K,gs", [
    (1, 1, 64, 64), (1, 16, 128, 128), (2, 17, 192, 64), (3, 100, 320, 64), (8, 33, 256, 128), (9, 50, 640, 128), (16, 64, 1024, 64),
    (17, 40, 384, 128), (33, 70, 512, 64), (40, 129, 2048, 128), (1, 4096, 2048, 64), (5, 3000, 4096, 128), (1, 300, 16384, 64),
    (12, 48, 8192, 128), (1, 40000, 256, 64)])
def test_qmm4_matches_64_bits(M, N, K, gs, dtype):
    w, s, b = weights(N, K, gs, dtype)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(5)).to(R.TD[dtype])
    y = head.qmm4(x.cuda(), w.cuda(), s.cuda(), b.cuda(), gs=gs)
    check_qmm4(y, x, w, s, b, gs)


@pytest.mark.parametrize("M", [1, 3])
@pytest.mark.parametrize("off", [0, 1, 3])
def test_qmm4_strides_and_alignment(M, off):
    """x and out inside wider buffers from any element on; scales that start on 2 bytes only."""
    N, K, gs = 70, 512, 64
    w, s, b = weights(N, K, gs, "bf16", 1)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(6)).bfloat16()
    ref = head.qmm4(x.cuda(), w.cuda(), s.cuda(), b.cuda(), gs=gs)
    wide = torch.zeros(M, K + 24, dtype=x.dtype, device="cuda")
    wide[:, off:off + K] = x.cuda()
    flat = [torch.zeros(t.numel() + 8, dtype=t.dtype, device="cuda") for t in (s, b)]
    views = []
    for f, t in zip(flat, (s, b)):
        f[off:off + t.numel()] = t.cuda().flatten()
        views.append(f[off:off + t.numel()].view(t.shape))
    out = torch.full((M, N + 5), 9.0, dtype=x.dtype, device="cuda")
    y = head.qmm4(wide[:, off:off + K], w.cuda(), *views, gs=gs, out=out[:, 2:2 + N])
    assert y.data_ptr() == out[:, 2:].data_ptr()
    assert torch.equal(y, ref) and (out[:, :2] == 9).all() and (out[:, 2 + N:] == 9).all()


def test_qmm4_magnitudes_and_rows_apart():
    """Tokens of very different size in one call; zeros; a token with an infinity
    or NaN spoils its own row alone."""
    N, K, gs = 40, 256, 64
    w, s, b = weights(N, K, gs, "bf16", 2)
    g = torch.Generator().manual_seed(7)
    x = (torch.randn(6, K, generator=g) * torch.tensor([1.0, 2.0 ** 90, 2.0 ** -90, 0.0, 1.0, 1.0])[:, None]).bfloat16()
    x[4, 3], x[5, 7] = math.inf, math.nan
    y = head.qmm4(x.cuda(), w.cuda(), s.cuda(), b.cuda(), gs=gs)
    check_qmm4(y[:4], x[:4], w, s, b, gs)
    assert (y[3] == 0).all() and not torch.isfinite(y[4:]).any()
    x[0, 1:] = 0  # one element alone, and elements 2^-20 of the largest
    x[0, 0], x[2, 0] = 3.0, x[2].abs().max() * 2.0 ** 20
    y = head.qmm4(x[:4].cuda(), w.cuda(), s.cuda(), b.cuda(), gs=gs)
    check_qmm4(y, x[:4], w, s, b, gs)


def test_qmm4_matrix_past_32_bits():
    """4.4 GB of codes: the last rows."""
    N, K, gs = 2_150_000, 4096, 128
    w = torch.zeros(N, K // 8, dtype=torch.int32, device="cuda")
    s = torch.zeros(N, K // gs, dtype=torch.bfloat16, device="cuda")
    b = torch.zeros(N, K // gs, dtype=torch.bfloat16, device="cuda")
    wt, st, bt = weights(40, K, gs, "bf16", 3)
    w[-40:], s[-40:], b[-40:] = wt.cuda(), st.cuda(), bt.cuda()
    x = torch.randn(1, K, generator=torch.Generator().manual_seed(8)).bfloat16()
    y = head.qmm4(x.cuda(), w, s, b, gs=gs)
    check_qmm4(y[:, -40:], x, wt, st, bt, gs)
    assert (y[:, :-40] == 0).all()


def test_qmm4_stream_graph_and_refusals():
    w, s, b = (t.cuda() for t in weights(64, 256, 64, "bf16", 4))
    x = torch.randn(2, 256, device="cuda").bfloat16()
    ref = head.qmm4(x, w, s, b)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    y = head.qmm4(x, w, s, b, stream=st)
    st.synchronize()
    assert torch.equal(y, ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        z = head.qmm4(x, w, s, b)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(z, ref)
    assert head.qmm4(x[:0], w, s, b).shape == (0, 64)
    for bad, err in ((dict(gs=32), (ValueError, moe.SeedlessError)), (dict(gs=0), ValueError)):
        with pytest.raises(err):
            head.qmm4(x, w, s, b, **bad)
    with pytest.raises(TypeError):
        head.qmm4(x.float(), w, s, b)
    with pytest.raises(TypeError):
        head.qmm4(x, w, s.half(), b)
    with pytest.raises(ValueError):
        head.qmm4(x[:, :128], w, s, b)
    with pytest.raises(ValueError):
        head.qmm4(x.cpu(), w, s, b)
    odd = torch.zeros(64 * 32 + 1, dtype=torch.int32, device="cuda")[1:].view(64, 32)
    with pytest.raises(moe.SeedlessError) as e:
        head.qmm4(x, odd, s, b)
    assert e.value.status == moe.INVALID_ARGUMENT


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K,gs", [
    (2, 128, 256, 64), (2, 129, 320, 64), (3, 1000, 1088, 64), (9, 5000, 384, 128), (16, 300, 2048, 64), (17, 257, 640, 128), (32, 4100, 2112, 64),
    (33, 513, 4096, 128), (20, 20000, 1024, 64), (7, 2500, 12800, 128), (32, 640, 8192, 64), (30, 130, 14336, 128)])
def test_qmm4_several_tokens_match_64_bits(M, N, K, gs, dtype):
    """Sizes with a last tile, batch and token group that are not full, matrices of
    few rows and many columns (shared by several blocks), many rounds of tiles."""
    w, s, b = weights(N, K, gs, dtype, 11)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(12)).to(R.TD[dtype])
    y = head.qmm4(x.cuda(), w.cuda(), s.cuda(), b.cuda(), gs=gs)
    check_qmm4(y, x, w, s, b, gs)
    again = head.qmm4(x.cuda(), w.cuda(), s.cuda(), b.cuda(), gs=gs)
    assert torch.equal(y, again)


@pytest.mark.parametrize("M", [2, 18])
@pytest.mark.parametrize("off", [0, 1, 3])
def test_qmm4_several_tokens_strides_and_alignment(M, off):
    N, K, gs = 200, 1024, 64
    w, s, b = weights(N, K, gs, "bf16", 13)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(14)).bfloat16()
    ref = head.qmm4(x.cuda(), w.cuda(), s.cuda(), b.cuda(), gs=gs)
    check_qmm4(ref, x, w, s, b, gs)
    wide = torch.zeros(M, K + 24, dtype=x.dtype, device="cuda")
    wide[:, off:off + K] = x.cuda()
    views = []
    for t in (s, b):
        f = torch.zeros(t.numel() + 8, dtype=t.dtype, device="cuda")
        f[off:off + t.numel()] = t.cuda().flatten()
        views.append(f[off:off + t.numel()].view(t.shape))
    out = torch.full((M, N + 5), 9.0, dtype=x.dtype, device="cuda")
    y = head.qmm4(wide[:, off:off + K], w.cuda(), *views, gs=gs, out=out[:, 2:2 + N])
    assert torch.equal(y, ref) and (out[:, :2] == 9).all() and (out[:, 2 + N:] == 9).all()


def test_qmm4_several_tokens_magnitudes():
    N, K, gs = 150, 512, 64
    w, s, b = weights(N, K, gs, "bf16", 15)
    g = torch.Generator().manual_seed(16)
    x = (torch.randn(6, K, generator=g) * torch.tensor([1.0, 2.0 ** 90, 2.0 ** -90, 0.0, 1.0, 1.0])[:, None]).bfloat16()
    x[4, 3], x[5, 400] = math.inf, math.nan
    y = head.qmm4(x.cuda(), w.cuda(), s.cuda(), b.cuda(), gs=gs)
    check_qmm4(y[:4], x[:4], w, s, b, gs)
    assert (y[3] == 0).all() and not torch.isfinite(y[4:]).any()


def test_qmm4_matrix_past_32_bits_several_tokens():
    N, K, gs = 2_150_000, 4096, 128
    w = torch.zeros(N, K // 8, dtype=torch.int32, device="cuda")
    s = torch.zeros(N, K // gs, dtype=torch.bfloat16, device="cuda")
    b = torch.zeros(N, K // gs, dtype=torch.bfloat16, device="cuda")
    wt, st, bt = weights(40, K, gs, "bf16", 3)
    w[-40:], s[-40:], b[-40:] = wt.cuda(), st.cuda(), bt.cuda()
    x = torch.randn(3, K, generator=torch.Generator().manual_seed(8)).bfloat16()
    y = head.qmm4(x.cuda(), w, s, b, gs=gs)
    check_qmm4(y[:, -40:], x, wt, st, bt, gs)
    assert (y[:, :-40] == 0).all()


def test_qmm4_stop_flag_and_wait_limit():
    """A raised stop flag leaves the output as it was; waits that give up at once show
    as NaN or not at all, and the next call is right."""
    w, s, b = (t.cuda() for t in weights(3000, 2048, 64, "bf16", 17))
    x = torch.randn(12, 2048, device="cuda").bfloat16()
    ref = head.qmm4(x, w, s, b)
    out = torch.full_like(ref, 5.0)
    flag = torch.ones(1, dtype=torch.int32, device="cuda")
    moe.set_stop_flag(flag)
    try:
        head.qmm4(x, w, s, b, out=out)
        torch.cuda.synchronize()
    finally:
        moe.set_stop_flag(None)
    assert (out == 5).all()
    moe.set_spin_limit(-1)
    try:
        head.qmm4(x, w, s, b, out=out)
        torch.cuda.synchronize()
    finally:
        moe.set_spin_limit(0)
    assert bool((torch.isnan(out) | (out == ref)).all())
    for _ in range(2):
        assert torch.equal(head.qmm4(x, w, s, b), ref)


# ---- logits -----------------------------------------------------------------------------

def check_logits(out, ref, size):
    """Five fp32 steps at most, each relative to what it adds up."""
    out = out.cpu().double()
    inf = torch.isinf(ref)
    assert torch.equal(out[inf], ref[inf])
    err = (out - ref).abs()[~inf]
    assert bool((err <= 5 * 2.0 ** -24 * size[~inf] + 1e-30).all()), float(err.max())


def make_logits(B, V, hist, nb, mask, dtype, seed=0, skew=True):
    g = torch.Generator().manual_seed(seed)
    l = (3 * torch.randn(B, V, generator=g)).to({"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[dtype])
    counts = [hist if b == 0 else (hist * ((b * 7) % 5)) // 5 for b in range(B)]
    ids = (torch.rand(sum(counts), generator=g) ** (3 if skew else 1) * (V + 2)).int() - 1  # -1 and V among them
    cub = R.offsets([nb if b % 3 else nb // 2 for b in range(B)])
    bids = (torch.rand(cub[-1], generator=g) ** 2 * (V + 1)).int()  # doubles among them
    return dict(l=l, hist=ids, cu=R.offsets(counts), rep=1 + 0.4 * torch.rand(B, generator=g), pres=torch.rand(B, generator=g),
                freq=0.3 * torch.rand(B, generator=g), ids=bids, bias=4 * torch.randn(cub[-1], generator=g), cub=cub,
                allowed=torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32), generator=g, dtype=torch.int64).int() if mask else None)


def run_logits(a, **kw):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    return head.process_logits(kw.pop("logits", None) if "logits" in kw else a["l"].cuda(), history=a["hist"].cuda(), cu_history=i32(a["cu"]),
                               repetition=a["rep"].cuda(), presence=a["pres"].cuda(), frequency=a["freq"].cuda(), bias_ids=a["ids"].cuda(),
                               bias=a["bias"].cuda(), cu_bias=i32(a["cub"]), allowed=None if a["allowed"] is None else a["allowed"].cuda(), **kw)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,V,hist,nb,mask", [
    (1, 1, 3, 2, True), (1, 33, 1, 0, True), (3, 1000, 50, 9, False), (2, 1027, 700, 40, True), (5, 5000, 3000, 300, True),
    (4, 151936 // 4, 1, 1, True), (2, 70001, 20000, 5, True)])
def test_logits_match_64_bits(B, V, hist, nb, mask, dtype):
    a = make_logits(B, V, hist, nb, mask, dtype)
    check_logits(run_logits(a), *R.logits(**a))


@pytest.mark.parametrize("V", [130_000, 129_999])
def test_logits_large_batch(V):
    """Enough tokens for the copy and the named tokens to be kernels of their own."""
    a = make_logits(20, V, 3000, 100, True, "bf16", seed=2)
    check_logits(run_logits(a), *R.logits(**a))


def test_logits_parts_left_out():
    a = make_logits(3, 999, 100, 10, True, "f32", seed=3)
    x = a["l"].cuda()
    assert torch.equal(head.process_logits(x), x)
    none = dict(hist=None, cu=None, rep=None, pres=None, freq=None, ids=None, bias=None, cub=None)
    out = head.process_logits(x, allowed=a["allowed"].cuda())
    check_logits(out, *R.logits(a["l"], **none, allowed=a["allowed"]))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    out = head.process_logits(x, history=a["hist"].cuda(), cu_history=i32(a["cu"]), presence=a["pres"].cuda())
    one = dict(none, hist=a["hist"], cu=a["cu"], rep=torch.ones(3), pres=a["pres"], freq=torch.zeros(3))
    check_logits(out, *R.logits(a["l"], **one, allowed=None))
    out = head.process_logits(x, bias_ids=a["ids"].cuda(), bias=a["bias"].cuda(), cu_bias=i32(a["cub"]))
    check_logits(out, *R.logits(a["l"], **dict(none, ids=a["ids"], bias=a["bias"], cub=a["cub"]), allowed=None))


@pytest.mark.parametrize("B", [2, 20])
def test_logits_rows_masked_whole_and_special_values(B):
    V = 130_000 if B == 20 else 500
    a = make_logits(B, V, 60, 6, True, "f32", seed=4)
    a["allowed"][0] = 0
    a["l"][1, 5], a["l"][1, 6], a["l"][1, 7] = math.inf, -math.inf, math.nan
    a["hist"][a["cu"][1]:a["cu"][1] + 3] = torch.tensor([5, 6, 7], dtype=torch.int32)
    a["allowed"][1, 0] = -1
    out = run_logits(a)
    assert (out[0] == -math.inf).all()
    assert out[1, 5] == math.inf and out[1, 6] == -math.inf and torch.isnan(out[1, 7])
    ref, size = R.logits(**a)
    check_logits(out[2:], ref[2:], size[2:])


def test_logits_strides_alignment_and_in_place():
    a = make_logits(3, 1000, 200, 20, True, "f32", seed=5)
    ref = run_logits(a)
    wide = torch.zeros(3, 1100, device="cuda")
    for off in (0, 1, 4):
        wide[:, off:off + 1000] = a["l"].cuda()
        assert torch.equal(run_logits(a, logits=wide[:, off:off + 1000]), ref)
    for off in (1, 2, 3):  # histories that start anywhere
        flat = torch.zeros(a["hist"].numel() + 4, dtype=torch.int32)
        flat[off:off + a["hist"].numel()] = a["hist"]
        i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
        out = head.process_logits(a["l"].cuda(), history=flat.cuda()[off:off + a["hist"].numel()], cu_history=i32(a["cu"]),
                                  repetition=a["rep"].cuda(), presence=a["pres"].cuda(), frequency=a["freq"].cuda(),
                                  bias_ids=a["ids"].cuda(), bias=a["bias"].cuda(), cu_bias=i32(a["cub"]), allowed=a["allowed"].cuda())
        assert torch.equal(out, ref)
    x = a["l"].cuda()
    assert torch.equal(run_logits(a, logits=x, out=x), ref) and torch.equal(x, ref)
    big = make_logits(20, 130_000, 500, 20, True, "f32", seed=6)
    y = big["l"].cuda()
    want = run_logits(big)
    assert torch.equal(run_logits(big, logits=y, out=y), want)


def test_logits_refusals():
    x = torch.zeros(2, 100, device="cuda")
    h = torch.zeros(3, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        head.process_logits(x, history=h)
    with pytest.raises(ValueError):
        head.process_logits(x, history=h, cu_history=cu[:2])
    with pytest.raises(TypeError):
        head.process_logits(x, history=h.long(), cu_history=cu)
    with pytest.raises(TypeError):
        head.process_logits(x.double())
    with pytest.raises(ValueError):
        head.process_logits(x, repetition=torch.ones(3, device="cuda"))
    with pytest.raises(ValueError):
        head.process_logits(x, bias_ids=h, bias=torch.zeros(2, device="cuda"), cu_bias=cu)
    with pytest.raises(ValueError):
        head.process_logits(x, allowed=torch.zeros(2, 3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        head.process_logits(x.cpu())
    assert head.process_logits(x[:0]).shape == (0, 100)
