"""GPU tests of examples/decode_loop.py: the operators together, a prompt and then
decode steps, against 64-bit restatements and against themselves."""
from __future__ import annotations

import importlib.util
import math
import os

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu


def load():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode_loop.py")
    spec = importlib.util.spec_from_file_location("decode_loop", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def small(ex, layers=2, batch=2, max_len=200):
    cfg = ex.MapleConfig(hidden_size=1024, moe_intermediate_size=512, num_attention_heads=8, num_key_value_heads=2, head_dim=64,
                         vocab_size=5003, num_experts=16, num_experts_per_tok=4, sliding_window=48)
    return ex.Decoder(cfg, layers, batch, max_len)


def prompt(d, n):
    return torch.randint(0, d.cfg.vocab_size, (d.B, n), generator=torch.Generator("cuda").manual_seed(3), device="cuda")


def test_graph_steps_equal_plain_steps():
    ex = load()
    said = []
    for graph in (False, True):
        d = small(ex)
        d.advance(prompt(d, 60))
        step = d.capture().replay if graph else lambda: d.advance(d.token[:, None].clone())  # noqa: B023
        tokens = []
        for _ in range(12):
            step()
            tokens.append(d.token.clone())
        d.check()
        assert d.lens.tolist() == [72, 72] and int((d.history >= 0).sum()) == 144
        said.append(torch.stack(tokens))
    assert torch.equal(*said)


def test_masked_tokens_are_never_said():
    d = small(load())
    d.allowed.zero_()
    d.allowed[:, 3] = 0b1010
    d.advance(prompt(d, 5))
    for _ in range(6):
        assert set(d.token.tolist()) <= {97, 99}
        d.advance(d.token[:, None].clone())
    d.check()


@pytest.mark.parametrize("n", [3, 40])
def test_a_layer_and_the_head_match_64_bits(n):
    """One attention half and the head in 64 bits on the same weights, every result
    rounded to bf16 where the path stores one: norm, projection, queries, attention,
    projection, sum, norm, logits.  Eight roundings of 2^-9 each, at most 2^-8 apart
    where the two sides round to different neighbours, and codes that differ by one of
    127 for a few values: 8 * 2^-8 of the largest magnitudes, in the mean far less."""
    ex = load()
    d = small(ex, layers=1)
    c, la = d.cfg, d.layers[0]
    la["experts"] = {k: torch.zeros_like(v) for k, v in la["experts"].items()}  # experts that add nothing
    tokens = prompt(d, n)
    d.lens += n
    got = d.logits(tokens).cpu().double()
    d.check()

    def bf(x):
        return x.to(torch.bfloat16)

    def rms(x):
        x = x.double()
        return bf(x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + c.rms_norm_eps))

    def mm(x, m):
        return bf(R.qmm4(x, m["w"].cpu(), m["scales"].cpu(), m["biases"].cpu(), ex.GS)[0])

    Hq, Hkv, D = c.num_attention_heads, c.num_key_value_heads, c.head_dim
    h = d.embed[tokens.flatten()].cpu()
    lens, cu, table = [n, n], [0, n, 2 * n], d.table.cpu()
    pages = table.numel()
    empty = (torch.full((pages, Hkv, 64, D), 128, dtype=torch.uint8), torch.full((pages, Hkv, D, 64), 128, dtype=torch.uint8),
             torch.zeros(pages, Hkv), torch.zeros(pages, Hkv))
    one = torch.ones(D)
    q, kk, vv, ks, vs = R.append(mm(rms(h), la["qkv"]), empty, table, lens, cu, Hq, one, one, c.rms_norm_eps, d.rope.cpu(), False)
    code = [torch.nan_to_num(torch.round(x / torch.where(s > 0, s, torch.ones_like(s))[:, :, None, None]) + 128, nan=128.0).to(torch.uint8)
            for x, s in ((kk, ks), (vv, vs))]
    o = R.attention(bf(q), code[0], code[1].transpose(2, 3), ks, vs, table, lens, cu, c.sliding_window)[0]
    h = bf(h.double() + mm(bf(o).flatten(1), la["o"]).double())
    ref = mm(rms(h.view(2, n, -1)[:, -1]), d.head).double()
    assert float((got - ref).norm() / ref.norm()) <= 8 * 2.0 ** -8
    assert not math.isnan(float(got.sum()))
