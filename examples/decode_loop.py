"""Prompt and decoding loop over the operators of momij_b200: head norms with
rotation and append, attention over the 8-bit paged cache, 4-bit projections, the
MoE block, and logits with penalties and a mask.

    python examples/decode_loop.py --layers 4 --batch 2 --prompt 200 --steps 64

Weights are random (the shapes are loader.MapleConfig's, or what the options say),
so the tokens mean nothing; the calls, their buffers and their order are those of a
decoder.  A decode step is one CUDA graph: every length, table and history lies on
the device at a fixed address, and the step itself moves them on.
"""
from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from momij_b200 import attn, head, moe  # noqa: E402
from momij_b200.loader import MapleConfig  # noqa: E402

GS = 64  # columns per scale of the 4-bit matrices and the experts


def random_qmm4(n: int, k: int, seed: int) -> dict:
    """A random 4-bit matrix [n, k] with entries of variance 1/k."""
    g = torch.Generator("cuda").manual_seed(seed)
    w = torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), generator=g, dtype=torch.int64, device="cuda").to(torch.int32)
    s = torch.full((n, k // GS), (12 / 255 / k) ** 0.5, dtype=torch.bfloat16, device="cuda")
    return dict(w=w, scales=s, biases=(-7.5 * s.float()).bfloat16())


class Decoder:
    def __init__(self, cfg: MapleConfig, layers: int, batch: int, max_len: int, seed: int = 0):
        self.cfg, self.B, self.max_len = cfg, batch, max_len
        H, Hq, Hkv, D = cfg.hidden_size, cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
        one = torch.ones(H, dtype=torch.bfloat16, device="cuda")
        g = torch.Generator("cuda").manual_seed(seed)
        self.embed = torch.randn(cfg.vocab_size, H, generator=g, device="cuda", dtype=torch.bfloat16)
        columns = -(-max_len // attn.PAGE)
        self.table = torch.arange(batch * columns, dtype=torch.int32, device="cuda").view(batch, columns)
        self.layers = []
        for i in range(layers):
            s = seed + 100 * (i + 1)
            self.layers.append(dict(
                norm=one, qkv=random_qmm4((Hq + 2 * Hkv) * D, H, s + 1), o=random_qmm4(H, Hq * D, s + 2),
                q_norm=one[:D].contiguous(), k_norm=one[:D].contiguous(), cache=attn.new_kv_cache(batch * columns, Hkv, D),
                gate=(torch.randn(cfg.num_experts, H, generator=g, device="cuda") * H ** -0.5).bfloat16(),
                experts=moe.device_expert_weights(cfg.num_experts, H, cfg.moe_intermediate_size, GS, layer=i, seed=seed)))
        self.norm, self.head = one, random_qmm4(cfg.vocab_size, H, seed + 3)
        self.rope = attn.rope_table(max_len, int(D * cfg.partial_rotary_factor), cfg.rope_theta)
        # What a sequence has said: unused places hold -1, which names no token.
        self.history = torch.full((batch, max_len), -1, dtype=torch.int32, device="cuda")
        self.cu_history = torch.arange(batch + 1, dtype=torch.int32, device="cuda") * max_len
        self.repetition = torch.full((batch,), 1.1, device="cuda")
        self.frequency = torch.full((batch,), 0.2, device="cuda")
        self.allowed = torch.full((batch, -(-cfg.vocab_size // 32)), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.token = torch.zeros(batch, dtype=torch.long, device="cuda")
        self.workspaces = {}

    def buffers(self, n: int) -> tuple:
        """Workspaces of a call with ``n`` tokens a sequence, kept for the next one."""
        if n not in self.workspaces:
            c, M = self.cfg, self.B * n
            self.workspaces[n] = (attn.new_workspace(M, c.num_attention_heads),
                                  torch.zeros(moe.block_workspace_size(M, c.num_experts_per_tok, c.hidden_size, c.moe_intermediate_size,
                                                                       c.num_experts), dtype=torch.uint8, device="cuda"))
        return self.workspaces[n]

    def logits(self, tokens: torch.Tensor) -> torch.Tensor:
        """Logits [B, V] after the next ``tokens`` [B, n]; ``lens`` counts them already."""
        c, (B, n) = self.cfg, tokens.shape
        ws, block_ws = self.buffers(n)
        h = self.embed[tokens.flatten()]
        for la in self.layers:
            x = moe.rms_norm(h, la["norm"], c.rms_norm_eps)
            qkv = head.qmm4(x, **la["qkv"], gs=GS)
            q = attn.qk_norm_rope_append(qkv, la["cache"], self.table, self.lens, n_heads=c.num_attention_heads, q_weight=la["q_norm"],
                                         k_weight=la["k_norm"], eps=c.rms_norm_eps, rope=self.rope, workspace=ws)
            o = attn.attention(q, la["cache"], self.table, self.lens, window=c.sliding_window, workspace=ws)
            h += head.qmm4(o.flatten(1), **la["o"], gs=GS)
            moe.moe_block(h, la["norm"], c.rms_norm_eps, la["gate"], la["experts"], I=c.moe_intermediate_size,
                          Ktop=c.num_experts_per_tok, gs=GS, workspace=block_ws)
        last = h.view(B, n, -1)[:, -1].contiguous()
        return head.qmm4(moe.rms_norm(last, self.norm, c.rms_norm_eps), **self.head, gs=GS)

    def advance(self, tokens: torch.Tensor) -> torch.Tensor:
        """Takes ``tokens`` [B, n] and chooses the next ones (greedily), [B]."""
        n = tokens.shape[1]
        at = self.lens.long()[:, None] + torch.arange(n, device="cuda")
        self.history.scatter_(1, at, tokens.int())
        self.lens += n
        out = head.process_logits(self.logits(tokens), history=self.history.view(-1), cu_history=self.cu_history,
                                  repetition=self.repetition, frequency=self.frequency, allowed=self.allowed)
        self.token.copy_(out.argmax(dim=1))
        return self.token

    def capture(self) -> torch.cuda.CUDAGraph:
        """One decode step of every sequence as a graph; the state is as it was before."""
        kept = self.lens.clone(), self.token.clone(), self.history.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # first use of buffers and kernels outside the capture
            self.advance(self.token[:, None])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self.advance(self.token[:, None])
        for t, k in zip((self.lens, self.token, self.history), kept):
            t.copy_(k)
        return graph

    def check(self) -> None:
        """Raises what the kernels reported since the last check."""
        for pair in self.workspaces.values():
            for ws in pair:
                moe.synchronize(workspace=ws)


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--batch", type=int, default=1)
    ap.add_argument("--prompt", type=int, default=200)
    ap.add_argument("--steps", type=int, default=64)
    a = ap.parse_args()
    d = Decoder(MapleConfig(), a.layers, a.batch, a.prompt + a.steps + 1)
    g = torch.Generator("cuda").manual_seed(1)
    d.advance(torch.randint(0, d.cfg.vocab_size, (a.batch, a.prompt), generator=g, device="cuda"))
    graph = d.capture()
    said = []
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    t0.record()
    for _ in range(a.steps):
        said.append(d.token.clone())
        graph.replay()
    t1.record()
    d.check()
    ms = t0.elapsed_time(t1) / a.steps
    print("tokens of sequence 0:", [int(t[0]) for t in said][:16])
    print(f"{a.layers} layers, {a.batch} sequences, lengths to {int(d.lens.max())}: {ms * 1e3:.0f} us a step, {a.batch / ms * 1e3:.0f} tokens/s")


if __name__ == "__main__":
    main()
