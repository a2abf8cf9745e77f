"""A small hybrid decoder on the package's operators: a gated-delta-rule layer and a sliding-window attention layer, trained
for some steps on a counting task, then served token by token. Run it on a B200 (the package built first):

    python examples/hybrid_decoder.py

What it shows, in the order of a layer:
    add_rms_norm          the residual stream and its norm, at the head of both layers
    conv_qkv, gates, chunk_gated_delta_rule, gated_rms_norm        the linear-attention mixer
    rotary, window_attention                                       the softmax mixer, trained and prefilled
    window_attention_step                                          its single tokens, over a rolling cache
    add_rms_norm_fp8                                               the last norm with an 8-bit output and scales
"""
from __future__ import annotations

import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mac-ai-engineering_b200"))
from macai_b200.conv import conv_qkv  # noqa: E402
from macai_b200.gated_delta import chunk_gated_delta_rule  # noqa: E402
from macai_b200.gated_norm import gated_rms_norm  # noqa: E402
from macai_b200.gates import gates  # noqa: E402
from macai_b200.norm import add_rms_norm, add_rms_norm_fp8  # noqa: E402
from macai_b200.rotary import rotary, rotary_table  # noqa: E402
from macai_b200.window_attention import window_attention, window_attention_step  # noqa: E402

DIM, HEADS, KEY_HEADS, WIDTH = 256, 4, 2, 64      # the attention layer's
RULE_HEADS, RULE_WIDTH = 2, 128                   # the rule's
WINDOW, SINKS, VOCAB = 64, 4, 64


def linear(i, o):
    m = nn.Linear(i, o, bias=False)
    nn.init.normal_(m.weight, std=i ** -0.5)
    return m


class DeltaMixer(nn.Module):
    """The linear-attention mixer: projections around the convolution, the gates, the rule and the gated norm."""

    def __init__(self):
        super().__init__()
        inner = RULE_HEADS * RULE_WIDTH
        self.qkv, self.z, self.ba, self.out = linear(DIM, 3 * inner), linear(DIM, inner), linear(DIM, 2 * RULE_HEADS), linear(inner, DIM)
        self.conv = nn.Parameter(torch.randn(3 * inner, 1, 4) * 0.3)
        self.A_log, self.dt_bias = nn.Parameter(torch.rand(RULE_HEADS)), nn.Parameter(torch.zeros(RULE_HEADS))
        self.norm = nn.Parameter(torch.ones(RULE_WIDTH))

    def forward(self, x):
        B, T, _ = x.shape
        q, k, v = conv_qkv(self.qkv(x), self.conv, RULE_HEADS * RULE_WIDTH, RULE_WIDTH, 1, RULE_WIDTH)
        b, a = self.ba(x).chunk(2, -1)
        beta, g = gates(b, a, self.A_log, self.dt_bias)
        o, _ = chunk_gated_delta_rule(q, k, v, g, beta, use_qk_l2norm_in_kernel=True)
        o = gated_rms_norm(o, self.z(x).view(B, T, RULE_HEADS, RULE_WIDTH), self.norm, 1e-6)
        return self.out(o.flatten(2))


class WindowMixer(nn.Module):
    """The softmax mixer: one fused projection, read in place as q, k, v; rotary on a quarter of the head."""

    def __init__(self):
        super().__init__()
        self.qkv, self.out = linear(DIM, (HEADS + 2 * KEY_HEADS) * WIDTH), linear(HEADS * WIDTH, DIM)

    def split(self, x):
        qkv = self.qkv(x).unflatten(-1, (HEADS + 2 * KEY_HEADS, WIDTH))
        return qkv[:, :, :HEADS], qkv[:, :, HEADS:HEADS + KEY_HEADS], qkv[:, :, HEADS + KEY_HEADS:]

    def forward(self, x, table):
        q, k, v = self.split(x)
        q, k = rotary(q, k, table)
        return self.out(window_attention(q, k, v, window=WINDOW, sinks=SINKS).flatten(2)), k, v

    def step(self, x, table, cache, lengths):
        """One token a request: x [B, 1, DIM]; stores its key and value in the cache."""
        q, k, v = self.split(x)
        q, k = rotary(q, k, table, lengths[:, None])
        return self.out(window_attention_step(q, k, v, *cache, lengths, window=WINDOW, sinks=SINKS).flatten(2))


class Decoder(nn.Module):
    def __init__(self):
        super().__init__()
        self.embed, self.head = nn.Embedding(VOCAB, DIM), linear(DIM, VOCAB)
        self.delta, self.window = DeltaMixer(), WindowMixer()
        self.norms = nn.ParameterList([nn.Parameter(torch.zeros(DIM)) for _ in range(3)])   # zero-centred: 1 + w

    def forward(self, tokens, table):
        """Logits [B, T, VOCAB]."""
        x = self.embed(tokens)
        y, s = add_rms_norm(x, None, self.norms[0], zero_centered=True)
        y, s = add_rms_norm(self.delta(y), s, self.norms[1], zero_centered=True)
        y, s = add_rms_norm(self.window(y, table)[0], s, self.norms[2], zero_centered=True)
        return self.head(y)


def train(steps=30, B=4, T=256, device="cuda", seed=0):
    """The model, its table, and the first and last loss of a counting task: every row counts up from a random token."""
    torch.manual_seed(seed)
    model = Decoder().to(device, torch.bfloat16)
    table = rotary_table(4096, WIDTH // 4, device=device)
    opt = torch.optim.AdamW(model.parameters(), lr=2e-3)
    losses = []
    for _ in range(steps):
        tokens = (torch.randint(0, VOCAB, (B, 1), device=device) + torch.arange(T, device=device)) % VOCAB
        logits = model(tokens, table)
        loss = nn.functional.cross_entropy(logits[:, :-1].float().flatten(0, 1), tokens[:, 1:].flatten())
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return model, table, float(losses[0]), float(losses[-1])


@torch.no_grad()
def serve(model, table, B=3, prompt=100, more=80, seed=1):
    """The window layer fed a prompt at once, then single tokens through a rolling cache; returns the largest difference
    from the layer run over the whole row."""
    layer, dev = model.window, table.device
    x = torch.randn(B, prompt + more, DIM, generator=torch.Generator().manual_seed(seed)).to(dev, torch.bfloat16)
    whole, _, _ = layer(x, table)
    _, k, v = layer(x[:, :prompt], table)
    S = SINKS + WINDOW                                  # the cache rolls: its slots are the window's and the first tokens'
    cache = tuple(torch.zeros(B, S, KEY_HEADS, WIDTH, dtype=torch.bfloat16, device=dev) for _ in range(2))
    at = torch.arange(max(0, prompt - WINDOW), prompt, device=dev)
    at = torch.cat([torch.arange(min(SINKS, int(at[0])), device=dev), at])
    slot = torch.where(at < S, at, SINKS + (at - SINKS) % (S - SINKS))
    for c, t in zip(cache, (k, v)):
        c[:, slot] = t[:, at]
    lengths = torch.full((B,), prompt, dtype=torch.int32, device=dev)
    worst = 0.0
    for t in range(prompt, prompt + more):
        y = layer.step(x[:, t:t + 1], table, cache, lengths)
        lengths += 1
        worst = max(worst, float((y.float() - whole[:, t:t + 1].float()).abs().max()))
    q, scale, _ = add_rms_norm_fp8(whole, x, model.norms[2], zero_centered=True)   # what an 8-bit head would read
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (B, prompt + more, DIM // 128)
    return worst


if __name__ == "__main__":
    model, table, first, last = train()
    print(f"training: loss {first:.3f} -> {last:.3f}")
    print(f"serving: largest difference between single tokens and the whole row {serve(model, table):.4f}")
