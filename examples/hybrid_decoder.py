"""A small hybrid decoder on the package's operators: a gated-delta-rule layer and a sliding-window attention layer, each with
its feed-forward block, trained for some steps on a counting task, then served token by token. Run it on a B200 (the package
built first):

    python examples/hybrid_decoder.py

What it shows, in the order of a layer:
    add_rms_norm          the residual stream and its norm, at the head of both layers
    conv_qkv, gates, chunk_gated_delta_rule, gated_rms_norm        the linear-attention mixer
    rotary, window_attention                                       the softmax mixer, trained and prefilled
    window_attention_step                                          its single tokens, over a rolling cache
    gated_delta_step                                               the rule's single tokens, over a pool of states
    gated_feed_forward                                             the layer's other half, trained and for single tokens
    linear_cross_entropy                                           the loss, without the logits
    add_rms_norm_fp8                                               the last norm with an 8-bit output and scales
"""
from __future__ import annotations

import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mac-ai-engineering_b200"))
from macai_b200.conv import conv_qkv  # noqa: E402
from macai_b200.feed_forward import gated_feed_forward  # noqa: E402
from macai_b200.gated_delta import chunk_gated_delta_rule, gated_delta_step  # noqa: E402
from macai_b200.gated_norm import gated_rms_norm  # noqa: E402
from macai_b200.gates import gates  # noqa: E402
from macai_b200.loss import linear_cross_entropy  # noqa: E402
from macai_b200.norm import add_rms_norm, add_rms_norm_fp8  # noqa: E402
from macai_b200.rotary import rotary, rotary_table  # noqa: E402
from macai_b200.window_attention import window_attention, window_attention_step  # noqa: E402

DIM, HEADS, KEY_HEADS, WIDTH = 256, 4, 2, 64      # the attention layer's
RULE_HEADS, RULE_WIDTH = 2, 128                   # the rule's
WINDOW, SINKS, VOCAB, INNER = 64, 4, 64, 512


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

    def rows(self, qkv, x):
        """The rule's inputs of the tokens that qkv (and x) has, qkv's first tokens standing before them."""
        n = qkv.shape[1] - x.shape[1]
        q, k, v = (t[:, n:] for t in conv_qkv(qkv, self.conv, RULE_HEADS * RULE_WIDTH, RULE_WIDTH, 1, RULE_WIDTH))
        b, a = self.ba(x).chunk(2, -1)
        beta, g = gates(b, a, self.A_log, self.dt_bias)
        return q, k, v, g, beta

    def close(self, o, x):
        o = gated_rms_norm(o, self.z(x).unflatten(-1, (RULE_HEADS, RULE_WIDTH)), self.norm, 1e-6)
        return self.out(o.flatten(2))

    def forward(self, x):
        o, _ = chunk_gated_delta_rule(*self.rows(self.qkv(x), x), use_qk_l2norm_in_kernel=True)
        return self.close(o, x)

    def prefill(self, x):
        """The output and what single tokens go on from: the convolution's last three inputs (zeros where the prompt has fewer,
        as the convolution has before a row's first token) and the states."""
        qkv = self.qkv(x)
        o, state = chunk_gated_delta_rule(*self.rows(qkv, x), output_final_state=True, use_qk_l2norm_in_kernel=True)
        before = qkv.new_zeros(qkv.shape[0], 3, qkv.shape[2])
        n = min(3, qkv.shape[1])
        before[:, 3 - n:] = qkv[:, qkv.shape[1] - n:]
        return self.close(o, x), before, state

    def step(self, x, before, state):
        """One token a request: x [B, 1, DIM]; carries on `before` and the states in place."""
        qkv = torch.cat([before, self.qkv(x)], 1)
        before.copy_(qkv[:, 1:])
        return self.close(gated_delta_step(*self.rows(qkv, x), state, use_qk_l2norm_in_kernel=True), x)


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


class FeedForward(nn.Module):
    def __init__(self):
        super().__init__()
        self.gate, self.up, self.down = linear(DIM, INNER), linear(DIM, INNER), linear(INNER, DIM)

    def forward(self, x):
        return gated_feed_forward(x, self.gate.weight, self.up.weight, self.down.weight)


class Decoder(nn.Module):
    def __init__(self):
        super().__init__()
        self.embed, self.head = nn.Embedding(VOCAB, DIM), linear(DIM, VOCAB)
        self.delta, self.window = DeltaMixer(), WindowMixer()
        self.ff = nn.ModuleList([FeedForward(), FeedForward()])
        self.norms = nn.ParameterList([nn.Parameter(torch.zeros(DIM)) for _ in range(5)])   # zero-centred: 1 + w

    def layers(self, tokens, delta, window):
        """The last norm's output, the mixers given as functions."""
        y, s = add_rms_norm(self.embed(tokens), None, self.norms[0], zero_centered=True)
        for i, f in enumerate((delta, self.ff[0], window, self.ff[1])):
            y, s = add_rms_norm(f(y), s, self.norms[i + 1], zero_centered=True)
        return y

    def hidden(self, tokens, table):
        return self.layers(tokens, self.delta, lambda y: self.window(y, table)[0])

    def forward(self, tokens, table):
        """Logits [B, T, VOCAB]."""
        return self.head(self.hidden(tokens, table))

    def loss(self, tokens, table):
        """The mean loss of every next token; a row's last token has none."""
        labels = torch.cat([tokens[:, 1:], torch.full_like(tokens[:, :1], -100)], 1)
        return linear_cross_entropy(self.hidden(tokens, table), self.head.weight, labels)


def train(steps=30, B=4, T=256, device="cuda", seed=0):
    """The model, its table, and the first and last loss of a counting task: every row counts up from a random token."""
    torch.manual_seed(seed)
    model = Decoder().to(device, torch.bfloat16)
    table = rotary_table(4096, WIDTH // 4, device=device)
    opt = torch.optim.AdamW(model.parameters(), lr=2e-3)
    losses = []
    for _ in range(steps):
        tokens = (torch.randint(0, VOCAB, (B, 1), device=device) + torch.arange(T, device=device)) % VOCAB
        loss = model.loss(tokens, table)
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return model, table, float(losses[0]), float(losses[-1])


def rolling_cache(keys, values, prompt):
    """A prompt's keys and values in a cache whose slots are the window's and the first tokens'."""
    B, dev, S = keys.shape[0], keys.device, SINKS + WINDOW
    cache = tuple(torch.zeros(B, S, KEY_HEADS, WIDTH, dtype=keys.dtype, device=dev) for _ in range(2))
    at = torch.arange(max(0, prompt - WINDOW), prompt, device=dev)
    at = torch.cat([torch.arange(min(SINKS, int(at[0])), device=dev), at])
    slot = torch.where(at < S, at, SINKS + (at - SINKS) % (S - SINKS))
    for c, t in zip(cache, (keys, values)):
        c[:, slot] = t[:, at]
    return cache


@torch.no_grad()
def serve(model, table, B=3, prompt=100, more=80, seed=1):
    """The window layer fed a prompt at once, then single tokens through a rolling cache; returns the largest difference
    from the layer run over the whole row."""
    layer, dev = model.window, table.device
    x = torch.randn(B, prompt + more, DIM, generator=torch.Generator().manual_seed(seed)).to(dev, torch.bfloat16)
    whole, _, _ = layer(x, table)
    _, k, v = layer(x[:, :prompt], table)
    cache = rolling_cache(k, v, prompt)
    lengths = torch.full((B,), prompt, dtype=torch.int32, device=dev)
    worst = 0.0
    for t in range(prompt, prompt + more):
        y = layer.step(x[:, t:t + 1], table, cache, lengths)
        lengths += 1
        worst = max(worst, float((y.float() - whole[:, t:t + 1].float()).abs().max()))
    q, scale, _ = add_rms_norm_fp8(whole, x, model.norms[2], zero_centered=True)   # what an 8-bit head would read
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (B, prompt + more, DIM // 128)
    return worst


@torch.no_grad()
def generate(model, table, tokens, more):
    """tokens [B, prompt] continued greedily by `more` tokens, one at a time through both layers; also the logits each of
    them was taken from."""
    B, prompt = tokens.shape
    kept = {}

    def delta(y):
        o, kept["before"], kept["state"] = model.delta.prefill(y)
        return o

    def window(y):
        o, k, v = model.window(y, table)
        kept["cache"] = rolling_cache(k, v, prompt)
        return o
    logits = [model.head(model.layers(tokens, delta, window)[:, -1:])]
    lengths = torch.full((B,), prompt, dtype=torch.int32, device=tokens.device)
    for _ in range(more):
        tokens = torch.cat([tokens, logits[-1].argmax(-1)], 1)
        y = model.layers(tokens[:, -1:], lambda y: model.delta.step(y, kept["before"], kept["state"]),
                         lambda y: model.window.step(y, table, kept["cache"], lengths))
        lengths += 1
        logits.append(model.head(y))
    return tokens, torch.cat(logits[:-1], 1)


if __name__ == "__main__":
    model, table, first, last = train()
    print(f"training: loss {first:.3f} -> {last:.3f}")
    print(f"serving: largest difference between single tokens and the whole row {serve(model, table):.4f}")
    tokens, _ = generate(model, table, torch.arange(5, 25, device=table.device)[None], 20)
    print(f"counting on from {int(tokens[0, 19])}: {tokens[0, 20:].tolist()}")
