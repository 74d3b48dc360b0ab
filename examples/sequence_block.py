"""A small sequence model on the ferrum_gpu.sequence operators.

    python examples/sequence_block.py [--steps N]

Three layers, each  norm_before -> mixer -> norm_after onto the residual stream:
the first mixes along the sequence with causal_conv1d and selective_scan, the
second with long_conv (through the FFT), the third with gated_recurrence, and
drops some of what it adds (dropout). The loss is linear_cross_entropy against the
vocabulary. Trains on a synthetic task (repeat the token seen LAG steps ago) and
then answers token by token on kept state, checking that both forms agree. Needs
a B200.
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "ferrum-gpu_b200"))

from ferrum_gpu import sequence as sq  # noqa: E402

VOCAB, WIDTH, STATES, TAPS, LAG, DROP = 16, 64, 16, 4, 5, 0.05


# Each operator with its gradient, as torch.autograd sees it.

class Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        ctx.save_for_backward(x, weight, bias)
        return sq.causal_conv1d(x, weight, bias, activation="silu")

    @staticmethod
    def backward(ctx, dy):
        g = sq.causal_conv1d_backward(dy.contiguous(), *ctx.saved_tensors, activation="silu")
        return g.dx, g.dweight, g.dbias


class Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, delta_bias):
        r = sq.selective_scan(u, delta, A, B, C, D=D, z=z, delta_bias=delta_bias,
                              delta_softplus=True, save_states=True)
        ctx.save_for_backward(u, delta, A, B, C, r.states, D, z, delta_bias)
        return r.out

    @staticmethod
    def backward(ctx, dout):
        u, delta, A, B, C, states, D, z, bias = ctx.saved_tensors
        g = sq.selective_scan_backward(dout.contiguous(), u, delta, A, B, C, states, D=D, z=z,
                                       delta_bias=bias, delta_softplus=True)
        return g.du, g.ddelta, g.dA, g.dB, g.dC, g.dD, g.dz, g.ddelta_bias


class LongConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kernel, skip):
        ctx.save_for_backward(x, kernel, skip)
        return sq.long_conv(x, kernel, skip)

    @staticmethod
    def backward(ctx, dy):
        g = sq.long_conv_backward(dy, *ctx.saved_tensors)
        return g.dx, g.dkernel, g.dskip


class Recurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, input_gate, recurrence_gate, decay):
        r = sq.gated_recurrence(x, input_gate, recurrence_gate, decay, save_states=True)
        ctx.save_for_backward(x, input_gate, recurrence_gate, decay, r.states)
        return r.out

    @staticmethod
    def backward(ctx, dout):
        g = sq.gated_recurrence_backward(dout.contiguous(), *ctx.saved_tensors)
        return g.dx, g.dinput_gate, g.drecurrence_gate, g.ddecay


class Dropout(torch.autograd.Function):
    """residual + dropout(x), the mask drawn again for the gradient."""

    @staticmethod
    def forward(ctx, x, residual, p, seed, offset=0):
        ctx.p, ctx.seed, ctx.offset, ctx.dtype = p, seed, offset, x.dtype
        return sq.dropout(x, p, seed, offset=offset, residual=residual)

    @staticmethod
    def backward(ctx, dy):
        dy = dy.contiguous()
        dx = sq.dropout_backward(dy, ctx.p, ctx.seed, offset=ctx.offset, dtype=ctx.dtype)
        return dx, dy, None, None, None


class Loss(torch.autograd.Function):
    """Each token's loss against the vocabulary; targets outside it have none."""

    @staticmethod
    def forward(ctx, x, weight, targets):
        r = sq.linear_cross_entropy(x, weight, targets)
        ctx.save_for_backward(x, weight, targets, r.lse)
        return r.loss

    @staticmethod
    def backward(ctx, dloss):
        g = sq.linear_cross_entropy_backward(dloss.contiguous(), *ctx.saved_tensors)
        return g.dx, g.dweight, None


class NormBefore(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight):
        y, r = sq.norm_before(x, weight)
        ctx.save_for_backward(r, weight)
        return y

    @staticmethod
    def backward(ctx, dy):
        r, weight = ctx.saved_tensors
        g = sq.norm_before_backward(dy.contiguous(), r, weight)
        return g.dx, g.dweight


class NormAfter(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, gate, residual, scale):
        ctx.save_for_backward(x, weight, gate, scale)
        return sq.norm_after(x, weight, gate=gate, residual=residual, scale=scale)

    @staticmethod
    def backward(ctx, dout):
        x, weight, gate, scale = ctx.saved_tensors
        dout = dout.contiguous()
        g = sq.norm_after_backward(dout, x, weight, gate=gate, scale=scale)
        return g.dx, g.dweight, g.dgate, dout, g.dscale


class ScanLayer(nn.Module):
    def __init__(self):
        super().__init__()
        self.norm_in, self.norm_out = nn.Parameter(torch.ones(WIDTH)), nn.Parameter(torch.ones(WIDTH))
        self.scale = nn.Parameter(torch.full((WIDTH,), 0.5))
        self.proj_in = nn.Linear(WIDTH, 3 * WIDTH, bias=False)     # u, z, gate
        self.weight = nn.Parameter(torch.randn(WIDTH, TAPS) / TAPS)
        self.bias = nn.Parameter(torch.zeros(WIDTH))
        self.proj_x = nn.Linear(WIDTH, WIDTH + 2 * STATES, bias=False)   # delta, B, C
        self.log_a = nn.Parameter(torch.log(torch.arange(1, STATES + 1.0)).repeat(WIDTH, 1))
        self.skip = nn.Parameter(torch.ones(WIDTH))
        step = torch.exp(torch.linspace(math.log(1e-2), math.log(0.5), WIDTH))
        self.delta_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))

    def forward(self, h):
        u, z, gate = self.proj_in(NormBefore.apply(h, self.norm_in)).split(WIDTH, -1)
        u = Conv.apply(u, self.weight, self.bias)
        delta, B, C = self.proj_x(u).split([WIDTH, STATES, STATES], -1)
        y = Scan.apply(u, delta, -torch.exp(self.log_a), B, C, self.skip, z, self.delta_bias)
        return NormAfter.apply(y, self.norm_out, gate, h, self.scale)

    def start(self, batch):
        dev = self.weight.device
        return {"conv": torch.zeros(batch, TAPS - 1, WIDTH, device=dev),
                "scan": torch.zeros(batch, WIDTH, STATES, device=dev)}

    def step(self, h, s):
        y, _ = sq.norm_before(h, self.norm_in)
        u, z, gate = self.proj_in(y).split(WIDTH, -1)
        u = sq.causal_conv1d_step(u, s["conv"], self.weight, self.bias, activation="silu")
        delta, B, C = self.proj_x(u).split([WIDTH, STATES, STATES], -1)
        y = sq.selective_scan_step(u, delta, -torch.exp(self.log_a), B, C, s["scan"], D=self.skip,
                                   z=z, delta_bias=self.delta_bias, delta_softplus=True)
        return sq.norm_after(y, self.norm_out, gate=gate, residual=h, scale=self.scale)


class LongLayer(nn.Module):
    def __init__(self, length):
        super().__init__()
        self.length = length
        self.norm_in, self.norm_out = nn.Parameter(torch.ones(WIDTH)), nn.Parameter(torch.ones(WIDTH))
        self.scale = nn.Parameter(torch.full((WIDTH,), 0.5))
        self.proj_in = nn.Linear(WIDTH, 2 * WIDTH, bias=False)
        fade = torch.exp(-torch.arange(length) * (8.0 / length))
        self.kernel = nn.Parameter(torch.randn(WIDTH, length) * fade / math.sqrt(length))
        self.skip = nn.Parameter(torch.ones(WIDTH))

    def forward(self, h):
        x, gate = self.proj_in(NormBefore.apply(h, self.norm_in)).split(WIDTH, -1)
        y = LongConv.apply(x.transpose(1, 2), self.kernel, self.skip)
        return NormAfter.apply(y.transpose(1, 2).contiguous(), self.norm_out, gate, h, self.scale)

    def start(self, batch):
        dev = self.kernel.device
        return {"history": torch.zeros(batch, WIDTH, self.length, device=dev),
                "position": torch.zeros(batch, dtype=torch.int32, device=dev)}

    def step(self, h, s):
        y, _ = sq.norm_before(h, self.norm_in)
        x, gate = self.proj_in(y).split(WIDTH, -1)
        y = sq.long_conv_step(x, s["history"], s["position"], self.kernel, self.skip)
        s["position"] += 1
        return sq.norm_after(y, self.norm_out, gate=gate, residual=h, scale=self.scale)


class RecurrenceLayer(nn.Module):
    def __init__(self, index=0):
        super().__init__()
        self.index = index        # layers count seeds alike: each draws masks of its own by it
        self.norm_in, self.norm_out = nn.Parameter(torch.ones(WIDTH)), nn.Parameter(torch.ones(WIDTH))
        self.scale = nn.Parameter(torch.full((WIDTH,), 0.5))
        self.proj_in = nn.Linear(WIDTH, 4 * WIDTH, bias=False)     # x, both gates, gate
        # at half open gates, memories of 2 to 200 steps
        self.log_decay = nn.Parameter(torch.linspace(math.log(1e-2), 0.0, WIDTH))
        # read when the mask is drawn: a captured step draws another mask once it changes
        self.register_buffer("seed", torch.zeros(1, dtype=torch.int64))

    def forward(self, h):
        x, i, r, gate = self.proj_in(NormBefore.apply(h, self.norm_in)).split(WIDTH, -1)
        y = Recurrence.apply(x, i, r, torch.exp(self.log_decay))
        if not self.training:
            return NormAfter.apply(y, self.norm_out, gate, h, self.scale)
        self.seed += 1
        y = NormAfter.apply(y, self.norm_out, gate, torch.zeros_like(h), self.scale)
        return Dropout.apply(y, h, DROP, self.seed.clone(), self.index)

    def start(self, batch):
        return {"state": torch.zeros(batch, WIDTH, device=self.scale.device)}

    def step(self, h, s):
        y, _ = sq.norm_before(h, self.norm_in)
        x, i, r, gate = self.proj_in(y).split(WIDTH, -1)
        y = sq.gated_recurrence_step(x, i, r, torch.exp(self.log_decay), s["state"])
        return sq.norm_after(y, self.norm_out, gate=gate, residual=h, scale=self.scale)


class Model(nn.Module):
    def __init__(self, length):
        super().__init__()
        self.embed = nn.Embedding(VOCAB, WIDTH)
        self.layers = nn.ModuleList([ScanLayer(), LongLayer(length), RecurrenceLayer(2)])
        self.head = nn.Linear(WIDTH, VOCAB, bias=False)

    def hidden(self, tokens):
        h = self.embed(tokens)
        for layer in self.layers:
            h = layer(h)
        return h

    def forward(self, tokens):
        return self.head(self.hidden(tokens))

    def loss(self, tokens, targets):
        """The mean over the tokens whose target lies in the vocabulary; no logits."""
        losses = Loss.apply(self.hidden(tokens), self.head.weight, targets)
        return losses.sum() / ((targets >= 0) & (targets < VOCAB)).sum()

    @torch.no_grad()
    def decode(self, tokens):
        """The same logits, one token at a time."""
        states = [layer.start(tokens.shape[0]) for layer in self.layers]
        out = []
        for t in range(tokens.shape[1]):
            h = self.embed(tokens[:, t])
            for layer, s in zip(self.layers, states):
                h = layer.step(h, s)
            out.append(self.head(h))
        return torch.stack(out, 1)


def main(steps: int = 200, batch: int = 16, length: int = 96):
    torch.manual_seed(0)
    model = Model(length).cuda()
    opt = torch.optim.AdamW(model.parameters(), lr=3e-3)
    losses = []
    for _ in range(steps):
        tokens = torch.randint(VOCAB, (batch, length), device="cuda")
        targets = torch.full_like(tokens, -100)
        targets[:, LAG:] = tokens[:, :-LAG]
        loss = model.loss(tokens, targets)
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    losses = torch.stack(losses).tolist()
    model.eval()
    with torch.no_grad():
        prompt, stepped = model(tokens), model.decode(tokens)
    gap = ((prompt - stepped).abs().max() / prompt.abs().max()).item()
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} in {steps} steps "
          f"(guessing: {math.log(VOCAB):.3f}); token by token differs by {gap:.1e}")
    return losses, gap


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=200)
    main(ap.parse_args().steps)
