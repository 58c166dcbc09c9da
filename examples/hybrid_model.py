"""A small hybrid language model on this package's operators: layers of the
gated delta rule, of the elementwise gated recurrence and of windowed attention,
with the residual stream in fp32 between them.

    python examples/hybrid_model.py [--steps 30]

trains it on synthetic text (a noisy cycle of symbols) and then answers token by
token, the states and caches going from step to step.

Training runs gated_scan, window_attn, add_rms_norm and chunk_gated_delta_rule
through autograd; answering runs gated_scan and chunk_gated_delta_rule on one row
with their states, window_attn_decode over a cache, and, with fp8=True,
add_rms_norm_fp8 before the projections.
"""

import argparse
import importlib
import os
import sys

import torch
import torch.nn.functional as F
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
gdn = importlib.import_module("v100-attention-lab_amd")

DTYPE = torch.bfloat16


class DeltaRule(nn.Module):
    """Gated delta rule: a K x V state per head."""

    def __init__(self, width, heads, dim):
        super().__init__()
        self.heads, self.dim = heads, dim
        self.inp = nn.Linear(width, heads * (3 * dim + 2), bias=False, dtype=DTYPE)
        self.out = nn.Linear(heads * dim, width, bias=False, dtype=DTYPE)

    def start(self, batch, length, device):
        return torch.zeros(batch, self.heads, self.dim, self.dim, device=device)

    def forward(self, y, state=None, length=None):
        B, T, _ = y.shape
        n, d = self.heads, self.dim
        q, k, v, b, g = self.inp(y).split([n * d, n * d, n * d, n, n], -1)
        q, k = (F.normalize(x.view(B, T, n, d), dim=-1) for x in (q, k))
        o, state = gdn.chunk_gated_delta_rule(
            q=q, k=k, v=v.reshape(B, T, n, d), g=F.logsigmoid(g.float() + 4), beta=torch.sigmoid(b.float()),
            initial_state=state, output_final_state=True)
        return self.out(o.reshape(B, T, n * d)), state


class Recurrence(nn.Module):
    """Elementwise gated recurrence: one state value per channel."""

    def __init__(self, width):
        super().__init__()
        self.inp = nn.Linear(width, 3 * width, bias=False, dtype=DTYPE)
        self.out = nn.Linear(width, width, bias=False, dtype=DTYPE)

    def start(self, batch, length, device):
        return torch.zeros(batch, self.out.in_features, device=device)

    def forward(self, y, state=None, length=None):
        x, g, z = self.inp(y).chunk(3, -1)
        h, state = gdn.gated_scan(x, F.logsigmoid(g.float() + 3), state)
        return self.out(h * F.silu(z)), state


class WindowAttention(nn.Module):
    """Attention with a sliding window, sinks and shared key heads; the state of
    a running sequence is its cache and length."""

    def __init__(self, width, heads, key_heads, dim, window, sinks):
        super().__init__()
        self.heads, self.key_heads, self.dim, self.window, self.sinks = heads, key_heads, dim, window, sinks
        self.inp = nn.Linear(width, (heads + 2 * key_heads) * dim, bias=False, dtype=DTYPE)
        self.out = nn.Linear(heads * dim, width, bias=False, dtype=DTYPE)

    def start(self, batch, length, device):
        cache = torch.zeros(2, batch, length, self.key_heads, self.dim, dtype=DTYPE, device=device)
        return cache[0], cache[1], torch.zeros(batch, dtype=torch.int32, device=device)

    def forward(self, y, state=None, length=None):
        B, T, _ = y.shape
        qkv = self.inp(y).view(B, T, -1, self.dim)
        q, k, v = qkv.split([self.heads, self.key_heads, self.key_heads], 2)
        if state is None:
            o = gdn.window_attn(q, k, v, self.window, self.sinks)
        else:
            kc, vc, n = state
            rows = n[:, None].long() + torch.arange(T, device=y.device)
            seq = torch.arange(B, device=y.device)[:, None]
            kc[seq, rows], vc[seq, rows] = k, v
            n += T
            o = gdn.window_attn_decode(q, kc, vc, n, self.window, self.sinks)
        return self.out(o.reshape(B, T, -1)), state


class HybridModel(nn.Module):
    def __init__(self, vocab=64, width=256, layers=2, window=48, sinks=4):
        super().__init__()
        self.embed = nn.Embedding(vocab, width)
        self.mixers = nn.ModuleList()
        for _ in range(layers):
            self.mixers += [DeltaRule(width, 4, 64), Recurrence(width), WindowAttention(width, 4, 2, 64, window, sinks)]
        self.norms = nn.ParameterList(nn.Parameter(torch.ones(width)) for _ in range(len(self.mixers) + 1))
        self.head = nn.Linear(width, vocab, bias=False, dtype=DTYPE)

    def start(self, batch, length, device):
        """States and caches of `batch` sequences of up to `length` tokens."""
        return [m.start(batch, length, device) for m in self.mixers]

    def _norm(self, x, i, r, fp8):
        if not fp8:
            return gdn.add_rms_norm(x, self.norms[i], r)
        y, scale, r = gdn.add_rms_norm_fp8(x, self.norms[i].detach(), r)
        return (y.float() * scale).to(DTYPE), r      # (an 8-bit product would take y and scale)

    def forward(self, tokens, states=None, fp8=False):
        """Logits of [B, T] tokens; with states (see start) they are continued in place."""
        r = self.embed(tokens)
        x = torch.zeros_like(r, dtype=DTYPE)
        for i, mixer in enumerate(self.mixers):
            y, r = self._norm(x, i, r, fp8)
            x, state = mixer(y, None if states is None else states[i])
            if states is not None:
                states[i] = state
        y, _ = self._norm(x, len(self.mixers), r, fp8)
        return self.head(y).float()


def text(batch, length, vocab, seed, device):
    """A cycle of symbols with a step of its own for each row, a tenth of them noise."""
    gen = torch.Generator().manual_seed(seed)
    step = torch.randint(1, 6, (batch, 1), generator=gen)
    t = (torch.randint(0, vocab, (batch, 1), generator=gen) + step * torch.arange(length)) % vocab
    noise = torch.rand(batch, length, generator=gen) < 0.1
    return torch.where(noise, torch.randint(0, vocab, (batch, length), generator=gen), t).to(device)


def train(model, steps, batch=8, length=256, device="cuda", log=None):
    """`steps` steps of AdamW; returns the losses."""
    opt = torch.optim.AdamW(model.parameters(), lr=3e-3)
    losses = []
    for i in range(steps):
        t = text(batch, length + 1, model.embed.num_embeddings, i, device)
        loss = F.cross_entropy(model(t[:, :-1]).flatten(0, 1), t[:, 1:].flatten())
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if log and (i + 1) % 10 == 0:
            log(f"step {i + 1}: loss {losses[-1].item():.3f}")
    return [x.item() for x in losses]


@torch.no_grad()
def answer(model, tokens, new, fp8=False):
    """Reads [B, T] tokens one at a time, then appends `new` of the model's own
    choice; returns them all, and the logits of every step."""
    B, T = tokens.shape
    states = model.start(B, T + new, tokens.device)
    out, logits = [tokens], []
    for t in range(T + new - 1):
        logits.append(model(torch.cat(out, 1)[:, t:t + 1], states, fp8))
        if t >= T - 1:
            out.append(logits[-1][:, -1:].argmax(-1))
    return torch.cat(out, 1), torch.cat(logits, 1)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=30)
    a = ap.parse_args()
    torch.manual_seed(0)
    model = HybridModel().cuda()
    train(model, a.steps, log=print)
    tokens, _ = answer(model, text(2, 40, 64, 999, "cuda"), 12)
    for row in tokens.tolist():
        print(" ".join(map(str, row[:40])), "->", " ".join(map(str, row[40:])))


if __name__ == "__main__":
    main()
