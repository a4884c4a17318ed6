"""A tiny Monarch language model trained on synthetic text, every part on this library's kernels:

    python -m monarch_muon_amd.example [steps]

``embedding`` -> decoder blocks (``rms_norm`` with the residual's addition, ``rotary``, ``differential_attention`` and an MLP
between Monarch projections, ``butterfly_blk``) -> ``linear_cross_entropy`` -> backward -> ``MonarchMuonOptimizer`` (Monarch
factors by Muon, the rest by AdamW), and then a few tokens sampled greedily, one at a time over a cache, and scored.
"""
from __future__ import annotations

import sys

import torch
import torch.nn.functional as F

from . import (MonarchMuonOptimizer, butterfly_blk, differential_attention, embedding, linear_cross_entropy, rms_norm,
               rotary, rotary_table)
from .workloads import factor_shapes

VOCAB, WIDTH, HIDDEN, NBLOCKS, LAYERS = 509, 256, 512, 2, 2
PAD = 0
BATCH, SEQ = 8, 96
HEADS, DIM = 4, 32            # a head: two maps of DIM columns, values of twice as many


def factors(*sizes):
    return torch.nn.ParameterList(torch.randn(s) / s[2] ** 0.5 for din, dout in sizes for s in factor_shapes(din, dout, NBLOCKS))


class Attention(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.w = factors(*[(WIDTH, WIDTH)] * 4)
        self.lam = torch.nn.Parameter(torch.full((HEADS,), 0.3))
        self.norm = torch.nn.Parameter(torch.ones(2 * DIM))

    def forward(self, x, table, cache=None, at=0):
        B, T, _ = x.shape
        q, k, v = (butterfly_blk(x, self.w[i], self.w[i + 1]) for i in (0, 2, 4))
        q, k, v = q.view(B, T, 2 * HEADS, DIM), k.view(B, T, 2 * HEADS, DIM), v.view(B, T, HEADS, 2 * DIM)
        q, k = rotary(q, k, table, torch.arange(at, at + T, device=x.device))
        lengths = None
        if cache is not None:          # (keys, values) of the tokens before, with room for these
            cache[0][:, at:at + T], cache[1][:, at:at + T] = k, v
            (k, v), lengths = cache, torch.full((B,), at + T, device=x.device)
        o = rms_norm(differential_attention(q, k, v, self.lam, lengths=lengths), self.norm)
        return butterfly_blk(o.view(B, T, WIDTH), self.w[6], self.w[7])


class Block(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.norms = torch.nn.ParameterList(torch.ones(WIDTH) for _ in range(2))
        self.attention = Attention()
        self.w = factors((WIDTH, HIDDEN), (HIDDEN, WIDTH))

    def forward(self, x, stream, table, cache=None, at=0):
        """``x``: what the block before adds to the residual ``stream``, and so returned."""
        x, stream = (rms_norm(x, self.norms[0]), x) if stream is None else rms_norm(x, self.norms[0], residual=stream)
        x, stream = rms_norm(self.attention(x, table, cache, at), self.norms[1], residual=stream)
        return butterfly_blk(F.silu(butterfly_blk(x, self.w[0], self.w[1])), self.w[2], self.w[3]), stream


class TinyMonarchLM(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.wte = torch.nn.Parameter(torch.randn(VOCAB, WIDTH) * 0.02)
        self.blocks = torch.nn.ModuleList(Block() for _ in range(LAYERS))
        self.ln_f = torch.nn.Parameter(torch.ones(WIDTH))
        self.lm_head = torch.nn.Parameter(torch.randn(VOCAB, WIDTH) * 0.02)
        self.to(torch.bfloat16)
        self.register_buffer("table", rotary_table(DIM, SEQ), persistent=False)

    def hidden(self, ids, caches=None, at=0):
        """Of ``ids`` (..., T), which stand at ``at`` on; ``caches``: one of each block for the tokens before."""
        end = at + ids.shape[-1]
        if end > self.table.shape[0]:
            self.table = rotary_table(DIM, 2 * end, device=self.table.device)
        rows = ids.reshape(ids.shape[:-1].numel(), ids.shape[-1])
        x, stream = embedding(rows, self.wte, scale=WIDTH ** 0.5, padding_idx=PAD), None
        for i, b in enumerate(self.blocks):
            x, stream = b(x, stream, self.table, None if caches is None else caches[i], at)
        return rms_norm(x, self.ln_f, residual=stream)[0].view(*ids.shape, WIDTH)

    def caches(self, batch, length):
        new = lambda heads, width: torch.empty(batch, length, heads, width, dtype=torch.bfloat16, device=self.wte.device)  # noqa: E731
        return [(new(2 * HEADS, DIM), new(HEADS, 2 * DIM)) for _ in self.blocks]

    def loss(self, ids, targets, reduction="mean"):
        return linear_cross_entropy(self.hidden(ids), self.lm_head, targets, ignore_index=PAD, reduction=reduction)


def text(generator, device):
    """Sequences that a model can learn: each token is mostly a fixed function of the one before; ragged, padded."""
    ids = torch.randint(1, VOCAB, (BATCH, 1), generator=generator)
    for _ in range(SEQ):
        step = (ids[:, -1:] * 17 + 5) % (VOCAB - 1) + 1
        noise = torch.randint(1, VOCAB, (BATCH, 1), generator=generator)
        ids = torch.cat([ids, torch.where(torch.rand(BATCH, 1, generator=generator) < 0.1, noise, step)], 1)
    length = torch.randint(SEQ // 2, SEQ + 1, (BATCH, 1), generator=generator)
    ids = torch.where(torch.arange(SEQ + 1) <= length, ids, PAD)
    return ids[:, :-1].to(device), ids[:, 1:].to(device)


def train(steps: int = 60, seed: int = 0, device: str = "cuda", verbose: bool = False):
    """(model, losses of the steps)."""
    torch.manual_seed(seed)
    generator = torch.Generator().manual_seed(seed)
    model = TinyMonarchLM().to(device)
    muon = [p for p in model.parameters() if p.dim() == 3]
    rest = [p for p in model.parameters() if p.dim() != 3]
    opt = MonarchMuonOptimizer(muon, rest, lr=0.02, momentum=0.95)
    losses = []
    for step in range(steps):
        loss = model.loss(*text(generator, device))
        loss.backward()
        opt.clip_grad_norm_(1.0)
        opt.step()
        opt.zero_grad()
        losses.append(loss.detach())
        if verbose and step % 10 == 0:
            print(f"step {step:3d}  loss {float(losses[-1]):.3f}", flush=True)
    return model, torch.stack(losses).cpu()


@torch.no_grad()
def generate(model: TinyMonarchLM, token: int, count: int):
    """``count`` tokens after ``token``, the likeliest at each step, and the log-probability of each."""
    dev = model.wte.device
    ids, scores, caches = [token], [], model.caches(1, count)
    for at in range(count):
        h = model.hidden(torch.tensor([[ids[-1]]], device=dev), caches, at)[0]
        best = (h.float() @ model.lm_head.float().T).argmax(-1)
        scores.append(-float(linear_cross_entropy(h, model.lm_head, best, reduction="sum")))
        ids.append(int(best))
    return ids[1:], scores


if __name__ == "__main__":
    lm, history = train(int(sys.argv[1]) if len(sys.argv) > 1 else 60, verbose=True)
    print(f"loss {float(history[0]):.3f} -> {float(history[-5:].mean()):.3f}")
    tokens, logp = generate(lm, 7, 5)
    print("after 7:", tokens, "log-probabilities", [round(s, 2) for s in logp])
