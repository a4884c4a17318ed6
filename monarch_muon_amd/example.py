"""A tiny Monarch language model trained on synthetic text, every part on this library's kernels:

    python -m monarch_muon_amd.example [steps]

``embedding`` -> residual MLP blocks of Monarch projections (``butterfly_blk``) -> ``linear_cross_entropy`` ->
backward -> ``MonarchMuonOptimizer`` (Monarch factors by Muon, the table, the norms and the head by AdamW), and then a
few tokens sampled greedily, one at a time, and scored.
"""
from __future__ import annotations

import sys

import torch
import torch.nn.functional as F

from . import MonarchMuonOptimizer, butterfly_blk, embedding, linear_cross_entropy
from .workloads import factor_shapes

VOCAB, WIDTH, HIDDEN, NBLOCKS, LAYERS = 509, 256, 512, 2, 2
PAD = 0
BATCH, SEQ = 8, 96


class Block(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.norm = torch.nn.Parameter(torch.ones(WIDTH, dtype=torch.bfloat16))
        self.w = torch.nn.ParameterList(torch.randn(s) / s[2] ** 0.5 for din, dout in ((WIDTH, HIDDEN), (HIDDEN, WIDTH))
                                        for s in factor_shapes(din, dout, NBLOCKS))

    def forward(self, x):
        h = F.rms_norm(x, (WIDTH,), self.norm)
        h = F.silu(butterfly_blk(h, self.w[0], self.w[1]))
        return x + butterfly_blk(h, self.w[2], self.w[3])


class TinyMonarchLM(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.wte = torch.nn.Parameter(torch.randn(VOCAB, WIDTH) * 0.02)
        self.blocks = torch.nn.ModuleList(Block() for _ in range(LAYERS))
        self.ln_f = torch.nn.Parameter(torch.ones(WIDTH, dtype=torch.bfloat16))
        self.lm_head = torch.nn.Parameter(torch.randn(VOCAB, WIDTH) * 0.02)
        self.to(torch.bfloat16)

    def hidden(self, ids):
        x = embedding(ids, self.wte, scale=WIDTH ** 0.5, padding_idx=PAD)
        for b in self.blocks:
            x = b(x)
        return F.rms_norm(x, (WIDTH,), self.ln_f)

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
    ids, scores = [token], []
    for _ in range(count):
        h = model.hidden(torch.tensor([ids[-1]], device=dev))
        best = (h.float() @ model.lm_head.float().T).argmax(-1)
        scores.append(-float(linear_cross_entropy(h, model.lm_head, best, reduction="sum")))
        ids.append(int(best))
    return ids[1:], scores


if __name__ == "__main__":
    lm, history = train(int(sys.argv[1]) if len(sys.argv) > 1 else 60, verbose=True)
    print(f"loss {float(history[0]):.3f} -> {float(history[-5:].mean()):.3f}")
    tokens, logp = generate(lm, 7, 5)
    print("after 7:", tokens, "log-probabilities", [round(s, 2) for s in logp])
