"""The two ends of a language model as cases to time and to compare: the head with its loss, and the embedding.

* ``op="loss"``: ``linear_cross_entropy`` of hidden states against a head of ``vocab`` rows.  ``train`` False is the
  loss alone (evaluation; with ``reduction`` "none" the scoring of given tokens), True the loss and its gradients.
* ``op="lookup"`` / ``op="embed"``: ``embedding`` of token ids; alone, or with the gradient of its table (training).

Widths and the vocabulary of 50304 are those of the benchmark configurations (toy 512, 257M 1024, 1.3B 2048, 6.89B
4096: ``monarch_muon_amd/workloads.py``) and of a 124M model (768); 1024 tokens are one training sequence.
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"
VOCAB = 50304
IGNORE = -100
_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
#: Tokens x vocabulary x width of the largest loss case, forward products; a training case makes three of them.
MOST_PRODUCT = 3 * 4096 * VOCAB * 4096
MOST_TOKENS = 16384


def _loss(name, tokens, width, train, reduction="mean", vocab=VOCAB, ignored=0.0):
    """``ignored``: the share of targets that are ``ignore_index``."""
    return dict(name=name, op="loss", tokens=tokens, width=width, vocab=vocab, train=train, reduction=reduction,
                ignored=ignored)


def _emb(name, op, tokens, width, dtype="bf16", vocab=VOCAB, scale=1.0, padded=0.0):
    """``padded``: the share of ids that are the padding id, which takes no gradient."""
    return dict(name=name, op=op, tokens=tokens, width=width, vocab=vocab, dtype=dtype, scale=scale, padded=padded)


def listed():
    return [
        # generation: the log-probability of one token under the 6.89B head, which is one read of the head
        _loss("score-1-6.89b", 1, 4096, False, "none"),
        # scoring the next tokens of a ragged batch of 33 sequences under the 1.3B head
        _loss("score-33-1.3b", 33, 2048, False, "none"),
        # evaluation: one micro-batch (4 x 1024) of the 6.89B model
        _loss("eval-6.89b", 4096, 4096, False),
        # training the toy model: one short ragged micro-batch
        _loss("train-toy", 1000, 512, True),
        # fine-tuning a 124M model on the GPT-2 vocabulary (odd, not padded), a third of the tokens a masked prompt
        _loss("train-124m-odd", 2047, 768, True, vocab=50257, ignored=0.33),
        # training the 257M model: 16 sequences of 1024
        _loss("train-257m", 16384, 1024, True),
        # training the 6.89B model at the benchmark's micro-batch (4 x 1024)
        _loss("train-6.89b", 4096, 4096, True),
        # generation: the embeddings of a batch of eight sequences, one token each
        _emb("lookup-8-6.89b", "lookup", 8, 4096),
        # training and prompt processing: the embeddings of 16 sequences of 1024, scaled by the root of the width
        _emb("lookup-6.89b", "lookup", 16384, 4096, scale=64.0),
        # training the toy model in fp32: one short ragged micro-batch
        _emb("embed-toy-f32", "embed", 1000, 512, "f32"),
        # training the 257M model: 64 sequences of 1024, an eighth padding; a common word occurs thousands of times
        _emb("embed-257m", "embed", 65536, 1024, padded=0.125),
        # training the 6.89B model: 16 sequences of 1024
        _emb("embed-6.89b", "embed", 16384, 4096, scale=64.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    vocab = rng.choice([VOCAB, 50257, _log(rng, 1000, 131072)])
    width = 8 * _log(rng, 32, 512)                       # 256 .. 4096
    if rng.random() < 0.6:
        train = rng.random() < 0.6
        most = MOST_PRODUCT // (width * vocab * (3 if train else 1))
        tokens = _log(rng, 64 if train else 1, min(MOST_TOKENS, most))
        reduction = rng.choice(["mean", "sum"]) if train else rng.choice(["mean", "none"])
        c = _loss("", tokens, width, train, reduction, vocab, rng.choice([0.0, round(rng.random(), 3)]))
    else:
        op, dtype = rng.choice(["lookup", "embed"]), rng.choice(["bf16", "bf16", "f32"])
        width += rng.choice([0, 0, rng.randint(1, 7)])
        most = 65536 * 1024 // width // (1 if dtype == "bf16" else 2)
        most_vocab = VOCAB * 4096 // width // (1 if dtype == "bf16" else 2)
        c = _emb("", op, _log(rng, 1, most), width, dtype, min(vocab, most_vocab), rng.choice([1.0, round(width ** 0.5, 3)]),
                 rng.choice([0.0, round(0.5 * rng.random(), 3)]))
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ids(g, n, vocab):
    """Token ids as text has them: the k-th commonest with a frequency of about 1 / k."""
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1)).long() - 1).clamp_(0, vocab - 1)


def prepare(case, seed):
    g = _gen(seed)
    T, D, V = case["tokens"], case["width"], case["vocab"]
    if case["op"] == "loss":
        w = (torch.randn(V, D, generator=g, device=DEV) * 0.02).bfloat16()
        y = _ids(g, T, V)
        # normalised hidden states that know their target more or less well: it stands 0 to 12 above a random logit
        wy = w[y].float()
        lift = 12 * torch.rand(T, 1, generator=g, device=DEV) / wy.square().sum(1, keepdim=True).clamp_min(1e-6)
        x = (torch.randn(T, D, generator=g, device=DEV) + lift * wy).bfloat16()
        masked = torch.rand(T, generator=g, device=DEV) < case["ignored"]
        masked[0] = False
        y = torch.where(masked, IGNORE, y)
        return dict(case=case, x=x.requires_grad_(case["train"]), w=w.requires_grad_(case["train"]), y=y)
    dt = _DT[case["dtype"]]
    pad = V - 1
    i = _ids(g, T, V)
    i = torch.where(torch.rand(T, generator=g, device=DEV) < case["padded"], pad, i)
    s = dict(case=case, i=i, pad=pad if case["padded"] else None)
    s["w"] = (torch.randn(V, D, generator=g, device=DEV) * 0.02).to(dt).requires_grad_(case["op"] == "embed")
    if case["op"] == "embed":
        s["dy"] = (torch.randn(T, D, generator=g, device=DEV) * 1e-3).to(dt)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if c["op"] == "loss":
        return (_own_loss if own else _plain_loss)(c, s["x"], s["w"], s["y"])
    return (_own_embedding if own else _plain_embedding)(c, s)


def _own_loss(c, x, w, y):
    from monarch_muon_amd import linear_cross_entropy
    loss = linear_cross_entropy(x, w, y, ignore_index=IGNORE, reduction=c["reduction"])
    if not c["train"]:
        return loss
    dx, dw = torch.autograd.grad(loss, (x, w))
    return loss.detach(), dx, dw


def _own_embedding(c, s):
    from monarch_muon_amd import embedding
    out = embedding(s["i"], s["w"], scale=c["scale"], padding_idx=s["pad"])
    if c["op"] == "lookup":
        return out
    return out.detach(), torch.autograd.grad(out, s["w"], s["dy"])[0]


@torch.no_grad()
def _plain_loss(c, x, w, y):
    xf, wf = x.float(), w.float()
    logits = xf @ wf.T
    top = logits.amax(1, keepdim=True)
    p = (logits - top).exp_()
    total = p.sum(1, keepdim=True)
    valid = y != IGNORE
    at = torch.where(valid, y, 0).unsqueeze(1)
    nll = torch.where(valid, (total.log() + top - logits.gather(1, at)).squeeze(1), 0.0)
    count = valid.sum()
    loss = nll if c["reduction"] == "none" else nll.sum() if c["reduction"] == "sum" else nll.sum() / count
    if not c["train"]:
        return loss
    d = p.div_(total)
    d.scatter_add_(1, at, torch.full_like(top, -1.0))
    d *= (valid / count if c["reduction"] == "mean" else valid.float()).unsqueeze(1)
    return loss, (d @ wf).bfloat16(), (d.T @ xf).bfloat16()


@torch.no_grad()
def _plain_embedding(c, s):
    w, i = s["w"], s["i"]
    out = (w[i].float() * c["scale"]).to(w.dtype)
    if c["op"] == "lookup":
        return out
    dy = s["dy"].float() * c["scale"]
    if s["pad"] is not None:
        dy = dy * (i != s["pad"]).unsqueeze(1)
    return out, torch.zeros(w.shape, device=w.device).index_add_(0, i, dy).to(w.dtype)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and what it should return
# ---------------------------------------------------------------------------
def _distinct(tokens, vocab):
    """The expected number of distinct ids among ``tokens`` of ``_ids``."""
    p = np.diff(np.log(np.arange(1, vocab + 2))) / math.log(vocab + 1)
    return float((-np.expm1(tokens * np.log1p(-np.minimum(p, 1 - 1e-12)))).sum())


def work(case):
    T, D, V = case["tokens"], case["width"], case["vocab"]
    if case["op"] == "loss":
        train = case["train"]
        return {"bytes": (4 if train else 2) * (T + V) * D + 8 * T, "flops": (6 if train else 2) * T * V * D}
    b = 2 if case["dtype"] == "bf16" else 4
    lookup = b * D * (T + _distinct(T, V)) + 8 * T
    return {"bytes": lookup + (b * D * (T + V) if case["op"] == "embed" else 0), "flops": 0}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "loss":
            return _exact_loss(case, s["x"].double(), s["w"].double(), s["y"])
        w, i = s["w"].double(), s["i"]
        out = torch.index_select(w, 0, i) * case["scale"]
        if case["op"] == "lookup":
            return out
        grad = torch.zeros_like(w)
        keep = i != s["pad"] if s["pad"] is not None else torch.ones_like(i, dtype=torch.bool)
        grad.index_put_((i[keep],), s["dy"].double()[keep], accumulate=True)
        return out, grad * case["scale"]


def _exact_loss(case, x, w, y):
    lp = torch.log_softmax(x @ w.T, 1)
    kept = torch.nonzero(y != IGNORE).squeeze(1)
    nll = torch.zeros_like(lp[:, 0])
    nll[kept] = -lp[kept, y[kept]]
    share = 1.0 / len(kept) if case["reduction"] == "mean" else 1.0
    loss = nll if case["reduction"] == "none" else nll.sum() * share
    if not case["train"]:
        return loss
    d = torch.zeros_like(lp)
    d[kept] = lp[kept].exp() * share
    d[kept, y[kept]] -= share
    return loss, d @ w, d.T @ x
