"""Losses at the vocabulary projection of a language model: cases, plain forms and what they cost.

Two operators over the logits z = hidden @ weight.T of a projection onto a large vocabulary, neither of
which keeps the logits:

  ce  cross entropy against one token per row; rows of IGNORE carry no token
  kd  distillation: KL(q || softmax(z / tau)) * tau^2, q = softmax(teacher / tau) over the few logits that
      a teacher kept for the row; entries of index -1 are padding, a row of nothing else carries no loss

`way` "forward" is the loss alone (scoring, evaluation), "train" the loss with the gradients of hidden and
weight. `run` computes them in elementary torch operations, or through b200gemm where `own` is true.
"""
import math
import os
import sys

import torch

own = False

IGNORE = -100
_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gb300-gemm-anatomy_b200")
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}

# The largest case bounds what a drawn one may cost: rows x vocabulary x hidden of a training step.
_MOST = 8192 * 128256 * 4096


def _case(name, op, way, rows, vocab, hidden, dtype="bf16", reduction="mean", ignored=0.0, top=1, tau=1.0):
    return {"name": name, "op": op, "way": way, "rows": rows, "vocab": vocab, "hidden": hidden, "dtype": dtype,
            "reduction": reduction, "ignored": ignored, "top": top, "tau": tau}


def listed():
    return [
        # The log-probability of one token while serving: the projection is read once, latency counts.
        _case("ce_token", "ce", "forward", 1, 128256, 4096, reduction="none"),
        # One token for each of a batch of sequences.
        _case("ce_batch", "ce", "forward", 64, 128256, 4096, reduction="none"),
        # Scoring of a short prompt, odd sizes, half precision, a few padded positions.
        _case("ce_prompt", "ce", "forward", 173, 32003, 2048, "fp16", "none", 0.1),
        # The log-probabilities of a long batch, for its perplexity.
        _case("ce_eval", "ce", "forward", 8192, 128256, 4096, reduction="none"),
        # The smallest training step: launches are all that counts.
        _case("ce_train_small", "ce", "train", 512, 512, 512),
        # A ragged training step in half precision, summed, a quarter of the tokens padded.
        _case("ce_train_ragged", "ce", "train", 1021, 50001, 1016, "fp16", "sum", 0.25),
        # Fine-tuning on answers: half of the tokens are prompts that carry no loss.
        _case("ce_train_masked", "ce", "train", 4096, 32000, 4096, ignored=0.5),
        # A full pre-training step on a large vocabulary.
        _case("ce_train_large", "ce", "train", 8192, 128256, 4096),
        # A small student with a handful of teacher logits.
        _case("kd_train_small", "kd", "train", 64, 1000, 256, top=8, tau=2.0),
        # How far a student is from its teacher, without a step.
        _case("kd_eval", "kd", "forward", 2048, 32000, 4096, reduction="none", top=64),
        # A ragged distillation step in half precision with padded rows, softened.
        _case("kd_train_ragged", "kd", "train", 999, 32003, 1000, "fp16", "sum", 0.2, top=37, tau=2.0),
        # A full distillation step from stored teacher logits.
        _case("kd_train_large", "kd", "train", 4096, 128256, 4096, top=128),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["ce", "ce", "kd"])
    way = rng.choice(["forward", "train"])
    while True:
        rows = _spread(rng, 1, 8192)
        vocab = _spread(rng, 256, 128256)
        hidden = 8 * _spread(rng, 8, 640)  # rows of the operands are whole 16-byte units
        if rows * vocab * hidden <= _MOST:
            break
    return {"op": op, "way": way, "rows": rows, "vocab": vocab, "hidden": hidden, "dtype": rng.choice(["bf16", "bf16", "fp16"]),
            "reduction": rng.choice(["mean", "sum", "none"]), "ignored": rng.choice([0.0, 0.0, round(rng.uniform(0.05, 0.7), 3)]),
            "top": _spread(rng, 1, 128) if op == "kd" else 1, "tau": rng.choice([1.0, 1.0, 2.0, 4.0]) if op == "kd" else 1.0}


def _kept(case):
    """Rows that carry a loss."""
    return case["rows"] - int(case["rows"] * case["ignored"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, V, D, K = case["rows"], case["vocab"], case["hidden"], case["top"]
    dtype = _DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def rand(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    weight = torch.empty((V, D), dtype=dtype, device="cuda")
    for v in range(0, V, 16384):
        weight[v:v + 16384] = randn(min(16384, V - v), D) * 0.02
    target = torch.randint(0, V, (T,), generator=g, device="cuda")
    # The model knows something of the token: its logit stands up to 10 above the others'.
    pull = 10 * rand(T, 1) / (D * 0.02 ** 2) * min(1.0, D / 1024)
    hidden = (randn(T, D) + weight[target].float() * pull).to(dtype)
    drop = torch.randperm(T, generator=g, device="cuda")[:T - _kept(case)]
    state = {"case": dict(case), "hidden": hidden, "weight": weight}
    # What reaches the loss from above, as from a loss scale or a weight for each row.
    up = (rand(T) + 0.5) if case["reduction"] == "none" else (rand(1) + 0.5).reshape(())
    state["up"] = up
    if case["op"] == "ce":
        target[drop] = IGNORE
        state["target"] = target
    else:
        # K different tokens, the first the likeliest; some rows kept fewer.
        step = 1 + (rand(T, 1) * (max(V // K, 1) - 1)).long()
        index = (target[:, None] + torch.arange(K, device="cuda") * step) % V
        teacher = (10 - 1.5 * torch.arange(1, K + 1, device="cuda").float().log2() + randn(T, K)).sort(dim=1, descending=True).values
        short = rand(T) < 0.1
        index[short, K - K // 4:] = -1
        index[drop] = -1
        state["index"], state["teacher"] = index, teacher
    return state


def run(s):
    c = s["case"]
    return _run_own(s, c) if own else _run_plain(s, c)


def _run_own(s, c):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from b200gemm import vocab_loss
    train = c["way"] == "train"
    h, w = s["hidden"].detach().requires_grad_(train), s["weight"].detach().requires_grad_(train)
    if c["op"] == "ce":
        loss = vocab_loss.linear_cross_entropy(h, w, s["target"], ignore_index=IGNORE, reduction=c["reduction"])
    else:
        loss = vocab_loss.linear_distillation(h, w, s["teacher"], s["index"], temperature=c["tau"], reduction=c["reduction"])
    if not train:
        return {"loss": loss}
    dh, dw = torch.autograd.grad(loss, (h, w), s["up"])
    return {"loss": loss.detach(), "d_hidden": dh, "d_weight": dw}


def _run_plain(s, c):
    tau = c["tau"]
    h, w = s["hidden"].float(), s["weight"].float()
    z = h @ w.t()
    if tau != 1.0:
        z = z / tau
    top = z.max(dim=1, keepdim=True).values
    lse = (z - top).exp().sum(dim=1, keepdim=True).log() + top
    if c["op"] == "ce":
        kept = s["target"] != IGNORE
        index = torch.where(kept, s["target"], 0)[:, None]
        loss = (lse - z.gather(1, index))[:, 0]
        q = torch.ones_like(index, dtype=torch.float32)
    else:
        there = s["index"] >= 0
        kept = there.any(dim=1)
        index = torch.where(there, s["index"], 0)
        t = torch.where(there, s["teacher"].float() / tau, -math.inf)
        t = torch.where(kept[:, None], t, 0.0)
        t = t - t.max(dim=1, keepdim=True).values
        q = t.exp() / t.exp().sum(dim=1, keepdim=True)
        logq = t - t.exp().sum(dim=1, keepdim=True).log()
        loss = torch.where(q > 0, q * (logq + (lse - z.gather(1, index))), 0.0).sum(dim=1) * tau ** 2
    loss = torch.where(kept, loss, 0.0)
    if c["reduction"] == "mean":
        n = kept.sum().clamp(min=1)
        out, up = loss.sum() / n, s["up"] / n
    elif c["reduction"] == "sum":
        out, up = loss.sum(), s["up"]
    else:
        out, up = loss, s["up"]
    if c["way"] != "train":
        return {"loss": out}
    # dloss/dz = (softmax(z) - q) * tau, for the rows that carry a loss.
    d = (z - lse).exp().scatter_add_(1, index, -q)
    d = d * torch.where(kept, up * tau, 0.0)[:, None]
    return {"loss": out, "d_hidden": (d @ w).to(s["hidden"].dtype), "d_weight": (d.t() @ h).to(s["weight"].dtype)}


def work(case):
    n, T, V, D, K = _kept(case), case["rows"], case["vocab"], case["hidden"], case["top"]
    side = T * 8 if case["op"] == "ce" else T * K * 12  # tokens, or the teacher's indices and logits
    out = 4 * T if case["reduction"] == "none" else 4
    bytes_ = 2 * (n * D + V * D) + side + out
    flops = 2 * n * V * D
    if case["way"] == "train":
        bytes_ += 2 * (T * D + V * D) + out
        flops *= 3  # the logits, and a product for each gradient
    return {"bytes": bytes_, "flops": flops}


def exact(case, seed):
    """The same in 64 bits, from the definition: log-probabilities of the rows that carry a loss, in pieces of the
    rows, and torch's derivative of the logits' loss."""
    s = prepare(case, seed)
    T, V, D = case["rows"], case["vocab"], case["hidden"]
    train, tau = case["way"] == "train", case["tau"]
    w = s["weight"].double()
    rows = (s["target"] != IGNORE if case["op"] == "ce" else (s["index"] >= 0).any(1)).nonzero()[:, 0]
    up = s["up"].double().expand(T) if case["reduction"] != "mean" else (s["up"].double() / max(len(rows), 1)).expand(T)
    loss = torch.zeros(T, dtype=torch.float64, device="cuda")
    dh = torch.zeros((T, D), dtype=torch.float64, device="cuda") if train else None
    dw = torch.zeros((V, D), dtype=torch.float64, device="cuda") if train else None
    for r in rows.split(1024):
        h = s["hidden"][r].double()
        z = (h @ w.t()).requires_grad_(train)
        logp = torch.log_softmax(z / tau, dim=1)
        if case["op"] == "ce":
            part = -logp.gather(1, s["target"][r][:, None])[:, 0]
        else:
            there = s["index"][r] >= 0
            logq = torch.log_softmax(s["teacher"][r].double().div(tau).masked_fill(~there, -math.inf), dim=1)
            term = logq.exp() * (logq.masked_fill(~there, 0.0) - logp.gather(1, s["index"][r].clamp(min=0)))
            part = term.sum(dim=1) * tau ** 2
        loss[r] = part.detach()
        if train:
            dz, = torch.autograd.grad(part, z, up[r])
            dh[r] = dz @ w
            dw.addmm_(dz.t(), h)
    if case["reduction"] == "mean":
        loss = loss.sum() / max(len(rows), 1)
    elif case["reduction"] == "sum":
        loss = loss.sum()
    return {"loss": loss, "d_hidden": dh, "d_weight": dw} if train else {"loss": loss}
