"""Losses at the vocabulary projection: probabilities of a large vocabulary, and weights of rows, in half precision."""
import math

import pytest
import torch

import vocab_loss_reference as ref
import vocab_loss_rows_reference as rows_ref

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def make(rows, vocab, hidden, dtype, seed=0, spread=0.5, common=0.0):
    """Logits of standard deviation `spread`; the rows of weight share a component of size `common`."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(rows, hidden, generator=g, device="cuda").to(dtype)
    w = torch.randn(vocab, hidden, generator=g, device="cuda") * (spread / math.sqrt(hidden))
    w = (w + common * torch.randn(hidden, generator=g, device="cuda")).to(dtype)
    return g, h, w


def targets(kind, g, rows, vocab, top=5):
    if kind == "ce":
        return (torch.randint(0, vocab, (rows,), generator=g, device="cuda"),)
    return (torch.randn(rows, top, generator=g, device="cuda"), torch.randint(0, vocab, (rows, top), generator=g, device="cuda"))


def step(kind, h, w, args, up, reduction="none", tau=1.0):
    from b200gemm import vocab_loss
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    if kind == "ce":
        loss = vocab_loss.linear_cross_entropy(h, w, *args, reduction=reduction)
    else:
        loss = vocab_loss.linear_distillation(h, w, *args, reduction=reduction, temperature=tau)
    return (loss.detach(), *torch.autograd.grad(loss, (h, w), up))


def distribution(kind, args, tau):
    return ref.targets_of(args[0], -100) if kind == "ce" else ref.teacher_of(*args, tau)


def check(kind, h, w, args, up, got, tau=1.0):
    dh, bh, dw, bw = rows_ref.gradients(h, w, *distribution(kind, args, tau), tau, up)
    ref.check("d_hidden", got[1], dh, bh)
    ref.check("d_weight", got[2], dw, bw)
    return dh, bh, dw, bw


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("kind,tau", [("ce", 1.0), ("kd", 2.0)])
@pytest.mark.parametrize("vocab,common", [(128256, 0.0), (128256, 1.0), (32003, 1.0)])
def test_small_probabilities(dtype, kind, tau, vocab, common):
    """Probabilities near 2^-17 keep the type's own precision. All rows weigh the same, as in a sum."""
    g, h, w = make(24, vocab, 64, dtype, common=common)
    args = targets(kind, g, 24, vocab)
    up = torch.full((24,), 1024.0, device="cuda")  # the results' own steps are no limit
    got = step(kind, h, w, args, up[0], "sum", tau)
    dh, bh, dw, bw = check(kind, h, w, args, up, got, tau)
    # The bounds tell something: zeros, or tokens without their probability, are outside of them.
    assert not bool((dw.abs() <= bw).all(1).any()) and not bool((dh.abs() <= bh).all(1).any())


@pytest.mark.parametrize("kind", ["ce", "kd"])
def test_confident_rows_reach_all_tokens(kind):
    """Rows that are sure of their token leave the others 2^-20 and less: none of it is lost."""
    g, h, w = make(16, 50001, 64, FP16, spread=0.1)
    args = targets(kind, g, 16, 50001, 1)
    token = args[-1].reshape(-1)
    h[:, 0], w[:, 0] = 4.0, 0.0
    w[token, 0] = 3.5  # 14 above the others
    up = torch.full((16,), 512.0, device="cuda")
    got = step(kind, h, w, args, up[0], "sum")
    dh, bh, dw, bw = check(kind, h, w, args, up, got)
    other = torch.ones(50001, dtype=torch.bool, device="cuda")
    other[token] = False
    assert not bool((dw[other].abs() <= bw[other]).all(1).any())
