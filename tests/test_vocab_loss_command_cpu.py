"""The check that the losses' command makes before it times anything: what it must not let pass."""
import math

import pytest
import torch

from b200gemm.cli import vocab_loss as cli


def step(loss, tau):
    g = torch.Generator().manual_seed(1)
    rows, vocab, hidden, top = 60, 200, 32, 4
    h, w = torch.randn(rows, hidden, generator=g), torch.randn(vocab, hidden, generator=g) / 4
    kept = torch.ones(rows, dtype=torch.bool)
    kept[::6] = False
    if loss == "ce":
        index, q = torch.randint(0, vocab, (rows, 1), generator=g), kept[:, None].float()
    else:
        index = torch.randint(0, vocab, (rows, top), generator=g)
        q = torch.softmax(torch.randn(rows, top, generator=g), 1) * kept[:, None]
    h.requires_grad_()
    w.requires_grad_()
    logp = torch.log_softmax(h @ w.t() / tau, 1)
    dense = torch.zeros(rows, vocab).scatter_add_(1, index, q)
    losses = tau ** 2 * (torch.xlogy(dense, dense) - dense * logp).sum(1)
    dh, dw = torch.autograd.grad(losses.sum() / int(kept.sum()), (h, w))
    return h.detach(), w.detach(), index, q, kept, tau, losses.detach(), dh, dw


@pytest.mark.parametrize("loss,tau", [("ce", 1.0), ("kd", 2.0)])
def test_right_results_pass(loss, tau):
    *given, losses, dh, dw = step(loss, tau)
    cli._check(*given, losses, None, None)
    cli._check(*given, None, dh, dw)


@pytest.mark.parametrize("loss,tau", [("ce", 1.0), ("kd", 2.0)])
@pytest.mark.parametrize("value", [math.nan, math.inf, 3.0])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_wrong_results_do_not(loss, tau, value, which):
    *given, losses, dh, dw = step(loss, tau)
    index, kept = given[2], given[4]
    out = [losses, dh, dw]
    # The first row, or lowest token, of those that are sampled.
    out[which][int(index[kept].min()) if which == 2 else int(kept.nonzero()[0, 0])] += value
    with pytest.raises(RuntimeError, match=("losses", "activations", "weight")[which]):
        cli._check(*given, *(out if which else (losses, None, None)))
