"""Distillation at the vocabulary projection at the ends of the range of temperatures."""
import math

import pytest
import torch

import vocab_loss_reference as ref
import vocab_loss_rows_reference as rows_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hidden", [64, 1000])
@pytest.mark.parametrize("tau", [2.0 ** -20, 2.0 ** -14, 2.0 ** -6, 2.0 ** 10, 2.0 ** 20])
@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_ends_of_the_range(dtype, hidden, tau, reduction):
    """Where z / tau is 2^24 and more, its steps in 32 bits are whole powers of e: which tokens share the
    probability is open, but it stays one, and the gradients what that allows."""
    from b200gemm import vocab_loss
    rows, vocab, top = 60, 700, 5
    g = torch.Generator(device="cuda").manual_seed(2)
    h = torch.randn(rows, hidden, generator=g, device="cuda").to(dtype).requires_grad_()
    w = (torch.randn(vocab, hidden, generator=g, device="cuda") * (8 / math.sqrt(hidden))).to(dtype).requires_grad_()
    logits = torch.randn(rows, top, generator=g, device="cuda") * min(tau, 1.0)
    index = torch.randint(0, vocab, (rows, top), generator=g, device="cuda")
    up = torch.rand(rows, generator=g, device="cuda") + 1.0 if reduction == "none" else torch.tensor(1.9, device="cuda")
    up = up / tau  # gradients of the size of the weights'
    loss = vocab_loss.linear_distillation(h, w, logits, index, temperature=tau, reduction=reduction)
    dh, dw = torch.autograd.grad(loss, (h, w), up)
    kept, i64, q = ref.teacher_of(logits, index, tau)
    want, bound, *_ = ref.reference(h.detach(), w.detach(), kept, i64, q, tau, reduction, up)
    ref.check("loss", loss.detach(), want, bound)
    want_h, bh, want_w, bw = rows_ref.gradients(h.detach(), w.detach(), kept, i64, q, tau, up.expand(rows))
    ref.check("d_hidden", dh, want_h, bh)
    ref.check("d_weight", dw, want_w, bw)
    # p and q are distributions: no row moves by more than twice the largest weight, nor a token by more than
    # twice the rows' sum. 1 + 2^-6 for the roundings to 16 bits (a half step twice) and the sums in 32.
    gmax = tau * up.abs().expand(rows)[:, None].double() * (1 + 2.0 ** -6)
    w64, h64 = w.detach().double().abs(), h.detach().double().abs()
    assert bool((dh.double().abs() <= gmax * 2 * w64.max(0).values).all())
    assert bool((dw.double().abs() <= (gmax * h64).sum(0) * (1 + 2.0 ** -6)).all())
