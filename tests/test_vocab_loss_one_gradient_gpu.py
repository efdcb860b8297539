"""Losses at the vocabulary projection: one gradient alone is, bit for bit, that of a full step.

Without d_hidden, dW waits for G by itself; without d_weight, the next piece's G follows dH directly."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def problem(kind, rows, vocab, hidden, ignored, dtype):
    from b200gemm import vocab_loss
    g = torch.Generator(device="cuda").manual_seed(rows)
    h = torch.randn(rows, hidden, generator=g, device="cuda").to(dtype)
    w = (torch.randn(vocab, hidden, generator=g, device="cuda") / 8).to(dtype)
    drop = torch.randperm(rows, generator=g, device="cuda")[:round(rows * ignored)]
    h[drop] = float("nan")
    if kind == "ce":
        f = vocab_loss.linear_cross_entropy
        args = (torch.randint(0, vocab, (rows,), generator=g, device="cuda"),)
        args[0][drop] = -100
    else:
        f = vocab_loss.linear_distillation
        args = (torch.randn(rows, 6, generator=g, device="cuda"), torch.randint(0, vocab, (rows, 6), generator=g, device="cuda"))
        args[1][drop] = -1
    up = torch.rand(rows, generator=g, device="cuda") + 0.5

    def step(want_h, want_w):
        a, b = h.detach().requires_grad_(want_h), w.detach().requires_grad_(want_w)
        return torch.autograd.grad(f(a, b, *args, reduction="none"), [t for t in (a, b) if t.requires_grad], up)
    return step


@pytest.mark.parametrize("kind,dtype", [("ce", torch.bfloat16), ("kd", torch.bfloat16), ("ce", torch.float16)])
@pytest.mark.parametrize("rows,vocab,hidden,ignored,what", [
    (4096, 40007, 64, 0.3, "pieces"), (4090, 56976, 264, 0.97, "pieces"), (5000, 300, 64, 0.2, "splits_weight"),
    (5000, 300, 64, 0.995, "splits_weight"), (130, 20000, 64, 0.5, "splits_hidden"), (257, 700, 136, 1.0, "launches_forward")])
def test_one_gradient_at_a_time(kind, dtype, rows, vocab, hidden, ignored, what):
    from b200gemm import vocab_loss
    assert vocab_loss.policy(rows, vocab, hidden, top=6 if kind == "kd" else 0, dtype=dtype)[what] > 1
    step = problem(kind, rows, vocab, hidden, ignored, dtype)
    dh, dw = step(True, True)
    torch.cuda.synchronize()
    differ = torch.zeros((), dtype=torch.bool, device="cuda")
    for _ in range(10):  # close behind one another, in turn
        for got, want in zip((*step(True, False), *step(False, True), *step(True, True)), (dh, dw, dh, dw)):
            differ |= (got != want).any()
    assert not differ
    assert dh.isfinite().all() and dw.isfinite().all() and bool(dh.any()) == (ignored < 1)
