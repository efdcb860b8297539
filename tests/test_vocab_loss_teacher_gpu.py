"""Distillation at the vocabulary projection: a teacher's logits at the ends of their type's range."""
import math

import pytest
import torch

import vocab_loss_reference as ref

pytestmark = pytest.mark.gpu


def check(logits, index, tau, hidden=64, vocab=300, reduction="none"):
    from b200gemm import vocab_loss
    rows = logits.shape[0]
    g = torch.Generator(device="cuda").manual_seed(rows)
    h = torch.randn(rows, hidden, generator=g, device="cuda").bfloat16().requires_grad_()
    w = (torch.randn(vocab, hidden, generator=g, device="cuda") / 4).bfloat16().requires_grad_()
    up = torch.rand(rows, generator=g, device="cuda") + 0.5
    loss = vocab_loss.linear_distillation(h, w, logits, index, temperature=tau, reduction=reduction)
    dh, dw = torch.autograd.grad(loss, (h, w), up)
    kept, i64, q = ref.teacher_of(logits, index, tau)
    rl, bl, rh, bh, rw, bw = ref.reference(h.detach(), w.detach(), kept, i64, q, tau, reduction, up)
    for name, a, b, c in (("loss", loss.detach(), rl, bl), ("d_hidden", dh, rh, bh), ("d_weight", dw, rw, bw)):
        ref.check(name, a, b, c)
    return loss.detach()


def entries(rows, top, dtype, vocab=300, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    index = torch.stack([torch.randperm(vocab, generator=g, device="cuda")[:top] for _ in range(rows)])
    return torch.randn(rows, top, generator=g, device="cuda").to(dtype), index


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tau", [0.25, 0.9, 1.0, 3.0])
def test_masks_of_the_lowest_value(dtype, tau):
    """The lowest finite value is a logit, not padding: nothing beside others, a uniform teacher alone."""
    logits, index = entries(40, 9, dtype)
    low = torch.finfo(dtype).min
    logits[::3, 4:] = low
    logits[5] = low
    logits[7, :4] = low
    logits[7, 4:] = -math.inf
    logits[8] = -math.inf
    loss = check(logits, index, tau)
    assert loss.isfinite().all() and loss[8] == 0 and loss[5] != 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tau", [0.25, 1.0, 3.0])
def test_logits_of_the_highest_value(dtype, tau):
    logits, index = entries(40, 9, dtype, seed=1)
    info = torch.finfo(dtype)
    logits[::3, 2] = info.max
    logits[1::3, 5:7] = info.max  # two of them share the row
    logits[6, 0] = info.min
    assert check(logits, index, tau).isfinite().all()


@pytest.mark.parametrize("tau", [0.5, 1.0])
def test_no_distribution(tau):
    """NaN and +infinity in an entry that counts are no distribution; in padding they are padding."""
    logits, index = entries(6, 5, torch.float32)
    logits[1, 2], logits[2, 0] = math.nan, math.inf
    logits[3, 3], index[3, 3] = math.nan, -1
    logits[4, 1], index[4, 1] = math.inf, -5
    from b200gemm import vocab_loss
    g = torch.Generator(device="cuda").manual_seed(0)
    h, w = (torch.randn(n, 64, generator=g, device="cuda").bfloat16() for n in (6, 300))
    loss = vocab_loss.linear_distillation(h, w, logits, index, temperature=tau, reduction="none")
    assert loss.isnan().tolist() == [False, True, True, False, False, False]
