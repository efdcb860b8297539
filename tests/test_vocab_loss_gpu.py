"""Losses at the vocabulary projection on the GPU against 64-bit results, element by element."""
import math

import pytest
import torch

import vocab_loss_reference as ref

pytestmark = pytest.mark.gpu

IGNORE = -100
BF16, FP16 = torch.bfloat16, torch.float16


def make(rows, vocab, hidden, dtype=BF16, seed=0, std=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(rows, hidden, generator=g, device="cuda").to(dtype)
    w = (torch.randn(vocab, hidden, generator=g, device="cuda") * (std or 2.0 / math.sqrt(hidden))).to(dtype)
    return g, h, w


def upstream(g, rows, reduction):
    if reduction == "none":
        return torch.randn(rows, generator=g, device="cuda")
    return torch.rand((), generator=g, device="cuda") + 0.5


def run(fn, h, w, args, up, **kw):
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = fn(h, w, *args, **kw)
    dh, dw = torch.autograd.grad(loss, (h, w), up)
    return loss.detach(), dh, dw


def check_all(got, want):
    loss, dh, dw = got
    rl, bl, rh, bh, rw, bw = want
    ref.check("loss", loss, rl, bl)
    ref.check("d_hidden", dh, rh, bh)
    ref.check("d_weight", dw, rw, bw)


def ce(rows, vocab, hidden, dtype=BF16, reduction="mean", ignored=0.0, seed=0, index=torch.int64, poison=True):
    from b200gemm import vocab_loss
    g, h, w = make(rows, vocab, hidden, dtype, seed)
    target = torch.randint(0, vocab, (rows,), generator=g, device="cuda").to(index)
    drop = torch.randperm(rows, generator=g, device="cuda")[:round(rows * ignored)]
    target[drop] = IGNORE
    if poison and len(drop):  # what padding holds must not matter
        h[drop[::2]] = math.nan
        h[drop[1::2]] = math.inf
    up = upstream(g, rows, reduction)
    got = run(vocab_loss.linear_cross_entropy, h, w, (target,), up, reduction=reduction)
    kept, idx, q = ref.targets_of(target, IGNORE)
    check_all(got, ref.reference(h, w, kept, idx, q, 1.0, reduction, up))
    return got


SIZES = [(1, 1, 8), (1, 300, 64), (3, 257, 72), (127, 1000, 136), (128, 512, 128), (129, 513, 200), (256, 256, 256),
         (300, 4099, 328), (513, 700, 64), (1000, 31, 1032)]


@pytest.mark.parametrize("rows,vocab,hidden", SIZES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_cross_entropy(rows, vocab, hidden, dtype):
    ce(rows, vocab, hidden, dtype)


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("ignored", [0.0, 0.3, 1.0])
@pytest.mark.parametrize("rows", [1, 5, 100, 257, 700])
def test_cross_entropy_masks(rows, ignored, reduction):
    loss, dh, dw = ce(rows, 777, 96, BF16 if rows % 2 else FP16, reduction, ignored, seed=rows, index=torch.int32)
    if ignored == 1.0:
        assert not loss.any() and not dh.any() and not dw.any()


@pytest.mark.parametrize("vocab", [32768, 32769, 40007])
def test_cross_entropy_several_pieces(vocab):
    """More columns than one piece of the backward pass holds; a last piece of one column."""
    from b200gemm import vocab_loss
    assert (vocab_loss.policy(4096, vocab, 64)["pieces"] > 1) == (vocab > 32768)
    ce(4096, vocab, 64, reduction="sum", ignored=0.1)


def kd(rows, vocab, hidden, top, dtype=BF16, reduction="mean", tau=1.0, ignored=0.0, seed=0, tdtype=torch.float32,
       index=torch.int64, change=None):
    from b200gemm import vocab_loss
    g, h, w = make(rows, vocab, hidden, dtype, seed)
    logits = (torch.randn(rows, top, generator=g, device="cuda") * 3).to(tdtype)
    idx = torch.randint(0, vocab, (rows, top), generator=g, device="cuda").to(index)
    short = torch.rand(rows, generator=g, device="cuda") < 0.3
    idx[short, top - top // 3:] = -1
    drop = torch.randperm(rows, generator=g, device="cuda")[:round(rows * ignored)]
    idx[drop] = -1
    h[drop] = math.nan
    if change is not None:
        change(logits, idx)
    up = upstream(g, rows, reduction)
    got = run(vocab_loss.linear_distillation, h, w, (logits, idx), up, temperature=tau, reduction=reduction)
    kept, i64, q = ref.teacher_of(logits, idx, tau)
    check_all(got, ref.reference(h, w, kept, i64, q, tau, reduction, up))
    return got


@pytest.mark.parametrize("rows,vocab,hidden,top", [(1, 1, 8, 1), (1, 500, 64, 7), (7, 33, 64, 256), (130, 1000, 136, 32),
                                                   (300, 4099, 200, 37), (513, 700, 64, 129)])
@pytest.mark.parametrize("dtype,tau", [(BF16, 1.0), (FP16, 2.5)])
def test_distillation(rows, vocab, hidden, top, dtype, tau):
    kd(rows, vocab, hidden, top, dtype, tau=tau)


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("ignored", [0.0, 0.4, 1.0])
@pytest.mark.parametrize("tdtype", [torch.float32, BF16, FP16])
def test_distillation_masks(reduction, ignored, tdtype):
    kd(205, 900, 72, 20, reduction=reduction, ignored=ignored, tau=0.7, tdtype=tdtype, index=torch.int32)


def test_distillation_several_pieces():
    kd(4096, 40007, 64, 16, reduction="sum", tau=2.0)


def test_distillation_all_entries_of_one_tile():
    """Every entry of every row within the same few columns, and the same token often."""
    def change(logits, idx):
        idx.copy_(torch.randint(290, 300, idx.shape, device=idx.device))
    kd(160, 1000, 64, 64, change=change)


def test_distillation_minus_infinity_is_padding():
    def change(logits, idx):
        logits[::2, ::3] = -math.inf
        logits[5] = -math.inf
    loss, dh, _ = kd(60, 300, 64, 9, reduction="none", change=change)
    assert loss[5] == 0 and not dh[5].any()
