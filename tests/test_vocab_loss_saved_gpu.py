"""Losses at the vocabulary projection: what the backward pass reads again may come back in another layout.

Saved-tensor hooks may give back the same values with other strides or another start; the gradients are
those of the values, bit for bit, and a tensor that is not what was saved is refused."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def inputs(kind, rows=70, vocab=301, hidden=80, dtype=BF16, pitched=True):
    """hidden and weight as column slices of wider tensors whose other columns are NaN."""
    g = torch.Generator(device="cuda").manual_seed(3)
    wide_h = torch.full((rows, hidden + 24), math.nan, dtype=dtype, device="cuda")
    wide_w = torch.full((vocab, hidden + 16), math.nan, dtype=dtype, device="cuda")
    h, w = (wide_h[:, 16:16 + hidden], wide_w[:, 8:8 + hidden]) if pitched else (
        torch.empty(rows, hidden, dtype=dtype, device="cuda"), torch.empty(vocab, hidden, dtype=dtype, device="cuda"))
    h.copy_(torch.randn(rows, hidden, generator=g, device="cuda"))
    w.copy_(torch.randn(vocab, hidden, generator=g, device="cuda") / 4)
    if kind == "ce":
        t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        t[::7] = -100
        args = (t,)
    else:
        idx = torch.randint(-1, vocab, (rows, 6), generator=g, device="cuda")
        idx[::7] = -1
        args = (torch.randn(rows, 6, generator=g, device="cuda"), idx)
    return h, w, args, torch.rand(rows, generator=g, device="cuda")


def loss_of(kind, h, w, args):
    from b200gemm import vocab_loss
    f = vocab_loss.linear_cross_entropy if kind == "ce" else vocab_loss.linear_distillation
    return f(h, w, *args, reduction="none")


def gradients(kind, h, w, args, up, want_h=True, want_w=True):
    h, w = h.detach().requires_grad_(want_h), w.detach().requires_grad_(want_w)
    return torch.autograd.grad(loss_of(kind, h, w, args), [t for t in (h, w) if t.requires_grad], up)


@pytest.mark.parametrize("kind", ["ce", "kd"])
@pytest.mark.parametrize("pin", [False, True])
@pytest.mark.parametrize("wants", [(True, True), (True, False), (False, True)])
def test_saved_on_the_host(kind, pin, wants):
    h, w, args, up = inputs(kind)
    want = gradients(kind, h, w, args, up, *wants)
    with torch.autograd.graph.save_on_cpu(pin_memory=pin):
        got = gradients(kind, h, w, args, up, *wants)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(x.isfinite().all() for x in got)


def wider(t):
    out = torch.full((t.shape[0], t.shape[1] + 40), math.nan, dtype=t.dtype, device=t.device)[:, 32:32 + t.shape[1]]
    return out.copy_(t)


def odd_pitch(t):
    return torch.full((t.shape[0], t.shape[1] + 3), math.nan, dtype=t.dtype, device=t.device)[:, :t.shape[1]].copy_(t)


def odd_start(t):
    flat = torch.full((t.numel() + 1,), math.nan, dtype=t.dtype, device=t.device)
    return flat[1:].view(t.shape).copy_(t)


def by_columns(t):
    return t.t().contiguous().t()


def spread(t):
    """Every second element of a longer one, in any number of dimensions."""
    return torch.empty(*t.shape, 2, dtype=t.dtype, device=t.device)[..., 0].copy_(t)


@pytest.mark.parametrize("kind,dtype", [("ce", BF16), ("kd", FP16)])
@pytest.mark.parametrize("layout", [wider, odd_pitch, odd_start, by_columns, spread])
@pytest.mark.parametrize("pitched", [True, False])
def test_saved_in_another_layout(kind, dtype, layout, pitched):
    h, w, args, up = inputs(kind, dtype=dtype, pitched=pitched)
    want = gradients(kind, h, w, args, up)

    def unpack(t):
        return layout(t) if t.dim() == 2 and t.dtype == dtype else (spread(t) if t.dim() else t)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        got = gradients(kind, h, w, args, up)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("kind", ["ce", "kd"])
@pytest.mark.parametrize("change", [lambda t: t[:1], lambda t: t.double(), lambda t: t.cpu(), lambda t: t[..., :-1]])
@pytest.mark.parametrize("which", range(5))
def test_saved_as_something_else_is_refused(kind, change, which):
    h, w, args, up = inputs(kind, rows=9)
    seen = []

    def unpack(t):
        seen.append(t)
        return change(t) if len(seen) == which + 1 else t
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        if kind == "ce" and which == 4:
            return  # a token for each row: four tensors are saved
        with pytest.raises(RuntimeError, match="came back"):
            gradients(kind, h, w, args, up)


@pytest.mark.parametrize("kind", ["ce", "kd"])
def test_checkpointed(kind):
    from torch.utils.checkpoint import checkpoint
    h, w, args, up = inputs(kind)
    want = gradients(kind, h, w, args, up)
    hg, wg = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = checkpoint(lambda a, b: loss_of(kind, a, b, args), hg, wg, use_reentrant=False)
    got = torch.autograd.grad(loss, (hg, wg), up)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
