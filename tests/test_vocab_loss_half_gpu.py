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


# --------------------------------------------------------------------------
# Weights of rows
# --------------------------------------------------------------------------
def weights(g, rows, low, high):
    """Of either sign, powers of two apart and no powers of two themselves."""
    e = torch.randint(low, high + 1, (rows,), generator=g, device="cuda").float()
    return torch.exp2(e) * (1 + torch.rand(rows, generator=g, device="cuda")) * (
        1 - 2 * torch.randint(0, 2, (rows,), generator=g, device="cuda"))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("kind,tau", [("ce", 1.0), ("kd", 0.5)])
@pytest.mark.parametrize("vocab,common", [(50001, 0.0), (128256, 1.0), (700, 0.0)])
def test_weights_far_apart(dtype, kind, tau, vocab, common):
    """Rows that weigh 2^20 less than others keep their own gradients' precision."""
    g, h, w = make(40, vocab, 64, dtype, seed=vocab, common=common)
    args = targets(kind, g, 40, vocab)
    up = weights(g, 40, -8, 12)
    got = step(kind, h, w, args, up, tau=tau)
    dh, bh, dw, bw = check(kind, h, w, args, up, got, tau)
    assert not bool((dh.abs() <= bh).all(1).any()) and not bool((dw.abs() <= bw).all(1).any())


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("kind", ["ce", "kd"])
def test_a_row_does_not_see_other_weights(dtype, kind):
    g, h, w = make(30, 32003, 72, dtype, common=1.0)
    args = targets(kind, g, 30, 32003)
    up = weights(g, 30, -2, 2)
    _, dh, dw = step(kind, h, w, args, up)
    for row, factor in ((3, 2.0 ** 12), (17, 3.0e5), (29, 0.0), (0, math.inf), (11, math.nan)):
        other = up.clone()
        other[row] *= factor
        _, changed, cw = step(kind, h, w, args, other)
        rest = torch.arange(30, device="cuda") != row
        assert torch.equal(changed[rest], dh[rest])
        if math.isfinite(factor):
            want, bound, *_ = rows_ref.gradients(h, w, *distribution(kind, args, 1.0), 1.0, other)
            inside = want[row].abs() + bound[row] < torch.finfo(dtype).max
            assert bool(((changed[row].double() - want[row]).abs() <= bound[row])[inside].all()) and bool(inside.any())
        else:
            assert not changed[row].isfinite().any() and not cw.isfinite().any()
        if factor == 0.0:
            assert not changed[row].any()
    # All weights times a power of two: everything times that.
    _, dh4, dw4 = step(kind, h, w, args, up * 4)
    if dtype == BF16:
        assert torch.equal(dh4, dh * 4) and torch.equal(dw4, dw * 4)
    else:  # but for results below 2^-14
        assert bool(((dh4 / 4 - dh).abs() <= 2.0 ** -24).all()) and bool(((dw4 / 4 - dw).abs() <= 2.0 ** -24).all())


@pytest.mark.parametrize("rows,vocab,hidden,ignored", [
    (9, 300, 8, 0.0), (130, 20000, 72, 0.3), (700, 3000, 1000, 0.5), (5000, 300, 64, 0.2), (5000, 300, 64, 0.997),
    (4090, 56976, 264, 0.9), (4096, 40007, 64, 0.95), (300, 500, 128, 0.0)])
def test_weights_in_every_form_of_the_products(rows, vocab, hidden, ignored):
    """One piece and several, dW whole, in tiles of two blocks and in runs; rows left out, and what they hold."""
    g, h, w = make(rows, vocab, hidden, FP16, seed=rows, spread=2.0)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    drop = torch.randperm(rows, generator=g, device="cuda")[:round(rows * ignored)]
    t[drop] = -100
    h[drop[::2]], h[drop[1::2]] = math.nan, math.inf
    up = weights(g, rows, -10, 6)
    up[drop[::3]] = math.inf  # nobody's weight
    got = step("ce", h, w, (t,), up)
    check("ce", h, w, (t,), up, got)
    assert not got[1][drop].any()
    again = step("ce", h, w, (t,), up)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("scales", [(1.0, 6e4), (1e-4, 1.0), (2.0 ** -24, 2.0 ** -20), (100.0, 1e-3)])
def test_weights_and_the_size_of_hidden(scales):
    """Rows of hidden near both ends of half precision's range, the light rows larger or smaller than the heavy."""
    g, h, w = make(32, 600, 64, FP16)
    h = torch.rand(32, 64, generator=g, device="cuda") - 0.5
    h[:16] *= scales[0]
    h[16:] *= scales[1]
    h = h.to(FP16)
    w = (w.float() * min(1 / max(scales), 1024.0)).to(FP16)
    args = targets("ce", g, 32, 600)
    up = weights(g, 32, -5, -3)  # d_weight stays below 65504
    up[:16] *= 2.0 ** -9
    check("ce", h, w, args, up, step("ce", h, w, args, up))


def test_weights_of_nothing():
    for dtype in (BF16, FP16):
        g, h, w = make(20, 500, 64, dtype)
        args = targets("ce", g, 20, 500)
        _, dh, dw = step("ce", h, w, args, torch.zeros(20, device="cuda"))
        assert not dh.any() and not dw.any()
        up = torch.zeros(20, device="cuda")
        up[4] = 3.0
        _, dh, dw = step("ce", h, w, args, up)
        check("ce", h, w, args, up, (None, dh, dw))
        assert not dh[:4].any() and not dh[5:].any()
        _, dh, dw = step("ce", h, w, (torch.full_like(args[0], -100),), torch.ones(20, device="cuda"))
        assert not dh.any() and not dw.any()


def test_weights_at_the_ends_of_their_range():
    """bf16 reaches as far as the weights do; half precision's results overflow or vanish, without a NaN."""
    g, h, w = make(20, 500, 64, BF16)
    args = targets("ce", g, 20, 500)
    base = weights(g, 20, 0, 3)
    _, dh, dw = step("ce", h, w, args, base)
    for scale in (2.0 ** 100, 2.0 ** -100):
        _, dh2, dw2 = step("ce", h, w, args, base * scale)
        assert torch.equal(dh2.float(), dh.float() * scale) and torch.equal(dw2.float(), dw.float() * scale)
    h, w = h.to(FP16), w.to(FP16)
    for scale in (2.0 ** 120, 2.0 ** -120, 2.0 ** -140):
        _, dh, dw = step("ce", h, w, args, base * scale)
        assert not dh.isnan().any() and not dw.isnan().any()
        assert bool(dh.any()) == (scale > 1) and bool(dw.any()) == (scale > 1)


def test_weights_without_one_of_the_gradients():
    from b200gemm import vocab_loss
    g, h, w = make(70, 3000, 136, FP16)
    args = targets("ce", g, 70, 3000)
    up = weights(g, 70, -6, 6)
    _, dh, dw = step("ce", h, w, args, up)
    hg, wg = h.detach().requires_grad_(), w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(vocab_loss.linear_cross_entropy(hg, w, *args, reduction="none"), hg, up)[0], dh)
    assert torch.equal(torch.autograd.grad(vocab_loss.linear_cross_entropy(h, wg, *args, reduction="none"), wg, up)[0], dw)


@pytest.mark.parametrize("rows,vocab,hidden", [(300, 2000, 128), (5000, 300, 64), (4096, 40007, 64)])
def test_weights_overlapping_and_replayed(rows, vocab, hidden):
    g, h, w = make(rows, vocab, hidden, FP16)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    t[::5] = -100
    up = weights(g, rows, -8, 8)
    first = step("ce", h, w, (t,), up)
    differ = torch.zeros((), dtype=torch.bool, device="cuda")
    for _ in range(20):
        for x, y in zip(step("ce", h, w, (t,), up), first):
            differ |= (x != y).any()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step("ce", h, w, (t,), up)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step("ce", h, w, (t,), up)
    for _ in range(20):
        graph.replay()
        for x, y in zip(out, first):
            differ |= (x != y).any()
    assert not differ
    up.mul_(2.0 ** -5)
    up[1] = 2.0 ** 11
    h[7].mul_(16.0)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, step("ce", h, w, (t,), up)))
