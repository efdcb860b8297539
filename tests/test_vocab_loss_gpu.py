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


@pytest.mark.parametrize("rows,hidden,ignored,reduction", [(4097, 64, 1 / 4097, "mean"), (8192, 64, 0.0, "none"),
                                                           (9001, 72, 0.4, "none"), (12291, 72, 0.0, "sum"),
                                                           (4096, 136, 0.999, "none"), (9001, 64, 1.0, "mean")])
def test_many_rows_left_out(rows, hidden, ignored, reduction):
    """Rows beyond one step of their numbering (4096), one of them or nearly all left out."""
    ce(rows, 300, hidden, BF16 if rows % 2 else FP16, reduction, ignored, seed=rows)


@pytest.mark.parametrize("rows,vocab,top", [(1, 512 * 64, 0), (1, 512 * 64 + 1, 0), (8, 32000, 0), (26, 718, 0),
                                            (512, 500, 0), (513, 500, 0), (33, 5000, 0), (4000, 60, 0), (4097, 60, 0),
                                            (16, 300, 256), (17, 300, 256), (320, 400, 12), (70, 3000, 3)])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_merged_by_the_last_block(rows, vocab, top, reduction):
    """Both sides of the rule, and every number of lanes per row."""
    if top:
        kd(rows, vocab, 72, top, reduction=reduction)
    else:
        ce(rows, vocab, 72, FP16, reduction, 0.2, seed=rows)


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


def test_distillation_vanishing_probabilities():
    """Teacher logits hundreds apart: entries of probability 0 are still part of the student's softmax."""
    def change(logits, idx):
        logits[:, 1::2] -= 200.0
    kd(90, 400, 64, 12, change=change)
    kd(90, 400, 1024, 12, change=change)


def test_distillation_minus_infinity_is_padding():
    def change(logits, idx):
        logits[::2, ::3] = -math.inf
        logits[5] = -math.inf
    loss, dh, _ = kd(60, 300, 64, 9, reduction="none", change=change)
    assert loss[5] == 0 and not dh[5].any()


# --------------------------------------------------------------------------
# Every tile shape and split that the host can choose
# --------------------------------------------------------------------------
@pytest.mark.parametrize("rows,vocab,hidden,want", [
    (40, 600, 72, dict(cta_group=1, tile_n=128)),                      # one row block, few columns
    (100, 38000, 72, dict(cta_group=1, tile_n=256)),
    (250, 18000, 72, dict(cta_group=2, tile_n=256)),
    (90, 700, 1096, dict(cta_group=1, tile_n=128)),                    # statistics over several units
    (120, 37801, 520, dict(cta_group=1, tile_n=256)),
    (1000, 9000, 584, dict(cta_group=2, tile_n=256)),
    (3000, 300, 136, dict(tile_n=128)),                                # dW in runs over the rows
])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_cross_entropy_tile_shapes(rows, vocab, hidden, want, dtype):
    from b200gemm import vocab_loss
    p = vocab_loss.policy(rows, vocab, hidden)
    assert {k: p[k] for k in want} == want, p
    ce(rows, vocab, hidden, dtype, reduction="none", ignored=0.2, seed=3)


def test_weight_gradient_in_runs():
    from b200gemm import vocab_loss
    p = vocab_loss.policy(5000, 300, 64)
    assert p["splits_weight"] > 1 and p["splits_hidden"] >= 1
    ce(5000, 300, 64, reduction="sum")
    # So few rows with a loss that most runs have none.
    ce(5000, 300, 64, reduction="sum", ignored=0.995)


@pytest.mark.parametrize("rows,vocab,dtype", [(4096, 28990, BF16), (4090, 56976, FP16)])
def test_weight_gradient_two_blocks_per_tile(rows, vocab, dtype):
    """Tiles of 512 rows of dW, the last of them with one block or less; one piece and two."""
    from b200gemm import vocab_loss
    assert vocab_loss.policy(rows, vocab, 264)["tile_m_weight"] == 512
    ce(rows, vocab, 264, dtype, reduction="sum")
    ce(rows, vocab, 264, dtype, reduction="sum", ignored=0.97)


def test_hidden_gradient_in_runs():
    from b200gemm import vocab_loss
    assert vocab_loss.policy(130, 20000, 64)["splits_hidden"] > 1
    ce(130, 20000, 64, reduction="sum", ignored=0.5)


# --------------------------------------------------------------------------
# How a program calls them
# --------------------------------------------------------------------------
def test_same_call_same_bits():
    a = ce(700, 5000, 264, ignored=0.3, reduction="none", seed=5)
    b = ce(700, 5000, 264, ignored=0.3, reduction="none", seed=5)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_strides_and_leading_dimensions():
    from b200gemm import vocab_loss
    g, h, w = make(6 * 35, 901, 80)
    wide_h, wide_w = torch.full((6, 35, 104), math.nan, dtype=BF16, device="cuda"), torch.full((901, 96), math.nan, dtype=BF16, device="cuda")
    wide_h[..., 16:96] = h.reshape(6, 35, 80)
    wide_w[:, 8:88] = w
    target = torch.randint(0, 901, (35, 6), generator=g, device="cuda").t()  # not contiguous
    up = torch.randn(6, 35, generator=g, device="cuda")
    hs, ws = wide_h[..., 16:96].detach().requires_grad_(), wide_w[:, 8:88].detach().requires_grad_()
    loss = vocab_loss.linear_cross_entropy(hs, ws, target, reduction="none")
    assert loss.shape == (6, 35)
    dh, dw = torch.autograd.grad(loss, (hs, ws), up)
    plain = run(vocab_loss.linear_cross_entropy, h, w, (target.reshape(-1).contiguous(),), up.reshape(-1), reduction="none")
    assert torch.equal(loss.detach().reshape(-1), plain[0])
    assert torch.equal(dh.reshape(-1, 80), plain[1]) and torch.equal(dw, plain[2])


def test_single_row_without_leading_dimension():
    from b200gemm import vocab_loss
    g, h, w = make(1, 500, 64)
    t = torch.tensor(7, device="cuda")
    a = vocab_loss.linear_cross_entropy(h[0], w, t, reduction="none")
    b = vocab_loss.linear_cross_entropy(h, w, t[None], reduction="none")
    assert a.shape == () and torch.equal(a, b[0])


def test_one_gradient_at_a_time():
    from b200gemm import vocab_loss
    g, h, w = make(300, 1000, 136)
    t = torch.randint(0, 1000, (300,), generator=g, device="cuda")
    both = run(vocab_loss.linear_cross_entropy, h, w, (t,), torch.ones((), device="cuda"))
    hg, wg = h.detach().requires_grad_(), w.detach().requires_grad_()
    vocab_loss.linear_cross_entropy(hg, w, t).backward()
    assert torch.equal(hg.grad, both[1])
    vocab_loss.linear_cross_entropy(h, wg, t).backward()
    assert torch.equal(wg.grad, both[2])
    loss = vocab_loss.linear_cross_entropy(hg, wg, t)
    assert torch.equal(torch.autograd.grad(loss, wg, retain_graph=True)[0], both[2])
    assert torch.equal(torch.autograd.grad(loss, hg, retain_graph=True)[0], both[1])  # twice on one graph
    with torch.no_grad():
        assert torch.equal(vocab_loss.linear_cross_entropy(hg, wg, t), both[0])


def test_refused_layouts():
    from b200gemm import vocab_loss
    g, h, w = make(6, 100, 64)
    t = torch.zeros(6, dtype=torch.long, device="cuda")
    flat = torch.zeros(7 * 80, dtype=BF16, device="cuda")
    for bad in (flat[4:4 + 6 * 64].view(6, 64), flat.as_strided((6, 64), (68, 1)), h[:1].expand(6, 64)):
        with pytest.raises(ValueError):
            vocab_loss.linear_cross_entropy(bad, w, t)
    wide = torch.zeros(100, 80, dtype=BF16, device="cuda")
    for bad in (wide[:, 4:68], wide.view(-1)[: 99 * 76 + 64].as_strided((100, 64), (76, 1))):
        with pytest.raises(ValueError):
            vocab_loss.linear_cross_entropy(h, bad, t)
    with pytest.raises(ValueError, match="target must be on"):
        vocab_loss.linear_cross_entropy(h, w, t.cpu())
    with pytest.raises(ValueError, match="weight must be on"):
        vocab_loss.linear_cross_entropy(h, w.cpu(), t)


def test_first_call_of_a_process_may_be_captured():
    import subprocess
    import sys
    from pathlib import Path
    root = Path(__file__).resolve().parents[1]
    code = """
import sys; sys.path.insert(0, %r)
import torch
from b200gemm import vocab_loss
h = torch.randn(300, 64, device="cuda").bfloat16().requires_grad_()
w = torch.randn(900, 64, device="cuda").bfloat16().requires_grad_()
t = torch.randint(0, 900, (300,), device="cuda")
up = torch.ones((), device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    loss = vocab_loss.linear_cross_entropy(h, w, t)
    grads = torch.autograd.grad(loss, (h, w), up)
graph.replay()
want = vocab_loss.linear_cross_entropy(h, w, t)
assert torch.equal(loss, want) and all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(want, (h, w), up)))
print("same")
""" % str(root / "gb300-gemm-anatomy_b200")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_differentiable_once():
    from b200gemm import vocab_loss
    g, h, w = make(10, 100, 64)
    h.requires_grad_()
    loss = vocab_loss.linear_cross_entropy(h, w, torch.zeros(10, dtype=torch.long, device="cuda"))
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(loss, h, create_graph=True)


def test_no_rows():
    from b200gemm import vocab_loss
    for reduction in ("none", "mean", "sum"):
        h = torch.empty(0, 64, dtype=BF16, device="cuda", requires_grad=True)
        w = torch.ones(30, 64, dtype=BF16, device="cuda", requires_grad=True)
        loss = vocab_loss.linear_cross_entropy(h, w, torch.empty(0, dtype=torch.long, device="cuda"), reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ()) and not loss.any()
        dh, dw = torch.autograd.grad(loss.sum(), (h, w))
        assert dh.shape == h.shape and dw.shape == w.shape and not dw.any()
    h = torch.empty(3, 0, 64, dtype=BF16, device="cuda")
    loss = vocab_loss.linear_distillation(h, w, torch.empty(3, 0, 5, device="cuda"),
                                          torch.empty(3, 0, 5, dtype=torch.int32, device="cuda"), reduction="none")
    assert loss.shape == (3, 0)


def test_loss_alone_is_the_loss_of_a_step():
    """Without a backward pass another path allocates; forward mode is refused."""
    from b200gemm import vocab_loss
    g, h, w = make(301, 700, 72)
    t = torch.randint(0, 700, (301,), generator=g, device="cuda")
    q = torch.randn(301, 5, generator=g, device="cuda")
    idx = torch.randint(-1, 700, (301, 5), generator=g, device="cuda")
    for fn, args in ((vocab_loss.linear_cross_entropy, (t,)), (vocab_loss.linear_distillation, (q, idx))):
        for reduction in ("none", "mean", "sum"):
            step = fn(h.detach().requires_grad_(), w, *args, reduction=reduction)
            alone = fn(h, w, *args, reduction=reduction)
            with torch.no_grad():
                quiet = fn(h.detach().requires_grad_(), w, *args, reduction=reduction)
            with torch.inference_mode():
                inferred = fn(h, w, *args, reduction=reduction)
            assert step.requires_grad and not alone.requires_grad and not quiet.requires_grad
            assert torch.equal(step, alone) and torch.equal(step, quiet) and torch.equal(step, inferred)
        with pytest.raises(RuntimeError):
            torch.func.jvp(lambda x: fn(x, w, *args), (h,), (h,))


@pytest.mark.parametrize("rows,vocab,hidden,top", [(512, 512, 512, 0), (130, 5000, 72, 0), (4096, 40007, 64, 0),
                                                   (700, 3000, 1000, 9), (8, 700, 64, 3)])
def test_overlapping_kernels_give_the_same_bits(rows, vocab, hidden, top):
    """Steps close behind one another, eager and as a graph that is replayed: the kernels of a step
    start while others end, on a workspace that the step before has used."""
    from b200gemm import vocab_loss
    g, h, w = make(rows, vocab, hidden)
    up = torch.rand(rows, generator=g, device="cuda")
    if top:
        fn = vocab_loss.linear_distillation
        args = (torch.randn(rows, top, generator=g, device="cuda"),
                torch.randint(-1, vocab, (rows, top), generator=g, device="cuda"))
    else:
        fn = vocab_loss.linear_cross_entropy
        args = (torch.randint(0, vocab, (rows,), generator=g, device="cuda"),)
        args[0][::5] = IGNORE
    first = run(fn, h, w, args, up, reduction="none")
    torch.cuda.synchronize()
    differ = torch.zeros((), dtype=torch.bool, device="cuda")
    for _ in range(30):
        for x, y in zip(run(fn, h, w, args, up, reduction="none"), first):
            differ |= (x != y).any()
    assert not differ
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(fn, h, w, args, up, reduction="none")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = run(fn, h, w, args, up, reduction="none")
    for _ in range(30):
        graph.replay()
        graph.replay()
        for x, y in zip(out, first):
            differ |= (x != y).any()
    assert not differ


def test_two_streams_at_once():
    from b200gemm import vocab_loss
    jobs = []
    for seed, (rows, vocab, hidden) in enumerate([(900, 20000, 512), (64, 30000, 1024), (2000, 3000, 256)]):
        g, h, w = make(rows, vocab, hidden, seed=seed)
        t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        jobs.append((h, w, t))
    one = torch.ones((), device="cuda")
    want = [run(vocab_loss.linear_cross_entropy, h, w, (t,), one) for h, w, t in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for (h, w, t), s in zip(jobs, streams):
            with torch.cuda.stream(s):
                got.append(run(vocab_loss.linear_cross_entropy, h, w, (t,), one))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_and_replayed():
    """Two graphs with their own inputs, replayed in turn and on new data."""
    from b200gemm import vocab_loss
    graphs = []
    for seed, (rows, vocab, hidden) in enumerate([(300, 2000, 128), (40, 5000, 64)]):
        g, h, w = make(rows, vocab, hidden, seed=seed)
        t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        one = torch.ones((), device="cuda")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run(vocab_loss.linear_cross_entropy, h, w, (t,), one)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(vocab_loss.linear_cross_entropy, h, w, (t,), one)
        graphs.append((graph, h, w, t, one, out))
    for step in range(3):
        for graph, h, w, t, one, out in graphs:
            h.copy_(torch.randn_like(h))
            t.copy_(torch.randint_like(t, w.shape[0]))
            t[::3] = IGNORE
            one.fill_(step + 0.5)
        for graph, *_ in graphs:
            graph.replay()
        for graph, h, w, t, one, out in graphs:
            want = run(vocab_loss.linear_cross_entropy, h, w, (t,), one)
            assert all(torch.equal(a, b) for a, b in zip(out, want))


# --------------------------------------------------------------------------
# Values
# --------------------------------------------------------------------------
def test_target_outside_the_vocabulary():
    """The row's loss is NaN, and the gradients that it reaches; other rows' are not."""
    from b200gemm import vocab_loss
    g, h, w = make(9, 50, 64)
    t = torch.arange(9, device="cuda")
    t[2], t[5] = 50, -7
    loss, dh, dw = run(vocab_loss.linear_cross_entropy, h, w, (t,), torch.ones(9, device="cuda"), reduction="none")
    bad = torch.zeros(9, dtype=torch.bool, device="cuda")
    bad[[2, 5]] = True
    assert torch.equal(loss.isnan(), bad) and torch.equal(dh.isnan().all(1), bad) and torch.equal(dh.isnan().any(1), bad)
    assert dw.isnan().all()
    idx = torch.randint(0, 50, (9, 4), generator=g, device="cuda")
    idx[2, 1] = 50
    loss = vocab_loss.linear_distillation(h, w, torch.zeros(9, 4, device="cuda"), idx, reduction="none")
    bad[5] = False
    assert torch.equal(loss.isnan(), bad)
    assert vocab_loss.linear_cross_entropy(h, w, t).isnan()


def test_upstream_zeros_and_scales():
    from b200gemm import vocab_loss
    for dtype in (BF16, FP16):
        g, h, w = make(140, 400, 64, dtype)
        t = torch.randint(0, 400, (140,), generator=g, device="cuda")
        up = torch.zeros(140, device="cuda")
        _, dh, dw = run(vocab_loss.linear_cross_entropy, h, w, (t,), up, reduction="none")
        assert not dh.any() and not dw.any()
        # Loss scales far from 1, as mixed precision uses them, and weights 2^20 apart.
        up = torch.exp2(torch.randint(-10, 11, (140,), generator=g, device="cuda").float()) * (1 if dtype == FP16 else 2.0 ** 40)
        kept, idx, q = ref.targets_of(t, IGNORE)
        check_all(run(vocab_loss.linear_cross_entropy, h, w, (t,), up, reduction="none"),
                  ref.reference(h, w, kept, idx, q, 1.0, "none", up))


def test_upstream_infinities_stay_in_their_rows():
    from b200gemm import vocab_loss
    g, h, w = make(140, 400, 64)
    t = torch.randint(0, 400, (140,), generator=g, device="cuda")
    up = torch.ones(140, device="cuda")
    _, want, _ = run(vocab_loss.linear_cross_entropy, h, w, (t,), up, reduction="none")
    up[7], up[130] = math.inf, math.nan
    _, dh, dw = run(vocab_loss.linear_cross_entropy, h, w, (t,), up, reduction="none")
    other = torch.ones(140, dtype=torch.bool, device="cuda")
    other[[7, 130]] = False
    assert torch.equal(dh[other], want[other]) and not dh[~other].isfinite().any()
    assert not dw.isfinite().any()


@pytest.mark.parametrize("std", [0.0, 3.0])
def test_flat_and_peaked_logits(std):
    """All logits equal; logits hundreds apart, where all but one probability vanish."""
    from b200gemm import vocab_loss
    g, h, w = make(200, 700, 512, seed=1, std=std or 1.0)
    if not std:
        w.zero_()
    t = torch.randint(0, 700, (200,), generator=g, device="cuda")
    t[::2] = (h @ w.t()).argmax(1)[::2]
    up = torch.rand((), device="cuda") + 0.5
    kept, idx, q = ref.targets_of(t, IGNORE)
    check_all(run(vocab_loss.linear_cross_entropy, h, w, (t,), up), ref.reference(h, w, kept, idx, q, 1.0, "mean", up))


@pytest.mark.parametrize("hidden", [64, 1024])
@pytest.mark.parametrize("shift", [-300.0, 300.0])
@pytest.mark.parametrize("vocab", [1, 100, 1000, 5000])
def test_logits_far_from_zero(hidden, shift, vocab):
    """All logits near the same large number: exp of it, or of its negative, is beyond 32 bits."""
    from b200gemm import vocab_loss
    g, h, w = make(150, vocab, hidden)
    h[:, 0] = 20.0
    w[:, 0] = shift / 20
    t = torch.randint(0, vocab, (150,), generator=g, device="cuda")
    up = torch.rand(150, generator=g, device="cuda")
    kept, idx, q = ref.targets_of(t, IGNORE)
    check_all(run(vocab_loss.linear_cross_entropy, h, w, (t,), up, reduction="none"),
              ref.reference(h, w, kept, idx, q, 1.0, "none", up))


@pytest.mark.parametrize("hidden", [64, 1024])
def test_infinite_logits(hidden):
    """Tokens that the projection masks with -inf have no part in the loss."""
    from b200gemm import vocab_loss
    g, h, w = make(70, 600, hidden)
    h = h.abs().clamp(min=0.01)
    w[100:400] = -math.inf
    t = torch.randint(0, 100, (70,), generator=g, device="cuda")
    loss = vocab_loss.linear_cross_entropy(h, w, t, reduction="none")
    live = torch.cat([w[:100], w[400:]])
    kept, idx, q = ref.targets_of(t, IGNORE)
    want = ref.reference(h, live, kept, idx, q, 1.0, "none", torch.ones(70, device="cuda"))
    ref.check("loss", loss, want[0], want[1])
    t[3] = 200
    assert vocab_loss.linear_cross_entropy(h, w, t, reduction="none")[3] == math.inf


def test_gradients_against_differences():
    """Central differences of the loss itself along a direction. hidden +- step * u is exact in bf16; the
    remainder is the third cumulant of the logits' change over 6, at most R^3 / (36 sqrt(3)) a row for a
    change of range R; the losses are off by 2^-19 each, the inner product by half a step of its terms."""
    from b200gemm import vocab_loss
    g = torch.Generator(device="cuda").manual_seed(11)
    rows, vocab, hidden, step = 50, 300, 64, 2.0 ** -4
    h = (torch.randint(-16, 17, (rows, hidden), generator=g, device="cuda") / 16).to(BF16)
    w = (torch.randn(vocab, hidden, generator=g, device="cuda") / 16).to(BF16)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    logits, index = torch.randn(rows, 5, generator=g, device="cuda"), torch.randint(0, vocab, (rows, 5), generator=g, device="cuda")
    u = torch.randint(0, 2, (rows, hidden), generator=g, device="cuda") * 2.0 - 1
    change = step * (u.double() @ w.double().t())
    spread = change.max(1).values - change.min(1).values
    for tau, f in ((1.0, lambda x: vocab_loss.linear_cross_entropy(x, w, t, reduction="none")),
                   (1.5, lambda x: vocab_loss.linear_distillation(x, w, logits, index, temperature=1.5, reduction="none"))):
        x = h.detach().requires_grad_()
        dh, = torch.autograd.grad(f(x).sum(), x)
        plus, minus = f((h + step * u).to(BF16)), f((h - step * u).to(BF16))
        got = step * (dh.double() * u).sum(1)
        diff = (plus.double() - minus.double()) / 2
        bound = (tau ** 2 * (spread / tau) ** 3 / (36 * math.sqrt(3)) + 2.0 ** -19 * (plus.abs() + minus.abs() + 1)
                 + step * (2.0 ** -8 + 2.0 ** -8) * dh.double().abs().sum(1) + step * 2.0 ** -8 * tau * 2 * w.double().abs().max(0).values.sum())
        assert bool(((got - diff).abs() <= bound).all())
        # The bound is no empty one: it is below the difference itself in most rows.
        assert float((diff.abs() > bound).double().mean()) > 0.5


def test_gradients_of_confident_rows():
    """Where the model is sure and right, p - 1 is small: its own precision counts, not that of 1 or of lse.
    log p is a difference from the largest logit: off by 2^-21 (a sum of up to 256 terms, its logarithm) and by
    how far the logits are off (dz, see the reference), the target's own cancelling but for the share 1 - p."""
    from b200gemm import vocab_loss
    rows, vocab, hidden = 64, 500, 2048
    g, h, w = make(rows, vocab, hidden, seed=4, std=0.02)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    h = (h + w[t].float() * torch.linspace(14, 20, rows, device="cuda")[:, None]).to(BF16)
    z = h.double() @ w.double().t()
    p = torch.softmax(z, 1)
    G = p.clone()
    G.scatter_(1, t[:, None], 0.0)
    miss = G.sum(1, keepdim=True)  # 1 - p
    assert float(miss.min()) < 1e-3 and float(miss.max()) > 1e-2
    up = (1 / miss[:, 0]).float()  # each row's gradient at one size
    loss, dh, _ = run(vocab_loss.linear_cross_entropy, h, w, (t,), up, reduction="none")
    dz = (hidden / 16 + 16) * 2.0 ** -23 * (h.double().abs() @ w.double().abs().t()).max(1, keepdim=True).values
    off = 2.0 ** -21 + 2 * dz * miss
    assert bool(((loss.double() + torch.log1p(-miss[:, 0])).abs() <= off[:, 0]).all())
    E = G * (2.0 ** -8 + 2 * dz + 2.0 ** -18)
    E.scatter_(1, t[:, None], 2.0 ** -8 * miss + off)
    G.scatter_(1, t[:, None], -miss)
    want = (G / miss) @ w.double()
    bound = (E / miss) @ w.double().abs() + 2.0 ** -8 * want.abs() + 2.0 ** -16 * (G / miss).abs() @ w.double().abs()
    assert bool(((dh.double() - want).abs() <= bound).all())


def test_many_rows():
    """More rows than a grid's second dimension, and than a pass of the row numbering."""
    ce(70001, 256, 64, ignored=0.4, reduction="none")


def test_weight_beyond_32_bit_offsets():
    """V x D above 2^31 elements: the last rows of the projection are read and written."""
    from b200gemm import vocab_loss
    V, D, T = 262400, 8192, 3
    assert V * D > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.empty(V, D, dtype=BF16, device="cuda")
    for v in range(0, V, 16400):
        w[v:v + 16400] = torch.randn(16400, D, generator=g, device="cuda") * 0.02
    h = torch.randn(T, D, generator=g, device="cuda").to(BF16)
    t = torch.tensor([0, V - 1, V // 2], device="cuda")
    loss, dh, dw = run(vocab_loss.linear_cross_entropy, h, w, (t,), torch.ones(T, device="cuda"), reduction="none")
    z = torch.cat([h.double() @ w[v:v + 16400].double().t() for v in range(0, V, 16400)], 1)
    p = torch.softmax(z, 1)
    dz = (D / 16 + 16) * 2.0 ** -23 * float((h.double().abs() @ w[:16400].double().abs().t()).max()) * 1.2
    want = torch.logsumexp(z, 1) - z.gather(1, t[:, None])[:, 0]
    assert bool(((loss.double() - want).abs() <= 2 * dz + 2.0 ** -18 + 2.0 ** -20 * want).all())
    G = p.scatter_add(1, t[:, None], -torch.ones(T, 1, dtype=torch.float64, device="cuda"))
    for rows in (slice(0, 40), slice(V // 2 - 20, V // 2 + 20), slice(V - 40, V)):
        exact = G[:, rows].t() @ h.double()
        bound = (2.0 ** -8 + 2.0 ** -8 + 2 * dz + 2.0 ** -17) * (G[:, rows].abs().t() @ h.double().abs()) + 2.0 ** -17
        assert bool(((dw[rows].double() - exact).abs() <= bound).all())
    assert bool(dw.isfinite().all()) and bool(dh.isfinite().all())


# --------------------------------------------------------------------------
# Together
# --------------------------------------------------------------------------
def test_losses_of_one_step_together():
    """A distillation step: both losses on the same hidden states and projection, gradients added by torch,
    next to the framework's GEMM, which gives the same logits."""
    from b200gemm import gemm, vocab_loss
    rows, vocab, hidden, top = 260, 1200, 128, 12
    g, h, w = make(rows, vocab, hidden, seed=2)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    t[-20:] = IGNORE
    logits = torch.randn(rows, top, generator=g, device="cuda")
    index = torch.randint(0, vocab, (rows, top), generator=g, device="cuda")
    index[-20:] = -1
    hg, wg = h.detach().requires_grad_(), w.detach().requires_grad_()
    a = vocab_loss.linear_cross_entropy(hg, wg, t)
    b = vocab_loss.linear_distillation(hg, wg, logits, index, temperature=2.0)
    (0.25 * a + 0.75 * b).backward()
    ra = ref.reference(h, w, *ref.targets_of(t, IGNORE), 1.0, "mean", torch.tensor(0.25, device="cuda"))
    rb = ref.reference(h, w, *ref.teacher_of(logits, index, 2.0), 2.0, "mean", torch.tensor(0.75, device="cuda"))
    ref.check("ce", a.detach(), ra[0], ra[1])
    ref.check("kd", b.detach(), rb[0], rb[1])
    for i, got in ((2, hg.grad), (4, wg.grad)):
        want = ra[i] + rb[i]
        ref.check("gradient", got, want, ra[i + 1] + rb[i + 1] + 2.0 ** -8 * (ra[i].abs() + rb[i].abs() + ra[i + 1] + rb[i + 1]))
    z = gemm.gemm(h, w, out_dtype=torch.float32).double()
    loss = (torch.logsumexp(z, 1) - z.gather(1, t.clamp(min=0)[:, None])[:, 0])[:-20].mean()
    assert abs(float(loss) - float(a.detach())) <= 2 * float(ra[1])


@pytest.mark.parametrize("args", [["--loss", "ce", "--ignored", "0.25"], ["--loss", "kd", "--top", "9", "--temperature", "2"],
                                  ["--loss", "ce", "--dtype", "fp16", "--way", "forward"]])
def test_command(args, capsys):
    from b200gemm.cli import vocab_loss as cli
    assert cli.main(args + ["--rows", "300", "--vocab", "5000", "--hidden", "256", "--iterations", "2", "--warmup", "1"]) == 0
    lines = capsys.readouterr().out.strip().splitlines()
    assert lines[0].startswith("loss,way,") and len(lines) == (2 if "--way" in args else 3)
    for line in lines[1:]:
        r = dict(zip(lines[0].split(","), line.split(",")))
        assert float(r["ms"]) > 0 and int(r["rows_with_loss"]) == (225 if "0.25" in args else 300)
