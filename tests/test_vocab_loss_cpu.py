"""Losses at the vocabulary projection without a GPU: refusals, the host's choices, the 64-bit reference."""
import ctypes
import math

import pytest
import torch

import vocab_loss_reference as ref
from b200gemm import _lib, vocab_loss

BF16, FP16 = torch.bfloat16, torch.float16


def operands(rows=4, vocab=32, hidden=16, dtype=BF16):
    return torch.zeros(rows, hidden, dtype=dtype), torch.zeros(vocab, hidden, dtype=dtype)


def longs(*shape):
    return torch.zeros(*shape, dtype=torch.long)


@pytest.mark.parametrize("change,match", [
    (dict(hidden=torch.zeros(4, 16)), "bfloat16 or float16"),
    (dict(weight=torch.zeros(32, 16, dtype=FP16)), "like hidden"),
    (dict(weight=torch.zeros(32, 24, dtype=BF16)), "do not match"),
    (dict(weight=torch.zeros(16, dtype=BF16)), "do not match"),
    (dict(weight=torch.zeros(0, 16, dtype=BF16)), "must be positive"),
    (dict(hidden=torch.zeros(4, 12, dtype=BF16), weight=torch.zeros(32, 12, dtype=BF16)), "multiple of 8"),
    (dict(hidden=torch.zeros(16, 4, dtype=BF16).t()), "contiguous rows"),
    (dict(weight=torch.zeros(16, 32, dtype=BF16).t()), "contiguous rows"),
    (dict(target=longs(5)), "expected"),
    (dict(target=longs(4, 1)), "expected"),
    (dict(target=torch.zeros(4)), "int32 or int64"),
    (dict(reduction="batchmean"), "reduction"),
    (dict(ignore_index=1.5), "integer"),
    (dict(ignore_index=2 ** 63), "64-bit"),
    (dict(), "CUDA device"),
])
def test_cross_entropy_refusals(change, match):
    h, w = operands()
    args = dict(hidden=h, weight=w, target=longs(4), reduction="mean", ignore_index=-100)
    args.update(change)
    with pytest.raises(ValueError, match=match):
        vocab_loss.linear_cross_entropy(args["hidden"], args["weight"], args["target"], reduction=args["reduction"],
                                        ignore_index=args["ignore_index"])


@pytest.mark.parametrize("change,match", [
    (dict(logits=torch.zeros(4, 3, dtype=torch.float64)), "float32"),
    (dict(index=torch.zeros(4, 3)), "int32 or int64"),
    (dict(index=longs(4, 2)), "x K"),
    (dict(logits=torch.zeros(4), index=longs(4)), "x K"),
    (dict(logits=torch.zeros(5, 3), index=longs(5, 3)), "x K"),
    (dict(logits=torch.zeros(4, 0), index=longs(4, 0)), "1 to 256"),
    (dict(logits=torch.zeros(4, 257), index=longs(4, 257)), "1 to 256"),
    (dict(logits=torch.zeros(4, 3, requires_grad=True)), "detach"),
    (dict(temperature=0.0), "temperature"),
    (dict(temperature=-1.0), "temperature"),
    (dict(temperature=1e-7), "temperature"),
    (dict(temperature=2e6), "temperature"),
    (dict(temperature=math.inf), "temperature"),
    (dict(temperature=math.nan), "temperature"),
    (dict(reduction="none "), "reduction"),
    (dict(), "CUDA device"),
])
def test_distillation_refusals(change, match):
    h, w = operands()
    args = dict(logits=torch.zeros(4, 3), index=longs(4, 3), temperature=1.0, reduction="mean")
    args.update(change)
    with pytest.raises(ValueError, match=match):
        vocab_loss.linear_distillation(h, w, args["logits"], args["index"], temperature=args["temperature"],
                                       reduction=args["reduction"])


def test_not_tensors():
    h, w = operands()
    with pytest.raises(TypeError, match="target"):
        vocab_loss.linear_cross_entropy(h, w, [0, 1, 2, 3])
    with pytest.raises(TypeError, match="hidden"):
        vocab_loss.linear_cross_entropy(None, w, longs(4))
    with pytest.raises(TypeError, match="teacher_logits"):
        vocab_loss.linear_distillation(h, w, None, longs(4, 3))


def desc(**change):
    fields = dict(rows=64, vocab=1000, hidden=128, ld_hidden=128, ld_weight=128, dtype=_lib.VL_BF16, top=0, index_bytes=8,
                  ld_index=0, ld_teacher=0, teacher_dtype=0, ignore_index=-100, reduction=_lib.VL_MEAN, temperature=1.0)
    fields.update(change)
    return _lib.VocabLossDesc(*(fields[n] for n, _ in _lib.VocabLossDesc._fields_))


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), _lib.ERR_INVALID_ARGUMENT), (dict(vocab=0), _lib.ERR_INVALID_ARGUMENT),
    (dict(hidden=0), _lib.ERR_INVALID_ARGUMENT), (dict(rows=2 ** 31), _lib.ERR_UNSUPPORTED),
    (dict(vocab=2 ** 31 - 512), _lib.ERR_UNSUPPORTED), (dict(hidden=100, ld_hidden=104), _lib.ERR_UNSUPPORTED),
    (dict(rows=2 ** 30, hidden=2 ** 20, ld_hidden=2 ** 20, ld_weight=2 ** 20), _lib.ERR_UNSUPPORTED),
    (dict(rows=2 ** 28, vocab=2 ** 28, hidden=8, ld_hidden=8, ld_weight=8), _lib.ERR_UNSUPPORTED),
    (dict(ld_hidden=120), _lib.ERR_INVALID_ARGUMENT), (dict(ld_weight=130), _lib.ERR_UNSUPPORTED),
    (dict(dtype=2), _lib.ERR_INVALID_ARGUMENT), (dict(index_bytes=2), _lib.ERR_INVALID_ARGUMENT),
    (dict(reduction=3), _lib.ERR_INVALID_ARGUMENT), (dict(top=257, ld_index=257, ld_teacher=257), _lib.ERR_UNSUPPORTED),
    (dict(top=-1), _lib.ERR_UNSUPPORTED), (dict(top=4, ld_index=3, ld_teacher=4), _lib.ERR_INVALID_ARGUMENT),
    (dict(top=4, ld_index=4, ld_teacher=4, teacher_dtype=3), _lib.ERR_INVALID_ARGUMENT),
    (dict(top=4, ld_index=4, ld_teacher=4, temperature=0.0), _lib.ERR_INVALID_ARGUMENT),
    (dict(temperature=2.0), _lib.ERR_INVALID_ARGUMENT),
])
def test_c_abi_refuses_descriptions(change, code):
    lib = _lib.load()
    d, info = desc(**change), _lib.VocabLossInfo()
    assert lib.b200_vocab_loss_info(ctypes.byref(d), 148, ctypes.byref(info)) == code
    assert _lib.last_error(lib)
    assert lib.b200_vocab_loss_forward(ctypes.byref(d), *([256] * 8), 1 << 40, None) == code
    assert lib.b200_vocab_loss_backward(ctypes.byref(d), *([256] * 10), 1 << 40, None) == code


def test_c_abi_refuses_pointers():
    lib = _lib.load()
    d, info = desc(), _lib.VocabLossInfo()
    assert lib.b200_vocab_loss_info(ctypes.byref(d), 0, ctypes.byref(info)) == _lib.ERR_INVALID_ARGUMENT
    assert lib.b200_vocab_loss_info(ctypes.byref(d), 148, None) == _lib.ERR_INVALID_ARGUMENT
    assert lib.b200_vocab_loss_info(None, 148, ctypes.byref(info)) == _lib.ERR_INVALID_ARGUMENT
    good = [256] * 8 + [1 << 40, None]
    for i in (0, 1, 2, 4, 5, 6, 7):  # hidden, weight, index, loss, lse, target_logp, workspace
        args = list(good)
        args[i] = None
        assert lib.b200_vocab_loss_forward(ctypes.byref(d), *args) == _lib.ERR_INVALID_ARGUMENT
    for i in (0, 1):
        args = list(good)
        args[i] = 264
        assert lib.b200_vocab_loss_forward(ctypes.byref(d), *args) == _lib.ERR_UNSUPPORTED
    t = desc(top=4, ld_index=4, ld_teacher=4)
    assert lib.b200_vocab_loss_forward(ctypes.byref(t), 256, 256, 256, None, *good[4:]) == _lib.ERR_INVALID_ARGUMENT
    good = [256] * 10 + [1 << 40, None]
    for i in (0, 1, 2, 4, 5, 6, 9):
        args = list(good)
        args[i] = None
        assert lib.b200_vocab_loss_backward(ctypes.byref(d), *args) == _lib.ERR_INVALID_ARGUMENT
    args = list(good)
    args[7] = args[8] = None
    assert lib.b200_vocab_loss_backward(ctypes.byref(d), *args) == _lib.ERR_UNSUPPORTED  # nothing asked for
    empty = desc(rows=0)
    assert lib.b200_vocab_loss_forward(ctypes.byref(empty), *([256] * 8), 1 << 40, None) == _lib.ERR_UNSUPPORTED


def sizes():
    import random
    r = random.Random(3)
    for _ in range(300):
        yield (round(math.exp(r.uniform(0, math.log(2e5)))), round(math.exp(r.uniform(0, math.log(3e5)))),
               8 * round(math.exp(r.uniform(0, math.log(1500)))), r.choice([0, 0, 1, 37, 256]))


@pytest.mark.parametrize("sms", [148, 132, 2, 1])
def test_policy_invariants(sms):
    """What the kernels rely on, over sizes of the whole range."""
    for rows, vocab, hidden, top in sizes():
        p = vocab_loss.policy(rows, vocab, hidden, top=top, sm_count=sms)
        assert (p["cta_group"], p["tile_n"]) in ((2, 256), (1, 256), (1, 128)) and p["tile_m"] == 128 * p["cta_group"]
        assert p["cta_group"] == 1 or rows > 128
        assert p["piece"] % 256 == 0 and (p["pieces"] - 1) * p["piece"] < vocab <= p["pieces"] * p["piece"]
        # Every run of dH's contraction has a k-slice in the first piece, which writes its sums.
        assert 1 <= p["splits_hidden"] <= 16 and p["splits_hidden"] <= -(-min(vocab, p["piece"]) // 64)
        assert 1 <= p["splits_weight"] <= 16 and (p["pieces"] == 1 or p["splits_weight"] == 1)
        # Room for G: 256 MiB, or what H takes, or one block of columns.
        pad = -(-rows // 256) * 256
        assert 2 * rows * p["piece"] <= max(256 << 20, 2 * pad * hidden, 2 * pad * 256)
        assert p["workspace_forward"] % 256 == 0 and p["workspace_backward"] >= 2 * rows * (p["piece"] + hidden)
        assert p["launches_backward"] == 2 + (top > 0) + 3 * p["pieces"]


def test_policy_of_known_sizes():
    p = vocab_loss.policy(8192, 128256, 4096)
    assert (p["cta_group"], p["tile_n"], p["splits_weight"]) == (2, 256, 1) and p["pieces"] > 1
    p = vocab_loss.policy(1, 128256, 4096)  # one token: the weight is read in narrow tiles, H not gathered
    assert (p["cta_group"], p["tile_n"], p["pieces"], p["launches_forward"]) == (1, 128, 1, 3)
    assert vocab_loss.policy(8192, 256, 512)["splits_weight"] > 1
    # A small call's rows are merged by the product's last block.
    assert vocab_loss.policy(26, 718, 120)["launches_forward"] == 2
    assert vocab_loss.policy(64, 1000, 256, top=8)["launches_forward"] == 2
    assert vocab_loss.policy(64, 32000, 256, top=8)["launches_forward"] == 3
    assert vocab_loss.policy(2048, 32000, 256, top=8)["launches_forward"] == 4
    assert vocab_loss.policy(64, 32000, 256)["launches_forward"] == 3
    assert vocab_loss.policy(0, 10, 8)["launches_forward"] == 0
    with pytest.raises(ValueError):
        vocab_loss.policy(1, 1, 8, dtype=torch.float32)
    with pytest.raises(_lib.BridgeError):
        vocab_loss.policy(1, 1, 12)


# --------------------------------------------------------------------------
# The reference
# --------------------------------------------------------------------------
def case(seed=0, rows=13, vocab=40, hidden=16, top=5):
    g = torch.Generator().manual_seed(seed)
    h, w = torch.randn(rows, hidden, generator=g).to(BF16), torch.randn(vocab, hidden, generator=g).to(BF16)
    t = torch.randint(0, vocab, (rows,), generator=g)
    t[[1, 7]] = -100
    logits, index = torch.randn(rows, top, generator=g), torch.randint(0, vocab, (rows, top), generator=g)
    index[3], index[4, 2:] = -1, -1
    index[5] = 9  # one token in every entry
    logits[6, 0] = -math.inf
    return h, w, t, logits, index


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_reference_cross_entropy(reduction):
    h, w, t, _, _ = case()
    up = torch.rand(13) + 0.5 if reduction == "none" else torch.tensor(0.7)
    hd, wd = h.double().requires_grad_(), w.double().requires_grad_()
    loss = torch.nn.functional.cross_entropy(hd @ wd.t(), t, ignore_index=-100, reduction=reduction)
    dh, dw = torch.autograd.grad(loss, (hd, wd), up.double())
    got = ref.reference(h, w, *ref.targets_of(t, -100), 1.0, reduction, up)
    for a, b in zip((loss, dh, dw), got[::2]):
        torch.testing.assert_close(a.detach(), b, rtol=1e-12, atol=1e-13)
    assert all(bool((b >= 0).all()) for b in got[1::2])


def test_reference_distillation():
    h, w, _, logits, index = case()
    hd, wd = h.double().requires_grad_(), w.double().requires_grad_()
    z = hd @ wd.t() / 2
    dense = torch.zeros_like(z)
    for r in range(13):
        there = [k for k in range(5) if index[r, k] >= 0 and logits[r, k] > -math.inf]
        if there:
            q = torch.softmax(logits[r, there].double() / 2, 0)
            for k, x in zip(there, q):
                dense[r, index[r, k]] += x
    kept = dense.sum(1) > 0
    want = 4 * (torch.xlogy(dense, dense) - dense * torch.log_softmax(z, 1)).sum(1)
    want = torch.where(kept, want, 0.0)
    dh, dw = torch.autograd.grad(want.sum(), (hd, wd), torch.tensor(1.3, dtype=torch.float64))
    got = ref.reference(h, w, *ref.teacher_of(logits, index, 2.0), 2.0, "sum", torch.tensor(1.3, dtype=torch.float64))
    for a, b in zip((want.sum(), dh, dw), got[::2]):
        torch.testing.assert_close(a.detach(), b, rtol=1e-12, atol=1e-13)


def test_bounds_notice_mistakes():
    """What a wrong kernel would give is outside the bounds: planted here in the results."""
    h, w, t, _, _ = case(rows=13)
    up = torch.tensor(1.0)
    loss, bl, dh, bh, dw, bw = ref.reference(h, w, *ref.targets_of(t, -100), 1.0, "sum", up)
    ref.check("same", dh, dh, bh)
    wrong = dh.clone()
    wrong[0] += w[t[0]].double()  # the target's term left out
    with pytest.raises(AssertionError):
        ref.check("target", wrong, dh, bh)
    with pytest.raises(AssertionError):
        ref.check("scale", dw * 1.05, dw, bw)
    with pytest.raises(AssertionError):
        ref.check("loss", loss * 1.001, loss, bl)
    with pytest.raises(AssertionError):
        ref.check("nan", torch.full_like(dh, math.nan), dh, bh)
    with pytest.raises(AssertionError):
        ref.check("shape", dh[:1], dh, bh)


# --------------------------------------------------------------------------
# The command
# --------------------------------------------------------------------------
@pytest.mark.parametrize("args", [["--loss", "mse"], ["--iterations", "0"], ["--rows", "0"], ["--ignored", "1.0"],
                                  ["--temperature", "2.0"], ["--way", "backward"]])
def test_command_usage_errors(args, capsys):
    from b200gemm.cli import vocab_loss as cli
    assert cli.main(args) == 2
    assert capsys.readouterr().out == ""


def test_command_needs_a_gpu(capsys):
    from b200gemm.cli import vocab_loss as cli
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    assert cli.main([]) == 1
    got = capsys.readouterr()
    assert got.out == "" and "ERROR" in got.err
