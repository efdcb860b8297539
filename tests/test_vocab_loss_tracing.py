"""Losses at the vocabulary projection: tensors that only stand for others are refused, not read."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

from b200gemm import vocab_loss


def call(kind, h, w, index, logits):
    if kind == "ce":
        return vocab_loss.linear_cross_entropy(h, w, index[:, 0])
    return vocab_loss.linear_distillation(h, w, logits, index)


def tensors(device):
    return (torch.empty(4, 16, dtype=torch.bfloat16, device=device), torch.empty(32, 16, dtype=torch.bfloat16, device=device),
            torch.zeros(4, 3, dtype=torch.long, device=device), torch.zeros(4, 3, device=device))


@pytest.mark.parametrize("kind", ["ce", "kd"])
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("device", ["cuda", "cpu"])
def test_fake_tensors(kind, grad, device):
    with FakeTensorMode():
        args = tensors(device)
        args[0].requires_grad_(grad)
        with pytest.raises(TypeError, match="torch.compiler.disable"):
            call(kind, *args)
    with pytest.raises(TypeError, match="torch.compiler.disable"):
        call(kind, *args)


@pytest.mark.parametrize("kind,which,name", [("ce", 0, "hidden"), ("ce", 1, "weight"), ("ce", 2, "target"),
                                             ("kd", 2, "teacher_index"), ("kd", 3, "teacher_logits")])
def test_one_fake_tensor(kind, which, name):
    args = list(tensors("cpu"))
    with FakeTensorMode() as mode:
        args[which] = mode.from_tensor(args[which])
    with pytest.raises(TypeError, match=name):
        call(kind, *args)


def test_modes_that_only_look():
    """A dispatch mode that passes every call on is no reason to refuse: the next check is the device's."""
    class Look(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    with Look(), pytest.raises(ValueError, match="CUDA device"):
        call("ce", *tensors("cpu"))


def test_compile_says_so():
    def step(h, w, index, logits):
        return call("ce", h, w, index, logits) * 2
    with pytest.raises(Exception, match="torch.compiler.disable"):
        torch.compile(step, backend="eager", fullgraph=True)(*tensors("cpu"))


@pytest.mark.parametrize("which", [0, 1])
def test_autocast_does_not_cast(which):
    args = list(tensors("cpu"))
    args[which] = args[which].float()
    with torch.autocast("cpu", dtype=torch.bfloat16), pytest.raises(ValueError, match="bfloat16|like hidden"):
        call("ce", *args)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["ce", "kd"])
def test_called_beside_a_compiled_graph(kind):
    g = torch.Generator(device="cuda").manual_seed(0)
    h = torch.randn(9, 64, generator=g, device="cuda").bfloat16().requires_grad_()
    w = torch.randn(50, 64, generator=g, device="cuda").bfloat16().requires_grad_()
    index = torch.randint(0, 50, (9, 3), generator=g, device="cuda")
    logits = torch.randn(9, 3, generator=g, device="cuda")
    outside = torch.compiler.disable(call)

    def step(f):
        return f(kind, h * 2, w, index, logits) * 3
    want = step(call)
    got = torch.compile(lambda: step(outside), backend="eager")()
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, (h, w)), torch.autograd.grad(want, (h, w))))


@pytest.mark.gpu
def test_backward_of_fake_tensors():
    g = torch.Generator(device="cuda").manual_seed(0)
    h = torch.randn(9, 64, generator=g, device="cuda").bfloat16().requires_grad_()
    w = torch.randn(50, 64, generator=g, device="cuda").bfloat16()
    t = torch.randint(0, 50, (9,), generator=g, device="cuda")
    mode = FakeTensorMode()
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, mode.from_tensor):
        loss = vocab_loss.linear_cross_entropy(h, w, t)
        with pytest.raises(TypeError, match="ordinary"):
            torch.autograd.grad(loss, h)
    loss = vocab_loss.linear_cross_entropy(h, w, t, reduction="none")
    up = mode.from_tensor(torch.ones(9, device="cuda"))
    with pytest.raises(TypeError, match="ordinary"):
        torch.autograd.grad(loss, h, up)
