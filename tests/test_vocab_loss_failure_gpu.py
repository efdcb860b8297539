"""Losses at the vocabulary projection: a call that is given up says so, and leaves the GPU as it was.

A wait runs out where a tile takes longer than the limit, or the status word of a running call is set
from another stream, as a role that gives up sets it. Neither faults or hangs: every wait of the kernels
is bounded, and a CTA leaves when the loads and products that it has started have ended."""
import ctypes
import os
import subprocess
import sys
import time
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]

_LONG_TILE_CHILD = r"""
import sys
sys.path.insert(0, "gb300-gemm-anatomy_b200")
import torch
from b200gemm import vocab_loss
def step(rows, vocab, hidden, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(rows, hidden, generator=g, device="cuda").bfloat16().requires_grad_()
    w = torch.empty(vocab, hidden, dtype=torch.bfloat16, device="cuda")
    for v in range(0, vocab, 64):
        w[v:v + 64] = torch.randn(min(64, vocab - v), hidden, generator=g, device="cuda") / hidden ** 0.5
    w.requires_grad_()
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    loss = vocab_loss.linear_cross_entropy(h, w, t)
    return loss.detach(), *torch.autograd.grad(loss, (h, w))
before = step(40, 700, 128)
# One tile of the backward pass: 25000 k-slices of 64, which take it several milliseconds.
loss, dh, dw = step(8, 256, 1600000)
torch.cuda.synchronize()
print("LOSS", bool(loss.isfinite()))
print("DH", bool(dh.isnan().all()))
print("DW", all(bool(x.isnan().all()) for x in dw.split(64)))
del loss, dh, dw
after = step(40, 700, 128)
print("AFTER", all(torch.equal(a, b) for a, b in zip(before, after)) and all(bool(a.isfinite().all()) for a in after))
"""


def child(code, **env):
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env=dict(os.environ, **env), capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    return dict(line.split(" ", 1) for line in r.stdout.strip().splitlines())


def test_wait_that_runs_out_leaves_nan_in_both_gradients():
    """The limit is read once per process: 1 ms, less than the tile takes. The forward pass drains its
    accumulators after a few k-slices each, so none of its waits is as long."""
    assert child(_LONG_TILE_CHILD, B200_WAIT_TIMEOUT_MS="1") == dict(LOSS="True", DH="True", DW="True", AFTER="True")


def test_the_same_tile_within_the_limit():
    assert child(_LONG_TILE_CHILD) == dict(LOSS="True", DH="False", DW="False", AFTER="True")


class Raw:
    """A call through the C ABI, with its workspace in hand: the status word is its first 32 bits."""

    def __init__(self, rows, vocab, hidden, top=0, reduction=None):
        from b200gemm import _lib
        self.lib, self._lib = _lib.load(), _lib
        reduction = _lib.VL_MEAN if reduction is None else reduction
        self.desc = _lib.VocabLossDesc(rows, vocab, hidden, hidden, hidden, _lib.VL_BF16, top, 8, top, top, _lib.VL_F32, -100,
                                       reduction, 1.0)
        self.info = _lib.VocabLossInfo()
        sms = torch.cuda.get_device_properties(0).multi_processor_count
        assert self.lib.b200_vocab_loss_info(ctypes.byref(self.desc), sms, ctypes.byref(self.info)) == _lib.OK
        g = torch.Generator(device="cuda").manual_seed(1)
        f32 = dict(dtype=torch.float32, device="cuda")
        self.h = torch.randn(rows, hidden, generator=g, device="cuda").bfloat16()
        self.w = torch.empty(vocab, hidden, dtype=torch.bfloat16, device="cuda")
        for v in range(0, vocab, 16384):
            self.w[v:v + 16384] = torch.randn(min(16384, vocab - v), hidden, generator=g, device="cuda") * 0.02
        self.index = torch.randint(0, vocab, (rows, top) if top else (rows,), generator=g, device="cuda")
        self.teacher = torch.randn(rows, top, generator=g, device="cuda") if top else None
        self.loss = torch.empty(rows if reduction == _lib.VL_NONE else 1, **f32)
        self.lse, self.logp = torch.empty(rows, **f32), torch.empty(rows, max(top, 1), **f32)
        self.up = torch.ones(rows if reduction == _lib.VL_NONE else 1, **f32)
        self.dh, self.dw = torch.empty_like(self.h), torch.empty_like(self.w)
        self.ws = torch.empty(max(self.info.workspace_forward, self.info.workspace_backward), dtype=torch.uint8, device="cuda")
        self.stream = torch.cuda.Stream()
        torch.cuda.synchronize()

    def _ptrs(self, *tensors):
        return [None if t is None else t.data_ptr() for t in tensors]

    def forward(self):
        rc = self.lib.b200_vocab_loss_forward(
            ctypes.byref(self.desc), *self._ptrs(self.h, self.w, self.index, self.teacher, self.loss, self.lse, self.logp, self.ws),
            self.info.workspace_forward, self.stream.cuda_stream)
        assert rc == self._lib.OK, self._lib.last_error()

    def backward(self):
        rc = self.lib.b200_vocab_loss_backward(
            ctypes.byref(self.desc),
            *self._ptrs(self.h, self.w, self.index, self.teacher, self.lse, self.logp, self.up, self.dh, self.dw, self.ws),
            self.info.workspace_backward, self.stream.cuda_stream)
        assert rc == self._lib.OK, self._lib.last_error()

    def given_up(self, call, share):
        """Runs `call`, and sets its status word when about `share` of it has run; tries until the word was
        set while it ran."""
        word = torch.full((4,), 0x7f, dtype=torch.uint8).pin_memory()
        other = torch.cuda.Stream()

        def timed(poke_after):
            e0, e1, poked = (torch.cuda.Event(enable_timing=True) for _ in range(3))
            torch.cuda.synchronize()
            with torch.cuda.stream(self.stream):
                e0.record()
                call()
                e1.record()
            if poke_after is not None:
                e0.synchronize()
                time.sleep(poke_after)
                with torch.cuda.stream(other):
                    self.ws[:4].copy_(word, non_blocking=True)
                    poked.record()
            torch.cuda.synchronize()
            return e0.elapsed_time(e1), e0.elapsed_time(poked) if poke_after is not None else None
        timed(None)
        whole, _ = timed(None)
        for _ in range(20):
            took, at = timed(share * whole / 1e3)
            if 0.1 * whole < at < 0.95 * whole and took > at:
                return whole, took, at
        pytest.fail(f"the word was never set while the call ran ({whole} ms)")


@pytest.mark.parametrize("top,reduction", [(0, 0), (0, 1), (16, 2)])
def test_forward_given_up(top, reduction):
    c = Raw(4096, 128256, 4096, top, reduction)
    c.forward()
    torch.cuda.synchronize()
    want = c.loss.clone(), c.lse.clone(), c.logp.clone()
    assert all(x.isfinite().all() for x in want)
    _, took, at = c.given_up(c.forward, 0.4)
    assert c.loss.isnan().all() and c.lse.isnan().all()
    # A backward pass that goes on from there gives no numbers either.
    c.backward()
    torch.cuda.synchronize()
    assert c.dh.isnan().all() and all(x.isnan().all() for x in c.dw.split(16384))
    # The next call on the same workspace is whole again.
    c.forward()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((c.loss, c.lse, c.logp), want))


@pytest.mark.parametrize("share", [0.2, 0.4, 0.6, 0.8])
def test_backward_given_up(share):
    """In the middle of each of the products of several pieces."""
    c = Raw(4096, 128256, 4096)
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    want = c.dh.clone(), c.dw.clone()
    assert all(x.isfinite().all() for x in want[0].split(4096)) and not want[1][:100].isnan().any()
    c.dh.zero_()
    c.dw.zero_()
    c.given_up(c.backward, share)
    assert c.dh.isnan().all() and all(x.isnan().all() for x in c.dw.split(16384))
    c.backward()
    torch.cuda.synchronize()
    assert torch.equal(c.dh, want[0]) and all(torch.equal(a, b) for a, b in zip(c.dw.split(16384), want[1].split(16384)))
