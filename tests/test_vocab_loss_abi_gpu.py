"""Losses at the vocabulary projection through the C ABI: every output is written, whatever was in its memory
and in the workspace, and a teacher's rows may have pitches of their own."""
import ctypes
import math

import pytest
import torch

import vocab_loss_reference as ref

pytestmark = pytest.mark.gpu


class Call:
    def __init__(self, rows, vocab, hidden, top=0, reduction="none", tau=1.0, pitch=0, ignored=0.3, index_dtype=torch.int64):
        from b200gemm import _lib
        self.lib, self.ok = _lib.load(), _lib.OK
        g = torch.Generator(device="cuda").manual_seed(5)
        self.h = torch.randn(rows, hidden, generator=g, device="cuda").bfloat16()
        self.w = (torch.randn(vocab, hidden, generator=g, device="cuda") / 8).bfloat16()
        drop = torch.randperm(rows, generator=g, device="cuda")[:int(rows * ignored)]
        self.tau, self.reduction, self.teacher = tau, reduction, None
        if top:
            # Columns behind the top ones: tokens that would count, logits that would dominate.
            index = torch.randint(0, vocab, (rows, top + pitch), generator=g, device="cuda").to(index_dtype)
            teacher = torch.full((rows, top + 2 * pitch), 1e4, device="cuda")
            self.index, self.teacher = index[:, :top], teacher[:, :top]
            self.index[:, top // 2:] = self.index[:, :1]  # a token that comes again
            self.index[drop] = -1
            self.teacher.copy_(torch.randn(rows, top, generator=g, device="cuda"))
        else:
            self.index = torch.randint(0, vocab, (rows,), generator=g, device="cuda").to(index_dtype)
            self.index[drop] = -100
        code = {"none": _lib.VL_NONE, "mean": _lib.VL_MEAN, "sum": _lib.VL_SUM}[reduction]
        self.desc = _lib.VocabLossDesc(rows, vocab, hidden, hidden, hidden, _lib.VL_BF16, top, self.index.element_size(), top + pitch,
                                       top + 2 * pitch, _lib.VL_F32, -100, code, tau)
        self.info = _lib.VocabLossInfo()
        sms = torch.cuda.get_device_properties(0).multi_processor_count
        assert self.lib.b200_vocab_loss_info(ctypes.byref(self.desc), sms, ctypes.byref(self.info)) == self.ok
        n = rows if reduction == "none" else 1
        self.up = torch.rand(n, generator=g, device="cuda")
        f32 = dict(dtype=torch.float32, device="cuda")
        self.loss, self.lse, self.logp = torch.empty(n, **f32), torch.empty(rows, **f32), torch.empty(rows, max(top, 1), **f32)
        self.dh, self.dw = torch.empty_like(self.h), torch.empty_like(self.w)
        self.ws = torch.empty(max(self.info.workspace_forward, self.info.workspace_backward), dtype=torch.uint8, device="cuda")

    def run(self, fill):
        """Both directions, on memory filled with the byte `fill`."""
        outputs = self.loss, self.lse, self.logp, self.dh, self.dw
        for t in outputs + (self.ws,):
            t.view(torch.uint8).fill_(fill)
        ptr = lambda *ts: [None if t is None else t.data_ptr() for t in ts]  # noqa: E731
        stream = torch.cuda.current_stream().cuda_stream
        assert self.lib.b200_vocab_loss_forward(
            ctypes.byref(self.desc), *ptr(self.h, self.w, self.index, self.teacher, self.loss, self.lse, self.logp, self.ws),
            self.info.workspace_forward, stream) == self.ok
        self.ws.fill_(fill ^ 0x55)  # nothing goes from one direction to the other there
        assert self.lib.b200_vocab_loss_backward(
            ctypes.byref(self.desc),
            *ptr(self.h, self.w, self.index, self.teacher, self.lse, self.logp, self.up, self.dh, self.dw, self.ws),
            self.info.workspace_backward, stream) == self.ok
        torch.cuda.synchronize()
        return [t.clone() for t in outputs]

    def check(self, got):
        kept, index, q = (ref.teacher_of(self.teacher, self.index, self.tau) if self.teacher is not None
                          else ref.targets_of(self.index, -100))
        up = self.up if self.reduction == "none" else self.up[0]
        loss, bl, dh, bh, dw, bw = ref.reference(self.h, self.w, kept, index, q, self.tau, self.reduction, up)
        ref.check("loss", got[0] if self.reduction == "none" else got[0][0], loss, bl)
        ref.check("d_hidden", got[3], dh, bh)
        ref.check("d_weight", got[4], dw, bw)


@pytest.mark.parametrize("rows,vocab,hidden,top", [(1, 300, 64, 0), (70, 900, 72, 0), (70, 900, 72, 12), (40, 300, 1000, 33),
                                                   (700, 20000, 136, 7), (2000, 3000, 64, 0), (17, 300, 64, 256)])
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_every_output_is_written(rows, vocab, hidden, top, reduction):
    c = Call(rows, vocab, hidden, top, reduction)
    zeros, ones, odd = c.run(0), c.run(0xff), c.run(0x7b)
    c.check(ones)
    for a, b, d in zip(zeros, ones, odd):
        assert torch.equal(a, b) and torch.equal(a, d)  # and so no NaN of the fill


@pytest.mark.parametrize("rows,vocab,hidden,top", [(9, 300, 64, 5), (300, 2000, 136, 30), (1500, 9000, 72, 6)])
@pytest.mark.parametrize("pitch", [1, 13])
@pytest.mark.parametrize("index_dtype", [torch.int32, torch.int64])
def test_pitches_of_a_teacher(rows, vocab, hidden, top, pitch, index_dtype):
    c = Call(rows, vocab, hidden, top, "sum", tau=2.0, pitch=pitch, index_dtype=index_dtype)
    c.check(c.run(0xff))
    assert not math.isnan(float(c.loss))
