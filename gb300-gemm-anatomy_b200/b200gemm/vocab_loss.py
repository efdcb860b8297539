"""Losses at the vocabulary projection: cross entropy and distillation without the logits.

``hidden`` (rows of a model's last layer) and ``weight`` (the vocabulary
projection, one row per token) have the layout of the GEMM's operands: row-major
``... x D`` and ``V x D``, so the logits would be ``gemm(hidden, weight)``. They
are computed tile by tile on the tensor cores, reduced in the kernel and never
written (``b200_vocab_loss_forward`` / ``_backward`` in ``include/b200gemm.h``).

Both functions are differentiable in ``hidden`` and ``weight`` (once), run on
the current stream of the operands' device, never synchronise and can be
captured into a CUDA graph. (As everywhere in torch, a backward pass that
accumulates into leaves is captured only while no eager graph of the same leaves
is alive.) Results do not depend on the order in which tiles run: the same call
gives the same bits.

A kernel wait that runs out (``B200_WAIT_TIMEOUT_MS``) leaves NaN in the results.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib

IGNORE_INDEX = -100
MAX_TOP = 256  # teacher logits per row

_OPERAND_CODE = {torch.bfloat16: _lib.VL_BF16, torch.float16: _lib.VL_F16}
_TEACHER_CODE = {**_OPERAND_CODE, torch.float32: _lib.VL_F32}
_INDEX_BYTES = {torch.int32: 4, torch.int64: 8}
_REDUCTION_CODE = {"none": _lib.VL_NONE, "mean": _lib.VL_MEAN, "sum": _lib.VL_SUM}


def _require_tensor(t, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")


def _require_operands(hidden, weight) -> None:
    _require_tensor(hidden, "hidden")
    _require_tensor(weight, "weight")
    if hidden.dtype not in _OPERAND_CODE:
        raise ValueError(f"hidden must be bfloat16 or float16, got {hidden.dtype}")
    if weight.dtype != hidden.dtype:
        raise ValueError(f"weight must be {hidden.dtype} like hidden, got {weight.dtype}")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden (... x D) and weight (V x D) do not match: shapes "
                         f"{tuple(hidden.shape)} and {tuple(weight.shape)}")
    d = weight.shape[1]
    if weight.shape[0] < 1 or d < 1 or d % 8 != 0:
        raise ValueError(f"weight has shape {tuple(weight.shape)}: V and D must be positive and D a "
                         "multiple of 8 (rows of whole 16-byte units)")
    for t, name in ((hidden, "hidden"), (weight, "weight")):
        if t.numel() and t.stride(-1) != 1:
            raise ValueError(f"{name} must have contiguous rows (D innermost), strides {t.stride()}")


def _require_same_device(hidden, **others) -> None:
    if hidden.device.type != "cuda":
        raise ValueError(f"hidden must live on a CUDA device, got {hidden.device}")
    for name, t in others.items():
        if t.device != hidden.device:
            raise ValueError(f"{name} must be on {hidden.device} like hidden, got {t.device}")


def _require_pitch(t: torch.Tensor, name: str) -> None:
    if t.shape[0] > 1 and (t.stride(0) < t.shape[1] or t.stride(0) % 8 != 0):
        raise ValueError(f"{name} rows must be a multiple of 8 elements apart and not overlap, "
                         f"strides {t.stride()}")
    if t.data_ptr() % 16 != 0:
        raise ValueError(f"{name} must start on a 16-byte boundary")


def _pitch(t: torch.Tensor) -> int:
    return int(t.stride(0)) if t.shape[0] > 1 else int(t.shape[1])


@functools.lru_cache(maxsize=256)
def _info(fields: tuple, temperature: float, sm_count: int):
    lib = _lib.load()
    info = _lib.VocabLossInfo()
    desc = _lib.VocabLossDesc(*fields, temperature)
    _lib.check(lib.b200_vocab_loss_info(ctypes.byref(desc), sm_count, ctypes.byref(info)),
               "b200_vocab_loss_info", lib)
    return info


def policy(rows: int, vocab: int, hidden: int, *, top: int = 0, dtype=torch.bfloat16,
           sm_count: int = 148) -> dict:
    """The host's choices for a call (b200_vocab_loss_info), computed without a device: tile
    shape, pieces of the vocabulary, runs of the contraction, workspace bytes, launches.
    ``top=0`` is the cross entropy."""
    fields = (int(rows), int(vocab), int(hidden), int(hidden), int(hidden), _OPERAND_CODE[dtype], int(top),
              8, int(top), int(top), _lib.VL_F32, IGNORE_INDEX, _lib.VL_MEAN)
    info = _info(fields, 1.0, int(sm_count))
    return {name: getattr(info, name) for name, _ in info._fields_}


class _VocabLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, index, teacher, ignore_index, reduction, temperature):
        rows, d = hidden.shape
        per_row = reduction == _lib.VL_NONE
        ctx.empty = rows == 0
        ctx.shape = (hidden.shape, weight.shape)
        loss = torch.empty((rows,) if per_row else (), dtype=torch.float32, device=hidden.device)
        if ctx.empty:
            ctx.like = (hidden.dtype, hidden.device)
            return loss if per_row else loss.zero_()
        top = 0 if teacher is None else int(teacher.shape[1])
        fields = (rows, int(weight.shape[0]), d, _pitch(hidden), _pitch(weight), _OPERAND_CODE[hidden.dtype], top,
                  _INDEX_BYTES[index.dtype], _pitch(index) if top else 0, _pitch(teacher) if top else 0,
                  _TEACHER_CODE[teacher.dtype] if top else 0, ignore_index, reduction)
        sms = torch.cuda.get_device_properties(hidden.device).multi_processor_count
        info = _info(fields, temperature, sms)
        lib = _lib.load()
        desc = _lib.VocabLossDesc(*fields, temperature)
        lse = torch.empty(rows, dtype=torch.float32, device=hidden.device)
        with torch.cuda.device(hidden.device):
            ws = torch.empty(info.workspace_forward, dtype=torch.uint8, device=hidden.device)
            stream = torch.cuda.current_stream().cuda_stream
            rc = lib.b200_vocab_loss_forward(
                ctypes.byref(desc), hidden.data_ptr(), weight.data_ptr(), index.data_ptr(),
                teacher.data_ptr() if top else None, loss.data_ptr(), lse.data_ptr(), ws.data_ptr(),
                info.workspace_forward, stream)
        _lib.check(rc, "b200_vocab_loss_forward", lib)
        ctx.save_for_backward(hidden, weight, index, teacher, lse)
        ctx.desc, ctx.info = desc, info
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        want_h, want_w = ctx.needs_input_grad[:2]
        if ctx.empty:
            dtype, device = ctx.like
            dh, dw = (torch.zeros(s, dtype=dtype, device=device) if want else None
                      for s, want in zip(ctx.shape, (want_h, want_w)))
            return dh, dw, None, None, None, None, None
        hidden, weight, index, teacher, lse = ctx.saved_tensors
        lib = _lib.load()
        grad = grad.to(torch.float32).contiguous()
        dh = torch.empty(hidden.shape, dtype=hidden.dtype, device=hidden.device) if want_h else None
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device) if want_w else None
        with torch.cuda.device(hidden.device):
            ws = torch.empty(ctx.info.workspace_backward, dtype=torch.uint8, device=hidden.device)
            stream = torch.cuda.current_stream().cuda_stream
            rc = lib.b200_vocab_loss_backward(
                ctypes.byref(ctx.desc), hidden.data_ptr(), weight.data_ptr(), index.data_ptr(),
                None if teacher is None else teacher.data_ptr(), lse.data_ptr(), grad.data_ptr(),
                dh.data_ptr() if want_h else None, dw.data_ptr() if want_w else None, ws.data_ptr(),
                ctx.info.workspace_backward, stream)
        _lib.check(rc, "b200_vocab_loss_backward", lib)
        return dh, dw, None, None, None, None, None


def _reduction(reduction: str) -> int:
    if reduction not in _REDUCTION_CODE:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTION_CODE)}, got {reduction!r}")
    return _REDUCTION_CODE[reduction]


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *,
                         ignore_index: int = IGNORE_INDEX, reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of ``softmax(hidden @ weight.T)`` against one token per row.

    hidden: ``... x D`` bf16 or fp16, weight: ``V x D`` of the same type, target: ``...`` int32 or
    int64. Rows whose target is ``ignore_index`` have no loss: they count 0, get zero gradients and
    meet no other row whatever they hold, and cost nothing in the products. A target outside
    ``[0, V)`` makes the loss NaN. reduction: "none" (shape of target), "mean" over the rows with a
    loss (0 without any) or "sum"; fp32. The gradients have the operands' type.
    """
    _require_operands(hidden, weight)
    _require_tensor(target, "target")
    code = _reduction(reduction)
    if target.dtype not in _INDEX_BYTES:
        raise ValueError(f"target must be int32 or int64, got {target.dtype}")
    if target.shape != hidden.shape[:-1]:
        raise ValueError(f"target has shape {tuple(target.shape)}, expected {tuple(hidden.shape[:-1])}")
    if not -2 ** 63 <= int(ignore_index) < 2 ** 63:
        raise ValueError(f"ignore_index={ignore_index} is no 64-bit integer")
    _require_same_device(hidden, weight=weight, target=target)
    h = hidden.reshape(-1, hidden.shape[-1])
    _require_pitch(h, "hidden")
    _require_pitch(weight, "weight")
    loss = _VocabLoss.apply(h, weight, target.reshape(-1).contiguous(), None, int(ignore_index), code, 1.0)
    return loss.reshape(target.shape) if reduction == "none" else loss


def linear_distillation(hidden: torch.Tensor, weight: torch.Tensor, teacher_logits: torch.Tensor,
                        teacher_index: torch.Tensor, *, temperature: float = 1.0,
                        reduction: str = "mean") -> torch.Tensor:
    """``temperature**2 * KL(q || softmax(hidden @ weight.T / temperature))`` against a teacher's top logits.

    teacher_logits: ``... x K`` fp32, bf16 or fp16, the logits a teacher kept for each row;
    teacher_index: ``... x K`` int32 or int64, their tokens, in any order; K from 1 to 256. q is the
    softmax of ``teacher_logits / temperature`` over the row's entries: those with a negative index
    or a logit of -inf are padding, entries of the same token add up. A row of nothing but padding
    has no loss, like an ignored target in ``linear_cross_entropy``; an index of V or more makes it
    NaN. The teacher gets no gradient. Everything else as in ``linear_cross_entropy``.
    """
    _require_operands(hidden, weight)
    _require_tensor(teacher_logits, "teacher_logits")
    _require_tensor(teacher_index, "teacher_index")
    code = _reduction(reduction)
    if teacher_logits.dtype not in _TEACHER_CODE:
        raise ValueError(f"teacher_logits must be float32, bfloat16 or float16, got {teacher_logits.dtype}")
    if teacher_index.dtype not in _INDEX_BYTES:
        raise ValueError(f"teacher_index must be int32 or int64, got {teacher_index.dtype}")
    if teacher_logits.shape != teacher_index.shape or teacher_logits.dim() != hidden.dim() or \
            teacher_logits.shape[:-1] != hidden.shape[:-1]:
        raise ValueError(f"teacher_logits and teacher_index must both be {tuple(hidden.shape[:-1])} x K, got "
                         f"{tuple(teacher_logits.shape)} and {tuple(teacher_index.shape)}")
    if not 1 <= teacher_logits.shape[-1] <= MAX_TOP:
        raise ValueError(f"a teacher's row holds 1 to {MAX_TOP} logits, got {teacher_logits.shape[-1]}")
    if teacher_logits.requires_grad:
        raise ValueError("teacher_logits gets no gradient: detach it")
    temperature = float(temperature)
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    _require_same_device(hidden, weight=weight, teacher_logits=teacher_logits, teacher_index=teacher_index)
    h = hidden.reshape(-1, hidden.shape[-1])
    _require_pitch(h, "hidden")
    _require_pitch(weight, "weight")
    k = teacher_logits.shape[-1]
    loss = _VocabLoss.apply(h, weight, teacher_index.reshape(-1, k).contiguous(),
                            teacher_logits.reshape(-1, k).contiguous(), 0, code, temperature)
    return loss.reshape(hidden.shape[:-1]) if reduction == "none" else loss
