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

Tensors without storage of their own are refused, so ``torch.compile`` cannot trace these losses:
call them through ``torch.compiler.disable``. Autocast does not cast for them: an fp32 operand is
refused under it as without it.
"""
from __future__ import annotations

import ctypes
import operator

import torch

from . import _lib

IGNORE_INDEX = -100
MAX_TOP = 256  # teacher logits per row

_OPERAND_CODE = {torch.bfloat16: _lib.VL_BF16, torch.float16: _lib.VL_F16}
_REDUCTION_CODE = {"none": _lib.VL_NONE, "mean": _lib.VL_MEAN, "sum": _lib.VL_SUM}


def policy(rows: int, vocab: int, hidden: int, *, top: int = 0, dtype=torch.bfloat16,
           reduction: str = "mean", sm_count: int = 148) -> dict:
    """The host's choices for a call (b200_vocab_loss_info), computed without a device: tile
    shape, pieces of the vocabulary, runs of the contraction, workspace bytes, launches.
    ``top=0`` is the cross entropy. In half precision reduction "none" takes two launches and a
    copy of hidden more (the weights of rows)."""
    lib = _lib.load()
    if dtype not in _OPERAND_CODE:
        raise ValueError(f"dtype must be bfloat16 or float16, got {dtype}")
    if reduction not in _REDUCTION_CODE:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTION_CODE)}, got {reduction!r}")
    desc = _lib.VocabLossDesc(rows, vocab, hidden, hidden, hidden, _OPERAND_CODE[dtype], top, 8, top, top,
                              _lib.VL_F32, IGNORE_INDEX, _REDUCTION_CODE[reduction], 1.0)
    info = _lib.VocabLossInfo()
    _lib.check(lib.b200_vocab_loss_info(ctypes.byref(desc), sm_count, ctypes.byref(info)),
               "b200_vocab_loss_info", lib)
    return {name: getattr(info, name) for name, _ in info._fields_}


_op = None


def _call(hidden, weight, index, teacher, names, ignore_index, reduction, temperature):
    """The operator checks everything else (shapes, types, strides, devices) and raises ValueError."""
    global _op
    if reduction not in _REDUCTION_CODE:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTION_CODE)}, got {reduction!r}")
    for t, name in zip((hidden, weight, index, teacher), names):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if _op is None:
        _op = _lib.torch_ops().vocab_loss.default
    return _op(hidden, weight, index, teacher, ignore_index, _REDUCTION_CODE[reduction], temperature)


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *,
                         ignore_index: int = IGNORE_INDEX, reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of ``softmax(hidden @ weight.T)`` against one token per row.

    hidden: ``... x D`` bf16 or fp16, weight: ``V x D`` of the same type, target: ``...`` int32 or
    int64. Rows whose target is ``ignore_index`` have no loss: they count 0, get zero gradients and
    meet no other row whatever they hold, and cost nothing in the products. A target outside
    ``[0, V)`` makes the loss NaN. reduction: "none" (shape of target), "mean" over the rows with a
    loss (0 without any) or "sum"; fp32. The gradients have the operands' type.
    """
    try:
        ignore_index = operator.index(ignore_index)
    except TypeError:
        raise ValueError(f"ignore_index={ignore_index!r} is no integer") from None
    if not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError(f"ignore_index={ignore_index} is no 64-bit integer")
    return _call(hidden, weight, target, None, ("hidden", "weight", "target"), ignore_index, reduction, 1.0)


def linear_distillation(hidden: torch.Tensor, weight: torch.Tensor, teacher_logits: torch.Tensor,
                        teacher_index: torch.Tensor, *, temperature: float = 1.0,
                        reduction: str = "mean") -> torch.Tensor:
    """``temperature**2 * KL(q || softmax(hidden @ weight.T / temperature))`` against a teacher's top logits.

    teacher_logits: ``... x K`` fp32, bf16 or fp16, the logits a teacher kept for each row;
    teacher_index: ``... x K`` int32 or int64, their tokens, in any order; K from 1 to 256. q is the
    softmax of ``teacher_logits / temperature`` (from 2^-20 to 2^20) over the row's entries: those with a negative index
    or a logit of -inf are padding, entries of the same token add up. A row of nothing but padding
    has no loss, like an ignored target in ``linear_cross_entropy``; an index of V or more makes it
    NaN. The teacher gets no gradient. Everything else as in ``linear_cross_entropy``.
    """
    return _call(hidden, weight, teacher_index, teacher_logits,
                 ("hidden", "weight", "teacher_index", "teacher_logits"), 0, reduction, float(temperature))
