"""RMS norm in front of the quantized matmuls: the residual's addition, the norm, and its output as the activation blocks
that the products read, in one launch (``lloom_b200_rms_norm``)."""
from __future__ import annotations

import torch

from . import _lib
from ._lib import LloomError
from .quantized import GgmlDType, QActs, _native, act_type


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, residual: torch.Tensor | None = None,
             act_for: GgmlDType | None = None):
    """``h = x + residual`` (in x's type), ``y = h / sqrt(mean(h^2) + eps) * weight`` over the last dimension.

    Returns ``y``, or ``(y, h)`` where a residual is given.  ``y`` has x's type; with ``act_for``, the dtype of the weights that
    read it next, it is a ``QActs`` of their block type instead, for ``QMatMul.forward_quantized`` and ``forward_group``.
    ``x`` and ``residual`` are f32, f16 or bf16, of one type and shape, contiguous or matrices with contiguous rows; ``weight``
    has any of the three types.  The blocks are those of the f32 values of ``y``, whose every rounding is defined but the last bits
    of a 64-bit sum: a row has the same blocks in every batch, but for about one in 10^8, whose 1 / sqrt lies on the border of two
    f32 values."""
    act = None if act_for is None else act_type(act_for)
    got = _native().rms_norm(x, weight, eps, residual, -1 if act is None else act)
    if got is None:
        _refuse(x, weight, residual, act_for)
    if act is None:
        return got
    shape = tuple(x.shape)
    if residual is None:
        return QActs._own(got, act, shape)
    return QActs._own(got[0], act, shape), got[1]


def _refuse(x, weight, residual, act_for):
    types = (torch.float32, torch.float16, torch.bfloat16)
    given = [("x", x), ("weight", weight)] + ([] if residual is None else [("residual", residual)])
    for name, t in given:
        if not isinstance(t, torch.Tensor) or t.dtype not in types:
            raise LloomError(_lib.ERR_DTYPE, "rms_norm", f"{name} is f32, f16 or bf16")
    for name, t in given:
        if t.device != x.device or not t.is_cuda:
            raise LloomError(_lib.ERR_DEVICE, "rms_norm", f"{name} is on {t.device}, x on {x.device}: one GPU is wanted")
    if residual is not None and (residual.dtype != x.dtype or residual.shape != x.shape):
        raise LloomError(_lib.ERR_SHAPE, "rms_norm", f"residual {tuple(residual.shape)} {residual.dtype} for x {tuple(x.shape)} {x.dtype}")
    if x.dim() < 1 or weight.shape != x.shape[-1:] or x.shape[-1] == 0:
        raise LloomError(_lib.ERR_SHAPE, "rms_norm", f"weight {tuple(weight.shape)} for x {tuple(x.shape)}")
    if act_for is not None and x.shape[-1] % act_type(act_for).block_size() != 0:
        raise LloomError(_lib.ERR_SHAPE, "rms_norm", f"rows of {x.shape[-1]} elements are no whole {act_type(act_for)!r} blocks")
    raise LloomError(_lib.ERR_SHAPE, "rms_norm", "x, residual and weight have contiguous rows")
