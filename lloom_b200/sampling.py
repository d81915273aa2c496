"""The next token of every row of logits (``lloom_b200_sample``): what follows the output head's product in a decode step."""
from __future__ import annotations

import torch

from . import _lib
from ._lib import LloomError
from .quantized import _native

MAX_VOCAB = 327680


def sample(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Draws a token per row of ``logits [.., vocab]`` (f32, f16 or bf16, on the GPU) with the uniform numbers ``u`` (f32, the leading
    shape, in [0, 1)).  Returns ``(ids, probs)``: int64 and f32 of the leading shape.

    With w = exp((l - max) / temperature) and the tokens ordered by falling logit, equal ones by index, the kept ones are the
    shortest of the first ``top_k`` (0: all), the first whose weights reach ``top_p`` times those of the first ``top_k``, and those with
    w >= ``min_p``.  The token is the first kept one, by index, whose running sum of weights exceeds u times their sum; its
    probability is its share of that sum.  ``temperature`` 0 takes the first of the largest logits.  A row with nothing above
    -infinity gives -1 and 0; NaN counts as -infinity.

    Each setting is a number, or a tensor on the same GPU with a value per row (f32; ``top_k`` int32)."""
    got = _native().sample(logits, u, temperature, top_k, top_p, min_p)
    if got is None:
        _refuse(logits, u, {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p})
    return got


def _refuse(logits, u, settings):
    if logits.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise LloomError(_lib.ERR_DTYPE, "sample", f"logits are f32, f16 or bf16, not {logits.dtype}")
    if u.dtype != torch.float32:
        raise LloomError(_lib.ERR_DTYPE, "sample", f"u is f32, not {u.dtype}")
    if not logits.is_cuda or u.device != logits.device:
        raise LloomError(_lib.ERR_DEVICE, "sample", f"logits on {logits.device}, u on {u.device}: one GPU is wanted")
    if logits.dim() < 1 or logits.shape[-1] == 0 or u.shape != logits.shape[:-1] or not u.is_contiguous():
        raise LloomError(_lib.ERR_SHAPE, "sample", f"u {tuple(u.shape)} for logits {tuple(logits.shape)}")
    for name, v in settings.items():
        if not isinstance(v, torch.Tensor):
            continue
        want = torch.int32 if name == "top_k" else torch.float32
        if v.dtype != want:
            raise LloomError(_lib.ERR_DTYPE, "sample", f"{name} is {want}, not {v.dtype}")
        if v.device != logits.device:
            raise LloomError(_lib.ERR_DEVICE, "sample", f"{name} on {v.device}, logits on {logits.device}")
        if v.numel() != u.numel() or not v.is_contiguous():
            raise LloomError(_lib.ERR_SHAPE, "sample", f"{name} {tuple(v.shape)} for {u.numel()} rows")
    raise LloomError(_lib.ERR_SHAPE, "sample", "logits have contiguous rows")
