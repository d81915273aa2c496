"""Microscaled 4-bit floating point (OCP MX: E2M1 elements, one E8M0 scale per 32 elements of a row): weights in that format
and the product that quantizes its activations to it, on the tensor cores' block-scaled instructions.

The format of GGUF type 39 (MXFP4), which the reference reads but refuses on CUDA (``lloom-tensor/src/quantized/mod.rs:206-221``).
Beside ``QTensor`` / ``QMatMul``, whose products keep the activations in 8 bits."""
from __future__ import annotations

from typing import Sequence

import numpy as np
import torch

from . import _lib
from ._lib import LloomError
from .quantized import _native

MX_BLOCK, MX_BLOCK_BYTES = 32, 17


class MxTensor:
    """A matrix ``[n, k]`` of microscaled 4-bit values on the GPU, k a multiple of 32, laid out for the tensor cores (4.25 bits
    an element, rows padded to 128 and k to 256)."""

    __slots__ = ("_native",)

    def __init__(self, native):
        self._native = native

    @property
    def shape(self) -> tuple:
        return self._native.shape()

    @classmethod
    def quantize(cls, src: torch.Tensor) -> "MxTensor":
        """Values ``[.., k]`` (f32, f16 or bf16, on the GPU, contiguous) to the nearest codes under the scale 2^(floor(log2 max) - 2)
        of their block; leading dimensions become rows.  A block with a NaN or an infinity becomes NaN."""
        st = _native().mx_quantize(src)
        if st is None:
            _refuse("MxTensor.quantize", src, src.shape[-1] if src.dim() else 0, None)
        return cls(st)

    @classmethod
    def from_data(cls, data, shape: Sequence[int], device="cuda") -> "MxTensor":
        """From a file's MXFP4 blocks (17 bytes per 32 elements): bytes, an array, or a uint8 tensor on either side."""
        shape = tuple(int(s) for s in shape)
        device = torch.device(device)
        if len(shape) != 2 or min(shape) <= 0 or shape[1] % MX_BLOCK != 0:
            raise LloomError(_lib.ERR_SHAPE, "MxTensor.from_data", f"shape {shape} is not [n, k] with k a multiple of {MX_BLOCK}")
        if isinstance(data, torch.Tensor):
            if data.dtype != torch.uint8:
                raise LloomError(_lib.ERR_DTYPE, "MxTensor.from_data", f"blocks are bytes, not {data.dtype}")
            blocks = data.contiguous().reshape(-1)
        else:
            host = np.frombuffer(data, dtype=np.uint8) if isinstance(data, (bytes, bytearray, memoryview)) else np.asarray(data, np.uint8)
            blocks = torch.from_numpy(np.array(host).reshape(-1))
        want = shape[0] * shape[1] // MX_BLOCK * MX_BLOCK_BYTES
        if blocks.numel() != want:
            raise LloomError(_lib.ERR_SHAPE, "MxTensor.from_data", f"{blocks.numel()} bytes, shape {shape} needs {want}")
        if device.type != "cuda":
            raise LloomError(_lib.ERR_DEVICE, "MxTensor.from_data", f"{device} is not a GPU")
        blocks = blocks.to(device)
        st = _native().mx_from_blocks(blocks, shape)
        if st is None:
            raise LloomError(_lib.ERR_SHAPE, "MxTensor.from_data", f"unsupported shape {shape}")
        return cls(st)

    def device(self) -> torch.device:
        return self._native.device()

    def storage_size_in_bytes(self) -> int:
        """Of the blocks; the image takes the padding on top."""
        n, k = self.shape
        return n * k // MX_BLOCK * MX_BLOCK_BYTES

    def data(self) -> bytes:
        """The blocks as a file stores them."""
        return self._native.to_blocks().cpu().numpy().tobytes()

    def dequantize(self) -> torch.Tensor:
        return self._native.dequantize(False)

    def dequantize_f16(self) -> torch.Tensor:
        return self._native.dequantize(True)


class MxMatMul:
    """``forward(xs) = xs @ W^T`` over an ``MxTensor``, the activations quantized to the same format on the way."""

    def __init__(self, tensor: MxTensor):
        if not isinstance(tensor, MxTensor):
            raise LloomError(_lib.ERR_DTYPE, "MxMatMul", f"{type(tensor).__name__} is not an MxTensor")
        self.tensor = tensor

    @classmethod
    def from_tensor(cls, tensor: MxTensor) -> "MxMatMul":
        return cls(tensor)

    def forward(self, xs: torch.Tensor) -> torch.Tensor:
        """``xs [.., k]`` f32, f16 or bf16, contiguous, any number of rows; ``[.., n]`` of xs's type.  Products are exact and summed
        in f32."""
        y = self.tensor._native.forward(xs)
        if y is None:
            _refuse("MxMatMul.forward", xs, self.tensor.shape[1], self.tensor.device())
        return y

    __call__ = forward


def _refuse(where, x, k, device):
    if x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise LloomError(_lib.ERR_DTYPE, where, f"values are f32, f16 or bf16, not {x.dtype}")
    if not x.is_cuda or (device is not None and x.device != device):
        raise LloomError(_lib.ERR_DEVICE, where, f"input on {x.device}, wanted on {device or 'a GPU'}")
    if x.dim() < 2:
        raise LloomError(_lib.ERR_SHAPE, where, f"input tensor has only one dimension {tuple(x.shape)}")
    if not x.is_contiguous():
        raise LloomError(_lib.ERR_SHAPE, where, f"input tensor is not contiguous {tuple(x.shape)}")
    if x.shape[-1] != k:
        raise LloomError(_lib.ERR_SHAPE, where, f"input tensor {tuple(x.shape)} incompatible with rows of {k}")
    raise LloomError(_lib.ERR_SHAPE, where, f"unsupported shape {tuple(x.shape)}: rows of a multiple of {MX_BLOCK} elements, at least one")
