"""Refusals of the microscaled entries, and MXFP4 tensors in a GGUF header: nothing is launched."""
import ctypes as C
import io

import pytest
import torch


def test_c_entries_refuse(cuda_lib):
    from lloom_b200 import _lib

    L = cuda_lib
    buf = (C.c_uint8 * (1 << 17))()
    p = (C.addressof(buf) + 1023) & ~1023
    big = 1 << 16
    assert L.lloom_b200_mx_image_bytes(1, 32) == 128 * 128 + 1024
    assert L.lloom_b200_mx_image_bytes(129, 288) == 4 * (128 * 128 + 1024)
    assert L.lloom_b200_mx_image_bytes(1, 31) == 0 and L.lloom_b200_mx_image_bytes(0, 32) == 0 and L.lloom_b200_mx_image_bytes(4, 1 << 25) == 0
    assert L.lloom_b200_mx_workspace_bytes(1, 8, 256) > 0 and L.lloom_b200_mx_workspace_bytes(1, 8, 100) == 0
    for bad in ((0, 32), (4, 0), (4, 48), (1 << 31, 32)):
        assert L.lloom_b200_mx_quantize(p, 0, *bad, p, big, None) == _lib.ERR_SHAPE, bad
        assert L.lloom_b200_mx_from_blocks(p, *bad, p, big, None) == _lib.ERR_SHAPE, bad
        assert L.lloom_b200_mx_to_blocks(p, *bad, p, None) == _lib.ERR_SHAPE, bad
        assert L.lloom_b200_mx_dequantize(p, *bad, p, 0, None) == _lib.ERR_SHAPE, bad
    assert L.lloom_b200_mx_quantize(p, 8, 1, 32, p, big, None) == _lib.ERR_DTYPE
    assert L.lloom_b200_mx_quantize(None, 0, 1, 32, p, big, None) == _lib.ERR_NULL
    assert L.lloom_b200_mx_quantize(p, 0, 1, 32, p, 100, None) == _lib.ERR_WORKSPACE
    assert L.lloom_b200_mx_quantize(p + 4, 0, 1, 32, p, big, None) == _lib.ERR_ALIGN
    assert L.lloom_b200_mx_quantize(p, 0, 1, 32, p + 16, big, None) == _lib.ERR_ALIGN
    assert L.lloom_b200_mx_from_blocks(p, 1, 32, p, 100, None) == _lib.ERR_WORKSPACE
    assert L.lloom_b200_mx_from_blocks(p, 1, 32, None, big, None) == _lib.ERR_NULL
    assert L.lloom_b200_mx_dequantize(p, 1, 32, p + 4, 0, None) == _lib.ERR_ALIGN

    def fwd(img=p, x=p, xt=0, y=p, yt=0, m=1, n=4, k=256, ldy=4, ws=p, nb=big):
        return L.lloom_b200_mx_fwd(img, x, xt, y, yt, m, n, k, ldy, ws, nb, None)

    assert fwd(k=100) == _lib.ERR_SHAPE and fwd(m=0) == _lib.ERR_SHAPE and fwd(ldy=3) == _lib.ERR_SHAPE
    assert fwd(xt=8) == _lib.ERR_DTYPE and fwd(yt=39) == _lib.ERR_DTYPE
    assert fwd(img=None) == _lib.ERR_NULL and fwd(x=None) == _lib.ERR_NULL and fwd(y=None) == _lib.ERR_NULL
    assert fwd(ws=None) == _lib.ERR_WORKSPACE and fwd(nb=8) == _lib.ERR_WORKSPACE
    assert fwd(x=p + 8) == _lib.ERR_ALIGN and fwd(img=p + 16) == _lib.ERR_ALIGN and fwd(ws=p + 16) == _lib.ERR_ALIGN and fwd(y=p + 2) == _lib.ERR_ALIGN


def test_python_refuses(cuda_lib):
    from lloom_b200 import LloomError, MxTensor, _lib

    def status(fn, *a):
        with pytest.raises(LloomError) as e:
            fn(*a)
        return e.value.status

    assert status(MxTensor.quantize, torch.zeros(2, 32)) == _lib.ERR_DEVICE
    assert status(MxTensor.quantize, torch.zeros(2, 32, dtype=torch.int32)) == _lib.ERR_DTYPE
    assert status(MxTensor.from_data, bytes(17), (1, 32), "cpu") == _lib.ERR_DEVICE
    assert status(MxTensor.from_data, bytes(16), (1, 32)) == _lib.ERR_SHAPE
    assert status(MxTensor.from_data, bytes(17), (1, 31)) == _lib.ERR_SHAPE
    assert status(MxTensor.from_data, bytes(17), (32,)) == _lib.ERR_SHAPE
    assert status(MxTensor.from_data, torch.zeros(17), (1, 32)) == _lib.ERR_DTYPE


def test_gguf_lists_mxfp4():
    from lloom_b200 import gguf_file as G

    f = io.BytesIO()
    data = bytes(range(34))
    G.write(f, [], [("w", G.MXFP4, (2, 32), data)])
    c = G.Content.read(io.BytesIO(f.getvalue()))
    assert c.tensor_infos["w"].size_in_bytes() == 34
    assert bytes(c.tensor_infos["w"].read_bytes(io.BytesIO(f.getvalue()), c.tensor_data_offset).numpy()) == data


def test_products_take_their_own_tensors(cuda_lib):
    """A GGUF file's tensors are of two kinds: the product of the other kind refuses one at once, not at its first forward."""
    from lloom_b200 import GgmlDType, LloomError, MxMatMul, MxTensor, QCudaStorage, QMatMul, QTensor, _lib

    q, mx = QTensor(QCudaStorage.load_quantized("cpu", bytes(144 * 4), GgmlDType.Q4K), (4, 256)), MxTensor(None)
    assert QMatMul.from_qtensor(q).qtensor is q and MxMatMul.from_tensor(mx).tensor is mx
    for fn, other in ((QMatMul, mx), (QMatMul.from_qtensor, mx), (QMatMul.from_arc, mx), (MxMatMul, q), (MxMatMul.from_tensor, q)):
        with pytest.raises(LloomError) as e:
            fn(other)
        assert e.value.status == _lib.ERR_DTYPE
