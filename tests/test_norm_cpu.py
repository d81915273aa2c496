"""Refusals of the norm and of the products that read blocks: nothing is launched."""
import ctypes as C

import pytest
import torch


def test_c_entry_refuses(cuda_lib):
    from lloom_b200 import _lib

    L = cuda_lib
    buf = (C.c_uint8 * 8192)()
    p = (C.addressof(buf) + 15) & ~15

    def norm(x=p, r=None, w=p, xt=0, wt=0, m=1, k=256, ldx=256, ldr=0, h=None, y=p, yt=0):
        return L.lloom_b200_rms_norm(x, r, w, xt, wt, 1e-5, m, k, ldx, ldr, h, y, yt, None)

    assert norm(xt=8) == _lib.ERR_DTYPE and norm(wt=2) == _lib.ERR_DTYPE
    assert norm(yt=1) == _lib.ERR_DTYPE  # y has x's type, or is blocks
    assert norm(yt=12) == _lib.ERR_DTYPE  # weights' type, not the activations'
    for bad in ({"m": 0}, {"k": 0}, {"ldx": 255}, {"r": p, "h": p, "ldr": 255}, {"k": 255, "yt": 8}, {"k": 224, "yt": 15}, {"k": 1 << 25, "ldx": 1 << 25}):
        assert norm(**bad) == _lib.ERR_SHAPE, bad
    for bad in ({"x": None}, {"w": None}, {"y": None}, {"r": p, "ldr": 256}):
        assert norm(**bad) == _lib.ERR_NULL, bad
    for bad in ({"x": p + 2}, {"w": p + 1}, {"y": p + 2}, {"r": p + 1, "h": p, "ldr": 256}, {"y": p + 2, "yt": 15}):
        assert norm(**bad) == _lib.ERR_ALIGN, bad
    assert L.lloom_b200_dequantize_act(12, p, 256, p, None) == _lib.ERR_DTYPE
    assert L.lloom_b200_dequantize_act(15, p, 32, p, None) == _lib.ERR_SHAPE
    assert L.lloom_b200_dequantize_act(8, None, 32, p, None) == _lib.ERR_NULL
    assert L.lloom_b200_dequantize_act(8, p, 32, p + 4, None) == _lib.ERR_ALIGN


def test_products_of_blocks_refuse(cuda_lib):
    from lloom_b200 import _lib

    L = cuda_lib
    buf = (C.c_uint8 * 65536)()
    p = (C.addressof(buf) + 1023) & ~1023

    def fwd(dt=12, w=p, img=None, act=p, y=p, yt=0, m=1, n=4, k=256, ldy=4, ws=p, nb=60000):
        return L.lloom_b200_qmatmul_fwd_acts(dt, w, img, act, y, yt, m, n, k, ldy, ws, nb, None)

    assert fwd(dt=3) == _lib.ERR_DTYPE and fwd(yt=8) == _lib.ERR_DTYPE
    assert fwd(k=100) == _lib.ERR_SHAPE and fwd(ldy=3) == _lib.ERR_SHAPE and fwd(m=0) == _lib.ERR_SHAPE
    assert fwd(w=None) == _lib.ERR_NULL and fwd(act=None) == _lib.ERR_NULL and fwd(y=None) == _lib.ERR_NULL
    assert fwd(ws=None) == _lib.ERR_WORKSPACE and fwd(nb=16) == _lib.ERR_WORKSPACE
    assert fwd(act=p + 2) == _lib.ERR_ALIGN and fwd(w=p + 8) == _lib.ERR_ALIGN and fwd(img=p + 16, m=9) == _lib.ERR_ALIGN

    vp, i64 = C.c_void_p * 1, C.c_int64 * 1
    def group(act=p, m=1, stores=None, nb=60000):
        return L.lloom_b200_qmatmul_fwd_acts_group(12, 1, vp(p), act, vp(p), i64(4), i64(4), stores, m, 256, p, nb, None)

    assert group(act=None) == _lib.ERR_NULL and group(m=9) == _lib.ERR_SHAPE and group(act=p + 2) == _lib.ERR_ALIGN
    assert group(stores=(C.c_int * 1)(3)) == _lib.ERR_SHAPE and group(nb=16) == _lib.ERR_WORKSPACE


def test_python_refuses(cuda_lib):
    from lloom_b200 import GgmlDType, LloomError, QActs, QCudaStorage, QMatMul, QTensor, _lib, rms_norm
    from lloom_b200.quantized import forward_group

    x, w = torch.zeros(2, 256), torch.ones(256)

    def status(fn, *a, **kw):
        with pytest.raises(LloomError) as e:
            fn(*a, **kw)
        return e.value.status

    assert status(rms_norm, x, w) == _lib.ERR_DEVICE
    assert status(rms_norm, x.int(), w) == _lib.ERR_DTYPE
    assert status(rms_norm, x, w.double()) == _lib.ERR_DTYPE
    assert status(rms_norm, x, w, act_for=GgmlDType.Q8K) == _lib.ERR_DTYPE  # not a weight type
    assert status(QActs, torch.zeros(2, 33, dtype=torch.uint8), GgmlDType.Q8_0) == _lib.ERR_SHAPE
    assert status(QActs, torch.zeros(2, 34), GgmlDType.Q8_0) == _lib.ERR_SHAPE
    assert status(QActs, torch.zeros(2, 144, dtype=torch.uint8), GgmlDType.Q4K) == _lib.ERR_DTYPE
    acts = QActs(torch.zeros(2, 292, dtype=torch.uint8), GgmlDType.Q8K)
    assert acts.shape == (2, 256)
    assert status(acts.dequantize) == _lib.ERR_SHAPE
    mm = QMatMul(QTensor(QCudaStorage.load_quantized("cpu", bytes(144 * 4), GgmlDType.Q4K), (4, 256)))
    assert status(mm.forward_quantized, QActs(torch.zeros(2, 34 * 8, dtype=torch.uint8), GgmlDType.Q8_0)) == _lib.ERR_SHAPE
    assert status(mm.forward_quantized, QActs(torch.zeros(2, 584, dtype=torch.uint8), GgmlDType.Q8K)) == _lib.ERR_SHAPE
    assert status(mm.forward_quantized, acts, torch.float64) == _lib.ERR_DTYPE
    assert status(mm.forward_quantized, QActs(torch.zeros(4, 292, dtype=torch.uint8)[::2], GgmlDType.Q8K)) == _lib.ERR_SHAPE
    assert status(forward_group, [mm], QActs(torch.zeros(2, 34 * 8, dtype=torch.uint8), GgmlDType.Q8_0)) == _lib.ERR_SHAPE


def test_stream_in_place_needs_rows_that_follow_each_other(cuda_lib):
    """h is contiguous: in the residual's own buffer its rows would run over those of a wider residual before they are read."""
    from lloom_b200 import _lib

    p = 1 << 20
    assert _lib.lib().lloom_b200_rms_norm(p, p + 65536, p, 0, 0, 1e-5, 4, 64, 64, 80, p + 65536, p + 131072, 0, None) == _lib.ERR_SHAPE


def test_blocks_of_values_refuse(cuda_lib):
    """The quantizer reads f32: of anything else it would read past the end."""
    from lloom_b200 import GgmlDType, LloomError, QActs, _lib
    from lloom_b200.quantized import quantize_act

    for x, want in ((torch.zeros(2, 256, dtype=torch.float16), _lib.ERR_DTYPE), (torch.zeros(2, 256, dtype=torch.bfloat16), _lib.ERR_DTYPE),
                    (torch.zeros(2, 256, dtype=torch.int8), _lib.ERR_DTYPE), (torch.zeros(2, 256), _lib.ERR_DEVICE)):
        for fn in (lambda: QActs.quantize(x, GgmlDType.Q4K), lambda: quantize_act(GgmlDType.Q8_0, x)):
            with pytest.raises(LloomError) as e:
                fn()
            assert e.value.status == want, x.dtype


def test_stacks_of_experts_are_no_matrices(cuda_lib):
    """[8, 256, 256]: its first two extents look like an [n, k] that fits the input."""
    from lloom_b200 import GgmlDType, LloomError, QActs, QCudaStorage, QMatMul, QTensor, _lib
    from lloom_b200.quantized import forward_group

    mm = QMatMul(QTensor(QCudaStorage.load_quantized("cpu", bytes(144 * 8 * 256), GgmlDType.Q4K), (8, 256, 256)))
    acts = QActs(torch.zeros(2, 292, dtype=torch.uint8), GgmlDType.Q8K)
    for fn in (lambda: mm.forward_quantized(acts), lambda: forward_group([mm], acts), lambda: forward_group([mm], torch.zeros(2, 256))):
        with pytest.raises(LloomError) as e:
            fn()
        assert e.value.status == _lib.ERR_SHAPE and "[n, k]" in str(e.value)


def test_group_refuses_destinations_that_do_not_fit(cuda_lib):
    """Every destination is written as f32 rows of n: another type, device or size would be written past its end."""
    from lloom_b200 import GgmlDType, LloomError, QActs, QCudaStorage, QMatMul, QTensor, _lib
    from lloom_b200.quantized import forward_group

    mm = QMatMul(QTensor(QCudaStorage.load_quantized("cpu", bytes(144 * 4), GgmlDType.Q4K), (4, 256)))
    for x in (torch.zeros(2, 256), QActs(torch.zeros(2, 292, dtype=torch.uint8), GgmlDType.Q8K)):
        for out in (torch.zeros(2, 4, dtype=torch.float16), torch.zeros(1, 4), torch.zeros(2, 5), torch.zeros(8), torch.zeros(2, 8)[:, ::2], torch.zeros(4, 2).t(),
                    torch.zeros(1, 4).expand(2, 4), torch.zeros(2, 4, device="meta"), None):
            with pytest.raises(LloomError) as e:
                forward_group([mm], x, outs=[out])
            assert e.value.status == _lib.ERR_SHAPE
        with pytest.raises(LloomError) as e:
            forward_group([mm], x, stores=[2])
        assert e.value.status == _lib.ERR_NULL
