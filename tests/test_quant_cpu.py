"""CPU: argument checks of the dense 8-bit product, in the library and in the Python layer."""
import ctypes as C

import pytest
import torch


def test_library_refusals_need_no_gpu(bsx):
    from brainstate_b200._lib import BSX_ERR_INVALID_ARG, BSX_ERR_UNSUPPORTED
    buf = (C.c_char * 64)()
    at = (C.addressof(buf) + 15) // 16 * 16
    assert [bsx.bsx_int8_row_bytes(n) for n in (0, 1, 16, 17, 4096)] == [0, 16, 16, 32, 4096]
    dense = lambda x=at, fmt=0, w=at, m=4, k=8, n=8, out=at, kind=0, ws=None, size=0: bsx.bsx_int8_dense(
        x, fmt, k, w, at, m, k, n, out, kind, ws, size, None)
    for bad in (dict(m=-1), dict(k=-1), dict(n=-1), dict(fmt=5), dict(fmt=-1), dict(kind=3), dict(x=None), dict(w=None),
                dict(out=None), dict(w=at + 4)):
        assert dense(**bad) == BSX_ERR_INVALID_ARG, bad
    for bad in (dict(k=131073), dict(m=2 ** 31), dict(n=2 ** 31), dict(k=0)):
        assert dense(**bad) == BSX_ERR_UNSUPPORTED, bad
    assert dense(m=0) == 0 and dense(n=0) == 0
    mul = lambda q=at, m=4, k=8, n=8, out=at, kind=0: bsx.bsx_int8_matmul(q, at, at, at, m, k, n, out, kind, None, 0, None)
    assert mul(q=None) == BSX_ERR_INVALID_ARG and mul(q=at + 8) == BSX_ERR_INVALID_ARG and mul(kind=4) == BSX_ERR_INVALID_ARG
    assert mul(k=0) == BSX_ERR_UNSUPPORTED and mul(m=0) == 0
    rows = lambda x=at, fmt=0, m=2, k=8, q=at, s=at: bsx.bsx_int8_quantize_rows(x, fmt, k, m, k, q, s, None)
    assert rows(x=None) == rows(fmt=7) == rows(s=None) == rows(q=at + 1) == BSX_ERR_INVALID_ARG
    assert rows(k=131073) == BSX_ERR_UNSUPPORTED and rows(m=0) == 0
    cols = lambda w=at, kind=0, k=8, n=8: bsx.bsx_int8_quantize_weights(w, kind, k, n, at, at, None)
    assert cols(w=None) == cols(kind=3) == BSX_ERR_INVALID_ARG and cols(k=0) == BSX_ERR_UNSUPPORTED and cols(n=0) == 0
    assert bsx.bsx_int8_dense_workspace_bytes(5, 100, 8) >= 5 * 112 + 20
    assert bsx.bsx_int8_dense_workspace_bytes(4, 200000, 8) == 0


def test_python_refuses_cpu_tensors():
    from brainstate_b200 import EventArray, nn, quant
    with pytest.raises(RuntimeError, match='GPU only'):
        quant.Int8Dense(torch.zeros(4, 4))
    with pytest.raises(RuntimeError, match='GPU only'):
        quant.quantize_rows(torch.zeros(4, 4))
    with pytest.raises(RuntimeError, match='GPU only'):
        quant.quantize_rows(EventArray(torch.zeros(4, 4)))
    with pytest.raises(TypeError, match='tensor or an EventArray'):
        quant.quantize_rows([1., 2.])
    with pytest.raises(TypeError, match='Int8Dense'):
        quant.int8_matmul(torch.zeros(4, 4), torch.zeros(4, 4))
    with pytest.raises(RuntimeError, match='GPU only'):
        nn.Int8Linear(4, 4, torch.zeros(4, 4))
