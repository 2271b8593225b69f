"""CPU: argument checks of the gated delta rule, in the library and in the Python layer, and the reference itself."""
import ctypes as C

import pytest
import torch

from plastic_reference import delta_rule as reference
from plastic_reference import inputs


def _desc(**kw):
    from brainstate_b200._lib import BsxDelta
    d = BsxDelta()
    d.batch, d.tokens, d.k_heads, d.v_heads, d.dk, d.dv, d.dtype, d.scale = 2, 100, 1, 2, 64, 32, 0, 1.0
    for n, v in kw.items():
        setattr(d, n, v)
    return d


def test_struct_layout_matches_header(bsx):
    from brainstate_b200._lib import BsxDelta
    assert C.sizeof(BsxDelta) == 2 * 8 + 6 * 4 + 7 * 8 + 15 * 8
    assert BsxDelta.q.offset == 40 and BsxDelta.q_stride.offset == 96


def test_library_refusals_need_no_gpu(bsx):
    from brainstate_b200._lib import BSX_ERR_INVALID_ARG, BSX_ERR_UNSUPPORTED, BSX_ERR_WORKSPACE
    buf = (C.c_float * 8)()
    at = C.addressof(buf)
    full = dict(q=at, k=at, v=at, g=at, beta=at)
    fwd = lambda d, out=at, ws=None, n=0: bsx.bsx_delta_forward(C.byref(d) if d else None, out, None, ws, n, None)
    assert fwd(None) == BSX_ERR_INVALID_ARG
    assert fwd(_desc()) == BSX_ERR_INVALID_ARG and b'NULL input' in bsx.bsx_last_error_string()
    assert fwd(_desc(**full), None) == BSX_ERR_INVALID_ARG and b'out' in bsx.bsx_last_error_string()
    assert fwd(_desc(**full)) == BSX_ERR_WORKSPACE
    for bad in (dict(batch=-1), dict(tokens=-1), dict(dtype=3), dict(k_heads=0), dict(v_heads=3, k_heads=2), dict(dk=0),
                dict(dv=0)):
        assert fwd(_desc(**full, **bad)) == BSX_ERR_INVALID_ARG, bad
    for bad in (dict(dk=129), dict(dv=4097), dict(tokens=2 ** 31), dict(batch=2 ** 31), dict(batch=2 ** 25, tokens=2 ** 12)):
        assert fwd(_desc(**full, **bad)) == BSX_ERR_UNSUPPORTED, bad
    assert fwd(_desc(batch=0)) == 0 and bsx.bsx_delta_recurrent(C.byref(_desc(batch=0)), None, None, None) == 0
    assert bsx.bsx_delta_backward(C.byref(_desc(**full)), None, None, None, None, None, None, None, None, None, 0,
                                  None) == BSX_ERR_INVALID_ARG
    # at least T and P of two chunks of two heads of two rows; reverse mode needs more
    assert bsx.bsx_delta_workspace_bytes(C.byref(_desc())) >= 2 * 2 * 2 * 2 * 36 * 64 * 4
    assert bsx.bsx_delta_backward_workspace_bytes(C.byref(_desc())) > bsx.bsx_delta_workspace_bytes(C.byref(_desc()))
    assert bsx.bsx_delta_workspace_bytes(C.byref(_desc(dk=500))) == 0


def test_python_refuses_cpu_tensors():
    from brainstate_b200 import nn, plastic
    a = list(inputs(1, 4, 1, 1, 8, 8, torch.float32).values())
    with pytest.raises(RuntimeError, match='GPU only'):
        plastic.delta_rule(*a[:5])
    with pytest.raises(RuntimeError, match='GPU only'):
        plastic.delta_rule_step(*(x[:, 0] for x in a[:5]), a[5])
    with pytest.raises(TypeError, match='must be a tensor'):
        plastic.delta_rule_step(*(x[:, 0] for x in a[:5]), None)
    with pytest.raises(ValueError, match='evenly'):
        nn.DeltaSynapse(8, 8, k_heads=2, v_heads=3)


def test_reference_learns_an_association():
    """One key, beta = 1, no decay: the matrix answers the key with the value exactly, whatever it held."""
    k = torch.zeros(1, 1, 1, 4, dtype=torch.float64)
    k[..., 2] = 1.
    v = torch.tensor([3., -1.], dtype=torch.float64).view(1, 1, 1, 2)
    o, s = reference(k, k, v, torch.zeros(1, 1, 1), torch.ones(1, 1, 1), 1.0,
                     torch.randn(1, 1, 4, 2, dtype=torch.float64))
    assert torch.allclose(o, v)
