"""The Python module between operators and entry points: what it is not given on a GPU, or not given at all, it leaves to others."""
import ctypes

import pytest
import torch

import _paged_oracle as oracle
from ghost_flow_b200.ops import _lib
from ghost_flow_b200.ops.fused import follows


def _args():
    s = oracle.batch([7, 20], [1, 2], 4, 2, 64, 16)
    return s["q"], s["kp"], s["vp"], s["table"], s["lens"], s["cu"]


def test_tensors_of_the_host_are_not_the_kernels():
    calls, (q, k, v, table, lens, cu), t = _lib.calls(), _args(), torch.zeros(8, 32)
    assert calls.attention(q, k, v, table, lens, cu) is None
    assert calls.append(torch.zeros(3, 8, 64).bfloat16(), 4, 2, k, v, table, lens, cu, t, t) is None
    assert calls.logits(torch.zeros(2, 9), None, None, None, 1.0, 0.0, 0, None, None) is None


@pytest.mark.parametrize("at", range(6))
@pytest.mark.parametrize("what", [None, 3, "text", torch.eye(3).to_sparse(), torch.zeros(2, device="meta")], ids=["none", "int", "str", "sparse", "meta"])
def test_what_is_no_tensor_with_memory(at, what):
    a = list(_args())
    a[at] = what
    assert _lib.calls().attention(*a) is None


def test_wrong_numbers_of_arguments_and_what_is_no_call():
    calls = _lib.calls()
    for f in (calls.bind, calls.append, calls.attention, calls.logits, calls.run_append, calls.run_attention, calls.run_logits):
        with pytest.raises(TypeError, match="arguments"):
            f(1)
    y = torch.zeros(2)
    for f, n in ((calls.run_append, 5), (calls.run_attention, 9), (calls.run_logits, 4)):
        for call in (None, b"", b"x" * 100, y):
            with pytest.raises(TypeError, match="not a call"):
                f(call, y, *[0] * (n - 2))
    with pytest.raises(TypeError):
        calls.append(y, "4", 2, *[y] * 7)


def test_other_versions_of_the_exchange_interface_are_refused():
    new = ctypes.pythonapi.PyCapsule_New
    new.restype, new.argtypes = ctypes.py_object, [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_void_p]
    table = (ctypes.c_uint32 * 16)(2, 0)
    with pytest.raises(RuntimeError, match="version 2"):
        _lib.calls().bind(new(ctypes.addressof(table), b"dlpack_exchange_api", None), 1, 1, 1, 1, *follows())
    with pytest.raises(ValueError):
        _lib.calls().bind(new(ctypes.addressof(table), b"another", None), 1, 1, 1, 1, *follows())
