"""What the recurrence with a rest refuses (no GPU needed)."""
import ctypes as C

import torch
import pytest

from isaacgym_amd import _abi, _lib, ops
from tests.test_sequence_host import FAKE, rec


def test_refusals():
    L = _lib.lib()
    rest, none = _abi.RecurrenceRest(codes=FAKE, stride=(16, 8)), _abi.RecurrenceRest()
    g = _abi.RecurrenceGrad(d_gate=FAKE, d_gate_stride=(16, 8))
    for dtype, r, code in ((_abi.IGX_F32, rest, _abi.IGX_E_PARAM), (_abi.IGX_BF16, none, _abi.IGX_E_NULL), (_abi.IGX_F16, none, _abi.IGX_E_NULL),
                           (7, rest, _abi.IGX_E_PARAM)):
        assert L.igx_linear_recurrence_with_rest(C.byref(rec(dtype=dtype)), C.byref(r), None) == code
        assert b"igx_linear_recurrence_with_rest" in L.igx_last_error_string()
        assert L.igx_linear_recurrence_backward_with_rest(C.byref(rec(dtype=dtype)), C.byref(g), C.byref(r), None) == code
    assert L.igx_linear_recurrence_with_rest(None, C.byref(rest), None) == _abi.IGX_E_NULL
    # nothing to do
    bf16 = dict(dtype=_abi.IGX_BF16)
    assert L.igx_linear_recurrence_with_rest(C.byref(rec(envs=0, **bf16)), C.byref(none), None) == _abi.IGX_OK
    assert L.igx_linear_recurrence_backward_with_rest(C.byref(rec(**bf16)), C.byref(_abi.RecurrenceGrad()), C.byref(none), None) == _abi.IGX_OK


def test_struct_layout_matches_the_header(tmp_path):
    import os
    import subprocess
    (tmp_path / "s.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "igx.h"\nint main(void){printf("%zu %zu %zu", '
                                  'sizeof(igx_recurrence_rest), offsetof(igx_recurrence_rest, codes), offsetof(igx_recurrence_rest, stride));'
                                  'return 0;}\n')
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.check_call(["gcc", "-I", inc, str(tmp_path / "s.c"), "-o", str(tmp_path / "s")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "s")]).split()]
    assert got == [C.sizeof(_abi.RecurrenceRest), _abi.RecurrenceRest.codes.offset, _abi.RecurrenceRest.stride.offset]


def test_host_tensors_are_refused():
    x = torch.zeros(3, 2, 4, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device tensors only"):
        ops.linear_recurrence(x, x, x.clone(), rest=torch.zeros(3, 2, 4, dtype=torch.int8))
