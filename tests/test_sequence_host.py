"""What the sequence operators refuse, and the plain forms that the GPU tests compare with (no GPU needed)."""
import ctypes as C

import pytest
import torch

from isaacgym_amd import _abi, _lib, ops, sequence
from tests import seq_cases as S

FAKE = 4096  # a non-NULL address: the refused calls return before any launch


def rec(**kw):
    base = dict(dtype=_abi.IGX_F32, steps=4, envs=2, width=8, gate=FAKE, gate_stride=(16, 8, 1), inp=FAKE, inp_stride=(16, 8),
                out=FAKE, out_stride=(16, 8))
    return _abi.Recurrence(**{**base, **kw})


def norm(**kw):
    base = dict(dtype=_abi.IGX_F32, activation=_abi.IGX_GATE_SILU, rows=4, width=8, eps=1e-5, x=FAKE, x_stride=8, y=FAKE,
                y_stride=8, weight=FAKE, next_weight=FAKE, out=FAKE, next=FAKE, y_inv_rms=FAKE, out_inv_rms=FAKE)
    return _abi.BlockNorm(**{**base, **kw})


@pytest.mark.parametrize("change,code", [
    (dict(dtype=3), _abi.IGX_E_PARAM), (dict(dtype=-1), _abi.IGX_E_PARAM), (dict(steps=-1), _abi.IGX_E_SIZE),
    (dict(envs=-2), _abi.IGX_E_SIZE), (dict(width=-8), _abi.IGX_E_SIZE), (dict(envs=1 << 20, width=1 << 20), _abi.IGX_E_SIZE),
    (dict(gate_stride=(16, 8, 2)), _abi.IGX_E_PARAM), (dict(gate=None), _abi.IGX_E_NULL), (dict(out=None), _abi.IGX_E_NULL)])
def test_recurrence_refusals(change, code):
    L = _lib.lib()
    r, g = rec(**change), _abi.RecurrenceGrad(d_gate=FAKE, d_gate_stride=(16, 8))
    assert L.igx_linear_recurrence(C.byref(r), None) == code
    assert b"igx_linear_recurrence" in L.igx_last_error_string()
    assert L.igx_linear_recurrence_backward(C.byref(r), C.byref(g), None) == code
    if "gate" not in change and "out" not in change:
        assert L.igx_linear_recurrence_workspace(C.byref(r)) == code


def test_recurrence_null_structs_and_nothing_to_do():
    L = _lib.lib()
    assert L.igx_linear_recurrence(None, None) == _abi.IGX_E_NULL
    assert L.igx_linear_recurrence_backward(C.byref(rec()), None, None) == _abi.IGX_E_NULL
    assert L.igx_linear_recurrence_workspace(None) == _abi.IGX_E_NULL
    assert L.igx_linear_recurrence(C.byref(rec(inp=None)), None) == _abi.IGX_E_NULL
    for kw in (dict(envs=0), dict(width=0), dict(steps=0)):  # no channels, or no steps and no carried value asked for
        assert L.igx_linear_recurrence(C.byref(rec(gate=None, inp=None, out=None, **kw)), None) == _abi.IGX_OK
    assert L.igx_linear_recurrence_backward(C.byref(rec()), C.byref(_abi.RecurrenceGrad()), None) == _abi.IGX_OK


@pytest.mark.parametrize("change,code", [
    (dict(dtype=9), _abi.IGX_E_PARAM), (dict(rows=-1), _abi.IGX_E_SIZE), (dict(width=0), _abi.IGX_E_SIZE),
    (dict(width=8193), _abi.IGX_E_SIZE), (dict(activation=3), _abi.IGX_E_PARAM), (dict(y=None, next_weight=None), _abi.IGX_E_NULL),
    (dict(y=None, weight=None, gate=FAKE), _abi.IGX_E_PARAM), (dict(weight=None), _abi.IGX_E_NULL),
    (dict(x_stride=-8), _abi.IGX_E_PARAM), (dict(eps=-1e-5), _abi.IGX_E_PARAM), (dict(eps=float("nan")), _abi.IGX_E_PARAM), (dict(y8=FAKE), _abi.IGX_E_NULL), (dict(x=None), _abi.IGX_E_NULL),
    (dict(gate=FAKE, gate_stride=8, y8=FAKE, y8_scale=FAKE), _abi.IGX_E_PARAM)])
def test_block_norm_refusals(change, code):
    L = _lib.lib()
    b = norm(**change)
    g = _abi.BlockNormGrad(d_out=FAKE, d_out_stride=8, d_x=FAKE)
    assert L.igx_block_norm_forward(C.byref(b), None) == code
    assert L.igx_block_norm_backward(C.byref(b), C.byref(g), None) == code


@pytest.mark.parametrize("b,g,code", [
    (dict(), dict(d_out_stride=-1, d_x=FAKE), _abi.IGX_E_PARAM),
    (dict(), dict(d_gate=FAKE), _abi.IGX_E_PARAM),
    (dict(next_weight=None), dict(d_next_weight=FAKE), _abi.IGX_E_PARAM),
    (dict(y=None, weight=None), dict(d_y=FAKE), _abi.IGX_E_PARAM),
    (dict(), dict(d_weight=FAKE), _abi.IGX_E_NULL),
    (dict(), dict(d_weight=FAKE, workspace=FAKE + 8, workspace_bytes=1 << 20), _abi.IGX_E_ALIGN),
    (dict(), dict(d_weight=FAKE, workspace=FAKE, workspace_bytes=16), _abi.IGX_E_SIZE),
    (dict(y_inv_rms=None), dict(d_y=FAKE), _abi.IGX_E_NULL),
    (dict(out_inv_rms=None), dict(d_y=FAKE), _abi.IGX_E_NULL)])
def test_block_norm_backward_refusals(b, g, code):
    assert _lib.lib().igx_block_norm_backward(C.byref(norm(**b)), C.byref(_abi.BlockNormGrad(**g)), None) == code


def test_block_norm_nothing_to_do_and_null():
    L = _lib.lib()
    assert L.igx_block_norm_forward(None, None) == _abi.IGX_E_NULL
    assert L.igx_block_norm_backward(C.byref(norm()), None, None) == _abi.IGX_E_NULL
    assert L.igx_block_norm_workspace(None) == _abi.IGX_E_NULL
    assert L.igx_block_norm_forward(C.byref(norm(rows=0, x=None, out=None, next=None)), None) == _abi.IGX_OK
    assert L.igx_block_norm_backward(C.byref(norm()), C.byref(_abi.BlockNormGrad(d_out=FAKE)), None) == _abi.IGX_OK
    assert L.igx_block_norm_workspace(C.byref(norm())) > 0


def test_pack8_refusals():
    L = _lib.lib()
    assert L.igx_pack8(FAKE, 7, 4, 8, 8, FAKE, FAKE, None) == _abi.IGX_E_PARAM
    assert L.igx_pack8(FAKE, 0, -4, 8, 8, FAKE, FAKE, None) == _abi.IGX_E_SIZE
    assert L.igx_pack8(FAKE, 0, 4, 8, -8, FAKE, FAKE, None) == _abi.IGX_E_PARAM
    assert L.igx_pack8(FAKE, 0, 1 << 40, 1 << 40, 8, FAKE, FAKE, None) == _abi.IGX_E_SIZE
    for i in (0, 1, 2):
        args = [None if j == i else FAKE for j in range(3)]
        assert L.igx_pack8(args[0], 0, 4, 8, 8, args[1], args[2], None) == _abi.IGX_E_NULL
        assert L.igx_unpack8(args[0], args[1], 0, 4, 8, args[2], None) == _abi.IGX_E_NULL
    assert L.igx_unpack8(FAKE, FAKE, 5, 4, 8, FAKE, None) == _abi.IGX_E_PARAM
    assert L.igx_pack8(None, 0, 0, 8, 8, None, None, None) == _abi.IGX_OK


def test_struct_layouts_match_the_header(tmp_path):
    import os
    import subprocess
    names = dict(Recurrence="igx_recurrence", RecurrenceGrad="igx_recurrence_grad", BlockNorm="igx_block_norm",
                 BlockNormGrad="igx_block_norm_grad")
    lines = []
    for py, c in names.items():
        lines.append('printf("%s - %%zu\\n", sizeof(%s));' % (py, c))
        lines += ['printf("%s %s %%zu\\n", offsetof(%s, %s));' % (py, f, c, f) for f, _ in getattr(_abi, py)._fields_]
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "igx.h"\nint main(void){\n%s\nreturn 0; }\n' % "\n".join(lines)
    (tmp_path / "s.c").write_text(src)
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.check_call(["gcc", "-I", inc, str(tmp_path / "s.c"), "-o", str(tmp_path / "s")])
    for line in subprocess.check_output([str(tmp_path / "s")]).decode().splitlines():
        py, field, value = line.split()
        cls = getattr(_abi, py)
        assert (C.sizeof(cls) if field == "-" else getattr(cls, field).offset) == int(value), line


def test_host_tensors_wrong_types_and_shapes_are_refused():
    x = torch.zeros(3, 2, 4)
    with pytest.raises(ValueError, match="device tensors only"):
        sequence.linear_recurrence(x, x)
    with pytest.raises(ValueError, match="device tensors only"):
        sequence.linear_recurrence_step(x[0], x[0], x[0].clone())
    with pytest.raises(ValueError, match="device tensors only"):
        sequence.rms_norm(x, torch.ones(4))
    with pytest.raises(ValueError, match="device tensors only"):
        sequence.residual_norm(x, x, torch.ones(4))
    with pytest.raises(ValueError, match="device tensors only"):
        sequence.pack8(x)
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        sequence.linear_recurrence(x.double(), x.double())
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        sequence.pack8(x.to(torch.int32))
    with pytest.raises(ValueError, match="steps, environments, channels"):
        ops.linear_recurrence(x[0], x[0], x[0])
    with pytest.raises(ValueError, match="environments, channels"):
        sequence.linear_recurrence_step(x, x, x)
    with pytest.raises(ValueError, match="activation"):
        sequence.residual_norm(x, x, torch.ones(4), activation="tanh")
    with pytest.raises(RuntimeError):
        sequence.linear_recurrence(torch.zeros(3, 3, 4), x)  # does not broadcast


def test_plain_recurrence_is_the_loop_and_its_autograd():
    g = torch.Generator().manual_seed(1)
    for reverse in (False, True):
        a, b = (torch.randn(9, 2, 3, generator=g, dtype=torch.float64) for _ in range(2))
        h0 = torch.randn(2, 3, generator=g, dtype=torch.float64)
        reset = (torch.rand(9, 2, generator=g) < 0.3).long()
        go, gl = torch.randn(9, 2, 3, generator=g, dtype=torch.float64), torch.randn(2, 3, generator=g, dtype=torch.float64)
        r = S.recurrence(a.float(), b.float(), h0.float(), reset, reverse, go.float(), gl.float())
        leaves = [t.float().double().requires_grad_(True) for t in (a, b, h0)]
        h, outs = leaves[2], [None] * 9
        for t in (range(8, -1, -1) if reverse else range(9)):
            h = leaves[0][t] * h * (reset[t] == 0).double()[:, None] + leaves[1][t]
            outs[t] = h
        grads = torch.autograd.grad((torch.stack(outs), h), leaves, (go.float().double(), gl.float().double()))
        for name, want in zip(("out", "last", "d_gate", "d_inp", "d_state"), (torch.stack(outs), h) + grads):
            assert torch.allclose(r[name][0], want, rtol=1e-12, atol=1e-12), name


@pytest.mark.parametrize("activation", ["silu", "sigmoid", "none"])
def test_plain_norm_is_its_autograd(activation):
    g = torch.Generator().manual_seed(2)
    x, y, z, do, dn = (torch.randn(5, 7, generator=g) for _ in range(5))
    w, s, w2 = (torch.randn(7, generator=g) for _ in range(3))
    t = dict(x=x, y=y, gate=z, weight=w, scale=s, next_weight=w2)
    r = S.block_norm(**t, activation=activation, d_out=do, d_next=dn)
    q = {k: v.double().requires_grad_(True) for k, v in t.items()}
    f = {"silu": q["gate"] * torch.sigmoid(q["gate"]), "sigmoid": torch.sigmoid(q["gate"]), "none": q["gate"]}[activation]

    def rms(v):
        return v / (v.square().mean(-1, keepdim=True) + 1e-5).sqrt()

    out = q["x"] + q["scale"] * f * rms(q["y"]) * q["weight"]
    nxt = rms(out) * q["next_weight"]
    assert torch.allclose(r["out"][0], out, rtol=1e-12, atol=1e-12) and torch.allclose(r["next"][0], nxt, rtol=1e-12, atol=1e-12)
    for k, want in zip(q, torch.autograd.grad((out, nxt), list(q.values()), (do.double(), dn.double()))):
        assert torch.allclose(r["d_" + k][0], want, rtol=1e-11, atol=1e-11), k
