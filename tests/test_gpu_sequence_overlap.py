"""Written tensors that share memory with others of the call are refused also where only part of them does; views that lie
between each other's rows are taken."""
import pytest
import torch

from isaacgym_amd import ops, sequence
from tests import seq_cases as S
from tests.test_gpu_sequence import BF16, DEV, F32, rollout

pytestmark = pytest.mark.gpu


def test_a_step_into_shifted_views_is_refused():
    N, D = 33, 12
    gate, inp, state, reset, _, _ = (t.to(DEV) for t in rollout(1, N, D, F32, 401, resets=0.2))
    gate, inp, reset = gate[0], inp[0], reset[0]
    buf = torch.zeros(N + 1, D, device=DEV)
    buf[:N] = state
    kept = buf.clone()
    for kw in (dict(state_out=buf[1:]), dict(out=buf[1:]), dict(state_out=buf[:N], out=buf[1:])):
        with pytest.raises(ValueError, match="overlap"):
            sequence.linear_recurrence_step(gate, inp, buf[:N], reset=reset, **kw)
    wide = torch.zeros(N + 1, D, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        sequence.linear_recurrence_step(gate, wide[1:], state, out=wide[:N])
    with pytest.raises(ValueError, match="overlap"):
        sequence.linear_recurrence_step(wide[1:], inp, state, state_out=wide[:N])
    flags = torch.zeros(N * D, device=DEV).view(torch.int64)  # the flags inside what is written
    with pytest.raises(ValueError, match="overlap"):
        sequence.linear_recurrence_step(gate, inp, state, reset=flags[:N], out=flags.view(F32).view(N, D))
    with pytest.raises(ValueError, match="overlap"):
        sequence.linear_recurrence_step(gate, inp, flags.view(F32).view(N, D), reset=flags[:N])
    torch.cuda.synchronize()
    assert torch.equal(buf, kept) and (wide == 0).all()  # nothing was launched
    # state_out as another view of state is the step in place
    want = sequence.linear_recurrence_step(gate, inp, buf[:N].clone(), reset=reset)
    assert torch.equal(sequence.linear_recurrence_step(gate, inp, buf[:N], reset=reset, state_out=buf[:N].view(N, D)), want)


def test_columns_of_one_buffer_are_taken():
    """gate, inp and out side by side in one allocation, and steps that lie between each other."""
    T, N, D = 40, 3, 13
    gate, inp, state, reset, _, _ = rollout(T, N, D, BF16, 402, resets=0.1)
    big = torch.zeros(2 * T, N, 3 * D, dtype=BF16, device=DEV)
    big[::2, :, :D], big[::2, :, D:2 * D] = gate.to(DEV), inp.to(DEV)
    ref = S.recurrence(gate, inp, state, reset)["out"]
    for out in (big[::2, :, 2 * D:], big[1::2, :, :D], big[1::2, :, 5:5 + D]):
        last = state.to(DEV)
        ops.linear_recurrence(big[::2, :, :D], big[::2, :, D:2 * D], out, state=last, reset=reset.to(DEV), last=last.view(N, D))
        S.close(out, *ref, "out")
    for out in (big[::2, :, D - 1:2 * D - 1], big[::2, :, D + 1:2 * D + 1], big[1:1 + T, :, :D]):
        with pytest.raises(ValueError, match="overlap"):
            ops.linear_recurrence(big[::2, :, :D], big[::2, :, D:2 * D], out, state=state.to(DEV))


def test_calls_on_own_buffers_refuse_shifted_views():
    T, N, D = 6, 3, 64
    gate, inp, state, reset, d_out, d_last = (t.to(DEV) for t in rollout(T, N, D, F32, 403))
    long = torch.zeros(T + 2, N, D, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        ops.linear_recurrence(gate, long[:T], long[2:])
    with pytest.raises(ValueError, match="overlap"):
        ops.linear_recurrence(gate, inp, long[:T], last=long[T - 1])
    with pytest.raises(ValueError, match="overlap"):
        ops.linear_recurrence(gate, inp, long[:T], state=long[0], last=long[0])
    with pytest.raises(ValueError, match="overlap"):
        ops.linear_recurrence_backward(gate, long[:T], d_out=d_out, d_gate=long[1:T + 1])
    with pytest.raises(ValueError, match="overlap"):
        ops.linear_recurrence_backward(gate, inp, d_out=d_out, d_gate=long[:T], d_inp=long[1:T + 1])
    rows, w = torch.zeros(9, 64, device=DEV), torch.ones(64, device=DEV)
    x = torch.randn(8, 64, device=DEV)
    inv = torch.ones(2, 8, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        ops.block_norm(rows[:8], next_weight=w, next=rows[1:])
    with pytest.raises(ValueError, match="overlap"):
        ops.block_norm(x, y=x, weight=w, next_weight=w, out=rows[:8], next=rows[1:])
    with pytest.raises(ValueError, match="overlap"):
        ops.block_norm(x, next_weight=w, next=rows[:8], inv_rms=rows[0, :16].view(2, 8))
    with pytest.raises(ValueError, match="overlap"):
        ops.block_norm_backward(x, x=x, next_weight=w, inv_rms=inv, d_next=rows[:8], d_x=rows[1:])
    with pytest.raises(ValueError, match="overlap"):
        ops.block_norm_backward(x, x=x, next_weight=w, inv_rms=inv, d_next=x, d_x=rows[:8], d_next_weight=rows[3])
    codes, scales = rows.view(torch.int8)[:8, :64].contiguous(), torch.zeros(8, 1, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        ops.pack8(rows[:8], rows.view(-1).view(torch.int8)[:512].view(8, 64), scales)
    with pytest.raises(ValueError, match="overlap"):
        ops.pack8(x, codes, codes.view(F32).view(-1)[:8].view(8, 1))
    with pytest.raises(ValueError, match="overlap"):
        ops.unpack8(rows.view(-1).view(torch.int8)[64:576].view(8, 64), scales, rows[:8])
    torch.cuda.synchronize()
    assert (rows == 0).all() and (long == 0).all() and (codes == 0).all()
