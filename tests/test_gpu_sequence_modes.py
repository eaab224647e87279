"""The sequence operators under autograd's other modes: what they do not have raises, what they share with torch works."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from isaacgym_amd import sequence
from isaacgym_amd.utils.rlgames_utils import discount_values
from tests.test_gpu_sequence import BF16, DEV, F32, block_inputs, block_pass, rollout

pytestmark = pytest.mark.gpu


def test_forward_mode_raises_in_place_of_a_lost_tangent():
    x, w = torch.randn(6, 2, 24, device=DEV), torch.ones(24, device=DEV)
    with fwAD.dual_level():
        d = fwAD.make_dual(x, torch.ones_like(x))
        for call in (lambda: x + sequence.rms_norm(d, w), lambda: sequence.residual_norm(d, x, w),
                     lambda: sequence.linear_recurrence(x, d), lambda: sequence.linear_recurrence(d.sigmoid(), x)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            sequence.rms_norm(d, w)
        # without gradients by its documentation
        done = torch.zeros(6, 2, dtype=torch.int64, device=DEV)
        adv = discount_values(done, x, d, x, 0.99, 0.95)
        assert fwAD.unpack_dual(adv).tangent is None and torch.equal(adv, discount_values(done, x, x, x, 0.99, 0.95))
    assert torch.isfinite(sequence.rms_norm(x, w)).all()  # and afterwards as before


def test_trace_raises_in_place_of_unwritten_memory():
    x, w = torch.randn(6, 2, 24, device=DEV), torch.ones(24, device=DEV)
    with pytest.raises(NotImplementedError, match="torch.jit.trace"):
        torch.jit.trace(lambda t: sequence.rms_norm(t, w), (x,), check_trace=False)
    with pytest.raises(NotImplementedError, match="torch.jit.trace"):
        torch.jit.trace(lambda t: sequence.linear_recurrence(t, t)[0], (x,), check_trace=False)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_saved_tensor_hooks_see_every_saved_tensor(dtype):
    """A hook that moves what the graph keeps to host memory and back changes no bit of the gradients."""
    args = block_inputs(40, 3, 72, dtype)
    want = block_pass(*args)
    seen = []

    def pack(t):
        seen.append(t.dtype)
        return t.cpu(), t.stride()

    def unpack(kept):
        t = torch.empty_strided(kept[0].shape, kept[1], dtype=kept[0].dtype, device=DEV)
        t.copy_(kept[0])
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        got = block_pass(*args)
    assert torch.int8 in seen and dtype in seen
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_saved_tensor_hooks_see_the_unrounded_part():
    gate, inp, state, reset, d_out, d_last = (t.to(DEV) for t in rollout(40, 3, 9, BF16, 301, resets=0.1))
    gate.requires_grad_(True)
    run = lambda: torch.autograd.grad(sequence.linear_recurrence(gate, inp, state=state, reset=reset, unrounded=True), gate,
                                      (d_out, d_last))[0]
    want, kinds = run(), []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (kinds.append(t.dtype), t.clone())[1], lambda t: t):
        got = run()
    assert torch.int8 in kinds and torch.equal(want, got)


@pytest.mark.parametrize("wrong", [lambda t: t.cpu(), lambda t: t[:1], lambda t: t.to(torch.int16 if t.dtype == torch.int8 else torch.float64)])
@pytest.mark.parametrize("kind", [torch.int8, F32])
def test_what_a_hook_hands_back_is_checked(wrong, kind):
    """A hook that gives the backward pass another device, shape or type gets an error, for the tensors that only the nodes
    know (codes, their scales, the rows' inverse roots) like for the caller's own."""
    def back(t):
        return wrong(t) if t.dtype == kind and t.dim() > 1 else t

    x = torch.randn(40, 130, device=DEV, dtype=BF16)
    w = torch.ones(130, device=DEV)
    gate, inp, state, reset, d_out, d_last = (t.to(DEV) for t in rollout(40, 3, 9, BF16, 302, resets=0.1))
    calls = [lambda: sequence.residual_norm(x, x, w, gate=x, next_weight=w, checkpoint=True), lambda: (sequence.rms_norm(x, w, checkpoint=True),)]
    if kind == torch.int8:
        calls.append(lambda: sequence.linear_recurrence(gate, inp, unrounded=True))
    else:
        calls.append(lambda: sequence.linear_recurrence(gate, inp, state=state))
    x.requires_grad_(True)
    gate.requires_grad_(True)
    for call in calls:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
            outs = call()
        with pytest.raises((ValueError, TypeError, RuntimeError), match="device tensors only|expected shape|expected dtype"):
            torch.autograd.backward(outs, [torch.ones_like(o) for o in outs])


def test_a_step_that_is_refused_has_not_been_taken():
    """A state that was made in inference mode may be advanced there, not outside; refused, it still holds its values."""
    gate, inp, start, reset, _, _ = (t.to(DEV) for t in rollout(1, 5, 12, F32, 303, resets=0.2))
    want = start.clone()
    out = sequence.linear_recurrence_step(gate[0], inp[0], want, reset=reset[0])
    with torch.inference_mode():
        state, to, result = start.clone(), torch.full_like(start, 7.0), torch.full_like(start, 7.0)
        inner = start.clone()
        assert torch.equal(sequence.linear_recurrence_step(gate[0], inp[0], inner, reset=reset[0]), out) and torch.equal(inner, want)
    for kw in (dict(), dict(state_out=to), dict(out=result), dict(state_out=to, out=torch.empty_like(start)),
               dict(state_out=torch.empty_like(start), out=result)):
        given = start.clone() if kw else state
        kept = given.clone()
        with pytest.raises(RuntimeError, match="inference tensor"):
            sequence.linear_recurrence_step(gate[0], inp[0], given, reset=reset[0], **kw)
        assert torch.equal(given, kept) and (to == 7).all() and (result == 7).all()
    with torch.inference_mode():
        sequence.linear_recurrence_step(gate[0], inp[0], state, reset=reset[0])
    assert torch.equal(state, want)
    # the other operators read inference tensors, and write none of them
    with torch.inference_mode():
        x, w = torch.randn(4, 24, device=DEV), torch.ones(24, device=DEV)
        inside = sequence.rms_norm(x, w)
    assert torch.equal(sequence.rms_norm(x, w), inside)
