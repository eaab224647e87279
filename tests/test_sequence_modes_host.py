"""Ways of differentiating and recording that the sequence operators do not have are refused before anything else is
looked at (no GPU needed)."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from isaacgym_amd import sequence

X, W = torch.ones(3, 2, 4), torch.ones(4)


@pytest.mark.parametrize("which", range(3))
def test_forward_mode_is_refused_for_the_recurrence(which):
    with fwAD.dual_level():
        args = [X.clone(), X.clone(), X[0].clone()]
        args[which] = fwAD.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            sequence.linear_recurrence(args[0], args[1], state=args[2])


@pytest.mark.parametrize("which", range(6))
def test_forward_mode_is_refused_for_the_norms(which):
    with fwAD.dual_level():
        args = [X.clone(), X.clone(), W.clone(), X.clone(), W.clone(), W.clone()]
        args[which] = fwAD.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            sequence.residual_norm(*args[:3], gate=args[3], scale=args[4], next_weight=args[5])
        if which in (0, 2):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                sequence.rms_norm(args[0], args[2])


@pytest.mark.parametrize("call", [
    lambda x: sequence.linear_recurrence(x, x)[0], lambda x: sequence.linear_recurrence_step(x[0], x[0], x[0].clone()),
    lambda x: sequence.rms_norm(x, W), lambda x: sequence.residual_norm(x, x, W), lambda x: sequence.pack8(x)[0],
    lambda x: sequence.unpack8(x.to(torch.int8), torch.ones(3, 2, 1))])
def test_tracing_is_refused(call):
    with pytest.raises(NotImplementedError, match="torch.jit.trace"):
        torch.jit.trace(call, (X,), check_trace=False)
