"""Sequence operators for policies trained on rollouts: the parts of a recurrent residual network that are bound by
memory, as HIP kernels with gradients.

A rollout is [T, N, D] - step, environment, channel - and its episodes begin where the step kernels raised the reset
flag, so the operators take `reset_buf` (int64) as it is:

* `linear_recurrence`: out[t] = gate[t] * out[t - 1] + inp[t], the state dropped where an episode begins; reversed in time
  it is the discounted sum behind returns and advantages (utils/rlgames_utils.py: `discount_values`).
  `linear_recurrence_step` is one step of it for a running policy.
* `rms_norm`, `residual_norm`: the norms before and after a block, with the branch's gate, its residual scale and the
  next block's norm in the same pass.
* `pack8` / `unpack8`: activations as 8-bit codes with a scale for every 64 elements; with `checkpoint=True` the norms keep
  what their backward pass needs of their inputs in that form.

Element types are float32, float16 and bfloat16; states, statistics, sums and parameters are float32.  There is no CPU
fallback; forward-mode derivatives and torch.jit.trace are refused.  Calls only enqueue work on the current stream and
can be captured into a HIP graph, forward and backward together; a capture while an eager graph of one of the same leaf
tensors is alive is refused, because torch would add the captured gradient to the leaf on the eager stream.
`ops.linear_recurrence`, `ops.block_norm`, `ops.pack8` and their `_backward` are the same calls on buffers that the
caller owns.
"""
import ctypes as C
import importlib

import torch

from . import _lib

_BOUND = ("igx_last_error_string", "igx_linear_recurrence_workspace", "igx_linear_recurrence_with_rest",
          "igx_linear_recurrence_backward_with_rest", "igx_block_norm_workspace", "igx_block_norm_forward",
          "igx_block_norm_backward", "igx_pack8", "igx_unpack8")
_loaded = None


def _native():
    """The C++ side (isaacgym_amd/_sequence.so, autograd nodes and checks), on the entry points of the loaded libigx.so."""
    global _loaded
    if _loaded is None:
        library = _lib.lib()
        try:
            module = importlib.import_module("._sequence", __package__)
        except ImportError as e:
            raise ImportError("isaacgym_amd/_sequence.so cannot be loaded (%s): build it with `make -C isaacgym_amd/csrc` "
                              "(or __graft_entry__.build())" % e) from e
        module.bind({name: C.cast(getattr(library, name), C.c_void_p).value for name in _BOUND}, _lib.IgxError)
        _loaded = module
    return _loaded


def linear_recurrence(gate, inp, state=None, reset=None, reverse=False, unrounded=False):
    """out[t] = gate[t] * out[t - 1] + inp[t] over a rollout; returns (out [T, N, D], last [N, D] float32).

    gate broadcasts against inp [T, N, D] (same type); both need adjacent channels, any strides otherwise, so a rollout
    kept environment by environment is passed as `x.transpose(0, 1)`.  state [N, D] float32: the value before the first
    step (None: zeros); reset [T, N] int64: where it is not 0 an episode begins and the value before is dropped.
    reverse=True runs from the last step to the first.  Differentiable (once) in gate, inp and state; where gate is
    broadcast its full-size gradient is summed by torch afterwards.
    Steps behind the end of a shorter rollout are padded with gate 1 and input 0: they hand the value through.

    The carried value is float32 whatever the type; `out` is its rounding.  The gradient of a 16-bit gate is computed from
    `out` as stored, which makes its error 1.4 times what its own rounding gives.  unrounded=True: from the carried value,
    of which 8 bits more are kept beside `out` for the backward pass (a byte an element, written and read once; float32
    needs none).  Products of consecutive gates have to stay within float32's range (gates in [-1, 1] always do)."""
    return _native().linear_recurrence(gate, inp, state, reset, bool(reverse), bool(unrounded))


def linear_recurrence_step(gate, inp, state, reset=None, state_out=None, out=None):
    """One step for a running policy: state_out = gate * state + inp (without gradients), [N, D] each, state float32;
    environments whose reset flag (int64 [N]) is set start from zero.  state_out None: state is advanced in place.
    Returns out (the new state in the inputs' type; allocated when None)."""
    return _native().linear_recurrence_step(gate, inp, state, reset, state_out, out)


def rms_norm(x, weight, eps=1e-5, checkpoint=False):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension (at most 8192 wide): the norm in front of a block.

    x [..., D] float32 / float16 / bfloat16 with adjacent columns and rows that are evenly spaced in some order of their
    dimensions (a transposed rollout is fine, and its result is laid out like it), weight [D] float32.  checkpoint=True: the backward
    pass sees x through its 8-bit codes (`pack8`), and x itself need not be kept for it."""
    return _native().block_norm(x, None, None, None, None, weight, "none", float(eps), bool(checkpoint))[1]


def residual_norm(x, y, weight, gate=None, scale=None, next_weight=None, activation="silu", eps=1e-5, checkpoint=False):
    """out = x + scale * act(gate) * (rms(y) * weight) behind a block with output y on the residual stream x; with
    next_weight returns (out, rms(out) * next_weight), the norm in front of the next block, from the same pass.

    x, y, gate [..., D] of one shape and type, their rows evenly spaced in one order of the dimensions that all three
    share and in which the results are laid out; weight, scale, next_weight [D] float32; activation of the gate: "silu",
    "sigmoid" or "none".  Differentiable (once) in all of them.  checkpoint=True: y and gate are kept for the backward pass
    as 8-bit codes (`pack8`) and the gradients are those at the values the codes stand for, with the rows' statistics of
    the forward pass; x is kept as it is.  There a gate counts as >= -16 with "silu" and within +-16 with "sigmoid", so
    that one that is shut by a very low value leaves the other 63 of its group their precision."""
    out, after = _native().block_norm(x, y, weight, gate, scale, next_weight, activation, float(eps), bool(checkpoint))
    return out if next_weight is None else (out, after)


def pack8(x):
    """(codes int8 [..., D], scales float32 [..., ceil(D / 64)]) of x [..., D]: groups of 64 elements along the last
    dimension share scale = max|x| / 127, a code is the nearest integer of x * (127 / max|x|).  A group that holds an inf
    or NaN decodes to NaN, one whose largest magnitude is below 2^-120 to zeros.  Not differentiable."""
    return _native().pack8(x)


def unpack8(codes, scales, dtype=torch.float32):
    """The values that pack8's codes and scales stand for."""
    return _native().unpack8(codes, scales, dtype)
