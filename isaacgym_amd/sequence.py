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
fallback.  Calls only enqueue work on the current stream and can be captured into a HIP graph, forward and backward
together; a capture while an eager graph of one of the same leaf tensors is alive is refused, because torch would add
the captured gradient to the leaf on the eager stream.
"""
from weakref import WeakSet

import torch
from torch.autograd.function import once_differentiable

from . import _abi, ops

_live = WeakSet()  # the autograd nodes of eager calls that hang on leaf tensors, as long as their graphs live


def _capture_guard(ctx, tensors):
    """Eager: remember that this node hangs on its leaves.  Captured: refuse leaves on which an eager node still hangs."""
    leaves = [id(t) for t in tensors if t is not None and t.requires_grad and t.is_leaf]
    if not leaves:
        return
    if torch.cuda.is_current_stream_capturing():
        for node in list(_live):
            if not node.leaves.isdisjoint(leaves):
                raise RuntimeError("a tensor that requires grad is still part of an eager autograd graph: release that "
                                   "graph's outputs before capturing one with the same tensor")
        return
    ctx.leaves = frozenset(leaves)  # the graph keeps the leaves alive, so their ids stay theirs
    _live.add(ctx)


def _differentiated(*tensors):
    """Whether autograd has to see the call (going past it saves half the host time of a small one)."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- gated linear recurrence -------------------------------------------------------------------

def _run_recurrence(gate, inp, state, reset, reverse):
    out = torch.empty_like(inp)  # in inp's layout, so that neighbouring operators see the one they were given
    if not _adjacent(out):
        out = torch.empty(inp.shape, dtype=inp.dtype, device=inp.device)
    last = torch.empty(inp.shape[1:], dtype=torch.float32, device=inp.device)
    ops.linear_recurrence(gate, inp, out, state=state, reset=reset, last=last, reverse=reverse)
    return out, last


class _LinearRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, inp, state, reset, reverse):
        ctx.set_materialize_grads(False)
        needed = any(ctx.needs_input_grad)
        if needed and inp.is_cuda:
            _capture_guard(ctx, (gate, inp, state))
        out, last = _run_recurrence(gate, inp, state, reset, reverse)
        if needed:
            ctx.save_for_backward(gate, out, state, reset)
            ctx.reverse = reverse
        return out, last

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_last):
        if d_out is None and d_last is None:
            return None, None, None, None, None
        gate, out, state, reset = ctx.saved_tensors
        if d_out is not None and not _adjacent(d_out):
            d_out = d_out.contiguous()
        if d_last is not None:
            d_last = d_last.contiguous()
        want_gate, want_inp, want_state = ctx.needs_input_grad[:3]
        d_gate = torch.empty_like(out) if want_gate else None
        d_inp = torch.empty_like(out) if want_inp else None
        d_state = torch.empty_like(state) if want_state else None
        ops.linear_recurrence_backward(gate, out, d_out=d_out, d_last=d_last, d_gate=d_gate, d_inp=d_inp, d_state=d_state,
                                       state=state, reset=reset, reverse=ctx.reverse)
        return d_gate, d_inp, d_state, None, None


def _adjacent(t):
    return t.shape[-1] <= 1 or t.stride(-1) == 1


def linear_recurrence(gate, inp, state=None, reset=None, reverse=False):
    """out[t] = gate[t] * out[t - 1] + inp[t] over a rollout; returns (out [T, N, D], last [N, D] float32).

    gate broadcasts against inp [T, N, D] (same type); both need adjacent channels, any strides otherwise, so a rollout
    kept environment by environment is passed as `x.transpose(0, 1)`.  state [N, D] float32: the value before the first
    step (None: zeros); reset [T, N] int64: where it is not 0 an episode begins and the value before is dropped.
    reverse=True runs from the last step to the first.  Differentiable in gate, inp and state; where gate is broadcast
    its full-size gradient is summed by torch afterwards.

    The carried value is float32 whatever the type; `out` is its rounding, and the gradient of gate is computed from
    `out` as stored.  Products of consecutive gates have to stay within float32's range (gates in [-1, 1] always do)."""
    if gate.shape != inp.shape:
        gate = gate.expand(inp.shape)
    run = _LinearRecurrence.apply if _differentiated(gate, inp, state) else _run_recurrence
    return run(gate, inp, state, reset, bool(reverse))


def linear_recurrence_step(gate, inp, state, reset=None, state_out=None, out=None):
    """One step for a running policy: state_out = gate * state + inp (without gradients), [N, D] each, state float32;
    environments whose reset flag (int64 [N]) is set start from zero.  state_out None: state is advanced in place.
    Returns out (the new state in the inputs' type; allocated when None)."""
    if not isinstance(inp, torch.Tensor) or inp.dim() != 2:
        raise ValueError("linear_recurrence_step: gate and inp are [environments, channels] tensors")
    if out is None:
        out = torch.empty(inp.shape, dtype=inp.dtype, device=inp.device)
    if gate.shape != inp.shape:
        gate = gate.expand(inp.shape)
    ops.linear_recurrence(gate[None], inp[None], out[None], state=state, reset=None if reset is None else reset[None],
                          last=state if state_out is None else state_out)
    return out


# ---- norms before and after a block --------------------------------------------------------------

def _row_grad(t):
    """An incoming gradient with adjacent columns and evenly spaced rows; autograd may hand in any strides."""
    return t if t is None or t.is_contiguous() else t.contiguous()


def _code_buffers(t):
    return (torch.empty(t.shape, dtype=torch.int8, device=t.device),
            torch.empty(t.shape[:-1] + (-(-t.shape[-1] // _abi.IGX_PACK8_GROUP),), dtype=torch.float32, device=t.device))


def _run_block_norm(x, y, weight, gate, scale, next_weight, activation, eps, inv_rms=None, codes=None):
    """(out, next) of ops.block_norm; without y (a norm in front of the first block) out is None."""
    out = None if y is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    nxt = None if next_weight is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    ops.block_norm(x, y=y, weight=weight, gate=gate, scale=scale, next_weight=next_weight, out=out, next=nxt,
                   inv_rms=inv_rms, codes=codes, activation=activation, eps=eps)
    return out, nxt


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, weight, gate, scale, next_weight, activation, eps, checkpoint):
        ctx.set_materialize_grads(False)
        needed = any(ctx.needs_input_grad)
        if needed and x.is_cuda:
            _capture_guard(ctx, (x, y, weight, gate, scale, next_weight))
        width = x.shape[-1]
        inv_rms = torch.empty(2, x.numel() // width if width else 0, dtype=torch.float32, device=x.device) if needed else None
        codes = None
        if needed and checkpoint:
            codes = _code_buffers(x) + (_code_buffers(x) if gate is not None else ())
        out, nxt = _run_block_norm(x, y, weight, gate, scale, next_weight, activation, eps, inv_rms, codes)
        if needed:
            keep_x = next_weight is not None and (y is not None or codes is None)
            ctx.save_for_backward(x if keep_x else None, *((y, gate) if codes is None else (None, None)), weight, scale,
                                  next_weight, inv_rms, *(codes or ()))
            ctx.activation, ctx.eps = activation, eps
        return out, nxt

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_next):
        if d_out is None and d_next is None:
            return (None,) * 9
        x, y, gate, weight, scale, next_weight, inv_rms, *codes = ctx.saved_tensors
        want_x, want_y, want_weight, want_gate, want_scale, want_next = ctx.needs_input_grad[:6]
        do, dn = _row_grad(d_out), _row_grad(d_next)
        like = dn if do is None else do
        # without a norm behind, the gradient of x is that of out
        passed = dn is None
        d_x = torch.empty_like(like) if want_x and not passed else None
        d_y = torch.empty_like(like) if want_y else None
        d_gate = torch.empty_like(like) if want_gate else None
        wanted = want_weight + want_scale + want_next
        sums = iter(torch.empty(wanted, like.shape[-1], dtype=torch.float32, device=like.device).unbind(0) if wanted else ())
        d_weight = next(sums) if want_weight else None
        d_scale = next(sums) if want_scale else None
        d_next_weight = next(sums) if want_next else None
        ops.block_norm_backward(like, x=x, y=y, weight=weight, gate=gate, scale=scale, next_weight=next_weight, inv_rms=inv_rms,
                                codes=codes or None, activation=ctx.activation, eps=ctx.eps, d_out=do, d_next=dn, d_x=d_x,
                                d_y=d_y, d_gate=d_gate, d_weight=d_weight, d_scale=d_scale, d_next_weight=d_next_weight)
        return d_out if want_x and passed else d_x, d_y, d_weight, d_gate, d_scale, d_next_weight, None, None, None


def _block_norm(x, y, weight, gate, scale, next_weight, activation, eps, checkpoint):
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise ValueError("x must be a tensor of at least one dimension")
    if _differentiated(x, y, weight, gate, scale, next_weight):
        return _BlockNorm.apply(x, y, weight, gate, scale, next_weight, activation, eps, checkpoint)
    return _run_block_norm(x, y, weight, gate, scale, next_weight, activation, eps)


def rms_norm(x, weight, eps=1e-5, checkpoint=False):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension (at most 8192 wide): the norm in front of a block.

    x [..., D] float32 / float16 / bfloat16, weight [D] float32.  checkpoint=True: the backward pass sees x through its
    8-bit codes (`pack8`), and x itself need not be kept for it."""
    return _block_norm(x, None, None, None, None, weight, "none", eps, checkpoint)[1]


def residual_norm(x, y, weight, gate=None, scale=None, next_weight=None, activation="silu", eps=1e-5, checkpoint=False):
    """out = x + scale * act(gate) * (rms(y) * weight) behind a block with output y on the residual stream x; with
    next_weight returns (out, rms(out) * next_weight), the norm in front of the next block, from the same pass.

    x, y, gate [..., D] of one shape and type; weight, scale, next_weight [D] float32; activation of the gate: "silu",
    "sigmoid" or "none".  Differentiable in all of them.  checkpoint=True: y and gate are kept for the backward pass as
    8-bit codes (`pack8`) and their gradients are those at the values the codes stand for; x is kept as it is."""
    out, nxt = _block_norm(x, y, weight, gate, scale, next_weight, activation, eps, checkpoint)
    return out if next_weight is None else (out, nxt)


# ---- 8-bit checkpoints -----------------------------------------------------------------------------

def pack8(x):
    """(codes int8 [..., D], scales float32 [..., ceil(D / 64)]) of x [..., D]: groups of 64 elements along the last
    dimension share scale = max|x| / 127, a code is the nearest integer of x * (127 / max|x|).  A group that holds an inf
    or NaN decodes to NaN, one whose largest magnitude is below 2^-120 to zeros.  Not differentiable."""
    x = x.detach()
    codes, scales = _code_buffers(x)
    ops.pack8(x, codes, scales)
    return codes, scales


def unpack8(codes, scales, dtype=torch.float32):
    """The values that pack8's codes and scales stand for."""
    out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    ops.unpack8(codes, scales, out)
    return out
