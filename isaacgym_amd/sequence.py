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
import torch
from torch.autograd.function import once_differentiable
from torch.utils.weak import WeakIdKeyDictionary
from weakref import WeakSet

from . import _abi, ops

_eager_nodes = WeakIdKeyDictionary()  # leaf -> the live autograd nodes that an eager call made with it


def _capture_guard(ctx, tensors):
    """Eager: remember that this node hangs on its leaves.  Captured: refuse leaves on which an eager node still hangs."""
    leaves = [t for t in tensors if t is not None and t.requires_grad and t.is_leaf]
    if not leaves:
        return
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        for t in leaves:
            if len(_eager_nodes.get(t, ())):
                raise RuntimeError("a tensor that requires grad is still part of an eager autograd graph: release that "
                                   "graph's outputs before capturing one with the same tensor")
        return
    for t in leaves:
        nodes = _eager_nodes.get(t)
        if nodes is None:
            nodes = _eager_nodes[t] = WeakSet()
        nodes.add(ctx)


# ---- gated linear recurrence -------------------------------------------------------------------

class _LinearRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, inp, state, reset, reverse):
        ctx.set_materialize_grads(False)
        out = torch.empty_like(inp)  # in inp's layout, so that neighbouring operators see the one they were given
        if not _adjacent(out):
            out = torch.empty(inp.shape, dtype=inp.dtype, device=inp.device)
        last = torch.empty(inp.shape[1:], dtype=torch.float32, device=inp.device)
        ops.linear_recurrence(gate, inp, out, state=state, reset=reset, last=last, reverse=reverse)
        if any(ctx.needs_input_grad[:3]):
            _capture_guard(ctx, (gate, inp, state))
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
    return _LinearRecurrence.apply(gate, inp, state, reset, bool(reverse))


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

def _rows(t, name):
    """t [..., width] as [rows, width], never copied."""
    if not isinstance(t, torch.Tensor) or t.dim() < 1:
        raise ValueError("%s must be a tensor of at least one dimension" % name)
    width = t.shape[-1]
    try:
        return t.view(t.numel() // width if width else 0, width)
    except RuntimeError:
        raise ValueError("%s: its rows (all but the last dimension) must be evenly spaced" % name) from None


def _row_grad(t, rows, width):
    """An incoming gradient as [rows, width] with adjacent columns; autograd may hand in any strides."""
    if t is None:
        return None
    t = t.reshape(rows, width)
    return t if width <= 1 or t.stride(1) == 1 else t.contiguous()


def _code_buffers(t):
    rows, width = t.shape
    return (torch.empty(rows, width, dtype=torch.int8, device=t.device),
            torch.empty(rows, -(-width // _abi.IGX_PACK8_GROUP), dtype=torch.float32, device=t.device))


class _BlockNorm(torch.autograd.Function):
    """(out, next) of ops.block_norm; without y (a norm in front of the first block) out is None."""

    @staticmethod
    def forward(ctx, x, y, weight, gate, scale, next_weight, activation, eps, checkpoint):
        ctx.set_materialize_grads(False)
        xr = _rows(x, "x")
        yr = None if y is None else _rows(y, "y")
        gr = None if gate is None else _rows(gate, "gate")
        rows, width = xr.shape
        needed = any(ctx.needs_input_grad)
        dev = x.device

        def row_stat(wanted):
            return torch.empty(rows, dtype=torch.float32, device=dev) if wanted and needed else None

        out = None if y is None else torch.empty(x.shape, dtype=x.dtype, device=dev)
        nxt = None if next_weight is None else torch.empty(x.shape, dtype=x.dtype, device=dev)
        y_inv, out_inv = row_stat(y is not None), row_stat(next_weight is not None)
        codes = needed and checkpoint
        y_codes = _code_buffers(xr) if codes else None
        gate_codes = _code_buffers(xr) if codes and gate is not None else None
        ops.block_norm(xr, y=yr, weight=weight, gate=gr, scale=scale, next_weight=next_weight,
                       out=None if out is None else out.view(rows, width), next=None if nxt is None else nxt.view(rows, width),
                       y_inv_rms=y_inv, out_inv_rms=out_inv, y_codes=y_codes, gate_codes=gate_codes, activation=activation,
                       eps=eps)
        if needed:
            _capture_guard(ctx, (x, y, weight, gate, scale, next_weight))
            keep_x = next_weight is not None and (y is not None or not codes)
            ctx.save_for_backward(xr if keep_x else None, None if codes else yr, None if codes else gr, weight, scale,
                                  next_weight, y_inv, out_inv, *(y_codes or (None, None)), *(gate_codes or (None, None)))
            ctx.shape, ctx.rows, ctx.width, ctx.dtype, ctx.device = x.shape, rows, width, x.dtype, dev
            ctx.has_block, ctx.activation, ctx.eps = y is not None, activation, eps
        return out, nxt

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_next):
        if d_out is None and d_next is None:
            return (None,) * 9
        x, y, gate, weight, scale, next_weight, y_inv, out_inv, y8, y8s, g8, g8s = ctx.saved_tensors
        want_x, want_y, want_weight, want_gate, want_scale, want_next = ctx.needs_input_grad[:6]
        rows, width = ctx.rows, ctx.width
        do, dn = _row_grad(d_out, rows, width), _row_grad(d_next, rows, width)

        def rows_like():
            return torch.empty(rows, width, dtype=ctx.dtype, device=ctx.device)

        def sums_like(wanted):
            return torch.empty(width, dtype=torch.float32, device=ctx.device) if wanted else None

        # behind a block and without a norm the gradient of x is that of out
        passed = next_weight is None or dn is None
        d_x = rows_like() if want_x and not passed else None
        d_y = rows_like() if want_y else None
        d_gate = rows_like() if want_gate else None
        d_weight, d_scale, d_next_weight = sums_like(want_weight), sums_like(want_scale), sums_like(want_next)
        ops.block_norm_backward(do if do is not None else dn, x=x, y=y, weight=weight, gate=gate, scale=scale,
                                next_weight=next_weight, y_inv_rms=y_inv, out_inv_rms=out_inv,
                                y_codes=None if y8 is None else (y8, y8s), gate_codes=None if g8 is None else (g8, g8s),
                                activation=ctx.activation, eps=ctx.eps, d_out=do, d_next=dn, d_x=d_x, d_y=d_y, d_gate=d_gate,
                                d_weight=d_weight, d_scale=d_scale, d_next_weight=d_next_weight)

        def shaped(t):
            return None if t is None else t.view(ctx.shape)

        return (d_out if want_x and passed else shaped(d_x), shaped(d_y), d_weight, shaped(d_gate), d_scale, d_next_weight,
                None, None, None)


def rms_norm(x, weight, eps=1e-5, checkpoint=False):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension (at most 8192 wide): the norm in front of a block.

    x [..., D] float32 / float16 / bfloat16, weight [D] float32.  checkpoint=True: the backward pass sees x through its
    8-bit codes (`pack8`), and x itself need not be kept for it."""
    return _BlockNorm.apply(x, None, None, None, None, weight, "none", eps, checkpoint)[1]


def residual_norm(x, y, weight, gate=None, scale=None, next_weight=None, activation="silu", eps=1e-5, checkpoint=False):
    """out = x + scale * act(gate) * (rms(y) * weight) behind a block with output y on the residual stream x; with
    next_weight returns (out, rms(out) * next_weight), the norm in front of the next block, from the same pass.

    x, y, gate [..., D] of one shape and type; weight, scale, next_weight [D] float32; activation of the gate: "silu",
    "sigmoid" or "none".  Differentiable in all of them.  checkpoint=True: y and gate are kept for the backward pass as
    8-bit codes (`pack8`) and their gradients are those at the values the codes stand for; x is kept as it is."""
    out, nxt = _BlockNorm.apply(x, y, weight, gate, scale, next_weight, activation, eps, checkpoint)
    return out if next_weight is None else (out, nxt)


# ---- 8-bit checkpoints -----------------------------------------------------------------------------

def pack8(x):
    """(codes int8 [..., D], scales float32 [..., ceil(D / 64)]) of x [..., D]: groups of 64 elements along the last
    dimension share scale = max|x| / 127, a code is the nearest integer of x * (127 / max|x|).  A group that holds an inf
    or NaN decodes to NaN, one whose largest magnitude is below 2^-120 to zeros.  Not differentiable."""
    xr = _rows(x.detach(), "x")
    codes, scales = _code_buffers(xr)
    ops.pack8(xr, codes, scales)
    return codes.view(x.shape), scales.view(x.shape[:-1] + scales.shape[1:])


def unpack8(codes, scales, dtype=torch.float32):
    """The values that pack8's codes and scales stand for."""
    out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    q = _rows(codes, "codes")
    ops.unpack8(q, _rows(scales, "scales"), _rows(out, "out"))
    return out
