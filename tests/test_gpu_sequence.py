"""The sequence operators against their plain 64-bit forms (tests/seq_cases.py), within the error that their types allow:
lengths from none to long, odd widths, every layout that is accepted, resets, non-finite values where they must not
count, gradients against formula and differences, streams, graphs and in-place steps."""
import gc

import pytest
import torch

from isaacgym_amd import ops, sequence
from isaacgym_amd._lib import IgxError
from tests import seq_cases as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def lay(t, layout):
    """t [T, N, D] (CPU) on the device with its elements laid out in the given way."""
    T, N, D = t.shape
    if layout == "time":
        return t.to(DEV).contiguous()
    if layout == "env":
        return t.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
    if layout == "slice":  # columns 3 ... of wider rows: neither aligned nor adjacent rows
        big = torch.full((T, N, D + 5), float("nan"), dtype=t.dtype, device=DEV)
        big[:, :, 3:3 + D] = t.to(DEV)
        return big[:, :, 3:3 + D]
    if layout == "steps":  # every second step of a longer rollout
        big = torch.full((2 * T, N, D), float("nan"), dtype=t.dtype, device=DEV)
        big[::2] = t.to(DEV)
        return big[::2]
    raise AssertionError(layout)


def rollout(T, N, D, dtype, seed, resets=0.0, gate_shape=None):
    g = gen(seed)
    gate = torch.sigmoid(torch.randn(gate_shape or (T, N, D), generator=g) * 2 + 1).to(dtype)
    inp = torch.randn(T, N, D, generator=g).to(dtype)
    state = torch.randn(N, D, generator=g)
    reset = (torch.rand(T, N, generator=g) < resets).to(torch.int64) * 3
    d_out = torch.randn(T, N, D, generator=g).to(dtype)
    d_last = torch.randn(N, D, generator=g)
    return gate, inp, state, reset, d_out, d_last


def check_recurrence(gate, inp, state, reset, d_out, d_last, reverse=False, layout="time", grad_layout="time"):
    """Forward and backward through autograd on the device, against the plain form of the same values."""
    full = gate.shape == inp.shape
    a = lay(gate, layout) if full else gate.to(DEV)
    b = lay(inp, layout)
    h = None if state is None else state.to(DEV)
    f = None if reset is None else reset.to(DEV)
    leaves = [t.requires_grad_(True) for t in (a, b, h) if t is not None]
    out, last = sequence.linear_recurrence(a, b, state=h, reset=f, reverse=reverse)
    assert out.shape == b.shape and out.dtype == b.dtype and last.dtype == F32
    ref = S.recurrence(gate, inp, state, reset, reverse, d_out, d_last)
    S.close(out, *ref["out"], "out")
    S.close(last, *ref["last"], "last")
    grads = torch.autograd.grad((out, last), leaves, (lay(d_out, grad_layout), d_last.to(DEV)))
    names = ["d_gate", "d_inp"] + (["d_state"] if h is not None else [])
    for name, got in zip(names, grads):
        if name == "d_gate" and not full:
            continue
        S.close(got, *ref[name], name)
    return out, last, grads


SHAPES = [(1, 1, 1), (1, 5, 3), (2, 3, 8), (7, 2, 60), (8, 37, 5), (9, 4, 105), (31, 1, 64), (33, 3, 211), (64, 130, 4),
          (129, 2, 17), (300, 1, 7), (1000, 3, 33), (1025, 1, 129), (4100, 1, 3), (2500, 1, 260)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_recurrence_shapes(shape, dtype):
    T, N, D = shape
    check_recurrence(*rollout(T, N, D, dtype, 1, resets=min(0.3, 4.0 / T)))


MANY = [(13, 1100, 64), (11, 700, 105), (12, 25000, 3), (11, 5000, 105), (10, 9001, 64), (9, 180000, 3),
        (600, 17, 1000), (517, 330, 50)]  # ... or many groups share a long sequence, with one flag a lane or two


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", MANY)
def test_recurrence_many_channels(shape, dtype):
    """Enough channels that a few groups of lanes share the steps, or that every lane walks alone."""
    T, N, D = shape
    check_recurrence(*rollout(T, N, D, dtype, 13, resets=0.1))


@pytest.mark.parametrize("layout", ["env", "slice"])
def test_recurrence_many_short_rows(layout):
    """Environments that do not follow each other, narrower than a lane's vector or not divided by it."""
    for T, N, D in ((11, 20000, 3), (10, 4000, 21), (9, 27000, 20)):
        check_recurrence(*rollout(T, N, D, F32, 14, resets=0.1), layout=layout, grad_layout="time")


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("layout", ["time", "env", "slice", "steps"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_recurrence_layouts(layout, dtype, reverse):
    other = {"time": "env", "env": "slice", "slice": "time", "steps": "env"}[layout]
    for T, N, D in ((150, 3, 12), (17, 6, 1), (20, 5, 9)):
        check_recurrence(*rollout(T, N, D, dtype, 2, resets=0.05), reverse=reverse, layout=layout, grad_layout=other)


@pytest.mark.parametrize("T,N,D", [(16, 5, 24), (400, 1, 8), (5, 6, 1)])
@pytest.mark.parametrize("shape", ["one", "per_step", "per_env", "per_channel", "per_step_env"])
def test_recurrence_broadcast_gate(T, N, D, shape):
    gs = {"one": (1, 1, 1), "per_step": (T, 1, 1), "per_env": (1, N, 1), "per_channel": (1, 1, D), "per_step_env": (T, N, 1)}[shape]
    gate, inp, state, reset, d_out, d_last = rollout(T, N, D, F32, 3, resets=0.05, gate_shape=gs)
    _, _, grads = check_recurrence(gate, inp, state, reset, d_out, d_last)
    ref, bound = S.recurrence(gate, inp, state, reset, False, d_out, d_last)["d_gate"]
    dims = [i for i in range(3) if gs[i] == 1 and ref.shape[i] > 1]
    assert grads[0].shape == gs
    total = ref.sum(dims, keepdim=True) if dims else ref
    count = ref.numel() // total.numel()
    slack = ((bound + count * S.U * ref.abs()).sum(dims, keepdim=True)) if dims else bound
    S.close(grads[0], total, slack, "summed d_gate")


@pytest.mark.parametrize("dtype", [F32, F16])
def test_recurrence_optional_arguments(dtype):
    gate, inp, state, reset, d_out, d_last = rollout(21, 4, 10, dtype, 4, resets=0.1)
    check_recurrence(gate, inp, None, reset, d_out, d_last)
    check_recurrence(gate, inp, state, None, d_out, d_last)
    check_recurrence(gate, inp, None, None, d_out, d_last, reverse=True)
    # only one of the outputs used, only one of the inputs differentiated
    a, b, h, f = gate.to(DEV), inp.to(DEV), state.to(DEV), reset.to(DEV)
    for use_out in (True, False):
        ref = S.recurrence(gate, inp, state, reset, False, d_out if use_out else None, None if use_out else d_last)
        for i, name in enumerate(("d_gate", "d_inp", "d_state")):
            args = [a.clone(), b.clone(), h.clone()]
            args[i].requires_grad_(True)
            out, last = sequence.linear_recurrence(args[0], args[1], state=args[2], reset=f)
            head = (out, d_out.to(DEV)) if use_out else (last, d_last.to(DEV))
            got, = torch.autograd.grad(head[0], args[i], head[1])
            S.close(got, *ref[name], "%s alone" % name)
    # a gradient that autograd hands in with stride 0
    args = [t.clone().requires_grad_(True) for t in (a, b, h)]
    sequence.linear_recurrence(*args, reset=f)[0].sum().backward()
    ref = S.recurrence(gate, inp, state, reset, False, torch.ones(inp.shape), None)
    for t, name in zip(args, ("d_gate", "d_inp", "d_state")):
        S.close(t.grad, *ref[name], "%s of a sum" % name)


@pytest.mark.parametrize("T,N,D", [(6, 4, 8), (700, 1, 12), (40, 3, 3)])
def test_recurrence_nothing_passes_an_episode_start(T, N, D):
    """Gates, state and earlier values that are inf or NaN must not reach what lies behind a reset."""
    gate, inp, state, _, d_out, d_last = rollout(T, N, D, F32, 5)
    reset = torch.zeros(T, N, dtype=torch.int64)
    at = T // 2
    reset[at] = 1
    reset[0] = -7
    gate[0], gate[at] = float("nan"), float("inf")
    state[:] = float("nan")
    inp[at - 1] = float("inf")
    clean_gate, clean_inp, clean_state = gate.clone(), inp.clone(), torch.zeros_like(state)
    clean_gate[0] = clean_gate[at] = 0.0
    ref = S.recurrence(clean_gate, clean_inp, clean_state, reset)
    out, last = sequence.linear_recurrence(gate.to(DEV), inp.to(DEV), state=state.to(DEV), reset=reset.to(DEV))
    S.close(out[:at - 1], ref["out"][0][:at - 1], ref["out"][1][:at - 1], "before")
    S.close(out[at:], ref["out"][0][at:], ref["out"][1][at:], "behind")
    assert torch.isinf(out[at - 1]).all()
    d_gate, d_inp, d_state = torch.empty_like(out), torch.empty_like(out), torch.empty_like(last)
    d_out[at:] = float("nan")  # what lies behind must not flow back over the start either
    ops.linear_recurrence_backward(gate.to(DEV), out, d_out=d_out.to(DEV), d_last=d_last.to(DEV), d_gate=d_gate, d_inp=d_inp,
                                   d_state=d_state, state=state.to(DEV), reset=reset.to(DEV))
    assert torch.isfinite(d_inp[:at]).all() and torch.isnan(d_inp[at:]).all()
    assert (d_gate[0] == 0).all() and (d_gate[at] == 0).all() and (d_state == 0).all()


def test_recurrence_every_step_reset_and_zero_state():
    gate, inp, state, _, d_out, d_last = rollout(200, 2, 8, BF16, 6)
    reset = torch.ones(200, 2, dtype=torch.int64)
    out, last, grads = check_recurrence(gate, inp, state, reset, d_out, d_last)
    assert torch.equal(out.cpu(), inp) and (grads[0] == 0).all() and (grads[2] == 0).all()


def test_recurrence_growing_gates_from_a_zero_state():
    """Gates of 2 over 300 steps: their product overflows fp32, the state stays 0 until the last step.  A state that is not
    0 overflows with it: inf, never a finite value."""
    for T, N in ((300, 1), (3000, 1), (700, 2100)):
        inp = torch.zeros(T, N, 8)
        inp[-1] = 1.0
        gate = torch.full((T, N, 8), 2.0, device=DEV)
        out, last = sequence.linear_recurrence(gate, inp.to(DEV))
        assert torch.equal(out.cpu(), inp) and (last == 1).all()
        assert torch.isinf(sequence.linear_recurrence(gate, inp.to(DEV), state=torch.full((N, 8), 2.0 ** -40, device=DEV))[1]).all()


@pytest.mark.parametrize("T,N,D", [(0, 3, 4), (5, 0, 4), (5, 3, 0), (0, 0, 0)])
def test_recurrence_empty(T, N, D):
    a = torch.empty(T, N, D, device=DEV, requires_grad=True)
    b = torch.empty(T, N, D, device=DEV, requires_grad=True)
    h = torch.randn(N, D, device=DEV, requires_grad=True)
    out, last = sequence.linear_recurrence(a, b, state=h, reset=torch.zeros(T, N, dtype=torch.int64, device=DEV))
    assert out.shape == (T, N, D)
    if T == 0:
        assert torch.equal(last, h)
        g = torch.randn_like(last)
        assert torch.equal(torch.autograd.grad(last, h, g)[0], g)
        assert (sequence.linear_recurrence(a.detach(), b.detach())[1] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("N,D", [(1, 1), (5, 3), (130, 60), (4096, 64)])
def test_recurrence_step(N, D, dtype):
    gate, inp, state, reset, _, _ = rollout(1, N, D, dtype, 7, resets=0.2)
    ref = S.recurrence(gate, inp, state, reset)
    a, b, h, f = gate[0].to(DEV), inp[0].to(DEV), state.to(DEV), reset[0].to(DEV)
    kept, to = h.clone(), torch.full_like(h, float("nan"))
    out = sequence.linear_recurrence_step(a, b, h, reset=f, state_out=to)
    S.close(out, ref["out"][0][0], ref["out"][1][0], "out")
    S.close(to, *ref["last"], "state_out")
    assert torch.equal(h, kept)
    again = sequence.linear_recurrence_step(a, b, h, reset=f)
    assert torch.equal(h, to) and torch.equal(again, out)  # in place: the same bits


def test_recurrence_step_in_place_where_lanes_share_channels():
    """A width that the 16-byte vector does not divide: the last lane of a row overlaps the one before."""
    for N, D in ((1, 13), (3001, 5), (1, 100003)):
        gate, inp, state, _, _, _ = rollout(1, N, D, BF16, 8)
        wide = torch.zeros(N, D + 3, dtype=BF16, device=DEV)  # rows apart: lanes per environment
        wide[:, 1:1 + D] = inp[0].to(DEV)
        for b in (inp[0].to(DEV), wide[:, 1:1 + D]):
            h, to = state.to(DEV), torch.empty(N, D, device=DEV)
            sequence.linear_recurrence_step(gate[0].to(DEV), b, h, state_out=to)
            sequence.linear_recurrence_step(gate[0].to(DEV), b, h)
            assert torch.equal(h, to)


@pytest.mark.parametrize("T,N,D", [(60, 7, 20), (2000, 1, 24)])
def test_recurrence_in_two_calls(T, N, D):
    """A rollout cut in two, `last` handed on as `state`: outputs and gradients are those of the whole."""
    gate, inp, state, reset, d_out, d_last = rollout(T, N, D, F32, 16, resets=0.02)
    ref = S.recurrence(gate, inp, state, reset, False, d_out, d_last)
    a, b, h = (t.to(DEV).requires_grad_(True) for t in (gate, inp, state))
    f, cut = reset.to(DEV), T // 3
    one, mid = sequence.linear_recurrence(a[:cut], b[:cut], state=h, reset=f[:cut])
    two, end = sequence.linear_recurrence(a[cut:], b[cut:], state=mid, reset=f[cut:])
    out = torch.cat((one, two))
    S.close(out, *ref["out"], "out")
    S.close(end, *ref["last"], "last")
    for name, got in zip(("d_gate", "d_inp", "d_state"), torch.autograd.grad((out, end), (a, b, h), (d_out.to(DEV), d_last.to(DEV)))):
        S.close(got, *ref[name], name)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("shape", [(7, 5, 12), (40, 6, 12), (3000, 1, 8), (700, 2100, 8), (20, 9000, 8), (10, 70000, 8)])
def test_recurrence_last_is_what_the_last_step_left(shape, reverse):
    """In every split of the time `last` is the fp32 value whose rounding is out's last step, and steps with gate 1 and input
    0 behind an environment's last one hand its state through."""
    T, N, D = shape
    g = torch.Generator(device=DEV).manual_seed(17)
    gate, inp = torch.rand(T, N, D, device=DEV, generator=g), torch.randn(T, N, D, device=DEV, generator=g)
    length = torch.randint(1, T, (N,), device=DEV, generator=g)
    pad = torch.arange(T, device=DEV)[:, None] >= length
    gate[pad], inp[pad] = 1.0, 0.0
    if reverse:
        gate, inp = gate.flip(0), inp.flip(0)
    for dtype in (F32, BF16):
        out, last = sequence.linear_recurrence(gate.to(dtype), inp.to(dtype), reverse=reverse)
        assert torch.equal(out[0 if reverse else -1], last.to(dtype))
    out, last = sequence.linear_recurrence(gate, inp, reverse=reverse)
    end = out.flip(0)[length - 1, torch.arange(N, device=DEV)] if reverse else out[length - 1, torch.arange(N, device=DEV)]
    # |out| < 1 + the magnitudes' sum of a recurrence with gates below 1 and inputs below 7; 3 u of it a step, T steps
    assert float((end - last).abs().max()) <= 3 * S.U * T * 7 * min(T, 20)


def test_recurrence_writes_only_its_elements():
    gate, inp, state, reset, _, _ = rollout(70, 3, 13, F16, 9, resets=0.1)
    big = torch.full((140, 3, 20), 7.0, dtype=F16, device=DEV)
    out = big[::2, :, 4:17]
    ops.linear_recurrence(gate.to(DEV), inp.to(DEV), out, state=state.to(DEV), reset=reset.to(DEV))
    ref = S.recurrence(gate, inp, state, reset)
    S.close(out, *ref["out"], "out")
    assert (big[1::2] == 7).all() and (big[:, :, :4] == 7).all() and (big[:, :, 17:] == 7).all()


def test_recurrence_offsets_past_32_bits():
    """Steps and environments more than 2^32 bytes apart."""
    far = torch.zeros(3 * (1 << 30) + 64, dtype=F32, device=DEV)
    gate, inp, state, _, _, _ = rollout(3, 2, 8, F32, 10)
    for strides in (((1 << 30), 16, 1), (16, (1 << 30) + (1 << 29), 1)):
        b = far.as_strided((3, 2, 8), strides)
        b.copy_(inp)
        out = torch.empty(3, 2, 8, device=DEV)
        ops.linear_recurrence(gate.to(DEV), b, out, state=state.to(DEV))
        S.close(out, *S.recurrence(gate, inp, state)["out"], "out")
        ops.linear_recurrence(gate.to(DEV), inp.to(DEV), b, state=state.to(DEV))
        assert torch.equal(b, out)


def test_recurrence_gradient_against_differences():
    """<gradient, v> against (f(x + e v) - f(x - e v)) / 2e of the 64-bit plain form, e = 1e-6: the difference's own error
    is 2^-53 |f| / e + e^2 |f'''| < 1e-8 of the magnitudes, below the fp32 gradient's."""
    gate, inp, state, reset, d_out, d_last = rollout(40, 2, 6, F32, 11, resets=0.05)
    gate, inp, state, d_out, d_last = (t.double() for t in (gate, inp, state, d_out, d_last))
    _, _, grads = check_recurrence(gate.float(), inp.float(), state.float(), reset, d_out.float(), d_last.float())

    def f(a, b, h):
        r = S.recurrence(a, b, h, reset)
        return float((r["out"][0] * d_out).sum() + (r["last"][0] * d_last).sum())

    e = 1e-6
    for i, x in enumerate((gate, inp, state)):
        v = torch.randn(x.shape, generator=gen(12 + i), dtype=torch.float64)
        plus, minus = ([y + s * e * v if y is x else y for y in (gate, inp, state)] for s in (1, -1))
        diff = (f(*plus) - f(*minus)) / (2 * e)
        g = grads[i].double().cpu()
        # every element of the gradient is within 40 steps' roundings of 3 u each; magnitudes from |g| plus one per step
        assert abs(float((g * v).sum()) - diff) <= 1e-5 * float((g.abs() * v.abs()).sum() + v.abs().sum())


@pytest.mark.parametrize("D", [0, 1, 3])
@pytest.mark.parametrize("dones", [torch.int64, torch.float32, torch.bool])
def test_discount_values(D, dones):
    """The agent's loop in 64 bits: two roundings of the difference, two of the gate, one of the sum, every step."""
    from isaacgym_amd.utils.rlgames_utils import discount_values
    T, N = 33, 70
    g = gen(15)
    shape = (T, N, D) if D else (T, N)
    rew, val, nxt = (torch.randn(*shape, generator=g) for _ in range(3))
    done = (torch.rand(T, N, generator=g) < 0.1)
    adv = discount_values(done.to(dones).to(DEV), val.to(DEV), rew.to(DEV), nxt.to(DEV), 0.99, 0.95)
    assert adv.shape == shape and not adv.requires_grad
    a, m = torch.zeros(shape[1:], dtype=torch.float64), torch.zeros(shape[1:], dtype=torch.float64)
    for t in range(T - 1, -1, -1):
        live = 0.99 * 0.95 * (~done[t]).double().view(N, *([1] if D else []))
        a = rew[t].double() + 0.99 * nxt[t].double() - val[t].double() + live * a
        m = rew[t].double().abs() + nxt[t].double().abs() + val[t].double().abs() + live * m
        assert ((adv[t].double().cpu() - a).abs() <= 5 * (T - t) * S.U * m).all()


# ---- norms ----------------------------------------------------------------------------------------------------------

def norm_inputs(R, D, dtype, seed, gate=True, scale=True, next=True, spread=True):
    g = gen(seed)
    x, y, z, do, dn = (torch.randn(R, D, generator=g) for _ in range(5))
    if spread and R:  # rows of very different sizes, one of them empty
        y = y * torch.logspace(-3, 2, R)[:, None]
        y[R // 2] = 0
    w, s, w2 = (1 + 0.2 * torch.randn(D, generator=g) for _ in range(3))
    t = dict(x=x.to(dtype), y=y.to(dtype), gate=(2 * z).to(dtype) if gate else None, weight=w, scale=s if scale else None,
             next_weight=w2 if next else None)
    return t, do.to(dtype), dn.to(dtype)


def check_norm(t, d_out, d_next, activation="silu", checkpoint=False, place=None):
    """residual_norm (or rms_norm where there is no y) forward and backward against the plain form."""
    place = place or (lambda v: v.to(DEV))
    dev = {k: (place(v) if v.dim() == 2 else v.to(DEV)).requires_grad_(True) for k, v in t.items() if v is not None}
    if t.get("y") is None:
        outs = (sequence.rms_norm(dev["x"], dev["next_weight"], checkpoint=checkpoint),)
        heads, names = (place(d_next),), ("next",)
        d_out = None
    else:
        outs = sequence.residual_norm(**dev, activation=activation, checkpoint=checkpoint)
        outs = outs if "next_weight" in dev else (outs,)
        heads, names = (place(d_out), place(d_next))[:len(outs)], ("out", "next")
    ref = S.block_norm(**t, activation=activation, d_out=d_out, d_next=d_next if t["next_weight"] is not None else None,
                       checkpoint=checkpoint)
    for name, got in zip(names, outs):
        S.close(got, *ref[name], name)
    keys = list(dev)
    grads = torch.autograd.grad(outs, [dev[k] for k in keys], heads)
    for k, got in zip(keys, grads):
        assert got.dtype == dev[k].dtype and got.shape == dev[k].shape
        S.close(got, *ref["d_" + k], "d_" + k)
    return outs, dict(zip(keys, grads))


NORM_SHAPES = [(1, 1), (3, 2), (5, 7), (64, 8), (33, 60), (7, 64), (130, 65), (19, 105), (6, 128), (300, 211), (5, 256),
               (9, 500), (4, 512), (3, 513), (5, 1025), (2, 2048), (3, 4099), (2, 8192)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_residual_norm_shapes(shape, dtype):
    t, do, dn = norm_inputs(*shape, dtype, 20)
    check_norm(t, do, dn)


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1, 1), (70, 33), (40, 64), (9, 130), (5, 700), (3, 2049), (2, 5000)])
def test_rms_norm(shape, dtype, checkpoint):
    t, _, dn = norm_inputs(*shape, dtype, 21)
    check_norm(dict(x=t["y"], y=None, next_weight=t["next_weight"]), None, dn, checkpoint=checkpoint)


@pytest.mark.parametrize("activation", ["silu", "sigmoid", "none"])
@pytest.mark.parametrize("gate,scale,nxt", [(True, True, False), (True, False, True), (False, True, True), (False, False, False)])
@pytest.mark.parametrize("checkpoint", [False, True])
def test_residual_norm_parts(gate, scale, nxt, activation, checkpoint):
    for (R, D), dtype in (((50, 60), F32), ((37, 264), BF16), ((6, 1100), F16)):
        t, do, dn = norm_inputs(R, D, dtype, 22, gate=gate, scale=scale, next=nxt)
        check_norm(t, do, dn, activation=activation, checkpoint=checkpoint)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_residual_norm_strided_rows(dtype):
    def place(v):  # rows of a wider array, from an odd column
        big = torch.full((v.shape[0], v.shape[1] + 9), float("nan"), dtype=v.dtype, device=DEV)
        big[:, 5:5 + v.shape[1]] = v.to(DEV)
        return big[:, 5:5 + v.shape[1]]

    for R, D in ((20, 60), (11, 211), (4, 1030)):
        t, do, dn = norm_inputs(R, D, dtype, 23)
        check_norm(t, do, dn, place=place)


@pytest.mark.parametrize("activation", ["silu", "sigmoid", "none"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_residual_norm_extreme_gates(dtype, activation):
    """Gates up to the type's ends: where exp(-z) leaves fp32 the gate is shut or open, not NaN."""
    z = [0.0, -0.0, 1e-30, 8.0, 17.0, 40.0, 87.0, 88.5, 89.0, 100.0, 104.0, 110.0, 111.5, 128.0, 200.0, 1e4, torch.finfo(dtype).max]
    z = torch.tensor(z + [-v for v in z])
    t, do, dn = norm_inputs(3, z.numel(), dtype, 36, spread=False)
    if activation == "none":
        z = z.clamp(-100, 100)  # the gate is then a factor of out, whose square has to stay in fp32
    t["gate"] = z.expand(3, -1).to(dtype).contiguous()
    if activation == "silu":
        big = t["gate"] > 1e3
        t["gate"][big] = 1e3
    outs, grads = check_norm(t, do, dn, activation=activation)
    for v in list(outs) + list(grads.values()):
        assert torch.isfinite(v).all()


def test_residual_norm_broadcast_rows_and_one_row():
    """One gate row for all rows (stride 0): torch adds its full-size gradients up; a single row without other dimensions."""
    t, do, dn = norm_inputs(40, 36, F32, 35)
    row = t["gate"][:1].clone()
    t["gate"] = row.expand(40, 36)
    dev = {k: v.to(DEV).requires_grad_(True) for k, v in t.items() if k != "gate"}
    leaf = row.to(DEV).requires_grad_(True)
    outs = sequence.residual_norm(gate=leaf.expand(40, 36), **dev)
    ref = S.block_norm(**t, d_out=do, d_next=dn)
    S.close(outs[0], *ref["out"], "out")
    grads = torch.autograd.grad(outs, [leaf] + list(dev.values()), (do.to(DEV), dn.to(DEV)))
    value, bound = ref["d_gate"]
    S.close(grads[0], value.sum(0, keepdim=True), (bound + 40 * S.U * value.abs()).sum(0, keepdim=True), "summed d_gate")
    for k, got in zip(dev, grads[1:]):
        S.close(got, *ref["d_" + k], "d_" + k)
    one = sequence.rms_norm(dev["x"].detach()[3], dev["weight"].detach())
    assert one.shape == (36,) and torch.equal(one, sequence.rms_norm(dev["x"].detach(), dev["weight"].detach())[3])


def test_residual_norm_many_rows():
    """More rows than there are lane groups on the card: the groups walk, the column sums are joined."""
    t, do, dn = norm_inputs(40001, 24, F32, 24, spread=False)
    check_norm(t, do, dn)
    t, do, dn = norm_inputs(9001, 600, BF16, 25, spread=False)
    check_norm(t, do, dn)


@pytest.mark.parametrize("dtype,checkpoint", [(F32, False), (BF16, True)])
def test_norms_larger_than_the_caches(dtype, checkpoint):
    """A call that moves more than the caches hold gives every row the bits of a small call on it; its column sums are the
    small calls' sums, added up in another order: (rows + calls) roundings of the magnitudes' sum."""
    R, D, part = 1 << 18, 200, 1 << 14
    g = torch.Generator(device=DEV).manual_seed(33)
    x, y, z, do, dn = (torch.randn(R, D, device=DEV, generator=g).to(dtype) for _ in range(5))
    w, s, w2 = (torch.randn(D, device=DEV, generator=g) for _ in range(3))
    for post in (True, False):
        def run(lo, hi):
            leaves = [t[lo:hi].detach().requires_grad_(True) for t in ((x, y, z) if post else (x,))]
            leaves += [t.detach().requires_grad_(True) for t in ((w, s, w2) if post else (w2,))]
            if post:
                outs = sequence.residual_norm(leaves[0], leaves[1], leaves[3], gate=leaves[2], scale=leaves[4],
                                              next_weight=leaves[5], checkpoint=checkpoint)
                heads = (do[lo:hi], dn[lo:hi])
            else:
                outs, heads = (sequence.rms_norm(leaves[0], leaves[1], checkpoint=checkpoint),), (dn[lo:hi],)
            grads = torch.autograd.grad(outs, leaves, heads)
            rows = [o.detach() for o in outs] + list(grads[:3 if post else 1])
            return rows, [t.double() for t in grads[3 if post else 1:]]

        rows, sums = run(0, R)
        total = [torch.zeros_like(t) for t in sums]
        for lo in range(0, R, part):
            some, parts = run(lo, lo + part)
            for a, b in zip(rows, some):
                assert torch.equal(a[lo:lo + part], b)
            total = [a + b for a, b in zip(total, parts)]
        for a, b in zip(sums, total):
            # the terms are d * unit-sized values: their magnitudes' sum is below 16 a row
            assert ((a - b).abs() <= (R + R // part) * S.U * 16 * R ** 0.5).all()


def test_residual_norm_leading_dimensions_and_unused_outputs():
    t, do, dn = norm_inputs(24, 40, F32, 26)
    dev = {k: (v.view(2, 3, 4, 40) if v.dim() == 2 else v).to(DEV).requires_grad_(True) for k, v in t.items()}
    out, nxt = sequence.residual_norm(**dev)
    assert out.shape == nxt.shape == (2, 3, 4, 40)
    for used, head, args in ((out, do, dict(d_out=do)), (nxt, dn, dict(d_next=dn))):
        ref = S.block_norm(**t, **args)
        grads = torch.autograd.grad(used, [dev[k] for k in t], head.view(2, 3, 4, 40).to(DEV), retain_graph=True,
                                    allow_unused=True)
        for k, got in zip(t, grads):
            S.close(got.reshape(ref["d_" + k][0].shape), *ref["d_" + k], "d_" + k)
    # one leaf alone
    for k in t:
        args = {j: (v.detach().requires_grad_(j == k)) for j, v in dev.items()}
        o, n = sequence.residual_norm(**args)
        got, = torch.autograd.grad((o, n), args[k], (do.view(o.shape).to(DEV), dn.view(o.shape).to(DEV)))
        ref = S.block_norm(**t, d_out=do, d_next=dn)["d_" + k]
        S.close(got.reshape(ref[0].shape), *ref, "d_%s alone" % k)


def test_norms_empty():
    for R in (0,):
        x = torch.empty(R, 30, device=DEV, requires_grad=True)
        w = torch.ones(30, device=DEV, requires_grad=True)
        out = sequence.rms_norm(x, w)
        assert out.shape == (R, 30)
        gx, gw = torch.autograd.grad(out, (x, w), torch.empty_like(out))
        assert gx.shape == x.shape and (gw == 0).all()
        out, nxt = sequence.residual_norm(x, x, w, gate=x, scale=w, next_weight=w)
        gx, gw = torch.autograd.grad((out, nxt), (x, w), (torch.empty_like(out), torch.empty_like(nxt)))
        assert gx.shape == x.shape and (gw == 0).all()
        for checkpoint in (False, True):  # each input alone: none takes another one's place
            for i in range(6):
                leaves = [torch.empty(R, 30, device=DEV) for _ in range(3)] + [torch.ones(30, device=DEV) for _ in range(3)]
                leaves[i].requires_grad_(True)
                outs = sequence.residual_norm(leaves[0], leaves[1], leaves[3], gate=leaves[2], scale=leaves[4],
                                              next_weight=leaves[5], checkpoint=checkpoint)
                got, = torch.autograd.grad(outs, leaves[i], [torch.empty_like(o) for o in outs])
                assert got.shape == leaves[i].shape and (got == 0).all()


def test_norms_a_row_does_not_touch_its_neighbours():
    """NaN and inf in one row stay in it (and in the column sums); the others keep their bits."""
    t, do, dn = norm_inputs(65, 50, F32, 27)
    clean = {k: v.to(DEV) for k, v in t.items()}
    bad = {k: v.clone() for k, v in clean.items()}
    bad["y"][17], bad["x"][40], bad["gate"][3, 5] = float("nan"), float("inf"), float("nan")
    keep = torch.ones(65, dtype=torch.bool)
    keep[[17, 40, 3]] = False
    for a, b in zip(sequence.residual_norm(**clean), sequence.residual_norm(**bad)):
        assert torch.equal(a[keep], b[keep])
        assert torch.isnan(b[17]).all()


def test_norms_offsets_past_32_bits():
    far = torch.zeros(2 * (1 << 30) + 4096, dtype=F32, device=DEV)
    t, do, dn = norm_inputs(3, 40, F32, 28)
    x = far.as_strided((3, 40), (1 << 30, 1))
    x.copy_(t["x"])
    got = sequence.residual_norm(x, t["y"].to(DEV), t["weight"].to(DEV), gate=t["gate"].to(DEV), scale=t["scale"].to(DEV))
    t["next_weight"] = None
    S.close(got, *S.block_norm(**t)["out"], "out")
    codes, scales = torch.empty(3, 40, dtype=torch.int8, device=DEV), torch.empty(3, 1, device=DEV)
    ops.pack8(x, codes, scales)
    assert torch.equal(codes.cpu().float(), S.through8(t["x"])[1])


def test_norm_gradient_against_differences():
    """As for the recurrence: the 64-bit plain form's central differences, e = 1e-6."""
    t, do, dn = norm_inputs(12, 20, F32, 29, spread=False)
    _, grads = check_norm(t, do, dn)
    t = {k: v.double() for k, v in t.items()}

    def f(t):
        r = S.block_norm(**t)
        return float((r["out"][0] * do.double()).sum() + (r["next"][0] * dn.double()).sum())

    e = 1e-6
    for i, k in enumerate(t):
        v = torch.randn(t[k].shape, generator=gen(30 + i), dtype=torch.float64)
        diff = (f({**t, k: t[k] + e * v}) - f({**t, k: t[k] - e * v})) / (2 * e)
        g = grads[k].double().cpu()
        assert abs(float((g * v).sum()) - diff) <= 1e-5 * float((g.abs() * v.abs()).sum() + v.abs().sum()), k


# ---- 8-bit checkpoints ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (17, 63), (9, 64), (11, 65), (40, 105), (5, 128), (2, 1000), (3001, 211)])
def test_pack8_is_the_definition_bit_for_bit(shape, dtype):
    x = (torch.randn(*shape, generator=gen(40)) * torch.logspace(-4, 4, shape[0])[:, None]).to(dtype)
    value, code, scale = S.through8(x)
    codes, scales = sequence.pack8(x.to(DEV))
    assert torch.equal(codes.cpu().float(), code) and torch.equal(scales.cpu(), scale)
    for to in (dtype, F32):
        assert torch.equal(sequence.unpack8(codes, scales, dtype=to).cpu(), value.to(to))


def test_pack8_ends_of_the_range():
    """Zeros, subnormals, values at the type's ends, ties, and non-finite values, which mark their group."""
    x = torch.zeros(9, 130)
    x[1] = 1e-40
    x[2, 3] = 2.0 ** -120
    x[3] = torch.linspace(-127, 127, 130)
    x[4, :64] = torch.arange(64) + 0.5
    x[4, 0] = 127.0
    x[5] = 3.0e38
    x[6, 70], x[7, 1], x[8, 129] = float("nan"), float("inf"), float("-inf")
    value, code, scale = S.through8(x)
    codes, scales = sequence.pack8(x.to(DEV))
    assert torch.equal(codes.cpu().float(), code)
    got = sequence.unpack8(codes, scales).cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(value)) and torch.equal(got.nan_to_num(7.0), value.nan_to_num(7.0))
    assert torch.isfinite(got[6, :64]).all() and torch.isnan(got[6, 64:128]).all() and torch.isnan(got[8, 128:]).all()


def test_pack8_shapes_and_empty():
    x = torch.randn(2, 3, 70, device=DEV)
    codes, scales = sequence.pack8(x)
    assert codes.shape == (2, 3, 70) and scales.shape == (2, 3, 2)
    assert torch.equal(sequence.unpack8(codes, scales), S.through8(x.cpu().view(6, 70))[0].view(2, 3, 70).to(DEV))
    codes, scales = sequence.pack8(torch.empty(0, 70, device=DEV))
    assert sequence.unpack8(codes, scales).shape == (0, 70)


@pytest.mark.parametrize("activation", ["silu", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(40, 60), (9, 130), (3, 1100)])
def test_checkpointed_gates_shut_by_very_low_values(shape, dtype, activation):
    """A shut gate takes the others of its group no precision; the gradients are those at the limited gates' codes."""
    t, do, dn = norm_inputs(*shape, dtype, 46)
    shut = torch.rand(shape, generator=gen(47)) < 0.1
    shut[1] = True  # a row without any open one
    t["gate"] = torch.where(shut, torch.full_like(t["gate"], torch.finfo(dtype).min), t["gate"])
    if activation == "sigmoid":
        t["gate"][0, 3], t["gate"][2, 5] = float("inf"), float("-inf")
    dev = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    outs = sequence.residual_norm(**dev, activation=activation, checkpoint=True)
    grads = torch.autograd.grad(outs, list(dev.values()), (do.to(DEV), dn.to(DEV)))
    limited = t["gate"].clamp(min=-16, max=16 if activation == "sigmoid" else None)
    # Results and the rows' inverse roots come from the gates themselves, whose activations are off from the limited ones' by
    # less than 16 exp(-16) < 2^-19.  That moves a row's inverse root by less than 2^-18 of it, and no result holds more than
    # its third power: 2^-16 of the terms' magnitudes, of which twice the largest result is taken as the bound.
    ref = S.block_norm(**dict(t, gate=limited), activation=activation, d_out=do, d_next=dn, checkpoint=True)
    for name, got in list(zip(("out", "next"), outs)) + [("d_" + k, g) for k, g in zip(dev, grads)]:
        value, bound = ref[name]
        S.close(got, value, bound + 2.0 ** -15 * value.abs().max(), name)


def test_checkpoint_frees_what_it_replaces():
    """With checkpoint=True the graph holds codes, not the block's output and gate."""
    R, D = 8192, 512
    x = torch.randn(R, D, device=DEV, dtype=BF16, requires_grad=True)
    w = torch.ones(D, device=DEV)
    size = R * D * 2

    def held(checkpoint):
        gc.collect()
        torch.cuda.synchronize()
        start = torch.cuda.memory_allocated()
        out = sequence.residual_norm(x, x * 2, w, gate=x + 1, checkpoint=checkpoint)
        gc.collect()
        return torch.cuda.memory_allocated() - start, out

    plain, o1 = held(False)
    del o1
    packed, o2 = held(True)
    assert plain >= 3 * size and packed <= 2.2 * size


def test_layouts_that_are_refused():
    x = torch.zeros(3, 4, 5, 6, device=DEV)
    w = torch.ones(6, device=DEV)
    with pytest.raises(ValueError, match="evenly spaced"):
        sequence.rms_norm(x[:, ::2], w)
    with pytest.raises(ValueError, match="adjacent"):
        sequence.rms_norm(torch.zeros(6, 5, device=DEV).t(), w)
    with pytest.raises(ValueError, match="adjacent"):
        sequence.rms_norm(x.transpose(2, 3), torch.ones(5, device=DEV))
    with pytest.raises(ValueError, match="expected shape"):
        sequence.residual_norm(x, x[0], w)
    with pytest.raises(TypeError, match="expected dtype"):
        sequence.residual_norm(x, x.half(), w)
    with pytest.raises(TypeError, match="expected dtype"):
        sequence.rms_norm(x, w.half())
    with pytest.raises(ValueError, match="device tensors only"):
        sequence.rms_norm(x, w.cpu())
    with pytest.raises(ValueError, match="contiguous"):
        sequence.rms_norm(x, torch.ones(12, device=DEV)[::2])
    r = torch.zeros(3, 4, 6, device=DEV)
    with pytest.raises(ValueError, match="adjacent"):
        sequence.linear_recurrence(r, torch.zeros(3, 6, 4, device=DEV).transpose(1, 2))
    with pytest.raises(TypeError, match="expected dtype"):
        sequence.linear_recurrence(r, r, reset=torch.zeros(3, 4, device=DEV))
    with pytest.raises(ValueError, match="expected shape"):
        sequence.linear_recurrence(r, r, state=torch.zeros(4, 5, device=DEV))
    with pytest.raises(ValueError, match="overlap"):
        ops.linear_recurrence(r, r, r)
    with pytest.raises(ValueError, match="share one address"):
        ops.linear_recurrence(r, r, torch.zeros(4, 6, device=DEV).expand(3, 4, 6))
    step = torch.zeros(4, 6, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        sequence.linear_recurrence_step(r[0], step, torch.zeros(4, 6, device=DEV), state_out=step)
    with pytest.raises(ValueError, match="overlap"):
        sequence.linear_recurrence_step(r[0], r[1], step, out=step)
    with pytest.raises(ValueError, match="expected shape"):
        sequence.linear_recurrence_step(r[0], r[1], step[:2])
    with pytest.raises(TypeError, match="expected dtype"):
        sequence.linear_recurrence_step(r[0], r[1], step.half())
    with pytest.raises(IgxError, match="8192"):
        sequence.rms_norm(torch.zeros(2, 8193, device=DEV), torch.ones(8193, device=DEV))


# ---- streams, graphs, repeatability ---------------------------------------------------------------------------------

def block(x, p, state, reset):
    """norm -> recurrence -> gated norm on the residual stream: one block of a recurrent policy."""
    n = sequence.rms_norm(x, p["w_in"])
    h, last = sequence.linear_recurrence(torch.sigmoid(n), n, state=state, reset=reset)
    out, nxt = sequence.residual_norm(x, h, p["w_out"], gate=n, scale=p["s"], next_weight=p["w_next"], checkpoint=True)
    return out, nxt, last


def block_inputs(T, N, D, dtype=F32, seed=50):
    g = gen(seed)
    x = torch.randn(T, N, D, generator=g).to(dtype).to(DEV)
    p = {k: (1 + 0.1 * torch.randn(D, generator=g)).to(DEV) for k in ("w_in", "w_out", "s", "w_next")}
    state = torch.randn(N, D, generator=g).to(DEV)
    reset = (torch.rand(T, N, generator=g) < 0.1).to(torch.int64).to(DEV)
    heads = [torch.randn(T, N, D, generator=g).to(dtype).to(DEV) for _ in range(2)]
    return x, p, state, reset, heads


def block_pass(x, p, state, reset, heads):
    leaves = [x, state] + list(p.values())
    for t in leaves:
        t.requires_grad_(True)
    out, nxt, last = block(x, p, state, reset)
    grads = torch.autograd.grad((out, nxt), leaves, heads)
    return [out.detach(), nxt.detach(), last.detach()] + list(grads)


def test_same_call_same_bits():
    args = block_inputs(300, 5, 100)
    first = block_pass(*args)
    for _ in range(3):
        for a, b in zip(first, block_pass(*args)):
            assert torch.equal(a, b)


def test_side_stream():
    args = block_inputs(64, 7, 72, BF16)
    want = block_pass(*args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = block_pass(*args)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_host_threads_on_their_own_streams():
    """Four host threads, each on its own stream and inputs, give what the serial calls give."""
    import threading
    shapes = [(600, 1, 40), (40, 6, 130), (300, 5, 100), (33, 300, 64)]
    args = [block_inputs(*s, seed=100 + i) for i, s in enumerate(shapes)]
    want = [block_pass(*a) for a in args]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = block_pass(*args[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # the assertion below reports it
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_two_captured_graphs_replayed_with_eager_work_between():
    """Forward and backward of a block in two graphs, on new inputs every replay, against the eager pass."""
    graphs = []
    for i, (T, N, D) in enumerate(((2000, 1, 40), (40, 6, 130))):
        x, p, state, reset, heads = block_inputs(T, N, D, seed=60 + i)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                block_pass(x, p, state, reset, heads)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = block_pass(x, p, state, reset, heads)
        graphs.append((graph, (x, p, state, reset, heads), outs, (T, N, D)))
    for turn in range(4):
        for graph, args, outs, shape in graphs:
            x, p, state, reset, heads = args
            fresh = block_inputs(*shape, seed=70 + turn)
            with torch.no_grad():
                x.copy_(fresh[0])
                state.copy_(fresh[2])
                for k in p:
                    p[k].copy_(fresh[1][k])
                reset.copy_(fresh[3])
                for h, f in zip(heads, fresh[4]):
                    h.copy_(f)
            graph.replay()
            want = block_pass(*fresh)
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b)
            del want


def test_capture_with_a_live_eager_graph_of_the_same_leaf_is_refused():
    x, p, state, reset, heads = block_inputs(8, 2, 16)
    x.requires_grad_(True)
    w = torch.ones(16, device=DEV, requires_grad=True)
    alive = sequence.rms_norm(x, w)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(graph):
            torch.zeros(1, device=DEV).add_(1)
            sequence.rms_norm(x, w)
    del alive, graph
    torch.cuda.synchronize()
    out = sequence.rms_norm(x, w)  # eager work goes on as before
    S.close(out.view(16, 16), *S.block_norm(x.detach().view(16, 16), next_weight=w)["next"], "next")


def test_capture_above_an_eager_graph_is_refused():
    """The same where the leaf is not the operator's own input: an eager graph further up, or one that is alive beside it."""
    x = torch.randn(8, 2, 16, device=DEV, requires_grad=True)
    w = torch.ones(16, device=DEV)
    alive = x * 2
    for make in (lambda: alive, lambda: x * 3):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager autograd graph"):
            with torch.cuda.graph(graph):
                torch.zeros(1, device=DEV).add_(1)
                sequence.rms_norm(make(), w)
        del graph
    with torch.no_grad():  # nothing to differentiate: captured
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = sequence.rms_norm(alive, w)
    graph.replay()
    assert torch.equal(out, sequence.rms_norm(alive.detach(), w))


def test_captured_backward_accumulates_into_leaves():
    """backward() inside the capture writes the leaves' grad at every replay."""
    x, p, state, reset, heads = block_inputs(20, 3, 24, seed=90)
    leaves = [t.requires_grad_(True) for t in [x, state] + list(p.values())]

    def step():
        for t in leaves:
            t.grad = None
        out, nxt, _ = block(x, p, state, reset)
        torch.autograd.backward((out, nxt), heads)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(3):
        fresh = block_inputs(20, 3, 24, seed=91 + turn)
        with torch.no_grad():
            x.copy_(fresh[0])
            state.copy_(fresh[2])
            reset.copy_(fresh[3])
            for k in p:
                p[k].copy_(fresh[1][k])
            for h, f in zip(heads, fresh[4]):
                h.copy_(f)
        graph.replay()
        want = block_pass(*fresh)[3:]
        for t, w in zip(leaves, want):
            assert torch.equal(t.grad, w)


def test_gradients_are_not_differentiated_again():
    x = torch.randn(4, 16, device=DEV, requires_grad=True)
    out = sequence.rms_norm(x, torch.ones(16, device=DEV))
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(out.sum(), x, create_graph=True)
    r = torch.randn(4, 2, 16, device=DEV, requires_grad=True)
    out, _ = sequence.linear_recurrence(r, r)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(out.sum(), r, create_graph=True)


def test_inputs_changed_between_forward_and_backward_are_noticed():
    r = torch.randn(4, 2, 16, device=DEV, requires_grad=True)
    g = torch.rand(4, 2, 16, device=DEV)
    out, _ = sequence.linear_recurrence(g, r)
    g.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_a_step_in_place_is_noticed_by_graphs_that_saved_the_state():
    r = torch.randn(4, 2, 16, device=DEV, requires_grad=True)
    state = torch.randn(2, 16, device=DEV)
    out, _ = sequence.linear_recurrence(torch.sigmoid(r), r, state=state)
    sequence.linear_recurrence_step(r.detach()[0], r.detach()[1], state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


# ---- the calls on the caller's buffers ---------------------------------------------------------------------------------

@pytest.mark.parametrize("checkpoint", [False, True])
def test_calls_on_own_buffers_equal_the_differentiable_ones(checkpoint):
    T, N, D = 200, 2, 70
    gate, inp, state, reset, d_out, d_last = (t.to(DEV) for t in rollout(T, N, D, BF16, 95, resets=0.05))
    leaves = [t.requires_grad_(True) for t in (gate, inp, state)]
    out, last = sequence.linear_recurrence(*leaves[:2], state=state, reset=reset)
    grads = torch.autograd.grad((out, last), leaves, (d_out, d_last))
    mine, end = torch.empty_like(out), torch.empty_like(last)
    own = [torch.empty_like(t) for t in leaves]
    with torch.no_grad():
        ops.linear_recurrence(gate, inp, mine, state=state, reset=reset, last=end)
        ops.linear_recurrence_backward(gate, mine, d_out=d_out, d_last=d_last, d_gate=own[0], d_inp=own[1], d_state=own[2],
                                       state=state, reset=reset)
    for a, b in zip([out, last, *grads], [mine, end, *own]):
        assert torch.equal(a, b)

    t, do, dn = norm_inputs(60, 130, F32, 96)
    dev = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    outs = sequence.residual_norm(**dev, activation="sigmoid", checkpoint=checkpoint)
    want = list(outs) + list(torch.autograd.grad(outs, list(dev.values()), (do.to(DEV), dn.to(DEV))))
    rows = [torch.empty(60, 130, device=DEV) for _ in range(2)]
    inv = torch.empty(2, 60, device=DEV)
    codes = None
    if checkpoint:
        codes = tuple(torch.empty(*s, dtype=d, device=DEV) for _ in range(2) for s, d in (((60, 130), torch.int8), ((60, 3), F32)))
    p = {k: dev[k].detach() for k in ("weight", "scale", "next_weight")}
    args = dict(activation="sigmoid", inv_rms=inv, codes=codes, **p)
    x, y, z = (dev[k].detach() for k in ("x", "y", "gate"))
    ops.block_norm(x, y=y, gate=z, out=rows[0], next=rows[1], **args)
    got = {k: torch.empty_like(v) for k, v in dev.items()}
    ops.block_norm_backward(x, x=x, y=None if checkpoint else y, gate=None if checkpoint else z, d_out=do.to(DEV),
                            d_next=dn.to(DEV), **{"d_" + k: v for k, v in got.items()}, **args)
    for a, b in zip(want, rows + list(got.values())):
        assert torch.equal(a, b)
    if checkpoint:
        for i, v in ((0, y), (2, z)):
            q, s = sequence.pack8(v)
            assert torch.equal(q, codes[i]) and torch.equal(s, codes[i + 1])
            mine = [torch.empty_like(q), torch.empty_like(s), torch.empty_like(v)]
            ops.pack8(v, mine[0], mine[1])
            ops.unpack8(mine[0], mine[1], mine[2])
            assert torch.equal(mine[0], q) and torch.equal(mine[1], s) and torch.equal(mine[2], sequence.unpack8(q, s))
    with pytest.raises(ValueError, match="overlap"):
        ops.block_norm(x, y=y, out=x, next=rows[1], **args)
    with pytest.raises(ValueError, match="overlap"):
        ops.linear_recurrence_backward(gate.detach(), out.detach(), d_out=d_out, d_inp=d_out)


# ---- as they are used: a policy on an environment's rollout ------------------------------------------------------------

def test_policy_block_on_a_task_rollout():
    """A recurrent policy runs a task step by step; the rollout is then trained on as a whole.  The training pass gives
    the running policy's outputs again, its gradients are the plain form's, and the advantages are the agent's loop."""
    from isaacgym_amd import tasks
    from isaacgym_amd.utils.rlgames_utils import discount_values

    T, N = 24, 64
    env = tasks.make("Ant", num_envs=N, device=DEV)
    D = env.num_obs
    g = gen(80)
    w_in, w_out, s, w_next = ((1 + 0.1 * torch.randn(D, generator=g)).to(DEV) for _ in range(4))
    k = torch.randn(D, generator=g).to(DEV)
    env.reset_done()
    state = torch.zeros(N, D, device=DEV)
    start = state.clone()
    begins = torch.ones(N, dtype=torch.int64, device=DEV)  # the first step starts every episode
    xs, flags, outs, rewards, dones = [], [], [], [], []
    obs = env.obs_buf.clone()
    env.progress_buf[::5] = 990  # some episodes end inside the rollout
    for t in range(T):
        n = sequence.rms_norm(obs, w_in)
        h = sequence.linear_recurrence_step(torch.sigmoid(n * k), n, state, reset=begins)
        out, nxt = sequence.residual_norm(obs, h, w_out, gate=n, scale=s, next_weight=w_next)
        xs.append(obs)
        flags.append(begins)
        outs.append((out, nxt))
        obs_dict, rew, reset, _ = env.step(nxt[:, :env.num_actions].tanh())
        obs, begins = obs_dict["obs"].clone(), reset.clone()
        rewards.append(rew.clone())
        dones.append(begins)
    assert sum(int(f.sum()) for f in flags[1:]) > 0
    x, reset = torch.stack(xs), torch.stack(flags)
    leaves = [t.requires_grad_(True) for t in (x, w_in, w_out, s, w_next)]
    n = sequence.rms_norm(x, w_in)
    gates = torch.sigmoid(n * k)
    h, last = sequence.linear_recurrence(gates, n, state=start, reset=reset)
    out, nxt = sequence.residual_norm(x, h, w_out, gate=n, scale=s, next_weight=w_next)
    # one step or many: a chain of at most T + 3 fp32 operators, about 100 u each (the norms' own bounds), on either side
    chain = (T + 3) * 100 * S.U
    for t in range(T):
        for a, b in ((out.detach()[t], outs[t][0]), (nxt.detach()[t], outs[t][1])):
            assert float((a - b).abs().max()) <= 2 * chain * float(out.detach().abs().max())
    assert float((last.detach() - state).abs().max()) <= 2 * chain * float(h.detach().abs().max())

    d = [torch.randn(out.shape, generator=g).to(DEV) for _ in range(2)]
    grads = torch.autograd.grad((out, nxt), leaves, d)
    # the whole block in 64 bits, differentiated by torch
    q = [t.detach().double().cpu().requires_grad_(True) for t in leaves]
    X, W, WO, SS, WN = q

    def rms(v):
        return v / (v.square().mean(-1, keepdim=True) + 1e-5).sqrt()

    NN = rms(X) * W
    A = torch.sigmoid(NN * k.double().cpu())
    H, hs = torch.zeros(N, D, dtype=torch.float64), []
    for t in range(T):
        H = torch.where(reset[t].cpu().bool()[:, None], torch.zeros_like(H), A[t] * H) + NN[t]
        hs.append(H)
    O = X + SS * (NN * torch.sigmoid(NN)) * rms(torch.stack(hs)) * WO
    ref = torch.autograd.grad((O, rms(O) * WN), q, [t.double().cpu() for t in d])
    for got, want in zip(grads, ref):
        assert float((got.double().cpu() - want).abs().max()) <= chain * float(want.abs().max())

    rew, done = torch.stack(rewards), torch.stack(dones)
    values, nxt_values = torch.randn(2, T, N, generator=g).to(DEV)
    adv = discount_values(done, values, rew, nxt_values, 0.99, 0.95)
    r64, v64, n64 = rew.double(), values.double(), nxt_values.double()
    want, mag = torch.zeros(T, N, dtype=torch.float64, device=DEV), torch.zeros(T, N, dtype=torch.float64, device=DEV)
    a, m = 0.0, 0.0
    for t in range(T - 1, -1, -1):
        live = 0.99 * 0.95 * (1.0 - done[t].double())
        a = r64[t] + 0.99 * n64[t] - v64[t] + live * a
        m = r64[t].abs() + n64[t].abs() + v64[t].abs() + live * m
        want[t], mag[t] = a, m
    # two roundings of the difference, one of the gate (twice: gamma * tau, its product) and one of the sum, every step
    assert ((adv.double() - want).abs() <= 5 * T * S.U * mag).all()
