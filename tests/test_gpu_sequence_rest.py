"""The recurrence with what out's rounding took kept beside it: the gradient of a 16-bit gate has one rounding of its type."""
import pytest
import torch

from isaacgym_amd import ops, sequence
from tests import seq_cases as S
from tests.test_gpu_sequence import BF16, DEV, F16, F32, gen, lay, rollout

pytestmark = pytest.mark.gpu
SHIFT = {BF16: 8, F16: 5}  # a code counts 1 / 256 of the type's step: 2^16 and 2^13 patterns of fp32


def gate_gradient(gate, inp, state, reset, reverse, d_out, d_last):
    """(value, bound) of d_gate from carried values that are off by at most 2^-7 of out's half step, rounded once.  The 64-bit
    form on the same values as fp32 gives the bound of the fp32 arithmetic."""
    dt = inp.dtype
    r = S.recurrence(gate.float(), inp.float(), state, reset, reverse, d_out.float(), d_last)
    value, bound = r["d_gate"]
    least = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2  # half a step of a subnormal out: there is no gain there
    kept = value.abs() * S.half_step(dt) * 2.0 ** -7 + r["d_inp"][0].abs() * least
    return value, bound + kept + S.stored(value, dt)


def check(gate, inp, state, reset, d_out, d_last, reverse=False, layout="time", grad_layout="time"):
    leaves = [lay(gate, layout), lay(inp, layout), state.to(DEV)]
    for t in leaves:
        t.requires_grad_(True)
    heads = (lay(d_out, grad_layout), d_last.to(DEV))
    f = reset.to(DEV)
    runs = []
    for unrounded in (True, False):
        outs = sequence.linear_recurrence(leaves[0], leaves[1], state=leaves[2], reset=f, reverse=reverse, unrounded=unrounded)
        runs.append([t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, heads)))
    for i in (0, 1, 3, 4):  # everything but d_gate is the same call
        assert torch.equal(runs[0][i], runs[1][i])
    S.close(runs[0][2], *gate_gradient(gate, inp, state, reset, reverse, d_out, d_last), "d_gate")


SHAPES = [(1, 1, 1), (2, 3, 8), (7, 2, 60), (9, 4, 105), (33, 3, 211), (300, 1, 7), (1025, 1, 129), (2500, 1, 260),
          (13, 1100, 64), (11, 5000, 105), (12, 25000, 3), (10, 20000, 64), (600, 17, 1000), (517, 330, 50)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(shape, dtype):
    T, N, D = shape
    check(*rollout(T, N, D, dtype, 201, resets=min(0.3, 4.0 / T)))


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("layout", ["time", "env", "slice", "steps"])
def test_layouts(layout, reverse):
    other = {"time": "env", "env": "slice", "slice": "time", "steps": "env"}[layout]
    for T, N, D in ((150, 3, 12), (17, 6, 1), (20, 5, 9), (9, 3000, 60)):
        check(*rollout(T, N, D, BF16, 202, resets=0.05), reverse=reverse, layout=layout, grad_layout=other)


def test_float32_keeps_nothing_more():
    gate, inp, state, reset, d_out, d_last = (t.to(DEV) for t in rollout(40, 3, 9, F32, 203, resets=0.1))
    gate.requires_grad_(True)
    got = [torch.autograd.grad(sequence.linear_recurrence(gate, inp, state=state, reset=reset, unrounded=u), gate, (d_out, d_last))[0]
           for u in (True, False)]
    assert torch.equal(*got)


def decoded(out, codes):
    """out and its codes as fp32."""
    bits = out.float().contiguous().view(torch.int32) + (codes.to(torch.int32) << SHIFT[out.dtype])
    return bits.view(F32)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_codes_are_what_the_rounding_took(dtype):
    """One step with gate 1 and input 0: out is the rounding of the state, out and code together the state to 2^-7 of half a
    step.  Ties, the neighbours of powers of two, subnormals, values that round to inf, inf and NaN."""
    info = torch.finfo(dtype)
    steps = torch.arange(-600, 600).float()
    v = torch.cat([torch.randn(4000, generator=gen(204)) * 10 ** (4 * torch.rand(4000, generator=gen(205)) - 2),
                   1 + steps * info.eps / 512, -2 + steps * info.eps / 512, 3 * info.eps / 2 * steps,
                   info.max * (1 + steps * info.eps / 1024), info.smallest_normal * (1 + steps * info.eps / 16),
                   info.smallest_normal * info.eps * steps / 64,
                   torch.tensor([0.0, -0.0, float("inf"), float("-inf"), float("nan"), 1e38, -1e38, 1e-45])])
    n = v.numel()
    for width in (n, 13, 1):  # whole vectors, rows with a moved last vector, single elements
        rows = n // width
        state = v[:rows * width].view(rows, width).to(DEV)
        wide = torch.zeros(1, rows, width + 3, dtype=dtype, device=DEV)
        for inp in (torch.zeros(1, rows, width, dtype=dtype, device=DEV), wide[:, :, :width]):
            out, codes = torch.empty(1, rows, width, dtype=dtype, device=DEV), torch.full((1, rows, width), 77, dtype=torch.int8, device=DEV)
            ops.linear_recurrence(torch.ones(1, rows, width, dtype=dtype, device=DEV), inp, out, state=state, rest=codes)
            h, o, q = state.cpu().double(), out[0].cpu(), codes[0].cpu()
            assert torch.equal(o.float().nan_to_num(7), state.cpu().to(dtype).float().nan_to_num(7))
            special = ~torch.isfinite(o.float())
            assert (q[special] == 0).all()
            assert (q[o.double() == h] == 0).all()
            err = (decoded(o, q).double() - h).abs()[~special]
            half = (S.stored(o.double(), dtype))[~special]
            # Where the value is normal a step is 256 codes on both sides of out.  In fp16's subnormals the step stays 2^-24, which
            # in the binade below 2^-14 is 2^14 patterns of fp32, twice what 256 codes of 2^5 reach (and more further down): a
            # code that ends at -128 leaves up to half of the half step, so that binade's upper end, 2^-14, belongs to them.
            normal = h.abs()[~special] >= info.smallest_normal
            assert (err[normal] <= half[normal] * 2.0 ** -7).all()
            assert (err <= half).all()


def test_codes_stay_in_their_elements():
    gate, inp, state, reset, _, _ = (t.to(DEV) for t in rollout(70, 3, 13, F16, 206, resets=0.1))
    big = torch.full((140, 3, 20), 77, dtype=torch.int8, device=DEV)
    tight = torch.empty(70, 3, 13, dtype=torch.int8, device=DEV)
    out = torch.empty_like(inp)
    ops.linear_recurrence(gate, inp, out, state=state, reset=reset, rest=big[::2, :, 4:17])
    ops.linear_recurrence(gate, inp, out, state=state, reset=reset, rest=tight)
    assert torch.equal(big[::2, :, 4:17], tight)
    assert (big[1::2] == 77).all() and (big[:, :, :4] == 77).all() and (big[:, :, 17:] == 77).all()


def test_own_buffers_equal_the_differentiable_call():
    gate, inp, state, reset, d_out, d_last = (t.to(DEV) for t in rollout(200, 2, 70, BF16, 207, resets=0.05))
    leaves = [t.requires_grad_(True) for t in (gate, inp, state)]
    outs = sequence.linear_recurrence(gate, inp, state=state, reset=reset, unrounded=True)
    want = list(torch.autograd.grad(outs, leaves, (d_out, d_last)))
    with torch.no_grad():
        mine, codes, got = torch.empty_like(inp), torch.empty(inp.shape, dtype=torch.int8, device=DEV), [torch.empty_like(t) for t in leaves]
        ops.linear_recurrence(gate, inp, mine, state=state, reset=reset, rest=codes)
        ops.linear_recurrence_backward(gate, mine, d_out=d_out, d_last=d_last, d_gate=got[0], d_inp=got[1], d_state=got[2],
                                       state=state, reset=reset, rest=codes)
    for a, b in zip([outs[0]] + want, [mine] + got):
        assert torch.equal(a, b)
    with pytest.raises(ValueError, match="overlap"):
        ops.linear_recurrence(gate, inp, mine, rest=mine.view(torch.int8)[:, :, :70])
    with pytest.raises(TypeError, match="expected dtype"):
        ops.linear_recurrence(gate, inp, mine, rest=codes.to(torch.uint8))
    with pytest.raises(ValueError, match="adjacent"):
        ops.linear_recurrence(gate, inp, mine, rest=torch.empty(200, 70, 2, dtype=torch.int8, device=DEV).transpose(1, 2))


def test_captured_and_replayed():
    gate, inp, state, reset, d_out, d_last = (t.to(DEV) for t in rollout(300, 2, 40, BF16, 208, resets=0.05))
    leaves = [gate, inp, state]

    def run():
        for t in leaves:
            t.requires_grad_(True)
        outs = sequence.linear_recurrence(*leaves[:2], state=state, reset=reset, unrounded=True)
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, (d_out, d_last)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for turn in range(3):
        with torch.no_grad():
            for t, f in zip(leaves + [reset, d_out, d_last], rollout(300, 2, 40, BF16, 209 + turn, resets=0.05)):
                t.copy_(f)
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
        del want
