"""The norms' column sums, exactly where the terms are whole numbers and by the chain of additions where they are not, and the
gates' gradients relative to themselves."""
import pytest
import torch

from isaacgym_amd import sequence
from tests import seq_bounds as B
from tests import seq_cases as S
from tests.test_gpu_sequence import BF16, DEV, F16, F32, norm_inputs

pytestmark = pytest.mark.gpu

# one row; fewer row groups than workgroups, just as many, one more; several rounds with an odd end; whole workgroups on a row;
# past the caches
SHAPES = [(1, 64), (6143, 128), (6145, 128), (24577, 8), (40001, 24), (300007, 10), (20011, 200), (9001, 600), (1537, 2046),
          (3001, 4100), (700, 8192), (16411, 211), (1 << 18, 200)]


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_sums_of_whole_numbers_are_exact(shape, dtype, checkpoint):
    """y is +-1, so its rms is 1 (eps 0) and its codes stand for it; x = y (1 - gate), so out = y; d_next is orthogonal to out in
    every pair of columns, so nothing is divided.  Every term is a whole number below 2^6 and no sum reaches 2^24."""
    R, D = shape
    g = torch.Generator(device=DEV).manual_seed(601)

    def whole(lo, hi):
        return torch.randint(lo, hi + 1, (R, D), device=DEV, generator=g).float()

    y = whole(0, 1) * 2 - 1
    # As codes of a group with top 3, gates of 1 and 2 are 42 and 85 times 3 / 127 = 0.9921 and 2.0079, no whole numbers; 0 and the
    # top itself are (127 times the fp32 number nearest to 2 / 127 rounds to 2).
    gate = 2 * whole(0, 1) if checkpoint else whole(1, 3)
    x = y * (1 - gate)
    d_out = whole(-8, 8)
    pairs = whole(-8, 8)[:, ::2].repeat_interleave(2, dim=1)[:, :D]
    sign = torch.ones(D, device=DEV)
    sign[1::2] = -1
    if D % 2:
        sign[-1] = 0
    d_next = pairs * sign * y
    weight = 2.0 ** torch.randint(0, 3, (D,), device=DEV, generator=g).float()
    leaves = [t.to(dtype) for t in (x, y, gate)] + [weight.clone(), 1 / weight, torch.ones(D, device=DEV)]
    for t in leaves:
        t.requires_grad_(True)
    outs = sequence.residual_norm(leaves[0], leaves[1], leaves[3], gate=leaves[2], scale=leaves[4], next_weight=leaves[5],
                                  activation="none", eps=0.0, checkpoint=checkpoint)
    assert torch.equal(outs[0], y.to(dtype)) and torch.equal(outs[1], y.to(dtype))
    d_x, _, d_gate, d_weight, d_scale, d_next_weight = torch.autograd.grad(outs, leaves, (d_out.to(dtype), d_next.to(dtype)))
    d = (d_out + d_next).double()
    assert torch.equal(d_x.double(), d) and torch.equal(d_gate.double(), d * y)
    total = (d * gate * y).sum(0)
    assert total.abs().max() < 2 ** 24
    assert torch.equal(d_weight.double(), total / weight) and torch.equal(d_scale.double(), total * weight)
    assert torch.equal(d_next_weight.double(), (d_next.double() * y).sum(0))
    # the norm alone
    v, w = y.to(dtype).requires_grad_(True), torch.ones(D, device=DEV, requires_grad=True)
    out = sequence.rms_norm(v, w, eps=0.0, checkpoint=checkpoint)
    got, = torch.autograd.grad(out, w, d_out.to(dtype))
    assert torch.equal(out, v) and torch.equal(got.double(), (d_out.double() * y).sum(0))


@pytest.mark.parametrize("R,D,dtype", [(40001, 24, F32), (20011, 200, F32), (9001, 600, BF16)])
def test_sums_within_the_chain_of_additions(R, D, dtype):
    t, do, dn = norm_inputs(R, D, dtype, 602, spread=False)
    dev = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    outs = sequence.residual_norm(**dev)
    grads = torch.autograd.grad(outs, [dev[k] for k in ("next_weight", "weight", "scale")], (do.to(DEV), dn.to(DEV)))
    tn, tb, r = B.terms(**t, activation="silu", d_out=do, d_next=dn)
    ratio = (t["weight"] / t["scale"]).abs().double()
    for name, got, term, factor in zip(("d_next_weight", "d_weight", "d_scale"), grads, (tn, tb, tb), (1.0, 1.0, ratio)):
        S.close(got, *B.column(r[name], term, factor), name)


@pytest.mark.parametrize("activation", ["sigmoid", "silu"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_gate_gradients_relative_to_themselves(dtype, activation):
    """Where a sigmoid is all but open its slope is exp(-z), not the rounding of 1 - p."""
    z = [0.0, 0.5, 3.0, 8.0, 12.0, 16.0, 17.0, 18.5, 20.0, 25.0, 30.0, 36.0, 40.0, 60.0, 80.0, 86.0, 87.0, 88.5, 100.0]
    z = torch.tensor(z + [-v for v in z])
    t, do, dn = norm_inputs(40, z.numel(), dtype, 603, spread=False)
    t["gate"] = z.expand(40, -1).to(dtype).contiguous()
    dev = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    outs = sequence.residual_norm(**dev, activation=activation)
    got, = torch.autograd.grad(outs, dev["gate"], (do.to(DEV), dn.to(DEV)))
    S.close(got, *B.gate_gradient(t, do, dn, activation), "d_gate")
