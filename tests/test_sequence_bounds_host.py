"""That the closer bounds see what they are there for, with the mistakes made in the 64-bit forms (no GPU needed)."""
import pytest
import torch

from tests import seq_bounds as B
from tests import seq_cases as S


def inputs(R, D, seed):
    g = torch.Generator().manual_seed(seed)
    x, y, z, do, dn = (torch.randn(R, D, generator=g) for _ in range(5))
    w, s, w2 = (1 + 0.2 * torch.randn(D, generator=g) for _ in range(3))
    return dict(x=x, y=y, gate=2 * z, weight=w, scale=s, next_weight=w2), do, dn


def outside(got, ref, bound):
    return bool(((got - ref).abs() > bound).any())


@pytest.mark.parametrize("R,D,group", [(40001, 24, 32), (20011, 200, 4)])
def test_rows_that_go_missing_are_outside(R, D, group):
    """One tile (the rows that a workgroup takes at a time) less, or one tile twice, in any of eight places."""
    t, do, dn = inputs(R, D, 24)
    tn, tb, r = B.terms(**t, activation="silu", d_out=do, d_next=dn)
    for name, term, factor in (("d_next_weight", tn, 1.0), ("d_weight", tb, 1.0)):
        value, bound = B.column(r[name], term, factor)
        assert (bound > 0).all() and not outside(term.sum(0), value, bound)
        for k in range(8):
            lo = (R // 8) * k // group * group
            tile = term[lo:lo + group].sum(0)
            assert outside(value - tile, value, bound) and outside(value + tile, value, bound)


@pytest.mark.parametrize("activation", ["sigmoid", "silu"])
def test_the_difference_of_near_values_is_outside(activation):
    """p (1 - p) in 32 bits in place of exp(-z) p p: outside for every sigmoid gate from 17 on."""
    z = torch.linspace(17, 40, 47)
    t, do, dn = inputs(5, z.numel(), 25)
    t["gate"] = z.expand(5, -1).contiguous()
    value, bound = B.gate_gradient(t, do, dn, activation)
    p = 1 / (1 + torch.exp(-z))
    near = p * (1 - p)
    slope = S.block_norm(**t, activation=activation, d_out=do, d_next=dn)["d_gate"][0]
    exact = torch.sigmoid(z.double()) * torch.sigmoid(-z.double())
    if activation == "sigmoid":  # the SiLU's slope is p + z q with p near 1
        assert ((value * (near.double() / exact) - value).abs() > bound).all()
        assert (value.abs() > bound).all()  # 0 in its place, or the other sign
    assert torch.allclose(slope, value, rtol=1e-9, atol=0)
