"""discount_values in every shape and layout that it documents."""
import pytest
import torch

from isaacgym_amd.utils.rlgames_utils import discount_values
from tests import seq_cases as S
from tests.test_gpu_sequence import DEV, gen

pytestmark = pytest.mark.gpu
T, N = 19, 21


def loop(done, values, rewards, next_values):
    """(advantages, allowed error) of [T, N, D] in 64 bits: two roundings of the difference, two of the gate, one of the sum."""
    a = m = torch.zeros(values.shape[1:], dtype=torch.float64)
    out, bound = [None] * T, [None] * T
    for t in range(T - 1, -1, -1):
        live = 0.99 * 0.95 * (done[t] == 0).double()[:, None]
        a = rewards[t].double() + 0.99 * next_values[t].double() - values[t].double() + live * a
        m = rewards[t].double().abs() + next_values[t].double().abs() + values[t].double().abs() + live * m
        out[t], bound[t] = a, 5 * (T - t) * S.U * m
    return torch.stack(out), torch.stack(bound)


@pytest.mark.parametrize("kind", [torch.int64, torch.float32, torch.bool, torch.uint8])
@pytest.mark.parametrize("done_last", [False, True])
@pytest.mark.parametrize("D", [0, 1, 3])
def test_shapes(D, done_last, kind):
    g = gen(501)
    val, rew, nxt = (torch.randn(T, N, max(D, 1), generator=g) for _ in range(3))
    done = (torch.rand(T, N, generator=g) < 0.15).to(kind)
    want, bound = loop(done, val, rew, nxt)
    args = [t if D else t.squeeze(-1) for t in (val, rew, nxt)]
    flags = done.unsqueeze(-1) if done_last else done
    got = discount_values(flags.to(DEV), *(t.to(DEV) for t in args), 0.99, 0.95)
    assert got.shape == args[0].shape
    S.close(got.reshape(want.shape), want, bound, "advantages")


@pytest.mark.parametrize("order", [(0, 1, 2), (1, 0, 2), (2, 0, 1), (0, 2, 1), (1, 2, 0), (2, 1, 0)])
def test_layouts(order):
    """Channels that are not adjacent in any of the inputs, environments first, steps last."""
    g = gen(502)
    val, rew, nxt = (torch.randn(T, N, 3, generator=g) for _ in range(3))
    done = (torch.rand(T, N, generator=g) < 0.15).long()
    back = [order.index(i) for i in range(3)]
    place = [t.permute(order).contiguous().to(DEV).permute(back) for t in (val, rew, nxt)]
    want, bound = loop(done, val, rew, nxt)
    S.close(discount_values(done.to(DEV), *place, 0.99, 0.95), want, bound, "advantages")
    flat = [t[..., 0] for t in place]
    S.close(discount_values(done.t().contiguous().to(DEV).t(), *flat, 0.99, 0.95), want[..., 0], bound[..., 0], "advantages")


def test_flags_of_every_value_are_refused():
    x = torch.zeros(T, N, 3, device=DEV)
    with pytest.raises(ValueError, match="expected shape"):
        discount_values(torch.zeros(T, N, 3, dtype=torch.int64, device=DEV), x, x, x, 0.99, 0.95)
