"""Which tensors share memory: the check in front of the sequence operators' calls, against the sets of their bytes (no GPU
needed)."""
import random
import time

import pytest
import torch

from isaacgym_amd import ops, sequence


def overlap(a, b):
    return sequence._native().overlap(a, b)


def bytes_of(t):
    at = {t.data_ptr()}
    for n, s in zip(t.shape, t.stride()):
        at = {p + i * s * t.element_size() for p in at for i in range(n)}
    return {p + k for p in at for k in range(t.element_size())}


@pytest.mark.parametrize("seed", range(40))
def test_against_the_sets_of_bytes(seed):
    """Views of one buffer with any sizes, strides and types: nested, interleaved, broadcast, windows over themselves."""
    rng = random.Random(seed)
    buf = torch.zeros(4000, dtype=torch.uint8)
    seen = set()
    for _ in range(150):
        views = []
        while len(views) < 2:
            dt = rng.choice([torch.uint8, torch.int16, torch.float32, torch.int64])
            e = torch.empty((), dtype=dt).element_size()
            dims = rng.randint(1, 4)
            sizes = [rng.choice([1, 1, 2, 3, 5, 8]) for _ in range(dims)]
            strides = [rng.choice([0, 1, 1, 2, 3, 5, 7, 12, 20, 30, 64]) for _ in range(dims)]
            reach = sum((n - 1) * s for n, s in zip(sizes, strides)) + 1
            room = buf.numel() // e - reach
            if room < 0:
                continue
            views.append(buf.view(dt).as_strided(sizes, strides, rng.randint(0, room)))
        want = bool(bytes_of(views[0]) & bytes_of(views[1]))
        seen.add(want)
        assert overlap(*views) == want and overlap(*views[::-1]) == want, [(v.shape, v.stride(), v.data_ptr() - buf.data_ptr()) for v in views]
        assert overlap(views[0], views[0])
    assert seen == {True, False}


def test_views_that_a_rollout_is_made_of():
    big = torch.zeros(140, 30, 60)
    a, b, c = big[..., :20], big[..., 20:40], big[..., 40:]
    assert not overlap(a, b) and not overlap(b, c) and not overlap(a, c)
    assert overlap(big[..., :21], b) and overlap(a, big[70])
    assert not overlap(big[::2], big[1::2]) and not overlap(big[::2, :, 4:17], big[1::2, :, 4:17])
    assert overlap(big[::2], big[::3])
    assert not overlap(big[:, ::2], big[:, 1::2]) and not overlap(big[:, :10], big[:, 10:])
    assert not overlap(big[::2, 1:, 5:], big[1::2, :7].transpose(0, 1))
    assert overlap(big[1:], big[:-1]) and not overlap(big[:70], big[70:])
    assert not overlap(big[:0], big) and not overlap(big, torch.zeros(140, 30, 60))
    row = torch.zeros(60)
    assert overlap(row.expand(30, 60), row) and not overlap(row.expand(30, 60)[:, :30], row[30:])


def test_it_is_quick_for_large_tensors():
    """Views of half a million rows that lie between each other's rows, in every order of the strides: no row is visited."""
    big = torch.zeros(1 << 22, dtype=torch.uint8)
    views = [big.as_strided((1 << 10, 1 << 9, 3), (4096, 8, 1), k) for k in (0, 3, 4096 * 0 + 4)]
    views += [big.as_strided((511, 1 << 9, 3), (8192, 8, 1), 4096 + 3), big.as_strided((1 << 9, 1 << 10, 3), (8, 4096, 1), 5)]
    start = time.perf_counter()
    got = [[overlap(a, b) for b in views] for a in views]
    assert time.perf_counter() - start < 0.5
    want = [[True, False, False, False, False], [False, True, True, True, True], [False, True, True, True, True],
            [False, True, True, True, True], [False, True, True, True, True]]
    assert got == want


def test_calls_on_host_tensors_reach_the_check():
    x = torch.zeros(6, 4)
    with pytest.raises(ValueError, match="overlap"):
        ops._apart((x[1:],), (x[:-1],))
    with pytest.raises(ValueError, match="overlap"):
        ops._apart((x[1:], None, x[:2]), (None,))
    ops._apart((x[:3], x[3:]), (None, torch.zeros(3)))
