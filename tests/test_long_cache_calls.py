"""The long-cache calls' host checks on the CPU, where they need no device tensors."""
import ctypes
import random

import pytest
import torch


@pytest.fixture(scope="module")
def eager(pkg):
    from breeze_tts_2_flash_amd import kernels
    return kernels.eager()


def elements(t, base):
    """The bytes that a view of `base` holds."""
    at = torch.zeros(t.shape, dtype=torch.int64)
    for i, (n, step) in enumerate(zip(t.shape, t.stride())):
        at += (torch.arange(n) * step).view([-1 if j == i else 1 for j in range(t.dim())])
    size = t.element_size()
    return {t.data_ptr() - base.data_ptr() + size * p + k for p in at.flatten().tolist() for k in range(size)}


def test_apart_side_by_side(eager):
    """K and V as halves of one tensor, in any of its dims, share nothing; shifted over one another they do."""
    for shape, dim in [((2, 3, 2, 5, 8), 0), ((3, 2, 2, 5, 8), 1), ((3, 2, 2, 5, 8), 2), ((3, 2, 5, 2, 8), 3)]:
        kv = torch.zeros(shape)
        k, v = kv.select(dim, 0), kv.select(dim, 1)
        assert eager.apart(k, v) and eager.apart(v, k), (shape, dim)
        assert not eager.apart(k, k) and not eager.apart(v, v[..., :1].expand_as(v)), (shape, dim)
    kv = torch.zeros(3, 5, 2, 2, 8).permute(0, 2, 1, 3, 4)  # [B, capacity, NKV, 2, D]
    assert eager.apart(kv[:, :, :, 0], kv[:, :, :, 1])
    one = torch.zeros(3, 2, 64 * 68, dtype=torch.uint8)  # a head's codes, then its scales
    codes = one.as_strided((3, 2, 64, 64), (2 * 64 * 68, 64 * 68, 64, 1))
    scales = one.as_strided((3, 2, 64, 4), (2 * 64 * 68, 64 * 68, 4, 1), 64 * 64)
    assert eager.apart(codes, scales) and not eager.apart(codes, one.as_strided(scales.shape, scales.stride(), 64 * 64 - 1))
    rows = torch.zeros(2, 3, 10, 8)
    assert not eager.apart(rows[:, :, :9], rows[:, :, 1:]) and eager.apart(rows[:, :, :5], rows[:, :, 5:])
    assert eager.apart(rows[:, :, ::2], rows[:, :, 1::2]) and eager.apart(rows[:, :1], rows[:, 2:])


def test_apart_against_brute_force(eager):
    """Never apart where two views share a byte; and apart wherever both are slices of one tensor that share none."""
    rng = random.Random(1)
    base = torch.zeros(6000, dtype=torch.uint8)
    shared = 0
    for _ in range(1500):
        if rng.random() < 0.5:  # any strides
            views = []
            for _ in range(2):
                sizes = [rng.randint(1, 4) for _ in range(4)]
                steps = [rng.choice([1, 2, 3, 7, 8, 16, 40, 64, 130, 200]) for _ in range(4)]
                views.append(base.as_strided(sizes, steps, rng.randint(0, 60)))
            exact = False
        else:  # the same steps, over slices
            whole = base[:4 * 3 * 5 * 6].view(4, 3, 5, 6).permute(*rng.sample(range(3), 3), 3)
            views = [whole[tuple(slice(lo, rng.randint(lo + 1, n)) for n in whole.shape for lo in [rng.randint(0, n - 1)])]
                     for _ in range(2)]
            exact = all(n > 1 for v in views for n in v.shape)
        meet = bool(elements(views[0], base) & elements(views[1], base))
        apart = eager.apart(*views)
        assert not (apart and meet), (views[0].shape, views[0].stride(), views[1].shape, views[1].stride())
        if exact:
            assert apart != meet, (views[0].shape, views[1].shape)
        shared += meet
    assert 100 < shared < 1400


@pytest.mark.parametrize("kind,T", [(0, 1), (1, 1), (1, 16), (2, 1)])
def test_workspaces_of_large_batches_have_one_layout(pkg, kind, T):
    """The counters take a power of two of lines, so that batches of many sizes can use one workspace."""
    lib, n = pkg.load(), ctypes.c_size_t(0)

    def size(B, splits):
        assert lib.bz_long_workspace_size(kind, B, 16, 8, 128, 4096, T, 0, 0, splits, 0, ctypes.byref(n)) == 0
        return n.value

    up = lambda x: (x + 255) // 256 * 256  # noqa: E731
    columns = 2 * T  # of a (row, kv head), by two q heads
    tiles = -(-T // 8)
    for units in (8, 64, 512, 520, 528, 1016, 1024, 1032, 2048, 4000):
        B = units // 8 // tiles
        if B == 0:
            continue
        lines = 512
        while lines < B * 8 * tiles:
            lines *= 2
        cols = B * 8 * columns * 2
        want = up(up(lines * 256 + cols * 8) + cols * 128 * 4)
        if kind == 2:
            want = up(want + B * 16 * 8) + B * 16 * 4096 * 4
        assert size(B, 2) == want, units
