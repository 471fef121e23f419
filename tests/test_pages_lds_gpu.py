"""Shared tables at pool sizes around those where a kernel's LDS passes 64 KB in all: the bit maps by themselves, or with what the kernel
has besides them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("pool", [240000, 244900, 245600, 250000, 261000, 262144, 262145, 262200])
def test_compact(dev, pool):
    from atflash import ops
    table, lens = ints([[pool - 1, 7, -1], [pool - 2, pool - 3, 0]], dev), ints([32, 47], dev)
    free = ints([pool - 5, 3, 2, 9, -1], dev)
    out, left_pages, left, src, dst, n = ops.compact_tables(table, lens, free, ints([4], dev), pool)
    assert n.item() == 3 and src[:3].tolist() == [pool - 1, pool - 2, pool - 3] and dst[:3].tolist() == [2, 3, 9]
    assert out.tolist() == [[2, 7, -1], [3, 9, 0]]
    assert left.item() == 4 and left_pages.tolist() == [pool - 1, pool - 2, pool - 3, pool - 5, -1]


@pytest.mark.parametrize("batch,pool", [(3, 300), (8, 2 ** 19), (8191, 262000), (8191, 262145), (8191, 262176), (8191, 262177), (8191, 2 ** 19)])
def test_select(dev, batch, pool):
    from atflash import ops
    table = torch.full((batch, 2), -1, dtype=torch.int32, device=dev)
    lens = torch.zeros(batch, dtype=torch.int32, device=dev)
    table[0, 0], table[1, 0], table[1, 1] = pool - 1, pool - 2, 5
    lens[0], lens[1] = 16, 20
    parents = torch.full((batch,), -1, dtype=torch.int32, device=dev)
    parents[1], parents[2] = 1, 1
    free = ints([8, 3, -1], dev)
    out, new, left, src, dst = ops.select_tables(table, lens, free, ints([2], dev), parents, pool)
    assert free.tolist() == [8, 3, pool - 1] and left.item() == 2
    assert out[:3].tolist() == [[-1, -1], [pool - 2, 5], [pool - 2, pool - 1]] and new[:3].tolist() == [0, 20, 20]
    assert src[:3].tolist() == [-1, -1, 5] and dst[:3].tolist() == [-1, -1, pool - 1]
    assert (out[3:] == -1).all() and (new[3:] == 0).all() and (src[3:] == -1).all()
