"""Prefill over an 8-bit cache whose call's bound lies far past its sequences' lengths, or whose sequences share pages: the
temporary bf16 pages are as many as the pool's at most, and the results the same."""
import pytest
import torch

from q8_ref import F8
from test_packed_gpu import D, SCALE, cumulate, ints, level_table, paged, ropes, rows

pytestmark = pytest.mark.gpu


def peak_of(call, dev):
    """(the call's result, bytes that it took at most beyond those in use before)"""
    torch.cuda.synchronize(dev)
    before = torch.cuda.memory_allocated(dev)
    torch.cuda.reset_peak_memory_stats(dev)
    out = call()
    torch.cuda.synchronize(dev)
    return out, torch.cuda.max_memory_allocated(dev) - before


def widened(table, width):
    return torch.nn.functional.pad(table, (0, width - table.shape[1]), value=-1).contiguous()


@pytest.mark.parametrize("whole", [False, True])
def test_a_bound_far_past_the_lengths(dev, whole):
    from atflash import interface
    held = [300, 1, 64, 0, 90, 17, 5, 333] * 2
    new = held if whole else [min(n, 40) for n in held]
    hq, hkv, bound = 6, 2, 65536
    k, v = rows(41, dev, (sum(held), hkv, D), (sum(held), hkv, D))
    (q,) = rows(42, dev, (sum(new), hq, D))
    cs = ropes(bound).to(dev)
    cache, table = paged(k, v, held, dev, cs, F8)
    zhi = level_table(k_ret=0.5)
    cu, n = ints(cumulate(new), dev), None if whole else ints(held, dev)
    want = interface.prefill_packed(q, cache, table, cu, n, max(held), zhi=zhi, rope=cs)
    wide = widened(table, bound // 16)
    got, peak = peak_of(lambda: interface.prefill_packed(q, cache, wide, cu, n, bound, zhi=zhi, rope=cs), dev)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # the pool in bf16, the outputs, and small change; 16 sequences of the bound would be 1 GB
    assert peak <= 2 * cache.kv.numel() + 8 * q.numel() + (1 << 20)


def test_sequences_that_share_their_pages(dev):
    from atflash import interface
    n, nq, hq, hkv, batch = 200, 30, 4, 2, 9
    k, v = rows(43, dev, (n, hkv, D), (n, hkv, D))
    cache, table = paged(k, v, [n], dev, None, F8)
    (q,) = rows(44, dev, (batch, nq, hq, D))
    shared = table.expand(batch, -1).contiguous()
    (out, lse), peak = peak_of(lambda: interface.prefill_paged(q, cache, shared, n, n - nq), dev)
    assert peak <= 2 * cache.kv.numel() + 8 * q.numel() + (1 << 20)
    for b in range(batch):
        o, l = interface.prefill_paged(q[b:b + 1], cache, table, n, n - nq)
        assert torch.equal(out[b], o[0]) and torch.equal(lse[b], l[0])


def test_captured_with_the_tables_full_width(dev):
    from atflash import interface
    held, new, hq, hkv = [100, 40, 7, 64], [20, 40, 1, 3], 4, 2
    k, v = rows(45, dev, (sum(held), hkv, D), (sum(held), hkv, D))
    (q,) = rows(46, dev, (sum(new), hq, D))
    cache, table = paged(k, v, held, dev, None, F8)
    wide, cu, n = widened(table, 64), ints(cumulate(new), dev), ints(held, dev)
    interface.prefill_packed(q, cache, wide, cu, n, 1024)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = interface.prefill_packed(q, cache, wide, cu, n, 1024)
    for i, lens in enumerate(([100, 40, 7, 64], [64, 40, 1, 50], [90, 41, 7, 3])):
        q.copy_(rows(47 + i, dev, q.shape)[0])
        n.copy_(ints(lens, dev))
        graph.replay()
        torch.cuda.synchronize()
        want = interface.prefill_packed(q, cache, wide, cu, n, 1024)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_entries_outside_the_pool_and_refusals(dev):
    from atflash import ops
    held = [100, 60]
    k, v = rows(48, dev, (160, 2, D), (160, 2, D))
    cache, table = paged(k, v, held, dev, None, F8)
    table[0, 2], table[1, 1] = -1, 10 ** 6
    wide = widened(table, 40)
    (q,) = rows(49, dev, (2, 5, 4, D))
    a = ops.prefill_q8(q, cache.kv, cache.exps, table, 60, 55, None, SCALE, None, 0)      # 8 entries of 13 pages
    b = ops.prefill_q8(q, cache.kv, cache.exps, wide, 60, 55, None, SCALE, None, 0)
    kv, used = ops.temporary_bf16(cache.kv, cache.exps, wide, 40, ints(held, dev))
    assert kv.shape == cache.kv.shape and used.data_ptr() == wide.data_ptr()
    c = ops.prefill(q, kv, used, 60, 55, None, SCALE, None, 0)
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)
    for args in ((cache.kv, cache.exps, wide.long(), 40), (cache.kv, cache.exps, wide, 41), (cache.kv, cache.exps[:1], wide, 40),
                 (cache.kv, cache.exps, wide, 40, ints([1], dev)), (cache.kv, cache.exps, wide.cpu(), 40)):
        with pytest.raises(ValueError):
            ops.temporary_bf16(*args)
