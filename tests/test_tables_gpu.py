"""Block tables and slot maps built on the GPU against lists on the host."""
import pytest
import torch

pytestmark = pytest.mark.gpu
PAGE = 16


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def host_extend(table, lens, new, free, total, num_pages):
    """The same on lists.  Returns (table, lengths, free pages left, first tokens, positions, slots)."""
    table, free = [list(r) for r in table], list(free)
    short, after, cu, pos, slot = 0, [], [0], [], []
    for row, n, m in zip(table, lens, new):
        n, m = max(n, 0), max(m, 0)
        for p in range(-(-n // PAGE), min(-(-(n + m) // PAGE), len(row))):
            if free:
                row[p] = free.pop()
            else:
                row[p] = -1
                short += 1
        after.append(n + m)
        cu.append(cu[-1] + m)
        for t in range(n, n + m):
            pg = row[t // PAGE] if t // PAGE < len(row) else -1
            pos.append(t)
            slot.append(pg * PAGE + t % PAGE if 0 <= pg < num_pages else -1)
    pos, slot = pos[:total], slot[:total]
    pad = [-1] * (total - len(pos))
    return table, after, len(free) - short, cu, pos + pad, slot + pad


def case(seed, batch, width, max_len, max_new, pool, spare):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, max_len + 1, (batch,), generator=g).tolist()
    new = torch.randint(0, max_new + 1, (batch,), generator=g).tolist()
    ids = torch.randperm(pool, generator=g).tolist()
    table = [[-1] * width for _ in range(batch)]
    for b, n in enumerate(lens):
        for p in range(min(-(-n // PAGE), width)):
            table[b][p] = ids.pop()
    return table, lens, new, ids[:spare]


def check(dev, table, lens, new, free, total, num_pages, room=3):
    from atflash import ops
    t = ints(table, dev)
    pages = ints(free + [12345] * room, dev)  # entries past the count are not pages
    lens_t, new_t, count = ints(lens, dev), ints(new, dev), ints([len(free)], dev)
    want = host_extend(table, lens, new, free, total, num_pages)
    for _ in range(2):  # lengths and free pages are read only: the same again
        out = ops.extend_tables(t, lens_t, new_t, pages, count, total, num_pages)
        got = (t.tolist(), out[0].tolist(), int(out[1]), out[2].tolist(), out[3].tolist(), out[4].tolist())
        for g, w in zip(got, want):
            assert g == w
    assert out[4].dtype == torch.int64 and count.tolist() == [len(free)] and lens_t.tolist() == lens


@pytest.mark.parametrize("batch,width,max_len,max_new,pool,spare", [
    (1, 1, 0, 1, 4, 4), (1, 300, 100, 4000, 300, 290), (3, 9, 60, 60, 40, 25), (64, 70, 1000, 1, 5000, 70),
    (255, 12, 90, 80, 4000, 2000), (256, 12, 90, 80, 4000, 2000), (257, 12, 90, 80, 4000, 2000),
    (1000, 8, 60, 40, 9000, 3000), (8191, 4, 30, 9, 40000, 8000)])
def test_extend(dev, batch, width, max_len, max_new, pool, spare):
    table, lens, new, free = case(batch, batch, width, max_len, max_new, pool, spare)
    check(dev, table, lens, new, free, sum(new), pool)


def test_pages_run_out(dev):
    table, lens, new, free = case(5, 40, 20, 100, 100, 500, 60)
    check(dev, table, lens, new, free, sum(new), 500)
    check(dev, table, lens, new, [], sum(new), 500, room=0)


@pytest.mark.parametrize("total", [0, 1, 300, 5000])
def test_fewer_and_more_rows_than_new_tokens(dev, total):
    table, lens, new, free = case(6, 30, 20, 100, 100, 700, 400)
    check(dev, table, lens, new, free, total, 700)


def test_tables_that_are_too_narrow_and_lengths_below_zero(dev):
    table, lens, new, free = case(7, 30, 5, 120, 90, 700, 400)
    lens[3], new[4], lens[5], new[5] = -7, -5, -1, -1
    table[6][0], table[7][0] = 700, -3  # entries outside the pool: no slots
    check(dev, table, lens, new, free, sum(max(n, 0) for n in new), 700)


def test_lengths_past_31_bits_stay_in_bounds(dev):
    from atflash import ops
    top = 2 ** 31 - 1
    table = ints([[3, 1, 0, 2], [4, -1, -1, -1]], dev)
    free = ints([9, 8, 7, 6, 5], dev)
    lens, left, cu, pos, slot = ops.extend_tables(table, ints([top, 5], dev), ints([5, 20], dev), free, ints([5], dev), 25, 10)
    assert lens.tolist() == [top, 25] and cu.tolist() == [0, 5, 25] and int(left) == 4
    assert table.tolist() == [[3, 1, 0, 2], [4, 5, -1, -1]]
    assert slot[:5].tolist() == [-1] * 5 and pos[5:].tolist() == list(range(5, 25))
    assert slot[5:].tolist() == [(4 if t < 16 else 5) * 16 + t % 16 for t in range(5, 25)]
    # sums of new tokens that wrap: whatever is listed is -1 or a slot of the pool
    lens, left, cu, pos, slot = ops.extend_tables(table, ints([top, 5], dev), ints([top, top], dev), free, ints([5], dev), 60, 10)
    assert lens.tolist() == [top, top] and int(left) == 2 and table[1].tolist() == [4, 5, 6, 7]
    assert all(-1 <= x < 160 for x in slot.tolist())


def test_release(dev):
    from atflash import ops
    batch, width, pool = 6, 40, 200
    table, lens, _, free = case(8, batch, width, 600, 0, pool, 20)
    lens[2] = 0
    table[2] = [-1] * width
    short = -(-lens[4] // PAGE) - 1
    table[4][short] = -1  # the row ran out of pages
    rows = [4, 1, 9, 4, 2, -1, 0]
    want, left = list(free), [list(r) for r in table]
    for b in (4, 1, 2, 0):
        want += [p for p in table[b][:-(-lens[b] // PAGE)] if p >= 0]
        left[b][:-(-lens[b] // PAGE)] = [-1] * -(-lens[b] // PAGE)
    t, n, pages, count = ints(table, dev), ints(lens, dev), ints(free + [0] * (pool - len(free)), dev), ints([len(free)], dev)
    ops.release_tables(t, n, pages, count, ints(rows, dev), pool)
    assert int(count) == len(want) and pages[:len(want)].tolist() == want and t.tolist() == left
    assert n.tolist() == [0, 0, 0, lens[3], 0, lens[5]]
    ops.release_tables(t, n, pages, count, ints([], dev), pool)
    assert int(count) == len(want)


def test_release_after_running_out_and_into_a_full_list(dev):
    from atflash import ops
    t, n, count = ints([[0, 1, -1, -1]], dev), ints([60], dev), ints([-2], dev)
    pages = ints([9, 9, 9], dev)
    ops.release_tables(t, n, pages, count, ints([0], dev), 3)
    assert int(count) == 2 and pages.tolist() == [0, 1, 9] and t.tolist() == [[-1] * 4]
    t, n, count = ints([[5, 6, 7, 8]], dev), ints([64], dev), ints([1], dev)
    pages = ints([4, 9, 9, 77], dev)
    ops.release_tables(t, n, pages[:3], count, ints([0], dev), 10)
    assert int(count) == 3 and pages.tolist() == [4, 5, 6, 77]


def test_captured_decode_steps(dev):
    # one graph that extends the tables by a token each; replayed over page borders
    from atflash.cache import PageTables
    tabs, ref = PageTables(50, 3, 10, dev), PageTables(50, 3, 10, dev)
    one = ints([1, 1, 1], dev)
    first = ints([14, 1, 33], dev)
    for t in (tabs, ref):
        t.extend(first, 48)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        start, cu, pos, slots = tabs.extend(one, 3)
    for i in range(40):
        graph.replay()
        torch.cuda.synchronize()
        want = ref.extend(one, 3)
        for a, b in zip((start, cu, pos, slots, tabs.page_table, tabs.seq_lens, tabs.free_count),
                        (*want, ref.page_table, ref.seq_lens, ref.free_count)):
            assert torch.equal(a, b)
    assert tabs.seq_lens.tolist() == [54, 41, 73]


def test_registered_operators(dev):
    from atflash import ops
    table, lens, new, free = case(9, 5, 20, 100, 100, 200, 90)
    a = [ints(x, dev) for x in (table, lens, new, free, [len(free)])]
    b = [x.clone() for x in a]
    want = ops.extend_tables(*a, sum(new), 200)
    got = torch.ops.atflash.extend_tables(*b, sum(new), 200)
    for x, y in zip((*want, a[0]), (*got, b[0])):
        assert torch.equal(x, y)
    for f, x in ((ops.release_tables, a), (torch.ops.atflash.release_tables, b)):
        f(x[0], x[1], x[3], x[4], ints([1, 3], dev), 200)
    assert torch.equal(a[0], b[0]) and torch.equal(a[4], b[4])
