"""Forks, drops, beams and compaction of page tables, and copies of pages, against lists on the host."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
PAGE = 16


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def pages_of(n, width):
    return min(-(-max(n, 0) // PAGE), width)


def host_select(table, lens, free, count, parents, pool):
    """(table, lengths, free pages, pages left, copies' sources, destinations) by the rules, row by row."""
    B, W, F = len(table), len(table[0]), len(free)
    free, count = list(free), min(max(count, 0), F)
    rows, new, named, asks = [], [], set(), []
    for b, p in enumerate(parents):
        row = [-1] * W
        new.append(0)
        if 0 <= p < B:
            n = max(lens[p], 0)
            whole, have = min(n // PAGE, W), pages_of(n, W)
            row[:whole] = table[p][:whole]
            new[-1] = n
            if have > whole:
                keeper = p if parents[p] == p else min(i for i in range(B) if parents[i] == p)
                last = table[p][whole]
                if keeper == b:
                    row[whole] = last
                elif 0 <= last < pool:
                    asks.append((b, whole, last))
            named.update(x for x in row if x >= 0)
        rows.append(row)
    gone = {x for r, n in zip(table, lens) for x in r[:pages_of(n, W)] if 0 <= x < pool} - named
    for x in sorted(gone):
        if count < F:
            free[count] = x
            count += 1
    src, dst, left = [-1] * B, [-1] * B, count
    for b, col, last in asks:
        left -= 1
        page = free[left] if left >= 0 else -1
        rows[b][col] = page
        if 0 <= page < pool:
            src[b], dst[b] = last, page
    return rows, new, free, left, src, dst


def state(seed, B, W, max_len, pool, shared=True):
    """Tables in which some rows begin with others' whole pages; the other pages are free."""
    r = random.Random(seed)
    ids = list(range(pool))
    r.shuffle(ids)
    table, lens = [[-1] * W for _ in range(B)], []
    for b in range(B):
        n = min(r.choice([0, r.randint(0, max_len), r.randint(0, max_len), PAGE * r.randint(0, max_len // PAGE)]), W * PAGE)
        have, like = pages_of(n, W), r.randrange(b) if b and shared else None
        common = min(n // PAGE, lens[like] // PAGE, r.randint(0, W)) if like is not None else 0
        need = have - common
        if need > len(ids):
            n, have, common, need = 0, 0, 0, 0
        if common:
            table[b][:common] = table[like][:common]
        table[b][common:have] = [ids.pop() for _ in range(need)]
        lens.append(n)
    return table, lens, ids


def run_select(dev, table, lens, free, parents, pool, room=0, count=None):
    from atflash import ops
    t, n, c = ints(table, dev), ints(lens, dev), ints([len(free) if count is None else count], dev)
    f = ints(list(free) + [-7] * room, dev)
    want = host_select(table, lens, f.tolist(), int(c), parents, pool)
    for _ in range(2):  # the call's inputs are read only: the same again
        out = ops.select_tables(t, n, f, c, ints(parents, dev), pool)
        got = (out[0].tolist(), out[1].tolist(), f.tolist(), int(out[2]), out[3].tolist(), out[4].tolist())
        for g, w in zip(got, want):
            assert g == w
        assert t.tolist() == table and n.tolist() == lens
    return want


@pytest.mark.parametrize("B,W,max_len,pool", [(1, 1, 16, 3), (2, 3, 40, 20), (5, 9, 140, 60), (8, 300, 4500, 3000), (33, 70, 1000, 2500),
                                              (64, 4100, 9000, 40000), (1000, 6, 90, 7000), (1025, 3, 40, 4000), (8191, 2, 30, 20000)])
@pytest.mark.parametrize("kind", ["beams", "forks", "drops", "same"])
def test_select(dev, B, W, max_len, pool, kind):
    table, lens, free = state(B + W, B, W, max_len, pool)
    r = random.Random(B)
    parents = {"beams": [r.randrange(B) for _ in range(B)], "forks": [b if r.random() < 0.7 else r.randrange(B) for b in range(B)],
               "drops": [b if r.random() < 0.5 else r.choice([-1, B, -5, 2 ** 31 - 1]) for b in range(B)],
               "same": list(range(B))}[kind]
    want = run_select(dev, table, lens, free, parents, pool, room=pool - len(free))
    if kind == "same":
        assert want[2][:len(free)] == free and want[3] == len(free) and set(want[4]) == {-1}


def test_every_row_from_one_and_all_dropped(dev):
    table, lens, free = state(3, 40, 30, 400, 900)
    lens[7], table[7] = 299, table[7]
    have = pages_of(299, 30)
    table[7] = [free.pop() for _ in range(have)] + [-1] * (30 - have)
    run_select(dev, table, lens, free, [7] * 40, 900, room=900)
    run_select(dev, table, lens, free, [-1] * 40, 900, room=900)


def test_pages_run_out_and_a_full_list(dev):
    table, lens, free = state(4, 12, 20, 300, 200)
    r = random.Random(1)
    for left in (0, 1, 3):
        run_select(dev, table, lens, free[:left], [r.randrange(4) for _ in range(12)], 200)      # no room for what becomes free
        run_select(dev, table, lens, free[:left], [r.randrange(4) for _ in range(12)], 200, room=2)
        run_select(dev, table, lens, free[:left], [0] + [r.randrange(4) for _ in range(11)], 200, room=200, count=-2)
    run_select(dev, table, lens, [], [b // 2 for b in range(12)], 200)


def test_entries_that_are_no_pages_and_strange_lengths(dev):
    table, lens, free = state(5, 20, 9, 140, 200)
    lens[1], lens[2], lens[3] = -9, 16 * 9 + 70, 100
    table[2] = [free.pop() for _ in range(9)]
    table[3] = [free.pop() for _ in range(7)] + [-1, -1]
    table[3][6] = 200           # the last page of a row that is filled in part
    table[4][0] = -1
    lens[5], table[5][:2] = 40, [-3, 5000]
    parents = [3, 3, 2, 2, 4, 5, 5, 1, 3] + list(range(9, 20))
    run_select(dev, table, lens, free, parents, 200, room=200)
    run_select(dev, table, lens, free, [9 if b in (2, 3, 5) else b for b in range(20)], 200, room=200)


def test_a_large_pool(dev):
    table, lens, free = state(6, 9, 9000, 140000, 80000)
    pool = 2 ** 19
    far = {x: pool - 1 - 6 * x for x in range(80000)}  # ids over the whole pool
    table = [[far.get(x, -1) for x in r] for r in table]
    free = [far[x] for x in free]
    run_select(dev, table, lens, free, [0, 0, 2, 2, 8, 1, 1, 8, 8], pool, room=pool - len(free))


# ---- compaction ----

def host_compact(table, lens, free, count, pool):
    W = len(table[0])
    live = {x for r, n in zip(table, lens) for x in r[:pages_of(n, W)] if 0 <= x < pool}
    ids = sorted(live | {x for x in free[:max(count, 0)] if 0 <= x < pool})
    low, rest = ids[:len(live)], ids[len(live):]
    dst, src = [x for x in low if x not in live], [x for x in reversed(rest) if x in live]
    to = dict(zip(src, dst))
    rows = [[to.get(x, x) if i < pages_of(n, W) else -1 for i, x in enumerate(r)] for r, n in zip(table, lens)]
    return rows, rest[::-1], src, dst


def run_compact(dev, table, lens, free, pool, room=0):
    from atflash import ops
    t, n, f, c = ints(table, dev), ints(lens, dev), ints(list(free) + [3] * room, dev), ints([len(free)], dev)
    rows, rest, src, dst = host_compact(table, lens, f.tolist(), len(free), pool)
    assert len(src) == len(dst)
    for _ in range(2):
        out = ops.compact_tables(t, n, f, c, pool)
        assert out[0].tolist() == rows
        assert int(out[2]) == len(rest) and out[1].tolist() == (rest + [-1] * (f.numel() - len(rest)))[:f.numel()]
        assert int(out[5]) == len(src)
        pad = [-1] * (out[3].numel() - len(src))
        assert out[3].numel() == max(1, pool // 2) and out[3].tolist() == src + pad and out[4].tolist() == dst + pad
        assert t.tolist() == table and int(c) == len(free)
    return rows, rest, src, dst


@pytest.mark.parametrize("B,W,max_len,pool", [(1, 1, 16, 1), (1, 1, 16, 2), (2, 3, 40, 20), (5, 9, 140, 60), (8, 300, 4500, 3000),
                                              (33, 70, 1000, 2500), (64, 410, 6000, 33000), (1000, 6, 90, 7000), (8191, 2, 30, 20000)])
def test_compact(dev, B, W, max_len, pool):
    table, lens, free = state(B + W, B, W, max_len, pool)
    rows, rest, src, _ = run_compact(dev, table, lens, free, pool, room=pool - len(free))
    used = {x for r in rows for x in r if x >= 0}
    assert used == set(range(len(used))) and rest == list(range(pool - 1, len(used) - 1, -1))
    run_compact(dev, rows, lens, rest, pool)  # nothing moves
    held = free[::3]  # pages held elsewhere: neither in a row nor free
    rows, rest, _, _ = run_compact(dev, table, lens, [x for x in free if x not in set(held)], pool, room=3)
    assert not set(held) & ({x for r in rows for x in r} | set(rest))


def test_compact_empty_full_and_strange(dev):
    run_compact(dev, [[-1] * 5] * 3, [0, 0, 0], list(range(30)), 30)
    run_compact(dev, [[29 - 5 * b - i for i in range(5)] for b in range(6)], [80] * 6, [], 30, room=4)
    table, lens, free = state(7, 20, 9, 140, 200)
    lens[1], lens[2] = -5, 999
    table[2] = [free.pop() for _ in range(9)]
    table[3][0], table[4][0] = 200, -9
    run_compact(dev, table, lens, free + [free[0], -2, 777] + [x for x in table[2][:2]], 200, room=9)


def test_compact_a_large_pool(dev):
    pool = 2 ** 19
    table, lens, free = state(6, 9, 9000, 140000, 80000)
    far = {x: pool - 1 - 6 * x for x in range(80000)}
    table = [[far.get(x, -1) for x in r] for r in table]
    rest = sorted(set(range(pool)) - {x for r in table for x in r})
    random.Random(2).shuffle(rest)
    run_compact(dev, table, lens, rest, pool)


# ---- copies ----

@pytest.mark.parametrize("shapes", [[(40, 2, 2, 2048)], [(40, 4, 2, 2048)] * 30, [(40, 3, 2)], [(40, 5)], [(40, 8, 2, 2048), (40, 8, 2), (40, 1),
                                    (40, 7, 4)] * 40])
@pytest.mark.parametrize("n", [1, 9, 20])
def test_copy_pages(dev, shapes, n):
    from atflash import ops
    g = torch.Generator(device=dev).manual_seed(n)
    caches = [torch.randint(-128, 128, s, generator=g, device=dev, dtype=torch.int8) for s in shapes]
    if len(shapes) == 1 and len(shapes[0]) == 4:
        caches = [torch.randn(s, generator=g, device=dev).to(torch.bfloat16) for s in shapes]
    ids = torch.randperm(40, generator=torch.Generator().manual_seed(n))[:2 * n].tolist()
    src, dst = ids[:n], ids[n:]
    want = [c.clone() for c in caches]
    for w in want:
        w[dst] = w[src]
    # pairs that are none lie between the others and are left out
    s = [x for p in zip(src, [-1, 5, 40, 2 ** 31 - 1, 3] * 4) for x in p]
    d = [x for p in zip(dst, [6, -1, 3, 7, 40] * 4) for x in p]
    ops.copy_pages(caches, ints(s, dev), ints(d, dev))
    for c, w in zip(caches, want):
        assert torch.equal(c, w)


def test_copy_counted_pairs(dev):
    from atflash import ops
    for count in (-3, 0, 2, 5, 99):
        c = torch.arange(30 * 64, device=dev, dtype=torch.int32).view(30, 64)
        want = c.clone()
        k = min(max(count, 0), 5)
        want[[20, 21, 22, 23, 24][:k]] = want[[1, 2, 3, 4, 5][:k]]
        ops.copy_pages([c], ints([1, 2, 3, 4, 5], dev), ints([20, 21, 22, 23, 24], dev), ints([count], dev))
        assert torch.equal(c, want)
    ops.copy_pages([], ints([1], dev), ints([2], dev))
    ops.copy_pages([c], ints([], dev), ints([], dev))


def test_copy_past_32_bits(dev):
    from atflash import ops
    c = torch.zeros((3, 3 * 2 ** 30), dtype=torch.uint8, device=dev)
    c[1, ::4096] = torch.arange(3 * 2 ** 18, device=dev).to(torch.uint8)
    c[1, -1] = 77
    ops.copy_pages([c], ints([1], dev), ints([2], dev))
    assert torch.equal(c[2], c[1]) and c[0].eq(0).all()


# ---- together ----

def test_tables_of_beams_keep_their_tokens(dev):
    """Steps of extend, write, select, drop and compact on GPU tables; a cache whose pages hold the token's number, so that every
    sequence's history can be read back."""
    from atflash.cache import PageTables
    r = random.Random(5)
    B, pool = 6, 60
    tabs = PageTables(pool, B, 12, dev, sharing=True)
    caches = [torch.full((pool, PAGE), -1, dtype=torch.int32, device=dev) for _ in range(2)]
    hist, nxt = [[] for _ in range(B)], 0
    for step in range(60):
        new = [r.choice([0, 1, 1, 3, 17]) if len(h) < 100 else 0 for h in hist]
        _, _, _, slots = tabs.extend(ints(new, dev), sum(new))
        vals = list(range(nxt, nxt + sum(new)))
        nxt += sum(new)
        for c in caches:
            c.view(-1)[slots] = ints(vals, dev)
        for h, m in zip(hist, new):
            h += vals[:m]
            vals = vals[m:]
        what = r.choice(["beams", "drop", "none", "compact", "fork"])
        if what == "beams":
            parents = [r.randrange(B) for _ in range(B)]
        elif what == "fork":
            parents = [b if r.random() < 0.6 else r.randrange(B) for b in range(B)]
        if what in ("beams", "fork"):
            tabs.select(ints(parents, dev), caches)
            hist = [list(hist[p]) for p in parents]
        elif what == "drop":
            gone = r.sample(range(B), 2)
            tabs.release(ints(gone + [B, -1], dev))
            hist = [[] if b in gone else h for b, h in enumerate(hist)]
        elif what == "compact":
            tabs.compact(caches)
            used = {x for row in tabs.page_table.tolist() for x in row if x >= 0}
            assert used == set(range(len(used)))
        assert tabs.seq_lens.tolist() == [len(h) for h in hist]
        table = tabs.page_table.tolist()
        free = tabs.free_pages[:int(tabs.free_count)].tolist()
        used = {x for row in table for x in row if x >= 0}
        assert len(free) == len(set(free)) and not used & set(free) and len(used) + len(free) == pool
        for c in caches:
            flat = c.cpu()
            for b, h in enumerate(hist):
                got = [int(flat[table[b][t // PAGE], t % PAGE]) for t in range(len(h))]
                assert got == h, (step, what, b)


def test_captured_steps(dev):
    from atflash.cache import PageTables
    tabs, ref = (PageTables(40, 4, 8, dev, sharing=True) for _ in range(2))
    for t in (tabs, ref):
        t.extend(ints([20, 33, 5, 16], dev), 74)
    parents = ints([0, 1, 2, 3], dev)
    cache, want = (torch.arange(40 * 64, device=dev, dtype=torch.int32).view(40, 64).clone() for _ in range(2))
    warm = PageTables(40, 4, 8, dev, sharing=True)
    warm.select(parents, [cache])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tabs.select(parents, [cache])
        moved = tabs.compact([cache])
    r = random.Random(2)
    for _ in range(12):
        parents.copy_(ints([r.randrange(4) for _ in range(4)], dev))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ref.select(parents, [want])
        n = ref.compact([want])
        for a, b in zip((tabs.page_table, tabs.seq_lens, tabs.free_count, moved, cache), (ref.page_table, ref.seq_lens, ref.free_count, n, want)):
            assert torch.equal(a, b)
        assert torch.equal(tabs.free_pages[:int(ref.free_count)], ref.free_pages[:int(ref.free_count)])
        more = ints([r.choice([0, 1, 9]) for _ in range(4)], dev)
        for t in (tabs, ref):
            t.extend(more, 36)
        if int(ref.seq_lens.max()) > 100:
            for t in (tabs, ref):
                t.release(ints([0, 1, 2, 3], dev))


def test_captured_calls_on_a_large_pool(dev):
    from atflash import ops
    pool = 2 ** 19
    table, lens, free = state(11, 5, 300, 4700, 5000)
    far = {x: pool - 1 - 100 * x for x in range(5000)}
    t, n = ints([[far.get(x, -1) for x in r] for r in table], dev), ints(lens, dev)
    f, c, parents = ints([far[x] for x in free] + [0] * 5000, dev), ints([len(free)], dev), ints([0, 0, 2, 1, -1], dev)
    args = (t, n, f, c)
    want = (ops.select_tables(*args, parents, pool), ops.compact_tables(*args, pool))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = (ops.select_tables(*args, parents, pool), ops.compact_tables(*args, pool))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((*want[0], *want[1]), (*got[0], *got[1])):
            assert torch.equal(a, b)


def test_registered_operators(dev):
    from atflash import ops
    table, lens, free = state(9, 6, 9, 140, 100)
    args = [ints(x, dev) for x in (table, lens, free + [0] * (100 - len(free)), [len(free)])]
    copy = [x.clone() for x in args]
    parents = ints([1, 1, 0, 3, 3, -1], dev)
    for a, b in zip(ops.select_tables(*args, parents, 100), torch.ops.atflash.select_tables(*copy, parents, 100)):
        assert torch.equal(a, b)
    assert torch.equal(args[2], copy[2])
    a, b = ops.compact_tables(*args, 100), torch.ops.atflash.compact_tables(*args, 100)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    c = torch.arange(6400, device=dev, dtype=torch.int32).view(100, 64)
    d = c.clone()
    ops.copy_pages([c], a[3], a[4], a[5])
    torch.ops.atflash.copy_pages([d], a[3], a[4], a[5])
    assert torch.equal(c, d)
