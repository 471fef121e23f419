"""Norms into the caches, what test_qk_norm_gpu.py leaves open: the caches that a replayed call writes, and every byte of the 8-bit cache
where some tokens cannot be placed."""
import pytest
import torch

from test_qk_norm_gpu import D, PAGE, exact, ints, packed, table_of

pytestmark = pytest.mark.gpu


def same(a, b):
    return all(x is None and y is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


@pytest.mark.parametrize("lens,starts", [([1, 1, 1], [15, 16, 200]), ([30, 1, 200], [3, 40, 16])])
@pytest.mark.parametrize("eight", [False, True])
def test_replays_write_what_the_call_writes(dev, eight, lens, starts):
    from atflash import cache, ops
    hq, hkv = 6, 2
    q, k, v, qw, kw, cu, start, table, pool, _ = packed(lens, starts, hq, hkv, dev, 8, room=0)
    cs = table_of(400, dev)
    empty = cache.new_kv_cache_q8(pool, hkv, dev) if eight else (cache.new_kv_cache(pool, hkv, dev), None)
    copy = lambda c: [None if t is None else t.clone() for t in c]  # noqa: E731
    kv, exps = copy(empty)
    call = lambda kv, exps: ops.qk_norm_write(kv, exps, q, k, v, qw, kw, 1e-6, cu, max(lens), start, table, cs)  # noqa: E731
    call(kv, exps)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(kv, exps)
    for i in range(4):
        for t in (q, k, v):
            t.copy_(torch.roll(t.clone(), i + 1, 0) * 1.5)
        want_c = copy(empty)
        want = call(*want_c)
        kv.view(torch.uint8).copy_(empty[0].view(torch.uint8))
        if eight:
            exps.copy_(empty[1])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert same((kv, exps), want_c) and not same((kv, exps), empty), i


@pytest.mark.parametrize("room", [0, 2])
def test_tokens_that_cannot_be_placed_in_the_8_bit_cache(dev, room):
    """As test_tokens_that_cannot_be_placed: negative starts, positions past the RoPE table, pages of no pool, columns past the
    table.  K's codes against the formula, its exponents the smallest that hold what is placed, the slots beside it empty, all
    other pages as they were.  A value's tolerance is test_write_q8's."""
    from atflash import cache, ops
    lens, hq, hkv, limit = [20, 20, 40, 20, 7], 4, 2, 104
    starts = [-7, 90, 10, 40, -20]
    q, k, v, qw, kw, cu, start, table, pool, _ = packed(lens, [0, 90, 10, 40, 0], hq, hkv, dev, 77, room)
    start = ints(starts, dev)
    table[2, 1], table[2, 2] = -1, pool + 5
    table = table[:, :6].contiguous()
    cs = table_of(limit, dev)
    T = sum(lens)
    # rows that are not placed are the largest by far: any of them among a page's maximum or codes would show
    pos = torch.cat([torch.arange(s, s + n) for s, n in zip(starts, lens)])
    pages = table.tolist()
    where = [(pages[b][p // PAGE] if 0 <= p < limit and p // PAGE < 6 else -1, p % PAGE)
             for b, (s, n) in enumerate(zip(starts, lens)) for p in range(s, s + n)]
    placed = torch.tensor([0 <= pg < pool for pg, _ in where], device=dev)
    assert placed.any() and not placed.all()
    v[:T][~placed] *= 2.0 ** 20
    k[:T][~placed] = float("nan")
    k[T:], v[T:] = float("inf"), float("inf")
    kv, exps = cache.new_kv_cache_q8(pool, hkv, dev)
    g = torch.Generator(device=dev).manual_seed(9)
    kv.view(torch.uint8).copy_(torch.randint(0, 120, kv.shape, generator=g, device=dev, dtype=torch.uint8))
    exps.copy_(torch.randint(-20, -10, exps.shape, generator=g, device=dev, dtype=torch.int8))
    kv0, exps0 = kv.clone(), exps.clone()
    ops.qk_norm_write(kv, exps, q, k, v, qw, kw, 1e-6, cu, max(lens), start, table, cs)
    ek, off = exact(k[:T], kw, 1e-6, pos.clamp(0, limit - 1).to(dev), cs)
    ev = v[:T].double().cpu()
    got_k, got_v = (t.double().cpu() for t in cache.dequantize(kv, exps, range(pool)))
    old_k, old_v = (t.double().cpu() for t in cache.dequantize(kv0, exps0, range(pool)))
    order = torch.cat([torch.cat([torch.arange(60 - 4 * s, 64 - 4 * s), torch.arange(124 - 4 * s, 128 - 4 * s)]) for s in range(16)])
    e = exps.double().cpu()
    slots = {}
    for i, (pg, slot) in enumerate(where):
        if 0 <= pg < pool:
            slots.setdefault(pg, {})[slot] = i
    for pg in range(pool):
        mine = slots.get(pg)
        if mine is None:
            assert torch.equal(kv[pg].view(torch.uint8), kv0[pg].view(torch.uint8)) and torch.equal(exps[pg], exps0[pg]), pg
            continue
        first, last = min(mine), max(mine)
        assert sorted(mine) == list(range(first, last + 1))
        for h in range(hkv):
            uv, uk = 2.0 ** float(e[pg, h, 0]), 2.0 ** float(e[pg, h, 1])
            for slot in range(PAGE):
                if slot in mine:
                    i = mine[slot]
                    y, o = ek[i, h][order], off[i, h][order]
                    assert ((got_k[pg, slot, h] - y).abs() <= o + (y.abs() + o) * 2.0 ** -4 + uk * 2.0 ** -10).all(), (pg, slot, h)
                    assert ((got_v[pg, slot, h] - ev[i, h]).abs() <= ev[i, h].abs() * 2.0 ** -4 + uv * 2.0 ** -10).all(), (pg, slot, h)
                elif slot > last:
                    assert got_k[pg, slot, h].eq(0).all() and got_v[pg, slot, h].eq(0).all(), (pg, slot, h)
                else:  # kept, perhaps under a larger exponent
                    assert ((got_k[pg, slot, h] - old_k[pg, slot, h]).abs() <= old_k[pg, slot, h].abs() * 2.0 ** -4 + uk * 2.0 ** -10).all()
                    assert ((got_v[pg, slot, h] - old_v[pg, slot, h]).abs() <= old_v[pg, slot, h].abs() * 2.0 ** -4 + uv * 2.0 ** -10).all()
            # the smallest exponent that holds the new values, or what the page had where it keeps codes
            for half, unit, y, o in ((0, uv, ev, torch.zeros_like(ev)), (1, uk, ek, off)):
                rows = list(mine.values())
                top, slack = y[rows, h].abs().max(), o[rows, h].max()
                had = 2.0 ** float(exps0[pg, h, half]) if first > 0 else 0.0
                assert top - slack <= 448 * unit and (unit == had or top + slack > 448 * unit / 2), (pg, h, half)
