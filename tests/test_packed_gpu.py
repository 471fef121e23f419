"""Prefill of packed rows: each sequence's rows are the bits of a call of its own, which are compared with attention in
64 bits; rows outside every sequence stay as they were; and whole steps over ragged batches with tables kept on the GPU."""
import pytest
import torch

from helpers import BF, D
from q8_ref import F8, attend, to_slices

pytestmark = pytest.mark.gpu
PAGE = 16
SCALE = D ** -0.5


def ropes(n, base=1e7):
    inv = base ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()


def level_table(base=1e7, k_ret=2.0):
    from atflash import atflash_window as AW
    return list(AW.window_zhi_from_kret(D, base, k_ret, 1 << 20))


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def cumulate(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def rows(seed, dev, *shapes):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(s, generator=g, device=dev).to(BF) for s in shapes]


def paged(k, v, lens, dev, rope=None, kv_dtype=BF):
    """A cache holding sequences of these lengths (rows of k and v one after the other) on scattered pages."""
    from atflash import interface
    from atflash.cache import PagedKVCache
    need = [-(-n // PAGE) for n in lens]
    width = max(max(need), 1)
    cache = PagedKVCache(sum(need) + 2, k.shape[1], dev, kv_dtype=kv_dtype)
    order = torch.randperm(sum(need) + 2, generator=torch.Generator().manual_seed(len(lens))).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    table = table.to(dev)
    interface.kv_write_packed(cache, k, v, ints(cumulate(lens), dev), max(lens), ints([0] * len(lens), dev), table, rope)
    return cache, table


RAGGED = [[1], [32, 33, 31], [0, 700, 0, 1, 257, 256, 255, 0], [1500, 3, 40]]


@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("hq,hkv", [(6, 2), (28, 4), (4, 4)])
@pytest.mark.parametrize("lens", RAGGED)
def test_whole_prompts_are_the_bits_of_single_calls(dev, lens, hq, hkv, rope):
    from atflash import interface
    T = sum(lens)
    q, k, v = rows(100 + T, dev, (T, hq, D), (T, hkv, D), (T, hkv, D))
    cu = cumulate(lens)
    cs = ropes(max(lens)).to(dev) if rope else None
    for zhi in (None, level_table()):
        out, lse = interface.flash_attn_packed(q, k, v, ints(cu, dev), max(lens), zhi=zhi, rope=cs)
        for b, n in enumerate(lens):
            if n == 0:
                continue
            r = slice(cu[b], cu[b + 1])
            o1, l1 = interface._flash_attn_fwd(q[None, r], k[None, r], v[None, r], atflash_window_zhi=zhi, rope=cs)
            assert torch.equal(out[r], o1[0]) and torch.equal(lse[:, r], l1[0])


def test_a_bound_far_past_the_rows(dev):
    from atflash import interface
    lens = [40, 1, 300]
    q, k, v = rows(7, dev, (341, 4, D), (341, 2, D), (341, 2, D))
    cs, cu = ropes(341).to(dev), ints(cumulate(lens), dev)
    want = interface.flash_attn_packed(q, k, v, cu, 300, zhi=level_table(), rope=cs)
    got = interface.flash_attn_packed(q, k, v, cu, 1 << 20, zhi=level_table(), rope=cs)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("kv_dtype", [BF, F8])
@pytest.mark.parametrize("new,held", [([5, 64, 1, 0, 300], [5, 1000, 700, 90, 333]), ([256, 512], [2000, 512]), ([1], [40])])
def test_queries_behind_cached_prefixes(dev, new, held, kv_dtype):
    # the last `new` of `held` keys: chunks, single tokens, whole prompts in one call
    from atflash import interface
    hq, hkv = 14, 2
    k, v = rows(7, dev, (sum(held), hkv, D), (sum(held), hkv, D))
    (q,) = rows(8, dev, (sum(new), hq, D))
    cs = ropes(max(held)).to(dev)
    cache, table = paged(k, v, held, dev, cs, kv_dtype)
    cu = cumulate(new)
    zhi = level_table(k_ret=0.5)
    out, lse = interface.prefill_packed(q, cache, table, ints(cu, dev), ints(held, dev), max(held), zhi=zhi, rope=cs)
    for b, n in enumerate(new):
        if n == 0:
            continue
        r = slice(cu[b], cu[b + 1])
        o1, l1 = interface.prefill_paged(q[None, r], cache, table[b:b + 1].contiguous(), held[b], held[b] - n, zhi=zhi,
                                         rope=cs)
        assert torch.equal(out[r], o1[0]) and torch.equal(lse[:, r], l1[0])


@pytest.mark.parametrize("k_ret", [None, 0.3])
def test_against_64_bits(dev, k_ret):
    # pre-rotated rows: errors by the roundings of P and of the output (q8_ref.attend); the log-sum-exp by those of
    # 32-bit sums and exponentials, 2^-16 of its terms' magnitudes (scores up to about 8 in size)
    from atflash import interface
    lens, hq, hkv = [130, 1, 515], 6, 2
    q, k, v = rows(9, dev, (sum(lens), hq, D), (sum(lens), hkv, D), (sum(lens), hkv, D))
    cu = cumulate(lens)
    zhi = None if k_ret is None else level_table(k_ret=k_ret)
    out, lse = interface.flash_attn_packed(q, k, v, ints(cu, dev), max(lens), zhi=zhi)
    lims = None if zhi is None else [1 << 30] * 2 + [z for z in zhi[1:] for _ in range(2)]
    for b, n in enumerate(lens):
        ks, vs = to_slices(k[cu[b]:cu[b + 1]]), v[cu[b]:cu[b + 1]]
        for i in sorted({0, n // 3, n // 2, n - 1}):
            pos = torch.arange(i + 1, device=dev)
            age = (i // 32 * 32 - (pos // 32 * 32 + 31)).clamp(min=0)[:, None].expand(-1, 16)
            want, bound = attend(to_slices(q[cu[b] + i]), ks[:i + 1], vs[:i + 1], lims, age, SCALE, False)
            assert ((out[cu[b] + i].double() - want).abs() <= bound).all()
            kk = ks[:i + 1].double()
            if lims is not None:
                kk = kk * (age <= torch.tensor(lims, device=dev)).repeat_interleave(8, -1)[:, None]
            s = torch.stack([kk[:, h * hkv // hq] @ to_slices(q[cu[b] + i, h]).double() for h in range(hq)]) * SCALE
            ref = torch.logsumexp(s, -1)
            assert ((lse[:, cu[b] + i].double() - ref).abs() <= 2.0 ** -16 * (s.abs().amax(-1) + ref.abs() + 1)).all()


def test_many_sequences(dev):
    # more than 64, so that the plan counts them in several rounds; equal and empty ones among them
    from atflash import interface
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 90, (150,), generator=g).tolist() + [0] * 3 + [64] * 20 + [900, 128, 128]
    hq, hkv, T = 4, 1, sum(lens)
    q, k, v = rows(10, dev, (T, hq, D), (T, hkv, D), (T, hkv, D))
    cu = cumulate(lens)
    out, lse = interface.flash_attn_packed(q, k, v, ints(cu, dev), max(lens))
    for b in [0, 1, 63, 64, 65, 100, 149, 153, 172, 173, 174, 175]:
        if lens[b]:
            r = slice(cu[b], cu[b + 1])
            o1, l1 = interface._flash_attn_fwd(q[None, r], k[None, r], v[None, r])
            assert torch.equal(out[r], o1[0]) and torch.equal(lse[:, r], l1[0])
    assert torch.isfinite(out.float()).all() and torch.isfinite(lse).all()


def test_the_plan_lists_every_tile_once_heaviest_first(dev):
    from atflash import interface
    hq, r = 64, 256
    new, held = [700, 0, 40, 256, 1, 128, 300], [700, 9, 5000, 256, 257, 384, 2900]
    T = sum(new)
    plan = interface.packed_plan(ints(cumulate(new), dev), ints(held, dev), T, 5000, hq)
    tiles = plan.tiles.tolist()
    n = tiles[0]
    got = [(tiles[2 + 2 * i], tiles[3 + 2 * i]) for i in range(n)]
    assert plan.tiles.numel() == 2 + 2 * (T // r + len(new))
    keys = {(b, i): h - m + min(m, (i + 1) * r) for b, (m, h) in enumerate(zip(new, held)) for i in range(-(-m // r))}
    assert got == sorted(keys, key=lambda t: (-keys[t], t[0]))


def test_rows_outside_every_sequence_stay_as_they_were(dev):
    # rows before the first and behind the last sequence; sequences whose lengths do not fit
    from atflash import interface
    hq, hkv, T = 4, 2, 300
    held = [100, 20, 90, 400]
    k, v = rows(11, dev, (sum(held), hkv, D), (sum(held), hkv, D))
    (q,) = rows(12, dev, (T, hq, D))
    cache, table = paged(k, v, held, dev)
    cu = [10, 60, 90, 120, 250]           # sequence 1: 30 queries of 20 keys; sequence 3: 400 keys, more than 128
    out = torch.full((T, hq, D), 7.0, dtype=BF, device=dev)
    lse = torch.full((hq, T), 5.0, device=dev)
    got = interface.prefill_packed(q, cache, table, ints(cu, dev), ints(held, dev), 128, out=out, lse=lse)
    assert got[0] is out and got[1] is lse
    for a, b in ((0, 10), (60, 90), (120, 300)):
        assert (out[a:b] == 7.0).all() and (lse[:, a:b] == 5.0).all()
    for s in (0, 2):
        r = slice(cu[s], cu[s + 1])
        n = cu[s + 1] - cu[s]
        o1, l1 = interface.prefill_paged(q[None, r], cache, table[s:s + 1].contiguous(), held[s], held[s] - n)
        assert torch.equal(out[r], o1[0]) and torch.equal(lse[:, r], l1[0])


@pytest.mark.parametrize("cu", [[0, 50, 20, 80], [-40, 30, 60, 10 ** 6], [90, 70, 50, 10]])
def test_first_rows_that_make_no_sense_stay_in_bounds(dev, cu):
    from atflash import interface
    q, k, v = rows(13, dev, (80, 2, D), (80, 1, D), (80, 1, D))
    out, lse = interface.flash_attn_packed(q, k, v, ints(cu, dev), 80)
    torch.cuda.synchronize()
    assert out.shape == (80, 2, D) and lse.shape == (2, 80)


def test_strided_rows_of_one_projection(dev):
    from atflash import interface
    lens, hq, hkv = [77, 200], 6, 2
    T = sum(lens)
    (x,) = rows(14, dev, (T, (hq + 2 * hkv) * D + 16))
    q, k, v = (x[:, a * D:b * D].view(T, b - a, D) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    cu = ints(cumulate(lens), dev)
    got = interface.flash_attn_packed(q, k, v, cu, 200)
    want = interface.flash_attn_packed(q.contiguous(), k.contiguous(), v.contiguous(), cu, 200)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    sorted_pair = interface.flash_attn_packed(q, k, v, cu, 200, layout="sorted_pair")
    assert torch.isfinite(sorted_pair[0].float()).all()


def test_captured_steps_follow_the_lengths(dev):
    # one graph, other lengths and rows at every replay; the plan is made inside
    from atflash import interface
    hq, hkv, T = 12, 4, 600
    q, k, v = rows(15, dev, (T, hq, D), (T, hkv, D), (T, hkv, D))
    cu = ints([0, 100, 600], dev)
    zhi = level_table()
    interface.flash_attn_packed(q, k, v, cu, T, zhi=zhi)  # (outside capture first: the LDS attribute)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = interface.flash_attn_packed(q, k, v, cu, T, zhi=zhi)
    for i, lens in enumerate(([100, 500], [600, 0], [1, 599], [300, 300])):
        cu.copy_(ints(cumulate(lens), dev))
        for x, y in zip((q, k, v), rows(16 + i, dev, (T, hq, D), (T, hkv, D), (T, hkv, D))):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        want = interface.flash_attn_packed(q, k, v, cu, T, zhi=zhi)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_registered_operators(dev):
    from atflash import ops
    held, new = [100, 40], [60, 40]
    k, v = rows(18, dev, (140, 2, D), (140, 2, D))
    (q,) = rows(19, dev, (100, 4, D))
    cache, table = paged(k, v, held, dev)
    cu, n = ints([0, 60, 100], dev), ints(held, dev)
    want = ops.prefill_packed(q, cache.kv, table, cu, n, 100, level_table(), SCALE, None, 0)
    got = torch.ops.atflash.prefill_packed(q, cache.kv, table, cu, n, 100, level_table(), SCALE, None, 0)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_plan_shared_by_layers_and_its_refusals(dev):
    from atflash import interface
    hq, hkv, held = 48, 4, [900, 40, 300]
    T = sum(held)
    q, k, v = rows(22, dev, (T, hq, D), (T, hkv, D), (T, hkv, D))
    cache, table = paged(k, v, held, dev)
    cu, n = ints(cumulate(held), dev), ints(held, dev)
    plan = interface.packed_plan(cu, n, T, 900, hq)
    want = interface.prefill_packed(q, cache, table, cu, n, 900)
    for _ in range(2):
        got = interface.prefill_packed(q, cache, table, cu, n, 900, plan=plan)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for args in ((q[:-1], cu, n, 900), (q[:, :24], cu, n, 900), (q, cu.clone(), n, 900), (q, cu, None, 900), (q, cu, n, 901)):
        with pytest.raises(ValueError):
            interface.prefill_packed(args[0], cache, table, *args[1:], plan=plan)
    # other lengths in the same tensors: refreshed, right again; a stale list stays in bounds
    for lens in ([300, 500, 440], [1240, 0, 0]):
        cu.copy_(ints(cumulate(lens), dev))
        n.copy_(ints(lens, dev))
        interface.prefill_packed(q, cache, table, cu, n, 900, plan=plan)
        plan.refresh()
        got = interface.prefill_packed(q, cache, table, cu, n, 900, plan=plan)
        torch.cuda.synchronize()
        want = interface.prefill_packed(q, cache, table, cu, n, 900)
        for b, m in enumerate(lens):
            if 0 < m <= 900:  # (a sequence of 1240 keys is past the call's 900: not computed)
                r = slice(sum(lens[:b]), sum(lens[:b]) + m)
                assert torch.equal(got[0][r], want[0][r])


def test_two_streams_at_once(dev):
    from atflash import interface
    a = rows(20, dev, (500, 8, D), (500, 2, D), (500, 2, D))
    b = rows(21, dev, (700, 8, D), (700, 2, D), (700, 2, D))
    cu = [ints([0, 100, 500], dev), ints([0, 640, 700], dev)]
    want = [interface.flash_attn_packed(*x, c, 640) for x, c in zip((a, b), cu)]
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for x, c, st in zip((a, b), cu, s):
        with torch.cuda.stream(st):
            got.append(interface.flash_attn_packed(*x, c, 640))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


@pytest.mark.parametrize("kv_dtype", [BF, F8])
def test_a_serving_loop_with_tables_on_the_gpu(dev, kv_dtype):
    """Prompts admitted together, decode steps, a chunk beside single tokens, sequences released and others admitted on
    their pages: every step's outputs are those of the same calls with tables from the host."""
    from atflash import interface
    from atflash.cache import PagedKVCache, PageTables
    hq, hkv, batch, width, pages = 8, 2, 4, 12, 30
    cs = ropes(width * PAGE).to(dev)
    zhi = level_table(k_ret=0.5)
    tabs = PageTables(pages, batch, width, dev)
    cache, host = PagedKVCache(pages, hkv, dev, kv_dtype=kv_dtype), PagedKVCache(pages, hkv, dev, kv_dtype=kv_dtype)
    lens = [0] * batch
    for b in range(batch):
        host.add_sequence(b)

    def step(seed, new):
        T = sum(new)
        q, k, v = rows(seed, dev, (T, hq, D), (T, hkv, D), (T, hkv, D))
        start, cu, pos, slots = tabs.extend(ints(new, dev), T)
        assert start.tolist() == lens and cu.tolist() == cumulate(new)
        for b, n in enumerate(new):
            lens[b] += n
            host.reserve(b, lens[b])
        table = host.page_table(range(batch), width)
        assert torch.equal(tabs.page_table, table) and tabs.seq_lens.tolist() == lens
        interface.kv_write_packed(cache, k, v, cu, max(new), start, tabs.page_table, cs)
        interface.kv_write_packed(host, k, v, ints(cumulate(new), dev), max(new),
                                  ints([n - m for n, m in zip(lens, new)], dev), table, cs)
        at = 0
        for b, n in enumerate(new):
            p = torch.arange(lens[b] - n, lens[b])
            assert pos[at:at + n].tolist() == p.tolist()
            assert slots[at:at + n].tolist() == (table[b].cpu().long()[p // PAGE] * PAGE + p % PAGE).tolist()
            at += n
        if max(new) == 1 and all(n == 1 for n in new):
            got = interface.decode_paged(q, cache, tabs.page_table, tabs.seq_lens, width * PAGE, zhi=zhi, rope=cs)
            want = interface.decode_paged(q, host, table, ints(lens, dev), width * PAGE, zhi=zhi, rope=cs)
            assert torch.equal(got, want)
        else:
            got, _ = interface.prefill_packed(q, cache, tabs.page_table, cu, tabs.seq_lens, width * PAGE, zhi=zhi, rope=cs)
            for b, n in enumerate(new):
                if n:
                    r = slice(sum(new[:b]), sum(new[:b]) + n)
                    want, _ = interface.prefill_paged(q[None, r], host, table[b:b + 1].contiguous(), lens[b], lens[b] - n,
                                                      zhi=zhi, rope=cs)
                    assert torch.equal(got[r], want[0])

    step(1, [40, 17, 1, 100])
    for i in range(20):
        step(2 + i, [1, 1, 1, 1])
    step(50, [1, 60, 1, 1])
    tabs.release(ints([3, 1, 3], dev))
    for b in (3, 1):
        host.free_sequence(b)
        host.add_sequence(b)
        lens[b] = 0
    host._free = tabs.free_pages[:int(tabs.free_count)].tolist()
    assert sorted(host._free + [p for b in (0, 2) for p in host.pages[b]]) == list(range(pages))
    step(51, [1, 90, 1, 33])
    step(52, [1, 1, 1, 1])
