"""The paged cache of 8-bit floats: its writer against the plain restatement (codes and exponents to the bit), its
expansion, and the decode and prefill over it against attention in 64 bits on the values that the codes stand for."""
import pytest
import torch

from helpers import BF, D, randn_bf16
from q8_ref import Cache, E_MIN, F8, U_F8, ages, attend, rotate32, to_slices

pytestmark = pytest.mark.gpu
PAGE = 16
SCALE = D ** -0.5


def ropes(n, base=5e5):
    inv = base ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()


def tables(base=5e5, k_ret=2.0):
    from atflash import atflash_window as AW, fiwin_common as FW
    return list(AW.window_zhi_from_kret(D, base, k_ret, 1 << 20)), FW.zhi_slice_vec8(D, base, k_ret).tolist()


def new_cache(pages, heads, dev):
    from atflash.cache import PagedKVCache
    return PagedKVCache(pages, heads, dev, kv_dtype=F8)


def same_as(cache, ref, pages=None):
    from atflash.cache import dequantize
    ids = list(range(ref.k.shape[0])) if pages is None else pages
    k, v = dequantize(cache.kv, cache.exps, ids)
    assert torch.equal(cache.exps.cpu().int()[ids], ref.e[ids])
    for got, want in ((k.cpu(), ref.k[ids]), (v.cpu(), ref.v[ids])):
        assert torch.equal(torch.nan_to_num(got, nan=12345.0), torch.nan_to_num(want, nan=12345.0))


def row_of(pages, dev):
    return torch.tensor(pages, dtype=torch.int32, device=dev)


# ---------------------------------------------------------------- the writer

@pytest.mark.parametrize("layout,rope", [(0, True), (0, False), (1, False)])
@pytest.mark.parametrize("n,start", [(1, 0), (1, 15), (1, 16), (16, 0), (17, 0), (33, 7), (5, 14), (200, 3)])
def test_writer_codes_and_exponents(dev, n, start, layout, rope):
    from atflash import ops
    g = torch.Generator().manual_seed(n * 100 + start)
    heads, total = 3, start + n
    pages = -(-total // PAGE) + 2
    order = torch.randperm(pages, generator=g)[: -(-total // PAGE)].tolist()
    cs = ropes(total) if rope else None
    ref, cache = Cache(pages, heads), new_cache(pages, heads, dev)
    calls = ([(0, start)] if start else []) + [(start, n)]
    for at, m in calls:
        k = randn_bf16((1, m, heads, D), g) * (1.0 if at == 0 else 3.0)
        v = randn_bf16((1, m, heads, D), g)
        ops.kv_write_q8(cache.kv, cache.exps, k.to(dev), v.to(dev), row_of([at], dev), row_of([order], dev),
                        None if cs is None else cs.to(dev), layout)
        ref.write(k[0], v[0], at, order, cs, layout)
    same_as(cache, ref)


def test_codes_are_the_nearest(dev):
    # against 64 bits: at most half a step, of the value or of the smallest normal code
    from atflash import ops
    from atflash.cache import dequantize
    g = torch.Generator().manual_seed(5)
    n, heads = 320, 4
    k, v, cs = randn_bf16((n, heads, D), g), randn_bf16((n, heads, D), g), ropes(n)
    cache = new_cache(n // PAGE, heads, dev)
    ops.kv_write_q8(cache.kv, cache.exps, k[None].to(dev), v[None].to(dev), row_of([0], dev),
                    row_of([list(range(n // PAGE))], dev), cs.to(dev), 0)
    gk, gv = (x.cpu().double().flatten(0, 1) for x in dequantize(cache.kv, cache.exps, range(n // PAGE)))
    c, s = cs[:, None, :, 0].double(), cs[:, None, :, 1].double()
    a, b = k[..., :64].double(), k[..., 64:].double()
    want_k = to_slices(torch.cat([a * c - b * s, b * c + a * s], -1))
    step = torch.exp2(cache.exps.cpu().double()).repeat_interleave(PAGE, 0)
    for got, want, half in ((gk, want_k, 1), (gv, v.double(), 0)):
        unit = step[:, :, half, None]
        # the fp32 rotation adds at most 3 roundings of 2^-24 of the pair's magnitude (5)
        slack = torch.maximum(want.abs(), unit * 2.0 ** -6) * U_F8 + 5 * 3 * 2.0 ** -24
        assert ((got - want).abs() <= slack).all()


def test_tokens_one_by_one_and_growing_magnitudes(dev):
    # every append raises the page's exponent: kept codes are shifted, some to subnormals
    from atflash import ops
    g = torch.Generator().manual_seed(11)
    heads, n = 2, 40
    order = [4, 0, 2]
    cs = ropes(n)
    ref, cache = Cache(5, heads), new_cache(5, heads, dev)
    for t in range(n):
        k, v = (randn_bf16((1, 1, heads, D), g) * 1.7 ** (t % 23) for _ in range(2))
        k, v = k.to(BF), v.to(BF)
        ops.kv_write_q8(cache.kv, cache.exps, k.to(dev), v.to(dev), row_of([t], dev), row_of([order], dev), cs.to(dev), 0)
        ref.write(k[0], v[0], t, order, cs)
        if t % 7 == 0 or t == n - 1:
            same_as(cache, ref)


def test_rewriting_forgets_what_lay_behind(dev):
    from atflash import ops
    g = torch.Generator().manual_seed(12)
    heads, order = 2, [1, 3, 0]
    ref, cache = Cache(4, heads), new_cache(4, heads, dev)
    for at, m, scale in ((0, 45, 8.0), (20, 3, 0.5), (32, 2, 0.25), (16, 1, 0.1)):
        k, v = ((randn_bf16((1, m, heads, D), g) * scale).to(BF) for _ in range(2))
        ops.kv_write_q8(cache.kv, cache.exps, k.to(dev), v.to(dev), row_of([at], dev), row_of([order], dev), None, 0)
        ref.write(k[0], v[0], at, order, None)
        same_as(cache, ref)


@pytest.mark.parametrize("kind", ["inf", "nan", "huge", "tiny", "zero", "all_nan"])
def test_special_values(dev, kind):
    from atflash import ops
    g = torch.Generator().manual_seed(13)
    heads = 2
    k, v = (randn_bf16((1, 24, heads, D), g) for _ in range(2))
    if kind == "inf":
        k[0, 3, 0, 5], v[0, 17, 1, 100] = float("inf"), float("-inf")
    elif kind == "nan":
        k[0, 0, 1, 0], v[0, 23, 0, 127] = float("nan"), float("nan")
    elif kind == "all_nan":
        k[:], v[:] = float("nan"), float("nan")
    elif kind == "zero":
        k[:], v[:] = 0, 0
    else:
        f = 2.0 ** 125 if kind == "huge" else 2.0 ** -120
        k, v = (k * f).to(BF), (v * f).to(BF)
        assert torch.isfinite(k).all()
    ref, cache = Cache(2, heads), new_cache(2, heads, dev)
    ops.kv_write_q8(cache.kv, cache.exps, k.to(dev), v.to(dev), row_of([0], dev), row_of([[1, 0]], dev), None, 0)
    ref.write(k[0], v[0], 0, [1, 0], None)
    same_as(cache, ref)


def test_what_cannot_be_placed_is_skipped(dev):
    # negative positions, positions past the page table and the RoPE table, entries outside the pool
    from atflash import ops
    g = torch.Generator().manual_seed(14)
    heads, cs = 2, ropes(40)
    starts, table = [-5, 30, 10, 0], [[0, 1, 2], [3, 4, -1], [5, 99, 6], [-7, 7, 8]]
    ref, cache = Cache(9, heads), new_cache(9, heads, dev)
    k, v = (randn_bf16((4, 30, heads, D), g) for _ in range(2))
    ops.kv_write_q8(cache.kv, cache.exps, k.to(dev), v.to(dev), row_of(starts, dev), row_of(table, dev), cs.to(dev), 0)
    for b in range(4):
        ref.write(k[b], v[b], starts[b], table[b], cs)
    same_as(cache, ref)


def packed_case(seed, lens, starts, heads, width):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens)
    k, v = (randn_bf16((T, heads, D), g) for _ in range(2))
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    perm = torch.randperm(len(lens) * width, generator=g).view(len(lens), width).to(torch.int32)
    return k, v, cu, perm


@pytest.mark.parametrize("lens,starts", [([1, 1, 1], [0, 15, 33]), ([0, 5, 70, 0, 16], [9, 0, 3, 1, 32]), ([130], [0])])
def test_packed_rows(dev, lens, starts):
    from atflash import ops
    from atflash.cache import new_kv_cache
    heads, width = 3, 9
    k, v, cu, table = packed_case(21, lens, starts, heads, width)
    cs = ropes(width * PAGE)
    pages = len(lens) * width
    ref, cache = Cache(pages, heads), new_cache(pages, heads, dev)
    kv, kv_rect = new_kv_cache(pages, heads, dev), new_kv_cache(pages, heads, dev)
    args = (k.to(dev), v.to(dev), row_of(cu, dev), max(lens), row_of(starts, dev), table.to(dev), cs.to(dev), 0)
    ops.kv_write_packed(cache.kv, cache.exps, *args)
    ops.kv_write_packed(kv, None, *args)
    for b, n in enumerate(lens):
        rows = slice(cu[b], cu[b + 1])
        ref.write(k[rows], v[rows], starts[b], table[b].tolist(), cs)
        if n:
            ops.kv_write(kv_rect, k[None, rows].to(dev), v[None, rows].to(dev), row_of(starts[b:b + 1], dev),
                         table[b:b + 1].to(dev), cs.to(dev), 0)
    same_as(cache, ref)
    assert torch.equal(kv.view(torch.int16), kv_rect.view(torch.int16))


def test_packed_rows_outside_the_tensor_are_not_read(dev):
    # first rows that do not fit the tensor are cut to it; more tokens than max_tokens are left out
    from atflash import ops
    heads, width = 2, 4
    k, v, _, table = packed_case(22, [40], [0], heads, 3 * width)
    table = table.view(3, width)
    cu, starts = [-3, 10, 35, 90], [0, 0, 0]
    ref, cache = Cache(12, heads), new_cache(12, heads, dev)
    ops.kv_write_packed(cache.kv, cache.exps, k.to(dev), v.to(dev), row_of(cu, dev), 20, row_of(starts, dev),
                        table.contiguous().to(dev), None, 0)
    for b, (lo, hi) in enumerate(((0, 10), (10, 30), (35, 40))):
        ref.write(k[lo:hi], v[lo:hi], 0, table[b].tolist(), None)
    same_as(cache, ref)


def test_strided_sources(dev):
    from atflash import ops
    g = torch.Generator().manual_seed(23)
    heads, n = 3, 37
    qkv = randn_bf16((n, 5 * heads, D + 8), g).to(dev)
    k, v = qkv[:, heads:2 * heads, :D], qkv[:, 3 * heads:4 * heads, :D]
    table = row_of([[2, 0, 1]], dev)
    a, b = new_cache(3, heads, dev), new_cache(3, heads, dev)
    cu, zero = row_of([0, n], dev), row_of([0], dev)
    ops.kv_write_packed(a.kv, a.exps, k, v, cu, n, zero, table, None, 0)
    ops.kv_write_packed(b.kv, b.exps, k.contiguous(), v.contiguous(), cu, n, zero, table, None, 0)
    assert torch.equal(a.kv.view(torch.uint8), b.kv.view(torch.uint8)) and torch.equal(a.exps, b.exps)


# ---------------------------------------------------------------- codes as bf16

def test_expansion_is_exact_for_every_code(dev):
    # all 256 codes at exponents over the whole range, against the conversion of torch
    from atflash import ops
    from atflash.cache import dequantize, k_half, v_half
    exps = [E_MIN, -100, -30, -1, 0, 1, 7, 60, 119]
    heads = 2
    cache = new_cache(len(exps), heads, dev)
    codes = torch.arange(256, dtype=torch.uint8).repeat(len(exps) * heads * 2 * 8).view(len(exps), heads, 2, 2048)
    cache.kv.view(torch.uint8).copy_(codes)
    cache.exps.copy_(torch.tensor(exps, dtype=torch.int8)[:, None, None].expand(-1, heads, 2))
    table = torch.tensor([[8, 3, -1, 4], [7, 0, 1, 99], [2, 5, 6, -2]], dtype=torch.int32, device=dev)
    kv, out_table = ops.kv_expand_q8(cache.kv, cache.exps, table, 4)
    live = [(i, int(p)) for i, p in enumerate(table.flatten().tolist()) if 0 <= p < len(exps)]
    want_table = [i if (i, int(p)) in live else -1 for i, p in enumerate(table.flatten().tolist())]
    assert out_table.flatten().tolist() == want_table
    k, v = dequantize(cache.kv, cache.exps, [p for _, p in live])
    rows = [i for i, _ in live]
    # (values past the largest bf16 number exist at the largest exponent only as 448: finite)
    got_k = k_half(kv)[rows].permute(0, 3, 1, 2, 4).flatten(-2).float()          # [n, 16, heads, 128]
    slot = [0, 1, 2, 3, 8, 9, 10, 11, 4, 5, 6, 7, 12, 13, 14, 15]
    got_v = v_half(kv)[rows][..., slot].permute(0, 3, 1, 2).float()
    for got, want in ((got_k, k), (got_v, v)):
        assert torch.equal(torch.nan_to_num(got, nan=1.5), torch.nan_to_num(want, nan=1.5))


def test_expansion_of_the_pages_that_hold_tokens(dev):
    from atflash import ops
    cache = new_cache(6, 2, dev)
    cache.kv.view(torch.uint8).random_(0, 120)
    cache.exps.random_(-4, 5)
    table = torch.tensor([[5, 1, 0], [2, 3, 4], [4, 5, 5], [1, -1, 2]], dtype=torch.int32, device=dev)
    lens = torch.tensor([17, 48, 0, 40], dtype=torch.int32, device=dev)
    all_kv, all_table = ops.kv_expand_q8(cache.kv, cache.exps, table, 3)
    kv, out = ops.kv_expand_q8(cache.kv, cache.exps, table, 3, lens)
    assert out.tolist() == [[0, 1, -1], [3, 4, 5], [-1, -1, -1], [9, -1, 11]]
    live = out[out >= 0].long()
    assert torch.equal(kv[live], all_kv[live]) and all_table.tolist()[2] == [6, 7, 8]


# ---------------------------------------------------------------- decode

def filled(lens, heads, dev, seed, spare=3):
    """A cache with random codes for sequences of these lengths on scattered pages, values in `k`, `v` per sequence."""
    from atflash import ops
    from atflash.cache import dequantize
    g = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-n // PAGE) for n in lens]
    width = max(max(need), 1)
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    table = table.to(dev)
    cache = new_cache(sum(need) + spare, heads, dev)
    keys = []
    for b, n in enumerate(lens):
        if n:
            x = torch.randn((2, 1, n, heads, D), generator=g, device=dev).to(BF)
            ops.kv_write_q8(cache.kv, cache.exps, x[0], x[1], row_of([0], dev), table[b:b + 1], None, 0)
        ids = table[b, :need[b]].long()
        k, v = dequantize(cache.kv, cache.exps, ids)
        keys.append((k.flatten(0, 1)[:n], v.flatten(0, 1)[:n]))
    return cache, table, keys


def check_decode(dev, lens, hq, hkv, seed, kind, layout=0, rope=False, base=5e5, k_ret=2.0, max_len=None, subset=None):
    from atflash import interface
    cache, table, keys = filled(lens, hkv, dev, seed)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    q = torch.randn((len(lens), hq, D), generator=g, device=dev).to(BF)
    n_max = max(max(lens), 1) if max_len is None else max_len
    if table.shape[1] * PAGE < n_max:
        table = torch.nn.functional.pad(table, (0, -(-n_max // PAGE) - table.shape[1]), value=-1).contiguous()
    level, vec8 = tables(base, k_ret)
    zhi = {"off": None, "level": level, "vec8": vec8}[kind]
    cs = ropes(n_max, base).to(dev) if rope else None
    out = interface.decode_paged(q, cache, table, row_of(lens, dev), n_max, zhi=zhi, rope=cs,
                                 layout="half_split" if layout == 0 else "sorted_pair")
    for b in subset if subset is not None else range(len(lens)):
        n = lens[b]
        if n == 0:
            assert (out[b] == 0).all()
            continue
        qq = q[b][None]
        if rope:
            c, s = cs[n - 1, :, 0].double(), cs[n - 1, :, 1].double()
            x, y = qq[..., :64].double(), qq[..., 64:].double()
            qq = torch.cat([x * c - y * s, y * c + x * s], -1)
        lims = None if zhi is None else (vec8 if kind == "vec8" else [min(z, 1 << 30) for z in level for _ in range(2)])
        if kind == "level":
            lims = [1 << 30] * 2 + lims[2:]
        want, bound = attend(to_slices(qq[0], layout), *keys[b], lims, ages(n, "key" if kind == "vec8" else "page", dev),
                             SCALE, rope)
        err = (out[b].double() - want).abs()
        assert (err <= bound).all(), (b, n, float((err / bound).max()))
    return out, (q, cache, table, zhi, cs)


@pytest.mark.parametrize("kind", ["off", "level", "vec8"])
@pytest.mark.parametrize("hq,hkv", [(8, 8), (6, 2), (28, 4), (16, 1)])
@pytest.mark.parametrize("lens", [[1], [15, 16, 17], [300, 1, 0, 77], [1003], [4099, 2000]])
def test_decode(dev, lens, hq, hkv, kind):
    check_decode(dev, lens, hq, hkv, 31 + len(lens) + lens[0], kind)


@pytest.mark.parametrize("kind,layout,rope", [("vec8", 0, True), ("level", 0, True), ("vec8", 1, False), ("off", 1, False)])
def test_decode_layouts_and_rope(dev, kind, layout, rope):
    check_decode(dev, [2500, 130, 1], 24, 8, 47, kind, layout, rope)


@pytest.mark.parametrize("k_ret", [0.05, 0.5, 8.0])
def test_decode_slice_boundaries(dev, k_ret):
    # narrow windows: many boundaries inside pages, odd slice counts, keys past every slice
    check_decode(dev, [901, 333, 48, 5], 12, 4, 53, "vec8", rope=True, base=1e7, k_ret=k_ret)


@pytest.mark.parametrize("kind,layout,rope", [("vec8", 0, True), ("level", 1, False), ("off", 0, True)])
@pytest.mark.parametrize("lens", [[600, 1, 0, 577, 32, 384, 385, 511, 16, 600, 200, 33, 590, 592, 593, 600, 15, 17, 100, 400],
                                  [5003, 4096, 700, 1], [33, 3000, 1, 2999, 1500, 0, 2000, 16, 700, 1024, 2900, 256]])
def test_decode_every_form_of_a_launch(dev, lens, kind, layout, rope):
    # 24 / 8 heads: one split a head of up to 38 pages; 8 splits of 40 pages; more workgroups than CUs
    check_decode(dev, lens, 24, 8, 67, kind, layout, rope)


def test_decode_longer_bound_than_the_lengths(dev):
    check_decode(dev, [40, 7, 0], 8, 2, 59, "vec8", max_len=9000)


def test_decode_ragged_batch(dev):
    # sequences of one split and of many in a call; their results do not depend on the others'
    lens = [700, 9000, 33000, 1, 12000, 20000, 0, 31000, 16, 32768, 25000, 8000]
    out, (q, cache, table, zhi, cs) = check_decode(dev, lens, 24, 8, 61, "vec8", rope=True, subset=[0, 3, 6, 8, 9])
    from atflash import interface
    others = [33000 if i == 2 else 5 if i % 2 == 0 else n for i, n in enumerate(lens)]
    again = interface.decode_paged(q, cache, table, row_of(others, dev), 33000, zhi=zhi, rope=cs)
    for b in (1, 3, 5, 7, 9, 11):
        assert torch.equal(again[b], out[b])


def test_missing_pages_score_zero_and_hold_nothing(dev):
    # an entry outside the pool: keys and values of zero, as in the bf16 decode
    from atflash import interface
    cache, table, keys = filled([100], 2, dev, 67)
    table[0, 2], table[0, 4] = -1, 10 ** 6
    q = torch.randn((1, 4, D), generator=torch.Generator(device=dev).manual_seed(3), device=dev).to(BF)
    out = interface.decode_paged(q, cache, table, row_of([100], dev), 100)
    k, v = (x.clone() for x in keys[0])
    for p in (2, 4):
        k[p * PAGE:(p + 1) * PAGE] = 0
        v[p * PAGE:(p + 1) * PAGE] = 0
    want, bound = attend(to_slices(q[0]), k, v, None, None, SCALE, False)
    assert ((out[0].double() - want).abs() <= bound).all()


def test_stale_codes_behind_the_sequence_do_not_matter(dev):
    from atflash import interface
    cache, table, _ = filled([90, 33], 2, dev, 71)
    q = torch.randn((2, 8, D), generator=torch.Generator(device=dev).manual_seed(4), device=dev).to(BF)
    lens = row_of([85, 33], dev)
    want = interface.decode_paged(q, cache, table, lens, 90)
    last = cache.kv.view(torch.uint8)[table[0, 5].long()]       # slots 5.. of the last page: NaN codes
    v = last[:, 0].view(2, 2, 4, 16, 4, 4)
    for t in range(5, 16):
        v[:, :, t // 4, :, :, t % 4] = 0x7f
    last[:, 1].view(2, 8, 16, 16)[:, :, 5:] = 0x7f
    cache.kv.view(torch.uint8)[table[0, 5].long()] = last
    got = interface.decode_paged(q, cache, table, lens, 90)
    assert torch.equal(got, want) and torch.isfinite(got.float()).all()


def test_decode_captured_and_on_another_stream(dev):
    from atflash import interface
    lens = [5000, 1200, 64]
    cache, table, _ = filled(lens, 4, dev, 73)
    q = torch.randn((3, 28, D), generator=torch.Generator(device=dev).manual_seed(5), device=dev).to(BF)
    n = row_of(lens, dev)
    plan = interface.decode_plan(cache, table, n, 5000, 28, zhi=tables()[1])
    want = interface.decode_paged(q, cache, table, n, 5000, zhi=tables()[1])
    assert torch.equal(plan.run(q), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = interface.decode_paged(q, cache, table, n, 5000, zhi=tables()[1])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run(q, out=out)
    for _ in range(3):
        q.copy_(torch.randn((3, 28, D), generator=torch.Generator(device=dev).manual_seed(6), device=dev).to(BF))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, interface.decode_paged(q, cache, table, n, 5000, zhi=tables()[1]))


def test_captured_calls_have_a_workspace_of_their_own(dev):
    from atflash import interface, ops
    cache, table, _ = filled([9000, 300], 2, dev, 74)
    q = torch.randn((2, 8, D), generator=torch.Generator(device=dev).manual_seed(5), device=dev).to(BF)
    n = row_of([9000, 300], dev)
    want = interface.decode_paged(q, cache, table, n, 9000)
    before = dict(ops._DECODE_WS)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(interface.decode_paged(q, cache, table, n, 9000))
        graphs.append(g)
    assert ops._DECODE_WS == before
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_registered_operators(dev):
    from atflash import ops
    g = torch.Generator(device=dev).manual_seed(76)
    k, v = (torch.randn((2, 40, 2, D), generator=g, device=dev).to(BF) for _ in range(2))
    table, start, cs = row_of([[0, 1, 2], [5, 4, 3]], dev), row_of([0, 0], dev), ropes(48).to(dev)
    a, b, c = (new_cache(6, 2, dev) for _ in range(3))
    ops.kv_write_q8(a.kv, a.exps, k, v, start, table, cs, 0)
    torch.ops.atflash.kv_write_q8(b.kv, b.exps, k, v, start, table, cs, 0)
    torch.ops.atflash.kv_write_packed(c.kv, c.exps, k.flatten(0, 1), v.flatten(0, 1), row_of([0, 40, 80], dev), 40, start,
                                      table, cs, 0)
    for x in (b, c):
        assert torch.equal(a.kv.view(torch.uint8), x.kv.view(torch.uint8)) and torch.equal(a.exps, x.exps)
    q = torch.randn((2, 6, D), generator=g, device=dev).to(BF)
    n = row_of([40, 17], dev)
    assert torch.equal(ops.decode_paged_q8(q, a.kv, a.exps, table, n, 48, None, SCALE, cs, 0),
                       torch.ops.atflash.decode_paged_q8(q, a.kv, a.exps, table, n, 48, None, SCALE, cs, 0))
    q = torch.randn((2, 40, 6, D), generator=g, device=dev).to(BF)
    for x, y in zip(ops.prefill_q8(q, a.kv, a.exps, table, 40, 0, None, SCALE, cs, 0),
                    torch.ops.atflash.prefill_q8(q, a.kv, a.exps, table, 40, 0, None, SCALE, cs, 0)):
        assert torch.equal(x, y)


def test_pool_past_4_gib(dev):
    # block offsets past 32 bits: pages at the end of a pool of 4.5 GB
    from atflash import interface, ops
    pages, heads = 160_000, 7
    cache = new_cache(pages, heads, dev)
    n = 50
    g = torch.Generator(device=dev).manual_seed(7)
    k, v = (torch.randn((1, n, heads, D), generator=g, device=dev).to(BF) for _ in range(2))
    far, near = row_of([[pages - 1, pages - 9, 150_000, pages - 2]], dev), row_of([[3, 0, 1, 2]], dev)
    q = torch.randn((1, 14, D), generator=g, device=dev).to(BF)
    outs = []
    for table in (far, near):
        ops.kv_write_q8(cache.kv, cache.exps, k, v, row_of([0], dev), table, None, 0)
        outs.append(interface.decode_paged(q, cache, table, row_of([n], dev), n))
    assert torch.equal(outs[0], outs[1]) and outs[0].abs().max() > 0


# ---------------------------------------------------------------- prefill over the 8-bit cache

@pytest.mark.parametrize("n,nq", [(1, 1), (200, 200), (700, 100)])
def test_prefill_over_the_8_bit_cache(dev, n, nq):
    from atflash import interface
    hq, hkv = 6, 2
    cache, table, keys = filled([n, n], hkv, dev, 83 + n)
    q = torch.randn((2, nq, hq, D), generator=torch.Generator(device=dev).manual_seed(8), device=dev).to(BF)
    out, lse = interface.prefill_paged(q, cache, table, n, n - nq)
    for b in range(2):
        k, v = keys[b]
        for i in sorted({0, nq // 2, nq - 1}):
            m = n - nq + i + 1
            want, bound = attend(to_slices(q[b, i]), k[:m], v[:m], None, None, SCALE, False)
            assert ((out[b, i].double() - want).abs() <= bound).all()


def test_a_prompt_then_single_tokens(dev):
    """As a serving loop uses them: a prompt written and attended to, then tokens appended and decoded one by one."""
    from atflash import interface, ops
    hq, hkv, n, steps = 12, 4, 75, 20
    g = torch.Generator().manual_seed(9)
    cs = ropes(n + steps)
    k, v = (randn_bf16((1, n + steps, hkv, D), g) for _ in range(2))
    q = randn_bf16((1, n + steps, hq, D), g)
    order = [5, 2, 0, 6, 1, 3]
    table = row_of([order], dev)
    cache, ref = new_cache(7, hkv, dev), Cache(7, hkv)
    level, vec8 = tables()
    ops.kv_write_q8(cache.kv, cache.exps, k[:, :n].to(dev), v[:, :n].to(dev), row_of([0], dev), table, cs.to(dev), 0)
    ref.write(k[0, :n], v[0, :n], 0, order, cs)
    out, _ = interface.prefill_paged(q[:, :n].to(dev), cache, table, n, 0, zhi=level, rope=cs.to(dev))
    assert torch.isfinite(out.float()).all()
    for t in range(n, n + steps):
        ops.kv_write_q8(cache.kv, cache.exps, k[:, t:t + 1].to(dev), v[:, t:t + 1].to(dev), row_of([t], dev), table,
                        cs.to(dev), 0)
        ref.write(k[0, t:t + 1], v[0, t:t + 1], t, order, cs)
        got = interface.decode_paged(q[:, t].to(dev), cache, table, row_of([t + 1], dev), t + 1, zhi=vec8, rope=cs.to(dev))
        rows = [(p, s) for p in order for s in range(PAGE)][:t + 1]
        kk = torch.stack([ref.k[p, s] for p, s in rows])
        vv = torch.stack([ref.v[p, s] for p, s in rows])
        qq = to_slices(rotate32(q[0, t][None], torch.tensor([t]), cs)[0])
        want, bound = attend(qq, kk, vv, vec8, ages(t + 1, "key"), SCALE, True)
        assert ((got[0].cpu().double() - want).abs() <= bound).all()
    same_as(cache, ref)
