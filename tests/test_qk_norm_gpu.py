"""Norm and rotation of queries and keys in one pass, on rows and into the caches, against the formula in 64 bits.

Tolerance of a value z (pair y1, y2 before the rotation): half a bf16 step, 2^-8 |z|, and the fp32 steps before it: 16 + 3
sums of squares (half of their relative error after the root), root, two products and the rotation's two, at most 24
roundings of 2^-24 of |y1| + |y2|.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F8 = torch.bfloat16, torch.float8_e4m3fn
D, P, PAGE = 128, 64, 16


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def table_of(n, dev, base=1e6):
    from atflash import rope as R
    return R.rope_table(n, R.inv_freq(D, base, dev))


def exact(x, w, eps, pos, cs):
    """(z, what the fp32 steps may be off) in 64 bits, on the CPU."""
    x, w = x.double().cpu(), w.double().cpu()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    if cs is None:
        return y, y.abs() * (24 * 2.0 ** -24)
    c, s = cs[pos.long()].double().cpu().unbind(-1)
    c, s = c[:, None], s[:, None]
    a, b = y[..., :P], y[..., P:]
    z = torch.cat([a * c - b * s, b * c + a * s], -1)
    return z, 24 * 2.0 ** -24 * (a.abs() + b.abs()).repeat(1, 1, 2)


def near(got, x, w, eps, pos, cs):
    z, off = exact(x, w, eps, pos, cs)
    bad = (got.double().cpu() - z).abs() > off + (z.abs() + off) * 2.0 ** -8
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values, first at {bad.nonzero()[0].tolist()}"


def rows(T, hq, hk, dev, seed, wtype=BF, fused=True):
    """q, k, v as views of one fused projection (fused), or of tensors of their own; weights."""
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn((T, hq + 2 * hk, D), generator=g, device=dev) * torch.exp(2 * torch.randn((T, 1, 1), generator=g, device=dev))
    x = x.to(BF)
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    if not fused:
        q, k, v = (t.contiguous() for t in (q, k, v))
    w = [(1 + 0.5 * torch.randn(D, generator=g, device=dev)).to(wtype) for _ in range(2)]
    return q, k, v, *w


@pytest.mark.parametrize("T,hq,hk", [(1, 28, 4), (1, 1, 1), (3, 5, 1), (7, 7, 9), (24, 32, 2), (130, 24, 8), (1001, 8, 8), (5000, 28, 4)])
@pytest.mark.parametrize("wtype,fused", [(BF, True), (torch.float32, False)])
def test_rows(dev, T, hq, hk, wtype, fused):
    from atflash import ops
    q, k, _, qw, kw = rows(T, hq, hk, dev, T + hq, wtype, fused)
    cs = table_of(6000, dev)
    pos = torch.randint(0, 6000, (T,), device=dev, dtype=torch.int32, generator=torch.Generator(device=dev).manual_seed(1))
    oq, ok = ops.qk_norm_rope(q, k, qw, kw, 1e-6, pos, cs)
    assert oq.is_contiguous() and ok.is_contiguous() and oq.shape == q.shape and ok.shape == k.shape
    near(oq, q, qw, 1e-6, pos, cs)
    near(ok, k, kw, 1e-6, pos, cs)
    oq, ok = ops.qk_norm_rope(q, k, qw, kw, 1e-5, None, None)  # normed only
    near(oq, q, qw, 1e-5, None, None)
    near(ok, k, kw, 1e-5, None, None)


def test_one_side_without_heads_and_no_rows(dev):
    from atflash import ops
    q, k, _, qw, kw = rows(9, 6, 3, dev, 5)
    cs, pos = table_of(50, dev), torch.arange(9, device=dev, dtype=torch.int32)
    both = ops.qk_norm_rope(q, k, qw, kw, 1e-6, pos, cs)
    oq, none = ops.qk_norm_rope(q, k[:, :0], qw, kw, 1e-6, pos, cs)
    assert torch.equal(oq, both[0]) and none.shape == (9, 0, D)
    none, ok = ops.qk_norm_rope(q[:, :0], k, qw, kw, 1e-6, pos, cs)
    assert torch.equal(ok, both[1]) and none.shape == (9, 0, D)
    oq, ok = ops.qk_norm_rope(q[:0], k[:0], qw, kw, 1e-6, pos[:0], cs)
    assert oq.shape == (0, 6, D) and ok.shape == (0, 3, D)


def test_zeros_large_and_small_rows_infinities_and_nan(dev):
    from atflash import ops
    x = torch.zeros((7, 2, D), device=dev)
    g = torch.Generator(device=dev).manual_seed(2)
    x[1:] = torch.randn((6, 2, D), generator=g, device=dev)
    x[2] *= 2.0 ** 55       # squares stay below the largest fp32 number
    x[3] *= 2.0 ** -40      # far below eps
    x = x.to(BF)
    x[4, 0, 3] = float("inf")
    x[5, 0, 100] = float("nan")
    w = torch.ones(D, device=dev, dtype=BF)
    pos, cs = torch.arange(7, device=dev, dtype=torch.int32), table_of(7, dev)
    out, _ = ops.qk_norm_rope(x, x[:, :0], w, w, 1e-6, pos, cs)
    fine = [0, 1, 2, 3, 6]
    near(out[fine], x[fine], w, 1e-6, pos[fine], cs)
    assert out[0].eq(0).all() and torch.isnan(out[4, 0]).any() and torch.isnan(out[5, 0]).all()
    near(out[4:6, 1:], x[4:6, 1:], w, 1e-6, pos[4:6], cs)  # the rows beside them


def test_rows_without_a_position_are_left(dev):
    from atflash import _lib
    q, k, _, qw, kw = rows(6, 3, 2, dev, 9)
    cs = table_of(20, dev)
    pos = ints([0, -1, 19, 20, 7, -2 ** 31], dev)
    oq, ok = torch.full((6, 3, D), 7.0, dtype=BF, device=dev), torch.full((6, 2, D), 7.0, dtype=BF, device=dev)
    _lib.launch(0, _lib.lib().atf_qk_norm_rope_bf16, oq.data_ptr(), q.data_ptr(), q.stride(0), q.stride(1), 3, ok.data_ptr(),
                k.data_ptr(), k.stride(0), k.stride(1), 2, qw.data_ptr(), kw.data_ptr(), 0, 1e-6, 6, pos.data_ptr(),
                cs.data_ptr(), 20)
    good = [0, 2, 4]
    near(oq[good], q[good], qw, 1e-6, pos[good], cs)
    near(ok[good], k[good], kw, 1e-6, pos[good], cs)
    for i in (1, 3, 5):
        assert oq[i].eq(7).all() and ok[i].eq(7).all()


# ---- into the caches ----

def packed(lens, starts, hq, hkv, dev, seed, room=2):
    T = sum(lens) + room  # rows behind the last sequence
    q, k, v, qw, kw = rows(T, hq, hkv, dev, seed)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    width = max(-(-(s + n) // PAGE) for s, n in zip(starts, lens)) + 1
    need = [-(-(s + n) // PAGE) for s, n in zip(starts, lens)]
    ids = torch.randperm(sum(need) + 3, generator=torch.Generator().manual_seed(seed)).tolist()
    table = [[ids.pop() for _ in range(n)] + [-1] * (width - n) for n in need]
    pos = torch.full((T,), -1, dtype=torch.int32, device=dev)
    for b, (s, n) in enumerate(zip(starts, lens)):
        pos[cu[b]:cu[b] + n] = torch.arange(s, s + n, device=dev)
    return q, k, v, qw, kw, ints(cu, dev), ints(starts, dev), ints(table, dev), sum(need) + 3, pos


SHAPES = [([1], [0], 28, 4), ([1, 1, 1], [15, 16, 200], 24, 8), ([5, 1, 40], [3, 33, 0], 6, 2), ([16, 32], [0, 16], 8, 8),
          ([700, 0, 33, 1], [0, 9, 25, 100], 28, 4), ([4, 3, 2], [14, 30, 1], 9, 3), ([2000], [77], 5, 1)]


@pytest.mark.parametrize("lens,starts,hq,hkv", SHAPES)
@pytest.mark.parametrize("rope", [True, False])
def test_write_bf16_has_the_rows_bits(dev, lens, starts, hq, hkv, rope):
    from atflash import ops
    q, k, v, qw, kw, cu, start, table, pool, pos = packed(lens, starts, hq, hkv, dev, 11 + len(lens))
    cs = table_of(3000, dev) if rope else None
    g = torch.Generator(device=dev).manual_seed(4)
    kv = torch.randn((pool, hkv, 2, 2048), generator=g, device=dev).to(BF)
    want = kv.clone()
    T = sum(lens)
    wq, wk = ops.qk_norm_rope(q[:T], k[:T], qw, kw, 1e-6, pos[:T], cs)
    ops.kv_write_packed(want, None, wk, v[:T], cu, max(lens), start, table, None, 0)
    got = ops.qk_norm_write(kv, None, q, k, v, qw, kw, 1e-6, cu, max(lens), start, table, cs)
    assert torch.equal(got[:T], wq)
    assert torch.equal(kv, want)


@pytest.mark.parametrize("lens,starts,hq,hkv", SHAPES)
def test_write_q8(dev, lens, starts, hq, hkv):
    from atflash import cache, ops
    q, k, v, qw, kw, cu, start, table, pool, pos = packed(lens, starts, hq, hkv, dev, 31 + len(lens))
    cs = table_of(3000, dev)
    T = sum(lens)
    kv, exps = cache.new_kv_cache_q8(pool, hkv, dev)
    # what the pages hold before: small values, written as the framework writes them
    g = torch.Generator(device=dev).manual_seed(6)
    for b, s in enumerate(starts):
        if s:
            old = (torch.randn((1, s, hkv, D), generator=g, device=dev) * 0.01).to(BF)
            ops.kv_write_q8(kv, exps, old, old, ints([0], dev), table[b:b + 1].contiguous(), None, 0)
    kv0, exps0 = kv.clone(), exps.clone()
    want, wexps = kv.clone(), exps.clone()
    got = ops.qk_norm_write(kv, exps, q, k, v, qw, kw, 1e-6, cu, max(lens), start, table, cs)
    wq, wk = ops.qk_norm_rope(q[:T], k[:T], qw, kw, 1e-6, pos[:T], cs)
    assert torch.equal(got[:T], wq)
    # V: the bits of the writer; its exponents, and the kept and emptied slots, as well
    ops.kv_write_packed(want, wexps, wk, v[:T], cu, max(lens), start, table, None, 0)
    assert torch.equal(kv.view(torch.uint8)[:, :, 0], want.view(torch.uint8)[:, :, 0])
    assert torch.equal(exps[:, :, 0], wexps[:, :, 0])
    # K against the formula: a code is off by half its step, 2^-4 of it, or 2^-10 of its exponent's unit
    ek, off = exact(k[:T], kw, 1e-6, pos[:T], cs)
    deq, before = (cache.dequantize(*c, range(pool))[0].double().cpu() for c in ((kv, exps), (kv0, exps0)))
    pages = table.tolist()
    order = torch.cat([torch.cat([torch.arange(60 - 4 * s, 64 - 4 * s), torch.arange(124 - 4 * s, 128 - 4 * s)]) for s in range(16)])
    e, first = exps[:, :, 1].double().cpu()[..., None], cu.tolist()
    for b, (s, n) in enumerate(zip(starts, lens)):
        at = first[b]
        for t in range(n):
            p, slot = pages[b][(s + t) // PAGE], (s + t) % PAGE
            y, o = ek[at + t][:, order], off[at + t][:, order]
            assert ((deq[p, slot] - y).abs() <= o + (y.abs() + o) * 2.0 ** -4 + 2.0 ** (e[p] - 10)).all(), (b, t)
        if s % PAGE and n:  # kept codes, moved up to the new exponent: exact but for those that became subnormal
            p = pages[b][s // PAGE]
            assert ((deq[p, :s % PAGE] - before[p, :s % PAGE]).abs() <= 2.0 ** (e[p] - 10)).all()
        if n and (s + n) % PAGE:
            assert deq[pages[b][(s + n) // PAGE], (s + n) % PAGE:].eq(0).all()
        for p0 in range(-(-s // PAGE) * PAGE, s + n, PAGE):  # pages that the call begins: the smallest exponent that holds them
            part = slice(at + p0 - s, at + min(p0 + PAGE, s + n) - s)
            top, o, u = ek[part].abs().amax((0, 2)), off[part].amax((0, 2)), 2.0 ** e[pages[b][p0 // PAGE], :, 0]
            assert (top - o <= 448 * u).all() and (top + o > 448 * u / 2).all()


@pytest.mark.parametrize("eight", [False, True])
def test_tokens_that_cannot_be_placed(dev, eight):
    """Negative positions, positions past the RoPE table, pages outside the pool or the table: what cannot be placed is left, and
    what lies beside it is as without it."""
    from atflash import cache, ops
    lens, hq, hkv = [20, 20, 40, 20], 4, 2
    starts = [-7, 90, 10, 40]
    q, k, v, qw, kw, cu, start, table, pool, _ = packed(lens, [0, 90, 10, 40], hq, hkv, dev, 77)
    start = ints(starts, dev)
    table[2, 1], table[2, 2] = -1, pool + 5
    table = table[:, :6].contiguous()  # pages 6.. of sequence 1 (positions 96 on) lie outside the table
    cs = table_of(104, dev)
    pos = torch.cat([torch.arange(s, s + n) for s, n in zip(starts, lens)]).to(dev, torch.int32)
    if eight:
        kv, exps = cache.new_kv_cache_q8(pool, hkv, dev)
    else:
        kv, exps = cache.new_kv_cache(pool, hkv, dev), None
    kv2, exps2 = kv.clone(), None if exps is None else exps.clone()
    T = sum(lens)
    got = ops.qk_norm_write(kv, exps, q, k, v, qw, kw, 1e-6, cu, max(lens), start, table, cs)
    ok = ((pos >= 0) & (pos < 104)).nonzero()[:, 0]
    near(got[ok], q[ok], qw, 1e-6, pos[ok], cs)
    _, wk = ops.qk_norm_rope(q[:T], k[:T], qw, kw, 1e-6, pos.clamp(0, 103), cs)
    ops.kv_write_packed(kv2, exps2, wk, v[:T], cu, max(lens), start, table, None, 0)
    if eight:
        assert torch.equal(kv.view(torch.uint8)[:, :, 0], kv2.view(torch.uint8)[:, :, 0])
    else:
        assert torch.equal(kv, kv2)


def test_max_tokens_cuts_and_rows_outside_stay(dev):
    from atflash import _lib
    q, k, v, qw, kw, cu, start, table, pool, pos = packed([30, 9], [0, 5], 3, 1, dev, 3)
    from atflash import cache
    cs, kv = table_of(64, dev), cache.new_kv_cache(pool, 1, dev)
    out = torch.full((41, 3, D), 7.0, dtype=BF, device=dev)
    _lib.launch(0, _lib.lib().atf_qk_norm_write, out.data_ptr(), q.data_ptr(), q.stride(0), q.stride(1), 3, kv.data_ptr(), None,
                pool, 1, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), qw.data_ptr(),
                kw.data_ptr(), 0, 1e-6, 2, cu.data_ptr(), 41, 12, start.data_ptr(), table.data_ptr(), table.shape[1],
                cs.data_ptr(), 64)
    done = list(range(12)) + list(range(30, 39))
    near(out[done], q[done], qw, 1e-6, pos[done], cs)
    left = [i for i in range(41) if i not in done]
    assert out[left].eq(7).all()
    assert kv[int(table[0, 0]), 0, 1].view(16, 16, 8)[:, 12:].eq(0).all()


@pytest.mark.parametrize("n", [1, 9])
@pytest.mark.parametrize("eight", [False, True])
def test_keys_alone(dev, n, eight):
    """No query heads: the cache as with them."""
    from atflash import cache, ops
    q, k, v, qw, kw, cu, start, table, pool, _ = packed([n, n], [15, 0], 4, 3, dev, 21, room=0)
    cs = table_of(64, dev)
    made = [cache.new_kv_cache_q8(pool, 3, dev) if eight else (cache.new_kv_cache(pool, 3, dev), None) for _ in range(2)]
    for (kv, exps), qq in zip(made, (q, q[:, :0])):
        out = ops.qk_norm_write(kv, exps, qq, k, v, qw, kw, 1e-6, cu, n, start, table, cs)
        assert out.shape == qq.shape
    assert torch.equal(made[0][0].view(torch.uint8), made[1][0].view(torch.uint8)) and (not eight or torch.equal(made[0][1], made[1][1]))


def test_offsets_past_31_bits(dev):
    from atflash import cache, ops
    hq, hkv, T = 2, 1, 40
    wide = torch.zeros((T, 2 ** 26 + 8), dtype=BF, device=dev)  # 5.4 GB: row 32 on lies past 2^31 elements
    x = wide[:, 8:8 + (hq + 2 * hkv) * D].unflatten(1, (-1, D))
    q, k, v, qw, kw = rows(T, hq, hkv, dev, 2)
    x.copy_(torch.cat([q, k, v], 1))
    pool = 600000  # 4.9 GB of blocks
    kv, small = cache.new_kv_cache(pool, hkv, dev), cache.new_kv_cache(3, hkv, dev)
    cs, pos = table_of(T, dev), torch.arange(T, device=dev, dtype=torch.int32)
    cu, zero = ints([0, T], dev), ints([0], dev)
    want = ops.qk_norm_rope(q, k, qw, kw, 1e-6, pos, cs)
    for a, b in zip(ops.qk_norm_rope(x[:, :hq], x[:, hq:hq + 1], qw, kw, 1e-6, pos, cs), want):
        assert torch.equal(a, b)
    far = ints([[pool - 1, pool - 2, 7]], dev)
    out = ops.qk_norm_write(kv, None, x[:, :hq], x[:, hq:hq + 1], x[:, hq + 1:], qw, kw, 1e-6, cu, T, zero, far, cs)
    ops.qk_norm_write(small, None, q, k, v, qw, kw, 1e-6, cu, T, zero, ints([[0, 1, 2]], dev), cs)
    assert torch.equal(out, want[0]) and torch.equal(kv[far[0].long()], small)


def test_captured_and_on_another_stream(dev):
    from atflash import cache, ops
    q, k, v, qw, kw, cu, start, table, pool, pos = packed([1, 1, 1], [15, 16, 200], 28, 4, dev, 8, room=0)
    cs = table_of(300, dev)
    kv = cache.new_kv_cache(pool, 4, dev)
    ops.qk_norm_write(kv, None, q, k, v, qw, kw, 1e-6, cu, 1, start, table, cs)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        side = ops.qk_norm_write(kv, None, q, k, v, qw, kw, 1e-6, cu, 1, start, table, cs)
    with torch.cuda.graph(graph):
        out = ops.qk_norm_write(kv, None, q, k, v, qw, kw, 1e-6, cu, 1, start, table, cs)
        rq, rk = ops.qk_norm_rope(q, k, qw, kw, 1e-6, pos, cs)
    torch.cuda.synchronize()
    near(side, q, qw, 1e-6, pos, cs)
    for i in range(3):
        q.copy_(torch.roll(q.clone(), i + 1, 0))
        want_kv = kv.clone()
        want = ops.qk_norm_write(want_kv, None, q, k, v, qw, kw, 1e-6, cu, 1, start, table, cs)
        kv.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(rq, want) and not torch.equal(kv, torch.zeros_like(kv))


def test_registered_operators(dev):
    from atflash import cache, ops
    q, k, v, qw, kw, cu, start, table, pool, pos = packed([5, 30], [3, 0], 6, 2, dev, 12, room=0)
    cs = table_of(64, dev)
    for a, b in zip(ops.qk_norm_rope(q, k, qw, kw, 1e-6, pos, cs), torch.ops.atflash.qk_norm_rope(q, k, qw, kw, 1e-6, pos, cs)):
        assert torch.equal(a, b)
    kv1, kv2 = cache.new_kv_cache(pool, 2, dev), cache.new_kv_cache(pool, 2, dev)
    a = ops.qk_norm_write(kv1, None, q, k, v, qw, kw, 1e-6, cu, 30, start, table, cs)
    b = torch.ops.atflash.qk_norm_write(kv2, None, q, k, v, qw, kw, 1e-6, cu, 30, start, table, cs)
    assert torch.equal(a, b) and torch.equal(kv1, kv2)
