"""Norms of rows whose mean square leaves the range of normal fp32 numbers, with eps 0 or too small to hold it there.  Tolerances are
those that test_qk_norm_gpu.py derives (scaling by a power of two rounds nothing), and for results below the smallest
bf16 number, 2^-133: they may come out as 0 or as it (a row's numbers 2^-126 beside one of 2^90 have results of 2^-210)."""
import pytest
import torch

from test_qk_norm_gpu import BF, D, P, exact, ints, table_of

pytestmark = pytest.mark.gpu
SCALES = (-132, -120, -100, -80, -66, -64, -62, -51, -50, -49, 0, 60, 63, 64, 65, 100, 120)


def tiny_and_huge(dev, heads):
    """Rows of about 2^e each, then rows with one element far from the rest."""
    g = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn((len(SCALES) + 3, heads, D), generator=g, device=dev)
    for i, e in enumerate(SCALES):
        x[i] = (x[i].double() * 2.0 ** e).float()
    x[-3] *= 2.0 ** -126
    x[-3, :, 5] = 2.0 ** 90
    x[-2] = 0
    x[-2, :, 127] = 2.0 ** -133  # the smallest bf16 number
    x[-1] = 0
    x[-1, :, 64] = torch.finfo(BF).max
    return x.to(BF)


def near(got, x, w, eps, pos, cs):
    z, off = exact(x, w, eps, pos, cs)
    bad = ~((got.double().cpu() - z).abs() <= off + (z.abs() + off) * 2.0 ** -8 + 2.0 ** -133)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values, first at {bad.nonzero()[0].tolist()}"


@pytest.mark.parametrize("eps", [0.0, 1e-42, 1e-37])
def test_rows_far_from_one(dev, eps):
    from atflash import ops
    x = tiny_and_huge(dev, 3)
    w = (1 + 0.3 * torch.randn(D, device=dev, generator=torch.Generator(device=dev).manual_seed(1))).to(BF)
    pos, cs = torch.arange(len(x), device=dev, dtype=torch.int32), table_of(len(x), dev)
    eps32 = float(torch.tensor(eps))
    q, k = ops.qk_norm_rope(x[:, :2], x[:, 2:], w, w, eps, pos, cs)
    near(q, x[:, :2].cpu(), w, eps32, pos, cs)
    near(k, x[:, 2:].cpu(), w, eps32, pos, cs)
    q, k = ops.qk_norm_rope(x[:, :2], x[:, 2:], w, w, eps, None, None)
    near(q, x[:, :2].cpu(), w, eps32, None, None)


@pytest.mark.parametrize("most", [1, 20])
@pytest.mark.parametrize("eight", [False, True])
def test_keys_far_from_one_in_the_caches(dev, most, eight):
    """The same rows as keys: the bf16 cache's have the rows' bits, the 8-bit cache's are theirs to half a step of a code."""
    from atflash import cache, ops
    x = tiny_and_huge(dev, 3)
    n = len(x)
    w = torch.ones(D, device=dev, dtype=BF)
    lens = [1] * n if most == 1 else [n]
    B = len(lens)
    cu = ints([0, *torch.tensor(lens).cumsum(0).tolist()], dev)
    table = torch.arange(B * 2, device=dev, dtype=torch.int32).view(B, 2)
    start = ints([0] * B, dev)
    cs = table_of(32, dev)
    pos = torch.cat([torch.arange(m) for m in lens]).to(dev, torch.int32)
    q, k = ops.qk_norm_rope(x[:, :1], x[:, 1:], w, w, 0.0, pos, cs)
    kv, exps = cache.new_kv_cache_q8(2 * B, 2, dev) if eight else (cache.new_kv_cache(2 * B, 2, dev), None)
    out = ops.qk_norm_write(kv, exps, x[:, :1], x[:, 1:], x[:, 1:], w, w, 0.0, cu, most, start, table, cs)
    assert torch.equal(out, q)
    if not eight:
        want = cache.new_kv_cache(2 * B, 2, dev)
        ops.kv_write_packed(want, None, k, x[:, 1:], cu, most, start, table, None, 0)
        assert torch.equal(kv, want)
        return
    z, off = exact(x[:, 1:].cpu(), w, 0.0, pos, cs)
    order = torch.cat([torch.cat([torch.arange(60 - 4 * s, 64 - 4 * s), torch.arange(P + 60 - 4 * s, P + 64 - 4 * s)]) for s in range(16)])
    got = cache.dequantize(kv, exps, range(2 * B))[0].double().cpu().view(B, 32, 2, D)
    unit = torch.exp2(exps[:, :, 1].double().cpu().view(B, 2, 1, 2, 1) - 10).expand(B, 2, 16, 2, 1).reshape(B, 32, 2, 1)
    at = 0
    for b, m in enumerate(lens):
        y, o = z[at:at + m][..., order], off[at:at + m][..., order]
        assert ((got[b, :m] - y).abs() <= o + (y.abs() + o) * 2.0 ** -4 + unit[b, :m]).all(), b
        at += m


@pytest.mark.parametrize("eps", [0.0, 1e-6])
@pytest.mark.parametrize("eight", [False, True])
def test_heads_of_all_sizes_beside_each_other(dev, eps, eight):
    """Queries whose heads and tokens differ in size by chance: each row as by itself."""
    from atflash import cache, ops
    hq, n = 13, 45
    x = tiny_and_huge(dev, 1)[:, 0]
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.cat([x, torch.randn((60, D), generator=g, device=dev).to(BF)])
    pick = torch.randint(0, len(x), (n, hq + 2), generator=g, device=dev)
    rows = x[pick]
    w = torch.ones(D, device=dev, dtype=BF)
    pos, cs = torch.arange(n, device=dev, dtype=torch.int32), table_of(64, dev)
    kv, exps = cache.new_kv_cache_q8(4, 2, dev) if eight else (cache.new_kv_cache(4, 2, dev), None)
    out = ops.qk_norm_write(kv, exps, rows[:, :hq], rows[:, hq:], rows[:, hq:], w, w, eps, ints([0, n], dev), n, ints([0], dev),
                            ints([[2, 0, 3]], dev), cs)
    near(out, rows[:, :hq].cpu(), w, float(torch.tensor(eps)), pos, cs)
    q, _ = ops.qk_norm_rope(rows[:, :hq], rows[:, hq:], w, w, eps, pos, cs)
    assert torch.equal(out, q)
    one, _ = ops.qk_norm_rope(rows[:, 4:5].contiguous(), rows[:, :0], w, w, eps, pos, cs)
    assert torch.equal(out[:, 4:5], one)
