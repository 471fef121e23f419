"""The 8-bit decode rounds its output and nothing else that shows: Q and P enter its matrix products in two bf16 parts.

Measure: the 2-norm of the error against 64 bits over that of rounding the 64-bit result itself.  The parts leave 2^-17 of a
value, sums and exponentials of 32 bits less: some 1e-5 of a result, a hundredth of the half steps of bf16 (2^-8 at most,
1.7e-3 in the mean), so the ratio is 1 but for the few per cent of elements that such a distance moves to the next number.
With one part, P's half steps alone, independent of the output's and as large, make it sqrt(2), Q's alone about 1.2.  The
line is drawn at 1.1; the CPU test plants each of these mistakes in the arithmetic and finds it above."""
import pytest
import torch

from helpers import BF, D
from q8_ref import ages, attend, to_slices

LINE = 1.1
SCALE = D ** -0.5


def ratio(got, want):
    return float((got.double() - want).norm() / (want.to(BF).double() - want).norm())


def parts(x, n):
    """x as n bf16 parts, added up again."""
    out = torch.zeros_like(x)
    for _ in range(n):
        out = out + (x - out).to(BF).double()
    return out


def emulate(q, k, v, q_parts, p_parts):
    """Attention whose Q and P enter the products in so many bf16 parts; the sum of P is taken before."""
    out = torch.empty(q.shape, dtype=torch.float64)
    for h in range(q.shape[0]):
        kk, vv = (x[:, h * k.shape[1] // q.shape[0]].double() for x in (k, v))
        s = kk @ parts(q[h].double(), q_parts) * SCALE
        p = torch.exp(s - s.max())
        out[h] = parts(p, p_parts) @ vv / p.sum()
    return out.to(BF)


@pytest.mark.parametrize("n", [100, 300, 1003])
def test_the_line_tells_the_mistakes_apart(n):
    g = torch.Generator().manual_seed(n)
    k, v = (torch.randn((n, 4, D), generator=g).to(torch.float8_e4m3fn).float() for _ in range(2))
    q = torch.randn((28, D), generator=g)           # as RoPE leaves it: not a bf16 number
    want, _ = attend(q, k, v, None, None, SCALE, False)
    assert ratio(emulate(q, k, v, 2, 2), want) < 1.02
    for q_parts, p_parts in ((1, 2), (2, 1), (1, 1)):
        assert ratio(emulate(q, k, v, q_parts, p_parts), want) > LINE


@pytest.mark.gpu
@pytest.mark.parametrize("kind,rope", [("off", False), ("off", True), ("level", True), ("vec8", False), ("vec8", True)])
@pytest.mark.parametrize("hq,hkv", [(8, 8), (28, 4), (24, 2), (16, 1)])   # the last two: 9 to 16 heads a kv head
def test_only_the_output_is_rounded(dev, hq, hkv, kind, rope):
    from atflash import interface
    from test_q8_gpu import filled, ropes, row_of, tables
    lens = [300, 1003, 129, 4099]
    cache, table, keys = filled(lens, hkv, dev, 201)
    q = torch.randn((len(lens), hq, D), generator=torch.Generator(device=dev).manual_seed(202), device=dev).to(BF)
    level, vec8 = tables()
    cs = ropes(max(lens)).to(dev) if rope else None
    out = interface.decode_paged(q, cache, table, row_of(lens, dev), max(lens), rope=cs,
                                 zhi={"off": None, "level": level, "vec8": vec8}[kind])
    lims = {"off": None, "vec8": vec8, "level": [1 << 30] * 2 + [z for z in level[1:] for _ in range(2)]}[kind]
    for b, n in enumerate(lens):
        x = q[b].double()
        if rope:
            c, s = cs[n - 1, :, 0].double(), cs[n - 1, :, 1].double()
            x = torch.cat([x[:, :64] * c - x[:, 64:] * s, x[:, 64:] * c + x[:, :64] * s], -1)
        want, _ = attend(to_slices(x), *keys[b], lims, ages(n, "key" if kind == "vec8" else "page", dev), SCALE, rope)
        r = ratio(out[b], want)
        print(hq, hkv, kind, rope, n, round(r, 4))
        assert r <= LINE, (n, r)
