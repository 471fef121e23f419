"""Plain restatement of the 8-bit cache and of attention over it, for the tests: the cache's
layout, exponents and codes on the CPU, attention in 64 bits with bounds derived from the
roundings that the kernels make."""
import math

import torch

D, PAIRS, PAGE = 128, 64, 16
F8 = torch.float8_e4m3fn
E_MIN, E_MAX = -110, 119
U_BF16 = 2.0 ** -8   # half a step of bf16, relative
U_F8 = 2.0 ** -4     # half a step of e4m3, relative


def rotate32(x, pos, cs):
    """Rotate-half RoPE of x [n, h, 128] bf16 at positions pos, every product and sum rounded to fp32."""
    c, s = cs[pos][:, None, :, 0], cs[pos][:, None, :, 1]
    a, b = x[..., :PAIRS].float(), x[..., PAIRS:].float()
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def to_slices(x, layout=0):
    """x [..., 128] with its dims by slices in wavelength order."""
    if layout == 1:
        return x
    dims = [d for s in range(16) for half in (0, PAIRS) for d in range(half + 60 - 4 * s, half + 64 - 4 * s)]
    return x[..., dims]


def exponent(top):
    """The smallest e with top <= 448 * 2^e, between the limits."""
    if top == 0:
        return E_MIN
    e = math.frexp(top)[1] - 12
    while top > math.ldexp(448.0, e):
        e += 1
    return min(max(e, E_MIN), E_MAX)


class Cache:
    """A cache in the plain: fp32 values of K (by slices) and V per (page, token, head, dim) and the exponents."""

    def __init__(self, pages, heads):
        self.k = torch.zeros(pages, PAGE, heads, D)
        self.v = torch.zeros(pages, PAGE, heads, D)
        self.e = torch.full((pages, heads, 2), E_MIN, dtype=torch.int32)

    def write(self, k, v, start, row, cs, layout=0):
        """k, v [n, heads, 128] bf16 at positions start.. of a sequence whose page-table row is `row`."""
        n = k.shape[0]
        limit = len(row) * PAGE if cs is None else min(len(row) * PAGE, cs.shape[0])
        end = min(start + n, limit)
        first = max(start, 0)
        for p in range(first // PAGE, -(-end // PAGE)):
            pg = int(row[p])
            if not 0 <= pg < self.k.shape[0]:
                continue
            lo, hi = max(first, p * PAGE), min(end, (p + 1) * PAGE)
            s0, s1 = lo - p * PAGE, hi - p * PAGE
            pos = torch.arange(lo, hi)
            kk = k[lo - start:hi - start]
            kk = to_slices(rotate32(kk, pos, cs) if cs is not None else kk.float(), layout)
            vv = v[lo - start:hi - start].float()
            for half, store, new in ((0, self.v, vv), (1, self.k, kk)):
                for h in range(k.shape[1]):
                    x = new[:, h]
                    fin = x[torch.isfinite(x)]
                    e = exponent(float(fin.abs().max()) if fin.numel() else 0.0)
                    if s0 > 0:
                        e = max(e, int(self.e[pg, h, half]))
                    q = (x.double() * 2.0 ** -e).clamp(-448, 448)
                    q[~torch.isfinite(x)] = math.nan
                    old = (store[pg, :s0, h].double() * 2.0 ** -e).float().to(F8)
                    new_codes = q.float().to(F8)
                    store[pg, :, h] = 0
                    store[pg, :s0, h] = (old.double() * 2.0 ** e).float()
                    store[pg, s0:s1, h] = (new_codes.double() * 2.0 ** e).float()
                    self.e[pg, h, half] = e


def attend(q, k, v, lims, age, scale, q_rounded):
    """q [hq, 128] and k [n, hkv, 128] by slices, v [n, hkv, 128], in 64 bits: (out [hq, 128], bound).
    lims: per-slice distance limits (16) or None; age [n, 16] the distance that counts for each slice.
    The bound counts the roundings of P (each weight by at most half a bf16 step; the sum is taken before), of the
    output, of Q where it is rotated by the kernel (each score by at most half a step of its terms' magnitudes, twice
    that in the ratio of a weight to the sum) and 2^-16 for sums and exponentials of 32 bits."""
    q, k, v = q.double(), k.double(), v.double()
    hq, hkv = q.shape[0], k.shape[1]
    if lims is not None:
        keep = age <= torch.tensor(lims, dtype=age.dtype, device=age.device)
        k = k * keep.repeat_interleave(8, dim=-1)[:, None]
    out = torch.empty(hq, D, dtype=torch.float64, device=q.device)
    bound = torch.empty_like(out)
    for h in range(hq):
        kk, vv = k[:, h * hkv // hq], v[:, h * hkv // hq]
        s = kk @ q[h] * scale
        p = torch.softmax(s, 0)
        out[h] = p @ vv
        mag = p @ vv.abs()
        ds = (kk.abs() @ q[h].abs() * scale).max() * (U_BF16 if q_rounded else 0.0)
        bound[h] = mag * (U_BF16 + torch.expm1(2 * ds) + 2.0 ** -16) + out[h].abs() * U_BF16 + 1e-30
    return out, bound


def ages(n, rule, device="cpu"):
    """Distance of the query at n - 1 that counts for key and slice: "page" (level table) or "key"."""
    pos = torch.arange(n, device=device)
    a = (n - 1 - (pos // PAGE * PAGE + PAGE - 1)).clamp(min=0) if rule == "page" else n - 1 - pos
    return a[:, None].expand(n, 16)
