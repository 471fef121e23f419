"""Operators of a serving step over ragged batches and an 8-bit cache, as timed cases.

    tables   block tables and slot maps on the GPU: the pages that a step's new
             tokens need, taken from the free pages, and where each token goes
    write8   keys (RoPE at write) and values of packed new tokens into a paged cache
             of 8-bit floats with a scale for each page of 16 tokens and head
    decode8  one decode step over that cache, windowed or plain
    packed   causal attention over packed prompts of different lengths, windowed or
             plain, grouped heads

Every case is one call of an entry point at the sizes and options of real use:
the two model shapes the repository's benchmark names (28 query heads on 4 kv
heads with RoPE base 1e7; 24 on 8 with base 5e5); `draw` adds other head counts.

The 8-bit cache.  A block of 4096 bytes (e4m3) for each page and kv head, V half
first, and two powers of two (K's and V's exponent, whole numbers of 8 bits): a
code c of a half with exponent e stands for c * 2^e, e being the smallest with the
half's largest value at most 448 * 2^e (between -110 and 119; a page that keeps
earlier tokens keeps at least its earlier exponent).
    V half  [2][4][16][4 dims][4 tokens]: element (j, g, r, d, t) is dim 8r + 4j + d
            of token 4g + t
    K half  [8 levels][16 tokens][16]: the 8-dim slices 2l and 2l + 1 of a token;
            slice s holds rotary pairs 60 - 4s .. 63 - 4s, first halves, then second
"""
import math
import os
import random
import sys
import types

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
own = False

DEV = "cuda"
D, PAIRS, PAGE = 128, 64, 16
CAP = 1_100_000  # distance cap of the window tables, above every context
SCALE = D ** -0.5
E_MIN, E_MAX = -110, 119  # exponents of the 8-bit cache
F8 = torch.float8_e4m3fn


def listed():
    return [
        # A decode step's bookkeeping: one token more for each running request.
        {"name": "tables_step_64", "kind": "tables", "batch": 64, "min_new": 1, "max_new": 1, "max_len": 20000,
         "lens_seed": 1},
        # Admission of many prompts at once behind cached prefixes.
        {"name": "tables_admit_300", "kind": "tables", "batch": 300, "min_new": 1, "max_new": 1900, "max_len": 5000,
         "lens_seed": 2},
        # A decode step's append: one token for each of a batch, somewhere in a page.
        {"name": "write8_append_32", "kind": "write8", "batch": 32, "min_new": 1, "max_new": 1, "max_start": 9000,
         "lens_seed": 3, "hkv": 8, "base": 5e5},
        # A chat's next turns behind what the cache holds, odd lengths.
        {"name": "write8_turns_11", "kind": "write8", "batch": 11, "min_new": 30, "max_new": 1100, "max_start": 5000,
         "lens_seed": 4, "hkv": 4, "base": 1e7},
        # Long prompts into the cache.
        {"name": "write8_3x20000", "kind": "write8", "batch": 3, "min_new": 20000, "max_new": 20000, "max_start": 0,
         "lens_seed": 5, "hkv": 8, "base": 5e5},
        # The smallest decode step, early in a conversation: latency.
        {"name": "decode8_1003", "kind": "decode8", "batch": 1, "min_len": 1003, "max_len": 1003, "lens_seed": 0,
         "hq": 24, "hkv": 8, "base": 5e5, "k_ret": 2.0, "table": "vec8"},
        # Continuous batching: sequences of very different ages in one step.
        {"name": "decode8_12_ragged", "kind": "decode8", "batch": 12, "min_len": 700, "max_len": 32768, "lens_seed": 3,
         "hq": 24, "hkv": 8, "base": 5e5, "k_ret": 2.0, "table": "vec8"},
        # The benchmark's headline context, plain causal attention.
        {"name": "decode8_128k", "kind": "decode8", "batch": 1, "min_len": 131072, "max_len": 131072, "lens_seed": 0,
         "hq": 28, "hkv": 4, "base": 1e7, "k_ret": 0.0, "table": "vec8"},
        # Many requests of the same age, level table.
        {"name": "decode8_40x8192", "kind": "decode8", "batch": 40, "min_len": 8192, "max_len": 8192, "lens_seed": 0,
         "hq": 28, "hkv": 4, "base": 1e7, "k_ret": 2.0, "table": "level"},
        # A few short prompts admitted together, a one-token one among them.
        {"name": "packed_5_short", "kind": "packed", "batch": 5, "min_len": 1, "max_len": 517, "lens_seed": 6,
         "hq": 24, "hkv": 8, "base": 5e5, "k_ret": 0.0, "rope": False},
        # Prompts of very different lengths, window on, RoPE by the call.
        {"name": "packed_16_ragged", "kind": "packed", "batch": 16, "min_len": 300, "max_len": 9000, "lens_seed": 7,
         "hq": 28, "hkv": 4, "base": 1e7, "k_ret": 2.0, "rope": True},
        # A document beside short prompts, rotated rows, window on.
        {"name": "packed_document", "kind": "packed", "batch": 4, "min_len": 700, "max_len": 16384, "lens_seed": 8,
         "hq": 24, "hkv": 8, "base": 5e5, "k_ret": 2.0, "rope": False},
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tables", "write8", "write8", "decode8", "decode8", "decode8", "packed", "packed"])
    hq, hkv, base = rng.choice([(28, 4, 1e7), (24, 8, 5e5), (28, 4, 1e7), (24, 8, 5e5), (14, 2, 1e7), (32, 2, 1e7),
                                (8, 8, 5e5), (32, 8, 5e5)])
    k_ret = rng.choice([0.0, 2.0, 2.0, 64.0])
    seed = rng.randrange(1000)
    if kind == "tables":
        batch = _log(rng, 1, 600)
        top = rng.choice([1, 1, _log(rng, 2, 100_000 // batch)])
        return {"kind": kind, "batch": batch, "min_new": rng.choice([0, 1]) if top > 1 else 1, "max_new": top,
                "max_len": _log(rng, 20, 20000), "lens_seed": seed}
    if kind == "write8":
        batch = rng.choice([1, 1, 3, 11, 16, 40])
        top = rng.choice([1, _log(rng, 2, 50_000 // batch), _log(rng, 2, 50_000 // batch)])
        return {"kind": kind, "batch": batch, "min_new": max(1, top // rng.choice([1, 7])), "max_new": top,
                "max_start": rng.choice([0, 0, 40, 5000]), "lens_seed": seed, "hkv": hkv, "base": base}
    if kind == "decode8":
        batch = rng.choice([1, 1, 2, 4, 7, 12, 24, 40, 64])
        top = _log(rng, 100, 131072 if batch == 1 else 262144 // batch)
        return {"kind": kind, "batch": batch, "min_len": top if batch == 1 else max(1, top // rng.choice([1, 3, 30])),
                "max_len": top, "lens_seed": seed, "hq": hq, "hkv": hkv, "base": base, "k_ret": k_ret,
                "table": rng.choice(["vec8", "vec8", "level"])}
    batch = rng.choice([1, 2, 3, 5, 8, 16, 30])
    top = _log(rng, 40, min(12000, 40_000 // batch))
    return {"kind": kind, "batch": batch, "min_len": max(1, top // rng.choice([1, 3, 30, 1000])), "max_len": top,
            "lens_seed": seed, "hq": hq, "hkv": hkv, "base": base, "k_ret": k_ret, "rope": rng.choice([True, False])}


# ---- the inputs, from the seed alone ----

def _spread(case, lo, hi, salt=0):
    """case["batch"] whole numbers spread over the logarithm of [lo, hi], hi among them."""
    rng = random.Random(case["lens_seed"] * 31 + salt)
    out = [_log(rng, max(lo, 1), max(hi, 1)) if lo > 0 or rng.random() < 0.9 else 0 for _ in range(case["batch"])]
    out[rng.randrange(len(out))] = hi
    return out


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + 29)


def _randn(shape, gen):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _angles(n, base):
    """fp32 [n, 64, 2] of (cos, sin)(position * base^(-2r/128)), the table a
    program builds once for its model (angles of far positions in 64 bits)."""
    inv = float(base) ** (-torch.arange(0, D, 2, device=DEV).double() / D)
    ang = torch.arange(n, device=DEV).double()[:, None] * inv[None, :]
    return torch.stack([torch.cos(ang), torch.sin(ang)], dim=-1).float().contiguous()


def _page_rows(lens):
    """Page ids of sequences that grow 512 tokens at a time in turn, as requests
    that are served together do: one list for each."""
    pages = [[] for _ in lens]
    nxt = 0
    for upto in range(512, max(lens) + 512, 512):
        for row, n in zip(pages, lens):
            need = -(-min(n, upto) // PAGE) - len(row)
            row.extend(range(nxt, nxt + max(0, need)))
            nxt += max(0, need)
    return pages, nxt


def _page_table(lens):
    pages, n = _page_rows(lens)
    tab = torch.full((len(lens), max(max(len(p) for p in pages), 1)), -1, dtype=torch.int32)
    for i, p in enumerate(pages):
        tab[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
    return tab.to(DEV), max(n, 1)


def _limits(case, per):
    """Largest distance at which each group of `per` sorted pairs is read, by
    the window rule: the width k * 2 pi * base^(2r/128) of its longest pair."""
    if not case["k_ret"]:
        return None
    out = []
    for i in range(PAIRS // per):
        r = PAIRS - 1 - per * i
        w = torch.tensor(case["k_ret"] * 2.0 * math.pi * case["base"] ** (2.0 * r / D), dtype=torch.float64)
        out.append(int(min(CAP, math.floor(float(w.to(torch.float32))))))
    if per == 8:
        out[0] = CAP  # the level rule keeps one level at every distance
    return out


def _tables_inputs(case, seed):
    rng = random.Random(seed * 7919 + 5)
    lens = _spread(case, 0, case["max_len"], salt=1)
    new = _spread(case, case["min_new"], case["max_new"], salt=2)
    order = list(range(len(lens)))
    rng.shuffle(order)  # other inputs for another seed, the same work
    lens = [lens[i] for i in order]
    have = [-(-n // PAGE) for n in lens]
    width = -(-(case["max_len"] + case["max_new"]) // PAGE)
    need = sum(-(-(n + m) // PAGE) - h for n, m, h in zip(lens, new, have))
    ids = torch.randperm(sum(have) + need + 64, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    tab = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, h in enumerate(have):
        tab[b, :h] = ids[at:at + h]
        at += h
    return tab.to(DEV), _ints(lens), _ints(new), ids[at:].to(DEV), _ints([len(ids) - at]), sum(new), len(ids)


def prepare(case, seed):
    kind = case["kind"]
    s = types.SimpleNamespace(case=case)
    g = _gen(seed)
    if kind == "tables":
        s.table, s.lens, s.new, s.free, s.count, s.total, s.pool = _tables_inputs(case, seed)
    elif kind == "write8":
        new, start = _spread(case, case["min_new"], case["max_new"]), _starts(case)
        ends = [a + n for a, n in zip(start, new)]
        s.table, s.pool = _page_table(ends)
        s.max_new = max(new)
        s.cu, s.start, s.new = _ints(_cu(new)), _ints(start), new
        s.k = _randn((sum(new), case["hkv"], D), g).to(torch.bfloat16)
        s.v = (_randn((sum(new), case["hkv"], D), g) * 0.5).to(torch.bfloat16)
        s.rope = _angles(max(ends), case["base"])
        s.codes, s.exps = _filled(s.table, start, s.pool, case["hkv"], g)
    elif kind == "decode8":
        lens = _spread(case, case["min_len"], case["max_len"])
        s.table, s.pool = _page_table(lens)
        s.n, s.lens_list, s.lens = max(lens), lens, _ints(lens)
        s.codes, s.exps = _filled(s.table, lens, s.pool, case["hkv"], g)
        s.q = _randn((len(lens), case["hq"], D), g).to(torch.bfloat16)
        s.rope = _angles(s.n, case["base"])
    else:
        lens = _spread(case, case["min_len"], case["max_len"])
        s.n, s.lens_list, s.cu = max(lens), lens, _ints(_cu(lens))
        s.q = _randn((sum(lens), case["hq"], D), g).to(torch.bfloat16)
        s.k = _randn((sum(lens), case["hkv"], D), g).to(torch.bfloat16)
        s.v = _randn((sum(lens), case["hkv"], D), g).to(torch.bfloat16)
        s.rope = _angles(s.n, case["base"]) if case["rope"] else None
    if "k_ret" in case:
        s.lims = _limits(case, 8 if case.get("table") == "level" or kind == "packed" else 4)
        s.zhi = None if s.lims is None else tuple(s.lims)
    if own:
        _import_own(s)
        if kind == "decode8":
            s.cache = s.own.cache.PagedKVCache(s.pool, case["hkv"], DEV, kv_dtype=F8)
            s.cache.kv.copy_(s.codes)
            s.cache.exps.copy_(s.exps)
    return s


def _starts(case):
    if case["max_start"] == 0:
        return [0] * case["batch"]
    return _spread(case, 1, case["max_start"], salt=3)


def _import_own(s):
    pkg = os.path.join(ROOT, "atflash-kernel_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from atflash import cache, interface, ops
    s.own = types.SimpleNamespace(cache=cache, interface=interface, ops=ops)


def run(s):
    kind = s.case["kind"]
    if own:
        if kind == "tables":
            out = s.own.ops.extend_tables(s.table, s.lens, s.new, s.free, s.count, s.total, s.pool)
            return (s.table, *out)
        if kind == "write8":
            s.own.ops.kv_write_packed(s.codes, s.exps, s.k, s.v, s.cu, s.max_new, s.start, s.table, s.rope, 0)
            return s.codes, s.exps
        if kind == "decode8":
            return s.own.interface.decode_paged(s.q, s.cache, s.table, s.lens, s.n, zhi=s.zhi, rope=s.rope)
        out, lse = s.own.interface.flash_attn_packed(s.q, s.k, s.v, s.cu, s.n, zhi=s.zhi, rope=s.rope)
        return out if s.rope is not None else (out, lse)
    if kind == "tables":
        return _plain_tables(s)
    if kind == "write8":
        return _plain_write(s, torch.float32)
    if kind == "decode8":
        return _plain_decode(s, torch.float32).to(torch.bfloat16)
    out, lse = _plain_packed(s)
    return out.to(torch.bfloat16) if s.rope is not None else (out.to(torch.bfloat16), lse)


# ---- the plain forms ----

def _plain_tables(s):
    """A sequence of L tokens with n new ones needs pages ceil(L/16) .. ceil((L+n)/16) - 1:
    they are taken from the end of the free pages, sequence by sequence.  Returns (the page
    table, lengths afterwards, free pages left, first token of each sequence, position of each
    token, its slot page * 16 + position % 16)."""
    lens, new = s.lens.long(), s.new.long()
    table = s.table.clone()
    width = table.shape[1]
    first, last = (lens + PAGE - 1) // PAGE, ((lens + new + PAGE - 1) // PAGE).clamp(max=width)
    need = (last - first).clamp(min=0)
    base = torch.cumsum(need, 0) - need
    col = torch.arange(width, device=DEV)[None]
    take = (col >= first[:, None]) & (col < last[:, None])
    rank = base[:, None] + col - first[:, None]
    count = s.count.long()
    at = (count - 1 - rank).clamp(min=0, max=s.free.shape[0] - 1)
    got = torch.where(rank < count, s.free.long()[at], -1)
    table = torch.where(take, got.int(), table)
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), torch.cumsum(new, 0)])
    tok = torch.arange(s.total, device=DEV)
    seq = (torch.searchsorted(cu, tok, right=True) - 1).clamp(max=len(lens) - 1)
    pos = lens[seq] + tok - cu[seq]
    page = table[seq, (pos // PAGE).clamp(max=width - 1)].long()
    slot = torch.where((page >= 0) & (page < s.pool) & (pos // PAGE < width), page * PAGE + pos % PAGE, -1)
    return table, (lens + new).int(), (count - need.sum()).int(), cu.int(), pos.int(), slot


def _rotate(x, cs):
    """Rotate-half RoPE of x [n, h, 128] with cs [n, 64, 2], in x's type."""
    c, s = cs[:, None, :, 0].to(x.dtype), cs[:, None, :, 1].to(x.dtype)
    a, b = x[..., :PAIRS], x[..., PAIRS:]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _to_slices(x):
    """x [..., 128] (half-split) as [..., 16 slices, 8]: slice i holds rotary pairs
    60 - 4i .. 63 - 4i, their first halves and then their second halves."""
    a = x[..., :PAIRS].unflatten(-1, (16, 4)).flip(-2)
    b = x[..., PAIRS:].unflatten(-1, (16, 4)).flip(-2)
    return torch.cat([a, b], dim=-1)


def _to_blocks(k, v):
    """k, v [pages, 16 tokens, heads, 128] as the halves [pages, heads, 2, 2048], V first."""
    p, _, h, _ = k.shape
    kb = _to_slices(k).permute(0, 2, 3, 1, 4).reshape(p, h, 8, 2, PAGE, 8).transpose(3, 4)
    vb = v.reshape(p, 4, 4, h, 16, 2, 4).permute(0, 3, 5, 1, 4, 6, 2)
    return torch.stack([vb.reshape(p, h, -1), kb.reshape(p, h, -1)], dim=2)


def _from_blocks(x):
    """The halves [pages, heads, 2, 2048] as k [pages, 16 tokens, heads, 16 slices, 8]
    and v [pages, 16 tokens, heads, 128]."""
    p, h = x.shape[:2]
    k = x[:, :, 1].reshape(p, h, 8, PAGE, 2, 8).permute(0, 3, 1, 2, 4, 5).reshape(p, PAGE, h, 16, 8)
    v = x[:, :, 0].reshape(p, h, 2, 4, 16, 4, 4).permute(0, 3, 6, 1, 4, 2, 5).reshape(p, PAGE, h, D)
    return k, v


def _exponents(top):
    """The smallest e with top <= 448 * 2^e, between the cache's limits."""
    m, e = torch.frexp(top.float())  # top = m * 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.where(top > 0, e, E_MIN).clamp(E_MIN, E_MAX)


def _filled(table, lens, pool, hkv, gen):
    """An 8-bit cache that holds lens[b] tokens of each sequence (pages whose
    magnitudes differ), empty pages otherwise: (codes, exponents)."""
    codes = torch.zeros((pool, hkv, 2, 2048), dtype=F8, device=DEV)
    exps = torch.full((pool, hkv, 2), E_MIN, dtype=torch.int8, device=DEV)
    for b, n in enumerate(lens):
        for p0 in range(0, -(-n // PAGE), 4096):
            p1 = min(-(-n // PAGE), p0 + 4096)
            x = _randn((p1 - p0, PAGE, hkv, 2, D), gen)
            x *= torch.exp2(_randn((p1 - p0, 1, hkv, 2, 1), gen) * 0.4)
            live = torch.arange(p0 * PAGE, p1 * PAGE, device=DEV).view(-1, PAGE, 1, 1, 1) < n
            x *= live
            blk = _to_blocks(x[..., 0, :], x[..., 1, :])
            e = _exponents(blk.abs().amax(-1))
            ids = table[b, p0:p1].long()
            codes.view(torch.uint8)[ids] = (blk * torch.exp2(-e.float())[..., None]).to(F8).view(torch.uint8)
            exps[ids] = e.to(torch.int8)
    return codes, exps


def _plain_write(s, dt):
    """New tokens into their pages: rows to blocks, the pages' exponents, codes.  A page
    that keeps earlier tokens keeps at least its exponent, its codes are shifted to the
    new one; slots behind the last new token become zero.  dt float64: codes unrounded."""
    case = s.case
    codes = s.codes.to(dt)
    exps = s.exps.int().clone()
    lo = 0
    for b, (a, n) in enumerate(zip(_starts(case), s.new)):
        k = _rotate(s.k[lo:lo + n].to(dt), s.rope[a:a + n])
        v = s.v[lo:lo + n].to(dt)
        lo += n
        p0, p1 = a // PAGE, -(-(a + n) // PAGE)
        x = torch.zeros((2, (p1 - p0) * PAGE, case["hkv"], D), dtype=dt, device=DEV)
        x[0, a - p0 * PAGE:a - p0 * PAGE + n] = k
        x[1, a - p0 * PAGE:a - p0 * PAGE + n] = v
        x = x.unflatten(1, (-1, PAGE))
        blk = _to_blocks(x[0], x[1])
        e = _exponents(blk.abs().amax(-1))
        ids = s.table[b, p0:p1].long()
        if a % PAGE:
            e[0] = torch.maximum(e[0], exps[ids[0]])
        out = blk * torch.exp2(-e.to(dt))[..., None]
        if dt == torch.float32:
            out = out.to(F8).to(dt)
        if a % PAGE:
            kept = torch.arange(PAGE, device=DEV) < a % PAGE
            shape = (1, PAGE, case["hkv"], D)
            kept = _to_blocks(*(kept.view(1, PAGE, 1, 1).expand(shape),) * 2)
            old = codes[ids[:1]] * torch.exp2((exps[ids[:1]] - e[:1]).to(dt))[..., None]
            if dt == torch.float32:
                old = old.to(F8).to(dt)
            out[:1] = torch.where(kept, old, out[:1])
        codes[ids] = out
        exps[ids] = e
    return (codes.to(F8) if dt == torch.float32 else codes), exps.to(torch.int8)


def _rows(s, b, n, dt):
    """Keys (by slices) and values of a sequence's n tokens from the 8-bit cache."""
    ids = s.table[b, :-(-n // PAGE)].long()
    x = s.codes.view(torch.uint8)[ids].view(F8).to(dt) * torch.exp2(s.exps[ids].to(dt))[..., None]
    k, v = _from_blocks(x)
    return k.flatten(0, 1)[:n], v.flatten(0, 1)[:n]


def _plain_decode(s, dt):
    """softmax(q k / sqrt(128)) v of each sequence's last position; a slice of a key is
    read up to its distance limit (slice table: the key's distance; level table: the
    distance of the youngest key of its page)."""
    case = s.case
    hq, hkv = case["hq"], case["hkv"]
    out = torch.empty((len(s.lens_list), hq, D), dtype=dt, device=DEV)
    for b, n in enumerate(s.lens_list):
        k, v = _rows(s, b, n, dt)  # [n, hkv, 16, 8], [n, hkv, 128]
        q = _to_slices(_rotate(s.q[b][None].to(dt), s.rope[n - 1:n]))[0]
        if s.lims is not None:
            pos = torch.arange(n, device=DEV)
            if len(s.lims) == 8:
                dist = (n - 1 - (pos // PAGE * PAGE + PAGE - 1)).clamp(min=0)
                keep = torch.stack([dist <= z for z in s.lims for _ in range(2)], dim=-1)
            else:
                keep = torch.stack([n - 1 - pos <= z for z in s.lims], dim=-1)
            k = k * keep[:, None, :, None].to(dt)
        k = k.flatten(-2).transpose(0, 1).contiguous()  # [hkv, n, 128]
        v = v.transpose(0, 1).contiguous()
        sc = torch.bmm(q.flatten(-2).view(hkv, hq // hkv, D), k.transpose(1, 2).contiguous()) * SCALE
        e = (sc - sc.amax(-1, keepdim=True)).exp()
        out[b] = (torch.bmm(e, v) / e.sum(-1, keepdim=True)).view(hq, D)
    return out


def _plain_packed(s, dt=torch.float32):
    """Causal attention of each sequence's rows over its own: (out [rows, heads, 128],
    log-sum-exp [heads, rows]).  A level (16 dims) of the keys is read up to its distance
    limit, the distance being that of a 32-row by 32-key tile."""
    case = s.case
    hq, hkv = case["hq"], case["hkv"]
    grp = hq // hkv
    out = torch.empty((s.q.shape[0], hq, D), dtype=dt, device=DEV)
    lse = torch.empty((hq, s.q.shape[0]), dtype=dt, device=DEV)
    lo = 0
    for n in s.lens_list:
        q, k, v = (x[lo:lo + n].to(dt) for x in (s.q, s.k, s.v))
        if s.rope is not None:
            q, k = _rotate(q, s.rope[:n]), _rotate(k, s.rope[:n])
        q = _to_slices(q).flatten(-2).transpose(0, 1).contiguous()  # [hq, n, 128], levels first to last
        k = _to_slices(k).flatten(-2).transpose(0, 1).contiguous()
        v = v.transpose(0, 1).contiguous()
        pos = torch.arange(n, device=DEV)
        for i0 in range(0, n, 512):
            i1 = min(n, i0 + 512)
            rows, keys = pos[i0:i1], pos[:i1]
            dist = (rows // 32 * 32)[:, None] - (keys // 32 * 32 + 31)[None]
            hide = keys[None] > rows[:, None]
            lims = [] if s.lims is None else s.lims
            cut = [z < int(dist.max()) for z in lims]
            whole = cut.index(True) if True in cut else 8
            for h in range(hkv):
                qh, kh = q[h * grp:(h + 1) * grp, i0:i1].reshape(-1, D), k[h, :i1]
                sc = (qh[:, :16 * whole] @ kh[:, :16 * whole].T).view(grp, i1 - i0, i1)
                for lv in range(whole, 8):
                    near = dist <= lims[lv]
                    far = int((~near.any(0)).sum())  # keys that no row reads at this level
                    if far < i1:
                        t = (qh[:, 16 * lv:16 * lv + 16] @ kh[far:, 16 * lv:16 * lv + 16].T).view(grp, i1 - i0, -1)
                        sc[..., far:] += t * near[:, far:]
                sc = (sc * SCALE).masked_fill_(hide, float("-inf"))
                top = sc.amax(-1, keepdim=True)
                e = (sc - top).exp_()
                total = e.sum(-1, keepdim=True)
                o = (e.view(-1, i1) @ v[h, :i1]).view(grp, i1 - i0, D) / total
                out[lo + i0:lo + i1, h * grp:(h + 1) * grp] = o.transpose(0, 1)
                lse[h * grp:(h + 1) * grp, lo + i0:lo + i1] = (top + total.log())[..., 0]
        lo += n
    return out, lse


# ---- what a pass cannot do without ----

def _kept(lims, first, last):
    """Sum over distances first..last of the share of K dims that are read."""
    if lims is None:
        return float(last - first + 1)
    return sum(max(0, min(z, last) - first + 1) for z in lims) / len(lims)


def work(case):
    kind = case["kind"]
    if kind == "tables":
        lens, new = _spread(case, 0, case["max_len"], salt=1), _spread(case, case["min_new"], case["max_new"], salt=2)
        pages = sum(new) // PAGE + len(lens)
        # lengths read and written, first tokens written; free pages read, entries written; position and slot
        return {"bytes": 16 * len(lens) + 8 * pages + 12 * sum(new), "flops": 0}
    if kind == "write8":
        new, start = _spread(case, case["min_new"], case["max_new"]), _starts(case)
        tok = sum(new)
        # the rows as bf16 and their codes, the pages' exponents, the (cos, sin) rows used
        far = max(a + n for a, n in zip(start, new)) - min(start)
        return {"bytes": tok * case["hkv"] * D * 2 * 3 + tok // PAGE * case["hkv"] * 2 + min(tok, far) * PAIRS * 8,
                "flops": tok * case["hkv"] * D * 5}
    lens = _spread(case, case["min_len"], case["max_len"])
    hq, hkv = case["hq"], case["hkv"]
    if kind == "decode8":
        lims = _limits(case, 8 if case["table"] == "level" else 4)
        nbytes = flops = 0.0
        for n in lens:
            kept = _kept(lims, 0, n - 1)
            nbytes += D * hkv * (n + kept) + n / PAGE * hkv * 2 + 2 * 2 * D * hq
            flops += 2 * D * hq * (n + kept)
        return {"bytes": nbytes, "flops": flops}
    lims = _limits(case, 8)
    nbytes = flops = 0.0
    for n in lens:
        nbytes += 2 * 2 * n * (hq + hkv) * D + n * hq * 4
        for i0 in range(0, n, 32):  # by 32-row tiles: every row of one reads about the same
            rows = min(32, n - i0)
            mid = i0 + rows / 2
            flops += 2 * D * hq * rows * (mid + 0.5 + _kept(lims, 0, int(mid)))
    return {"bytes": nbytes, "flops": flops}


# ---- results in 64 bits ----

def exact(case, seed):
    kind = case["kind"]
    if kind == "tables":
        return _exact_tables(*_tables_inputs(case, seed))
    if kind == "packed" and sum(n * n for n in _spread(case, case["min_len"], case["max_len"])) * case["hq"] > 1.2e10:
        return None
    keep = globals()["own"]
    globals()["own"] = False
    try:
        s = prepare(case, seed)
    finally:
        globals()["own"] = keep
    if kind == "write8":
        return _plain_write(s, torch.float64)[0], None
    if kind == "decode8":
        return _exact_decode(s)
    out, lse = _exact_packed(s)
    return out if s.rope is not None else (out, lse)


def _exact_tables(table, lens, new, free, count, total, pool):
    """Page by page and token by token, as a program on the host does it."""
    table, lens, new, free = (x.tolist() for x in (table, lens, new, free))
    free = free[:int(count)]
    after, cu, pos, slot = [], [0], [], []
    for row, n, m in zip(table, lens, new):
        for p in range(-(-n // PAGE), -(-(n + m) // PAGE)):
            row[p] = free.pop() if free else -1
        after.append(n + m)
        cu.append(cu[-1] + m)
        pos += range(n, n + m)
        slot += [row[t // PAGE] * PAGE + t % PAGE if row[t // PAGE] >= 0 else -1 for t in range(n, n + m)]
    return _ints(table), _ints(after), _ints([len(free)]), _ints(cu), _ints(pos), torch.tensor(slot, device=DEV)


def _exact_decode(s):
    """Key by key from the definition: value c * 2^e, dims in place, limits by dim."""
    case = s.case
    hq, hkv = case["hq"], case["hkv"]
    dim_slice = torch.tensor([15 - (d % PAIRS) // 4 for d in range(D)], device=DEV)
    out = torch.empty((len(s.lens_list), hq, D), dtype=torch.float64, device=DEV)
    for b, n in enumerate(s.lens_list):
        pages = -(-n // PAGE)
        ids = s.table[b, :pages].long()
        raw = s.codes.view(torch.uint8)[ids].view(F8).double()
        scale = torch.pow(2.0, s.exps[ids].double())
        q = s.q[b].double()
        c, sn = s.rope[n - 1, :, 0].double(), s.rope[n - 1, :, 1].double()
        q = torch.cat([q[:, :PAIRS] * c - q[:, PAIRS:] * sn, q[:, PAIRS:] * c + q[:, :PAIRS] * sn], dim=-1)
        dims = torch.arange(D, device=DEV)
        sl = dim_slice
        in_slice = (dims % 4) + 4 * (dims >= PAIRS)
        tok = torch.arange(PAGE, device=DEV)
        k_at = (sl // 2 * 256 + sl % 2 * 8 + in_slice)[None] + tok[:, None] * 16
        v_at = ((dims % 8) // 4 * 1024 + dims // 8 * 16 + dims % 4 * 4)[None] + (tok // 4 * 256 + tok % 4)[:, None]
        for h in range(hkv):
            k = (raw[:, h, 1][:, k_at] * scale[:, h, 1, None, None]).flatten(0, 1)[:n]
            v = (raw[:, h, 0][:, v_at] * scale[:, h, 0, None, None]).flatten(0, 1)[:n]
            if s.lims is not None:
                pos = torch.arange(n, device=DEV)
                if len(s.lims) == 8:
                    far = (n - 1 - (pos | 15)).clamp(min=0)
                    lim = torch.tensor(s.lims, device=DEV)[sl // 2]
                else:
                    far, lim = n - 1 - pos, torch.tensor(s.lims, device=DEV)[sl]
                k = torch.where(far[:, None] > lim[None], 0.0, k)
            for i in range(h * hq // hkv, (h + 1) * hq // hkv):
                p = torch.softmax(k @ q[i] * SCALE, dim=0)
                out[b, i] = p @ v
    return out


def _exact_packed(s):
    case = s.case
    hq, hkv = case["hq"], case["hkv"]
    level = torch.tensor([7 - (d % PAIRS) // 8 for d in range(D)], device=DEV)
    out = torch.empty((s.q.shape[0], hq, D), dtype=torch.float64, device=DEV)
    lse = torch.empty((hq, s.q.shape[0]), dtype=torch.float64, device=DEV)
    for n, lo in zip(s.lens_list, _cu(s.lens_list)):
        pos = torch.arange(n, device=DEV)
        step = max(32, min(2048, (1 << 26) // max(n, 1) // 32 * 32))
        for h in range(hq):
            q, k, v = s.q[lo:lo + n, h].double(), s.k[lo:lo + n, h * hkv // hq].double(), s.v[lo:lo + n, h * hkv // hq].double()
            if s.rope is not None:
                c, sn = s.rope[:n, :, 0].double(), s.rope[:n, :, 1].double()
                q, k = (torch.cat([x[:, :PAIRS] * c - x[:, PAIRS:] * sn, x[:, PAIRS:] * c + x[:, :PAIRS] * sn], -1)
                        for x in (q, k))
            for i0 in range(0, n, step):
                i1 = min(n, i0 + step)
                tile = (pos[i0:i1] // 32 * 32)[:, None] - (pos[:i1] | 31)[None]
                sc = torch.zeros((i1 - i0, i1), dtype=torch.float64, device=DEV)
                for lv in range(8):
                    d = level == lv
                    t = q[i0:i1][:, d] @ k[:i1][:, d].T
                    sc += t if s.lims is None else torch.where(tile <= s.lims[lv], t, 0.0)
                sc = torch.where(pos[None, :i1] > pos[i0:i1, None], -math.inf, sc * SCALE)
                lse[h, lo + i0:lo + i1] = torch.logsumexp(sc, dim=-1)
                out[lo + i0:lo + i1, h] = torch.softmax(sc, dim=-1) @ v[:i1]
    return out, lse
