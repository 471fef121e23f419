"""Operators of a branching decode, as timed cases: one step norms, rotates and writes
new tokens, ranks each row's next tokens, and forks, drops and moves sequences.

    qknorm    RMS norm of the queries and keys of each head and the rotation of their
              positions in one pass over packed rows
    qkwrite   the same with the keys written, beside their values, into a paged cache
              (bf16, or 8-bit floats with a power of two for each page, head and half)
    logprobs  log probabilities of given tokens, entropy and top alternatives of rows of logits
    select    new rows of page tables from old ones (forks, drops, a beam's parents): whole
              pages shared, part-filled ones copied in every layer, pages without a row freed
    compact   the pages that rows hold moved to the front of the pool, in every layer

Every case is one pass of entry points at the sizes of real use: the model shapes that the
repository's benchmark names (28 query heads on 4 kv heads, RoPE base 1e7, 152064 tokens
of vocabulary; 24 on 8, base 5e5); `draw` adds others.

The caches (pages of 16 tokens, V half first):
    bf16   V half [128 dims][16 slots], token groups of four in the order 0, 2, 1, 3
           K half [16 slices][16 tokens][8 dims]
    8-bit  V half [2][4][16][4 dims][4 tokens]: element (j, g, r, d, t) is dim 8r + 4j + d
           of token 4g + t; K half [8 levels][16 tokens][slices 2l, 2l + 1]; a code c of a
           half with exponent e is c * 2^e, e the smallest with every magnitude of the
           half at most 448 * 2^e, between -110 and 119
    slice s holds rotary pairs 60 - 4s .. 63 - 4s, first halves, then second.
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
EPS = 1e-6
E_MIN, E_MAX = -110, 119
F8 = torch.float8_e4m3fn
FLOATS = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # A decode step: one token of each of a batch, every length its own.
        {"name": "qknorm_step_24", "kind": "qknorm", "batch": 24, "min_new": 1, "max_new": 1, "max_start": 9000,
         "lens_seed": 1, "hq": 28, "hkv": 4, "base": 1e7},
        # Packed prompts of different lengths, odd ones.
        {"name": "qknorm_prompts_7", "kind": "qknorm", "batch": 7, "min_new": 900, "max_new": 9001, "max_start": 0,
         "lens_seed": 2, "hq": 24, "hkv": 8, "base": 5e5},
        # A decode step's append to the bf16 cache.
        {"name": "qkwrite_append_32", "kind": "qkwrite", "batch": 32, "min_new": 1, "max_new": 1, "max_start": 9000,
         "lens_seed": 3, "hq": 28, "hkv": 4, "base": 1e7, "cache": "bf16"},
        # A chat's next turns behind what an 8-bit cache holds.
        {"name": "qkwrite8_turns_11", "kind": "qkwrite", "batch": 11, "min_new": 30, "max_new": 1100,
         "max_start": 5000, "lens_seed": 4, "hq": 24, "hkv": 8, "base": 5e5, "cache": "8bit"},
        # Long prompts into the bf16 cache.
        {"name": "qkwrite_2x16000", "kind": "qkwrite", "batch": 2, "min_new": 16000, "max_new": 16000, "max_start": 0,
         "lens_seed": 5, "hq": 28, "hkv": 4, "base": 1e7, "cache": "bf16"},
        # One request's step: the chosen token's log probability and five alternatives.
        {"name": "logprobs_step_1", "kind": "logprobs", "rows": 1, "vocab": 152064, "type": "bf16", "top": 5,
         "masked": 0.0},
        # A batch's step, fp32 logits, most of the vocabulary masked by a grammar.
        {"name": "logprobs_step_48", "kind": "logprobs", "rows": 48, "vocab": 50257, "type": "fp32", "top": 20,
         "masked": 0.9},
        # A scored prompt: every position's token, and the likeliest.
        {"name": "logprobs_prompt_2048", "kind": "logprobs", "rows": 2048, "vocab": 152064, "type": "bf16", "top": 1,
         "masked": 0.0},
        # A beam step: eight beams far into an answer, some dropped and some forked.
        {"name": "select_beams_8", "kind": "select", "batch": 8, "tokens": 6007, "common": 5000, "fork": 0,
         "layers": 28, "hkv": 4, "cache": "bf16", "lens_seed": 6},
        # A long prompt forked into samples.
        {"name": "select_fork_48", "kind": "select", "batch": 48, "tokens": 30011, "common": 0, "fork": 1,
         "layers": 24, "hkv": 8, "cache": "8bit", "lens_seed": 7},
        # A small pool after a few requests ended.
        {"name": "compact_300", "kind": "compact", "batch": 6, "pool": 300, "fill": 0.6, "layers": 4, "hkv": 4,
         "cache": "8bit", "lens_seed": 8},
        # A large pool, half empty, before it is cut.
        {"name": "compact_6000", "kind": "compact", "batch": 40, "pool": 6000, "fill": 0.5, "layers": 28, "hkv": 4,
         "cache": "bf16", "lens_seed": 9},
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["qknorm", "qknorm", "qkwrite", "qkwrite", "logprobs", "logprobs", "logprobs", "select", "select",
                       "compact"])
    hq, hkv, base = rng.choice([(28, 4, 1e7), (24, 8, 5e5), (28, 4, 1e7), (24, 8, 5e5), (14, 2, 1e7), (32, 2, 1e7),
                                (8, 8, 5e5), (5, 1, 5e5)])
    seed = rng.randrange(1000)
    if kind in ("qknorm", "qkwrite"):
        batch = rng.choice([1, 1, 3, 8, 11, 40])
        top = rng.choice([1, _log(rng, 2, 28000 // batch), _log(rng, 2, 28000 // batch)])
        case = {"kind": kind, "batch": batch, "min_new": max(1, top // rng.choice([1, 7])), "max_new": top,
                "max_start": rng.choice([0, 0, 40, 5000]), "lens_seed": seed, "hq": hq, "hkv": hkv, "base": base}
        if kind == "qkwrite":
            case["cache"] = rng.choice(["bf16", "8bit"])
        return case
    if kind == "logprobs":
        vocab = rng.choice([151, 32000, 50257, 128256, 152064, _log(rng, 300, 200_000)])
        kind_of = rng.choice(["bf16", "bf16", "fp32", "fp16"])
        most = 300_000_000 // vocab // (2 if kind_of == "fp32" else 1)
        return {"kind": kind, "rows": _log(rng, 1, min(4000, most)), "vocab": vocab, "type": kind_of,
                "top": rng.choice([0, 1, 1, 5, 20, 32]), "masked": rng.choice([0.0, 0.0, 0.5, 0.99])}
    if kind == "select":
        batch = rng.choice([2, 4, 5, 8, 16, 33])
        tokens = _log(rng, 30, 60_000 // batch)
        return {"kind": kind, "batch": batch, "tokens": tokens, "common": rng.choice([0, tokens // 2]),
                "fork": rng.choice([0, 0, 1]), "layers": rng.choice([2, 12, 28]), "hkv": rng.choice([1, 2, 4, 8]),
                "cache": rng.choice(["bf16", "8bit"]), "lens_seed": seed}
    return {"kind": kind, "batch": rng.choice([1, 3, 8, 40]), "pool": _log(rng, 50, 4000),
            "fill": rng.choice([0.2, 0.5, 0.8]), "layers": rng.choice([2, 12, 24]), "hkv": rng.choice([1, 2, 4, 8]),
            "cache": rng.choice(["bf16", "8bit"]), "lens_seed": seed}


# ---- the inputs, from the seed alone ----

def _spread(case, lo, hi, salt=0):
    """case["batch"] whole numbers spread over the logarithm of [lo, hi], hi among them."""
    rng = random.Random(case["lens_seed"] * 31 + salt)
    out = [_log(rng, max(lo, 1), max(hi, 1)) for _ in range(case["batch"])]
    out[rng.randrange(len(out))] = hi
    return out


def _starts(case):
    return _spread(case, 1, case["max_start"], salt=3) if case["max_start"] else [0] * case["batch"]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + 31)


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


def _page_table(lens):
    """Page ids of sequences that grow 512 tokens at a time in turn, as requests
    that are served together do."""
    pages, nxt = [[] for _ in lens], 0
    for upto in range(512, max(lens) + 512, 512):
        for row, n in zip(pages, lens):
            need = max(0, -(-min(n, upto) // PAGE) - len(row))
            row.extend(range(nxt, nxt + need))
            nxt += need
    tab = torch.full((len(lens), max(len(p) for p in pages)), -1, dtype=torch.int32)
    for i, p in enumerate(pages):
        tab[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
    return tab.to(DEV), nxt


def _caches(case, pool, gen):
    """Every layer's pages, any values: bf16 blocks, or codes and exponents."""
    out = []
    for _ in range(case["layers"]):
        shape = (pool, case["hkv"], 2, 2048)
        if case["cache"] == "bf16":
            out.append(torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(generator=gen))
        else:
            codes = torch.randint(0, 0x7fff, (shape[0], shape[1], 2, 2048 // 2), generator=gen, device=DEV, dtype=torch.int16)
            codes = (codes.view(torch.uint8) & 0x77).view(F8)
            out += [codes.view(shape), torch.randint(-9, 3, (*shape[:2], 2), generator=gen, device=DEV, dtype=torch.int8)]
    return out


def _select_tables(case, seed):
    """Rows that share the whole pages of their first `common` tokens, the pages in any
    order; parents: row 0's copies (fork), or a beam step's choice."""
    rng = random.Random(seed * 7919 + case["lens_seed"])
    batch, n = case["batch"], case["tokens"]
    lens = [n] + [0] * (batch - 1) if case["fork"] else [n] * batch
    shared = case["common"] // PAGE
    pool = shared + sum(max(0, -(-m // PAGE) - shared) for m in lens) + batch + 7
    ids = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    tab = torch.full((batch, -(-(n + 600) // PAGE)), -1, dtype=torch.int32)
    at = shared
    for b, m in enumerate(lens):
        have = -(-m // PAGE)
        if have:
            tab[b, :shared] = ids[:shared]
            tab[b, shared:have] = ids[at:at + have - shared]
            at += have - shared
    free = torch.full((pool,), -1, dtype=torch.int32)
    free[:pool - at] = ids[at:]
    picks = random.Random(case["lens_seed"])  # which ranks survive, the same work for every seed
    parents = [0] * batch if case["fork"] else [picks.randrange(batch) for _ in range(batch)]
    order = list(range(batch))
    if not case["fork"]:
        rng.shuffle(order)
    parents = [order[p] for p in parents]
    return tab.to(DEV), _ints(lens), free.to(DEV), _ints([pool - at]), _ints(parents), pool


def _compact_tables(case, seed):
    """Rows whose pages lie anywhere in the pool; the second half of the rows begin with the
    whole pages that row 0 begins with."""
    rng = random.Random(case["lens_seed"])
    pool, batch = case["pool"], case["batch"]
    live = max(batch, int(pool * case["fill"]))
    each = [live // batch] * batch
    lens = [max(1, n * PAGE - rng.randrange(PAGE)) for n in each]
    shared = each[0] // 3
    ids = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    tab = torch.full((batch, max(each) + 9), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(each):
        tab[b, :n] = ids[at:at + n]
        at += n
        if b > batch // 2:
            tab[b, :shared] = tab[0, :shared]
            at -= shared
            tab[b, shared:n] = ids[at - n + shared:at]
    free = torch.full((pool,), -1, dtype=torch.int32)
    free[:pool - at] = ids[at:]
    return tab.to(DEV), _ints(lens), free.to(DEV), _ints([pool - at]), pool


def prepare(case, seed):
    kind = case["kind"]
    s = types.SimpleNamespace(case=case)
    g = _gen(seed)
    if kind in ("qknorm", "qkwrite"):
        new, start = _spread(case, case["min_new"], case["max_new"]), _starts(case)
        ends = [a + n for a, n in zip(start, new)]
        hq, hkv, rows = case["hq"], case["hkv"], sum(new)
        # one fused projection's rows; tokens differ in magnitude
        qkv = _randn((rows, hq + 2 * hkv, D), g) * torch.exp(_randn((rows, 1, 1), g) * 0.7)
        qkv = qkv.to(torch.bfloat16)
        s.q, s.k, s.v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s.qw, s.kw = ((1 + 0.3 * _randn((D,), g)).to(torch.bfloat16) for _ in range(2))
        s.rope = _angles(max(ends), case["base"])
        s.cu, s.start, s.max_new = _ints(_cu(new)), _ints(start), max(new)
        s.pos = torch.cat([torch.arange(a, e, dtype=torch.int32) for a, e in zip(start, ends)]).to(DEV)
    if kind == "qkwrite":
        s.table, s.pool = _page_table(ends)
        s.touched = sum(-(-e // PAGE) - a // PAGE for a, e in zip(start, ends))  # pages that the rows lie in
        s.kv, s.exps = (_caches({**case, "layers": 1}, s.pool, g) + [None])[:2]
    elif kind == "logprobs":
        x = _randn((case["rows"], case["vocab"]), g) * 2.0
        x += 6.0 * (_randn((1, case["vocab"]), g) > 3.0)  # tokens that are likely everywhere
        s.tokens = torch.randint(0, case["vocab"], (case["rows"],), generator=g, device=DEV)
        if case["masked"]:
            allowed = _randn((1, case["vocab"]), g).argsort(-1)[:, :max(1, round(case["vocab"] * (1 - case["masked"])))]
            x = torch.full_like(x, -math.inf).scatter_(1, allowed.expand(case["rows"], -1), x.gather(1, allowed.expand(case["rows"], -1)))
            s.tokens = allowed[0][s.tokens % allowed.shape[1]]
        s.x = x.to(FLOATS[case["type"]])
    elif kind == "select":
        s.table, s.lens, s.free, s.count, s.parents, s.pool = _select_tables(case, seed)
        s.caches = _caches(case, s.pool, g)
    elif kind == "compact":
        s.table, s.lens, s.free, s.count, s.pool = _compact_tables(case, seed)
        s.caches = _caches(case, s.pool, g)
    return s


def _ops():
    pkg = os.path.join(ROOT, "atflash-kernel_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from atflash import ops
    return ops


def run(s):
    kind = s.case["kind"]
    if own:
        ops = _ops()
        if kind == "qknorm":
            return ops.qk_norm_rope(s.q, s.k, s.qw, s.kw, EPS, s.pos, s.rope)
        if kind == "qkwrite":
            q = ops.qk_norm_write(s.kv, s.exps, s.q, s.k, s.v, s.qw, s.kw, EPS, s.cu, s.max_new, s.start, s.table, s.rope)
            return q, s.kv, s.exps
        if kind == "logprobs":
            return ops.token_logprobs(s.x, s.tokens, s.case["top"])
        if kind == "select":
            table, lens, left, src, dst = ops.select_tables(s.table, s.lens, s.free, s.count, s.parents, s.pool)
            ops.copy_pages(s.caches, src, dst)
            return table, lens, s.free, left, src, dst, s.caches
        table, free, left, src, dst, moves = ops.compact_tables(s.table, s.lens, s.free, s.count, s.pool)
        ops.copy_pages(s.caches, src, dst, moves)
        return table, free, left, src, dst, moves, s.caches
    if kind == "qknorm":
        return tuple(_norm_rotate(x.float(), w.float(), s.rope[s.pos.long()]).to(torch.bfloat16)
                     for x, w in ((s.q, s.qw), (s.k, s.kw)))
    if kind == "qkwrite":
        cs = s.rope[s.pos.long()]
        q = _norm_rotate(s.q.float(), s.qw.float(), cs).to(torch.bfloat16)
        k = _norm_rotate(s.k.float(), s.kw.float(), cs)
        if s.exps is None:
            return q, _plain_pages(s, k.to(torch.bfloat16)), None
        return q, *_plain_pages_q8(s, k, s.v.float())
    if kind == "logprobs":
        return _plain_logprobs(s.x, s.tokens, s.case["top"])
    return _plain_select(s) if kind == "select" else _plain_compact(s)


# ---- the plain forms ----

def _norm_rotate(x, w, cs):
    """x [n, h, 128] / rms(x) * w, then rotate-half by cs [n, 64, 2], in x's type."""
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    c, s = cs[:, None, :, 0].to(x.dtype), cs[:, None, :, 1].to(x.dtype)
    a, b = y[..., :PAIRS], y[..., PAIRS:]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _to_slices(x):
    """x [..., 128] (half-split) as [..., 16 slices, 8]: slice i holds rotary pairs
    60 - 4i .. 63 - 4i, their first halves and then their second halves."""
    a = x[..., :PAIRS].unflatten(-1, (16, 4)).flip(-2)
    b = x[..., PAIRS:].unflatten(-1, (16, 4)).flip(-2)
    return torch.cat([a, b], dim=-1)


def _sequences(s):
    """The sequence of each row of the call."""
    rows = torch.arange(s.q.shape[0], device=DEV)
    return torch.searchsorted(s.cu.long(), rows, right=True) - 1


def _plain_pages(s, k):
    """Rotated keys and values into their slots of the bf16 cache, in place."""
    pos = s.pos.long()
    page, slot = s.table[_sequences(s), pos // PAGE].long(), pos % PAGE
    kv = s.kv
    kv[:, :, 1].view(-1, kv.shape[1], 16, PAGE, 8).permute(0, 3, 1, 2, 4)[page, slot] = _to_slices(k)
    order = torch.tensor([0, 2, 1, 3], device=DEV)[slot // 4] * 4 + slot % 4
    kv[:, :, 0].view(-1, kv.shape[1], D, PAGE).permute(0, 3, 1, 2)[page, order] = s.v
    return kv


def _to_blocks(k, v):
    """k, v [pages, 16 tokens, heads, 128] as the 8-bit halves [pages, heads, 2, 2048], V first."""
    p, _, h, _ = k.shape
    kb = _to_slices(k).permute(0, 2, 3, 1, 4).reshape(p, h, 8, 2, PAGE, 8).transpose(3, 4)
    vb = v.reshape(p, 4, 4, h, 16, 2, 4).permute(0, 3, 5, 1, 4, 6, 2)
    return torch.stack([vb.reshape(p, h, -1), kb.reshape(p, h, -1)], dim=2)


def _exponents(top):
    """The smallest e with top <= 448 * 2^e, between the cache's limits."""
    m, e = torch.frexp(top.float())  # top = m * 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.where(top > 0, e, E_MIN).clamp(E_MIN, E_MAX)


def _plain_pages_q8(s, k, v):
    """Rotated keys and values into the pages of the 8-bit cache: their exponents, codes.  A
    page that keeps earlier tokens keeps at least its exponent, its codes are moved to the
    new one; slots behind the last new token become zero.  k in float64: codes unrounded."""
    dt = k.dtype
    to = (lambda x: x.to(F8).to(dt)) if dt == torch.float32 else (lambda x: x)
    seq, pos, start, cu = _sequences(s), s.pos.long(), s.start.long(), s.cu.long()
    count = (start + cu[1:] - cu[:-1] + PAGE - 1) // PAGE - start // PAGE  # pages of each sequence
    base = torch.cumsum(count, 0) - count
    at = base[seq] + pos // PAGE - (start // PAGE)[seq]
    x = torch.zeros((2, s.touched, PAGE, s.case["hkv"], D), dtype=dt, device=DEV)
    x[0, at, pos % PAGE] = k
    x[1, at, pos % PAGE] = v
    ids = torch.empty(s.touched, dtype=torch.long, device=DEV)
    ids[at] = s.table[seq, pos // PAGE].long()
    kept = torch.zeros(s.touched, dtype=torch.long, device=DEV)
    kept[base] = start % PAGE  # tokens before the call's first in its first page
    blk = _to_blocks(x[0], x[1])
    e, had = _exponents(blk.abs().amax(-1)), s.exps[ids].int()
    e = torch.where((kept > 0)[:, None, None], torch.maximum(e, had), e)
    old = to(s.kv.view(torch.uint8)[ids].view(F8).to(dt) * torch.exp2((had - e).to(dt))[..., None])
    mask = (torch.arange(PAGE, device=DEV) < kept[:, None])[:, :, None, None].expand(-1, -1, s.case["hkv"], D)
    new = torch.where(_to_blocks(mask, mask), old, to(blk * torch.exp2(-e.to(dt))[..., None]))
    if dt == torch.float64:
        codes = s.kv.to(dt)
        codes[ids] = new
        return codes, None
    s.kv.view(torch.uint8)[ids] = new.to(F8).view(torch.uint8)
    s.exps[ids] = e.to(torch.int8)
    return s.kv, s.exps


def _plain_logprobs(x, tokens, top):
    """x - log sum exp x at the tokens, the entropy, and the `top` largest with their places
    (equal ones: the lowest place first)."""
    rows, vocab = x.shape
    x = x.float()
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(-1, keepdim=True)
    lse = m + total.log()
    logp = x - lse
    entropy = -torch.where(e > 0, e / total * logp, 0.0).sum(-1)
    best = torch.empty((rows, 0), dtype=torch.long, device=DEV)
    if top:
        bits = (x + 0.0).view(torch.int32).long()
        rank = torch.where(bits < 0, ~bits, bits | 0x80000000)  # ordered as the values are
        rank = (rank << 24) | (0xffffff - torch.arange(vocab, device=DEV))
        best = 0xffffff - (rank.topk(top, dim=-1).values & 0xffffff)
    return (logp.gather(1, tokens[:, None])[:, 0], entropy, logp.gather(1, best), best)


def _plain_copied(cache, src, dst):
    raw = cache.view(torch.uint8)
    raw[dst] = raw[src]
    return cache


def _plain_select(s):
    """New row b is old row parents[b]: its whole pages, and its part-filled last page if b
    keeps it (the parent itself, or else its first child), otherwise a page from the end of
    the free pages, to which the part-filled one is copied.  Pages that no new row names are
    appended to the free pages first, lowest id first."""
    batch, width = s.table.shape
    n, par = s.lens.long().clamp(min=0), s.parents.long()
    ok = (par >= 0) & (par < batch)
    p = torch.where(ok, par, 0)
    full, have = (n // PAGE).clamp(max=width), ((n + PAGE - 1) // PAGE).clamp(max=width)
    col, row = torch.arange(width, device=DEV)[None], torch.arange(batch, device=DEV)
    of = s.table[p].long()
    first = torch.where(par[:, None] == par[None], row[None], batch).amin(-1)
    keep = torch.where(par[p] == p, row == p, row == first)
    last = of.gather(1, full[p].clamp(max=width - 1)[:, None])[:, 0]
    fresh = ok & (have > full)[p] & ~keep & (last >= 0) & (last < s.pool)
    named = ok[:, None] & ((col < full[p][:, None]) | (keep[:, None] & (col < have[p][:, None])))
    inside = lambda t: (t >= 0) & (t < s.pool)  # noqa: E731
    old = s.table.long()
    mark = torch.zeros((2, s.pool + 1), dtype=torch.bool, device=DEV)
    mark[0, torch.where((col < have[:, None]) & inside(old), old, s.pool)] = True
    mark[1, torch.where(named & inside(of), of, s.pool)] = True
    freed = (mark[0] & ~mark[1])[:s.pool]
    size = s.free.shape[0]
    count = s.count.long().clamp(0, size)
    at = (count + torch.cumsum(freed, 0) - 1).clamp(max=size)
    pages = torch.cat([s.free.long(), s.free.new_zeros(1).long()])
    pages[torch.where(freed, at, size)] = torch.arange(s.pool, device=DEV)
    count = (count + freed.sum()).clamp(max=size)
    nth = count - torch.cumsum(fresh, 0)
    page = torch.where(nth >= 0, pages[nth.clamp(min=0)], -1)
    table = torch.where(named, of, -1)
    table = torch.where(fresh[:, None] & (col == full[p][:, None]), page[:, None], table)
    good = fresh & inside(page)
    src, dst = torch.where(good, last, -1), torch.where(good, page, -1)
    a, b = src[good], dst[good]
    return (table.int(), torch.where(ok, n[p], 0).int(), pages[:size].int(), (count - fresh.sum()).int(), src.int(),
            dst.int(), [_plain_copied(c, a, b) for c in s.caches])


def _plain_compact(s):
    """Of the ids that rows hold or that are free, the lowest become the rows': the i-th
    highest of the pages past those goes to the i-th lowest free one among them.  The free
    pages come out highest first."""
    col = torch.arange(s.table.shape[1], device=DEV)[None]
    have = (s.lens.long().clamp(min=0) + PAGE - 1) // PAGE
    old, free = s.table.long(), s.free.long()
    at = torch.arange(free.shape[0], device=DEV)
    mark = torch.zeros((2, s.pool + 1), dtype=torch.bool, device=DEV)
    held = (col < have[:, None]) & (old >= 0) & (old < s.pool)
    mark[0, torch.where(held, old, s.pool)] = True
    mark[1, torch.where((at < s.count) & (free >= 0) & (free < s.pool), free, s.pool)] = True
    live, idle = mark[0, :s.pool], (mark[1] & ~mark[0])[:s.pool]
    rank, n = torch.cumsum(live | idle, 0) - 1, live.sum()
    dst = (idle & (rank < n)).nonzero()[:, 0]
    src = (live & (rank >= n)).nonzero()[:, 0].flip(0)
    to = torch.arange(s.pool + 1, device=DEV)
    to[src] = dst
    table = torch.where(held, to[torch.where(held, old, s.pool)], torch.where(col < have[:, None], old, -1))
    rest = ((live | idle) & (rank >= n)).nonzero()[:, 0].flip(0)
    pad = lambda x, size: torch.cat([x, x.new_full((size - x.shape[0],), -1)]).int()  # noqa: E731
    half = max(1, s.pool // 2)
    return (table.int(), pad(rest, free.shape[0]), _ints([rest.shape[0]]), pad(src, half), pad(dst, half),
            _ints([src.shape[0]]), [_plain_copied(c, src, dst) for c in s.caches])


# ---- what a pass cannot do without ----

def _page_bytes(case):
    return case["layers"] * case["hkv"] * (8192 if case["cache"] == "bf16" else 4098)


def work(case):
    kind = case["kind"]
    if kind in ("qknorm", "qkwrite"):
        new, start = _spread(case, case["min_new"], case["max_new"]), _starts(case)
        tok, hq, hkv = sum(new), case["hq"], case["hkv"]
        far = max(a + n for a, n in zip(start, new)) - min(start)
        nbytes = tok * (hq + hkv) * D * 4 + min(tok, far) * PAIRS * 8  # rows read and written, (cos, sin) rows
        if kind == "qkwrite":
            nbytes += tok * hkv * D * 4  # values read and written
            if case["cache"] == "8bit":
                nbytes -= tok * hkv * D * 2  # codes have half the bytes
        return {"bytes": nbytes, "flops": tok * (hq + hkv) * D * 8}
    if kind == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["type"] == "fp32" else 2) + case["rows"] * (16 + 12 * case["top"]), "flops": n * 6}
    if kind == "select":
        batch, n = case["batch"], case["tokens"]
        entries = -(-n // PAGE) * batch
        picks = random.Random(case["lens_seed"])
        kinds = 1 if case["fork"] else len({picks.randrange(batch) for _ in range(batch)})
        copies = batch - kinds if n % PAGE else 0
        read = -(-n // PAGE) if case["fork"] else entries
        return {"bytes": 4 * (read + entries) + 2 * copies * _page_bytes(case), "flops": 0}
    live = case["fill"] * case["pool"]
    moves = live * (1 - case["fill"])
    return {"bytes": 4 * (2 * live + 2 * case["pool"]) + 2 * moves * _page_bytes(case), "flops": 0}


# ---- results in 64 bits ----

def exact(case, seed):
    kind = case["kind"]
    if kind == "logprobs" and case["rows"] * case["vocab"] > 400_000_000:
        return None
    keep = globals()["own"]
    globals()["own"] = False
    try:
        s = prepare(case, seed)
    finally:
        globals()["own"] = keep
    if kind in ("qknorm", "qkwrite"):
        q, k = _exact_rows(s, s.q, s.qw), _exact_rows(s, s.k, s.kw)
        if kind == "qknorm":
            return q, k
        if s.exps is not None:
            return q, *_plain_pages_q8(s, k, s.v.double())
        return q, _exact_pages(s, k), None
    if kind == "logprobs":
        return _exact_logprobs(s.x, s.tokens, case["top"])
    return _exact_select(s) if kind == "select" else _exact_compact(s)


def _exact_rows(s, x, w):
    """Dim by dim: x[d] w[d] / sqrt(mean of squares + eps), pair (r, r + 64) turned by its angle's (cos, sin)."""
    x, w, out = x.double(), w.double(), torch.empty(x.shape, dtype=torch.float64, device=DEV)
    size = torch.sqrt(torch.linalg.vector_norm(x, dim=-1) ** 2 / D + EPS)
    turn = torch.view_as_complex(s.rope.double().contiguous())[s.pos.long()][:, None]
    z = torch.complex(x[..., :PAIRS] * w[:PAIRS], x[..., PAIRS:] * w[PAIRS:]) / size[..., None] * turn
    out[..., :PAIRS], out[..., PAIRS:] = z.real, z.imag
    return out


def _exact_pages(s, k):
    """Element by element of the bf16 blocks: where dim d of the token in slot t lies."""
    kv, pos = s.kv.double().flatten(2), s.pos.long()
    seq = torch.repeat_interleave(torch.arange(len(s.start), device=DEV), (s.cu[1:] - s.cu[:-1]).long())
    page, t = s.table[seq, pos // PAGE].long()[:, None], (pos % PAGE)[:, None]
    dims = torch.arange(D, device=DEV)[None]
    r = dims % PAIRS
    k_at = 2048 + (15 - r // 4) * 128 + t * 8 + r % 4 + 4 * (dims >= PAIRS)
    group = t // 4
    v_at = dims * PAGE + torch.where(group == 1, 2, torch.where(group == 2, 1, group)) * 4 + t % 4
    for h in range(k.shape[1]):
        kv[page, h, k_at] = k[:, h]
        kv[page, h, v_at] = s.v[:, h].double()
    return kv.view(s.kv.shape)


def _exact_logprobs(x, tokens, top):
    lse = torch.cat([torch.logsumexp(r.double(), -1, keepdim=True) for r in x.split(64)])
    got, entropy, values, ids = [], [], [], []
    for r, z, t in zip(x.split(64), lse.split(64), tokens.split(64)):
        logp = r.double() - z
        got.append(logp.gather(1, t[:, None])[:, 0])
        entropy.append(torch.special.entr(logp.exp()).sum(-1))
        best = torch.sort(r, dim=-1, descending=True, stable=True).indices[:, :top] if top else t[:, None][:, :0]
        values.append(logp.gather(1, best))
        ids.append(best)
    return torch.cat(got), torch.cat(entropy), torch.cat(values), torch.cat(ids)


def _exact_select(s):
    """Row by row, as a program on the host does it."""
    table, lens, free, parents = (x.tolist() for x in (s.table, s.lens, s.free, s.parents))
    count, width = int(s.count), s.table.shape[1]
    rows, new, kept, ask = [], [], set(), []
    for b, p in enumerate(parents):
        if not 0 <= p < len(table):
            rows.append([])
            new.append(0)
            continue
        n = lens[p]
        row = table[p][:n // PAGE]
        if n % PAGE and n // PAGE < width:
            holder = p if parents[p] == p else parents.index(p)
            row.append(table[p][n // PAGE] if holder == b else None)
            if holder != b:
                ask.append((b, table[p][n // PAGE]))
        kept.update(x for x in row if x is not None)
        rows.append(row)
        new.append(n)
    for x in sorted({x for r, n in zip(table, lens) for x in r[:-(-n // PAGE)]} - kept):
        free[count] = x
        count += 1
    src, dst = [-1] * len(table), [-1] * len(table)
    for b, page in ask:
        count -= 1
        rows[b][-1] = free[count]
        src[b], dst[b] = page, free[count]
    rows = [r + [-1] * (width - len(r)) for r in rows]
    return (_ints(rows), _ints(new), _ints(free), _ints([count]), _ints(src), _ints(dst), _moved(s.caches, src, dst))


def _exact_compact(s):
    table, lens, free, count = s.table.tolist(), s.lens.tolist(), s.free.tolist(), int(s.count)
    live = {x for r, n in zip(table, lens) for x in r[:-(-n // PAGE)]}
    ids = sorted(live | set(free[:count]))
    low, rest = ids[:len(live)], ids[len(live):]
    dst = [x for x in low if x not in live]
    src = [x for x in reversed(rest) if x in live]
    to = dict(zip(src, dst))
    rows = [[to.get(x, x) if i < -(-n // PAGE) else -1 for i, x in enumerate(r)] for r, n in zip(table, lens)]
    half = max(1, s.pool // 2)
    pad = lambda x, n: _ints(x + [-1] * (n - len(x)))  # noqa: E731
    return (_ints(rows), pad(rest[::-1], len(free)), _ints([len(rest)]), pad(src, half), pad(dst, half),
            _ints([len(src)]), _moved(s.caches, src, dst))


def _moved(caches, src, dst):
    pairs = [(a, b) for a, b in zip(src, dst) if b >= 0]
    a, b = (torch.tensor([p[i] for p in pairs], dtype=torch.long, device=DEV) for i in (0, 1))
    for c in caches:
        c.view(torch.uint8).index_copy_(0, b, c.view(torch.uint8).index_select(0, a))
    return caches
