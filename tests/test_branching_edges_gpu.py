"""Calls at the ends of what the norms, log probabilities and shared pages allow: many short rows, many sequences of which few have
tokens, lists of tokens, calls on two streams at once, a step's calls captured as one graph.

Bounds are those that test_qk_norm_gpu.py and test_logprobs_gpu.py derive."""
import pytest
import torch

from test_logprobs_gpu import check, logits
from test_pages_gpu import ints, state
from test_qk_norm_gpu import BF, D, near, rows, table_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R,V,top", [(70001, 5, 2), (70001, 1, 1), (200000, 3, 0), (66000, 129, 3)])
def test_many_short_rows(dev, R, V, top):
    x, tokens = logits(R, V, "bf16", dev, R)
    check(x, tokens, top)


def test_lists_of_tokens(dev):
    """None, no tokens, and more of them than a workgroup has threads."""
    from atflash import ops
    for R in (2, 700):
        x, _ = logits(R, 9000, "bf16", dev, 3)
        for n in (0, 1, 257, 1500):
            tokens = torch.randint(0, 9000, (R, n), generator=torch.Generator().manual_seed(n)).to(dev)
            check(x, tokens, 2)
        logp, ent, vals, ids = ops.token_logprobs(x)
        assert logp.shape == (R, 0) and vals.shape == ids.shape == (R, 0)
        assert torch.equal(ent, ops.token_logprobs(x, tokens)[1])
    logp, ent, vals, ids = ops.token_logprobs(x[:0], tokens[:0], 5)
    assert logp.shape == (0, 1500) and ent.shape == (0,) and vals.shape == ids.shape == (0, 5)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("most", [1, 20])
def test_many_sequences_of_which_few_have_tokens(dev, eight, most):
    from atflash import cache, ops
    B, active = 65535, [0, 77, 40000, 65534]
    lens = torch.zeros(B, dtype=torch.int32)
    lens[active] = most
    cu = torch.cat([torch.zeros(1, dtype=torch.int32), lens.cumsum(0, dtype=torch.int32)]).to(dev)
    T = most * len(active)
    table = torch.full((B, 2), -1, dtype=torch.int32)
    for i, b in enumerate(active):
        table[b] = torch.tensor([2 * i, 2 * i + 1])
    start = torch.full((B,), 5, dtype=torch.int32, device=dev)
    pos = (5 + torch.arange(most, dtype=torch.int32)).repeat(len(active)).to(dev)
    q, k, v, qw, kw = rows(T, 3, 2, dev, most)
    cs = table_of(64, dev)
    kv, exps = cache.new_kv_cache_q8(8, 2, dev) if eight else (cache.new_kv_cache(8, 2, dev), None)
    want, wexps = kv.clone(), None if exps is None else exps.clone()
    out = ops.qk_norm_write(kv, exps, q, k, v, qw, kw, 1e-6, cu, most, start, table.to(dev), cs)
    near(out, q, qw, 1e-6, pos, cs)
    small = torch.arange(len(active) + 1, dtype=torch.int32, device=dev) * most
    ops.qk_norm_write(want, wexps, q, k, v, qw, kw, 1e-6, small, most, start[:len(active)], table[active].to(dev), cs)
    assert torch.equal(kv.view(torch.uint8), want.view(torch.uint8)) and (exps is None or torch.equal(exps, wexps))


def test_calls_on_two_streams_at_once(dev):
    """Nothing is shared between calls: each stream's results are those of the call by itself."""
    from atflash import ops
    xs = [logits(R, 50000, "bf16", dev, R)[0] for R in (40, 3)]
    tokens = [torch.arange(x.shape[0], device=dev) for x in xs]
    tabs = []
    for seed in (1, 2):
        table, lens, free = state(seed, 9, 40, 600, 700)
        tabs.append([ints(table, dev), ints(lens, dev), ints(free, dev), ints([len(free)], dev), ints([0, 0, 2, 2, 8, 1, 1, 8, 8], dev)])
    qs = [rows(n, 5, 2, dev, n) for n in (300, 9)]

    def calls(i):
        q, k, _, qw, kw = qs[i]
        t = tabs[i]
        free = t[2].clone()
        return [*ops.token_logprobs(xs[i], tokens[i], 7), *ops.select_tables(t[0], t[1], free, t[3], t[4], 700), free,
                *ops.qk_norm_rope(q, k, qw, kw, 1e-6, None, None)]
    alone = [calls(0), calls(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(calls(i))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, alone[i]))


@pytest.mark.parametrize("eight", [False, True])
def test_a_captured_step(dev, eight):
    """extend, norms into the cache, attention, log probabilities and the beams' choice as one graph, replayed with other inputs
    against the same calls made one by one."""
    from atflash import cache, ops
    B, hq, hkv, width, pool = 4, 6, 2, 6, 24
    qw, kw = rows(1, hq, hkv, dev, 1)[3:]
    cs = table_of(width * 16, dev)
    one = torch.ones(B, dtype=torch.int32, device=dev)

    def fresh():
        tabs = cache.PageTables(pool, B, width, dev, sharing=True)
        kv, exps = cache.new_kv_cache_q8(pool, hkv, dev) if eight else (cache.new_kv_cache(pool, hkv, dev), None)
        return tabs, kv, exps

    def step(s, x, proj, parents):
        tabs, kv, exps = s
        q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        start, cu, _, _ = tabs.extend(one, B)
        q = ops.qk_norm_write(kv, exps, q, k, v, qw, kw, 1e-6, cu, 1, start, tabs.page_table, cs)
        args = (tabs.page_table, tabs.seq_lens, width * 16, None, D ** -0.5, None, 0)
        o = ops.decode_paged_q8(q, kv, exps, *args) if eight else ops.decode_paged(q, kv, *args)
        said = ops.token_logprobs((o.flatten(1) * proj).contiguous(), None, 3)
        tabs.select(parents, [t for t in (kv, exps) if t is not None])
        return [o, *said]
    g = torch.Generator().manual_seed(3)
    xs = [torch.randn((B, hq + 2 * hkv, D), generator=g).to(BF).to(dev) for _ in range(40)]
    choice = [torch.randint(0, B, (B,), generator=g).to(torch.int32).to(dev) for _ in range(40)]
    proj = torch.randn((hq * D,), generator=g).to(BF).to(dev)
    x, parents = xs[0].clone(), choice[0].clone()
    a, b = fresh(), fresh()
    step(fresh(), x, proj, parents)  # (libraries and workspaces)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a, x, proj, parents)
    for i in range(40):
        x.copy_(xs[i])
        parents.copy_(choice[i])
        graph.replay()
        want = step(b, xs[i], proj, choice[i])
        torch.cuda.synchronize()
        assert all(torch.equal(p, w) for p, w in zip(out, want)), i
        assert torch.equal(a[0].page_table, b[0].page_table) and torch.equal(a[0].seq_lens, b[0].seq_lens)
        assert torch.equal(a[0].free_count, b[0].free_count)
        n = int(a[0].free_count)
        assert torch.equal(a[0].free_pages[:n], b[0].free_pages[:n])
        # every page is in use or free
        used = {p for r in a[0].page_table.tolist() for p in r if p >= 0}
        assert len(used) + n == pool and not used & set(a[0].free_pages[:n].tolist())


@pytest.mark.parametrize("order", ["random", "rising", "falling", "equal", "last few"])
@pytest.mark.parametrize("V,top", [(2_500_001, 0), (2_500_001, 1), (2_500_001, 9), (2_500_001, 30), (2_500_001, 64), (1_000_003, 17)])
def test_a_row_of_many_splits(dev, V, top, order):
    """More workgroups a row than a wave has lanes, and lists that are all alike, or of which one holds everything."""
    x = torch.randn((1, V), generator=torch.Generator(device=dev).manual_seed(V + top), device=dev) * 3
    if order == "rising":
        x = x.sort(-1).values
    elif order == "falling":
        x = x.sort(-1, descending=True).values
    elif order == "equal":
        x = torch.full_like(x, 0.25)
    elif order == "last few":
        x[:, -100:] += 20
    check(x.to(BF), torch.tensor([V // 2], device=dev), top)
