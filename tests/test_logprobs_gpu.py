"""Log probabilities, entropy and top alternatives of rows of logits against 64 bits.

Tolerances (u = 2^-24, d = a logit's distance to the row's largest, D its largest magnitude that still counts: exp(-104) is
below the smallest fp32 number).  A term exp(d) comes of a subtraction, a product and an exponential: relative error (2 D + 2) u.
Adding n terms in a row and then over the threads adds at most (n + 16) u, n = 64 a chunk of 16 bytes times 8 a thread.  So log s is
off by E = (V / 512 + 64 + 16 + 2 D + 2) u, a log probability by E + (D + 2 |log p|) u + log s's own rounding, and the entropy
log s - t / s, t's terms with two roundings more, by E (1 + |t / s|) + 4 u (|log s| + |t / s|).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def exact(x, tokens, top):
    """On the CPU in 64 bits, rows with finite sums: (logp of all, entropy, top ids)."""
    x = x.cpu()
    logp = torch.log_softmax(x.double(), -1)
    ent = torch.special.entr(logp.exp()).sum(-1)
    ids = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[:, :top]
    return logp, ent, ids


def check(x, tokens, top, got=None):
    from atflash import ops
    logp, ent, vals, ids = ops.token_logprobs(x, tokens, top) if got is None else got
    R, V = x.shape
    want, went, wids = exact(x, tokens, top)
    assert torch.equal(ids.cpu(), wids)
    xd = x.double().cpu()
    d = xd - xd.amax(-1, keepdim=True)
    D = d.abs().where(d > -104, 0.0).amax(-1)
    E = (V / 512 + 64 + 16 + 2 * D + 2) * U
    log_s = torch.logsumexp(d, -1)
    ts = (log_s - went).abs()

    def close(a, w):
        a, far = a.double().cpu().reshape(R, -1), w.reshape(R, -1)
        assert torch.equal(torch.isneginf(a), torch.isneginf(far))
        tol = E[:, None] + (D[:, None] + 2 * far.abs() + log_s[:, None]) * U
        bad = ((a - far).abs() > tol) & torch.isfinite(far)
        assert not bad.any(), ((a - far).abs() / tol)[torch.isfinite(far)].max()
    if tokens is not None:
        assert logp.shape == tokens.shape
        close(logp, want.gather(1, tokens.cpu().reshape(R, -1)))
    if top:
        close(vals, want.gather(1, wids))
    bad = (ent.double().cpu() - went).abs() > E * (1 + ts) + 4 * U * (log_s.abs() + ts)
    assert not bad.any(), (ent, went)


def logits(R, V, kind, dev, seed, scale=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn((R, V), generator=g, device=dev) * scale
    return x.to(TYPES[kind]), torch.randint(0, V, (R,), generator=g, device=dev)


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("R,V,top", [(1, 1, 1), (2, 2, 0), (3, 7, 7), (1, 8, 3), (5, 9, 9), (4, 63, 20), (4, 65, 64), (1, 151, 32),
                                     (7, 1000, 5), (1, 4096, 64), (3, 8191, 1), (2, 8193, 20), (600, 777, 5), (700, 70, 64),
                                     (1, 50257, 20), (48, 50257, 20), (300, 33000, 8), (1, 152064, 5), (520, 40001, 3)])
def test_sizes(dev, kind, R, V, top):
    x, tokens = logits(R, V, kind, dev, R + V)
    check(x, tokens, top)


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("R", [3, 600])
@pytest.mark.parametrize("skip,V", [(1, 3001), (3, 8200), (5, 12), (7, 9)])
def test_rows_at_any_alignment_and_stride(dev, kind, R, skip, V):
    wide, tokens = logits(R, V + 16 + skip, kind, dev, V)
    x = wide[:, skip:skip + V]
    before = wide.clone()
    check(x, tokens % V, 5)
    assert torch.equal(wide, before)


@pytest.mark.parametrize("R", [2, 600])
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
def test_ties_go_to_the_lowest_id(dev, kind, R):
    g = torch.Generator(device=dev).manual_seed(1)
    for levels, V in ((1, 5000), (2, 20000), (9, 9001)):
        x = torch.randint(0, levels, (R, V), generator=g, device=dev).to(TYPES[kind])
        x[0, ::3] *= -0.0 if levels == 1 else 1.0  # zeros of both signs are equal
        check(x, torch.zeros(R, dtype=torch.int64, device=dev), 33)


@pytest.mark.parametrize("R", [1, 600])
@pytest.mark.parametrize("kind,E", [("bf16", 8), ("fp32", 4)])
@pytest.mark.parametrize("order", ["up", "down", "lanes", "front", "back"])
def test_the_best_in_any_order(dev, R, kind, E, order):
    """Logits that rise, fall, lie together, or rise from lane to lane so that a chunk has more candidates than there is room for."""
    V = 40000
    i = torch.arange(V, device=dev)
    x = {"up": i, "down": -i, "lanes": (i // E) % 64, "front": -(i // 700), "back": i // 900}[order].float()
    x = (x * 0.01).repeat(R, 1).to(TYPES[kind])
    tokens = torch.randint(0, V, (R,), device=dev, generator=torch.Generator(device=dev).manual_seed(3))
    for top in (1, 20, 64):
        check(x, tokens, top)


@pytest.mark.parametrize("R", [4, 600])
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("V", [130, 9000])
def test_masks(dev, R, kind, V):
    """Masked logits of -inf and of the type's lowest value; fewer left than alternatives."""
    x, tokens = logits(R, V, kind, dev, 5)
    low = torch.finfo(x.dtype).min
    for mask in (-math.inf, low):
        y = x.clone()
        y[:, 3:V - 4] = mask
        y[1, 1:] = mask
        y[1, 0] = 2.0
        y[2] = torch.where(torch.arange(V, device=dev) % 7 == 0, y[2], mask)
        check(y, tokens, 20)
    y = torch.full_like(x, low)  # nothing left but the lowest value: all alike
    check(y, tokens, 9)


@pytest.mark.parametrize("R", [3, 600])
def test_rows_of_minus_infinity(dev, R):
    from atflash import ops
    x, tokens = logits(R, 9000, "fp32", dev, 6)
    x[1] = -math.inf
    logp, ent, vals, ids = ops.token_logprobs(x, tokens, 4)
    assert logp[1] == -math.inf and ent[1] == 0 and vals[1].tolist() == [-math.inf] * 4 and ids[1].tolist() == [0, 1, 2, 3]
    rest = torch.arange(R, device=dev) != 1
    check(x[rest], tokens[rest].contiguous(), 4, [t[rest] for t in (logp, ent, vals, ids)])


@pytest.mark.parametrize("R", [4, 600])
def test_nan_and_infinity_stay_in_their_rows(dev, R):
    from atflash import ops
    x, tokens = logits(R, 9000, "bf16", dev, 7)
    x[1, 77] = math.nan
    x[2, 8999] = math.inf
    logp, ent, vals, ids = ops.token_logprobs(x, tokens, 3)
    assert torch.isnan(logp[1:3]).all() and torch.isnan(ent[1:3]).all() and torch.isnan(vals[1:3]).all()
    clean = x[1].clone()
    clean[77] = -math.inf
    assert ids[1].tolist() == torch.sort(clean.float(), descending=True, stable=True).indices[:3].tolist()
    assert ids[2, 0] == 8999
    rest = torch.tensor([i not in (1, 2) for i in range(R)], device=dev)
    check(x[rest], tokens[rest].contiguous(), 3, [t[rest] for t in (logp, ent, vals, ids)])


def test_large_logits_and_one_that_has_all(dev):
    x, tokens = logits(5, 30000, "fp32", dev, 8)
    x[0] += 1e6
    x[1] *= 1e30
    x[2, 17] = 300.0
    x[3] -= 3e38
    tokens[2] = 17
    from atflash import ops
    check(x, tokens, 6)
    logp, ent, _, _ = ops.token_logprobs(x, tokens, 0)
    assert logp[2] == 0 and ent[2] == 0


def test_several_tokens_padding_and_tokens_past_the_vocabulary(dev):
    from atflash import ops
    x, _ = logits(6, 5000, "bf16", dev, 9)
    tokens = torch.randint(0, 5000, (6, 11), device=dev)
    check(x, tokens, 0)
    plain = ops.token_logprobs(x, tokens)[0]
    tokens[2, 3], tokens[4, 0], tokens[5, 10], tokens[0, 0] = -100, -1, 5000, 2 ** 40
    logp = ops.token_logprobs(x, tokens)[0]
    assert logp[2, 3] == 0 and logp[4, 0] == 0 and torch.isnan(logp[5, 10]) and torch.isnan(logp[0, 0])
    ok = (tokens >= 0) & (tokens < 5000)
    assert torch.equal(logp[ok], plain[ok])
    none = ops.token_logprobs(x, None, 2)
    assert none[0].shape == (6, 0) and none[3].shape == (6, 2)
    empty = ops.token_logprobs(x[:0], None, 2)
    assert empty[1].shape == (0,) and empty[3].shape == (0, 2)


def test_offsets_past_31_bits(dev):
    from atflash import ops
    wide = torch.zeros((3, 2 ** 30 + 2 ** 29), dtype=torch.bfloat16, device=dev)
    x = wide[:, 5:5 + 20000]
    x.copy_(logits(3, 20000, "bf16", dev, 10)[0])
    check(x, torch.tensor([1, 2, 3], device=dev), 5)


def test_the_same_bits_every_time_and_captured(dev):
    from atflash import ops
    for R in (2, 600):
        x, tokens = logits(R, 50257, "bf16", dev, 11)
        ops.token_logprobs(x, tokens, 20)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.token_logprobs(x, tokens, 20)
        side = torch.cuda.Stream()
        for i in range(4):
            x.copy_(torch.roll(x, 1000 + i, 1))
            want = ops.token_logprobs(x, tokens, 20)
            torch.cuda.synchronize()
            graph.replay()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                other = ops.token_logprobs(x, tokens, 20)
            torch.cuda.synchronize()
            for a, b, c in zip(out, want, other):
                assert torch.equal(a, b) and torch.equal(b, c)


def test_registered_operator(dev):
    from atflash import ops
    x, tokens = logits(3, 5000, "fp16", dev, 12)
    for a, b in zip(ops.token_logprobs(x, tokens, 7), torch.ops.atflash.token_logprobs(x, tokens, 7)):
        assert torch.equal(a, b)
