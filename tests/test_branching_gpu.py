"""The operators of a branching decode together, as a serving program runs them, and through the transformers hook."""
import types

import pytest
import torch

import helpers as H

pytestmark = pytest.mark.gpu
BF, F8 = torch.bfloat16, torch.float8_e4m3fn
D, P, PAGE = 128, 64, 16
EPS = 1e-6


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def norm_rope(x, w, pos, cs):
    """In 64 bits: x [n, h, 128], positions [n]."""
    x, w = x.double(), w.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    c, s = cs[pos, :, 0].double()[:, None], cs[pos, :, 1].double()[:, None]
    return torch.cat([y[..., :P] * c - y[..., P:] * s, y[..., P:] * c + y[..., :P] * s], -1)


@pytest.mark.parametrize("kv_dtype", [BF, F8])
def test_a_beam_search(dev, kv_dtype):
    """Two layers of attention with random projections, three prompts with four beams each: prompts prefilled once and forked, then steps
    of extend, qk_norm_write, decode, log probabilities, beams chosen among the alternatives, select and copies, with a
    compaction on the way.  Each step's log probabilities against a recomputation in 64 bits from the beams' own tokens.
      Tolerance of a log probability: helpers.assert_close's bar (2e-2 an attention output) through the head below, whose
    columns have 2-norm 1: a logit moves by at most 2e-2 times the columns' 1-norm, sqrt(hidden) at most, and log sum exp by as much;
    measured means are far smaller (1e-3), so the bar on the mean is taken too.  The 8-bit cache is off by 2^-4 of a value by
    design, so its keys and values are taken from the cache, not from the formula."""
    from atflash import cache as C, interface as I, ops, rope as R
    g = torch.Generator(device=dev).manual_seed(1)
    prompts, beams, hq, hkv, vocab, steps = [19, 32, 5], 4, 4, 2, 300, 12
    B, hid, layers = len(prompts) * beams, 256, 2
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    emb = rnd(vocab, hid).to(BF)
    proj = [(rnd(hid, (hq + 2 * hkv) * D) / hid ** 0.5).to(BF) for _ in range(layers)]
    out_w = [(rnd(hq * D, hid) / (hq * D) ** 0.5).to(BF) for _ in range(layers)]
    head = rnd(hid, vocab)
    head = (head / head.norm(dim=0)).to(BF)
    norms = [[(1 + 0.3 * rnd(D)).to(BF) for _ in range(2)] for _ in range(layers)]
    cs = R.rope_table(128, R.inv_freq(D, 1e4, dev))
    pool = 120
    caches = [C.PagedKVCache(pool, hkv, dev, kv_dtype=kv_dtype) for _ in range(layers)]
    pages = [t for c in caches for t in (c.kv, c.exps) if t is not None]
    tabs = C.PageTables(pool, B, 8, dev, sharing=True)

    def forward(tokens, new, most):
        """The last hidden states of packed new tokens (one launch a layer for norms, rotation and cache)."""
        start, cu, _, _ = tabs.extend(new, len(tokens))
        x = emb[tokens]
        for (qw, kw), w, o, c in zip(norms, proj, out_w, caches):
            y = (x @ w).view(-1, hq + 2 * hkv, D)
            q = I.qk_norm_write(c, y[:, :hq], y[:, hq:hq + hkv], y[:, hq + hkv:], qw, kw, cu, most, start, tabs.page_table, EPS, cs)
            if most == 1:
                a = I.decode_paged(q, c, tabs.page_table, tabs.seq_lens, 128)
            else:
                a, _ = I.prefill_packed(q, c, tabs.page_table, cu, tabs.seq_lens, 128)
            x = x + a.reshape(-1, hq * D) @ o
        return x

    def reference(history, rows):
        """Log probabilities behind each history, in 64 bits over the bf16 (or the cache's) keys and values; the bf16 steps
        between the layers as the program takes them."""
        res = []
        for b, toks in zip(rows, history):
            n = len(toks)
            x, pos = emb[torch.tensor(toks, device=dev)], torch.arange(n, device=dev)
            for (qw, kw), w, o, c in zip(norms, proj, out_w, caches):
                y = (x @ w).view(-1, hq + 2 * hkv, D)
                q, k, v = norm_rope(y[:, :hq], qw, pos, cs), norm_rope(y[:, hq:hq + hkv], kw, pos, cs).to(BF).double(), y[:, hq + hkv:].double()
                if kv_dtype == F8:
                    ids = tabs.page_table[b, :-(-n // PAGE)].tolist()
                    kk, vv = C.dequantize(c.kv, c.exps, ids)
                    order = torch.cat([torch.cat([torch.arange(60 - 4 * s, 64 - 4 * s), torch.arange(124 - 4 * s, 128 - 4 * s)]) for s in range(16)])
                    back = torch.empty(D, dtype=torch.long)
                    back[order] = torch.arange(D)
                    kk, vv = kk.flatten(0, 1)[:n][..., back.to(dev)].double(), vv.flatten(0, 1)[:n].double()
                    assert ((kk - k).abs() <= 2.0 ** -4 * 1.01 * k.abs() + 2.0 ** -7 * k.abs().amax()).all()  # what the cache holds is these keys
                    k, v = kk, vv
                k, v = (t.repeat_interleave(hq // hkv, 1) for t in (k, v))
                sc = torch.einsum("qhd,khd->hqk", q.cpu(), k.cpu()) * D ** -0.5
                sc = sc.masked_fill(torch.ones((n, n), dtype=torch.bool).triu(1), float("-inf"))
                a = torch.einsum("hqk,khd->qhd", sc.softmax(-1), v.cpu()).to(dev).to(BF)
                x = x + a.reshape(-1, hq * D) @ o
            res.append(torch.log_softmax((x[-1:] @ head).double(), -1)[0])
        return torch.stack(res)

    hist = [[int(t) for t in torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(n))] for n in prompts]
    first = [p * beams for p in range(len(prompts))]
    new = [0] * B
    for b, h in zip(first, hist):
        new[b] = len(h)
    tokens = torch.tensor([t for h in hist for t in h], device=dev)
    x = forward(tokens, ints(new, dev), max(prompts))
    last = torch.cumsum(torch.tensor(prompts), 0) - 1
    logits = x[last.to(dev)] @ head
    # fork every prompt into its beams, which start with its best tokens
    _, _, vals, ids = ops.token_logprobs(logits, None, beams)
    tabs.select(ints([b // beams * beams for b in range(B)], dev), pages)
    hist = [list(hist[b // beams]) + [int(ids[b // beams, b % beams])] for b in range(B)]
    score = vals.flatten().double().cpu()
    held = int(tabs.num_pages - tabs.free_count)
    assert held == sum(-(-n // PAGE) + (beams - 1) * (n % PAGE != 0) for n in prompts)  # whole pages are held once
    for step in range(steps):
        tok = torch.tensor([h[-1] for h in hist], device=dev)
        logits = forward(tok, ints([1] * B, dev), 1) @ head
        logp, ent, vals, ids = ops.token_logprobs(logits, ids.new_zeros(B), beams)
        rows = [0, 5, B - 1]
        want = reference([hist[b] for b in rows], rows)
        got = torch.log_softmax(logits[rows].double(), -1)
        diff = (got - want).abs()
        assert diff.max() <= 2 * 2e-2 * hid ** 0.5 and diff.mean() <= 2e-2, (step, diff.max(), diff.mean())
        full = torch.log_softmax(logits.double(), -1)
        assert (vals.double() - full.gather(1, ids)).abs().max() < 1e-5 and (logp.double() - full[:, 0]).abs().max() < 1e-5
        assert (ent.double() - torch.special.entr(full.exp()).sum(-1)).abs().max() < 1e-4
        cand = (score[:, None] + vals.double().cpu()).view(len(prompts), -1)
        best = cand.topk(beams, dim=-1)
        parents = (best.indices // beams + torch.arange(len(prompts))[:, None] * beams).flatten()
        chosen = ids.cpu()[parents, best.indices.flatten() % beams]
        score = best.values.flatten()
        tabs.select(parents.to(dev, torch.int32), pages)
        hist = [list(hist[p]) + [int(t)] for p, t in zip(parents.tolist(), chosen.tolist())]
        if step == 6:
            tabs.compact(pages)
            used = {p for r in tabs.page_table.tolist() for p in r if p >= 0}
            assert used == set(range(len(used)))
    tabs.release(ints(list(range(B)), dev))
    assert int(tabs.free_count) == pool and sorted(tabs.free_pages.tolist()) == list(range(pool))


# ---- through the transformers hook ----

transformers = pytest.importorskip("transformers")


def _qwen3(dev, layers=2):
    cfg = transformers.Qwen3Config(vocab_size=512, hidden_size=512, intermediate_size=1024, num_hidden_layers=layers, num_attention_heads=4,
                                   num_key_value_heads=2, head_dim=128, max_position_embeddings=4096, rope_theta=1e4)
    torch.manual_seed(0)
    model = transformers.Qwen3ForCausalLM(cfg).to(BF).to(dev).eval()
    with torch.no_grad():
        for layer in model.model.layers:
            for norm in (layer.self_attn.q_norm, layer.self_attn.k_norm):
                norm.weight.copy_(1 + 0.3 * torch.randn(128))
    model.set_attn_implementation("eager")
    return model


@pytest.mark.parametrize("mode", ["off", "win"])
@pytest.mark.parametrize("kind", ["paged", "plain"])
def test_hook_norms_against_64_bits(dev, kind, mode):
    """The hook called as a layer calls it, prompt in two chunks and steps: attention of the normed, rotated rows."""
    from atflash import hf
    from atflash.model_tables import window_from_config
    model = _qwen3(dev)
    win = window_from_config(model.config, 0.05, 0.05, 4096)
    mods = [(layer.self_attn.q_norm, layer.self_attn.k_norm) for layer in model.model.layers]
    hook = hf.WindowAttention(win, mode=mode, norms=mods)
    hq, hkv, b = 4, 2, 2
    cache = hook.new_cache(model.config, b, 90, dev)
    lyr, module = cache.layers[1], types.SimpleNamespace(layer_idx=1)
    cs = hook.rope_table(90, dev)
    g = torch.Generator().manual_seed(1)
    ks, vs, at = [], [], 0
    for m in (40, 33, 1, 1, 1):
        q, k, v = (torch.randn((b, h, m, D), generator=g).to(BF).to(dev) for h in (hq, hkv, hkv))
        ks.append(k)
        vs.append(v)
        K, V = torch.cat(ks, 2), torch.cat(vs, 2)
        if kind == "paged":
            k, v = lyr.update(k, v)
            out, _ = hook(module, q, k, v, None)
        else:
            out, _ = hook(module, q, K, V, None)
        n = at + m
        for i in range(b):
            qr = norm_rope(q[i].transpose(0, 1), mods[1][0].weight.detach(), torch.arange(at, n, device=dev), cs)
            kr = norm_rope(K[i].transpose(0, 1), mods[1][1].weight.detach(), torch.arange(n, device=dev), cs)
            vv = V[i].transpose(0, 1)
            base = 1e4
            if m == 1:
                ref = H.decode_oracle_vec8(qr[0].float().cpu(), kr.float().cpu(), vv.float().cpu(), base,
                                           win.decode_zhi8 if mode == "win" else None, False)
                got = out[i, 0]
            else:
                widths = H.wvec_for_levels(win.prefill_zhi) if mode == "win" else [1e9] * 64
                ref = H.prefill_oracle(qr[None].float().cpu(), kr[None].float().cpu(), vv[None].float().cpu(), base, None, False,
                                       q_offset=at, widths=widths)[0]
                got = out[i]
            H.assert_close(got, ref, f"{kind} {mode} rows {at}..{n - 1}")
        at = n


def test_model_with_norms_equals_eager(dev):
    """Window off: the logits of a model whose norms the kernels apply, against eager attention with the model's own."""
    from atflash import hf
    from test_hf_gpu import _close
    model = _qwen3(dev)
    ids = torch.randint(0, 512, (2, 150), generator=torch.Generator().manual_seed(3)).to(dev)
    with torch.no_grad():
        want = model(ids).logits.float()
        hook = hf.register(model, n_ctx=4096, mode="off", norm_at_load=True)
        _close(model(ids, use_cache=False).logits.float(), want, "norms by the kernels, no cache")
        cache = hook.new_cache(model.config, 2, 160, dev)
        parts = [model(ids[:, a:z], past_key_values=cache).logits.float() for a, z in ((0, 90), (90, 148), (148, 149), (149, 150))]
        _close(torch.cat(parts, 1), want, "norms by the kernels, paged")
        eight = hook.new_cache(model.config, 2, 160, dev, kv_dtype=F8)
        got = model(ids, past_key_values=eight).logits
        assert torch.isfinite(got).all() and eight.get_seq_length() == 150
        hook2 = hf.register(model, n_ctx=4096, mode="off")
        with pytest.raises(ValueError, match="norm mode"):
            model(ids[:, :4], past_key_values=hook.new_cache(model.config, 2, 16, dev))
        _close(model(ids, past_key_values=hook2.new_cache(model.config, 2, 160, dev)).logits.float(), want, "the model's own norms")
    hf.unregister(model)
    with torch.no_grad():
        assert torch.equal(model(ids).logits.float(), want)


@pytest.mark.parametrize("kv_dtype", [BF, F8])
@pytest.mark.parametrize("norm_at_load", [False, True])
def test_reordered_rows_are_their_histories(dev, kv_dtype, norm_at_load):
    """After any reordering every row's logits are, bit for bit, those of a cache that was fed the row's own tokens."""
    from atflash import hf
    model = _qwen3(dev)
    hook = hf.register(model, n_ctx=4096, norm_at_load=norm_at_load)
    B, n = 4, 45
    prompt = torch.randint(0, 512, (1, n), generator=torch.Generator().manual_seed(4)).expand(B, n).contiguous().to(dev)
    g = torch.Generator().manual_seed(5)
    cache = hook.new_cache(model.config, B, 80, dev, kv_dtype=kv_dtype, sharing=True)
    hist = [[] for _ in range(B)]
    with torch.no_grad():
        model(prompt, past_key_values=cache)
        cache.reorder_cache(torch.tensor([0, 0, 0, 0], device=dev))
        assert int(cache.tables.num_pages - cache.tables.free_count) == n // PAGE + B  # whole pages are held once
        for step in range(20):
            tok = torch.randint(0, 512, (B, 1), generator=g)
            got = model(tok.to(dev), past_key_values=cache).logits
            hist = [h + [int(t)] for h, t in zip(hist, tok)]
            if step in (1, 5, 12, 19):
                plain = hook.new_cache(model.config, B, 80, dev, kv_dtype=kv_dtype)
                model(prompt, past_key_values=plain)
                for i in range(len(hist[0])):
                    want = model(torch.tensor([[h[i]] for h in hist], device=dev), past_key_values=plain).logits
                assert torch.equal(got, want), step
            parents = torch.randint(0, B, (B,), generator=g) if step % 3 else torch.tensor([1, 2, 3, 0])
            cache.reorder_cache(parents.to(dev))
            hist = [list(hist[p]) for p in parents.tolist()]
        cache.reset()
        assert int(cache.tables.free_count) == cache.tables.num_pages
        again = model(prompt, past_key_values=cache).logits
        fresh = hook.new_cache(model.config, B, 80, dev, kv_dtype=kv_dtype)
        assert torch.equal(again, model(prompt, past_key_values=fresh).logits)
    hf.unregister(model)


def test_generate_with_beams(dev):
    """transformers' beam search on a cache that shares pages; the score it returns is the sequence's, taken anew.
      A token's log probability may differ by _close's bar on a logit, 0.1, twice (the token's and the sum's); the score is their mean."""
    from atflash import hf, ops
    model = _qwen3(dev)
    hook = hf.register(model, n_ctx=4096, mode="off", norm_at_load=True)
    n, new, beams = 37, 12, 3
    ids = torch.randint(2, 512, (2, n), generator=torch.Generator().manual_seed(6)).to(dev)
    cache = hook.new_cache(model.config, 2 * beams, n + new, dev, sharing=True)
    with torch.no_grad():
        out = model.generate(ids, past_key_values=cache, num_beams=beams, do_sample=False, max_new_tokens=new, min_new_tokens=new,
                             pad_token_id=0, return_dict_in_generate=True, output_scores=True, attention_mask=torch.ones_like(ids))
        assert out.sequences.shape == (2, n + new) and torch.equal(out.sequences[:, :n], ids)
        logits = model(out.sequences[:, :-1], use_cache=False).logits[:, n - 1:]
        logp = ops.token_logprobs(logits.reshape(-1, 512), out.sequences[:, n:].reshape(-1).contiguous())[0].view(2, new)
    for b in range(2):
        # (the length penalty divides by the generated length, with or without the prompt by version)
        total = float(logp[b].sum())
        assert min(abs(float(out.sequences_scores[b]) * m - total) for m in (new, n + new)) <= 0.2 * new
    hf.unregister(model)


def test_e2e_request_says_what_its_tokens_were_chosen_from(dev):
    from atflash import e2e, hf
    cfg = transformers.Qwen2Config(vocab_size=640, hidden_size=256, intermediate_size=256, num_hidden_layers=1, num_attention_heads=2,
                                   num_key_value_heads=1, max_position_embeddings=4096, rope_theta=1e4)
    model = e2e.build_model(cfg, dev)
    hook = e2e.use_mode(model, "off", 4096)
    ids = torch.randint(0, 640, (1, 96), generator=torch.Generator().manual_seed(7)).to(dev)
    plain = e2e.run_request(model, hook, ids, 64, 5)
    said = e2e.run_request(model, hook, ids, 64, 5, logprobs=3)
    assert "logprobs" not in plain and said["tokens"] == plain["tokens"] and len(said["logprobs"]) == 5
    for tok, s in zip(said["tokens"], said["logprobs"]):
        best = [x for _, x in s["top"]]
        assert len(best) == 3 and best == sorted(best, reverse=True) and s["logprob"] == best[0]  # greedy (equal logits: equal log probabilities)
        assert tok in [i for i, x in s["top"] if x == best[0]] or best[0] == best[-1]
        assert 0 <= s["entropy"] <= 6.47  # log 640
    hf.unregister(model)
