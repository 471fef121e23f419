"""The transformers hook on a PagedCache of 8-bit floats: its layers hold what the plain restatement of the writer holds,
its outputs are attention in 64 bits over those values, and a prompt in chunks is a prompt in one piece."""
import types

import pytest
import torch

transformers = pytest.importorskip("transformers")
from transformers import Qwen2Config, Qwen2ForCausalLM  # noqa: E402

from atflash import hf  # noqa: E402
from atflash.cache import dequantize  # noqa: E402
from atflash.model_tables import window_from_config  # noqa: E402
from q8_ref import Cache, E_MIN, F8, ages, attend, to_slices  # noqa: E402

CFG = dict(vocab_size=512, hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4,
           num_key_value_heads=2, max_position_embeddings=4096, rope_theta=1e4)


def test_layers_and_refusals_on_the_cpu():
    cfg = Qwen2Config(**CFG)
    c = hf.PagedCache(cfg, 2, 100, device="cpu", kv_dtype=F8)
    assert c.layers[0].kv.dtype == F8 and tuple(c.layers[1].exps.shape) == (14, 2, 2)
    assert (c.layers[0].exps == E_MIN).all()
    assert hf.PagedCache(cfg, 1, 20, device="cpu").layers[0].exps is None
    with pytest.raises(ValueError, match="kv_dtype"):
        hf.PagedCache(cfg, 1, 20, device="cpu", kv_dtype=torch.float16)
    k = torch.zeros((2, 2, 1, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU only"):
        c.layers[0].update(k, k)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["win", "off"])
def test_a_prompt_and_steps_through_the_hook(dev, mode):
    cfg = Qwen2Config(**CFG)
    win = window_from_config(cfg, 2.0, 2.0, 4096)
    hook = hf.WindowAttention(win, mode=mode)
    n, steps, hq, hkv = 70, 12, 4, 2
    cache = hook.new_cache(cfg, 2, n + steps, dev, kv_dtype=F8)
    lyr, module = cache.layers[1], types.SimpleNamespace(layer_idx=1)
    cs = cache.rope_cs.cpu()
    ref = Cache(lyr.kv.shape[0], hkv)
    g = torch.Generator().manual_seed(1)
    at = 0
    for m in [40, 30] + [1] * steps:
        q, k, v = (torch.randn((2, h, m, 128), generator=g).to(torch.bfloat16) for h in (hq, hkv, hkv))
        kd, vd = k.to(dev), v.to(dev)
        kd, vd = lyr.update(kd, vd)
        out, _ = hook(module, q.to(dev), kd, vd, None)
        for b in range(2):
            row = cache.page_table[b].tolist()
            ref.write(k[b].transpose(0, 1), v[b].transpose(0, 1), at, row, cs)
            rows = [(p, s) for p in row for s in range(16)][:at + m]
            kk, vv = (torch.stack([x[p, s] for p, s in rows]) for x in (ref.k, ref.v))
            for i in sorted({0, m - 1}):
                t = at + i + 1
                x = q[b, :, i].double()
                c, s = cs[t - 1, :, 0].double(), cs[t - 1, :, 1].double()
                x = torch.cat([x[:, :64] * c - x[:, 64:] * s, x[:, 64:] * c + x[:, :64] * s], -1)
                if mode == "off":
                    lims, age = None, None
                elif m == 1:
                    lims, age = list(win.decode_zhi8), ages(t, "key")
                else:
                    pos = torch.arange(t)
                    age = (at + i // 32 * 32 - (pos // 32 * 32 + 31)).clamp(min=0)[:, None].expand(-1, 16)
                    lims = [1 << 30] * 2 + [z for z in win.prefill_zhi[1:] for _ in range(2)]
                want, bound = attend(to_slices(x), kk[:t], vv[:t], lims, age, win.sm_scale, True)
                assert ((out[b, i].cpu().double() - want).abs() <= bound).all()
        at += m
    got_k, got_v = dequantize(lyr.kv, lyr.exps, range(lyr.kv.shape[0]))
    assert torch.equal(got_k.cpu(), ref.k) and torch.equal(got_v.cpu(), ref.v)


@pytest.mark.gpu
def test_chunks_of_a_model_are_the_single_shot(dev):
    torch.manual_seed(0)
    model = Qwen2ForCausalLM(Qwen2Config(**CFG)).to(torch.bfloat16).to(dev).eval()
    hook = hf.register(model, 2.0, 2.0, n_ctx=4096)
    ids = torch.randint(0, 512, (1, 200), generator=torch.Generator().manual_seed(3)).to(dev)
    logits = []
    for chunks in ([200], [64, 96, 40]):
        cache = hook.new_cache(model.config, 1, 210, dev, kv_dtype=F8)
        at = 0
        with torch.no_grad():
            for n in chunks:
                out = model(ids[:, at:at + n], past_key_values=cache, use_cache=True)
                at += n
            step = model(ids[:, :1], past_key_values=cache, use_cache=True)
        logits.append((out.logits[:, -1], step.logits[:, -1]))
        assert cache.get_seq_length() == 201 and torch.isfinite(step.logits.float()).all()
    assert torch.equal(logits[0][0], logits[1][0]) and torch.equal(logits[0][1], logits[1][1])
    hf.unregister(model)
