"""Norms of the heads left to the kernels: which models a hook with norms, or without them, runs."""
import pytest
import torch

transformers = pytest.importorskip("transformers")
BF = torch.bfloat16


def model_of(layers=2, cls="Qwen3", **kw):
    args = dict(vocab_size=64, hidden_size=256, intermediate_size=256, num_hidden_layers=layers, num_attention_heads=2, num_key_value_heads=1,
                head_dim=128, max_position_embeddings=4096, rope_theta=1e4)
    return getattr(transformers, cls + "ForCausalLM")(getattr(transformers, cls + "Config")(**{**args, **kw})).to(BF).eval()


def states():
    return [torch.zeros((1, h, 3, 128), dtype=BF) for h in (2, 1, 1)]


def test_a_hook_with_norms_refuses_models_that_apply_their_own():
    """Attention functions are registered by name, so the last hook gets every model's calls: a model that norms its heads itself would
    be normed twice, by this model's weights."""
    from atflash import hf
    a, b = model_of(3), model_of(2)
    ha = hf.register(a, n_ctx=4096)
    hb = hf.register(b, n_ctx=4096, norm_at_load=True)
    assert transformers.AttentionInterface()[hf.ATTN_NAME] is hb
    for layer in a.model.layers:  # (the third one has no counterpart in b)
        with pytest.raises(ValueError, match="another hook"):
            hb(layer.self_attn, *states(), None)
    with pytest.raises(ValueError, match="another hook"):
        a(input_ids=torch.zeros((1, 3), dtype=torch.long), use_cache=False)
    for layer in a.model.layers:
        ha._check_norms(layer.self_attn)
    for layer in b.model.layers:
        hb._check_norms(layer.self_attn)
    hf.unregister(a)
    hf.unregister(b)
    with pytest.raises(ValueError, match="another hook"):  # b norms its heads itself again
        hb(b.model.layers[0].self_attn, *states(), None)


def test_a_hook_with_norms_refuses_models_without_any():
    from atflash import hf
    a, b = model_of(cls="Qwen2"), model_of()
    hf.register(a, n_ctx=4096)
    hb = hf.register(b, n_ctx=4096, norm_at_load=True)
    with pytest.raises(ValueError, match="another hook"):
        hb(a.model.layers[0].self_attn, *states(), None)
    hf.unregister(a)
    hf.unregister(b)


@pytest.mark.parametrize("name", ["q_norm", "k_norm"])
def test_both_norms_are_looked_at(name):
    from atflash import hf
    a, b = model_of(), model_of()
    ha = hf.register(a, n_ctx=4096, norm_at_load=True)
    plain = hf.register(b, n_ctx=4096)
    attn = a.model.layers[1].self_attn
    ha._check_norms(attn)
    setattr(attn, name, getattr(attn, name).original)
    with pytest.raises(ValueError, match="another hook"):  # one of the two would be applied twice
        ha(attn, *states(), None)
    with pytest.raises(ValueError, match="another hook"):  # the other not at all
        plain(attn, *states(), None)
    setattr(attn, name, hf.IdentityNorm(getattr(b.model.layers[1].self_attn, name)))
    with pytest.raises(ValueError, match="another hook"):  # another model's
        ha(attn, *states(), None)
    hf.unregister(a)
    hf.unregister(b)
