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


class Norm(torch.nn.Module):
    """x f(x, eps) w of 128 dims, computed in fp32 and rounded as the models' norms are."""

    def __init__(self, f, eps=1e-6):
        super().__init__()
        self.weight, self.eps, self.f = torch.nn.Parameter((1 + 0.3 * torch.randn(128)).to(BF)), eps, f

    def forward(self, x):
        y = x.float() * self.f(x.float(), self.eps)
        return self.weight * y.to(x.dtype)


def mean(x):
    return x.square().mean(-1, keepdim=True)


EPS_ELSEWHERE = {
    "beside the root": lambda x, e: 1 / (mean(x).sqrt() + e),
    "a bound": lambda x, e: torch.rsqrt(mean(x).clamp(min=e)),
    "a bound of the root": lambda x, e: 1 / mean(x).sqrt().clamp(min=e),
    "of the sum": lambda x, e: torch.rsqrt((x.square().sum(-1, keepdim=True) + e) / 128),
    "squared": lambda x, e: torch.rsqrt(mean(x) + e * e),
    "not used": lambda x, e: torch.rsqrt(mean(x).clamp(min=1e-30)),
    "another": lambda x, e: torch.rsqrt(mean(x) + 1e-5),
}


@pytest.mark.parametrize("name", list(EPS_ELSEWHERE))
@pytest.mark.parametrize("side", ["q_norm", "k_norm"])
def test_norms_with_eps_elsewhere_are_refused(name, side):
    from atflash import hf
    model = model_of()
    setattr(model.model.layers[1].self_attn, side, Norm(EPS_ELSEWHERE[name]))
    with pytest.raises(ValueError, match="something else"):
        hf.register(model, n_ctx=4096, norm_at_load=True)


@pytest.mark.parametrize("eps", [0.0, 1e-12, 1e-6, 1e-5, 1e-3, 0.5])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_the_norm_itself_is_taken(eps, dtype):
    from atflash import hf
    g = torch.Generator().manual_seed(2)
    for norm in (Norm(lambda x, e: torch.rsqrt(mean(x) + e), eps), torch.nn.RMSNorm(128, eps=eps),
                 transformers.models.qwen3.modeling_qwen3.Qwen3RMSNorm(128, eps=eps)):
        norm = norm.to(dtype)
        with torch.no_grad():
            norm.weight.copy_(torch.randn(128, generator=g) * 2)
        assert hf._norm_eps(norm) == eps


def attention(model, how):
    """Layer 1's attention with its norms elsewhere."""
    Q = transformers.models.qwen3.modeling_qwen3
    base = type(model.model.layers[1].self_attn)

    class Changed(base):
        def forward(self, hidden_states, position_embeddings, attention_mask, past_key_values=None, **kwargs):
            if how == "raises":
                raise RuntimeError("not this way")
            shape = (*hidden_states.shape[:-1], -1, self.head_dim)
            q, k, v = (p(hidden_states).view(shape).transpose(1, 2) for p in (self.q_proj, self.k_proj, self.v_proj))
            cos, sin = position_embeddings
            if how == "one before, one behind":
                k = self.k_norm(k)
            q, k = Q.apply_rotary_pos_emb(q, k, cos, sin)
            if how != "one left out":
                q = self.q_norm(q)
            if how != "one before, one behind":
                k = self.k_norm(k)
            return q, k
    model.model.layers[1].self_attn.__class__ = Changed


@pytest.mark.parametrize("how", ["both behind", "one before, one behind", "one left out", "raises"])
@pytest.mark.parametrize("before", [False, True])
def test_norms_behind_the_rotation_are_refused(how, before):
    """The kernels norm before they rotate; the weight makes that another result than the other order."""
    from atflash import hf
    model = model_of()
    if before:
        hf.register(model, n_ctx=4096)  # (the rotation left to the kernels already)
    rot = model.model.rotary_emb
    attention(model, how)
    norms = [getattr(layer.self_attn, n) for layer in model.model.layers for n in ("q_norm", "k_norm")]
    with pytest.raises(ValueError, match="before the rotation"):
        hf.register(model, n_ctx=4096, norm_at_load=True)
    assert [getattr(layer.self_attn, n) for layer in model.model.layers for n in ("q_norm", "k_norm")] == norms
    assert all(not n._forward_pre_hooks for n in norms) and model.model.rotary_emb is rot
    assert hf.register(model, n_ctx=4096).norms is None  # without them as ever
    hf.unregister(model)


def test_the_trial_leaves_nothing():
    """Neither hooks, gradients, random numbers nor a cache's state; a model in training as well, twice, and behind another hook."""
    from atflash import hf
    model = model_of(3).train()
    state = torch.random.get_rng_state()
    for _ in range(2):
        hook = hf.register(model, n_ctx=4096, norm_at_load=True)
    assert len(hook.norms) == 3 and torch.equal(torch.random.get_rng_state(), state)
    for layer in model.model.layers:
        for n in (layer.self_attn.q_norm, layer.self_attn.k_norm):
            assert not n._forward_pre_hooks and not n.original._forward_pre_hooks and n.original.weight.grad is None
    hf.unregister(model)


def test_a_caller_without_an_attention_module_names_a_layer():
    import types
    from atflash import hf
    model = model_of(2)
    hook = hf.register(model, n_ctx=4096, norm_at_load=True)
    for i in range(2):
        hook._check_norms(types.SimpleNamespace(layer_idx=i))
    for wrong in (dict(layer_idx=2), dict(layer_idx=-1), dict(), dict(layer_idx=0, q_norm=model.model.layers[1].self_attn.q_norm),
                  dict(layer_idx=0, k_norm=model.model.layers[0].self_attn.k_norm.original)):
        with pytest.raises(ValueError, match="another hook"):
            hook(types.SimpleNamespace(**wrong), *states(), None)
    hf.unregister(model)
