"""Refusals of the norms, log probabilities, shared tables and page copies, before anything reaches the GPU: the C entry points'
validation, the Python operators' checks, and the host side of tables and caches that share pages."""
import ctypes
import math
import os

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
P = 1 << 20  # an address that no call may use


@pytest.fixture
def lib():
    """The library, where no GPU is visible: a call that passes validation would run on these addresses."""
    from atflash import _lib
    if torch.cuda.is_available():
        pytest.skip("validation with made-up addresses runs on the CPU tier only")
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("HIP library not built")
    return _lib.lib()


def call(fn, args, **change):
    assert set(change) <= set(args)
    return fn(*{**args, **change}.values())


NORM = dict(q_out=P, q=P, q_st=512, q_sh=128, hq=4, k_out=P, k=P, k_st=256, k_sh=128, hk=2, qw=P, kw=P, fp32=0, eps=1e-6, rows=9,
            pos=P, rope=P, rope_pos=64, stream=None)
WRITE = dict(q_out=P, q=P, q_st=512, q_sh=128, hq=4, kv=P, exps=None, pages=4, hkv=2, k=P, ks_t=256, ks_h=128, v=P, vs_t=256, vs_h=128,
             qw=P, kw=P, fp32=0, eps=1e-6, batch=1, cu=P, total=8, most=4, start=P, table=P, max_pages=4, rope=P, rope_pos=64,
             stream=None)
LOGP = dict(logp=P, entropy=P, values=P, ids=P, x=P, type=0, stride=5000, rows=600, vocab=5000, tokens=P, n=1, top=3, ws=None, bytes=0,
            stream=None)
SELECT = dict(out=P, table=2 * P, width=8, lens=P, free=P, n_free=8, count=P, parents=P, batch=4, pages=32, lens_out=2 * P, left=P, src=P,
              dst=P, stream=None)
COMPACT = dict(out=P, table=2 * P, width=8, lens=P, free_out=P, free=2 * P, n_free=8, count=P, batch=4, pages=32, left=P, src=P, dst=P,
               copies=16, n=P, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), 1), (dict(hq=-1), 1), (dict(hk=-1), 1), (dict(q=None), 1), (dict(q_out=None), 1), (dict(qw=None), 1), (dict(k=None), 1),
    (dict(k_out=None), 1), (dict(kw=None), 1), (dict(eps=-1.0), 1), (dict(eps=math.nan), 1), (dict(eps=math.inf), 1), (dict(q=P + 8), 1),
    (dict(k_out=P + 8), 1), (dict(kw=P + 4), 1), (dict(q_sh=4), 1), (dict(k_st=129), 1), (dict(pos=None), 1), (dict(rope=P + 4), 1),
    (dict(rope_pos=0), 1), (dict(hq=70000), 2), (dict(rows=0, q=None), 0), (dict(hq=0, hk=0, q=None), 0)])
def test_norm_validation(lib, change, code):
    assert call(lib.atf_qk_norm_rope_bf16, NORM, **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(batch=-1), 1), (dict(most=-1), 1), (dict(total=-1), 1), (dict(cu=None), 1), (dict(kv=None), 1), (dict(q=None), 1), (dict(k=None), 1),
    (dict(v=None), 1), (dict(start=None), 1), (dict(table=None), 1), (dict(kw=None), 1), (dict(qw=None), 1), (dict(q_out=None), 1),
    (dict(pages=0), 1), (dict(hkv=0), 1), (dict(max_pages=0), 1), (dict(hq=-1), 1), (dict(eps=-1e-9), 1), (dict(v=P + 2), 1), (dict(ks_t=4), 1),
    (dict(q_st=3), 1), (dict(rope_pos=0), 1), (dict(batch=70000), 2), (dict(hkv=70000), 2), (dict(hq=70000), 2), (dict(batch=0, kv=None), 0),
    (dict(total=0), 0), (dict(most=0, kv=None), 0)])
def test_norm_write_validation(lib, change, code):
    assert call(lib.atf_qk_norm_write, WRITE, **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), 1), (dict(n=-1), 1), (dict(top=-1), 1), (dict(type=3), 1), (dict(vocab=0), 1), (dict(top=9, vocab=8), 1), (dict(x=None), 1),
    (dict(entropy=None), 1), (dict(logp=None), 1), (dict(tokens=None), 1), (dict(values=None), 1), (dict(ids=None), 1), (dict(x=P + 1), 1),
    (dict(x=P + 2, type=2), 1), (dict(tokens=P + 4), 1), (dict(top=65), 2), (dict(vocab=(1 << 30) + 1), 2), (dict(rows=3, vocab=50000), 4),
    (dict(rows=3, vocab=50000, ws=P, bytes=64), 4), (dict(rows=3, vocab=50000, ws=P + 8, bytes=1 << 20), 4), (dict(rows=0, x=None), 0)])
def test_logprobs_validation(lib, change, code):
    assert call(lib.atf_token_logprobs, LOGP, **change) == code


def test_logprobs_workspace(lib):
    size = lib.atf_logprobs_workspace_bytes
    assert size(0, 5000, 0, 3) == 0 and size(3, 0, 0, 3) == 0 and size(3, 5000, 0, -1) == 0
    assert size(5000, 152064, 0, 20) == 0  # a workgroup a row
    for rows in (1, 7, 48, 300):
        for top in (0, 1, 20, 64):
            n = size(rows, 152064, 0, top)
            assert n > 0 and n % (rows * (16 + 8 * top)) == 0
            splits = n // (rows * (16 + 8 * top))
            assert 2 <= splits and splits * max(top, 1) <= 2048 and splits * rows <= 1024


@pytest.mark.parametrize("change,code", [
    (dict(batch=0), 1), (dict(width=0), 1), (dict(n_free=-1), 1), (dict(pages=0), 1), (dict(out=None), 1), (dict(table=None), 1), (dict(lens=None), 1),
    (dict(free=None), 1), (dict(count=None), 1), (dict(parents=None), 1), (dict(lens_out=None), 1), (dict(left=None), 1), (dict(src=None), 1),
    (dict(dst=None), 1), (dict(out=2 * P), 1), (dict(lens_out=P), 1), (dict(batch=8192), 2), (dict(batch=8000, width=1 << 18), 2),
    (dict(pages=(1 << 19) + 1), 2)])
def test_select_validation(lib, change, code):
    assert call(lib.atf_select_tables, SELECT, **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(batch=0), 1), (dict(width=0), 1), (dict(n_free=-1), 1), (dict(pages=0), 1), (dict(out=None), 1), (dict(free_out=None), 1),
    (dict(free=None), 1), (dict(count=None), 1), (dict(left=None), 1), (dict(src=None), 1), (dict(dst=None), 1), (dict(n=None), 1),
    (dict(copies=15), 1), (dict(out=2 * P), 1), (dict(free_out=2 * P), 1), (dict(batch=8192), 2), (dict(pages=(1 << 19) + 2, copies=1 << 20), 2)])
def test_compact_validation(lib, change, code):
    assert call(lib.atf_compact_tables, COMPACT, **change) == code


def test_copy_validation(lib):
    one, size = (ctypes.c_void_p * 1)(P), (ctypes.c_int64 * 1)(64)

    def copy(caches=one, sizes=size, n_caches=1, pages=8, src=P, dst=P, n=3):
        return lib.atf_copy_pages(caches, sizes, n_caches, pages, src, dst, n, None, None)
    assert copy(n_caches=-1) == 1 and copy(n=-1) == 1 and copy(caches=None) == 1 and copy(sizes=None) == 1
    assert copy(src=None) == 1 and copy(dst=None) == 1 and copy(pages=0) == 1
    assert copy(caches=(ctypes.c_void_p * 1)(None)) == 1 and copy(sizes=(ctypes.c_int64 * 1)(0)) == 1
    assert copy(sizes=(ctypes.c_int64 * 1)(1 << 50)) == 1
    assert copy(n_caches=0) == 0 and copy(n=0) == 0


# ---- the Python operators ----

def fake(*shape, dtype=BF, dev="cuda:0"):
    return torch.empty(shape, dtype=dtype, device=dev)


def valid():
    """name -> (operator, its arguments) of calls that would reach the library."""
    from atflash import ops
    i32 = torch.int32
    q, k, w = fake(9, 4, 128), fake(9, 2, 128), fake(128)
    cs, pos = fake(64, 64, 2, dtype=torch.float32), fake(9, dtype=i32)
    kv, kv8, exps = fake(8, 2, 2, 2048), fake(8, 2, 2, 2048, dtype=F8), fake(8, 2, 2, dtype=torch.int8)
    table, lens, free, one, cu = fake(2, 4, dtype=i32), fake(2, dtype=i32), fake(8, dtype=i32), fake(1, dtype=i32), fake(3, dtype=i32)
    norm = dict(q=q, k=k, q_weight=w, k_weight=w.clone(), eps=1e-6, positions=pos, rope_cs=cs)
    write = dict(kv_cache=kv, kv_exps=None, q=q, k=k, v=k.clone(), q_weight=w, k_weight=w.clone(), eps=1e-6, cu_seqlens=cu, max_tokens=5,
                 start_pos=lens, page_table=table, rope_cs=cs)
    tables = dict(page_table=table, seq_lens=lens, free_pages=free, free_count=one)
    return {"norm": (ops.qk_norm_rope, norm), "write": (ops.qk_norm_write, write),
            "write8": (ops.qk_norm_write, {**write, "kv_cache": kv8, "kv_exps": exps}),
            "logprobs": (ops.token_logprobs, dict(logits=fake(3, 500), tokens=fake(3, dtype=torch.int64), top=4)),
            "select": (ops.select_tables, {**tables, "parents": lens.clone(), "num_pages": 8}),
            "compact": (ops.compact_tables, {**tables, "num_pages": 8}),
            "copy": (ops.copy_pages, dict(caches=[kv, exps], src=lens, dst=lens.clone(), count=one))}


BAD = {
    "norm": [("q", lambda: fake(9, 4, 64)), ("q", lambda: fake(9, 4, 128, dtype=torch.float16)), ("q", lambda: fake(9, 128, 4).transpose(1, 2)),
             ("k", lambda: fake(8, 2, 128)), ("k", lambda: fake(9, 2, 128, dev="cuda:1")), ("q_weight", lambda: fake(64)),
             ("q_weight", lambda: fake(128, dtype=torch.float32)), ("k_weight", lambda: fake(256)[::2]), ("eps", lambda: -1.0),
             ("eps", lambda: math.nan), ("positions", lambda: None), ("positions", lambda: fake(9, dtype=torch.int64)),
             ("positions", lambda: fake(8, dtype=torch.int32)), ("rope_cs", lambda: fake(64, 64, 2)), ("rope_cs", lambda: fake(64, 32, 2, dtype=torch.float32)),
             ("q", lambda: fake(9, 4, 128, dev="cpu"))],
    "write": [("q", lambda: fake(8, 4, 128)), ("k", lambda: fake(9, 3, 128)), ("v", lambda: fake(9, 2, 64)), ("v", lambda: fake(9, 2, 128, dtype=torch.float32)),
              ("kv_cache", lambda: fake(8, 2, 2, 2048, dtype=F8)), ("kv_exps", lambda: fake(8, 2, 2, dtype=torch.int8)),
              ("cu_seqlens", lambda: fake(2, dtype=torch.int32)), ("start_pos", lambda: fake(2, dtype=torch.int64)),
              ("page_table", lambda: fake(2, 4, dtype=torch.int64)), ("max_tokens", lambda: -2 ** 33), ("eps", lambda: math.inf),
              ("page_table", lambda: fake(2, 4, dtype=torch.int32, dev="cuda:1"))],
    "write8": [("kv_exps", lambda: fake(8, 2, 2)), ("kv_exps", lambda: fake(7, 2, 2, dtype=torch.int8))],
    "logprobs": [("logits", lambda: fake(3, 500, dtype=torch.float64)), ("logits", lambda: fake(500)), ("logits", lambda: fake(500, 3).t()),
                 ("logits", lambda: fake(3, 0)), ("tokens", lambda: fake(3, dtype=torch.int32)), ("tokens", lambda: fake(4, dtype=torch.int64)),
                 ("tokens", lambda: fake(3, 2, 2, dtype=torch.int64)), ("tokens", lambda: fake(3, dtype=torch.int64, dev="cpu")),
                 ("top", lambda: -1), ("top", lambda: 65), ("tokens", lambda: fake(6, dtype=torch.int64)[::2])],
    "select": [("page_table", lambda: fake(2, 4, dtype=torch.int64)), ("seq_lens", lambda: fake(3, dtype=torch.int32)),
               ("parents", lambda: fake(2, dtype=torch.int64)), ("parents", lambda: fake(1, dtype=torch.int32)),
               ("free_count", lambda: fake(2, dtype=torch.int32)), ("free_pages", lambda: fake(2, 4, dtype=torch.int32)),
               ("num_pages", lambda: 2 ** 32 + 8), ("parents", lambda: fake(2, dtype=torch.int32, dev="cuda:1"))],
    "compact": [("seq_lens", lambda: fake(2, dtype=torch.int64)), ("free_pages", lambda: fake(16, dtype=torch.int32)[::2]),
                ("num_pages", lambda: -2 ** 32 + 8)],
    "copy": [("caches", lambda: [fake(8, 4), fake(7, 4)]), ("caches", lambda: [fake(8, 4).t()]), ("caches", lambda: [fake(8, 4, dev="cuda:1")]),
             ("caches", lambda: [fake()]), ("src", lambda: fake(3, dtype=torch.int32)), ("dst", lambda: fake(2, dtype=torch.int64)),
             ("src", lambda: fake(2, 1, dtype=torch.int32)), ("count", lambda: fake(2, dtype=torch.int32)),
             ("dst", lambda: fake(2, dtype=torch.int32, dev="cuda:1"))],
}


@pytest.mark.parametrize("name,i", [(n, i) for n, bad in BAD.items() for i in range(len(bad))])
def test_operators_refuse(monkeypatch, name, i):
    from atflash import _lib
    reached = []
    monkeypatch.setattr(_lib, "launch", lambda *a: reached.append(a))
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: 4096)
    from atflash import ops
    monkeypatch.setattr(ops, "_data_ptr", lambda t: 4096)
    with FakeTensorMode():
        op, args = valid()[name]
        op(**args)
        assert len(reached) == 1  # the call itself is a good one
        key, bad = BAD[name][i]
        with pytest.raises(ValueError):
            op(**{**args, key: bad()})
        assert len(reached) == 1


def test_cpu_tensors_are_refused():
    from atflash import ops
    with pytest.raises(ValueError, match="GPU only"):
        ops.token_logprobs(torch.zeros(2, 9))
    with pytest.raises(ValueError, match="GPU only"):
        ops.copy_pages([torch.zeros(4, 4)], torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    t = torch.zeros((2, 4), dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU only"):
        ops.select_tables(t, t[:, 0].contiguous(), t[0], t[0, :1], t[:, 1].contiguous(), 8)


def test_fakes_have_the_operators_shapes():
    import atflash.ops  # noqa: F401  (registers them)
    O = torch.ops.atflash
    with FakeTensorMode():
        a = valid()
        n = a["norm"][1]
        q, k = O.qk_norm_rope(*n.values())
        assert q.shape == n["q"].shape and k.shape == n["k"].shape and q.dtype == BF
        assert O.qk_norm_write(*a["write"][1].values()).shape == n["q"].shape
        logp, ent, vals, ids = O.token_logprobs(*a["logprobs"][1].values())
        assert logp.shape == (3,) and ent.shape == (3,) and vals.shape == (3, 4) and ids.dtype == torch.int64 and vals.dtype == torch.float32
        assert [tuple(x.shape) for x in O.select_tables(*a["select"][1].values())] == [(2, 4), (2,), (1,), (2,), (2,)]
        assert [tuple(x.shape) for x in O.compact_tables(*a["compact"][1].values())] == [(2, 4), (8,), (1,), (4,), (4,), (1,)]
        O.copy_pages(*a["copy"][1].values())


# ---- tables and caches that share pages ----

def test_tables_share_only_where_asked():
    from atflash.cache import PageTables
    t = PageTables(8, 2, 4, "cpu")
    with pytest.raises(ValueError, match="sharing"):
        t.select(torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="524288"):
        PageTables(2 ** 19 + 1, 2, 4, "cpu", sharing=True)
    shared = PageTables(8, 2, 4, "cpu", sharing=True)
    for call in (lambda c: shared.select(torch.zeros(2, dtype=torch.int32), [c]), lambda c: t.compact([c])):
        with pytest.raises(ValueError, match="8 pages"):
            call(torch.zeros(7, 4))


transformers = pytest.importorskip("transformers")


def config(cls="Qwen3Config", **kw):
    args = dict(vocab_size=64, hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=1,
                head_dim=128, max_position_embeddings=4096, rope_theta=1e4)
    return getattr(transformers, cls)(**{**args, **kw})


def test_shared_caches_refuse_what_pages_of_others_forbid():
    from atflash import hf
    c = hf.PagedCache(config(), 2, 100, device="cpu", sharing=True)
    assert c.page_table is c.tables.page_table and (c.page_table == -1).all() and len(c.page_tensors()) == 2
    assert len(hf.PagedCache(config(), 2, 100, device="cpu", sharing=True, kv_dtype=F8).page_tensors()) == 4
    lyr = c.layers[0]
    lyr.length = 20
    with pytest.raises(NotImplementedError, match="cropped"):
        lyr.crop(10)
    with pytest.raises(RuntimeError, match="given back"):
        c.reserve(20, 1)
    with pytest.raises(RuntimeError, match="inside a step"):
        c.reorder_cache(torch.tensor([0, 0]))
    with pytest.raises(ValueError, match="beam_idx"):
        c.reorder_cache(torch.tensor([0]))
    plain = hf.PagedCache(config(), 2, 100, device="cpu")
    with pytest.raises(NotImplementedError, match="sharing=True"):
        plain.reorder_cache(torch.tensor([0, 0]))


def test_norms_are_taken_and_given_back():
    from atflash import hf
    model = transformers.Qwen3ForCausalLM(config()).to(BF).eval()
    for layer in model.model.layers:
        with torch.no_grad():
            layer.self_attn.q_norm.weight.copy_(1 + 0.3 * torch.randn(128))
    norms = [layer.self_attn.q_norm for layer in model.model.layers]
    hook = hf.register(model, n_ctx=4096, norm_at_load=True)
    assert [n[0] for n in hook.norms] == norms and all(n[2] == model.config.rms_norm_eps for n in hook.norms)
    assert all(isinstance(layer.self_attn.k_norm, hf.IdentityNorm) for layer in model.model.layers)
    assert hook.new_cache(model.config, 1, 32, "cpu").layers[0].deferred
    again = hf.register(model, n_ctx=4096, norm_at_load=True)  # from the originals
    assert [n[0] for n in again.norms] == norms
    hook = hf.register(model, n_ctx=4096)
    assert hook.norms is None and [layer.self_attn.q_norm for layer in model.model.layers] == norms
    hf.register(model, n_ctx=4096, norm_at_load=True)
    hf.unregister(model)
    assert [layer.self_attn.q_norm for layer in model.model.layers] == norms
    with pytest.raises(ValueError, match="rope_at_load"):
        hf.register(model, n_ctx=4096, rope_at_load=False, norm_at_load=True)
    assert [layer.self_attn.q_norm for layer in model.model.layers] == norms


def test_other_norms_are_refused():
    from atflash import hf

    class PlusOne(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.weight, self.eps = torch.nn.Parameter(torch.full((128,), 0.1)), 1e-6

        def forward(self, x):
            x = x.float()
            return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.eps) * (1 + self.weight)
    model = transformers.Qwen3ForCausalLM(config()).eval()
    keep = model.model.layers[1].self_attn.k_norm
    for bad in (PlusOne(), torch.nn.LayerNorm(128), torch.nn.Identity(), torch.nn.RMSNorm(64, eps=1e-6)):
        model.model.layers[1].self_attn.k_norm = bad
        with pytest.raises(ValueError):
            hf.register(model, n_ctx=4096, norm_at_load=True)
        assert model.model.layers[1].self_attn.k_norm is bad
    model.model.layers[1].self_attn.k_norm = torch.nn.RMSNorm(128, eps=3e-5)
    with pytest.raises(ValueError, match="same eps"):
        hf.register(model, n_ctx=4096, norm_at_load=True)
    model.model.layers[1].self_attn.k_norm = keep
    without = transformers.Qwen2ForCausalLM(config("Qwen2Config")).eval()
    with pytest.raises(ValueError, match="q_norm"):
        hf.register(without, n_ctx=4096, norm_at_load=True)


def test_row_limits(lib):
    """A launch has 2^32 threads at most."""
    assert call(lib.atf_qk_norm_rope_bf16, NORM, rows=(1 << 25) + 1) == 2
    assert call(lib.atf_token_logprobs, LOGP, rows=(1 << 23) + 1, vocab=8) == 2


def test_models_with_kernel_norms_keep_their_state_dict():
    """Weights are saved and loaded under the norms' own names, replaced ones included; nothing of a model without its norms runs
    by another model's hook."""
    import copy
    from atflash import hf
    model = transformers.Qwen3ForCausalLM(config()).to(BF).eval()
    before = {n: p.clone() for n, p in model.state_dict().items()}
    names = [n for n, _ in model.named_parameters()]
    hook = hf.register(model, n_ctx=4096, norm_at_load=True)
    assert list(model.state_dict()) == list(before) and [n for n, _ in model.named_parameters()] == names
    new = {n: torch.randn(128).to(BF) if "q_norm" in n else p.clone() for n, p in before.items()}
    for assign in (False, True):
        model.load_state_dict(new, assign=assign)
        for i, layer in enumerate(model.model.layers):
            want = new[f"model.layers.{i}.self_attn.q_norm.weight"]
            assert torch.equal(hook.norms[i][0].weight, want) and torch.equal(layer.self_attn.q_norm.weight, want)
    model.float()
    assert all(q.weight.dtype == torch.float32 for q, _, _ in hook.norms)
    model.to(BF)
    x = [torch.zeros((1, h, 3, 128), dtype=BF) for h in (2, 1, 1)]
    other = transformers.Qwen3ForCausalLM(config()).to(BF).eval()
    plain = hf.register(other, n_ctx=4096)
    twin = hf.register(other, n_ctx=4096, norm_at_load=True)
    for wrong in (plain, twin):
        with pytest.raises(ValueError, match="another hook"):
            wrong(model.model.layers[0].self_attn, *x, None)
    with pytest.raises(ValueError, match="another hook"):
        hook(copy.deepcopy(model).model.layers[1].self_attn, *x, None)
    hf.unregister(model)
    assert isinstance(model.model.layers[0].self_attn.q_norm, type(other.model.layers[0].self_attn.q_norm.original))
    assert torch.equal(model.model.layers[1].self_attn.q_norm.weight, new["model.layers.1.self_attn.q_norm.weight"])


def test_e2e_refuses_too_many_alternatives():
    from atflash import e2e
    for n in ("65", "-1"):
        with pytest.raises(SystemExit, match="logprobs"):
            e2e.main(["--logprobs", n])
