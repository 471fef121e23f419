"""The 8-bit cache on the CPU: the validation of its C entry points before anything reaches the GPU, the refusals of
its Python operators, and the plain restatement that the GPU tests compare with."""
import math

import pytest
import torch

from q8_ref import Cache, E_MAX, E_MIN, F8, exponent


def call(fn, args, **change):
    """fn with the arguments of a valid call, some of them changed."""
    a = dict(args)
    a.update(change)
    return fn(*a.values())


WRITE = dict(kv=1 << 20, exps=1 << 20, pages=4, hkv=2, k=1 << 20, ks_b=1024, ks_t=256, ks_h=128, v=1 << 20, vs_b=1024,
             vs_t=256, vs_h=128, batch=1, n=4, cu=None, total=0, start=1 << 20, table=1 << 20, max_pages=4, rope=None,
             rope_pos=0, layout=0, stream=None)
PACKED = dict(kv=1 << 20, pages=4, hkv=2, k=1 << 20, ks_t=256, ks_h=128, v=1 << 20, vs_t=256, vs_h=128, batch=1,
              cu=1 << 20, total=8, most=4, start=1 << 20, table=1 << 20, max_pages=4, rope=None, rope_pos=0, layout=0,
              stream=None)
DECODE = dict(out=1 << 20, o_sb=512, o_sh=128, q=1 << 20, q_sb=512, q_sh=128, kv=1 << 20, exps=1 << 20, pages=4,
              table=1 << 20, max_pages=4, lens=1 << 20, batch=1, hq=4, hkv=2, most=64, zhi=None, entries=0, scale=0.1,
              rope=None, rope_pos=0, layout=0, ws=None, ws_bytes=0, stream=None)
EXPAND = dict(out=1 << 20, out_table=1 << 20, kv=1 << 20, exps=1 << 20, pages=4, hkv=2, table=1 << 20, batch=1,
              max_pages=4, n_pages=4, lens=None, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(batch=-1), 1), (dict(n=-1), 1), (dict(kv=None), 1), (dict(exps=None), 1), (dict(k=None), 1),
    (dict(start=None), 1), (dict(pages=0), 1), (dict(hkv=0), 1), (dict(max_pages=0), 1), (dict(layout=7), 1),
    (dict(layout=1, rope=1 << 20, rope_pos=9), 1), (dict(rope=1 << 20, rope_pos=0), 1), (dict(k=(1 << 20) + 8), 1),
    (dict(vs_t=129), 1), (dict(cu=1 << 20, total=-1, ks_b=0, vs_b=0), 1), (dict(cu=1 << 20, total=8), 1),
    (dict(batch=70000), 2), (dict(hkv=70000), 2), (dict(batch=0, kv=None), 0), (dict(n=0), 0)])
def test_write_validation(no_gpu, change, code):
    assert call(no_gpu.atf_kv_write_q8, WRITE, **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(cu=None), 1), (dict(total=-1), 1), (dict(most=-1), 1), (dict(kv=None), 1), (dict(ks_t=4), 1), (dict(v=8), 1),
    (dict(batch=0), 0), (dict(total=0), 0), (dict(most=0), 0)])
def test_packed_write_validation(no_gpu, change, code):
    assert call(no_gpu.atf_kv_write_packed_bf16, PACKED, **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(batch=-1), 1), (dict(exps=None), 1), (dict(kv=None), 1), (dict(q=None), 1), (dict(hq=5), 1), (dict(hkv=0), 1),
    (dict(most=0), 1), (dict(most=65), 1), (dict(most=1 << 24), 1), (dict(zhi=1 << 20, entries=9), 1), (dict(scale=0.0), 1),
    (dict(scale=math.nan), 1), (dict(q=(1 << 20) + 8), 1), (dict(q_sh=4), 1), (dict(o_sh=2), 1), (dict(hq=34, hkv=2), 2),
    (dict(batch=70000), 2), (dict(hq=9000, hkv=9000), 2), (dict(most=4096, max_pages=256), 4), (dict(batch=0), 0)])
def test_decode_validation(no_gpu, change, code):
    assert call(no_gpu.atf_decode_paged_q8, DECODE, **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(batch=-1), 1), (dict(n_pages=-1), 1), (dict(out=None), 1), (dict(out_table=None), 1), (dict(kv=None), 1),
    (dict(exps=None), 1), (dict(table=None), 1), (dict(pages=0), 1), (dict(n_pages=5), 1), (dict(out=8), 1),
    (dict(batch=70000), 2), (dict(batch=60000, n_pages=60000, max_pages=60000), 2), (dict(n_pages=0, out=None), 0)])
def test_expand_validation(no_gpu, change, code):
    assert call(no_gpu.atf_kv_expand_q8, EXPAND, **change) == code


@pytest.fixture
def no_gpu(monkeypatch):
    """The library; the calls here end at its checks (or do nothing)."""
    from atflash import _lib
    return _lib.lib()


def test_operators_refuse_cpu_tensors_and_malformed_caches():
    from atflash import interface, ops
    from atflash.cache import PagedKVCache
    cache = PagedKVCache(2, 1, "cpu", kv_dtype=F8)
    assert cache.kv.dtype == F8 and tuple(cache.kv.shape) == (2, 1, 2, 2048) and (cache.exps == E_MIN).all()
    table, one = torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    k = torch.zeros((1, 3, 1, 128), dtype=torch.bfloat16)
    q = torch.zeros((1, 1, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU only"):
        ops.kv_write_q8(cache.kv, cache.exps, k, k, one, table, None, 0)
    with pytest.raises(ValueError, match="GPU only"):
        ops.kv_write_packed(cache.kv, cache.exps, k[0], k[0], torch.zeros(2, dtype=torch.int32), 3, one, table, None, 0)
    with pytest.raises(ValueError, match="GPU only"):
        interface.decode_paged(q, cache, table, one, 16)
    with pytest.raises(ValueError, match="GPU only"):
        interface.prefill_paged(k, cache, table, 3, 0)
    with pytest.raises(ValueError, match="kv_dtype"):
        PagedKVCache(2, 1, "cpu", kv_dtype=torch.float16)
    meta = torch.device("meta")
    for kv, exps in ((torch.empty((2, 1, 2, 2048), dtype=torch.bfloat16), cache.exps),
                     (cache.kv[:, :, :1], cache.exps), (cache.kv, cache.exps[:1]), (cache.kv, cache.exps.int())):
        with pytest.raises(ValueError):
            ops._check_cache_q8(kv, exps)
    with pytest.raises(ValueError, match="one device"):
        ops._one_device(torch.empty(1, device=meta), one)


def test_registered_operators_have_fakes():
    from atflash import ops  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q = torch.empty((2, 4, 128), dtype=torch.bfloat16, device="cuda")
        kv = torch.empty((8, 2, 2, 2048), dtype=F8, device="cuda")
        exps = torch.empty((8, 2, 2), dtype=torch.int8, device="cuda")
        table, lens = (torch.empty(s, dtype=torch.int32, device="cuda") for s in ((2, 4), (2,)))
        o = torch.ops.atflash.decode_paged_q8(q, kv, exps, table, lens, 64, None, 0.1, None, 0)
        assert o.shape == q.shape and o.dtype == q.dtype
        out, lse = torch.ops.atflash.prefill_q8(q[None].expand(2, 2, 4, 128), kv, exps, table, 2, 0, None, 0.1, None, 0)
        assert out.shape == (2, 2, 4, 128) and lse.shape == (2, 4, 2)


@pytest.mark.parametrize("top,e", [(0.0, E_MIN), (448.0, 0), (448.0000305, 1), (1.75, -8), (1.7500001, -7), (2.0 ** -130, E_MIN),
                                   (3.38e38, E_MAX), (1.0, -8), (256.0, 0), (224.0, -1)])
def test_the_restated_exponent(top, e):
    assert exponent(top) == e


def test_the_restated_cache_keeps_and_forgets():
    c = Cache(2, 1)
    x = torch.ones((20, 1, 128), dtype=torch.bfloat16)
    c.write(x, 2 * x, 0, [1, 0], None)
    assert (c.k[1] == 1).all() and (c.v[0, :4] == 2).all() and (c.v[0, 4:] == 0).all()
    c.write(1000 * x[:1], x[:1], 5, [1, 0], None)
    assert (c.k[1, :5] == 1).all() and (c.k[1, 5] == 1024).all() and (c.k[1, 6:] == 0).all()
    assert int(c.e[1, 0, 1]) == exponent(1000.0) and int(c.e[1, 0, 0]) == exponent(2.0)


PLAN = dict(plan=1 << 20, plan_bytes=1 << 20, cu=1 << 20, lens=None, batch=2, total=90000, most=60, hq=4, stream=None)
FLASH = dict(out=1 << 20, o_st=512, o_sh=128, lse=None, q=1 << 20, q_st=512, q_sh=128, k=1 << 20, ks_t=256, ks_h=128,
             v=1 << 20, vs_t=256, vs_h=128, cu=1 << 20, batch=2, total=100, most=60, hq=4, hkv=2, zhi=None, scale=0.1,
             rope=None, rope_pos=0, layout=0, ws=1 << 20, ws_bytes=1 << 20, stream=None)
PREFILL = dict(out=1 << 20, o_st=512, o_sh=128, lse=None, q=1 << 20, q_st=512, q_sh=128, kv=1 << 20, pages=9, table=1 << 20,
               max_pages=4, cu=1 << 20, lens=None, batch=2, total=90000, most=60, hq=4, hkv=2, zhi=None, scale=0.1, rope=None,
               rope_pos=0, layout=0, plan=1 << 20, plan_bytes=1 << 20, stream=None)
EXTEND = dict(table=1 << 20, max_pages=4, lens=1 << 20, new=1 << 20, free=1 << 20, num_free=4, count=1 << 20, batch=2,
              total=9, pages=9, lens_out=1 << 20, left=1 << 20, cu=1 << 20, pos=1 << 20, slots=1 << 20, stream=None)
RELEASE = dict(table=1 << 20, max_pages=4, lens=1 << 20, free=1 << 20, num_free=4, count=1 << 20, rows=1 << 20, n=1, batch=2,
               pages=9, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(batch=-1), 1), (dict(total=-1), 1), (dict(cu=None), 1), (dict(most=0), 1), (dict(hq=0), 1), (dict(most=1 << 24), 2),
    (dict(plan=None), 4), (dict(plan_bytes=8), 4), (dict(plan=(1 << 20) + 4), 4), (dict(batch=0), 0), (dict(total=0), 0)])
def test_plan_validation(no_gpu, change, code):
    assert call(no_gpu.atf_prefill_plan, PLAN, **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(batch=-1), 1), (dict(total=-1), 1), (dict(most=0), 1), (dict(most=1 << 24), 2), (dict(hkv=3), 1), (dict(hq=0), 1),
    (dict(cu=None), 1), (dict(q=None), 1), (dict(k=None), 1), (dict(v=None), 1), (dict(out=None), 1), (dict(ks_t=4), 1),
    (dict(v=8), 1), (dict(q_st=3), 1), (dict(o_sh=2), 1), (dict(scale=0.0), 1), (dict(rope=1 << 20, rope_pos=59), 1),
    (dict(layout=2), 1), (dict(ws=None), 4), (dict(ws_bytes=1000), 4), (dict(ws=(1 << 20) + 8), 4), (dict(batch=0), 0),
    (dict(total=0), 0)])
def test_flash_packed_validation(no_gpu, change, code):
    assert call(no_gpu.atf_flash_packed_bf16, FLASH, **change) == code


def test_flash_packed_workspace_holds_its_parts(no_gpu):
    for b, t, most, hq, hkv in ((1, 1, 1, 4, 4), (5, 1000, 517, 24, 8), (300, 20000, 9000, 28, 4), (3, 48, 16, 2, 1)):
        pages = (t // 16 + b) * hkv * 8192
        rest = no_gpu.atf_prefill_plan_bytes(b, t, hq) + 4 * b * -(-most // 16)
        assert pages + rest <= no_gpu.atf_flash_packed_workspace_bytes(b, t, most, hq, hkv) <= pages + rest + 48
    assert no_gpu.atf_flash_packed_workspace_bytes(0, 1, 1, 1, 1) == 0


@pytest.mark.parametrize("change,code", [
    (dict(batch=-1), 1), (dict(total=-1), 1), (dict(cu=None), 1), (dict(out=None), 1), (dict(q=None), 1), (dict(kv=None), 1),
    (dict(hkv=3), 1), (dict(max_pages=3), 1), (dict(most=1 << 24), 2), (dict(scale=-1.0), 1), (dict(rope=1 << 20, rope_pos=59), 1),
    (dict(layout=1, rope=1 << 20, rope_pos=99), 1), (dict(q=(1 << 20) + 8), 1), (dict(out=(1 << 20) + 4), 1), (dict(q_st=4), 1),
    (dict(o_st=2), 1), (dict(plan=None), 4), (dict(plan_bytes=9), 4), (dict(batch=0), 0), (dict(total=0), 0)])
def test_packed_prefill_validation(no_gpu, change, code):
    assert call(no_gpu.atf_prefill_packed_bf16, PREFILL, **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(batch=0), 1), (dict(batch=-2), 1), (dict(total=-1), 1), (dict(max_pages=0), 1), (dict(pages=0), 1),
    (dict(num_free=-1), 1), (dict(table=None), 1), (dict(lens=None), 1), (dict(new=None), 1), (dict(free=None), 1),
    (dict(count=None), 1), (dict(pos=None), 1), (dict(slots=None), 1), (dict(slots=(1 << 20) + 4), 1), (dict(cu=None), 1),
    (dict(batch=8192), 2)])
def test_extend_validation(no_gpu, change, code):
    assert call(no_gpu.atf_extend_tables, EXTEND, **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(batch=0), 1), (dict(n=-1), 1), (dict(rows=None), 1), (dict(table=None), 1), (dict(free=None), 1), (dict(pages=0), 1),
    (dict(n=0, rows=None), 0)])
def test_release_validation(no_gpu, change, code):
    assert call(no_gpu.atf_release_tables, RELEASE, **change) == code


def test_plan_size_covers_every_split_of_the_rows(no_gpu):
    # tiles of `batch` sequences with total rows: at most one started tile more for each; no list for small calls
    for batch, total, hq in ((1, 9000, 28), (3, 1500, 28), (300, 20000, 8), (8, 900, 64)):
        assert (no_gpu.atf_prefill_plan_bytes(batch, total, hq) // 4 - 2) // 2 == total // 256 + batch
    assert no_gpu.atf_prefill_plan_bytes(1, 1, 4) == no_gpu.atf_prefill_plan_bytes(5, 900, 24) == 0
    assert no_gpu.atf_prefill_plan_bytes(0, 5, 4) == no_gpu.atf_prefill_plan_bytes(1, 0, 4) == 0


def test_tables_and_packed_operators_refuse():
    from atflash import interface, ops
    from atflash.cache import PagedKVCache, PageTables
    i32 = torch.int32
    tabs = PageTables(8, 2, 4, "cpu")
    assert tabs.free_pages.tolist() == [7, 6, 5, 4, 3, 2, 1, 0] and int(tabs.free_count) == 8
    with pytest.raises(ValueError, match="GPU only"):
        tabs.extend(torch.ones(2, dtype=i32), 2)
    with pytest.raises(ValueError, match="GPU only"):
        tabs.release(torch.zeros(1, dtype=i32))
    q, k = torch.zeros((4, 6, 128), dtype=torch.bfloat16), torch.zeros((4, 4, 128), dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=i32)
    with pytest.raises(ValueError, match="multiple"):
        interface.flash_attn_packed(q, k, k, cu, 4)
    with pytest.raises(ValueError, match="GPU only"):
        interface.flash_attn_packed(q, k[:, :2], k[:, :2], cu, 4)
    cache = PagedKVCache(2, 2, "cpu")
    with pytest.raises(ValueError, match="GPU only"):
        interface.prefill_packed(q, cache, torch.zeros((1, 1), dtype=i32), cu, None, 4)
    with pytest.raises(ValueError, match="too small"):
        interface.prefill_packed(q, PagedKVCache(2, 2, "cpu", kv_dtype=F8), torch.zeros((1, 1), dtype=i32), cu, None, 40)
    with pytest.raises(ValueError, match="GPU only"):
        ops.PackedPlan(cu, None, 4, 4, 6)


def test_decode_workspace_holds_every_split(no_gpu):
    # partials of (batch, kv head, split): 16 rows of 130 floats; none where a sequence is one split
    for shape in ((1, 28, 4, 131072), (12, 24, 8, 32768), (40, 28, 4, 8192), (1, 24, 8, 1003), (64, 32, 8, 4096), (1, 4, 4, 16),
                  (300, 8, 8, 5000), (4, 32, 2, 65536), (1, 28, 4, 1 << 20)):
        size = no_gpu.atf_decode_q8_workspace_bytes(*shape)
        unit = shape[0] * shape[2] * 16 * 130 * 4
        assert size % unit == 0 and size // unit <= max(1, -(-shape[3] // 16)) and size <= 64 << 20
    assert no_gpu.atf_decode_q8_workspace_bytes(1, 4, 4, 16) == 0 == no_gpu.atf_decode_q8_workspace_bytes(0, 4, 4, 16)


def test_page_tables_past_30_bits_of_entries_are_refused(no_gpu):
    assert call(no_gpu.atf_extend_tables, EXTEND, batch=1025, max_pages=1 << 20) == 2


def test_flash_packed_bound_past_the_rows_costs_nothing(no_gpu):
    # no sequence has more rows than the call: a generous bound takes no more workspace, nor a longer RoPE table
    size = no_gpu.atf_flash_packed_workspace_bytes
    assert size(300, 500, (1 << 24) - 1, 24, 8) == size(300, 500, 500, 24, 8)
    assert call(no_gpu.atf_flash_packed_bf16, FLASH, most=5000, rope=1 << 20, rope_pos=99) == 1
    assert call(no_gpu.atf_flash_packed_bf16, FLASH, most=5000, rope=1 << 20, rope_pos=100, ws_bytes=1000) == 4


def test_packed_prompts_without_kv_heads_are_refused():
    from atflash import interface
    q, k = torch.zeros((4, 6, 128), dtype=torch.bfloat16), torch.zeros((4, 0, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="multiple"):
        interface.flash_attn_packed(q, k, k, torch.tensor([0, 4], dtype=torch.int32), 4)
