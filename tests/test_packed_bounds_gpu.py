"""First rows of packed sequences that make no sense: rows outside the tensors are neither read (they hold NaN here, which
would show) nor written (guards around the outputs and the workspace), and whoever's rows do make sense is served."""
import pytest
import torch

from helpers import BF, D
from q8_ref import F8
from test_packed_gpu import SCALE, ints

pytestmark = pytest.mark.gpu
LO, HI = -2 ** 31, 2 ** 31 - 1
T, SPARE = 80, 300
NONSENSE = [[0, 50, 20, 80], [-40, 30, 60, 10 ** 6], [90, 70, 50, 10], [10, LO, 20, 80], [60, LO + 5, LO, 70], [HI, LO, HI, 80],
            [0, HI, LO, 80], [LO, LO, HI, HI], [0, 0, HI, 0]]


def inside_nan(shape, seed, dev):
    """T rows of a larger tensor that holds NaN in front of them and behind."""
    x = torch.full((T + 2 * SPARE, *shape), float("nan"), dtype=BF, device=dev)
    x[SPARE:SPARE + T] = torch.randn((T, *shape), generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(BF)
    return x[SPARE:SPARE + T]


@pytest.mark.parametrize("hq", [2, 320])      # without a list of tiles and with one
@pytest.mark.parametrize("cu", NONSENSE)
def test_packed_prompts_stay_in_bounds(dev, cu, hq):
    from atflash import _lib, interface
    L = _lib.lib()
    hkv, B = hq // 2, len(cu) - 1
    q, k, v = (inside_nan((h, D), i, dev) for i, h in enumerate((hq, hkv, hkv)))
    out = torch.full((T + 2, hq, D), 7.0, dtype=BF, device=dev)
    lse = torch.full((hq + 2, T), 5.0, device=dev)
    size = L.atf_flash_packed_workspace_bytes(B, T, T, hq, hkv)
    assert (L.atf_prefill_plan_bytes(B, T, hq) > 0) == (hq > 2)
    edge = 1 << 16
    ws = torch.full((size + 2 * edge,), 171, dtype=torch.uint8, device=dev)
    first = ints(cu, dev)
    _lib.check(L.atf_flash_packed_bf16(
        out[1:].data_ptr(), hq * D, D, lse[1:].data_ptr(), q.data_ptr(), hq * D, D, k.data_ptr(), hkv * D, D, v.data_ptr(),
        hkv * D, D, first.data_ptr(), B, T, T, hq, hkv, None, SCALE, None, 0, 0, ws.data_ptr() + edge, size,
        _lib.stream_of(q.device)))
    assert (ws[:edge] == 171).all() and (ws[edge + size:] == 171).all()
    assert (out[0] == 7.0).all() and (out[-1] == 7.0).all() and (lse[0] == 5.0).all() and (lse[-1] == 5.0).all()
    assert torch.isfinite(out.float()).all() and torch.isfinite(lse).all()
    starts = [min(max(c, 0), T) for c in cu]
    if starts == sorted(starts):  # sequences that do not overlap: each is its own call
        for a, b in zip(starts, starts[1:]):
            if a < b:
                o, s = interface._flash_attn_fwd(q[None, a:b], k[None, a:b], v[None, a:b])
                assert torch.equal(out[1 + a:1 + b], o[0]) and torch.equal(lse[1:-1, a:b], s[0])


@pytest.mark.parametrize("most", [2, T])      # token by token and by pages
@pytest.mark.parametrize("kv_dtype", [BF, F8])
@pytest.mark.parametrize("cu", NONSENSE)
def test_packed_writes_stay_in_bounds(dev, cu, kv_dtype, most):
    from atflash import interface
    from atflash.cache import PagedKVCache
    hkv, B, width = 2, len(cu) - 1, 5
    k, v = (inside_nan((hkv, D), i, dev) for i in range(2))
    a, b = (PagedKVCache(B * width + 2, hkv, dev, kv_dtype=kv_dtype) for _ in range(2))
    table = ints([[1 + i * width + j for j in range(width)] for i in range(B)], dev)
    zero = ints([0] * B, dev)
    interface.kv_write_packed(a, k, v, ints(cu, dev), most, zero, table)
    for i in range(B):  # the same, a sequence at a time
        lo, hi = max(cu[i], 0), min(max(cu[i + 1], 0), T)
        if lo < hi:
            interface.kv_write_packed(b, k[lo:hi], v[lo:hi], ints([0, hi - lo], dev), most, zero[:1], table[i:i + 1].contiguous())
    assert torch.equal(a.kv.view(torch.uint8), b.kv.view(torch.uint8))
    assert a.exps is None or torch.equal(a.exps, b.exps)
    assert torch.isfinite(a.kv.float()).all()
