"""The 8-bit decode through its C entry with each of the two workspace sizes that its header allows."""
import pytest
import torch

from helpers import BF, D
from q8_ref import attend, to_slices
from test_q8_gpu import PAGE, SCALE, filled, row_of

pytestmark = pytest.mark.gpu


def decode_with(size, q, cache, table, lens, most):
    """out of a call whose workspace has `size` bytes, with a guard behind them that stays as it was."""
    from atflash import _lib
    B, hq, _ = q.shape
    guard = 4096
    ws = torch.full((size + guard,), 171, dtype=torch.uint8, device=q.device)
    out = torch.empty_like(q)
    _lib.check(_lib.lib().atf_decode_paged_q8(
        out.data_ptr(), hq * D, D, q.data_ptr(), hq * D, D, cache.kv.data_ptr(), cache.exps.data_ptr(), cache.num_pages,
        table.data_ptr(), table.shape[1], lens.data_ptr(), B, hq, cache.num_kv_heads, most, None, 0, SCALE, None, 0, 0,
        ws.data_ptr(), size, _lib.stream_of(q.device)))
    assert (ws[size:] == 171).all()
    return out


@pytest.mark.parametrize("lens,hq,hkv", [([4096, 700, 1, 33, 0, 2049, 16, 4000] * 8, 24, 8), ([9000, 32000, 5, 700], 6, 2),
                                         ([2500, 130, 1], 32, 2), ([1003], 24, 8)])
def test_either_workspace_is_enough(dev, lens, hq, hkv):
    from atflash import _lib, interface
    cache, table, keys = filled(lens, hkv, dev, 91)
    q = torch.randn((len(lens), hq, D), generator=torch.Generator(device=dev).manual_seed(92), device=dev).to(BF)
    n, most = row_of(lens, dev), max(lens)
    shape = (len(lens), hq, hkv, most)
    full, least = _lib.lib().atf_decode_q8_workspace_bytes(*shape), _lib.lib().atf_decode_workspace_bytes(*shape)
    assert torch.equal(decode_with(full, q, cache, table, n, most), interface.decode_paged(q, cache, table, n, most))
    got = decode_with(least, q, cache, table, n, most)
    for b in range(min(len(lens), 8)):
        if lens[b] == 0:
            assert (got[b] == 0).all()
            continue
        want, bound = attend(to_slices(q[b]), *keys[b], None, None, SCALE, False)
        assert ((got[b].double() - want).abs() <= bound).all()


def test_less_than_either_is_refused(dev):
    from atflash import _lib
    cache, table, _ = filled([9000], 2, dev, 93)
    q = torch.zeros((1, 6, D), dtype=BF, device=dev)
    least = min(f(1, 6, 2, 9000) for f in (_lib.lib().atf_decode_q8_workspace_bytes, _lib.lib().atf_decode_workspace_bytes))
    with pytest.raises(_lib.AtflashError, match="workspace"):
        decode_with(least - 16, q, cache, table, row_of([9000], dev), 9000)
