"""Rejected tokens cut off an 8-bit hook cache and others written in their place, beside a run that never had them: a cut
at a page's border leaves no trace; one inside a page keeps the page's exponents, which the rejected tokens may have raised."""
import pytest
import torch

transformers = pytest.importorskip("transformers")
from transformers import Qwen2Config  # noqa: E402

from atflash import hf  # noqa: E402
from atflash.cache import dequantize  # noqa: E402
from atflash.model_tables import window_from_config  # noqa: E402
from q8_ref import F8, U_F8  # noqa: E402
from test_hf_q8 import CFG  # noqa: E402

pytestmark = pytest.mark.gpu


def written(dev, pieces):
    """The first layer after pieces (k, v, tokens kept afterwards or None)."""
    cfg = Qwen2Config(**CFG)
    cache = hf.WindowAttention(window_from_config(cfg, 2.0, 2.0, 4096)).new_cache(cfg, 1, 96, dev, kv_dtype=F8)
    lyr = cache.layers[0]
    for k, v, keep in pieces:
        lyr.update(k.to(dev), v.to(dev))
        lyr.last_key = None  # (as the hook does)
        if keep is not None:
            lyr.crop(keep)
    return lyr


@pytest.mark.parametrize("keep", [32, 37])
def test_after_a_cut(dev, keep):
    g = torch.Generator().manual_seed(keep)

    def rows(n, scale=1.0):
        return [(torch.randn((1, 2, n, 128), generator=g) * scale).to(torch.bfloat16) for _ in range(2)]
    prompt, draft, more = rows(keep), rows(7, 40.0), rows(20)
    a = written(dev, [(*prompt, None), (*draft, keep), (*more, None)])
    b = written(dev, [(*prompt, None), (*more, None)])
    assert a.length == b.length == keep + 20
    page = keep // 16
    others = [p for p in range(a.kv.shape[0]) if p != page]
    inside = keep % 16 != 0
    same = others if inside else range(a.kv.shape[0])
    for x, y in ((a.kv.view(torch.uint8), b.kv.view(torch.uint8)), (a.exps, b.exps)):
        assert all(torch.equal(x[p], y[p]) for p in same)
    if not inside:
        return
    assert (a.exps[page] > b.exps[page]).all()
    # Both runs round a value once to a code, by at most U_F8 of it or of the smallest normal code (2^-6 of the
    # exponent's power); codes that were there when an exponent rose were rounded once more, by half the smallest step
    # (2^-10 of that power) where they became subnormal and not at all elsewhere.
    for half, x, y in zip((1, 0), dequantize(a.kv, a.exps, [page]), dequantize(b.kv, b.exps, [page])):
        unit = torch.exp2(a.exps[page, :, half].float())[None, None, :, None]
        top = torch.maximum(x.abs(), y.abs()) / (1 - U_F8)
        assert ((x - y).abs() <= 2 * U_F8 * torch.maximum(top, unit * 2.0 ** -6) + 2 * 2.0 ** -10 * unit).all()
        assert not torch.equal(x, y)
