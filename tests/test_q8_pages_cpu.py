"""The expansion of an 8-bit cache into blocks by page: the checks of its C entry."""
import pytest

from test_q8_cpu import EXPAND, call, no_gpu  # noqa: F401

PAGES = {k: v for k, v in EXPAND.items() if k != "out_table"}


@pytest.mark.parametrize("change,code", [
    (dict(batch=-1), 1), (dict(n_pages=-1), 1), (dict(out=None), 1), (dict(kv=None), 1), (dict(exps=None), 1),
    (dict(table=None), 1), (dict(pages=0), 1), (dict(hkv=0), 1), (dict(n_pages=5), 1), (dict(out=8), 1), (dict(kv=8), 1),
    (dict(batch=70000), 2), (dict(hkv=70000), 2), (dict(n_pages=0, out=None), 0), (dict(batch=0, kv=None), 0)])
def test_expand_by_page_validation(no_gpu, change, code):  # noqa: F811
    assert call(no_gpu.atf_kv_expand_q8_pages, PAGES, **change) == code
