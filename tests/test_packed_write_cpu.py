"""kv_write_packed takes the caches that the other paged entry points take."""


def test_a_cache_without_exponents_of_its_own_is_a_bf16_cache(monkeypatch):
    # as prefill, decode and plan take it
    from atflash import interface, ops
    seen = []
    monkeypatch.setattr(ops, "kv_write_packed", lambda kv, exps, *a: seen.append((kv, exps)))

    class Pool:
        kv = "pages"
    interface.kv_write_packed(Pool, None, None, None, 1, None, None)
    assert seen == [("pages", None)]
