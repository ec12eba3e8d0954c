"""How the paged cache hands out pages: host logic, on the CPU."""
import pytest
import torch

from retrievalattention_amd.cache_hub import paged_cache


def _cache(**change):
    a = dict(layer_num=1, batch_size=3, max_length=64, num_key_value_heads=1, num_heads=2, head_dim=64, dtype=torch.bfloat16,
             device="cpu", page_size=16)
    a.update(change)
    return paged_cache(**a)


@pytest.fixture(autouse=True)
def no_launches(monkeypatch):
    from retrievalattention_amd import kernels
    monkeypatch.setattr(kernels, "paged_fill", lambda *a, **k: None)
    monkeypatch.setattr(kernels, "attention_weights", lambda *a, **k: None)


def _prompt(cache, b, T):
    x = torch.zeros(1, T, 1, 64, dtype=torch.bfloat16)
    cache.prefill_update_kv_cache(x, x, x, 0, b)


def _owned(cache):
    pages = [p for row in cache._table for p in row]
    assert len(set(pages)) == len(pages) and not set(pages) & set(cache._free)
    assert len(pages) + cache.free_pages == cache.k_pages[0].shape[0]
    for b, row in enumerate(cache._table):
        assert cache.block_table[b].tolist() == row + [-1] * (cache.block_table.shape[1] - len(row))
    return [len(row) for row in cache._table]


def test_refused_prompts_take_nothing():
    c = _cache()
    _prompt(c, 1, 5)
    for b, T in ((-1, 5), (3, 5), (0, 0)):
        with pytest.raises(ValueError, match="expected a prompt"):
            _prompt(c, b, T)
    assert _owned(c) == [0, 1, 0]


def test_pages_follow_the_rows():
    c = _cache()
    _prompt(c, 0, 16)
    _prompt(c, 2, 33)
    assert _owned(c) == [1, 0, 3] and c.context == 33 and c.active.tolist() == [1, 0, 1] and c.seen.tolist() == [16, 0, 33]
    c.prepare_token()                       # row 17 of the first sequence; the second place is none
    assert _owned(c) == [2, 0, 3]
    for _ in range(15):
        c.prepare_token()
    assert _owned(c) == [2, 0, 4 if c._rows[2] > 48 else 3]
    c.release(0)
    assert _owned(c)[0] == 0 and c.active.tolist() == [0, 0, 1]
    _prompt(c, 2, 5)                        # a new prompt ends the place's last sequence
    assert _owned(c) == [0, 0, 1]


def test_a_budget_bounds_the_pages():
    c = _cache(budget=24, sinks=2, recent=4)
    _prompt(c, 1, 60)
    assert _owned(c) == [0, 2, 0] and c.seen.tolist() == [0, 60, 0]
    for _ in range(100):
        c.prepare_token()
    assert _owned(c) == [0, 2, 0] and c.context == 24


def test_refusals():
    c = _cache(pages=4)
    with pytest.raises(ValueError, match="built for 64"):
        _prompt(c, 0, 65)
    _prompt(c, 0, 33)
    with pytest.raises(RuntimeError, match="2 pages wanted, 1 free"):
        _prompt(c, 1, 17)
    assert _owned(c) == [3, 0, 0]
    _prompt(c, 1, 16)
    c.prepare_token.__self__._rows[0] = 48
    with pytest.raises(RuntimeError, match="2 pages wanted, 0 free"):
        c.prepare_token()
    assert _owned(c) == [3, 1, 0] and c._rows == [48, 16, 0]
    c.release(1)
    for _ in range(16):
        c.prepare_token()
    with pytest.raises(RuntimeError, match="64 rows"):
        c.prepare_token()
    for bad in (dict(page_size=12), dict(head_dim=96), dict(num_heads=40), dict(dtype=torch.float32), dict(budget=10, sinks=4, recent=6),
                dict(budget=10, sinks=0, recent=0), dict(window=0)):
        with pytest.raises(ValueError):
            _cache(**bad)


def _state(c):
    return ([list(row) for row in c._table], list(c._rows), sorted(c._free), c.block_table.tolist(), c.seqlens.tolist(), c.seen.tolist(),
            c.active.tolist())


@pytest.mark.parametrize("budget", [None, 24])
def test_refused_tensors_change_nothing(budget, monkeypatch):
    """A prompt or a token of other shapes, types or layouts than the pages' is refused before a sequence ends or pages are taken."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    c = _cache(**({} if budget is None else dict(budget=budget, sinks=2, recent=4)))
    _prompt(c, 0, 16)
    _prompt(c, 2, 20)
    before = _state(c)
    key, token = torch.zeros(1, 30, 1, 64, dtype=torch.bfloat16), torch.zeros(3, 1, 1, 64, dtype=torch.bfloat16)
    query = torch.zeros(1, 30, 2, 64, dtype=torch.bfloat16)
    bad = [key.half(), key.float(), key[..., :32], torch.zeros(1, 30, 2, 64, dtype=torch.bfloat16), key[0], None, "key",
           torch.zeros(1, 30, 1, 128, dtype=torch.bfloat16)[..., ::2]]
    for x in bad:
        for k, v in ((x, key), (key, x)):
            with pytest.raises((ValueError, TypeError)):
                c.prefill_update_kv_cache(query, k, v, 0, 0)
            assert _state(c) == before
    with pytest.raises((ValueError, TypeError)):
        c.prefill_update_kv_cache(query, key, key[:, :29], 0, 0)
    if budget is not None:
        for x in (None, query.half(), query[:, :29], query[0], query[0, 0], torch.zeros(1, 30, 17, 64, dtype=torch.bfloat16)):
            with pytest.raises((ValueError, TypeError)):
                c.prefill_update_kv_cache(x, key, key, 0, 0)
    assert _state(c) == before
    for x in (token.half(), token[:2], token[..., :32], token[:, 0], None, torch.zeros(3, 2, 1, 64, dtype=torch.bfloat16)):
        for k, v in ((x, token), (token, x)):
            with pytest.raises((ValueError, TypeError)):
                c.decode_update_kv_cache(k, v, 0)
            assert _state(c) == before
    c.prefill_update_kv_cache(query, key, key, 0, 0)
    assert c._rows[0] == (30 if budget is None else 24)
