"""What the paged cache's entry points refuse, on the CPU: the C entries answer before they launch anything, the wrappers before
they call them."""
import ctypes

import pytest
import torch

from retrievalattention_amd import kernels
from retrievalattention_amd._lib import Paged, lib

ARG, WORKSPACE = -1, -3
A = 1 << 20   # an aligned address; nothing is read from it


def _cache(**change):
    s = dict(k_pages=A, v_pages=2 * A, block_table=A, k_page_stride=4096, k_head_stride=2048, k_row_stride=128, v_page_stride=4096,
             v_head_stride=2048, v_row_stride=128, table_stride=4, pages=9, heads=2, page_rows=16, dim=128, table_pages=4, half=0)
    s.update(change)
    return ctypes.byref(Paged(**s))


BAD_CACHES = [dict(k_pages=None), dict(v_pages=A + 8), dict(block_table=None), dict(k_page_stride=4100), dict(v_row_stride=-128),
              dict(k_head_stride=4), dict(pages=0), dict(heads=0), dict(page_rows=0), dict(page_rows=24), dict(dim=96), dict(dim=256),
              dict(table_pages=0), dict(table_pages=1 << 21), dict(table_stride=-1), dict(heads=70000)]


def _attention(cache=None, **change):
    a = dict(q=A, lens=A, starts=None, scores=None, sb=128, sh=64, out=A, lse=None, B=3, gs=4, max_len=64, scale=1.0, ws=A,
             bytes=1 << 30, stream=None)
    a.update(change)
    return lib().ri_paged_attention(cache or _cache(), *a.values())


def _append(cache=None, **change):
    a = dict(key=A, value=A, kb=256, kh=128, vb=256, vh=128, lens=A, new=A + 64, scores=A, sb=128, sh=64, positions=A, pb=128, ph=64,
             token=A, B=3, budget=64, sinks=4, recent=8, stream=None)
    a.update(change)
    return lib().ri_paged_append(cache or _cache(), *a.values())


def _fill(cache=None, **change):
    a = dict(key=A, value=A, kb=25600, kt=256, kh=128, vb=25600, vt=256, vh=128, lens=A, weights=A, wb=200, wh=100, new=A + 64,
             scores=2 * A, sb=128, sh=64, positions=A, pb=128, ph=64, B=3, T=100, budget=64, sinks=4, recent=8, ws=A, bytes=1 << 20,
             stream=None)
    a.update(change)
    return lib().ri_paged_fill(cache or _cache(), *a.values())


def _weigh(**change):
    a = dict(q=A, key=A, lens=None, out=A, qb=8192, qt=1024, qh=128, kb=25600, kt=256, kh=128, B=3, W=8, T=100, heads=2, gs=4, dim=128,
             scale=1.0, ws=A, bytes=1 << 30, stream=None)
    a.update(change)
    return lib().ri_attention_weights(*a.values())


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
@pytest.mark.parametrize("call", [_attention, _append, _fill])
def test_caches(call, bad):
    assert call(_cache(**bad)) == ARG


@pytest.mark.parametrize("bad", [dict(q=None), dict(q=A + 4), dict(lens=None), dict(out=None), dict(ws=None), dict(ws=A + 4), dict(B=0),
                                 dict(B=70000), dict(gs=0), dict(gs=17), dict(max_len=0), dict(max_len=65),
                                 dict(scores=A, sh=63), dict(scores=A, sb=-1)], ids=str)
def test_attention(bad):
    assert _attention(**bad) == ARG


@pytest.mark.parametrize("heads,B,answer", [(4096, 1, ARG), (2048, 1, ARG), (2047, 1, WORKSPACE), (65535, 1, ARG), (64, 2047, WORKSPACE),
                                            (64, 2048, ARG)])
def test_attention_of_more_rows_than_are_counted(heads, B, answer):
    """Sixteen rows of a sequence's heads, or of all sequences' one head, are counted in 32 bits; a small workspace is refused behind that."""
    big = _cache(heads=heads, table_pages=1 << 20)
    assert _attention(big, B=B, max_len=1 << 24, bytes=16) == answer


@pytest.mark.parametrize("scored", [0, 1])
def test_attention_workspace(scored):
    need = lib().ri_paged_attention_workspace_bytes(3, 2, 4, 128, 64, scored)
    assert need > 0
    assert _attention(bytes=need - 1, scores=A if scored else None) == WORKSPACE
    for bad in ((0, 2, 4, 128, 64), (3, 2, 17, 128, 64), (3, 2, 4, 96, 64), (3, 2, 4, 128, 0)):
        assert lib().ri_paged_attention_workspace_bytes(*bad, scored) == 0


@pytest.mark.parametrize("bad", [dict(key=None), dict(value=A + 2), dict(kb=4), dict(vh=-8), dict(lens=None), dict(new=A), dict(new=A + 8),
                                 dict(token=A + 72), dict(B=0), dict(budget=0), dict(budget=65), dict(sinks=-1), dict(recent=-1), dict(sinks=56),
                                 dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), dict(positions=None), dict(token=None),
                                 dict(sh=63), dict(ph=63), dict(sb=-1)], ids=str)
def test_append(bad):
    assert _append(**bad) == ARG


@pytest.mark.parametrize("bad", [dict(key=None), dict(value=A + 2), dict(kt=4), dict(vb=-8), dict(weights=None), dict(T=0), dict(B=0),
                                 dict(T=2 ** 24 + 1, wh=2 ** 25), dict(wh=99), dict(budget=0), dict(budget=65), dict(sinks=57),
                                 dict(sinks=-1), dict(recent=-1), dict(sh=63), dict(ph=63), dict(ws=None), dict(pb=-1),
                                 dict(scores=A), dict(T=64, scores=A), dict(new=A),
                                 dict(new=A - 8)], ids=str)
def test_fill(bad):
    assert _fill(**bad) == ARG


def test_writes_to_pages_of_both():
    assert _append(_cache(v_pages=A)) == ARG and _fill(_cache(v_pages=A)) == ARG


def test_fill_workspace():
    need = lib().ri_paged_fill_workspace_bytes(3, 2, 100, 64)
    assert need > 0 and lib().ri_paged_fill_workspace_bytes(3, 2, 64, 64) == 0
    assert _fill(bytes=need - 1) == WORKSPACE
    assert _fill(T=64, weights=None) == ARG   # (scores are the weights)


@pytest.mark.parametrize("bad", [dict(q=None), dict(key=A + 2), dict(out=None), dict(ws=None), dict(ws=A + 4), dict(B=0), dict(W=0),
                                 dict(W=101), dict(T=2 ** 24 + 1), dict(heads=0), dict(gs=0), dict(gs=17), dict(dim=96), dict(qb=4),
                                 dict(kt=-8), dict(B=40000)], ids=str)
def test_weights(bad):
    assert _weigh(**bad) == ARG


def test_weights_workspace():
    need = lib().ri_attention_weights_workspace_bytes(3, 2, 4, 8, 100)
    assert need >= 3 * 2 * 4 * 8 * 4
    assert _weigh(bytes=need - 1) == WORKSPACE


def test_wrappers_refuse_host_tensors():
    x = torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16)
    table, lens = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 1, 8, 128, dtype=torch.bfloat16)
    row = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16)
    for call in (lambda: kernels.paged_attention(q, x, x, table, lens), lambda: kernels.paged_append(row, row, x, x, table, lens),
                 lambda: kernels.paged_fill(row, row, x, x, table), lambda: kernels.attention_weights(q, row)):
        with pytest.raises(ValueError, match="device tensor"):
            call()
