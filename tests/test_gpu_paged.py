"""The paged cache's operators against their definition in 64 bits (oracle/paged.py), at the sizes and masks where they can go
wrong.  Tolerances count roundings: u = eps / 2 of the element type is a rounding's largest relative error, 2^-24 that of fp32."""
import math

import pytest
import torch

from oracle import paged as oracle
from retrievalattention_amd import kernels

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
F = 2.0 ** -24


def _u(dt):
    return torch.finfo(dt).eps / 2


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen)


def _pool(gen, dt, B, heads, dim, page, rows, junk=True):
    """Pages of B sequences, scattered, with NaN and infinities in the rows behind each sequence's `rows` and in a spare page."""
    per = -(-rows // page)
    pool = B * per + 2
    table = torch.randperm(pool - 1, generator=gen)[:B * per].view(B, per).to(torch.int32)
    k, v = _randn(gen, pool, heads, page, dim).to(dt), _randn(gen, pool, heads, page, dim).to(dt)
    if junk:
        k[pool - 1], v[pool - 1] = math.nan, math.inf
    return k, v, table


def _spoil(k, v, table, lens, starts=None):
    """Rows that are not attended hold NaN and infinities."""
    page = k.shape[2]
    for b in range(table.shape[0]):
        for r in range(table.shape[1] * page):
            if r >= int(lens[b]) or (starts is not None and r < int(starts[b])):
                p = int(table[b, r // page])
                if 0 <= p < k.shape[0]:
                    k[p, :, r % page] = math.nan if r % 2 else math.inf
                    v[p, :, r % page] = -math.inf if r % 3 else math.nan


def _check_attention(q, k, v, table, lens, starts, out, lse, scale, before=None, after=None):
    want, want_lse, p, absolute, size = oracle.attention(q, k, v, table, lens, starts, scale)
    dt, dim = q.dtype, q.shape[-1]
    n = table.shape[1] * k.shape[2]
    # a score is a sum of dim products in fp32, scaled (two roundings more); its exponential is off by that and by two units
    ds = (dim + 4) * F * size + 8 * F * (1 + size)
    # out: each probability rounded to the element type, the sums in fp32, the result rounded; a half below 2^-14 is off by 2^-25
    tol = _u(dt) * (absolute + want.abs()) + (2 * ds[:, None, :, None] + (64 + n / 16) * F) * absolute
    if dt == HF:
        tol = tol + 2.0 ** -25 * (n * 8 + 1)
    assert bool(((out.cpu().double() - want).abs() <= tol).all()), float(((out.cpu().double() - want).abs() - tol).max())
    finite = torch.isfinite(want_lse)
    got = lse.cpu().double()
    assert bool((got[~finite] == -math.inf).all())
    assert bool(((got - want_lse).abs() <= ds + (64 + n / 16) * F + 4 * F * want_lse.abs())[finite].all())
    if before is not None:
        heads = k.shape[1]
        w = p.view(p.shape[0], heads, -1, p.shape[-1])[..., :before.shape[-1]].sum(2)
        rel = (2 * ds.view(ds.shape[0], heads, -1).max(-1).values + (64 + n / 16) * F)[..., None]
        want_scores = before.double() + w
        # (a weight is exp(s - lse) with s and the maximum up to `size` in size, and the sum of up to 16 of them and the score)
        assert bool(((after.cpu().double() - want_scores).abs() <= rel * w + 18 * F * want_scores.abs()).all())
        assert torch.equal(after.cpu()[w == 0], before[w == 0])


CASES = [
    # dt, B, heads, gs, dim, page, lens, starts
    (BF, 1, 1, 1, 128, 16, [1], None),
    (BF, 1, 2, 4, 128, 16, [17], None),
    (HF, 3, 2, 7, 128, 16, [0, 1, 331], None),
    (BF, 2, 1, 16, 128, 64, [640, 63], None),
    (HF, 2, 3, 8, 64, 32, [100, 257], None),
    (BF, 4, 2, 3, 64, 8, [9, 8, 7, 200], None),
    (BF, 2, 2, 4, 128, 1, [5, 40], None),
    (HF, 2, 1, 5, 128, 4, [50, 3], [13, 3]),
    (BF, 4, 2, 4, 128, 16, [300, 300, 40, 16], [0, 290, 40, 15]),
    (BF, 2, 1, 9, 64, 256, [1500, 700], [700, 0]),
    (BF, 1, 2, 4, 128, 16, [5003], None),
    (HF, 2, 1, 12, 128, 2, [1111, 0], [1, 0]),
    # rows shared over workgroups: empty sequences first, between and last, parts of several groups in one share
    (BF, 7, 3, 4, 128, 16, [0, 3001, 0, 0, 17, 600, 0], [0, 5, 0, 0, 17, 590, 0]),
    (HF, 5, 2, 1, 64, 8, [1, 1025, 2049, 513, 0], None),
    (BF, 1, 1, 2, 64, 32, [0], None),
    (BF, 70, 1, 4, 64, 16, [(37 * i) % 640 for i in range(70)], [(37 * i) % 640 // 2 for i in range(70)]),
    # many groups: one workgroup to each
    (HF, 170, 1, 4, 64, 16, [(37 * i) % 1000 for i in range(170)], None),
]


@pytest.mark.parametrize("dt,B,heads,gs,dim,page,lens,starts", CASES)
@pytest.mark.parametrize("scored", [False, True])
def test_attention(dev, dt, B, heads, gs, dim, page, lens, starts, scored):
    gen = torch.Generator().manual_seed(B * 1000 + dim + page + lens[0])
    rows = max(lens) + 3 if B < 7 else max(max(lens), 600) + 3
    k, v, table = _pool(gen, dt, B, heads, dim, page, rows)
    lens, starts = torch.tensor(lens, dtype=torch.int32), None if starts is None else torch.tensor(starts, dtype=torch.int32)
    _spoil(k, v, table, lens, starts)
    q = (2 * _randn(gen, B, 1, heads * gs, dim)).to(dt)
    before = torch.rand(B, heads, table.shape[1] * page, generator=gen) if scored else None
    on = lambda t: None if t is None else t.to(dev)  # noqa: E731
    scores = on(before)
    out, lse = kernels.paged_attention(on(q), on(k), on(v), on(table), on(lens), starts=on(starts), scores=scores,
                                       return_softmax_lse=True)
    _check_attention(q, k, v, table, lens, starts, out, lse, dim ** -0.5, before, scores)
    again = kernels.paged_attention(on(q), on(k), on(v), on(table), on(lens), starts=on(starts))
    assert torch.equal(again, out)   # no order of arrival in the result


@pytest.mark.parametrize("lens", [[5, 16], [200, 331], [3, 5000]])
@pytest.mark.parametrize("what", ["query", "keys"])
def test_attention_passes_nan_on(dev, lens, what):
    """A NaN in what is attended is in the result, also where a part's scores are nothing else; other heads are as without it."""
    gen = torch.Generator().manual_seed(lens[1])
    B, heads, gs, dim = 2, 2, 3, 128
    k, v, table = _pool(gen, BF, B, heads, dim, 16, lens[1])
    q = (2 * _randn(gen, B, 1, heads * gs, dim)).to(BF)
    on = lambda t: t.to(dev)  # noqa: E731
    lens = torch.tensor(lens, dtype=torch.int32)
    room = table.shape[1] * 16
    scores, was = torch.zeros(B, heads, room, device=dev), torch.zeros(B, heads, room, device=dev)
    want, want_lse = kernels.paged_attention(on(q), on(k), on(v), on(table), on(lens), scores=was, return_softmax_lse=True)
    bad = torch.zeros(B, heads, gs, dtype=torch.bool)
    if what == "query":
        bad[0, 1, 2] = bad[1, 0, 0] = True
        q[0, 0, gs + 2, 7], q[1, 0, 0, 127] = math.nan, math.nan
    else:
        bad[1, 1] = True
        k[table[1].long(), 1] = math.nan
    out, lse = kernels.paged_attention(on(q), on(k), on(v), on(table), on(lens), scores=scores, return_softmax_lse=True)
    bad = bad.view(B, heads * gs)
    assert bool(out.cpu()[:, 0][bad].isnan().all()) and torch.equal(out.cpu()[:, 0][~bad], want.cpu()[:, 0][~bad])
    assert bool(lse.cpu()[bad].isnan().all()) and torch.equal(lse.cpu()[~bad], want_lse.cpu()[~bad])
    attended = torch.arange(room)[None, None] < lens[:, None, None]
    spoilt = bad.view(B, heads, gs).any(-1)[:, :, None] & attended
    assert bool(scores.cpu()[spoilt].isnan().all()) and torch.equal(scores.cpu()[~spoilt], was.cpu()[~spoilt])


def test_attention_max_len_scale_and_strides(dev):
    """Pages as [pages, rows, heads, dim], keys and values in one tensor, a table that is a part of a larger one, rows past max_len
    and pages that are not there left out, a scale of its own."""
    gen = torch.Generator().manual_seed(5)
    B, heads, gs, dim, page, per = 3, 2, 6, 128, 16, 5
    both = _randn(gen, B * per, 2, page, heads, dim).to(BF).to(dev)
    k, v = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    big = torch.randperm(B * per, generator=gen).view(B, per).to(torch.int32)
    wide = torch.full((B, per + 3), -7, dtype=torch.int32)
    wide[:, 1:per + 1] = big
    wide[1, 2], wide[2, 1] = -1, B * per    # no such pages: rows 16 .. 31 of the second sequence, 0 .. 15 of the third
    table = wide.to(dev)[:, 1:per + 1]
    lens = torch.tensor([80, 33, 10], dtype=torch.int32)
    q = _randn(gen, B, 1, heads * gs, dim).to(BF)
    out, lse = kernels.paged_attention(q.to(dev), k, v, table, lens.to(dev), scale=0.2, max_len=77, return_softmax_lse=True)
    _check_attention(q, k.cpu(), v.cpu(), table.cpu(), lens.clamp(max=77), None, out, lse, 0.2)
    assert bool((out[2] == 0).all()) and bool((lse[2] == -math.inf).all())


@pytest.mark.parametrize("B,room", [(600, 1024), (1300, 640)])
def test_attention_of_many_sequences(dev, B, room):
    """More sequences than a workgroup looks at at a time; most of them empty or short."""
    gen = torch.Generator().manual_seed(B)
    lens = torch.where(torch.rand(B, generator=gen) < 0.5, 0, (torch.rand(B, generator=gen) ** 6 * room).int()).to(torch.int32)
    lens[-1], lens[B // 2] = room, 513
    per, page = room // 64, 64
    k, v = _randn(gen, 40, 2, page, 64).to(BF), _randn(gen, 40, 2, page, 64).to(BF)
    table = torch.randint(40, (B, per), generator=gen).to(torch.int32)   # pages that sequences share
    q = _randn(gen, B, 1, 4, 64).to(BF)
    before = torch.rand(B, 2, room, generator=gen)
    scores = before.to(dev)
    out, lse = kernels.paged_attention(*(t.to(dev) for t in (q, k, v, table, lens)), scores=scores, return_softmax_lse=True)
    _check_attention(q, k, v, table, lens, None, out, lse, 0.125, before, scores)


def test_attention_of_extreme_scores(dev):
    """Scores far apart and all alike, keys with infinite elements, a sum that overflows without the running maximum."""
    gen = torch.Generator().manual_seed(6)
    k, v, table = _pool(gen, BF, 2, 1, 64, 16, 300, junk=False)
    lens = torch.tensor([300, 290], dtype=torch.int32)
    q = 60 * _randn(gen, 2, 1, 2, 64).to(BF)
    out, lse = kernels.paged_attention(*(t.to(dev) for t in (q, k, v, table, lens)), return_softmax_lse=True)
    _check_attention(q, k, v, table, lens, None, out, lse, 0.125)
    same = kernels.paged_attention(*(t.to(dev) for t in (q * 0, k, v, table, lens)))
    rows = oracle.rows_of(v, table[0], torch.arange(300))[0][0]
    assert torch.allclose(same[0, 0, 0].cpu().double(), rows.mean(0), atol=2 * _u(BF) * float(rows.abs().mean(0).max()))
    # a key of -inf where the query is positive: no weight
    q = q.abs()
    k[int(table[0, 2]), 0, 3] = -math.inf
    out = kernels.paged_attention(*(t.to(dev) for t in (q, k, v, table, lens)))
    assert bool(torch.isfinite(out).all())


def test_attention_on_a_long_cache_past_32_bits(dev):
    """Pages whose offsets pass 2^31 elements: only the last ones are looked at."""
    heads, dim, page, pages = 2, 128, 256, 33000
    k = torch.empty((pages, heads, page, dim), dtype=BF, device=dev)     # 4.3 GB, 2^31 elements and more
    v = torch.empty_like(k)
    gen = torch.Generator().manual_seed(7)
    at = torch.tensor([[pages - 1, pages - 2, 32769]], dtype=torch.int32)
    small_k, small_v = _randn(gen, 3, heads, page, dim).to(BF), _randn(gen, 3, heads, page, dim).to(BF)
    k[at[0].long().to(dev)], v[at[0].long().to(dev)] = small_k.to(dev), small_v.to(dev)
    q = _randn(gen, 1, 1, heads * 4, dim).to(BF)
    lens = torch.tensor([700], dtype=torch.int32)
    out, lse = kernels.paged_attention(q.to(dev), k, v, at.to(dev), lens.to(dev), return_softmax_lse=True)
    _check_attention(q, small_k, small_v, torch.tensor([[0, 1, 2]]), lens, None, out, lse, dim ** -0.5)
    key = _randn(gen, 1, 1, heads, dim).to(BF).to(dev)
    kernels.paged_append(key, key, k, v, at.to(dev), lens.to(dev))
    assert torch.equal(k[32769, :, 700 - 512], key[0, 0])


def _grid_scores(gen, dt, B, heads, gs, dim, page, rows, values):
    """Queries of 1 in the first dimension and keys whose first element, of `values`, is the score: exact in either type."""
    k, v, table = _pool(gen, dt, B, heads, dim, page, rows, junk=False)
    k[..., 0] = values[torch.randint(len(values), k.shape[:3], generator=gen)].to(dt)
    q = torch.zeros(B, 1, heads * gs, dim, dtype=dt)
    q[..., 0] = 1
    return q, k, v, table


@pytest.mark.parametrize("dt,B,heads,gs,dim,page,lens", [
    (BF, 2, 2, 4, 128, 16, [331, 64]),
    (HF, 2, 2, 7, 128, 32, [300, 17]),
    (BF, 1, 3, 16, 64, 8, [200]),
    (HF, 1, 1, 3, 64, 4, [513]),
    (BF, 2, 2, 4, 128, 16, [3001, 700]),
])
def test_attention_rounds_the_output_only(dev, dt, B, heads, gs, dim, page, lens):
    """Values of 1 and -1 that nearly cancel: the weights' own error shows, not that of the result's last rounding."""
    gen = torch.Generator().manual_seed(lens[0])
    values = torch.arange(-64, 65) / 16        # scores of -4 .. 4
    q, k, v, table = _grid_scores(gen, dt, B, heads, gs, dim, page, max(lens), values)
    v = torch.where(torch.rand(v.shape, generator=gen) < 0.5, 1.0, -1.0).to(dt)
    lens = torch.tensor(lens, dtype=torch.int32)
    out = kernels.paged_attention(*(t.to(dev) for t in (q, k, v, table, lens)), scale=1.0)
    want, _, _, absolute, size = oracle.attention(q, k, v, table, lens, None, 1.0)
    # a weight's parts add up to it within 2^-16 (2^-21 in half); its score is rounded twice and its exponential twice, the sums in fp32
    tol = _u(dt) * want.abs() + 2.0 ** (-16 if dt == BF else -21) * absolute + \
        (8 * F * (1 + size[:, None, :, None]) + (64 + int(lens.max()) / 16) * F) * absolute
    assert bool(((out.cpu().double() - want).abs() <= tol).all()), float(((out.cpu().double() - want).abs() / tol).max())


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("low", [9, 14, 18, 20])
@pytest.mark.parametrize("n", [400, 5000])
def test_attention_of_rows_that_weigh_little(dev, dt, low, n):
    """One row takes nearly all the weight and has nothing to say; the result is the many others', of e^-low each."""
    gen = torch.Generator().manual_seed(n + low)
    heads, gs, dim, page = 2, 4, 64, 16
    q, k, v, table = _grid_scores(gen, dt, 1, heads, gs, dim, page, n, torch.tensor([-float(low)]))
    v = v.abs() + 1
    k[int(table[0, 3]), :, 5, 0] = 0.0
    v[int(table[0, 3]), :, 5] = 0.0
    lens = torch.tensor([n], dtype=torch.int32)
    out = kernels.paged_attention(*(t.to(dev) for t in (q, k, v, table, lens)), scale=1.0)
    want, _, _, absolute, size = oracle.attention(q, k, v, table, lens, None, 1.0)
    # as above; half: a part below its normal numbers is off by 2^-25 of 2^15 times a weight, and so is a result
    tol = _u(dt) * want.abs() + 2.0 ** (-16 if dt == BF else -21) * absolute + (8 * F * (1 + low) + (64 + n / 16) * F) * absolute
    if dt == HF:
        tol = tol + n * 2.0 ** -40 * float(v.max()) + 2.0 ** -25
    assert bool(((out.cpu().double() - want).abs() <= tol).all()), float(((out.cpu().double() - want).abs() / tol).max())


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "f16"])
def test_attention_of_infinite_values(dev, dt):
    """A value of infinity that has weight is in the result, with the weight of the highest score as with others'."""
    gen = torch.Generator().manual_seed(14)
    heads, gs, dim, n = 1, 3, 64, 40
    q, k, v, table = _grid_scores(gen, dt, 1, heads, gs, dim, 16, n, torch.tensor([-7.0, -3.5, -0.25]))
    k[int(table[0, 1]), 0, 2, 0] = 0.0
    v[int(table[0, 1]), 0, 2, 5] = math.inf
    v[int(table[0, 2]), 0, 3, 9] = -math.inf
    lens = torch.tensor([n], dtype=torch.int32)
    out = kernels.paged_attention(*(t.to(dev) for t in (q, k, v, table, lens)), scale=1.0)
    assert bool((out[..., 5] == math.inf).all()) and bool((out[..., 9] == -math.inf).all())
    assert int(torch.isfinite(out).sum()) == heads * gs * (dim - 2)


@pytest.mark.parametrize("n", [40, 700, 5000])
def test_attention_of_scores_of_minus_infinity(dev, n):
    """A head all of whose scores are -inf attends nothing; one of which some are attends the others."""
    gen = torch.Generator().manual_seed(n)
    heads, gs, dim = 2, 3, 64
    q, k, v, table = _grid_scores(gen, BF, 1, heads, gs, dim, 16, n, torch.arange(-32, 33) / 16)
    rows = torch.arange(n)
    p = table[0].long()[rows // 16]
    k[p, 0, rows % 16, 0] = -math.inf
    some = rows[torch.rand(n, generator=gen) < 0.5]
    k[table[0].long()[some // 16], 1, some % 16, 0] = -math.inf
    lens = torch.tensor([n], dtype=torch.int32)
    before = torch.rand(1, heads, table.shape[1] * 16, generator=gen)
    scores = before.to(dev)
    out, lse = kernels.paged_attention(*(t.to(dev) for t in (q, k, v, table, lens)), scale=1.0, scores=scores, return_softmax_lse=True)
    assert bool((out[0, 0, :gs] == 0).all()) and bool((lse[0, :gs] == -math.inf).all()) and torch.equal(scores[0, 0].cpu(), before[0, 0])
    x = k[p, 1, rows % 16, 0].double()
    w = torch.softmax(x, 0)
    want = w @ v[p, 1, rows % 16].double()
    tol = _u(BF) * want.abs() + (2.0 ** -16 + (24 + 64 + n / 16) * F) * (w @ v[p, 1, rows % 16].double().abs())   # (scores of up to 2)
    assert bool(((out[0, 0, gs:].cpu().double() - want).abs() <= tol).all())
    got = scores[0, 1, :n].cpu().double()
    assert bool(((got - before[0, 1, :n].double() - gs * w).abs() <= (24 + 64 + n / 16) * F * gs * w + 18 * F * got).all())
    assert torch.equal(got.float()[w == 0], before[0, 1, :n][w == 0])


@pytest.mark.parametrize("page,n", [(16, 300), (8, 700), (64, 3000)])
@pytest.mark.parametrize("bad", [math.nan, math.inf], ids=["nan", "inf"])
def test_attention_leaves_scores_of_rows_that_are_not_there(dev, page, n, bad):
    """Also where a NaN makes the others' scores NaN, and with another head's weights as they are."""
    gen = torch.Generator().manual_seed(n)
    heads, gs, dim = 2, 3, 64
    k, v, table = _pool(gen, BF, 1, heads, dim, page, n)
    table[0, 1], table[0, n // page // 2] = -1, k.shape[0]
    q = (2 * _randn(gen, 1, 1, heads * gs, dim)).to(BF)
    lens = torch.tensor([n], dtype=torch.int32)
    before = torch.rand(1, heads, table.shape[1] * page, generator=gen)
    on = lambda t: t.to(dev)  # noqa: E731
    clean, spoilt = on(before), on(before)
    kernels.paged_attention(on(q), on(k), on(v), on(table), on(lens), scores=clean)
    q[0, 0, 1, 3] = bad
    kernels.paged_attention(on(q), on(k), on(v), on(table), on(lens), scores=spoilt)
    rows = torch.arange(before.shape[2])
    there = (rows < n) & (table[0].long()[rows // page] >= 0) & (table[0].long()[rows // page] < k.shape[0])
    for got in (clean.cpu(), spoilt.cpu()):
        assert torch.equal(got[:, :, ~there], before[:, :, ~there])
    assert bool(spoilt[0, 0].cpu()[there].isnan().all()) and torch.equal(spoilt[0, 1], clean[0, 1])


# ------------------------------------------------------------------------------------------------ append
def _append_state(gen, dt, B, heads, dim, page, budget, lens, seen, sinks, recent, ties):
    k, v, table = _pool(gen, dt, B, heads, dim, page, budget, junk=False)
    scores = torch.rand(B, heads, budget, generator=gen)
    if ties:
        scores = (scores * 4).floor() - 1      # -1, 0, 1, 2: rows share their score
        scores[scores == 0] = -0.0
    positions = torch.stack([torch.randperm(max(seen), generator=gen)[:budget].sort().values[torch.randperm(budget, generator=gen)]
                             for _ in range(B * heads)]).view(B, heads, budget).to(torch.int32)
    return k, v, table, scores, positions, torch.tensor(lens, dtype=torch.int32), torch.tensor(seen, dtype=torch.int32)


@pytest.mark.parametrize("dt,B,heads,dim,page,budget,lens,seen,sinks,recent,ties", [
    (BF, 1, 1, 128, 16, 1, [0], [0], 0, 0, False),
    (BF, 1, 1, 128, 16, 1, [1], [9], 0, 0, False),
    (HF, 3, 2, 64, 8, 37, [37, 36, 0], [90, 40, 0], 4, 5, False),
    (BF, 2, 3, 128, 32, 700, [700, 700], [3000 - 100, 800], 4, 64, True),
    (BF, 2, 2, 128, 64, 4111, [4111, 5000], [9000, 7000], 0, 0, True),
    (HF, 1, 8, 64, 1, 64, [64], [64], 20, 43, False),
    (BF, 1, 2, 64, 256, 20000, [20000], [30000], 4, 512, False),
])
def test_append(dev, dt, B, heads, dim, page, budget, lens, seen, sinks, recent, ties):
    gen = torch.Generator().manual_seed(budget + page)
    k, v, table, scores, positions, lens, seen = _append_state(gen, dt, B, heads, dim, page, budget, lens,
                                                               [max(x, budget) for x in seen], sinks, recent, ties)
    key = _randn(gen, B, 1, heads, dim + 8).to(dt)[..., :dim]    # strided rows
    value = _randn(gen, B, heads, 1, dim).to(dt).transpose(1, 2)
    d = [t.to(dev) for t in (k, v, table, lens, scores, positions, seen)]
    held = torch.full((B,), -5, dtype=torch.int32, device=dev)
    wide = torch.empty(B, 1, heads, dim + 8, dtype=dt, device=dev)[..., :dim].copy_(key)
    kernels.paged_append(wide, value.to(dev), d[0], d[1], d[2], d[3], held, scores=d[4], positions=d[5], token_positions=d[6],
                         budget=budget, sinks=sinks, recent=recent)
    for b in range(B):
        n = min(int(lens[b]), budget)
        for h in range(heads):
            r = n if n < budget else oracle.victim(scores[b, h], positions[b, h], n, int(seen[b]), sinks, recent)
            p = int(table[b, r // page])
            k[p, h, r % page], v[p, h, r % page] = key[b, 0, h], value[b, 0, h]
            scores[b, h, r], positions[b, h, r] = 0.0, seen[b]
        assert int(held[b]) == min(n + 1, budget)
    for got, want in zip((d[0], d[1], d[4], d[5]), (k, v, scores, positions)):
        assert torch.equal(got.cpu(), want)


def test_append_without_scores_and_with_odd_ones(dev):
    """Plain appends leave a full sequence as it is; NaN counts as the highest score, -inf as the lowest; where every row stays, the
    first one goes; a page that is not there takes nothing."""
    gen = torch.Generator().manual_seed(8)
    k, v, table, scores, positions, lens, seen = _append_state(gen, BF, 4, 1, 64, 16, 32, [31, 32, 7, 16], [40, 40, 40, 40], 0, 0, False)
    table[3, 1] = -1
    key = _randn(gen, 4, 1, 1, 64).to(BF)
    d = [t.to(dev) for t in (key, key, k, v, table, lens)]
    held = torch.zeros(4, dtype=torch.int32, device=dev)
    kernels.paged_append(*d, held)
    for b, r in ((0, 31), (2, 7)):
        k[int(table[b, r // 16]), :, r % 16] = key[b, 0]
    assert torch.equal(d[2].cpu(), k) and held.tolist() == [32, 32, 8, 17]
    lens = torch.full((4,), 32, dtype=torch.int32)
    scores[0, 0, :] = math.nan
    scores[0, 0, 9] = math.inf
    scores[1, 0, 21] = -math.inf
    positions[2] = 1
    full = [t.to(dev) for t in (key, key, k, v, table, lens)]
    s, p = scores.to(dev), positions.to(dev)
    kernels.paged_append(*full, scores=s, positions=p, token_positions=seen.to(dev), sinks=2, recent=3, budget=32)
    for b in range(3):
        r = oracle.victim(scores[b, 0], positions[b, 0], 32, 40, 2, 3)
        assert int(p[b, 0, r]) == 40 and float(s[b, 0, r]) == 0.0 and int((p[b, 0].cpu() != positions[b, 0]).sum()) <= 1
    assert oracle.victim(scores[2, 0], positions[2, 0], 32, 40, 2, 3) == 0


# ------------------------------------------------------------------------------------------------ fill
@pytest.mark.parametrize("dt,B,T,heads,dim,page,budget,lens,sinks,recent,weights", [
    (BF, 1, 1, 1, 128, 16, None, None, 0, 0, None),
    (HF, 2, 37, 3, 64, 8, None, [37, 0], 0, 0, None),
    (BF, 3, 300, 2, 128, 16, 64, [300, 64, 65], 4, 16, "any"),
    (BF, 2, 2500, 2, 64, 32, 1000, None, 0, 0, "few"),
    (HF, 1, 5000, 1, 128, 64, 4999, None, 4, 4000, "few"),
    (BF, 1, 1100, 2, 128, 4, 16, [1100], 8, 8, "any"),
    (BF, 2, 1030, 1, 128, 16, 100, [1030, 99], 1, 0, "zero"),
    (BF, 1, 4097, 2, 64, 256, 1, None, 0, 0, "odd"),
    (BF, 1, 70000, 2, 64, 256, 9000, None, 4, 64, "any"),
    (HF, 4, 9001, 2, 64, 64, 700, [9001, 4096, 4097, 100], 4, 64, "any"),
    (BF, 2, 8200, 1, 64, 32, 8100, None, 0, 4100, "zero"),
    (BF, 1, 12289, 2, 64, 32, 5000, [12288], 0, 0, "few"),
    (HF, 1, 16384, 1, 64, 128, 4097, None, 17, 0, "odd"),
    (HF, 4, 17001, 2, 64, 64, 700, [17001, 4096, 16385, 100], 4, 64, "any"),
    (BF, 2, 20500, 1, 64, 32, 20400, [20500, 20401], 0, 4100, "zero"),
    (BF, 1, 24577, 1, 64, 32, 5000, [24576], 0, 0, "few"),
    (HF, 1, 16400, 1, 64, 128, 4097, None, 17, 0, "odd"),
    (BF, 26, 16385, 4, 64, 8, 21, [16385 - 631 * b for b in range(26)], 3, 2, "any"),    # more chunks than run at a time
    (BF, 26, 16385, 4, 64, 8, 21, None, 0, 0, "few"),
])
def test_fill(dev, dt, B, T, heads, dim, page, budget, lens, sinks, recent, weights):
    gen = torch.Generator().manual_seed(T + page)
    room = budget or T
    k, v, table = _pool(gen, dt, B, heads, dim, page, room, junk=False)
    key, value = _randn(gen, B, T, heads, dim).to(dt), _randn(gen, B, T, heads, 2, dim).to(dt)[:, :, :, 1]
    lens_t = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    w = None
    if weights:
        w = torch.exp(4 * _randn(gen, B, heads, T)) if weights in ("any", "odd") else torch.zeros(B, heads, T)
        if weights == "few":
            w = (torch.rand(B, heads, T, generator=gen) * 5).floor()
        if weights == "odd":
            w[..., ::7], w[..., 5], w[..., 4000] = -1.0, math.inf, math.nan
    scores = torch.full((B, heads, room), 3.0) if w is not None else None
    positions = torch.full((B, heads, room), -9, dtype=torch.int32)
    on = lambda t: None if t is None else t.to(dev)  # noqa: E731
    d = [on(t) for t in (k, v, table, scores, positions)]
    held = torch.full((B,), -5, dtype=torch.int32, device=dev)
    wide = torch.empty(B, T, heads, 2, dim, dtype=dt, device=dev)
    wide[:, :, :, 1] = value.to(dev)
    kernels.paged_fill(key.to(dev), wide[:, :, :, 1], d[0], d[1], d[2], held, seqlens=on(lens_t), weights=on(w), scores=d[3],
                       positions=d[4], budget=budget, sinks=sinks, recent=recent)
    for b in range(B):
        n = T if lens is None else lens[b]
        for h in range(heads):
            rows = torch.tensor(oracle.kept(None if w is None else w[b, h].tolist(), n, room, sinks, recent), dtype=torch.long)
            r = torch.arange(rows.numel())
            at = table[b].long()[r // page]
            k[at, h, r % page], v[at, h, r % page] = key[b, rows, h], value[b, rows, h]
            positions[b, h, r] = rows.to(torch.int32)
            if scores is not None:
                scores[b, h, r] = w[b, h, rows]
        assert int(held[b]) == min(n, room)
    for got, want in zip((d[0], d[1], d[4]), (k, v, positions)):
        assert torch.equal(got.cpu(), want)
    if scores is not None:
        assert torch.equal(d[3].cpu().nan_to_num(-77), scores.nan_to_num(-77))


def test_fill_of_a_prompt_of_many_chunks(dev):
    """More than 1024 chunks of 4096 rows, equal weights among them."""
    T, budget, sinks, recent = 4_300_001, 70_000, 4, 100
    gen = torch.Generator(device=dev).manual_seed(11)
    w = torch.rand(1, 1, T, generator=gen, device=dev)
    w[..., ::3] = 0.99
    key = torch.randn(1, T, 1, 64, generator=gen, device=dev).to(BF)
    per = -(-budget // 256)
    table = torch.randperm(per, generator=gen, device=dev).view(1, per).to(torch.int32)
    k, v = torch.zeros(per, 1, 256, 64, dtype=BF, device=dev), torch.zeros(per, 1, 256, 64, dtype=BF, device=dev)
    positions = torch.zeros(1, 1, budget, dtype=torch.int32, device=dev)
    scores = torch.zeros(1, 1, budget, device=dev)
    kernels.paged_fill(key, key, k, v, table, weights=w, scores=scores, positions=positions, budget=budget, sinks=sinks, recent=recent)
    x = w[0, 0].clone()
    x[:sinks] = x[T - recent:] = 2.0
    want = torch.sort(x, descending=True, stable=True).indices[:budget].sort().values
    assert torch.equal(positions[0, 0].long(), want) and torch.equal(scores[0, 0], w[0, 0, want])
    r = torch.arange(budget, device=dev)
    at = table[0].long()[r // 256]
    assert torch.equal(k[at, 0, r % 256], key[0, want, 0]) and torch.equal(v[at, 0, r % 256], key[0, want, 0])


# ------------------------------------------------------------------------------------------------ weights of a prompt
@pytest.mark.parametrize("dt,B,T,W,heads,gs,dim,lens", [
    (BF, 1, 1, 1, 1, 1, 128, None),
    (HF, 2, 33, 33, 1, 3, 64, None),
    (BF, 3, 70, 9, 2, 4, 128, [70, 5, 0]),
    (BF, 1, 260, 40, 1, 7, 128, None),
    (HF, 2, 515, 16, 2, 16, 64, [515, 129]),
    (BF, 1, 130, 130, 2, 2, 128, [129]),
    (BF, 1, 3300, 3, 1, 5, 64, None),
    (BF, 1, 700, 700, 1, 4, 128, None),
    (HF, 2, 600, 300, 1, 3, 64, [600, 299]),
    (BF, 1, 1600, 40, 2, 16, 128, [1599]),
])
def test_prompt_weights(dev, dt, B, T, W, heads, gs, dim, lens):
    gen = torch.Generator().manual_seed(T + W)
    q, key = (2 * _randn(gen, B, W, heads * gs, dim)).to(dt), _randn(gen, B, T, heads, dim).to(dt)
    lens_t = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    want, size = oracle.weigh(q, key, lens_t, dim ** -0.5)
    if lens is not None:   # what lies behind a prompt's end has no say
        for b, n in enumerate(lens):
            key[b, n:] = math.nan
            q[b, :max(0, W - n)] = math.inf
    # heads first, as a transposed view, and a part of a wider tensor
    kd = key.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
    qd = torch.empty(B, W, heads * gs, dim + 8, dtype=dt, device=dev)[..., :dim].copy_(q)
    got = kernels.attention_weights(qd, kd, seqlens=None if lens is None else lens_t.to(dev))
    # relative errors: of the exponentials (their arguments are sums of dim products in fp32, up to `size`, less a log-sum-exp of
    # that order), of the sum of T terms in the lse and of W * gs terms here, all in fp32
    rel = 4 * (dim + 12) * F * (1 + size) + (64 + T / 32 + W * gs / 32) * F
    assert bool(((got.cpu().double() - want).abs() <= rel * want + 1e-30).all()), \
        float(((got.cpu().double() - want).abs() / want.clamp(min=1e-30)).max())
    again = kernels.attention_weights(q.to(dev), key.to(dev), seqlens=None if lens is None else lens_t.to(dev))
    assert torch.equal(again, got)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0])
def test_prompt_weights_scales(dev, scale):
    gen = torch.Generator().manual_seed(9)
    q, key = _randn(gen, 1, 50, 3, 64).to(BF), _randn(gen, 1, 300, 1, 64).to(BF)
    want, size = oracle.weigh(q, key, None, scale)
    got = kernels.attention_weights(q.to(dev), key.to(dev), scale=scale)
    rel = 4 * (64 + 12) * F * (1 + size.abs()) + (64 + 300 / 32 + 150 / 32) * F
    assert bool(((got.cpu().double() - want).abs() <= rel * want + 1e-30).all())


def test_writers_refuse_shared_memory(dev):
    """What a call writes while it still reads it elsewhere."""
    x, table = torch.zeros(3, 1, 16, 64, dtype=BF, device=dev), torch.arange(2, dtype=torch.int32, device=dev)[None]
    row, w, lens = torch.zeros(1, 40, 1, 64, dtype=BF, device=dev), torch.rand(1, 1, 40, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    v, one, places = x.clone(), row[:, :1], torch.zeros(1, 1, 32, dtype=torch.int32, device=dev)
    for call in (lambda: kernels.paged_fill(row, row, x, v, table, weights=w, scores=w),
                 lambda: kernels.paged_fill(row, row, x, x, table, weights=w),
                 lambda: kernels.paged_fill(row, row, x, v, table, lens, seqlens=lens, weights=w),
                 lambda: kernels.paged_append(one, one, x, x, table, lens),
                 lambda: kernels.paged_append(one, one, x, v, table, lens, lens),
                 lambda: kernels.paged_append(one, one, x, v, table, lens, table[0, :1], positions=places, token_positions=table[0, :1])):
        with pytest.raises(ValueError, match="memory"):
            call()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("T", [3, 7, 31])
def test_prompt_weights_of_equal_keys(dev, T, dim):
    """One query, T equal keys: each exponential is that of 0 whatever the score, sums are whole numbers, and the weight 1 / T
    carries one rounding of the inverse (another's room for the division), however large the score is."""
    gen = torch.Generator().manual_seed(T)
    q, key = _randn(gen, 8, 1, 16, dim).to(BF), (3 * _randn(gen, 8, 1, 16, dim)).to(BF).expand(8, T, 16, dim)
    got = kernels.attention_weights(q.to(dev), key.to(dev)).cpu().double()
    assert bool(((got * T - 1).abs() <= 2 * F).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf], ids=["nan", "inf"])
@pytest.mark.parametrize("where", [0.0, 0.4, 1.0], ids=["first", "middle", "last"])
@pytest.mark.parametrize("dt,T,W,heads,gs,dim,n", [
    (BF, 70, 9, 2, 4, 128, 70),
    (HF, 70, 40, 1, 3, 64, 33),
    (BF, 700, 300, 2, 2, 64, 640),
    (BF, 500, 500, 1, 4, 128, 500),
    (HF, 900, 70, 1, 3, 128, 901 - 13),
])
def test_prompt_weights_of_a_spoilt_query(dev, dt, T, W, heads, gs, dim, n, where, bad):
    """The keys that it sees have a NaN, those behind its token the other queries' weights, other heads what they had."""
    gen = torch.Generator().manual_seed(T + W + gs)
    q, key = _randn(gen, 2, W, heads * gs, dim).to(dt), _randn(gen, 2, T, heads, dim).to(dt)
    lens = torch.tensor([n, T], dtype=torch.int32)
    scale = dim ** -0.5
    clean, size = oracle.weigh(q, key, lens, scale)
    was = kernels.attention_weights(q.to(dev), key.to(dev), seqlens=lens.to(dev)).cpu()
    i, j = max(W - n, int(where * (W - 1))), gs - 1      # a query that is one of the prompt's; a head of the first key-value head
    last = n - W + i
    p = torch.softmax(key[0, :last + 1, 0].double() @ q[0, i, j].double() * scale, 0)
    clean[0, 0, :last + 1] -= p
    q[0, i, j, 5] = bad
    got = kernels.attention_weights(q.to(dev), key.to(dev), seqlens=lens.to(dev)).cpu()
    assert bool(got[0, 0, :last + 1].isnan().all())
    rel = 4 * (dim + 12) * F * (1 + size) + (64 + T / 32 + W * gs / 32) * F     # (as in test_prompt_weights)
    assert bool(((got[0, 0, last + 1:].double() - clean[0, 0, last + 1:]).abs() <= rel[0, 0] * clean[0, 0, last + 1:] + 1e-30).all())
    assert torch.equal(got[1], was[1]) and torch.equal(got[0, 1:], was[0, 1:])


@pytest.mark.parametrize("T,W,at", [(70, 9, 0), (300, 300, 299), (900, 20, 450)])
def test_prompt_weights_of_a_spoilt_key(dev, T, W, at):
    """Every query behind it sees it, so nothing of its head is known: the last token's query sees all."""
    gen = torch.Generator().manual_seed(T)
    q, key = _randn(gen, 1, W, 4, 64).to(BF), _randn(gen, 1, T, 2, 64).to(BF)
    was = kernels.attention_weights(q.to(dev), key.to(dev))
    key[0, at, 1, 9] = math.nan
    got = kernels.attention_weights(q.to(dev), key.to(dev))
    assert bool(got[0, 1].isnan().all()) and torch.equal(got[0, 0], was[0, 0])


def test_prompt_weights_far_apart(dev):
    """Scores that rise along the prompt by more than an exponential of fp32 can tell, and fall."""
    gen = torch.Generator().manual_seed(10)
    T = 900
    key = torch.zeros(1, T, 2, 64)
    key[0, :, 0, 0] = torch.arange(T) / 4       # 0 .. 225, exact in bfloat16
    key[0, :, 0, 0] = key[0, :, 0, 0].floor()
    key[0, :, 1, 0] = -key[0, :, 0, 0]
    key[..., 1] = _randn(gen, 1, T, 2)
    key = key.to(BF)
    q = torch.zeros(1, 7, 2, 64)
    q[..., 0], q[..., 1] = 16.0, 1.0
    want, size = oracle.weigh(q.to(BF), key, None, 1.0)
    got = kernels.attention_weights(q.to(BF).to(dev), key.to(dev), scale=1.0).cpu().double()
    # (each score is exact up to a rounding of its sum and one of its product with 1 / ln 2: 3 roundings of 3600 / ln 2 here)
    rel = 8 * F * (1 + size) * 1.5 + 64 * F
    assert bool(((got - want).abs() <= rel * want + 1e-30).all())


def test_native_and_general_calls_do_the_same(dev, monkeypatch):
    """The native calls launch what the wrappers' general way launches; arguments that are not in order reach the general way,
    which words the error."""
    gen = torch.Generator().manual_seed(12)
    B, heads, gs, dim, page, T, budget = 3, 2, 4, 64, 16, 200, 40
    k, v, table = _pool(gen, HF, B, heads, dim, page, budget, junk=False)
    key, q = _randn(gen, B, T, heads, dim).to(HF).to(dev), _randn(gen, B, T, heads * gs, dim).to(HF).to(dev)
    lens = torch.tensor([200, 40, 17], dtype=torch.int32, device=dev)

    class General:
        def __getattr__(self, name):
            return lambda *a: None

    def run():
        kk, vv, held, more = k.to(dev), v.to(dev), torch.zeros(B, dtype=torch.int32, device=dev), torch.zeros(B, dtype=torch.int32, device=dev)
        scores = torch.zeros(B, heads, budget, device=dev)
        positions = torch.zeros(B, heads, budget, dtype=torch.int32, device=dev)
        t = table.to(dev)
        w = kernels.attention_weights(q[:, -9:], key, seqlens=lens, scale=0.1)
        kernels.paged_fill(key, key * 2, kk, vv, t, held, seqlens=lens, weights=w, scores=scores, positions=positions, budget=budget,
                           sinks=1, recent=3)
        kernels.paged_append(key[:, :1], key[:, 1:2], kk, vv, t, held, more, scores=scores, positions=positions, token_positions=lens,
                             budget=budget, sinks=1, recent=3)
        out, lse = kernels.paged_attention(q[:, :1].contiguous(), kk, vv, t, more, scores=scores, max_len=budget, return_softmax_lse=True)
        return w, kk, vv, held, more, scores, positions, out, lse
    first = run()      # (sizes the scratch)
    native = run()
    with monkeypatch.context() as m:
        m.setattr(kernels, "step_calls", General)
        general = run()
    for a, b, c in zip(first, native, general):
        assert torch.equal(a, b) and torch.equal(b, c)
    w, kk, vv, held, more, scores, positions, _, _ = native
    odd = torch.zeros(B, T, heads, dim + 8, dtype=HF, device=dev)[..., 1:dim + 1]
    t = table.to(dev)
    one = q[:, :1].contiguous()
    for error, match, call in (
            (ValueError, "contiguous", lambda: kernels.paged_attention(q[:, :1, :, :].transpose(1, 2).contiguous().transpose(1, 2)[..., ::2], kk, vv, t, more)),
            (TypeError, "int32", lambda: kernels.paged_attention(one, kk, vv, t, more.long())),
            (ValueError, "max_len", lambda: kernels.paged_attention(one, kk, vv, t, more, max_len=49)),
            (ValueError, "scores", lambda: kernels.paged_attention(one, kk, vv, t, more, scores=scores)),   # (48 rows, scores of 40)
            (ValueError, "query heads", lambda: kernels.paged_attention(one[:, :, :7].contiguous(), kk, vv, t, more)),
            (ValueError, "cpu|cuda", lambda: kernels.paged_attention(one, kk, vv, table, more)),
            (TypeError, "float16", lambda: kernels.paged_attention(one.bfloat16(), kk, vv, t, more)),
            (ValueError, "another tensor", lambda: kernels.paged_append(key[:, :1], key[:, :1], kk, vv, t, held, held)),
            (ValueError, "budget", lambda: kernels.paged_append(key[:, :1], key[:, :1], kk, vv, t, held, budget=49)),
            (ValueError, "positions", lambda: kernels.paged_append(key[:, :1], key[:, :1], kk, vv, t, held, scores=scores, budget=40)),
            (ValueError, "share memory", lambda: kernels.paged_append(key[:, :1], key[:, :1], kk[:1].expand(kk.shape), vv, t, held)),
            (ValueError, "share memory", lambda: kernels.paged_attention(one, kk, vv, t, more, scores=scores[:1].expand(B, heads, 40), max_len=40)),
            (ValueError, "weights", lambda: kernels.paged_fill(key, key, kk, vv, t, held, budget=40)),
            (ValueError, "aligned", lambda: kernels.paged_fill(odd, odd, kk, vv, t, held, weights=w, budget=40)),
            (ValueError, "W <= T", lambda: kernels.attention_weights(q, key[:, :9])),
            (RuntimeError, "Half and BFloat16", lambda: kernels.attention_weights(q.float(), key.float()))):
        with pytest.raises(error, match=match):
            call()


def test_scratch_does_not_grow_in_a_capture(dev):
    gen = torch.Generator().manual_seed(13)
    k, v, table = _pool(gen, BF, 1, 1, 64, 16, 64, junk=False)
    args = [t.to(dev) for t in (_randn(gen, 1, 1, 4, 64).to(BF), k, v, table, torch.tensor([50], dtype=torch.int32))]
    own = kernels.Scratch()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capture"), torch.cuda.graph(graph):
        kernels.paged_attention(*args, scratch=own)
    want = kernels.paged_attention(*args, scratch=own)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernels.paged_attention(*args, scratch=own)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
