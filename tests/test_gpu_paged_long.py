"""The paged cache's operators where there is much to do: pages past a wave's first 64 table entries, groups of many parts,
more sequences than threads, many tiles and several column blocks of a prompt's weights.  Which sizes those are is the launches' rule;
tests/test_paged_plans.py asks it whether the cases here are still what they are meant to be.
Compared with 64 bits on the device; u = eps / 2 of the element type and F = 2^-24 count roundings."""
import math

import pytest
import torch

from retrievalattention_amd import kernels

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
F = 2.0 ** -24

# dt, heads, gs, dim, W, T, lens
ENDS = [20011, 19000 - 31, 16500, 321, 300, 250, 190, 130, 97, 5, 0]   # inside a split, of 1 to 6 tiles and odd halves of one, and nothing
STREAMED = [
    (BF, 4, 1, 128, 5, 20011, ENDS),          # a part of one block of columns
    (HF, 4, 4, 64, 16, 20011, ENDS),
    (BF, 4, 4, 128, 64, 20011, ENDS),         # two blocks in one workgroup
    (HF, 3, 7, 64, 33, 20011, ENDS),
    (BF, 2, 4, 64, 200, 20011, ENDS),         # several blocks
    (HF, 2, 5, 128, 100, 20011, ENDS),
    (BF, 1, 3, 128, 9000, 9000, [9000, 8199, 4097, 500]),   # whole prompts
    (HF, 2, 4, 128, 64, 90001, [90001, 61002]),             # splits that a launch of its own joins
]
# the same, and the (sequence, head) pairs that are compared: several blocks to a workgroup
BLOCKS = [
    (BF, 8, 16, 128, 1011, 8300, [8300, 8300, 4111, 1500, 700, 64, 1, 0], [(0, 0), (1, 7), (2, 3), (3, 0), (4, 6), (5, 1), (6, 2), (7, 4)]),
    (HF, 4, 16, 64, 8192, 24000, [24000, 23333], [(0, 1), (1, 3)]),
    (BF, 8, 4, 128, 17000, 17000, [17000], [(0, 0), (0, 7)]),
]

# dt, heads, gs, dim, page, lens, starts: long caches of few pages that repeat, whose rows many workgroups share
LONG = [(dt, 8, gs, 64, page, [180000 - 997 * b for b in range(8)], [0, 16, 40017, 5, 0, 1023, 77777, 64])
        for dt, gs, page in ((BF, 4, 1), (HF, 1, 2), (BF, 8, 4), (HF, 3, 8), (BF, 4, 16), (HF, 12, 64), (HF, 5, 16), (BF, 16, 8))]
LONG += [(BF, 2, 4, 128, 64, [1500000, 0, 1400001, 3000000], [7, 0, 1, 500003]),
         (HF, 2, 7, 128, 16, [2500000, 2600000], None),
         (BF, 4, 16, 128, 4, [600000, 900001], [0, 31])]
# the same: many parts to a group, which the join's waves take 64 at a time
PARTS = [(BF, 1, 4, 128, 64, [131072], None), (HF, 1, 7, 64, 16, [70001, 0, 41000], [3, 0, 999]), (BF, 2, 16, 64, 16, [300001], [70]),
         (HF, 1, 16, 128, 32, [600000], None), (BF, 1, 1, 64, 8, [16000, 270000, 17, 0, 33], [15999, 0, 0, 0, 32])]
# sequences beyond the 512 that a workgroup looks at at a time, sharing their rows: dt, heads, gs, dim, page, room, sequences
MANY = [(BF, 1, 4, 64, 16, 2304, 700), (HF, 2, 1, 64, 64, 2560, 1300), (BF, 1, 3, 128, 8, 3000, 513), (HF, 1, 8, 64, 32, 5000, 1025)]


def _randn(gen, dev, *shape):
    return torch.randn(*shape, generator=gen, device=dev)


def _weigh(q, key, n, scale):
    """Weights [n] that the queries [W, gs, dim] of the last W tokens give the first n keys [T, dim], and the largest sum of |q k| scale."""
    W, gs, dim = q.shape
    out, size = torch.zeros(n, dtype=torch.float64, device=q.device), 0.0
    k, w = key[:n].double().T.contiguous(), min(W, n)
    step = max(1, (1 << 24) // max(n, 1))
    for i0 in range(W - w, W, step):
        i1 = min(i0 + step, W)
        last = n - W + torch.arange(i0, i1, device=q.device)
        later = torch.arange(n, device=q.device)[None] > last[:, None]
        for j in range(gs):
            x = (q[i0:i1, j].double() @ k).mul_(scale)
            out += torch.softmax(x.masked_fill_(later, -math.inf), 1).sum(0)
            size = max(size, float((q[i0:i1, j].abs().float() @ k.abs().float()).max()) * scale * 1.0001)
    return out, size


def _check_weights(got, q, key, lens, gs, pairs):
    dim, W, T = q.shape[3], q.shape[1], key.shape[1]
    for b, h in pairs:
        n = lens[b]
        want, size = _weigh(q[b, :, h * gs:(h + 1) * gs], key[b, :, h], n, dim ** -0.5)
        # an exponential's argument is a sum of dim products in fp32, up to `size`, less one of that order; sums of T terms for a query
        # and of W * gs terms for a key
        rel = 4 * (dim + 12) * F * (1 + size) + (64 + T / 32 + W * gs / 32) * F
        d = (got[b, h, :n].double() - want).abs()
        assert bool((d <= rel * want + 1e-30).all()), (b, h, float((d / want.clamp(min=1e-30)).max()), rel)
        assert bool((got[b, h, n:] == 0).all()), (b, h)


def _prompts(dev, dt, heads, gs, dim, W, T, lens):
    gen = torch.Generator(device=dev).manual_seed(T + W + gs)
    B = len(lens)
    key = _randn(gen, dev, B, T, heads, dim).to(dt)
    q = _randn(gen, dev, B, W, heads * gs, dim).to(dt)
    for b, n in enumerate(lens):   # what lies behind a prompt's end has no say
        key[b, n:] = math.nan
        q[b, :max(0, W - n)] = math.nan
    return q, key, torch.tensor(lens, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("dt,heads,gs,dim,W,T,lens", STREAMED)
def test_prompt_weights_of_many_tiles(dev, dt, heads, gs, dim, W, T, lens):
    q, key, lens_t = _prompts(dev, dt, heads, gs, dim, W, T, lens)
    got = kernels.attention_weights(q, key, seqlens=lens_t)
    _check_weights(got, q, key, lens, gs, [(b, h) for b in range(len(lens)) for h in range(heads)])
    for _ in range(5):
        assert torch.equal(kernels.attention_weights(q, key, seqlens=lens_t), got)


@pytest.mark.parametrize("dt,heads,gs,dim,W,T,lens,pairs", BLOCKS)
def test_prompt_weights_of_several_blocks_to_a_workgroup(dev, dt, heads, gs, dim, W, T, lens, pairs):
    """Sums of several blocks of columns are added up in LDS where the parts of one each would be too many."""
    q, key, lens_t = _prompts(dev, dt, heads, gs, dim, W, T, lens)
    got = kernels.attention_weights(q, key, seqlens=lens_t)
    _check_weights(got, q, key, lens, gs, pairs)
    assert torch.equal(kernels.attention_weights(q, key, seqlens=lens_t), got)
    (b, h), n = pairs[0], lens[pairs[0][0]]
    for i in (W - min(W, n), W // 2, W - 1):    # a query with a NaN: what it sees, and only that
        bad = q.clone()
        bad[b, i, h * gs + gs // 2, 1] = math.nan
        spoilt = kernels.attention_weights(bad, key, seqlens=lens_t)
        last = n - W + i
        assert bool(spoilt[b, h, :last + 1].isnan().all()) and bool(spoilt[b, h, last + 1:].isfinite().all())
        spoilt[b, h] = got[b, h]
        assert torch.equal(spoilt, got)


def _attend(q, k_pages, v_pages, table, n, start, scale):
    """One sequence and head: q [gs, dim], pages [pages, page_rows, dim], table [n]; out, lse, weights, sums of p |v|, largest sum of |q k| scale."""
    page = k_pages.shape[1]
    k, v = k_pages.reshape(-1, k_pages.shape[2]).double(), v_pages.reshape(-1, v_pages.shape[2]).double()
    r = torch.arange(start, n, device=q.device)
    at = table.long()[r // page] * page + r % page
    x = (q.double() @ k.T.contiguous() * scale)[:, at]
    size = (q.double().abs() @ k.abs().T.contiguous() * scale).max(1).values
    p = torch.softmax(x, 1)
    # rows repeat: their weights first
    each = torch.zeros(q.shape[0], k.shape[0], dtype=torch.float64, device=q.device).index_add_(1, at, p)
    return each @ v, torch.logsumexp(x, 1), p, each @ v.abs(), size


def _check_attention(dev, dt, heads, gs, dim, page, lens, starts, pool=64):
    gen = torch.Generator(device=dev).manual_seed(lens[0] + page + gs)
    B, per = len(lens), -(-max(lens) // page)
    pool = max(pool, 2048 // page)
    k, v = _randn(gen, dev, pool, heads, page, dim).to(dt), _randn(gen, dev, pool, heads, page, dim).to(dt)
    table = torch.randint(pool, (B, per), generator=gen, device=dev, dtype=torch.int32)
    q = (2 * _randn(gen, dev, B, 1, heads * gs, dim)).to(dt)
    lens_t = torch.tensor(lens, dtype=torch.int32, device=dev)
    starts_t = None if starts is None else torch.tensor(starts, dtype=torch.int32, device=dev)
    before = torch.rand(B, heads, max(lens), generator=gen, device=dev)
    scores = before.clone()
    out, lse = kernels.paged_attention(q, k, v, table, lens_t, starts=starts_t, scores=scores, max_len=max(lens), return_softmax_lse=True)
    plain = kernels.paged_attention(q, k, v, table, lens_t, starts=starts_t, max_len=max(lens))
    assert torch.equal(plain, out)
    u = torch.finfo(dt).eps / 2
    for b in range(B):
        first = min(starts[b] if starts else 0, lens[b])
        for h in range(heads):
            mine = slice(h * gs, (h + 1) * gs)
            got, got_lse, after = out[b, 0, mine].double(), lse[b, mine].double(), scores[b, h]
            untouched = torch.ones(max(lens), dtype=torch.bool, device=dev)
            untouched[first:lens[b]] = False
            assert torch.equal(after[untouched], before[b, h][untouched])
            if first == lens[b]:
                assert bool((got == 0).all()) and bool((got_lse == -math.inf).all())
                continue
            want, want_lse, p, absolute, size = _attend(q[b, 0, mine], k[:, h], v[:, h], table[b], lens[b], first, dim ** -0.5)
            # a score is a sum of dim products in fp32, scaled (two roundings more); its exponential is off by that and by two units.
            # A weight's two parts add up to it within 2^-16 (2^-21 in half, and 2^-40 of what the highest score weighs); a result
            # below the normal halves is off by 2^-25.
            n = lens[b] - first
            ds = (dim + 4) * F * size + 8 * F * (1 + size)
            tol = u * want.abs() + (2.0 ** (-16 if dt == BF else -21) + 2 * ds[:, None] + (64 + n / 16) * F) * absolute
            if dt == HF:
                tol = tol + n * 2.0 ** -40 * p.max(1).values[:, None] * v[:, h].abs().max().double() + 2.0 ** -25
            assert bool(((got - want).abs() <= tol).all()), (b, h, float(((got - want).abs() / tol).max()))
            assert bool(((got_lse - want_lse).abs() <= ds + (64 + n / 16) * F + 4 * F * want_lse.abs()).all()), (b, h)
            w = p.sum(0)
            want_scores = before[b, h, first:lens[b]].double() + w
            rel = 2 * ds.max() + (64 + n / 16) * F
            assert bool(((after[first:lens[b]].double() - want_scores).abs() <= rel * w + 18 * F * want_scores).all()), (b, h)


@pytest.mark.parametrize("dt,heads,gs,dim,page,lens,starts", LONG)
def test_attention_past_a_waves_first_table_entries(dev, dt, heads, gs, dim, page, lens, starts):
    """A wave holds 64 entries of the table at a time, the next 64 behind them: every row's weight and the output tell which were used."""
    _check_attention(dev, dt, heads, gs, dim, page, lens, starts)


@pytest.mark.parametrize("dt,heads,gs,dim,page,lens,starts", PARTS)
def test_attention_of_many_parts(dev, dt, heads, gs, dim, page, lens, starts):
    _check_attention(dev, dt, heads, gs, dim, page, lens, starts)


def _many_lengths(room, B):
    """Most empty or short, long ones first, last, and on both sides of each 512th."""
    gen = torch.Generator().manual_seed(B)
    lens = (torch.rand(B, generator=gen) ** 6 * room).int()
    lens[torch.rand(B, generator=gen) < 0.5] = 0
    for b in (0, 1, 510, 511, 512, 513, 1023, 1024, B - 2, B - 1):
        if b < B:
            lens[b] = room - 7 * (b % 13)
    return lens.tolist()


@pytest.mark.parametrize("dt,heads,gs,dim,page,room,B", MANY)
def test_attention_shares_the_rows_of_many_sequences(dev, dt, heads, gs, dim, page, room, B):
    lens = _many_lengths(room, B)
    _check_attention(dev, dt, heads, gs, dim, page, lens, [n // 3 if b % 2 else 0 for b, n in enumerate(lens)])
