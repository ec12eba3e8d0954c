"""The paged cache's operators together, as a model uses them: prompts, tokens, evictions, captured tokens, pages that come and go."""
import pytest
import torch

from oracle import paged as oracle
from retrievalattention_amd.cache_hub import paged_cache
from tests.test_gpu_paged import F, _check_attention, _randn

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _models(dev, dt, config):
    from retrievalattention_amd.model_hub import LlamaModel, LlamaShape
    shape = LlamaShape(hidden_size=256, intermediate_size=512, num_layers=2, num_heads=8, num_key_value_heads=2,
                       head_dim=128, vocab_size=1000)
    B, ctx, new = 2, 700, 8
    gen = torch.Generator().manual_seed(3)
    ids = torch.randint(0, shape.vocab_size, (B, ctx), generator=gen).to(dev)
    models = []
    for kind, conf in (("Paged_Attn", config), ("Full_Flash_Attn", None)):
        m = LlamaModel(shape, ctx + new, dtype=dt, device=dev, seed=1)
        m.init_kv_cache(kind, B, ctx, new, conf)
        models.append(m)
    return *models, ids, new


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("config", [None, dict(page_size=8, pages=2 * 89), dict(budget=707, window=None)], ids=["plain", "small pages", "budget"])
def test_decodes_like_dense_attention(dev, dt, config):
    """Nothing is evicted (707 rows of 708 at most are there when the last token is appended): the model must decode like the same
    model over a dense cache, to the noise of its element type."""
    paged, dense, ids, new = _models(dev, dt, config)
    lp, ld = paged.prefill_forward(ids), dense.prefill_forward(ids)
    assert torch.equal(lp, ld)
    tok = ld.argmax(-1)
    for step in range(new - 1):
        lp, ld = paged.decode_forward(tok), dense.decode_forward(tok)
        d = (lp - ld).abs()
        assert float(d.max()) <= 5e-2 * max(1.0, float(ld.abs().max())), (step, float(d.max()))
        assert float(d.mean()) <= 1.5e-2 * float(ld.abs().mean())
        tok = ld.argmax(-1)
    assert paged.kv_cache.context == dense.kv_cache.context == ids.shape[1] + new - 1


def _inputs(gen, dev, dt, B, heads, gs, dim):
    q, k, v = _randn(gen, B, 1, heads * gs, dim), _randn(gen, B, 1, heads, dim), _randn(gen, B, 1, heads, dim)
    return [x.to(dt).to(dev) for x in (2 * q, k, v)]


@pytest.mark.parametrize("dt,heads,gs,dim,page,budget,sinks,recent,window,prompts", [
    (BF, 2, 4, 128, 16, 40, 4, 8, 16, [100, 33]),
    (HF, 1, 7, 64, 8, 37, 0, 1, None, [64, 200, 36]),
    (BF, 3, 1, 128, 32, 70, 2, 30, 5, [69, 3]),
])
def test_prompts_then_tokens_with_evictions(dev, dt, heads, gs, dim, page, budget, sinks, recent, window, prompts):
    """Every step against its definition on what the cache held before it: which rows a prompt keeps and a token takes (exactly, by
    the scores that were there), the attention's output, the scores that it leaves."""
    gen = torch.Generator().manual_seed(budget)
    B, layers, steps = len(prompts), 2, 12
    c = paged_cache(layers, B, 400, heads, heads * gs, dim, dt, dev, page_size=page, budget=budget, sinks=sinks, recent=recent,
                    window=window)
    for b, T in enumerate(prompts):
        for l in range(layers):
            q, k, v = ((s * _randn(gen, 1, T, n, dim)).to(dt) for s, n in ((2, heads * gs), (1, heads), (1, heads)))
            c.prefill_update_kv_cache(q.to(dev), k.to(dev), v.to(dev), l, b)
            w = T if window is None else min(T, window)
            want, size = oracle.weigh(q[:, T - w:], k, None, dim ** -0.5)
            rel = 4 * (dim + 12) * F * (1 + size) + (64 + T / 32 + w * gs / 32) * F
            n = min(T, budget)
            for h in range(heads):
                at, scores = c.positions[l][b, h, :n].cpu().long(), c.scores[l][b, h, :n].cpu().double()
                x = want[0, h]
                assert bool(((scores - x[at]).abs() <= rel[0, h] * x[at] + 1e-30).all())
                # the kept rows: the protected ones, and none left out that weighs more than one kept by more than the errors of both
                assert at.tolist() == sorted(set(at.tolist()))
                if T > budget:
                    out = torch.ones(T, dtype=torch.bool)
                    out[at] = False
                    assert not out[:sinks].any() and not out[T - recent:].any()
                    free = [int(t) for t in at if sinks <= t < T - recent]
                    assert float(x[out].max()) * (1 - float(rel[0, h])) <= min(float(x[t]) for t in free) * (1 + float(rel[0, h]))
                r = torch.arange(n)
                p = c.block_table[b].cpu().long()[r // page]
                assert torch.equal(c.k_pages[l].cpu()[p, h, r % page], k[0, at, h])
                assert torch.equal(c.v_pages[l].cpu()[p, h, r % page], v[0, at, h])
    assert c.seqlens.tolist() == [min(T, budget) for T in prompts]
    for step in range(steps):
        for l in range(layers):
            q, k, v = _inputs(gen, dev, dt, B, heads, gs, dim)
            lens, seen = c.seqlens.tolist(), c.seen.tolist()
            scores, positions = c.scores[l].cpu().clone(), c.positions[l].cpu().clone()
            c.decode_update_kv_cache(k, v, l)
            for b in range(B):
                assert seen[b] == prompts[b] + step
                for h in range(heads):
                    r = lens[b] if lens[b] < budget else oracle.victim(scores[b, h], positions[b, h], budget, seen[b], sinks, recent)
                    scores[b, h, r], positions[b, h, r] = 0.0, seen[b]
                    p = int(c.block_table[b, r // page])
                    assert torch.equal(c.k_pages[l][p, h, r % page], k[b, 0, h]) and torch.equal(c.v_pages[l][p, h, r % page], v[b, 0, h])
            assert torch.equal(c.scores[l].cpu(), scores) and torch.equal(c.positions[l].cpu(), positions)
            now = c.new_seqlens.cpu()
            assert now.tolist() == [min(n + 1, budget) for n in lens]
            pages = [t.cpu() for t in (c.k_pages[l], c.v_pages[l], c.block_table)]
            out = c.compute(q, l)
            from retrievalattention_amd import kernels
            _, lse = kernels.paged_attention(q, c.k_pages[l], c.v_pages[l], c.block_table, now.to(dev), return_softmax_lse=True)
            _check_attention(q.cpu(), *pages, now, None, out, lse, dim ** -0.5, scores, c.scores[l])


@pytest.mark.parametrize("budget", [None, 48])
def test_captured_tokens_replay_like_eager_ones(dev, budget):
    """One token of two layers captured and replayed, with the program's own work between the replays: every replay leaves what an
    eager twin has, to the bit."""
    gen = torch.Generator().manual_seed(4)
    B, heads, gs, dim, layers = 3, 2, 4, 128, 2
    caches = [paged_cache(layers, B, 100, heads, heads * gs, dim, BF, dev, page_size=8, budget=budget, sinks=2, recent=4)
              for _ in range(2)]
    for b, T in enumerate((60, 41, 7)):
        for l in range(layers):
            q, k, v = (_randn(gen, 1, T, n, dim).to(BF).to(dev) for n in (heads * gs, heads, heads))
            for c in caches:
                c.prefill_update_kv_cache(q, k, v, l, b)
    static = [[torch.zeros_like(x) for x in _inputs(gen, dev, BF, B, heads, gs, dim)] for _ in range(layers)]

    def token(c):
        outs = []
        for l in range(layers):
            c.decode_update_kv_cache(static[l][1], static[l][2], l)
            outs.append(c.compute(static[l][0], l))
        return outs

    eager, replayed = caches
    graph, got = torch.cuda.CUDAGraph(), None
    for step in range(20):
        for l in range(layers):
            for x, y in zip(static[l], _inputs(gen, dev, BF, B, heads, gs, dim)):
                x.copy_(y)
        want = token(eager)
        if step < 2:
            got = token(replayed)          # (the first token sizes the scratch)
        else:
            if step == 2:
                with torch.cuda.graph(graph):
                    got = token(replayed)
            replayed.prepare_token()
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b), step
        for name in ("seqlens", "new_seqlens", "seen", "block_table"):
            assert torch.equal(getattr(eager, name), getattr(replayed, name)), (step, name)
        for l in range(layers):
            assert torch.equal(eager.k_pages[l], replayed.k_pages[l])
            if budget:
                assert torch.equal(eager.scores[l], replayed.scores[l]) and torch.equal(eager.positions[l], replayed.positions[l])


def test_two_captured_caches_on_two_streams(dev):
    """Caches have scratch of their own: their captured tokens replay side by side."""
    gen = torch.Generator().manual_seed(5)
    heads, gs, dim = 2, 4, 64
    caches, graphs, outs, inputs, wants = [], [], [], [], []
    for i in range(2):
        c = paged_cache(1, 2, 2000, heads, heads * gs, dim, HF, dev, budget=900, recent=16)
        for b in range(2):
            q, k, v = (_randn(gen, 1, 1000 + 100 * i, n, dim).to(HF).to(dev) for n in (heads * gs, heads, heads))
            c.prefill_update_kv_cache(q, k, v, 0, b)
        x = _inputs(gen, dev, HF, 2, heads, gs, dim)
        c.decode_update_kv_cache(x[1], x[2], 0)
        c.compute(x[0], 0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.decode_update_kv_cache(x[1], x[2], 0)
            out = c.compute(x[0], 0)
        caches.append(c), graphs.append(graph), outs.append(out), inputs.append(x)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(5):
        for i in range(2):
            streams[i].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i, c in enumerate(caches):
            x = inputs[i]
            from retrievalattention_amd import kernels
            want = kernels.paged_attention(x[0], c.k_pages[0], c.v_pages[0], c.block_table, c.new_seqlens, max_len=900)
            assert torch.equal(want, outs[i]), (rep, i)


def test_places_come_and_go(dev):
    """A place without a sequence attends nothing and stays empty; its pages serve another; a new prompt starts from nothing."""
    gen = torch.Generator().manual_seed(6)
    heads, gs, dim = 1, 2, 64
    c = paged_cache(1, 3, 64, heads, heads * gs, dim, BF, dev, page_size=16, pages=8)
    prompt = lambda T: [_randn(gen, 1, T, n, dim).to(BF).to(dev) for n in (heads * gs, heads, heads)]  # noqa: E731
    for b, T in ((0, 40), (2, 20)):
        c.prefill_update_kv_cache(*prompt(T), 0, b)

    def token():
        q, k, v = _inputs(gen, dev, BF, 3, heads, gs, dim)
        c.decode_update_kv_cache(k, v, 0)
        now, pages = c.new_seqlens.cpu(), [t.cpu() for t in (c.k_pages[0], c.v_pages[0], c.block_table)]
        out = c.compute(q, 0)
        want, _, _, absolute, _ = oracle.attention(q.cpu(), *pages, now, None, dim ** -0.5)
        assert bool(((out.cpu().double() - want).abs() <= 2 ** -8 * (absolute + want.abs()) + 1e-4 * absolute).all())
        return out
    out = token()
    assert bool((out[1] == 0).all()) and c.seqlens.tolist() == [41, 0, 21] and c.free_pages == 8 - 3 - 2
    c.release(0)
    c.prefill_update_kv_cache(*prompt(60), 0, 1)
    for _ in range(3):
        out = token()
    assert bool((out[0] == 0).all()) and c.seqlens.tolist() == [0, 63, 24] and c.seen.tolist() == [0, 63, 24]
    c.prefill_update_kv_cache(*prompt(1), 0, 1)
    token()
    assert c.seqlens.tolist() == [0, 2, 25] and c.free_pages == 8 - 1 - 2
