"""The operators of the paged key-value cache as measurable cases: a new token's attention over the pages (with or without
adding its weights to the rows' scores), the append of a token that may take the place of the row with the lowest score,
the weights that a prompt's queries give its keys, and the write of a prompt's heaviest rows into pages.

`listed()` gives the named cases, `draw(rng)` one more of the same ranges.  With `own` false, `run` computes the operators
from elementary torch operations; with `own` true it calls the package."""
import math

import torch

own = False
DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # the single user with a short context: one layer's attention, launch and host time count
        dict(name="attend_one", kind="attend", dtype="bf16", dim=128, batch=1, heads=8, group=4, tokens=331, page=16,
             ragged=False, window=0, scored=False),
        # four long contexts, nothing evicted: the dense baseline of the benchmark's headline shape, bound by memory
        dict(name="attend_long", kind="attend", dtype="bf16", dim=128, batch=4, heads=8, group=4, tokens=131072, page=64,
             ragged=False, window=0, scored=False),
        # a serving batch of unequal lengths (empty and one-token sequences among them), seven heads to a key-value head,
        # some sequences attend a window only
        dict(name="attend_ragged", kind="attend", dtype="fp16", dim=128, batch=16, heads=4, group=7, tokens=61440, page=16,
             ragged=True, window=4096, scored=False),
        # a batch over caches of a budget: the weights are added to the rows' scores for the next eviction
        dict(name="attend_scored", kind="attend", dtype="bf16", dim=128, batch=32, heads=8, group=4, tokens=4096, page=32,
             ragged=False, window=0, scored=True),
        # a token of one sequence takes the place of the weakest of 1024 rows in every head
        dict(name="append_one", kind="append", dtype="bf16", dim=128, batch=1, heads=8, page=16, budget=1024, sinks=4,
             recent=64, ragged=False),
        # the same for a batch with large budgets, some sequences still below theirs
        dict(name="append_batch", kind="append", dtype="fp16", dim=128, batch=32, heads=8, page=64, budget=8192, sinks=4,
             recent=512, ragged=True),
        # the prompt's last queries weigh a short prompt's keys
        dict(name="weigh_short", kind="weigh", dtype="fp16", dim=128, batch=1, heads=4, group=7, window=32, tokens=1111,
             ragged=False),
        # an observation window at the end of a long prompt: the keys are streamed
        dict(name="weigh_window", kind="weigh", dtype="bf16", dim=128, batch=1, heads=8, group=4, window=64, tokens=131072,
             ragged=False),
        # every query of a prompt weighs the keys up to its own: matrix products and exponentials
        dict(name="weigh_prompt", kind="weigh", dtype="bf16", dim=128, batch=1, heads=8, group=4, window=8192, tokens=8192,
             ragged=False),
        # a short prompt goes into pages whole
        dict(name="fill_short", kind="fill", dtype="bf16", dim=128, batch=1, heads=8, tokens=1000, page=16, budget=0, sinks=0,
             recent=0, ragged=False),
        # the 8192 heaviest rows of a long prompt
        dict(name="fill_long", kind="fill", dtype="bf16", dim=128, batch=1, heads=8, tokens=131072, page=64, budget=8192,
             sinks=4, recent=512, ragged=False),
        # a padded batch of prompts, some of them shorter than the budget
        dict(name="fill_ragged", kind="fill", dtype="fp16", dim=128, batch=4, heads=4, tokens=30011, page=32, budget=2000,
             sinks=4, recent=64, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "append", "weigh", "weigh", "fill", "fill"))
    case = dict(kind=kind, dtype=rng.choice(("bf16", "bf16", "fp16")), dim=rng.choice((64, 128, 128)),
                heads=rng.choice((1, 2, 4, 8)))
    page = rng.choice((8, 16, 16, 32, 64, 256))
    if kind == "attend":
        tokens = _log(rng, 1, 131072)
        return dict(case, batch=min(_log(rng, 1, 64), max(1, 4194304 // (case["heads"] * tokens))),
                    group=rng.choice((1, 2, 3, 4, 4, 7, 8, 16)), tokens=tokens, page=page, ragged=rng.random() < 0.5,
                    window=rng.choice((0, 0, _log(rng, 1, tokens))), scored=rng.random() < 0.4)
    if kind == "append":
        budget = _log(rng, 16, 32768)
        sinks = rng.choice((0, 4))
        return dict(case, batch=min(_log(rng, 1, 64), max(1, 2097152 // (case["heads"] * budget))), page=page,
                    budget=budget, sinks=sinks, recent=rng.randrange(budget // 2), ragged=rng.random() < 0.5)
    if kind == "weigh":
        tokens, group = _log(rng, 1, 131072), rng.choice((1, 2, 3, 4, 4, 7, 8, 16))
        most = max(1, 2 ** 31 // (case["heads"] * group * tokens))
        window = min(tokens, rng.choice((_log(rng, 1, 256), _log(rng, 1, 8192))), most)
        return dict(case, batch=min(_log(rng, 1, 8), max(1, most // window)), group=group, window=window, tokens=tokens,
                    ragged=rng.random() < 0.5)
    tokens = _log(rng, 1, 131072)
    evicts = tokens > 64 and rng.random() < 0.7
    budget = _log(rng, 32, max(33, tokens // 2)) if evicts else 0
    return dict(case, batch=min(_log(rng, 1, 8), max(1, 1048576 // (case["heads"] * tokens))), tokens=tokens, page=page,
                budget=budget, sinks=rng.choice((0, 4)) if evicts else 0, recent=rng.randrange(budget // 2) if evicts else 0,
                ragged=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEVICE)


def _rows(gen, dtype, *shape):
    """Keys: a few channels of each head are several times as large as the others, as after rotary embedding."""
    scale = 1.0 + 3.0 * (torch.rand(shape[-1], generator=gen, device=DEVICE) < 4 / 128)
    return (_normal(gen, *shape) * scale).to(dtype)


def _lengths(gen, batch, most, ragged):
    """int32 [batch]: all `most`, or spread over the logarithm down to nothing, the first the longest."""
    if not ragged:
        return torch.full((batch,), most, dtype=torch.int32, device=DEVICE)
    part = torch.exp(-torch.rand(batch, generator=gen, device=DEVICE) * math.log(most + 1))
    lens = torch.floor(part * (most + 1)).to(torch.int32).clamp(max=most)
    lens[0] = most
    if batch > 2:
        lens[1] = 0
    return lens


def _table(gen, batch, per):
    """Pages of the sequences, scattered over a pool that has some to spare; int32 [batch, per]."""
    pool = batch * per + 3
    return torch.randperm(pool, generator=gen, device=DEVICE)[:batch * per].view(batch, per).to(torch.int32), pool


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, dim, B, H = TYPES[case["dtype"]], case["dim"], case["batch"], case["heads"]
    s = dict(kind=case["kind"])
    if case["kind"] == "weigh":
        T, W, G = case["tokens"], case["window"], case["group"]
        s["key"] = _rows(gen, dtype, B, T, H, dim)
        # the queries resemble the keys of some tokens of the prompt
        at = torch.randint(T, (W,), generator=gen, device=DEVICE)
        near = s["key"][:, at].float().repeat_interleave(G, 2)
        s["q"] = (_normal(gen, B, W, H * G, dim) + 0.35 * near).to(dtype)
        s["lens"] = _lengths(gen, B, T, True) if case["ragged"] else None
        return s
    if case["kind"] == "fill":
        T, page, budget = case["tokens"], case["page"], case["budget"]
        room = budget or T
        per = -(-room // page)
        s["key"], s["value"] = _rows(gen, dtype, B, T, H, dim), _normal(gen, B, T, H, dim).to(dtype)
        s["lens"] = _lengths(gen, B, T, True) if case["ragged"] else None
        s["table"], pool = _table(gen, B, per)
        s["k"] = torch.zeros((pool, H, page, dim), dtype=dtype, device=DEVICE)
        s["v"] = torch.zeros((pool, H, page, dim), dtype=dtype, device=DEVICE)
        s["held"] = torch.zeros((B,), dtype=torch.int32, device=DEVICE)
        s.update(budget=budget, sinks=case["sinks"], recent=case["recent"], weights=None, scores=None, positions=None)
        if budget:
            # accumulated weights, many of them too small to differ
            w = torch.exp(2.5 * _normal(gen, B, H, T)) * 1e-3
            s["weights"] = torch.where(w < 1e-4, torch.zeros_like(w), w)
            s["scores"] = torch.zeros((B, H, room), device=DEVICE)
            s["positions"] = torch.zeros((B, H, room), dtype=torch.int32, device=DEVICE)
        return s
    page = case["page"]
    if case["kind"] == "append":
        room = case["budget"]
        per = -(-room // page)
        s["table"], pool = _table(gen, B, per)
        s["k"], s["v"] = _rows(gen, dtype, pool, H, page, dim), _normal(gen, pool, H, page, dim).to(dtype)
        s["key"], s["value"] = _rows(gen, dtype, B, 1, H, dim), _normal(gen, B, 1, H, dim).to(dtype)
        lens = torch.full((B,), room, dtype=torch.int32, device=DEVICE)
        if case["ragged"]:   # every fourth sequence is not full yet
            part = torch.rand(B, generator=gen, device=DEVICE)
            lens = torch.where(torch.arange(B, device=DEVICE) % 4 == 3, (part * room).to(torch.int32), lens)
        s["lens"], s["held"] = lens, torch.zeros((B,), dtype=torch.int32, device=DEVICE)
        # rows hold tokens of the sequence in any order, as evictions leave them: the first `sinks`, the last of the
        # recent ones and some of those between
        seen = lens * 3 + 7
        order = torch.rand((B, H, room), generator=gen, device=DEVICE).argsort(-1)
        between = case["sinks"] + order * 2
        late = order >= lens[:, None, None] - case["recent"]
        s["positions"] = torch.where(order < case["sinks"], order, torch.where(
            late, seen[:, None, None] - lens[:, None, None] + order, between)).to(torch.int32)
        s["scores"] = torch.exp(2.5 * _normal(gen, B, H, room)) * 1e-3
        s["seen"] = seen.to(torch.int32)
        s.update(budget=room, sinks=case["sinks"], recent=case["recent"])
        return s
    T, G = case["tokens"], case["group"]
    per = -(-T // page)
    s["table"], pool = _table(gen, B, per)
    s["k"], s["v"] = _rows(gen, dtype, pool, H, page, dim), _normal(gen, pool, H, page, dim).to(dtype)
    s["lens"] = _lengths(gen, B, T, case["ragged"])
    s["starts"] = None
    if case["window"]:   # every second sequence attends its last rows only
        odd = torch.arange(B, device=DEVICE) % 2 == 1
        s["starts"] = torch.where(odd, (s["lens"] - case["window"]).clamp(min=0), 0).to(torch.int32)
    last = (s["lens"].long() - 1).clamp(min=0)
    at = (torch.rand((B, G), generator=gen, device=DEVICE) * last[:, None]).long()
    near = s["k"][s["table"].long().gather(1, at // page), :, at % page].float().transpose(1, 2)   # [B, H, G, dim]
    s["q"] = (_normal(gen, B, H, G, dim) + 0.35 * near).to(dtype).view(B, 1, H * G, dim)
    s["scores"] = torch.rand((B, H, T), generator=gen, device=DEVICE) if case["scored"] else None
    s["most"] = T
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return {"attend": _attend, "append": _append, "weigh": _weigh, "fill": _fill}[s["kind"]](s)


def _attend(s):
    if own:
        from retrievalattention_amd import kernels
        out, lse = kernels.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], starts=s["starts"],
                                           scores=s["scores"], max_len=s["most"], return_softmax_lse=True)
        return {"out": out, "lse": lse, "scores": s["scores"]}
    out, lse, p = _plain_attend(s)
    if s["scores"] is not None:
        s["scores"] += p.sum(2)
    return {"out": out, "lse": lse, "scores": s["scores"]}


def _plain_attend(s):
    _, H, page, dim = s["k"].shape
    B, T = s["q"].shape[0], s["most"]
    table = s["table"].long()
    rows = torch.arange(T, device=DEVICE)
    valid = rows < s["lens"][:, None]
    if s["starts"] is not None:
        valid = valid & (rows >= s["starts"][:, None])
    valid = valid[:, None, None]
    k = s["k"][table].transpose(1, 2).reshape(B, H, -1, dim)[:, :, :T].float()
    v = s["v"][table].transpose(1, 2).reshape(B, H, -1, dim)[:, :, :T].float()
    q = s["q"].view(B, H, -1, dim).float()
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * dim ** -0.5
    x = torch.where(valid, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    out = torch.matmul(p, torch.where(valid.transpose(-1, -2), v, 0.0))
    return out.to(s["q"].dtype).view(s["q"].shape), (m + torch.log(total)).view(B, -1), p


def _append(s):
    if own:
        from retrievalattention_amd import kernels
        kernels.paged_append(s["key"], s["value"], s["k"], s["v"], s["table"], s["lens"], s["held"], scores=s["scores"],
                             positions=s["positions"], token_positions=s["seen"], budget=s["budget"], sinks=s["sinks"],
                             recent=s["recent"])
    else:
        _plain_append(s)
    return {"k": s["k"], "v": s["v"], "scores": s["scores"], "positions": s["positions"], "held": s["held"]}


def _plain_append(s):
    H, page = s["k"].shape[1], s["k"].shape[2]
    lens, seen = s["lens"].long(), s["seen"].long()
    rows = torch.arange(s["scores"].shape[-1], device=DEVICE)
    held = s["positions"].long()
    free = (rows < lens[:, None, None]) & (held >= s["sinks"]) & (held <= seen[:, None, None] - s["recent"])
    x = torch.where(free, s["scores"], math.inf)
    weakest = torch.where(x == x.amin(-1, keepdim=True), rows, rows.shape[0]).amin(-1)
    row = torch.where(lens[:, None] < s["budget"], lens[:, None], weakest)          # [B, H]
    heads = torch.arange(H, device=DEVICE)
    at = s["table"].long().gather(1, row // page)
    s["k"][at, heads, row % page] = s["key"][:, 0]
    s["v"][at, heads, row % page] = s["value"][:, 0]
    s["scores"].scatter_(2, row[..., None], 0.0)
    s["positions"].scatter_(2, row[..., None], s["seen"][:, None, None].expand(-1, H, 1))
    s["held"].copy_((s["lens"] + 1).clamp(max=s["budget"]))


def _weigh(s):
    if own:
        from retrievalattention_amd import kernels
        return kernels.attention_weights(s["q"], s["key"], seqlens=s["lens"])
    return _plain_weigh(s)


def _plain_weigh(s):
    B, W, _, dim = s["q"].shape
    T, H = s["key"].shape[1], s["key"].shape[2]
    lens = torch.full((B,), T, device=DEVICE) if s["lens"] is None else s["lens"].long()
    q = s["q"].float().view(B, W, H, -1, dim).permute(0, 2, 3, 1, 4).reshape(B, H, -1, dim)
    x = torch.matmul(q, s["key"].float().permute(0, 2, 3, 1).contiguous()).view(B, H, -1, W, T) * dim ** -0.5
    at = lens[:, None] - W + torch.arange(W, device=DEVICE)              # [B, W]
    seen = (torch.arange(T, device=DEVICE) <= at[..., None])[:, None, None]
    x = torch.where(seen, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    total = x.sum(-1, keepdim=True)
    return x.div_(torch.where(total > 0, total, 1.0)).sum((2, 3))


def _fill(s):
    if own:
        from retrievalattention_amd import kernels
        kernels.paged_fill(s["key"], s["value"], s["k"], s["v"], s["table"], s["held"], seqlens=s["lens"],
                           weights=s["weights"], scores=s["scores"], positions=s["positions"], budget=s["budget"] or None,
                           sinks=s["sinks"], recent=s["recent"])
    else:
        _plain_fill(s)
    return {"k": s["k"], "v": s["v"], "scores": s["scores"], "positions": s["positions"], "held": s["held"]}


def _plain_fill(s):
    B, T, H, _ = s["key"].shape
    page = s["k"].shape[2]
    lens = torch.full((B,), T, device=DEVICE) if s["lens"] is None else s["lens"].long()
    budget = s["budget"] or T
    rows = torch.arange(T, device=DEVICE)
    inside = (rows < lens[:, None])[:, None].expand(B, H, T)
    keep = inside
    if s["budget"]:
        always = (rows < s["sinks"]) | (rows >= (lens - s["recent"])[:, None])
        x = torch.where(always[:, None], math.inf, s["weights"])
        x = torch.where(inside, x, -math.inf)
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices
        keep = inside & torch.zeros_like(inside).scatter(2, order[..., :budget], True)
    b, h, t = keep.nonzero(as_tuple=True)
    row = (keep.cumsum(-1) - 1)[b, h, t]
    at = s["table"].long()[b, row // page]
    s["k"][at, h, row % page] = s["key"][b, t, h]
    s["v"][at, h, row % page] = s["value"][b, t, h]
    if s["scores"] is not None:
        s["scores"][b, h, row] = s["weights"][b, h, t]
        s["positions"][b, h, row] = t.to(torch.int32)
    s["held"].copy_(lens.clamp(max=budget))


# ------------------------------------------------------------------------------------------------ cost
def _all_lengths(case):
    """Lengths as a host list of the case's typical shares: ragged ones are spread over the logarithm, of which the mean
    is (n - 1) / ln n."""
    n, B = case["tokens"], case["batch"]
    return [n] * B if not case["ragged"] else [n] + [n / math.log(n + 2)] * (B - 1)


def work(case):
    """Bytes and operations of one pass: every input that the result depends on read once, every output written once."""
    row, H, B = 2 * case["dim"], case["heads"], case["batch"]
    if case["kind"] == "attend":
        rows = sum(min(n, case["window"]) if case["window"] and b % 2 else n for b, n in enumerate(_all_lengths(case)))
        heads = H * case["group"]
        return {"bytes": rows * H * (2 * row + (8 if case["scored"] else 0)) + B * heads * (2 * row + 4) + rows / case["page"] * 4,
                "flops": 4 * rows * heads * case["dim"]}
    if case["kind"] == "append":   # scores and positions of the rows, the new rows read and written
        return {"bytes": B * H * ((0.8 if case["ragged"] else 1.0) * case["budget"] * 8 + 4 * row + 8), "flops": 0}
    if case["kind"] == "weigh":
        keys = pairs = 0
        for n in _all_lengths(case):
            w = min(case["window"], n)
            keys += n
            pairs += w * n - w * (w - 1) / 2
        return {"bytes": keys * H * (row + 4) + B * case["window"] * H * case["group"] * row,
                "flops": 2 * pairs * H * case["group"] * case["dim"]}
    bytes_ = 0
    for n in _all_lengths(case):
        kept = min(n, case["budget"] or n)
        bytes_ += kept * H * 4 * row + (H * (n * 4 + kept * 8) if case["budget"] else 0)
    return {"bytes": bytes_, "flops": 0}


# ------------------------------------------------------------------------------------------------ definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "weigh": _exact_weigh, "fill": _exact_fill}[s["kind"]](s)


def _exact_attend(s):
    B, _, heads, dim = s["q"].shape
    H, page = s["k"].shape[1], s["k"].shape[2]
    out = torch.zeros((B, 1, heads, dim), dtype=torch.float64, device=DEVICE)
    lse = torch.full((B, heads), -math.inf, dtype=torch.float64, device=DEVICE)
    scores = None if s["scores"] is None else s["scores"].double()
    starts = [0] * B if s["starts"] is None else s["starts"].tolist()
    for b, n in enumerate(s["lens"].tolist()):
        rows = torch.arange(starts[b], n, device=DEVICE)
        if not rows.numel():
            continue
        at = s["table"][b].long()[rows // page]
        for h in range(H):
            mine = slice(h * heads // H, (h + 1) * heads // H)
            k, v = s["k"][at, h, rows % page].double(), s["v"][at, h, rows % page].double()
            x = (k @ s["q"][b, 0, mine].double().T.contiguous()) / math.sqrt(dim)      # [rows, heads]
            lse[b, mine] = torch.logsumexp(x, 0)
            p = torch.softmax(x, 0)
            out[b, 0, mine] = (p[..., None] * v[:, None]).sum(0) if rows.numel() < 64 else p.T.contiguous() @ v
            if scores is not None:
                scores[b, h, rows] += p.sum(1)
    return {"out": out, "lse": lse, "scores": scores}


def _exact_append(s):
    k, v, scores, positions = s["k"].double(), s["v"].double(), s["scores"].double(), s["positions"].clone()
    page, budget = s["k"].shape[2], s["budget"]
    lens, seen = s["lens"].tolist(), s["seen"].tolist()
    host_scores, host_positions, table = s["scores"].double().cpu().numpy(), s["positions"].cpu().numpy(), s["table"].tolist()
    for b, n in enumerate(lens):
        for h in range(k.shape[1]):
            r = n
            if n >= budget:
                at = host_positions[b, h, :n]
                ok = ((at >= s["sinks"]) & (at <= seen[b] - s["recent"])).nonzero()[0]
                r = int(ok[host_scores[b, h, :n][ok].argmin()]) if ok.size else 0
            p = table[b][r // page]
            k[p, h, r % page], v[p, h, r % page] = s["key"][b, 0, h].double(), s["value"][b, 0, h].double()
            scores[b, h, r], positions[b, h, r] = 0.0, seen[b]
    held = torch.tensor([min(n + 1, budget) for n in lens], dtype=torch.int32, device=DEVICE)
    return {"k": k, "v": v, "scores": scores, "positions": positions, "held": held}


def _exact_weigh(s):
    B, W, heads, dim = s["q"].shape
    T, H = s["key"].shape[1], s["key"].shape[2]
    out = torch.zeros((B, H, T), dtype=torch.float64, device=DEVICE)
    lens = [T] * B if s["lens"] is None else s["lens"].tolist()
    for b, n in enumerate(lens):
        w = min(W, n)
        if not w:
            continue
        later = torch.arange(n, device=DEVICE)[None] > torch.arange(n - w, n, device=DEVICE)[:, None]
        for i in range(heads):
            h = i * H // heads
            x = s["q"][b, W - w:, i].double() @ s["key"][b, :n, h].double().T.contiguous()
            out[b, h, :n] += torch.softmax((x / math.sqrt(dim)).masked_fill_(later, -math.inf), 1).sum(0)
    return out


def _exact_fill(s):
    k, v = s["k"].double(), s["v"].double()
    scores = None if s["scores"] is None else s["scores"].double()
    positions = None if s["positions"] is None else s["positions"].clone()
    B, T, H, _ = s["key"].shape
    page = s["k"].shape[2]
    lens = [T] * B if s["lens"] is None else s["lens"].tolist()
    budget = s["budget"] or T
    for b, n in enumerate(lens):
        for h in range(H):
            kept = torch.arange(n, device=DEVICE)
            if n > budget:
                free = kept[s["sinks"]:n - s["recent"]]
                w = s["weights"][b, h, free].double()
                first = torch.argsort(-w, stable=True)[:budget - s["sinks"] - s["recent"]]
                kept = torch.cat((kept[:s["sinks"]], free[first].sort().values, kept[n - s["recent"]:]))
            r = torch.arange(kept.numel(), device=DEVICE)
            at = s["table"][b].long()[r // page]
            k[at, h, r % page], v[at, h, r % page] = s["key"][b, kept, h].double(), s["value"][b, kept, h].double()
            if scores is not None:
                scores[b, h, r] = s["weights"][b, h, kept].double()
                positions[b, h, r] = kept.to(torch.int32)
    held = torch.tensor([min(n, budget) for n in lens], dtype=torch.int32, device=DEVICE)
    return {"k": k, "v": v, "scores": scores, "positions": positions, "held": held}
