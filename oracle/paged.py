"""The paged cache's operators in 64 bits, one sequence and head at a time, and the sizes that errors are counted in."""
import math

import torch


def rows_of(pages, table_row, rows):
    """[heads, n, dim] of the given rows of a sequence, in 64 bits, and which of them there are."""
    page_rows = pages.shape[2]
    page = table_row.long()[rows // page_rows]
    there = (page >= 0) & (page < pages.shape[0])
    got = pages[page.clamp(0, pages.shape[0] - 1), :, rows % page_rows].double()    # [n, heads, dim]
    return got.transpose(0, 1), there


def attention(q, k_pages, v_pages, table, lens, starts, scale):
    """out, lse, weights [B, heads, rows] and, of each output, the sum of p |v| and, of each row, the sum of |q k| scale."""
    B, _, hq, dim = q.shape
    heads, room = k_pages.shape[1], table.shape[1] * k_pages.shape[2]
    gs = hq // heads
    out, absolute = torch.zeros(B, 1, hq, dim).double(), torch.zeros(B, 1, hq, dim).double()
    lse = torch.full((B, hq), -math.inf).double()
    weights, size = torch.zeros(B, hq, room).double(), torch.zeros(B, hq).double()
    for b in range(B):
        n = min(max(int(lens[b]), 0), room)
        first = 0 if starts is None else min(max(int(starts[b]), 0), n)
        rows = torch.arange(first, n)
        k, there = rows_of(k_pages, table[b], rows)
        v, _ = rows_of(v_pages, table[b], rows)
        rows, k, v = rows[there], k[:, there], v[:, there]
        if not rows.numel():
            continue
        for i in range(hq):
            x = (k[i // gs] * q[b, 0, i].double()).sum(-1) * scale
            p = torch.softmax(x, 0)
            out[b, 0, i], absolute[b, 0, i] = p @ v[i // gs], p @ v[i // gs].abs()
            lse[b, i] = torch.logsumexp(x, 0)
            weights[b, i, rows] = p
            size[b, i] = ((k[i // gs] * q[b, 0, i].double()).abs().sum(-1) * scale).max()
    return out, lse, weights, absolute, size


def weigh(q, key, lens, scale):
    """[B, heads, T] and, of each, the largest sum of |q k| scale of its sequence and head."""
    B, W, hq, dim = q.shape
    T, heads = key.shape[1:3]
    gs = hq // heads
    out, size = torch.zeros(B, heads, T).double(), torch.zeros(B, heads, 1).double()
    for b in range(B):
        n = T if lens is None else min(max(int(lens[b]), 0), T)
        for i in range(W):
            last = n - W + i
            if last < 0:
                continue
            for j in range(hq):
                k, x = key[b, :last + 1, j // gs].double(), q[b, i, j].double()
                out[b, j // gs, :last + 1] += torch.softmax((k * x).sum(-1) * scale, 0)
                size[b, j // gs] = max(float(size[b, j // gs]), float((k * x).abs().sum(-1).max() * scale))
    return out, size


def order(x):
    """Sort key of a score: NaN above everything."""
    x = float(x)
    return (1, 0.0) if math.isnan(x) else (0, x)


def victim(scores, positions, n, token, sinks, recent):
    """The row of a full head that a new token takes."""
    free = [r for r in range(n) if sinks <= int(positions[r]) <= token - recent]
    return min(free, key=lambda r: (order(scores[r]), r)) if free else 0


def kept(weights, n, budget, sinks, recent):
    """The rows of a prompt of n tokens that a head keeps."""
    if n <= budget:
        return list(range(n))
    free = sorted(range(sinks, n - recent), key=lambda r: tuple(-x for x in order(weights[r])) + (r,))
    return sorted(list(range(sinks)) + free[:budget - sinks - recent] + list(range(n - recent, n)))
