"""A paged key-value cache with eviction by accumulated attention weight (no counterpart in the reference; methods as those of
retroinfer_cache).

Each layer has a pool of pages [pages, kv heads, page_size, head_dim] for keys and one for values; a sequence holds as many pages as
its rows need, the same ones in every layer, through one block table.  With a `budget` a sequence keeps at most that many rows per
key-value head: of a longer prompt those to which the prompt's last `window` queries (None: all) give the most weight, and a
generated token then takes the place of the row with the least weight accumulated so far, the first `sinks` and the last `recent`
tokens excepted.  Heads keep different tokens, but equally many.

Everything that a step reads is on the device, so a captured step can be replayed token after token: call prepare_token() before
each replay, which hands out the pages that the token needs."""
import torch

from .. import kernels


class paged_cache:
    def __init__(self, layer_num, batch_size, max_length, num_key_value_heads, num_heads, head_dim, dtype, device, page_size=16,
                 budget=None, sinks=4, recent=64, window=64, pages=None):
        if page_size < 1 or page_size & (page_size - 1):
            raise ValueError("page_size: expected a power of two")
        if head_dim not in kernels.PAGED_DIMS:
            raise ValueError(f"head_dim: expected one of {kernels.PAGED_DIMS}")
        if num_heads % num_key_value_heads or num_heads // num_key_value_heads > kernels.MAX_GROUP_SIZE:
            raise ValueError(f"num_heads: expected 1 to {kernels.MAX_GROUP_SIZE} query heads to each key-value head")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("dtype: expected bfloat16 or float16")
        if budget is not None and (sinks < 0 or recent < 1 or sinks + recent >= budget):
            raise ValueError("budget: expected more than sinks + recent, and recent at least 1")
        if window is not None and window < 1:
            raise ValueError("window: expected at least one query")
        self.layer_num, self.batch_size, self.kv_head, self.num_heads = layer_num, batch_size, num_key_value_heads, num_heads
        self.head_dim, self.dtype, self.device = head_dim, dtype, torch.device(device)
        self.page_size, self.budget, self.sinks, self.recent, self.window = page_size, budget, sinks, recent, window
        self.max_length = max_length
        self.rows = max_length if budget is None else min(budget, max_length)   # of a sequence at most
        if budget is not None and self.rows < budget:   # nothing is ever evicted
            self.budget = None
        per = -(-self.rows // page_size)
        pages = batch_size * per if pages is None else pages
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=self.device)  # noqa: E731
        shape = (pages, num_key_value_heads, page_size, head_dim)
        self.k_pages = [torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(layer_num)]
        self.v_pages = [torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(layer_num)]
        self.block_table = torch.full((batch_size, per), -1, dtype=torch.int32, device=self.device)
        self.seqlens, self.new_seqlens = i32(batch_size), i32(batch_size)   # rows in use before and with the token being decoded
        self.seen, self.active = i32(batch_size), i32(batch_size)           # tokens of a sequence so far; whether it is one
        self.scores = self.positions = [None] * layer_num
        if self.budget is not None:
            shape = (batch_size, num_key_value_heads, self.rows)
            self.scores = [torch.zeros(shape, device=self.device) for _ in range(layer_num)]
            self.positions = [i32(*shape) for _ in range(layer_num)]
        self._table = [[] for _ in range(batch_size)]    # the host's copies
        self._rows = [0] * batch_size
        self._free = list(range(pages - 1, -1, -1))
        self._scratch = kernels.Scratch()

    @property
    def context(self):
        """Rows in use of the longest sequence."""
        return max(self._rows)

    @property
    def free_pages(self):
        return len(self._free)

    # ------------------------------------------------------------------ pages
    def _take(self, wanted):
        """Pages for `wanted` {sequence: rows}; all of them or none."""
        more = {b: -(-rows // self.page_size) - len(self._table[b]) for b, rows in wanted.items()}
        if sum(n for n in more.values() if n > 0) > len(self._free):
            raise RuntimeError(f"paged_cache: {sum(n for n in more.values() if n > 0)} pages wanted, {len(self._free)} free")
        for b, n in more.items():
            if n > 0:
                self._table[b] += [self._free.pop() for _ in range(n)]
                row = self._table[b]
                self.block_table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
        for b, rows in wanted.items():
            self._rows[b] = rows

    def release(self, batch_idx):
        """Ends a sequence: its pages can be handed out again, its place takes the next prompt."""
        self._free += self._table[batch_idx]
        self._table[batch_idx], self._rows[batch_idx] = [], 0
        self.block_table[batch_idx] = -1
        for t in (self.seqlens, self.new_seqlens, self.seen, self.active):
            t[batch_idx] = 0

    def prepare_token(self):
        """The pages of the next token of every sequence.  decode_update_kv_cache calls it, except during a stream capture: call
        it before each replay of a captured token."""
        if self.budget is None and any(self._table[b] and n >= self.rows for b, n in enumerate(self._rows)):
            raise RuntimeError(f"paged_cache: a sequence has {self.rows} rows, all that it was built for")
        self._take({b: min(n + 1, self.rows) for b, n in enumerate(self._rows) if self._table[b]})

    def _rows_of(self, t, batch, tokens, heads, name):
        """Refuses what the kernels would refuse of a layer's rows [batch, tokens, heads, head_dim] before pages are handed out for them."""
        kernels._strided(t, 4, self.dtype, self.block_table.device, name)
        if t.shape != (batch, tokens, heads, self.head_dim):
            raise ValueError(f"{name}: expected [{batch}, {tokens}, {heads}, {self.head_dim}]")

    # ------------------------------------------------------------------ prompt
    def prefill_update_kv_cache(self, query_states, key_states, value_states, layer_idx, batch_idx):
        """One sequence's prompt in one layer: query [1, T, heads, dim] (only read with a budget), key and value [1, T, kv heads,
        dim].  Returns key and value as they came, for the prompt's own attention."""
        if not isinstance(key_states, torch.Tensor) or key_states.dim() != 4:
            raise ValueError("paged_cache: expected key [1, T, kv heads, head_dim]")
        T, b = key_states.shape[1], batch_idx
        if not 0 <= b < self.batch_size or T < 1 or key_states.shape[0] != 1:
            raise ValueError(f"paged_cache: expected a prompt [1, 1 token or more, ..] and a place below {self.batch_size}")
        if layer_idx == 0:
            self._rows_of(key_states, 1, T, self.kv_head, "key_states")
            self._rows_of(value_states, 1, T, self.kv_head, "value_states")
            if self.budget is not None:
                heads = query_states.shape[2] if isinstance(query_states, torch.Tensor) and query_states.dim() == 4 else 0
                if heads % self.kv_head or not 1 <= heads // self.kv_head <= kernels.MAX_GROUP_SIZE:
                    raise ValueError(f"query_states: expected 1 to {kernels.MAX_GROUP_SIZE} heads to each key-value head")
                self._rows_of(query_states, 1, T, heads, "query_states")
            if self.budget is None and T > self.rows:
                raise ValueError(f"paged_cache: a prompt of {T} tokens, built for {self.rows}")
            wanted = -(-min(T, self.rows) // self.page_size)
            if wanted > len(self._free) + len(self._table[b]):
                raise RuntimeError(f"paged_cache: {wanted} pages wanted, {len(self._free)} free")
            if self._table[b]:   # the place's last sequence ends
                self.release(b)
            self._take({b: min(T, self.rows)})
            self.seen[b], self.active[b] = T, 1
        weights = None
        if self.budget is not None:
            window = T if self.window is None else min(T, self.window)
            weights = kernels.attention_weights(query_states[:, T - window:], key_states, scratch=self._scratch)
        one = slice(b, b + 1)
        kernels.paged_fill(key_states, value_states, self.k_pages[layer_idx], self.v_pages[layer_idx], self.block_table[one],
                           self.seqlens[one], weights=weights, **self._per_row(layer_idx, one), **self._keep(), scratch=self._scratch)
        return key_states, value_states

    def _keep(self):
        return {} if self.budget is None else dict(budget=self.budget, sinks=self.sinks, recent=self.recent)

    def _per_row(self, layer_idx, part=slice(None)):
        if self.budget is None:
            return {}
        return dict(scores=self.scores[layer_idx][part], positions=self.positions[layer_idx][part])

    # ------------------------------------------------------------------ tokens
    def decode_update_kv_cache(self, key_states, value_states, layer_idx):
        """The next token's key and value [B, 1, kv heads, dim] in one layer."""
        if layer_idx == 0 and not torch.cuda.is_current_stream_capturing():
            self._rows_of(key_states, self.batch_size, 1, self.kv_head, "key_states")
            self._rows_of(value_states, self.batch_size, 1, self.kv_head, "value_states")
            self.prepare_token()
        kernels.paged_append(key_states, value_states, self.k_pages[layer_idx], self.v_pages[layer_idx], self.block_table,
                             self.seqlens, self.new_seqlens, **self._per_row(layer_idx),
                             token_positions=None if self.budget is None else self.seen, **self._keep())
        return key_states, value_states

    def compute(self, query_states, layer_idx):
        """The token's attention [B, 1, heads, dim] in one layer; the last layer's call moves the sequences on by the token."""
        out = kernels.paged_attention(query_states, self.k_pages[layer_idx], self.v_pages[layer_idx], self.block_table,
                                      self.new_seqlens, scores=self.scores[layer_idx], max_len=self.rows, scratch=self._scratch)
        if layer_idx == self.layer_num - 1:
            torch.mul(self.new_seqlens, self.active, out=self.seqlens)   # (places without a sequence stay empty)
            self.seen.add_(self.active)
        return out
