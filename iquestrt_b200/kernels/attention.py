"""The attention between the prologue and the o_proj of a decode layer, over a paged KV cache
whose bookkeeping lives on the device: a captured step finds its own cache rows, positions
and lengths, attends, and (with a budget) evicts, so that replaying it decodes token after
token.  The reference's counterpart is its online split-KV attention over flat caches and
sliding-window rings (iquestrt/kernels/attention.py:40-57, iquestrt/kv.py:57-66)."""

import contextlib

import torch

from .. import ops


class PagedKvCache:
    """The paged keys and values of `batch` sequences for `layers` layers of a rank, and what a
    step needs to know about them.

    Row j of sequence b lies in page `page_table[b, j // page_size]` of every layer's caches;
    the default table gives each sequence the pages it needs for `rows` rows, in order (pass
    `page_table` and `capacity` to place them otherwise; sequences that are cut to a budget
    must not share pages).  `lengths` counts the rows held, `seen` the tokens seen; with a
    `budget` each layer also keeps every row's accumulated attention weight and position, and
    `evict` cuts sequences that have grown past it.  `rows` must leave room for the step's
    `q_len` tokens above the budget."""

    def __init__(self, layers: int, batch: int, kv_heads: int, head_dim: int, *, rows: int,
                 q_len: int = 1, page_size: int = 64, dtype=torch.float8_e4m3fn, device="cuda",
                 page_table=None, capacity: int | None = None, budget: int | None = None,
                 keep_first: int = 4, keep_last: int = 0, scratch=None):
        if not 1 <= q_len <= 8:
            raise ValueError(f"q_len must be 1..8, got {q_len}")
        if min(layers, batch, kv_heads, head_dim, rows, page_size) < 1:
            raise ValueError(f"sizes must be at least 1, got {layers} layers, batch {batch}, "
                             f"{kv_heads} heads of {head_dim}, {rows} rows, pages of {page_size}")
        if dtype not in (torch.bfloat16, torch.float8_e4m3fn):
            raise ValueError(f"the KV cache must be bf16 or e4m3, got {dtype}")
        if budget is not None and not 1 <= budget <= rows - q_len:
            raise ValueError(f"a budget of {budget} rows and {q_len} new ones need more than "
                             f"{rows} rows")
        if budget is not None and (min(keep_first, keep_last) < 0
                                   or keep_first + keep_last > budget):
            raise ValueError(f"a budget of {budget} rows does not hold the protected ones, "
                             f"{keep_first} + {keep_last}")
        pages = -(-rows // page_size)
        if page_table is None:
            page_table = torch.arange(batch * pages, dtype=torch.int32).view(batch, pages)
            capacity = batch * pages * page_size
        elif capacity is None:
            raise ValueError("a page table needs the caches' capacity")
        elif page_table.dim() != 2 or page_table.shape[0] != batch \
                or page_table.shape[1] * page_size < rows:
            raise ValueError(f"page_table {tuple(page_table.shape)} does not give {batch} sequences "
                             f"{rows} rows each in pages of {page_size}")
        self.batch, self.q_len, self.kv_heads, self.head_dim = batch, q_len, kv_heads, head_dim
        self.page_size, self.capacity = page_size, capacity
        self.budget, self.keep_first, self.keep_last = budget, keep_first, keep_last
        self.page_table = page_table.to(device=device, dtype=torch.int32).contiguous()
        self.rows = self.page_table.shape[1] * page_size
        dev = self.page_table.device
        shape = (capacity, kv_heads, head_dim)
        self.k = [torch.zeros(shape, dtype=dtype, device=dev) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=dev) for _ in range(layers)]
        ints = dict(dtype=torch.int32, device=dev)
        # rows held between steps, and with the step's tokens (one buffer without a budget)
        self.held = torch.zeros(batch, **ints)
        self.lengths = self.held if budget is None else torch.zeros(batch, **ints)
        self.seen = torch.zeros(batch, **ints)
        self.slot = torch.zeros(batch * q_len, dtype=torch.int64, device=dev)
        self.pos = torch.zeros(batch * q_len, dtype=torch.int64, device=dev)
        self.weights = self.positions = None
        if budget is not None:
            self.weights = [torch.zeros(batch, kv_heads, self.rows, device=dev)
                            for _ in range(layers)]
            self.positions = [torch.zeros(batch, kv_heads, self.rows, **ints)
                              for _ in range(layers)]
            self._evict_work = ops.EvictWork(batch=batch, kv_heads=kv_heads, rows=self.rows,
                                             device=dev)
        self._scratch = scratch

    @property
    def scratch(self):
        if self._scratch is None:
            self._scratch = ops.default_scratch(self.held.device)
        return self._scratch

    def set_lengths(self, lengths, seen=None, *, positions=None, weights=None) -> None:
        """Declares the rows already written (a prompt's) per sequence, and the tokens seen (as
        many, where nothing was evicted before).  Between steps only.

        With a budget the rows' positions and accumulated weights start anew: `positions` and
        `weights` are a tensor `[batch, kv_heads, rows]` a layer (int32, fp32; fewer rows will do
        if they hold the longest sequence).  Without `positions` row j is token j, which is so
        only where nothing was evicted; without `weights` every row starts at 0, and of rows that
        no step's attention has told apart the later go first.  The cache's own tensors
        (`cache.positions`, `cache.weights`) say that they are filled already."""
        n = torch.as_tensor(lengths, dtype=torch.int32).cpu()
        if n.shape != (self.batch,) or int(n.min()) < 0 or int(n.max()) > self.rows:
            raise ValueError(f"lengths must be [{self.batch}] within 0..{self.rows}, got "
                             f"{n.tolist()}")
        s = n if seen is None else torch.as_tensor(seen, dtype=torch.int32).cpu()
        if s.shape != (self.batch,) or bool((s < (0 if self.budget is None else n)).any()):
            raise ValueError(f"seen must be [{self.batch}], not negative and (with a budget) no less "
                             f"than the rows {n.tolist()}, got {s.tolist()}")
        if self.budget is None:
            if positions is not None or weights is not None:
                raise ValueError("positions and weights are kept with a budget only")
        else:
            if positions is None and not torch.equal(s, n):
                raise ValueError("sequences that have seen more tokens than they hold need their "
                                 "rows' positions")
            for name, given, kept in (("positions", positions, self.positions),
                                      ("weights", weights, self.weights)):
                self._check_state(name, given, kept, int(n.max()))
        self.held.copy_(n)
        self.seen.copy_(s)
        if self.budget is None:
            return
        order = torch.arange(self.rows, dtype=torch.int32, device=self.held.device)
        for i, (p, w) in enumerate(zip(self.positions, self.weights)):
            if positions is None:
                p.copy_(order.expand_as(p))
            elif positions[i] is not p:
                p[..., :positions[i].shape[2]].copy_(positions[i])
            if weights is None:
                w.zero_()
            elif weights[i] is not w:
                w[..., :weights[i].shape[2]].copy_(weights[i])

    def _check_state(self, name, given, kept, longest) -> None:
        if given is None:
            return
        if len(given) != len(kept):
            raise ValueError(f"{name} must be a tensor for each of {len(kept)} layers, got {len(given)}")
        for x in given:
            if not isinstance(x, torch.Tensor) or x.dtype != kept[0].dtype or x.dim() != 3 \
                    or x.shape[:2] != kept[0].shape[:2] or not longest <= x.shape[2] <= self.rows:
                what = f"{tuple(x.shape)} {x.dtype}" if isinstance(x, torch.Tensor) else type(x)
                raise ValueError(f"{name} must be [{self.batch}, {self.kv_heads}, {longest}.."
                                 f"{self.rows}] {kept[0].dtype} tensors, got {what}")

    @contextlib.contextmanager
    def rehearsal(self):
        """What runs inside, on the current stream, leaves the cache as it was: the warm-up step
        before a capture.  The sequences hold nothing meanwhile, and the rows of the steps' first
        tokens are the caches' first ones for all of them, so that these rows are all there is
        to put back (sequences that overwrite one another's change nothing but these).  The
        capture itself goes outside: inside, the page table is another."""
        table = self.page_table
        rows = min(self.q_len, self.page_size, self.capacity)
        kept = [self.held, self.lengths, self.seen, self.slot, self.pos]
        kept += [x[:rows] for x in self.k + self.v]
        if self.budget is not None:
            kept += [x[..., :self.q_len] for x in self.weights + self.positions]
        was = [x.clone() for x in kept]
        self.page_table = torch.zeros_like(table)
        self.held.zero_()
        self.seen.zero_()
        try:
            yield self
        finally:
            self.page_table = table
            for x, y in zip(kept, was):
                x.copy_(y)

    def advance(self, *, max_positions: int = 0, pdl: bool = False) -> None:
        """Rows and positions of the step's tokens into `slot` / `pos`; `lengths` and `seen`
        count them from here on.  A sequence without room for them (or that would reach
        `max_positions`) keeps its rows, counts, weights and positions, and the scratch's status
        word says so; the step's outputs for it mean nothing."""
        ops.kv_advance(self.page_table, self.held, self.seen, self.slot, self.pos,
                       page_size=self.page_size, capacity=self.capacity, q_len=self.q_len,
                       max_positions=max_positions, lengths_out=self.lengths, scratch=self.scratch, pdl=pdl)

    def evict(self, layer: int, *, pdl: bool = False) -> None:
        """Cuts `layer`'s sequences back to the budget, after the step's attention; `held` gets
        the lengths they then have (the same for every layer)."""
        ops.kv_evict(self.k[layer], self.v[layer], self.page_table, self.lengths,
                     self.weights[layer], self.positions[layer], self.seen,
                     page_size=self.page_size, budget=self.budget, keep_first=self.keep_first,
                     keep_last=self.keep_last, lengths_out=self.held, work=self._evict_work,
                     scratch=self.scratch, pdl=pdl)


class PagedAttention:
    """Attention of a step's rows over a `PagedKvCache`: q `[batch * q_len, q_heads, D]` (what
    `PrologueKernels` returns) -> `[batch * q_len, q_heads * D]` bf16 (what `OProjGemv` takes),
    in one arena slot.  `window` > 0: sliding-window attention, over a cache without a budget
    only: the window counts rows, and eviction gives up their order."""

    def __init__(self, q_heads: int, cache: PagedKvCache, *, ws, window: int = 0, scale=None):
        if q_heads % cache.kv_heads:
            raise ValueError(f"{q_heads} query heads do not share {cache.kv_heads} key/value heads")
        if window < 0:
            raise ValueError(f"window must not be negative, got {window}")
        if window and cache.budget is not None:
            raise ValueError("a sliding window needs a cache without a budget: eviction does not "
                             "keep the rows in the order of their tokens")
        self.q_heads, self.cache, self.window, self.scale = q_heads, cache, window, scale
        rows, d = cache.batch * cache.q_len, cache.head_dim
        self.out = ws.slot(("attention", "out"), (rows, q_heads * d), torch.bfloat16)
        self.work = ops.AttnWork(batch=cache.batch, q_len=cache.q_len, q_heads=q_heads,
                                 kv_heads=cache.kv_heads, head_dim=d, rows=cache.rows,
                                 weights=cache.weights is not None, device=cache.held.device)

    def __call__(self, q, layer: int, *, pdl: bool = False):
        c = self.cache
        shape = (c.batch, c.q_len, self.q_heads, c.head_dim)
        more = {}
        if c.weights is not None:
            more = dict(weights=c.weights[layer], positions=c.positions[layer], seen=c.seen,
                        slot=c.slot)
        ops.attn_decode(q.view(shape), c.k[layer], c.v[layer], c.page_table, c.lengths,
                        page_size=c.page_size, scale=self.scale, window=self.window,
                        out=self.out.view(shape), work=self.work, scratch=c.scratch, pdl=pdl, **more)
        return self.out
