"""The cache manager: pages of keys and values with a block table per request, and slots of
fixed-size state per request.

The model's mixers say what they need (`PagedKVNeed`, `StateNeed`). Schedule entries with the
same need form a *group*: a group of paged needs owns one pool tensor
`[layers of the group, 2 (K, V), pages + 1, kv_heads, page_tokens, head_dim]` and one page
allocator, and every request has one block table per group. (The reference has a single pool
for its one kind of layer, layover/kv/paged_cache.py:26-49, laid out block-major for its swap
path; here a page of one head is a contiguous run of page_tokens * head_dim elements per
layer, which is what the attention kernels read.) The last page of each pool is a scratch page
that is never handed out: padded rows of a captured decode step and table entries whose page
was given back point at it.

A group with a window only keeps the pages that a later query can still see: after a step,
pages that lie wholly below `tokens - window + 1` go back to the free list and are reused; where the
window keeps a sequence's first tokens visible (`keep_first`), the pages that hold them stay. A group
with a chunked mask (a query sees only the keys of its own chunk of positions) gives back the pages
that lie wholly before the chunk of the next token.
State groups own `[slots + 1, *shape]`; a request's slot is zeroed when it is opened.
A group whose values are the leading channels of its keys (`values_in_keys`) has one store, not two.
A mixer made of several mixers names several needs (a tuple); its view is a composite of their views.

A request can be *forked* (`fork`): its full pages are shared, which nobody writes any more, and the page that is
still being written, the state and the record are copied on the device. After a step over drafted tokens `accept`
moves the rows of those that are kept to the places behind what the request holds and gives back the pages behind them.

Beside the mixers' state every request has one *record* of `record_words` int32 words on the
device, `records[slot]`, written whole when the request is opened and never touched by the host
again: kernels index it by the request's slot, so a captured CUDA graph sees a fixed address.
What the words mean is the business of whoever writes and reads them (the sampler keeps the
request's seed, counter, temperature and last token there); the manager only hands out the row.
(The reference keeps such facts on the host, layover/engine.py:39-40; its nearest device-side
relative is the packed row at a fixed address of layover/decode_graphs.py:56-77.)

All bookkeeping is on the host and works without a device (`device=None` allocates no pools),
which is how the scheduler and the property tests use it.
"""

from __future__ import annotations

from collections import Counter
from dataclasses import dataclass, field

import torch

from ..parts.base import PagedKVNeed, StateNeed
from .allocator import BlockAllocator, OutOfBlocks


@dataclass
class PagedGroup:
    need: PagedKVNeed
    entries: list[int]                 # schedule entries that write into this group, in layer order
    allocator: BlockAllocator
    pool: torch.Tensor | None = None   # [layers, 2, pages + 1, kv_heads, page_tokens, head_dim]
    # where values have another size than keys the two cannot share a tensor: one pool each, `pool` stays None
    k_store: torch.Tensor | None = None  # [layers, pages + 1, kv_heads, page_tokens, head_dim]
    v_store: torch.Tensor | None = None  # [layers, pages + 1, kv_heads, page_tokens, v_head_dim]

    @property
    def scratch_page(self) -> int:
        return self.allocator.num_blocks


@dataclass
class StateGroup:
    need: StateNeed
    entries: list[int]
    pool: torch.Tensor | None = None   # [entries, slots + 1, *shape]


@dataclass
class CacheView:
    """What one schedule entry's mixer sees of the cache."""
    kind: str                          # "paged", "state", or "composite" (then only `parts` is set)
    group: int                         # index among the groups of its kind
    layer: int                         # index inside the group's pool
    writes: bool = True                # False when the entry reads another entry's keys and values
    k_pool: torch.Tensor | None = None # [pages + 1, kv_heads, page_tokens, head_dim]
    v_pool: torch.Tensor | None = None # [pages + 1, kv_heads, page_tokens, head_dim or the values' own size]
    pool: torch.Tensor | None = None   # the group's whole pool [layers, 2, pages + 1, kv_heads, page_tokens, head_dim]
                                       # (None where values have another size than keys)
    state: torch.Tensor | None = None  # [slots + 1, *shape]
    page_tokens: int = 0
    need: object = None
    parts: list | None = None          # a composite view: one view per need of the mixer, in its order


@dataclass
class BlockTable:
    """One request's pages in one group. Pages before index `first_live` (but not those that hold kept first
    tokens) were given back: `given_back` of them."""
    blocks: list[int] = field(default_factory=list)
    first_live: int = 0
    given_back: int = 0


@dataclass
class SequenceCache:
    """Everything the cache holds for one live request."""
    request_id: str
    slot: int
    tables: list[BlockTable]
    num_tokens: int = 0
    closed: bool = False
    # the parents of the drafts that the last step computed behind the held tokens (none: empty); None: no step has run yet
    drafts: list[int] | None = None


class CacheManager:
    def __init__(self, needs: list[tuple[int, object, int | None]], num_blocks: int, block_tokens: int = 16,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str | None = None,
                 max_requests: int = 64, record_words: int = 8):
        """`needs`: for every schedule entry (entry index, its need or None, the entry whose cache
        it reads instead of its own or None). `num_blocks` pages per paged group."""
        if block_tokens <= 0:
            raise ValueError("block_tokens must be positive")
        self.block_tokens = block_tokens
        self._num_blocks = num_blocks
        self.dtype = dtype
        self.device = None if device is None else torch.device(device)
        self.max_requests = max_requests
        self.paged: list[PagedGroup] = []
        self.states: list[StateGroup] = []
        self.views: dict[int, CacheView] = {}
        own = {entry: need for entry, need, reads in needs if reads is None and need is not None}
        for entry, need in own.items():
            if isinstance(need, (tuple, list)):
                self.views[entry] = CacheView("composite", -1, -1, parts=[self._own_view(entry, n) for n in need])
            else:
                self.views[entry] = self._own_view(entry, need)
        for entry, need, reads in needs:
            if reads is not None:
                if reads not in self.views or self.views[reads].kind != "paged":
                    raise ValueError(f"schedule entry {entry} reads the cache of entry {reads}, which has no pages")
                src = self.views[reads]
                self.views[entry] = CacheView("paged", src.group, src.layer, writes=False,
                                              page_tokens=block_tokens, need=src.need)
        self._slots = BlockAllocator(max_requests)
        self.live: dict[str, SequenceCache] = {}
        self.record_words = int(record_words)
        self.records: torch.Tensor | None = None     # [max_requests + 1, record_words] int32 on the device
        self._record_staging = None                  # the same rows in pinned host memory, and when each was last sent
        self._record_sent: list = [None] * (max_requests + 1)
        if self.device is not None:
            self._allocate_pools()

    def _own_view(self, entry: int, need) -> CacheView:
        """The view of one need of a schedule entry; needs that are equal share a group (and its pool)."""
        if isinstance(need, PagedKVNeed):
            group = next((g for g in self.paged if g.need == need), None)
            if group is None:
                group = PagedGroup(need, [], BlockAllocator(self._num_blocks))
                self.paged.append(group)
            group.entries.append(entry)
            return CacheView("paged", self.paged.index(group), len(group.entries) - 1, page_tokens=self.block_tokens, need=need)
        if isinstance(need, StateNeed):
            group = next((g for g in self.states if g.need == need), None)
            if group is None:
                group = StateGroup(need, [])
                self.states.append(group)
            group.entries.append(entry)
            return CacheView("state", self.states.index(group), len(group.entries) - 1, need=need)
        raise TypeError(f"schedule entry {entry}: unknown cache need {need!r}")

    def _all_views(self):
        for view in self.views.values():
            yield from (view.parts if view.kind == "composite" else [view])

    # ------------------------------------------------------------------ device memory
    def _allocate_pools(self) -> None:
        for group in self.paged:
            need = group.need
            shape = (group.allocator.num_blocks + 1, need.kv_heads, self.block_tokens)
            if getattr(need, "values_in_keys", False):
                group.k_store = torch.zeros((len(group.entries), *shape, need.head_dim), dtype=self.dtype, device=self.device)
            elif need.value_dim == need.head_dim:
                group.pool = torch.zeros((len(group.entries), 2, *shape, need.head_dim), dtype=self.dtype, device=self.device)
            else:
                group.k_store = torch.zeros((len(group.entries), *shape, need.head_dim), dtype=self.dtype, device=self.device)
                group.v_store = torch.zeros((len(group.entries), *shape, need.value_dim), dtype=self.dtype, device=self.device)
        for group in self.states:
            group.pool = torch.zeros((len(group.entries), self.max_requests + 1, *group.need.shape),
                                     dtype=group.need.dtype, device=self.device)
        self.records = torch.zeros((self.max_requests + 1, self.record_words), dtype=torch.int32, device=self.device)
        if self.device.type == "cuda":
            self._record_staging = torch.zeros((self.max_requests + 1, self.record_words), dtype=torch.int32,
                                               pin_memory=True)
        for view in self._all_views():
            if view.kind == "paged":
                group = self.paged[view.group]
                if group.pool is not None:
                    view.k_pool, view.v_pool, view.pool = group.pool[view.layer, 0], group.pool[view.layer, 1], group.pool
                elif group.v_store is None:       # the values are read from the keys' rows
                    view.k_pool = view.v_pool = group.k_store[view.layer]
                else:
                    view.k_pool, view.v_pool = group.k_store[view.layer], group.v_store[view.layer]
            else:
                view.state = self.states[view.group].pool[view.layer]

    def view(self, entry: int) -> CacheView | None:
        return self.views.get(entry)

    @property
    def scratch_slot(self) -> int:
        return self.max_requests

    @property
    def num_free_slots(self) -> int:
        return self._slots.num_free

    def pool_bytes(self) -> int:
        pools = [t for g in self.paged for t in (g.pool, g.k_store, g.v_store)] + [g.pool for g in self.states] + [self.records]
        return sum(p.numel() * p.element_size() for p in pools if p is not None)

    # ------------------------------------------------------------------ arithmetic
    def blocks_for(self, tokens: int) -> int:
        return -(-tokens // self.block_tokens)

    @property
    def num_blocks(self) -> int:
        return min((g.allocator.num_blocks for g in self.paged), default=0)

    @property
    def num_free(self) -> int:
        return min((g.allocator.num_free for g in self.paged), default=0)

    def _first_needed_page(self, group: PagedGroup, first_query: int) -> int:
        """Pages below this index (and past the kept first tokens' pages) hold no key that a query at
        `first_query` or later can see."""
        chunk = getattr(group.need, "chunk", None)
        if chunk:       # a query sees only its own chunk: everything before the chunk of `first_query` is done with
            return (first_query // chunk * chunk) // self.block_tokens
        if group.need.window is None:
            return 0
        return max(0, first_query - group.need.window + 1) // self.block_tokens

    def _kept_pages(self, group: PagedGroup) -> int:
        """Pages at the front of a table that hold first tokens which stay visible behind the window."""
        keep = getattr(group.need, "keep_first", 0) or 0
        return self.blocks_for(keep) if group.need.window is not None else 0

    def _dead(self, group: PagedGroup, first_query: int) -> tuple[int, int]:
        """[lo, hi): the page indices that no query at `first_query` or later can see."""
        lo = self._kept_pages(group)
        return lo, max(lo, self._first_needed_page(group, first_query))

    def peak_blocks(self, group_index: int, total_tokens: int, chunk: int) -> int:
        """The most pages of a group that a request of `total_tokens` holds at any time when it is
        fed at most `chunk` tokens a step."""
        group = self.paged[group_index]
        reach = getattr(group.need, "chunk", None) or group.need.window     # the most keys behind a query that stay visible
        if reach is None:
            return self.blocks_for(total_tokens)
        span = min(total_tokens, reach - 1 + max(1, chunk))
        return min(self.blocks_for(total_tokens), span // self.block_tokens + 2 + self._kept_pages(group))

    def blocks_missing(self, seq: SequenceCache, new_total: int) -> list[int]:
        """Per paged group: pages to allocate before tokens [seq.num_tokens, new_total) can be written."""
        out = []
        for group, table in zip(self.paged, seq.tables):
            lo, hi = self._dead(group, seq.num_tokens)
            have, want = len(table.blocks), self.blocks_for(new_total)
            dead = max(0, min(hi, want) - max(lo, have))          # new table entries that no query will read
            out.append(max(0, want - have - dead))
        return out

    # ------------------------------------------------------------------ life of a request
    def open(self, request_id: str, record: list[int] | None = None) -> SequenceCache:
        """A slot and empty tables for a new request. `record` (up to `record_words` int32 values, the
        rest zero) becomes the request's record on the device; the mixers' state of the slot is zeroed."""
        if request_id in self.live:
            raise ValueError(f"request {request_id!r} is already open")
        if record is not None and len(record) > self.record_words:
            raise ValueError(f"a record holds {self.record_words} words, got {len(record)}")
        try:
            slot = self._slots.alloc(1)[0]
        except OutOfBlocks:
            raise OutOfBlocks(f"all {self.max_requests} request slots are in use") from None
        for group in self.states:
            if group.pool is not None:
                group.pool[:, slot].zero_()
        if self.records is not None:
            words = torch.zeros(self.record_words, dtype=torch.int32)
            if record:
                words[: len(record)] = torch.tensor(record, dtype=torch.int64).to(torch.int32)
            if self._record_staging is not None:
                # stream-ordered behind every kernel that still uses the slot's previous owner
                if self._record_sent[slot] is not None:
                    self._record_sent[slot].synchronize()
                self._record_staging[slot] = words
                self.records[slot].copy_(self._record_staging[slot], non_blocking=True)
                self._record_sent[slot] = torch.cuda.Event()
                self._record_sent[slot].record()
            else:
                self.records[slot] = words
        seq = SequenceCache(request_id, slot, [BlockTable() for _ in self.paged])
        self.live[request_id] = seq
        return seq

    def grow(self, seq: SequenceCache, new_total: int) -> None:
        """Make room for tokens up to `new_total`, in every group or in none (OutOfBlocks)."""
        if seq.closed:
            raise ValueError(f"request {seq.request_id!r} is closed")
        missing = self.blocks_missing(seq, new_total)
        for group, count in zip(self.paged, missing):
            if count > group.allocator.num_free:
                raise OutOfBlocks(f"need {count} blocks, {group.allocator.num_free} free")
        for group, table in zip(self.paged, seq.tables):
            lo, hi = self._dead(group, seq.num_tokens)
            for index in range(len(table.blocks), self.blocks_for(new_total)):
                if lo <= index < hi:  # a page no query of this or a later step can see
                    table.blocks.append(group.scratch_page)
                    table.first_live = max(table.first_live, index + 1)
                    table.given_back += 1
                else:
                    table.blocks.append(group.allocator.alloc(1)[0])

    def commit(self, seq: SequenceCache, new_total: int) -> None:
        """The step that wrote tokens up to `new_total` has been issued: count them and give back
        the pages that a window has passed."""
        if new_total < seq.num_tokens:
            raise ValueError("a request's token count cannot shrink")
        if any(self.blocks_for(new_total) > len(t.blocks) for t in seq.tables):
            raise ValueError("commit past the pages that grow() made")
        seq.num_tokens = new_total
        for group, table in zip(self.paged, seq.tables):
            lo, hi = self._dead(group, new_total)
            hi = min(hi, len(table.blocks))
            for index in range(max(table.first_live, lo), hi):
                if table.blocks[index] != group.scratch_page:
                    group.allocator.free(table.blocks[index])
                    table.blocks[index] = group.scratch_page
                    table.given_back += 1
            table.first_live = max(table.first_live, hi)

    def close(self, seq: SequenceCache) -> None:
        """Give back every page and the state slot."""
        if seq.closed:
            raise ValueError(f"request {seq.request_id!r} was closed before")
        for group, table in zip(self.paged, seq.tables):
            for block in table.blocks:
                if block != group.scratch_page:
                    group.allocator.free(block)
            table.blocks = []
            table.first_live = 0
            table.given_back = 0
        self._slots.free(seq.slot)
        seq.closed = True
        seq.num_tokens = 0
        del self.live[seq.request_id]

    release = close

    # ------------------------------------------------------------------ several hypotheses of a request
    def _need_kernels(self) -> None:
        if self.device is not None and self.device.type != "cuda":
            from .. import ops
            raise ops.KernelError("rows of a cache are moved on a CUDA device: there is no CPU path")

    def _paged_pools(self, group: PagedGroup) -> list[torch.Tensor]:
        """A group's pools as [planes, pages, kv_heads, page_tokens, channels]."""
        return [p.flatten(0, 1) if p.dim() == 6 else p for p in (group.pool, group.k_store, group.v_store) if p is not None]

    def fork(self, forks: list[tuple[SequenceCache, str]]) -> list[SequenceCache]:
        """A new request for each (live request, new request id), holding the same tokens: all of them, or (OutOfBlocks) none. Pages
        that hold nothing but those tokens are shared; the page that is still being written, the state slot and the record are
        copied, in one launch a pool whatever the number of forks. Pages behind the held tokens are not taken over."""
        self._need_kernels()
        ids = [request_id for _, request_id in forks]
        if len(set(ids)) != len(ids) or any(i in self.live for i in ids):
            raise ValueError("a forked request needs an id of its own")
        for seq, _ in forks:
            if seq.closed or self.live.get(seq.request_id) is not seq:
                raise ValueError(f"request {seq.request_id!r} is closed or does not belong to this cache")
        open_page = [seq.num_tokens // self.block_tokens if seq.num_tokens % self.block_tokens else None for seq, _ in forks]
        for g, group in enumerate(self.paged):
            wanted = sum(at is not None and seq.tables[g].blocks[at] != group.scratch_page for (seq, _), at in zip(forks, open_page))
            if wanted > group.allocator.num_free:
                raise OutOfBlocks(f"forking needs {wanted} blocks, {group.allocator.num_free} free")
        if len(forks) > self._slots.num_free:
            raise OutOfBlocks(f"forking needs {len(forks)} request slots, {self._slots.num_free} free")
        made, copies = [], [[] for _ in self.paged]
        for (seq, request_id), at in zip(forks, open_page):
            child = SequenceCache(request_id, self._slots.alloc(1)[0], [], seq.num_tokens, drafts=None if seq.drafts is None else [])
            for g, group in enumerate(self.paged):
                source = seq.tables[g]
                blocks = source.blocks[: self.blocks_for(seq.num_tokens)]
                for index, block in enumerate(blocks):
                    if block == group.scratch_page:
                        continue
                    if index == at:
                        blocks[index] = group.allocator.alloc(1)[0]
                        copies[g].append((block, blocks[index]))
                    else:
                        group.allocator.share(block)
                child.tables.append(BlockTable(blocks, min(source.first_live, len(blocks)), sum(b == group.scratch_page for b in blocks)))
            self.live[request_id] = child
            made.append(child)
        if self.device is not None and forks:
            try:
                self._copy_for(forks, made, copies)
            except Exception:
                for child in made:
                    self.close(child)
                raise
        return made

    def _copy_for(self, forks: list[tuple[SequenceCache, str]], made: list[SequenceCache], copies: list[list[tuple[int, int]]]) -> None:
        """What forked requests own: pages (per group: from, to), state slots and records."""
        from .. import ops

        pair = lambda rows: torch.tensor(rows, dtype=torch.int32).T.contiguous().to(self.device)
        for group, pairs in zip(self.paged, copies):
            if pairs:
                src, dst = pair(pairs)
                for pool in self._paged_pools(group):
                    ops.copy_pages(pool, src, dst)
        src, dst = pair([[seq.slot, child.slot] for (seq, _), child in zip(forks, made)])
        for group in self.states:
            ops.copy_pages(group.pool, src, dst)
        ops.copy_pages(self.records.unsqueeze(0), src, dst)

    def accept(self, accepted: list[tuple[SequenceCache, list[int]]]) -> None:
        """After a step over drafted tokens: each request keeps the drafts listed (rising places among its drafts, a path down the tree
        that its last step brought). Their rows move to the places right behind what the request holds, in all layers; they are counted, and the pages
        behind them given back."""
        from .. import ops

        self._need_kernels()
        seen = set()
        for seq, path in accepted:
            if seq.closed or self.live.get(seq.request_id) is not seq or seq.request_id in seen:
                raise ValueError(f"request {seq.request_id!r} is closed, listed twice or does not belong to this cache")
            seen.add(seq.request_id)
            room = min((len(t.blocks) for t in seq.tables), default=0) * self.block_tokens - seq.num_tokens
            if any(b <= a for a, b in zip([-1, *path], path)) or (path and path[-1] >= room):
                raise ValueError(f"request {seq.request_id!r}: accepted drafts rise and lie in its pages, got {path} with room for {room}")
            if seq.drafts is not None and any(node >= len(seq.drafts) or seq.drafts[node] != before for before, node in zip([-1, *path], path)):
                raise ValueError(f"request {seq.request_id!r}: accepted drafts are a path down those of its last step, whose parents are "
                                 f"{seq.drafts}, got {path}")
        if self.device is not None and any(place != node for _, path in accepted for place, node in enumerate(path)):
            cu = [0]
            for _, path in accepted:
                cu.append(cu[-1] + len(path))
            lists = [[seq.num_tokens for seq, _ in accepted], [node for _, path in accepted for node in path], cu]
            for g, group in enumerate(self.paged):
                width = max(len(seq.tables[g].blocks) for seq, _ in accepted)
                rows = [seq.tables[g].blocks + [group.scratch_page] * (width - len(seq.tables[g].blocks)) for seq, _ in accepted]
                sizes = [len(accepted) * width, *(len(x) for x in lists)]
                flat = torch.tensor([b for row in rows for b in row] + [x for part in lists for x in part], dtype=torch.int32).to(self.device)
                table, first, picked, ends = flat.split(sizes)
                for pool in self._paged_pools(group):
                    ops.compact_tokens(pool, table.view(len(accepted), width), first, picked, ends)
        for seq, path in accepted:
            self.commit(seq, seq.num_tokens + len(path))
            if seq.drafts is not None:
                seq.drafts = []
            keep = self.blocks_for(seq.num_tokens)
            for group, table in zip(self.paged, seq.tables):
                for block in table.blocks[keep:]:
                    if block != group.scratch_page:
                        group.allocator.free(block)
                    else:
                        table.given_back -= 1
                del table.blocks[keep:]
                table.first_live = min(table.first_live, len(table.blocks))

    # ------------------------------------------------------------------ checks
    def check_tables(self, seq: SequenceCache, tokens: int | None = None) -> None:
        """What a kernel cannot check for itself, before every launch (layover/kv/paged_cache.py:160-165):
        the request is the one this manager opened, its slot is inside the pool, every page id of
        its tables is inside its group's pool and held (or the scratch page), and the tables cover
        `tokens` tokens (default: those it holds)."""
        if self.live.get(seq.request_id) is not seq:
            raise ValueError(f"request {seq.request_id!r} is not open in this cache")
        if not 0 <= seq.slot < self.max_requests or len(seq.tables) != len(self.paged):
            raise ValueError(f"request {seq.request_id!r}: slot {seq.slot} or its tables do not belong to this cache")
        needed = self.blocks_for(seq.num_tokens if tokens is None else tokens)
        for group, table in zip(self.paged, seq.tables):
            if len(table.blocks) < needed:
                raise ValueError(f"request {seq.request_id!r}: {needed} pages needed, its table has {len(table.blocks)}")
            held = group.allocator.is_held
            for block in table.blocks:
                if block != group.scratch_page and not held(block):
                    raise ValueError(f"request {seq.request_id!r}: block {block} is not an allocated page of its pool")

    def check_row(self, group_index: int, row, request_id: str = "?") -> None:
        """The same check on one request's page ids as an int32 numpy array (what the batch builder
        is about to send to the device): every id is the scratch page or a held page of the group's
        pool. Vectorised, so that it costs little on every step."""
        import numpy as np

        group = self.paged[group_index]
        if row.size == 0:
            return
        low, high = int(row.min()), int(row.max())
        if low < 0 or high > group.scratch_page:
            raise ValueError(f"request {request_id!r}: page id {low if low < 0 else high} is outside its pool of "
                             f"{group.allocator.num_blocks} pages")
        real = row[row != group.scratch_page]
        if real.size and not np.frombuffer(group.allocator._out, dtype=np.uint8)[real].all():
            bad = int(real[np.frombuffer(group.allocator._out, dtype=np.uint8)[real] == 0][0])
            raise ValueError(f"request {request_id!r}: block {bad} is not an allocated page of its pool")

    def check(self) -> None:
        """No page lost, held twice or both free and held, over all live requests."""
        for index, group in enumerate(self.paged):
            group.allocator.check()
            held = [b for seq in self.live.values() for b in seq.tables[index].blocks if b != group.scratch_page]
            counts = Counter(held)
            if any(count != max(1, group.allocator.holders(block)) for block, count in counts.items()):
                raise AssertionError("a page is held by two tables")
            if len(counts) != group.allocator.num_used:
                raise AssertionError(f"{group.allocator.num_used} pages are out, {len(counts)} are in tables")
            for block in held:
                if not group.allocator.is_held(block):
                    raise AssertionError(f"page {block} is in a table and on the free list")
        self._slots.check()
        if self._slots.num_used != len(self.live):
            raise AssertionError("state slots and live requests disagree")
