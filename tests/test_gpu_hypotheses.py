"""Kernels for several hypotheses of a request (attention for trees of drafts, compaction and copies of a cache, beam selection)
against float64, at the edges of their tiles, chunks, masks and lists."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def ops():
    from layover_b200 import ops as o
    return o


# ------------------------------------------------------------------------------- trees of drafts
def random_tree(gen, nodes):
    """Parents of a random tree, -1: hangs on the last held token."""
    return [-1 if i == 0 or torch.rand((), generator=gen) < 0.15 else int(torch.randint(max(0, i - 5), i, (), generator=gen)) for i in range(nodes)]


def seen_of(parents):
    seen = torch.zeros(len(parents), len(parents), dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i] = True
    return seen


def words_of(seen, words):
    out = torch.zeros(seen.shape[0], words, dtype=torch.int64)
    for j in range(seen.shape[1]):
        out[:, j // 32] |= seen[:, j].long() << (j % 32)
    return torch.where(out >= 1 << 31, out - (1 << 32), out).to(torch.int32)


class Trees:
    """Requests with (held tokens, drafts), their cache full of NaN wherever nobody wrote."""

    def __init__(self, lengths, q_heads, kv_heads, dim, page=16, dtype=torch.bfloat16, window=0, sinks=False, softcap=0.0, seed=0, seen=None,
                 extra_rows=2, scale=None):
        gen = torch.Generator().manual_seed(seed)
        self.lengths, self.q_heads, self.kv_heads, self.dim, self.page, self.window, self.softcap = lengths, q_heads, kv_heads, dim, page, window, softcap
        tokens = sum(n for _, n in lengths)
        self.max_nodes, self.max_ctx = max(n for _, n in lengths), max(1, max(h + n for h, n in lengths))
        words = -(-max(self.max_nodes, 1) // 32)
        self.seen = seen if seen is not None else [seen_of(random_tree(gen, n)) for _, n in lengths]
        depth = [m.sum(1) - 1 for m in self.seen]
        self.positions = torch.cat([h + d.clamp(min=0) for (h, _), d in zip(lengths, depth)] + [torch.zeros(extra_rows, dtype=torch.long)]).to(torch.int32)
        self.tree = torch.cat([words_of(m, words) for m in self.seen] + [torch.full((extra_rows, words), -1, dtype=torch.int32)])
        needed = [-(-(h + n) // page) for h, n in lengths]
        pages = sum(needed) + 3
        order = torch.randperm(pages, generator=gen).tolist()
        width = max(max(needed), 1) + 1
        self.table = torch.full((len(lengths), width), 1 << 30, dtype=torch.int32)        # behind a request's pages: no page of the pool
        for i, n in enumerate(needed):
            self.table[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        self.q = torch.randn(tokens + extra_rows, q_heads * dim, generator=gen).to(dtype)
        self.k_pool, self.v_pool = (torch.full((pages, kv_heads, page, dim), NAN, dtype=dtype) for _ in range(2))
        self.k, self.v = ([torch.randn(h + n, kv_heads, dim, generator=gen).to(dtype) for h, n in lengths] for _ in range(2))
        self.sinks = torch.randn(q_heads, generator=gen) if sinks else None
        self.cu_q = torch.tensor([sum(n for _, n in lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32)
        self.ctx = torch.tensor([h + n for h, n in lengths], dtype=torch.int32)
        self.scale = dim ** -0.5 if scale is None else scale

    def fill(self):
        for i in range(len(self.lengths)):
            at = torch.arange(self.k[i].shape[0])
            pages = self.table[i].long()[at // self.page]
            self.k_pool[pages, :, at % self.page], self.v_pool[pages, :, at % self.page] = self.k[i], self.v[i]
        return self

    def run(self, **over):
        o = ops()
        d = {name: getattr(self, name).cuda() for name in ("q", "k_pool", "v_pool", "table", "cu_q", "ctx", "positions", "tree")}
        out = torch.full((d["q"].numel() + over.get("shift", 0),), 7.0, dtype=d["q"].dtype, device="cuda")[over.get("shift", 0):].view_as(d["q"])
        o.attention_tree(d["q"], d["k_pool"], d["v_pool"], out, d["table"], d["cu_q"], d["ctx"], d["positions"] if self.window else None, d["tree"],
                         len(self.lengths), self.q_heads, self.kv_heads, self.dim, self.page, self.scale, over.get("max_nodes", self.max_nodes),
                         over.get("max_ctx", self.max_ctx), window=self.window, sinks=None if self.sinks is None else self.sinks.cuda(),
                         softcap=self.softcap)
        return out.cpu()

    def want(self):
        """(outputs, sums of weight times |value|, largest sum of |q k| of a score), in 64 bits."""
        outs, sums, sizes, group = [], [], [], self.q_heads // self.kv_heads
        for i, (held, n) in enumerate(self.lengths):
            rows = slice(int(self.cu_q[i]), int(self.cu_q[i + 1]))
            see = torch.ones(n, held + n, dtype=torch.bool)
            if self.window:
                see[:, :held] = self.positions[rows, None].long() - torch.arange(held) < self.window
            see[:, held:] = self.seen[i]
            for h in range(self.q_heads):
                q, k, v = self.q[rows].view(n, self.q_heads, self.dim)[:, h].double(), self.k[i][:, h // group].double(), self.v[i][:, h // group].double()
                z = q @ k.T * self.scale
                if self.softcap:
                    z = self.softcap * torch.tanh(z / self.softcap)
                z = z.masked_fill(~see, -INF)
                top = z.amax(1, keepdim=True) if held + n else torch.full((n, 1), -INF, dtype=torch.float64)
                if self.sinks is not None:
                    top = top.clamp(min=float(self.sinks[h]))
                w = torch.exp(z - torch.where(top == -INF, 0.0, top)).masked_fill(~see, 0.0)
                total = w.sum(1, keepdim=True) + (0.0 if self.sinks is None else torch.exp(float(self.sinks[h]) - top))
                p = w / torch.where(total == 0, 1.0, total)
                v = v[None].expand(n, -1, -1).masked_fill(~see[..., None], 0.0)             # what is not seen does not count, NaN neither
                outs.append(torch.einsum("nk,nkd->nd", p, v)); sums.append(torch.einsum("nk,nkd->nd", p, v.abs()))
                size = (q.abs() @ k.abs().T).masked_fill(~see, 0.0) * self.scale
                sizes.append(size.amax(1) if size.shape[1] else size.new_zeros(n))
        join = lambda parts: torch.cat([torch.stack(parts[i * self.q_heads: (i + 1) * self.q_heads], 1).flatten(1) for i in range(len(self.lengths))])
        return join(outs), join(sums), max(float(s.max()) if s.numel() else 0.0 for s in sizes)

    def check(self, got=None, finite=None):
        got = self.run() if got is None else got
        assert ops().attention_tree_status() == 0
        want, sums, size = self.want()
        tokens = int(self.cu_q[-1])
        assert (got[tokens:] == 7.0).all()                                     # rows behind the last draft
        got = got[:tokens].double()
        # a weight's exponent is off by the rounding of its score: (dim + 4) additions and products of 32 bits; the exponential and a soft
        # cap's (a quotient of 2^-21) add 2^-18 at most; the sums over the keys round once a key, those over tiles and chunks with them
        step = 2.0 ** -24
        weights = 2 * ((self.dim + 4) * step * size + 2.0 ** -18 + self.softcap * 2.0 ** -20) + 2 * (self.max_ctx + 64) * step
        bound = weights * sums + 1e-30
        if self.q.dtype == torch.bfloat16:       # the weights round to bfloat16 for the second product, the result once more
            bound = bound + 2.0 ** -8 * sums + 2.0 ** -8 * (want.abs() + bound)
        else:
            bound = bound + 2.0 ** -24 * want.abs()
        off = (got - want).abs()
        ok = (off <= bound) | (torch.isnan(want) & torch.isnan(got)) | ((want == got) & torch.isinf(want))
        assert ok.all(), f"{int((~ok).sum())} of {ok.numel()} off, at most {float((off / bound).nan_to_num(0).max()):.3g} bounds"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("q_heads, kv_heads, dim", [(4, 2, 16), (6, 1, 32), (8, 8, 64), (12, 2, 128), (5, 5, 48), (16, 1, 128), (3, 1, 256), (32, 8, 128)])
def test_tree_attention_over_head_layouts(q_heads, kv_heads, dim, dtype):
    """One draft and many; held tokens that end a tile, begin one, and none at all."""
    Trees([(0, 1), (63, 1), (64, 7), (1, 16), (130, 17), (0, 9)], q_heads, kv_heads, dim, dtype=dtype, seed=dim).fill().check()


@pytest.mark.parametrize("dtype, dim", [(torch.float32, 4), (torch.float32, 20), (torch.float32, 132), (torch.bfloat16, 176)])
def test_tree_attention_over_odd_head_sizes(dtype, dim):
    Trees([(70, 5), (3, 12)], 6, 2, dim, dtype=dtype, seed=dim).fill().check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page", [1, 4, 8, 24, 128])
def test_tree_attention_over_page_sizes(page, dtype):
    Trees([(200, 11), (37, 3)], 8, 2, 128, page=page, dtype=dtype, seed=page).fill().check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nodes", [1, 2, 31, 32, 33, 64, 65, 150])
def test_tree_attention_over_tree_sizes(nodes, dtype):
    """Words of the mask, row tiles, drafts over several key tiles."""
    Trees([(50, nodes), (300, max(1, nodes - 1))], 4, 1, 128, dtype=dtype, seed=nodes).fill().check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("context", [1000, 5003])
def test_tree_attention_splits_long_contexts(context, dtype):
    """Chunks of the keys joined afterwards; a short request beside the long one has chunks without a key."""
    Trees([(context, 6), (5, 6), (context // 3, 2)], 8, 2, 128, dtype=dtype, seed=context).fill().check()


@pytest.mark.parametrize("nodes", [1, 9, 33])
@pytest.mark.parametrize("window", [0, 150])
def test_tree_attention_of_more_sequences_than_blocks(nodes, window):
    """Shares of several whole row tiles and of ends of two, requests without drafts among them; keys of one tile and of some."""
    lengths = [((i * 37) % 400, (i * 5) % (nodes + 1)) for i in range(70)] + [(2500, nodes)]
    Trees(lengths, 16, 4, 128, window=window, seed=nodes).fill().check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window", [1, 3, 64, 100, 5000])
def test_tree_attention_behind_a_window(window, dtype):
    """The deeper a draft the fewer held keys it sees, none with the smallest windows."""
    Trees([(400, 20), (63, 9), (1200, 3)], 8, 2, 64, dtype=dtype, window=window, seed=window).fill().check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sinks, softcap, context", [(True, 0.0, 90), (True, 0.0, 3000), (False, 5.0, 90), (True, 30.0, 3000)])
def test_tree_attention_with_sinks_and_cap(sinks, softcap, context, dtype):
    Trees([(context, 12), (0, 5)], 8, 4, 128, dtype=dtype, sinks=sinks, softcap=softcap, seed=7).fill().check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("held, sinks, window", [(0, False, 0), (0, True, 0), (100, False, 1)])
def test_tree_attention_rows_that_see_nothing_are_zero(held, sinks, window, dtype):
    empty = torch.zeros(10, 10, dtype=torch.bool)
    empty[3, 3] = empty[7, 2] = True                       # a mask need not be a tree
    case = Trees([(held, 10)], 4, 2, 128, dtype=dtype, sinks=sinks, window=window, seen=[empty]).fill()
    case.positions[:10] = held + 5                         # behind a window of one nothing held is seen
    got = case.run()
    case.check(got)
    assert (got[0] == 0).all() and (got[3] != 0).any() and (got[7] != 0).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("q_heads, kv_heads, nodes, held", [(4, 1, 3, 40), (8, 1, 5, 100), (8, 2, 20, 61), (4, 2, 70, 1500)])
def test_a_draft_that_is_not_finite_reaches_only_who_sees_it(q_heads, kv_heads, nodes, held, dtype):
    gen = torch.Generator().manual_seed(nodes)
    case = Trees([(held, nodes), (held, nodes)], q_heads, kv_heads, 128, dtype=dtype, seed=nodes)
    for i, value in ((1, NAN), (nodes - 1, INF), (nodes // 2, -INF)):
        case.v[0][held + i, :, int(torch.randint(128, (), generator=gen))] = value
    clean = case.fill().run()
    case.check(clean)
    case.k[0][held + 1] = NAN                              # a key, too: then every row that sees it is NaN
    got = case.fill().run()
    touched = case.seen[0][:, 1]
    assert torch.isnan(got[:nodes][touched]).all()
    rest = got[:nodes][~touched]
    assert torch.equal(torch.nan_to_num(rest, 99.0), torch.nan_to_num(clean[:nodes][~touched], 99.0)) and torch.equal(got[nodes:2 * nodes], clean[nodes:2 * nodes])


@pytest.mark.parametrize("nodes, others, held", [(5, 30, 3000), (10, 32, 500), (3, 60, 2000), (40, 64, 9000)])
def test_drafts_that_are_not_finite_beside_larger_trees(nodes, others, held):
    """All rows of a small tree are made again where the launch is planned for larger ones."""
    case = Trees([(held, nodes), (held, others), (20, nodes)], 8, 2, 128, seed=nodes)
    for seq in (0, 2):
        case.v[seq][-nodes + 1, 0, 3], case.v[seq][-1, 1, 77] = NAN, INF
    case.fill().check()


def test_tree_attention_of_large_scores():
    """Scores far apart: the weights of all but one key vanish, and nothing overflows."""
    for dtype in (torch.bfloat16, torch.float32):
        Trees([(500, 9)], 4, 2, 128, dtype=dtype, scale=20.0, seed=5).fill().check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tree_attention_of_a_chain_is_causal_attention(dtype):
    """Drafts in a row are a prompt portion: the same rows as the framework's causal attention gives."""
    o, n, held = ops(), 37, 211
    case = Trees([(held, n)], 8, 2, 128, dtype=dtype, seen=[torch.ones(n, n).tril().bool()], extra_rows=0, seed=3).fill()
    got = case.run()
    case.check(got)
    d = {name: getattr(case, name).cuda() for name in ("q", "k_pool", "v_pool", "table", "cu_q", "ctx")}
    block = o.attention_simt_block_queries()
    tiles = torch.arange(0, n, block, dtype=torch.int32).cuda()
    out = torch.empty_like(d["q"])
    o.attention_simt(d["q"], d["k_pool"], d["v_pool"], out, d["table"], d["cu_q"], d["ctx"], torch.zeros_like(tiles), tiles, tiles.numel(), 8, 2, 128, 16,
                     case.scale)
    case.check(out.cpu())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tree_attention_bounds_may_be_larger_than_the_lengths(dtype):
    """A captured step is planned for more drafts and keys than there are; requests without drafts have no rows."""
    case = Trees([(90, 4), (7, 0), (300, 9)], 8, 2, 128, dtype=dtype, seed=1).fill()
    case.check(case.run(max_nodes=32, max_ctx=4000))
    case.check(case.run(max_ctx=100))                      # planned for fewer keys: all are read all the same


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nodes, most", [(9, 3), (70, 5), (70, 40)])
def test_tree_attention_leaves_drafts_behind_the_most_alone(nodes, most, dtype):
    """Rows of drafts behind `max_nodes` stay as they are; the others are as they would be."""
    case = Trees([(300, nodes), (40, 2), (0, nodes)], 8, 2, 128, dtype=dtype, seed=nodes).fill()
    whole, got = case.run(), case.run(max_nodes=most)
    case.check(whole)
    for first, n in ((0, nodes), (nodes, 2), (nodes + 2, nodes)):
        assert (got[first + min(n, most): first + n] == 7.0).all()
    keep = torch.cat([torch.arange(f, f + min(n, most)) for f, n in ((0, nodes), (nodes, 2), (nodes + 2, nodes))])
    whole[keep] = got[keep]
    case.check(whole)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tree_attention_of_very_many_requests(dtype):
    """More than a block keeps the lengths of; some bring no drafts, some hold nothing."""
    gen = torch.Generator().manual_seed(3)
    held, nodes = torch.randint(0, 90, (700,), generator=gen).tolist(), torch.randint(0, 4, (700,), generator=gen).tolist()
    Trees(list(zip(held, nodes)), 2, 1, 128, dtype=dtype, seed=4).fill().check()


@pytest.mark.parametrize("dtype, dim", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 128)])
def test_pages_behind_2_to_the_31_values(dtype, dim):
    """The same rows in a small pool and at the end of one of over 2^31 values: attention, compaction and copies."""
    o, (held, n, heads, page) = ops(), (70, 9, 2, 16)
    gen = torch.Generator().manual_seed(6)
    put = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    pages, far = 8, (1 << 31) // (heads * page * dim) + 10
    small = torch.randn(2, pages, heads, page, dim, generator=gen).to(dtype).cuda()
    q, tree = torch.randn(n, 8 * dim, generator=gen).to(dtype).cuda(), words_of(seen_of(random_tree(gen, n)), 1).cuda()
    big = torch.empty(2, far, heads, page, dim, dtype=dtype, device="cuda")
    big[:, -pages:] = small
    outs = []
    for pool in (small, big):
        first = pool.shape[1] - pages
        table, out = put([[first + i for i in (5, 1, 7, 0, 3)]]), torch.empty_like(q)
        o.attention_tree(q, pool[0], pool[1], out, table, put([0, n]), put([held + n]), None, tree, 1, 8, heads, dim, page, dim ** -0.5, n, held + n)
        o.compact_tokens(pool, table, put([held]), put([1, 4, 8]), put([0, 3]))
        o.copy_pages(pool, put([first + 5, first + 1]), put([first + 2, first + 4]))
        outs.append((out.cpu(), pool[:, first:].cpu()))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_tree_attention_writes_to_any_16_bytes():
    case = Trees([(90, 4), (200, 9)], 8, 2, 128, seed=2).fill()
    case.check(case.run(shift=8))


# ------------------------------------------------------------------------------- moves in a cache
@pytest.mark.parametrize("dtype, channels", [(torch.bfloat16, 128), (torch.float32, 20), (torch.bfloat16, 20), (torch.bfloat16, 7), (torch.float32, 256), (torch.int8, 3)])
@pytest.mark.parametrize("page", [1, 5, 16])
def test_compaction_moves_the_picked_rows_and_nothing_else(page, dtype, channels):
    o, gen = ops(), torch.Generator().manual_seed(page * channels)
    planes, heads, kept = 3, 2, [[0, 1, 2], [4, 7, 11, 12], [], [19], list(range(1, 25)), [0, 2, 3, 9, 10, 11, 12, 13, 20, 21]]
    held = [5, 0, 3, 16, 31, 7]
    needed = [-(-(h + 26) // page) for h in held]
    pages = sum(needed) + 2
    order = torch.randperm(pages, generator=gen).tolist()
    table = torch.full((len(held), max(needed)), pages + 5, dtype=torch.int32)
    for i, n in enumerate(needed):
        table[i, :n] = torch.tensor([order.pop() for _ in range(n)])
    pool = torch.randint(-100, 100, (planes, pages, heads, page, channels), generator=gen).to(dtype)
    want = pool.clone()
    for i, picks in enumerate(kept):
        for place, p in enumerate(picks):
            a, b = held[i] + p, held[i] + place
            want[:, table[i, b // page], :, b % page] = pool[:, table[i, a // page], :, a % page]
    put = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cu = [sum(len(k) for k in kept[:i]) for i in range(len(kept) + 1)]
    got = pool.cuda()
    o.compact_tokens(got, table.cuda(), put(held), put([p for k in kept for p in k]), put(cu))
    assert torch.equal(got.cpu(), want)


def test_compaction_leaves_out_what_is_outside():
    o = ops()
    pool = torch.arange(2 * 4 * 1 * 4 * 8, dtype=torch.float32).view(2, 4, 1, 4, 8).cuda()
    before, put = pool.clone(), (lambda x: torch.tensor(x, dtype=torch.int32, device="cuda"))
    table = put([[0, 1, -1], [2, 99, 3]])
    o.compact_tokens(pool, table, put([2, 1]), put([7, 90, 100, 4, 6]), put([0, 3, 5]))      # page -1, behind the table, page 99
    o.compact_tokens(pool, put([[0, 1, 2]]), put([0]), put([0, 1]), put([-9, 1000]))                                # ends behind the drafts that are there
    assert torch.equal(pool, before)


@pytest.mark.parametrize("dtype, shape", [(torch.bfloat16, (2, 8, 16, 128)), (torch.float32, (3, 5, 7)), (torch.bfloat16, (1,)), (torch.float32, (32, 128, 128)),
                                          (torch.uint8, (11,)), (torch.bfloat16, (6,))])
def test_copies_of_pages(dtype, shape):
    o, gen = ops(), torch.Generator().manual_seed(len(shape))
    pool = torch.randint(0, 100, (5, 9, *shape), generator=gen).to(dtype)
    src, dst = [1, 1, 4, 8, 30, 2, -1], [0, 3, 6, 7, 5, 9, 5]        # one source twice; indices outside
    want = pool.clone()
    for a, b in list(zip(src, dst))[:4]:
        want[:, b] = pool[:, a]
    got = pool.cuda()
    o.copy_pages(got, torch.tensor(src, dtype=torch.int32).cuda(), torch.tensor(dst, dtype=torch.int32).cuda())
    assert torch.equal(got.cpu(), want)


# ------------------------------------------------------------------------------- beams
def select(logits, scores, keep, ended=None, pad=0):
    o, shape = ops(), (scores.shape[0], keep)
    outs = torch.full(shape, 5.0).cuda(), torch.full(shape, 55, dtype=torch.int32).cuda(), torch.full(shape, 55, dtype=torch.int32).cuda()
    o.beam_select(logits, scores.cuda(), *outs, ended=None if ended is None else ended.cuda(), pad=pad)
    return [x.cpu() for x in outs]


def selected(logits, scores, keep, ended=None, pad=0):
    (requests, beams), vocab = scores.shape, logits.shape[1]
    outs = []
    for r in range(requests):
        found = torch.full((beams, vocab), -INF, dtype=torch.float64)
        for b in range(beams):
            z = logits[r * beams + b].double().cpu()
            if ended is not None and ended[r, b]:
                found[b, pad] = scores[r, b].double()
            elif scores[r, b] > -INF and torch.isfinite(z.max()) and not torch.isnan(z).any():
                found[b] = scores[r, b].double() + torch.log_softmax(z, 0)
        best = found.flatten().sort(descending=True, stable=True).indices[:keep]
        values = found.flatten()[best]
        outs.append((values, torch.where(values == -INF, -1, best // vocab), torch.where(values == -INF, -1, best % vocab)))
    want = [torch.stack(x) for x in zip(*outs)]
    if keep > beams * vocab:                               # fewer candidates than places
        want = [torch.nn.functional.pad(x, (0, keep - beams * vocab), value=v) for x, v in zip(want, (-INF, -1, -1))]
    return want


def check_beams(logits, scores, keep, ended=None, pad=0):
    got, want = select(logits, scores, keep, ended, pad), selected(logits, scores, keep, ended, pad)
    assert torch.equal(got[1].long(), want[1]) and torch.equal(got[2].long(), want[2])
    finite = torch.isfinite(want[0])
    assert torch.equal(got[0][~finite].double(), want[0][~finite])
    # the score rounds once; the log of the sum is off by the exponentials' 2^-21 and the sums' roundings, relative to the sum: 2^-18 in all
    off = (got[0].double() - want[0]).abs()[finite]
    assert (off <= 2.0 ** -24 * want[0].abs()[finite] + 2.0 ** -18).all()


@pytest.mark.parametrize("requests, beams, keep", [(1, 1, 1), (1, 4, 4), (3, 5, 10), (2, 32, 32), (17, 3, 7), (1, 64, 32)])
@pytest.mark.parametrize("vocab", [1, 2, 33, 2049, 32768, 50001])
def test_beam_selection(requests, beams, keep, vocab):
    gen = torch.Generator().manual_seed(vocab + beams)
    logits = (3 * torch.randn(requests * beams, vocab + 3, generator=gen)).cuda()[:, :vocab]       # rows of wider ones
    scores = -5 * torch.rand(requests, beams, generator=gen)
    check_beams(logits, scores, keep)
    ended = (torch.rand(requests, beams, generator=gen) < 0.3).int()
    check_beams(logits, scores, keep, ended, pad=vocab // 2)


def test_beam_selection_breaks_ties_by_the_lowest_place():
    for vocab in (40, 5000, 100_000):
        logits, scores = torch.zeros(6, vocab).cuda(), torch.zeros(2, 3)
        values, parents, tokens = select(logits, scores, 20)
        assert (parents == 0).all() and torch.equal(tokens, torch.arange(20, dtype=torch.int32).expand(2, -1))
        logits[:, [7, vocab - 1, 20]] = 1.0                # three equal ones a beam, of equal beams
        values, parents, tokens = select(logits, scores, 9)
        assert torch.equal(parents, torch.tensor([0, 0, 0, 1, 1, 1, 2, 2, 2], dtype=torch.int32).expand(2, -1))
        assert torch.equal(tokens, torch.tensor([7, 20, vocab - 1] * 3, dtype=torch.int32).expand(2, -1))


def test_beam_selection_of_rising_and_falling_logits():
    """Every value, and none but the first, is better than all before it."""
    rise = torch.linspace(-4, 4, 70_000)
    check_beams(torch.stack((rise, rise.flip(0), rise, rise.flip(0))).cuda(), torch.tensor([[-1.0, -2.0], [-2.0, -1.5]]), 32)


def test_beam_selection_of_masked_beams_and_tokens():
    gen = torch.Generator().manual_seed(4)
    low = torch.finfo(torch.float32).min
    logits = torch.randn(12, 3000, generator=gen)
    logits[0, 5:] = -INF                                   # five candidates
    logits[1] = -INF                                       # none
    logits[2, 7] = NAN                                     # no finite sum of exponentials
    logits[3, 9] = INF
    logits[4, 3:] = low                                    # three that count, then the lowest ones
    logits[5] = low                                        # all alike
    logits[6] = 1e30
    logits[7, ::2] = -INF
    scores = torch.tensor([[-1.0, -2.0, -0.5], [-0.1, -3.0, -INF], [-INF, -4.0, -INF], [-1.0, -1.0, -1.0]])
    for keep in (3, 8, 32):
        check_beams(logits.cuda(), scores, keep)
        check_beams(logits.cuda(), scores, keep, torch.tensor([[0, 1, 1], [0, 0, 1], [1, 1, 0], [1, 0, 1]], dtype=torch.int32), pad=2999)


def test_beam_selection_of_the_most_beams():
    gen = torch.Generator().manual_seed(12)
    logits = torch.randn(2 * 64, 30_000, generator=gen).cuda()
    logits[5] = 0.25                                   # a row of equal ones among the others
    check_beams(logits, -3 * torch.rand(2, 64, generator=gen), 32)
    few = torch.randn(3, 2, generator=gen).cuda()      # fewer candidates than places
    values, parents, tokens = select(few, torch.zeros(1, 3), 32)
    assert parents[0, :6].min() >= 0 and (parents[0, 6:] == -1).all() and (values[0, 6:] == -INF).all() and (tokens[0, 6:] == -1).all()


def test_beam_selection_does_not_read_beams_that_are_over():
    """Neither an ended beam's logits nor those of one that is not there reach the others."""
    gen = torch.Generator().manual_seed(10)
    logits = torch.randn(8, 9000, generator=gen)
    clean = logits.clone()
    logits[1] = float("nan"); logits[6] = INF; logits[7, 100:] = float("nan")
    scores = torch.tensor([[-1.0, -INF, -2.0, -1.5], [-1.0, -2.0, -1.5, -INF]])
    ended = torch.tensor([[0, 0, 0, 1], [0, 0, 1, 0]], dtype=torch.int32)
    found, expected = select(logits.cuda(), scores, 8, ended, 5), select(clean.cuda(), scores, 8, ended, 5)
    assert all(torch.equal(x, y) for x, y in zip(found, expected)) and bool((found[2] >= 0).all())


def test_first_step_of_a_beam_search_takes_one_beam():
    gen = torch.Generator().manual_seed(9)
    logits = torch.randn(8, 4096, generator=gen).cuda()
    scores = torch.tensor([[0.0, -INF, -INF, -INF], [-INF, -INF, 0.0, -INF]])
    check_beams(logits, scores, 4)


# ------------------------------------------------------------------------------- streams and graphs
def test_captured_and_on_another_stream():
    """Captured once, replayed on new inputs at the same addresses, two graphs in flight one after the other; then on a side stream."""
    o = ops()
    case = Trees([(900, 6), (41, 6)], 8, 2, 128, seed=11, extra_rows=0).fill()
    d = {name: getattr(case, name).cuda() for name in ("q", "k_pool", "v_pool", "table", "cu_q", "ctx", "positions", "tree")}
    logits, scores = torch.randn(4, 9000).cuda(), torch.randn(1, 4).cuda()
    outs = [torch.empty_like(d["q"]) for _ in range(2)]
    chosen = [(torch.empty(1, 4).cuda(), *(torch.empty(1, 4, dtype=torch.int32).cuda() for _ in range(2))) for _ in range(2)]

    def both(i):
        o.attention_tree(d["q"], d["k_pool"], d["v_pool"], outs[i], d["table"], d["cu_q"], d["ctx"], None, d["tree"], 2, 8, 2, 128, 16, case.scale, 6, 906)
        o.beam_select(logits, scores, *chosen[i])

    both(0); both(1)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph):
            both(i)
    d["q"].mul_(-1)
    logits.neg_()
    for x in (*outs, *chosen[0], *chosen[1]):
        x.zero_()
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    case.q = -case.q
    for i in range(2):
        case.check(outs[i].cpu())
        want = selected(logits, scores.cpu(), 4)
        assert torch.equal(chosen[i][1].cpu().long(), want[1]) and torch.equal(chosen[i][2].cpu().long(), want[2])
    side = torch.cuda.Stream()
    outs[0].zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(0)
    side.synchronize()
    case.check(outs[0].cpu())


def test_the_same_call_gives_the_same_bits():
    case = Trees([(2000, 9), (77, 3)], 8, 2, 128, seed=2).fill()
    assert torch.equal(case.run(), case.run())


# ------------------------------------------------------------------------------- as they are used
@pytest.fixture(scope="module", params=["fp32", "bf16"])
def served(request, tiny_folders):
    """A model with the head size of the served ones (tcgen05) and one of small heads, in either precision."""
    import layover_b200 as lb
    return {name: lb.load_model(str(tiny_folders[name][0]), device="cuda", dtype=request.param) for name in ("a", "c")}


def fresh(model, blocks=200, page=8):
    import layover_b200 as lb
    from layover_b200.engine.step import StepFunction
    cache = lb.PagedKVCache(model, blocks, block_tokens=page, max_requests=24)
    return cache, StepFunction(model, cache)


def feed(cache, step, name, tokens):
    """A request that holds `tokens`, fed as one portion; the logits of its last."""
    import layover_b200 as lb
    seq = cache.open(name)
    return seq, step([lb.StepEntry(seq, list(tokens), [len(tokens) - 1])]).clone()[0]


@pytest.mark.parametrize("name", ["a", "c"])
def test_a_step_over_drafts_and_what_follows_it(served, name):
    """Every draft's logits are those of its own branch fed as a request of its own; after some are accepted the request goes on as if it
    had been fed them; a second request's portion shares the step."""
    import layover_b200 as lb
    from conftest import random_prompt, tolerance
    model = served[name]
    cache, step = fresh(model)
    vocab = model.spec.vocab_size
    prompt, tokens = random_prompt(vocab, 45, 1), random_prompt(vocab, 9, 2)
    parents, other = [-1, 0, 0, 1, 1, 2, -1, 4, 7], random_prompt(vocab, 13, 3)
    seq, _ = feed(cache, step, "x", prompt)
    beside = cache.open("y")
    logits = step([lb.StepEntry(seq, tokens, list(range(9)), parents), lb.StepEntry(beside, other, [12])]).clone()
    assert seq.num_tokens == 45 and beside.num_tokens == 13
    branch = [[t] if p < 0 else None for t, p in zip(tokens, parents)]
    for i, p in enumerate(parents):
        branch[i] = branch[i] or branch[p] + [tokens[i]]
    for i in range(9):
        one, want = feed(cache, step, f"branch {i}", prompt + branch[i])
        assert (logits[i] - want).abs().max().item() <= tolerance(want, model.dtype)
        cache.close(one)
    _, want = feed(cache, step, "alone", other)
    assert (logits[9] - want).abs().max().item() <= tolerance(want, model.dtype)
    path = [0, 1, 4, 7, 8]
    cache.accept([(seq, path)])
    cache.check()
    assert seq.num_tokens == 50
    got = step([lb.StepEntry(seq, [3], [0])])[0].clone()
    _, want = feed(cache, step, "path", prompt + [tokens[i] for i in path] + [3])
    assert (got - want).abs().max().item() <= tolerance(want, model.dtype)
    assert ops().attention_tree_status() == 0


@pytest.mark.parametrize("window", [1, 3, 16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_drafts_behind_a_window_shorter_than_their_branch(tiny_folders, window, dtype):
    """As token by token: a window counts drafts too, and the tokens of a portion that shares the step."""
    import layover_b200 as lb
    from conftest import random_prompt, tolerance
    from test_gpu_engine import build_toy
    model = build_toy(tiny_folders, "a", dtype, window=window)[0]
    assert model.takes_drafts
    cache, step = fresh(model)
    vocab = model.spec.vocab_size
    prompt, other = random_prompt(vocab, 45, 1), random_prompt(vocab, 40, 3)
    parents = [-1, 0, 0, 1, 1, 2, *range(5, 30)]
    tokens = random_prompt(vocab, len(parents), 2)
    seq, _ = feed(cache, step, "x", prompt)
    beside = cache.open("y")
    logits = step([lb.StepEntry(seq, tokens, list(range(len(tokens))), parents), lb.StepEntry(beside, other, [39])]).clone()
    for i in (0, 2, 4, 8, 20, len(tokens) - 1):
        branch, at = [], i
        while at >= 0:
            branch, at = [tokens[at], *branch], parents[at]
        one, want = feed(cache, step, f"branch {i}", prompt + branch)
        assert (logits[i] - want).abs().max().item() <= tolerance(want, model.dtype)
        cache.close(one)
    _, want = feed(cache, step, "alone", other)
    assert (logits[-1] - want).abs().max().item() <= tolerance(want, model.dtype)
    path = [0, 2, *range(5, 25)]
    cache.accept([(seq, path)])
    cache.check()
    got = step([lb.StepEntry(seq, [3], [0])])[0].clone()
    _, want = feed(cache, step, "after", prompt + [tokens[i] for i in path] + [3])
    assert (got - want).abs().max().item() <= tolerance(want, model.dtype)


@pytest.mark.parametrize("name", ["a", "c"])
def test_forked_requests_go_their_own_ways(served, name):
    import layover_b200 as lb
    from conftest import random_prompt, tolerance
    model = served[name]
    cache, step = fresh(model)
    prompt = random_prompt(model.spec.vocab_size, 43, 5)
    seq, _ = feed(cache, step, "x", prompt)
    children = cache.fork([(seq, "b"), (seq, "c")])
    logits = step([lb.StepEntry(s, [t], [0]) for s, t in zip((seq, *children), (1, 2, 3))]).clone()
    cache.close(seq)
    for row, child, token in zip(logits[1:], children, (2, 3)):
        _, want = feed(cache, step, f"plain {token}", prompt + [token])
        assert (row - want).abs().max().item() <= tolerance(want, model.dtype)
        got = step([lb.StepEntry(child, [9, 8, 7], [2])])[0].clone()
        _, want = feed(cache, step, f"longer {token}", prompt + [token, 9, 8, 7])
        assert (got - want).abs().max().item() <= tolerance(want, model.dtype)
    cache.check()


def test_forks_copy_states_and_records(tmp_path):
    import layover_b200 as lb
    from layover_b200.engine.step import StepFunction
    model = lb.random_model(lb.preset("topidra-tiny"), seed=0, device="cuda", dtype="fp32")
    cache = lb.PagedKVCache(model, 100, block_tokens=8, max_requests=6)
    step = StepFunction(model, cache)
    prompt = [int(t) for t in torch.randint(0, model.spec.vocab_size, (29,), generator=torch.Generator().manual_seed(1))]
    seq, _ = feed(cache, step, "x", prompt)
    cache.records[seq.slot] = torch.arange(cache.record_words, dtype=torch.int32, device="cuda")
    (child,) = cache.fork([(seq, "y")])
    assert torch.equal(cache.records[child.slot], cache.records[seq.slot])
    for group in cache.states:
        assert torch.equal(group.pool[:, child.slot], group.pool[:, seq.slot])
    first, second = step([lb.StepEntry(seq, [4], [0]), lb.StepEntry(child, [4], [0])])
    assert torch.equal(first, second)
    with pytest.raises(ValueError, match="no form for a tree"):
        step([lb.StepEntry(seq, [1, 2], [0], [-1, -1])])
    cache.check()


@pytest.mark.parametrize("name", ["a", "c"])
def test_generation_with_drafts_is_greedy_generation(served, name):
    """Each token is the greedy choice after those before it, within the logits' tolerance; a text that repeats itself takes fewer steps."""
    import layover_b200 as lb
    from conftest import tolerance
    model = served[name]
    prompts = [[7, 8, 9, 10, 7, 8, 9, 10, 7, 8], [5, 6], [3]]
    out, counts = lb.generate_with_drafts(model, prompts, 40, lb.LookupDrafts(2, 5, 1), block_tokens=8, prefill_chunk=4)
    assert [len(o) for o in out] == [40, 40, 40] and counts["drafted"] >= counts["accepted"]
    cache, step = fresh(model)
    for i, (prompt, tokens) in enumerate(zip(prompts, out)):
        text = prompt + tokens
        seq = cache.open(f"{i}")
        logits = step([lb.StepEntry(seq, text, list(range(len(prompt) - 1, len(text) - 1)))])
        chosen = logits.gather(1, torch.tensor(tokens, device="cuda")[:, None])[:, 0]
        assert (logits.amax(1) - chosen).max().item() <= 2 * tolerance(logits, model.dtype)
    stop = out[0][5]
    again, _ = lb.generate_with_drafts(model, prompts[:1], 40, lb.LookupDrafts(2, 5, 1), stop_tokens={stop}, block_tokens=8, prefill_chunk=4)
    assert again[0] == out[0][: out[0].index(stop) + 1]


def test_beam_search_finds_the_best_beams(tiny_folders):
    """Against a search that feeds every beam's whole text anew: the same texts where their sums are apart, the same sums."""
    import layover_b200 as lb
    from conftest import random_prompt
    model = lb.load_model(str(tiny_folders["a"][0]), device="cuda", dtype="fp32")
    prompts, beams, new = [random_prompt(256, 11, 1), random_prompt(256, 1, 2), random_prompt(256, 24, 3)], 3, 7
    found = lb.beam_search(model, prompts, beams, new, block_tokens=4, prefill_chunk=8)
    cache, step = fresh(model, 800, 4)
    for r, prompt in enumerate(prompts):
        held = [(0.0, [])]
        for _ in range(new):
            rows = []
            for score, tokens in held:
                seq, logits = feed(cache, step, "t", prompt + tokens)
                cache.close(seq)
                rows += [(score + float(p), tokens + [t]) for t, p in enumerate(torch.log_softmax(logits.double(), 0).tolist())]
            held = sorted(rows, key=lambda x: -x[0])[:beams]
        assert [round(s, 3) for s, _ in found[r]] == pytest.approx([round(s, 3) for s, _ in held], abs=2e-3)
        for (score, tokens), (want, text) in zip(found[r], held):
            assert tokens == text or min(abs(want - s) for s, t in held if t != text) < 1e-3
    stop = found[0][0][1][2]
    stopped = lb.beam_search(model, prompts[:1], beams, new, stop_tokens={stop}, block_tokens=4)
    assert any(tokens[-1] == stop for _, tokens in stopped[0]) and all(stop not in tokens[:-1] for _, tokens in stopped[0])


def test_command_line_follows_beams_and_checks_drafts(capsys):
    import json
    from layover_b200.__main__ import main
    base = ["--preset", "tiny-b", "--random-weights", "--dtype", "fp32", "--prompt-lens", "9,20", "--max-new-tokens", "6"]
    assert main(base + ["--beams", "3"]) == 0
    beams = json.loads(capsys.readouterr().out)
    assert [len(b) for b in beams["generated"]] == [3, 3] and all(len(t) == 6 for b in beams["generated"] for t in b)
    assert main(base + ["--drafts", "4"]) == 0
    assert [len(t) for t in json.loads(capsys.readouterr().out)["generated"]] == [6, 6]
    with pytest.raises(SystemExit):
        main(base + ["--drafts", "4", "--beams", "2"])
