"""Several hypotheses of a request on the host: what the operators refuse, before any device is asked for."""

import pytest
import torch

from layover_b200 import ops

I32 = torch.int32


def zeros(*shape, dtype=I32):
    return torch.zeros(shape, dtype=dtype)


def tree_call(**over):
    """A call of 5 drafts of 2 requests, 4 heads over 2 of 16 channels, with some arguments changed."""
    a = dict(q=zeros(5, 64, dtype=torch.bfloat16), k_pool=zeros(3, 2, 4, 16, dtype=torch.bfloat16), v_pool=zeros(3, 2, 4, 16, dtype=torch.bfloat16),
             out=zeros(5, 64, dtype=torch.bfloat16), block_table=zeros(2, 2), cu_q=zeros(3), ctx_len=zeros(2), positions=zeros(5), tree=zeros(5, 1), n_seqs=2,
             q_heads=4, kv_heads=2, dim=16, page_tokens=4, scale=0.25, max_nodes=3, max_ctx=8)
    a.update(over)
    return ops.attention_tree(**a)


@pytest.mark.parametrize("over, message", [
    (dict(out=zeros(5, 64, dtype=torch.float32)), "out must be"), (dict(k_pool=zeros(3, 2, 4, 16, dtype=torch.float32)), "k_pool must be"),
    (dict(cu_q=zeros(3, dtype=torch.int64)), "cu_q must be"), (dict(tree=zeros(5)), "2 dimension"), (dict(tree=zeros(4, 1)), "a row of tree per draft"),
    (dict(tree=zeros(5, 2)[:, :1]), "contiguous"), (dict(q=zeros(64, 5, dtype=torch.bfloat16).T), "contiguous"), (dict(q_heads=3), "multiple of kv_heads"),
    (dict(kv_heads=0), "multiple of kv_heads"), (dict(dim=32), "do not match the heads"), (dict(page_tokens=8), "do not match the heads"),
    (dict(n_seqs=3), "a row of tree per draft"), (dict(max_nodes=33), "2 words"), (dict(max_nodes=0), "at least 1"), (dict(max_ctx=0), "at least 1"),
    (dict(scale=0.0), "scale is positive"), (dict(scale=float("nan")), "scale is positive"),
    (dict(window=-1), "not negative"), (dict(softcap=-1.0), "not negative"), (dict(window=4, positions=None), "needs positions"),
    (dict(window=4, positions=zeros(4)), "a position per draft"), (dict(sinks=zeros(3, dtype=torch.float32)), "one sink"),
    (dict(q=zeros(5, 64, dtype=torch.float16), out=zeros(5, 64, dtype=torch.float16), k_pool=zeros(3, 2, 4, 16, dtype=torch.float16),
          v_pool=zeros(3, 2, 4, 16, dtype=torch.float16)), "not supported"),
    (dict(dim=8, q=zeros(5, 32, dtype=torch.bfloat16), out=zeros(5, 32, dtype=torch.bfloat16), k_pool=zeros(3, 2, 4, 8, dtype=torch.bfloat16),
          v_pool=zeros(3, 2, 4, 8, dtype=torch.bfloat16)), "not supported"),
    (dict(dim=272, q=zeros(5, 1088, dtype=torch.bfloat16), out=zeros(5, 1088, dtype=torch.bfloat16), k_pool=zeros(3, 2, 4, 272, dtype=torch.bfloat16),
          v_pool=zeros(3, 2, 4, 272, dtype=torch.bfloat16)), "not supported"),
])
def test_tree_attention_refuses(over, message):
    with pytest.raises(ValueError, match=message):
        tree_call(**over)


def test_operators_have_no_cpu_path():
    with pytest.raises(ops.KernelError, match="no CPU path"):
        tree_call()
    with pytest.raises(ops.KernelError, match="no CPU path"):
        ops.copy_pages(zeros(2, 3, 4), zeros(1), zeros(1))
    with pytest.raises(ops.KernelError, match="no CPU path"):
        ops.compact_tokens(zeros(2, 3, 1, 4, 4), zeros(1, 2), zeros(1), zeros(2), zeros(2))
    with pytest.raises(ops.KernelError, match="no CPU path"):
        beam_call()


@pytest.mark.parametrize("args, message", [
    ((zeros(2, 6).T, zeros(1), zeros(1)), "contiguous"), ((zeros(2, 3), zeros(1, dtype=torch.int64), zeros(1)), "src must be"),
    ((zeros(2, 3), zeros(1), zeros(2)), "one index per copy"), ((zeros(6), zeros(1), zeros(1)), "planes, pages"), ((zeros(2, 3), zeros(1, 1), zeros(1, 1)), "one index"),
])
def test_copies_refuse(args, message):
    with pytest.raises(ValueError, match=message):
        ops.copy_pages(*args)


@pytest.mark.parametrize("over, message", [
    (dict(pool=zeros(2, 3, 4, 4)), "planes, pages"), (dict(block_table=zeros(1, 2)), "a table row"), (dict(cu_picked=zeros(2)), "an end per sequence"),
    (dict(picked=zeros(2, dtype=torch.int64)), "picked must be"), (dict(first=zeros(4)[::2]), "contiguous"),
])
def test_compaction_refuses(over, message):
    a = dict(pool=zeros(2, 3, 1, 4, 4), block_table=zeros(2, 2), first=zeros(2), picked=zeros(2), cu_picked=zeros(3))
    a.update(over)
    with pytest.raises(ValueError, match=message):
        ops.compact_tokens(**a)


def beam_call(**over):
    f = torch.float32
    a = dict(logits=zeros(6, 10, dtype=f), scores=zeros(2, 3, dtype=f), next_scores=zeros(2, 4, dtype=f), parents=zeros(2, 4), tokens=zeros(2, 4))
    a.update(over)
    return ops.beam_select(**a)


@pytest.mark.parametrize("over, message", [
    (dict(logits=zeros(6, 10, dtype=torch.bfloat16)), "float32"), (dict(logits=zeros(10, 6, dtype=torch.float32).T), "contiguous vocabulary"),
    (dict(logits=zeros(5, 10, dtype=torch.float32)), "a row of logits per beam"), (dict(parents=zeros(2, 3)), "the outputs"), (dict(tokens=zeros(2, 4, dtype=torch.int64)), "tokens must be"),
    (dict(pad=10), "pad a token"), (dict(pad=-1), "pad a token"), (dict(ended=zeros(2, 4)), "scores' shape"), (dict(ended=zeros(2, 3, dtype=torch.bool)), "ended must be"),
    (dict(next_scores=zeros(2, 33, dtype=torch.float32), parents=zeros(2, 33), tokens=zeros(2, 33)), "keep is"),
    (dict(next_scores=zeros(2, 0, dtype=torch.float32), parents=zeros(2, 0), tokens=zeros(2, 0)), "keep is"),
    (dict(logits=zeros(130, 10, dtype=torch.float32), scores=zeros(2, 65, dtype=torch.float32)), "beams 1"),
])
def test_beam_selection_refuses(over, message):
    with pytest.raises(ValueError, match=message):
        beam_call(**over)


@pytest.mark.parametrize("n_seqs, nodes, ctx, window, heads", [(1, 1, 1, 0, (32, 8, 128)), (1, 8, 708, 0, (32, 8, 128)), (40, 25, 8025, 0, (32, 8, 128)), (2, 64, 12409, 0, (16, 4, 128)),
                                                             (5, 13, 1544, 1024, (12, 2, 64)), (3, 700, 900, 16, (16, 1, 128)), (64, 64, 131072, 0, (64, 8, 256))])
def test_tree_plan_covers_rows_and_keys(n_seqs, nodes, ctx, window, heads):
    q_heads, kv_heads, dim = heads
    for wide in (False, True):
        tile_rows, row_tiles, chunks, chunk_tiles = ops.tree_plan(n_seqs, nodes, ctx, window, *heads, 148, wide)
        rows, keys = nodes * q_heads // kv_heads, min(ctx, nodes + window) if window else ctx
        assert (row_tiles - 1) * tile_rows < rows <= row_tiles * tile_rows
        tile = 64 if wide else 32
        assert chunks * chunk_tiles * tile >= keys and (chunks - 1) * chunk_tiles * tile < keys + 2 * tile
        assert chunks == 1 or n_seqs * kv_heads * row_tiles * chunks * tile_rows * (dim + 2) <= 64 << 20
    blocks, rows2, floats = ops.tree_share(n_seqs, nodes, ctx, window, q_heads, kv_heads, 148)
    assert 1 <= blocks <= 148 and rows2 == (nodes > 128 // (q_heads // kv_heads)) and floats > 2 * blocks * 128 * 130


# ------------------------------------------------------------------------------- the cache's bookkeeping
def manager(needs=None, blocks=20, page=4, max_requests=8):
    from layover_b200.cache import CacheManager
    from layover_b200.parts.base import PagedKVNeed, StateNeed

    needs = needs or [PagedKVNeed(2, 16, None), PagedKVNeed(2, 16, 6), StateNeed((3,), torch.float32)]
    return CacheManager([(i, n, None) for i, n in enumerate(needs)], blocks, page, torch.float32, None, max_requests)


def test_a_shared_page_returns_with_its_last_holder():
    from layover_b200.cache import BlockAllocator

    a = BlockAllocator(3)
    a.alloc(2)
    a.share(0); a.share(0)
    assert a.holders(0) == 3 and a.holders(1) == 1 and a.holders(2) == 0
    a.free(0); a.free(0)
    assert a.is_held(0) and a.num_free == 1 and a.holders(0) == 1
    a.free(0)
    assert not a.is_held(0) and a.num_free == 2
    with pytest.raises(ValueError, match="not allocated"):
        a.free(0)
    with pytest.raises(ValueError, match="cannot be shared"):
        a.share(2)
    a.check()


def test_a_fork_shares_full_pages_and_owns_the_one_that_is_written():
    m = manager()
    a = m.open("a")
    m.grow(a, 10); m.commit(a, 10)
    m.grow(a, 14)                                        # pages ahead of what is held are not taken over
    b, c = m.fork([(a, "b"), (a, "c")])
    assert b.num_tokens == 10 and b.slot != a.slot != c.slot and len(b.tables[0].blocks) == 3
    assert b.tables[0].blocks[:2] == a.tables[0].blocks[:2] and len({s.tables[0].blocks[2] for s in (a, b, c)}) == 3
    m.check(); m.check_tables(b)
    for seq, total in ((a, 14), (b, 21), (c, 11)):
        m.grow(seq, total); m.commit(seq, total)
        m.check()
    m.close(a); m.check()
    m.close(c); m.check()
    m.close(b)
    m.check()
    assert m.num_free == 20 and m.num_free_slots == 8


def test_a_fork_at_the_end_of_a_page_copies_none_and_an_empty_one_shares_none():
    m = manager()
    a = m.open("a")
    (e,) = m.fork([(a, "e")])
    assert e.tables[0].blocks == [] and e.num_tokens == 0
    m.grow(a, 8); m.commit(a, 8)
    free = m.num_free
    (b,) = m.fork([(a, "b")])
    assert m.num_free == free and b.tables[0].blocks == a.tables[0].blocks
    (d,) = m.fork([(b, "d")])                             # a fork of a fork
    m.check()
    for seq in (a, b, d, e):
        m.close(seq)
    m.check()


def test_forks_are_all_or_none():
    from layover_b200.cache import OutOfBlocks

    m = manager(blocks=4, max_requests=3)
    a = m.open("a")
    m.grow(a, 9); m.commit(a, 9)                         # three pages, one free
    with pytest.raises(OutOfBlocks, match="2 blocks"):
        m.fork([(a, "b"), (a, "c")])
    m.check()
    assert set(m.live) == {"a"}
    with pytest.raises(ValueError, match="id of its own"):
        m.fork([(a, "a")])
    with pytest.raises(ValueError, match="id of its own"):
        m.fork([(a, "b"), (a, "b")])
    m.grow(a, 12); m.commit(a, 12)
    with pytest.raises(OutOfBlocks, match="slots"):
        m.fork([(a, "b"), (a, "c"), (a, "d")])
    m.close(a)
    with pytest.raises(ValueError, match="closed"):
        m.fork([(a, "b")])
    m.check()


@pytest.mark.parametrize("path, pages", [([], 3), ([0], 3), ([0, 1, 2], 4), ([1, 4, 5, 9], 4)])
def test_accepted_drafts_are_counted_and_the_pages_behind_them_given_back(path, pages):
    m = manager([__import__("layover_b200").parts.base.PagedKVNeed(2, 16, None)])
    a = m.open("a")
    m.grow(a, 10); m.commit(a, 10)
    m.grow(a, 10 + 11)                                   # eleven drafts: six pages
    m.accept([(a, path)])
    assert a.num_tokens == 10 + len(path) and len(a.tables[0].blocks) == pages
    m.check(); m.check_tables(a)
    m.grow(a, a.num_tokens + 5); m.commit(a, a.num_tokens + 5)
    m.close(a)
    m.check()
    assert m.num_free == 20


def test_accept_behind_a_window_keeps_the_books():
    m = manager()
    a = m.open("a")
    for total in (3, 9, 17):
        m.grow(a, total); m.commit(a, total)
    for path in ([0, 2], [0], [1, 3, 6], [], [0, 1, 2, 3, 4, 5, 6, 7]):
        m.grow(a, a.num_tokens + 9)
        m.accept([(a, path)])
        m.check(); m.check_tables(a)
    m.close(a)
    m.check()


def test_accept_refuses():
    m = manager()
    a, b = m.open("a"), m.open("b")
    m.grow(a, 6)
    for path in ([2, 1], [1, 1], [-1], [8]):
        with pytest.raises(ValueError, match="accepted drafts rise"):
            m.accept([(a, path)])
    with pytest.raises(ValueError, match="listed twice"):
        m.accept([(a, [0]), (a, [0])])
    m.close(b)
    with pytest.raises(ValueError, match="closed"):
        m.accept([(b, [])])
    assert a.num_tokens == 0


def test_random_forks_lose_no_page():
    import random

    rng = random.Random(3)
    m = manager(blocks=60, max_requests=12)
    live, made = [m.open("0")], 1
    for _ in range(600):
        seq = rng.choice(live)
        kind = rng.random()
        if kind < 0.35 and len(live) < 10:
            if m.num_free >= 2:
                live += m.fork([(seq, str(made))])
                made += 1
        elif kind < 0.55 and len(live) > 1:
            live.remove(seq)
            m.close(seq)
        elif m.num_free >= 6:
            n = rng.randint(1, 9)
            m.grow(seq, seq.num_tokens + n)
            if kind < 0.8:
                m.commit(seq, seq.num_tokens + n)
            else:
                m.accept([(seq, sorted(rng.sample(range(n), rng.randint(0, n))))])
        elif len(live) > 1:
            live.remove(seq)
            m.close(seq)
        m.check()
    for seq in live:
        m.close(seq)
    m.check()
    assert m.num_free == 60


# ------------------------------------------------------------------------------- trees of drafts on the host
def test_a_batch_carries_the_tree_of_its_drafts():
    from layover_b200.engine.batch import BatchBuilder, StepEntry

    m = manager([__import__("layover_b200").parts.base.PagedKVNeed(2, 16, None)], blocks=40)
    a, b = m.open("a"), m.open("b")
    m.grow(a, 7); m.commit(a, 7)
    m.grow(a, 7 + 4); m.grow(b, 34)
    batch = BatchBuilder(m, torch.device("cpu")).build([StepEntry(a, [5, 6, 7, 8], [0, 3], parents=[-1, 0, 0, 2]), StepEntry(b, list(range(34)))])       # 34 tokens: two words a row
    assert batch.positions.tolist() == [7, 8, 8, 9] + list(range(34))
    assert batch.tree.shape == (38, 2) and batch.tree[:4].tolist() == [[1, 0], [3, 0], [5, 0], [13, 0]]
    assert batch.tree[4 + 32].tolist() == [-1, 1] and batch.tree[4 + 31].tolist() == [-1, 0]
    assert BatchBuilder(m, torch.device("cpu")).build([StepEntry(a, [5, 6, 7, 8])]).tree is None
    with pytest.raises(ValueError, match="come before"):
        BatchBuilder(m, torch.device("cpu")).build([StepEntry(a, [5, 6], parents=[0, 0])])
    with pytest.raises(ValueError, match="a parent per"):
        BatchBuilder(m, torch.device("cpu")).build([StepEntry(a, [5, 6], parents=[-1])])


def test_a_window_hides_ancestors_from_a_draft():
    """Groups whose window is shorter than a branch have a tree of their own, also for a portion beside the drafts."""
    from layover_b200.engine.batch import BatchBuilder, StepEntry, tree_rows, tree_rows_in_window

    PagedKVNeed = __import__("layover_b200").parts.base.PagedKVNeed
    m = manager([PagedKVNeed(2, 16, None), PagedKVNeed(2, 16, 2), PagedKVNeed(2, 16, 5)], blocks=40)
    a, b = m.open("a"), m.open("b")
    m.grow(a, 7); m.commit(a, 7)
    m.grow(a, 7 + 5); m.grow(b, 4)
    parents = [-1, 0, 0, 2, 3]
    batch = BatchBuilder(m, torch.device("cpu")).build([StepEntry(a, [5, 6, 7, 8, 9], [0, 3], parents=parents), StepEntry(b, [1, 2, 3, 4])])
    trees = [g.tree.flatten().tolist() for g in batch.groups]
    assert trees[0] == trees[2] == batch.tree.flatten().tolist() == [0b1, 0b11, 0b101, 0b1101, 0b11101, 0b1, 0b11, 0b111, 0b1111]
    assert trees[1] == [0b1, 0b11, 0b101, 0b1100, 0b11000, 0b1, 0b11, 0b110, 0b1100]
    seen, _ = tree_rows(parents)
    assert tree_rows_in_window(parents, seen, 1) == [1 << i for i in range(5)] and tree_rows_in_window(parents, seen, 9) == seen


def test_lookup_drafts_and_the_walk_down_them():
    import layover_b200 as lb
    from layover_b200.engine.drafts import walk

    guess = lb.LookupDrafts(width=2, depth=3, context=2)
    assert guess([1, 2, 3, 4, 1, 2, 3, 9, 1, 2], 10) == ([3, 9, 1, 4, 1], [-1, 0, 1, 0, 3])      # the latest first, one common beginning
    assert guess([1, 2, 3, 4, 1, 2, 3, 9, 1, 2], 1) == ([3], [-1])
    assert guess([1, 2], 4) == ([], []) and guess([1, 2, 3], 4) == ([], []) and guess([1, 2, 1, 2], 0) == ([], [])
    assert walk([7, 3, 9, 4], [-1, 0, 1, 1], [3, 9, 7, 5]) == [0, 1, 2]
    assert walk([7, 3, 3], [-1, 0, 0], [3, 5, 5]) == [0, 1] and walk([7], [-1], [7]) == [0] and walk([7, 8], [-1, 0], [9, 8]) == [0]
