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
        assert chunks * chunk_tiles * 64 >= keys and (chunks - 1) * chunk_tiles * 64 < keys + 128
        assert chunks == 1 or n_seqs * kv_heads * row_tiles * chunks * tile_rows * (dim + 2) <= 64 << 20
    blocks, rows2, floats = ops.tree_share(n_seqs, nodes, ctx, window, q_heads, kv_heads, 148)
    assert 1 <= blocks <= 148 and rows2 == (nodes > 128 // (q_heads // kv_heads)) and floats > 2 * blocks * 128 * 130
