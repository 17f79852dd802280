"""Several hypotheses of a request on the host: limits that the operators name, books that stay whole, refusals of the searches and of the
command line."""

import pytest
import torch

from layover_b200 import ops
from layover_b200.parts import PartSpec

I32 = torch.int32


# ------------------------------------------------------------------------------- limits
@pytest.mark.parametrize("requests, beams, vocab", [(1, 1, 2 ** 31 - 3600), (1, 1, 2 ** 31 - 2 ** 15 + 1), (1, 64, 2 ** 25), (2, 3, 2 ** 30)])
def test_beam_selection_names_its_largest_sizes(requests, beams, vocab):
    """Places of beams x vocabulary, and the ends of the pieces that are read ahead, are counted in 32 bits."""
    f = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device="meta")
    with pytest.raises(ValueError, match="at most"):
        ops.beam_select(f(requests * beams, vocab), f(requests, beams), f(requests, 4), f(requests, 4, dtype=I32), f(requests, 4, dtype=I32))


@pytest.mark.parametrize("call, message", [
    (lambda m: ops.copy_pages(m(2, 3, 4), m(65_536, dtype=I32), m(65_536, dtype=I32)), "at most 65535"),
    (lambda m: ops.copy_pages(m(65_536, 3, 4), m(1, dtype=I32), m(1, dtype=I32)), "at most 65535"),
    (lambda m: ops.compact_tokens(m(2, 3, 1, 4, 4), m(65_536, 2, dtype=I32), m(65_536, dtype=I32), m(5, dtype=I32), m(65_537, dtype=I32)), "at most 65535"),
    (lambda m: ops.compact_tokens(m(2 ** 16, 1, 2 ** 10, 1, 2 ** 9), m(1, 2, dtype=I32), m(1, dtype=I32), m(5, dtype=I32), m(2, dtype=I32)), "at most"),
])
def test_moves_name_their_largest_sizes(call, message):
    with pytest.raises(ValueError, match=message):
        call(lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device="meta"))


# ------------------------------------------------------------------------------- books
def manager(blocks=20, page=4, max_requests=8):
    from layover_b200.cache import CacheManager
    from layover_b200.parts.base import PagedKVNeed, StateNeed

    needs = [PagedKVNeed(2, 16, None), PagedKVNeed(2, 16, 6), StateNeed((3,), torch.float32)]
    return CacheManager([(i, n, None) for i, n in enumerate(needs)], blocks, page, torch.float32, None, max_requests)


@pytest.mark.parametrize("path", [[0, 3], [1], [0, 1, 2], [2], [0, 4]])
def test_accepted_drafts_are_a_branch_of_what_the_last_step_brought(path):
    m = manager()
    a = m.open("a")
    m.grow(a, 13)
    a.drafts = [-1, 0, 0, 1]                             # as a step leaves them
    with pytest.raises(ValueError, match="last step"):
        m.accept([(a, path)])
    assert a.num_tokens == 0 and a.drafts == [-1, 0, 0, 1]
    m.accept([(a, [0, 1, 3])])
    assert a.num_tokens == 3 and a.drafts == []
    with pytest.raises(ValueError, match="last step"):
        m.accept([(a, [0])])
    m.accept([(a, [])])
    m.check()


def test_a_fork_whose_copies_fail_leaves_the_books_as_they_were(monkeypatch):
    m = manager()
    a = m.open("a")
    m.grow(a, 10); m.commit(a, 10)
    m.device = torch.device("cpu")                        # rows would be moved, and that raises: no CPU path
    m.paged[0].pool = torch.zeros(1, 2, 21, 2, 4, 16)
    monkeypatch.setattr(m, "_need_kernels", lambda: None)
    free, slots, tables = m.num_free, m.num_free_slots, [list(t.blocks) for t in a.tables]
    with pytest.raises(ops.KernelError, match="no CPU path"):
        m.fork([(a, "b"), (a, "c")])
    m.check()
    assert (set(m.live), m.num_free, m.num_free_slots, [t.blocks for t in a.tables]) == ({"a"}, free, slots, tables)
    assert all(m.paged[0].allocator.holders(b) == 1 for b in a.tables[0].blocks)
    m.device = None
    (b,) = m.fork([(a, "b")])                             # and the ids are free
    m.close(a); m.close(b)
    m.check()


# ------------------------------------------------------------------------------- which models take drafts, and with what
def one_block(block):
    """A model of one block, without weights."""
    from types import SimpleNamespace

    from layover_b200.models.model import Model
    from layover_b200.parts import build_part

    model = Model.__new__(Model)
    model.blocks, model.final_norm = [build_part("block", block, "")], build_part("norm", NORM, "")
    model.spec = SimpleNamespace(schedule=[SimpleNamespace(layer=0, reads_cache_of=None)])
    return model


NORM = PartSpec("rmsnorm", {"dim": 16, "eps": 1e-5, "weight": "n"})
ATTENTION = dict(hidden=16, q_heads=2, kv_heads=1, head_dim=16, q="q", k="k", v="v", o="o")
STREAMS = dict(streams=2, hidden=16, connections=[{k: f"h{q}.{k}" for k in ("in", "out", "mix")} for q in (1, 2)], input_norm=NORM,
               mixer=PartSpec("attention", ATTENTION))


def test_a_block_that_keeps_a_state_beside_its_attention_takes_no_drafts():
    """A token shift mixes what stands next to one another, which drafts of a tree do not."""
    assert one_block(PartSpec("hyper_connected", STREAMS)).takes_drafts
    assert not one_block(PartSpec("hyper_connected", dict(STREAMS, shift="shift"))).takes_drafts
    assert not one_block(PartSpec("hyper_connected", dict(STREAMS, mixer=PartSpec("attention", dict(ATTENTION, sink="s"))))).takes_drafts


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_model_that_takes_drafts_lists_their_kernels(dtype):
    """Where a bounded wait of theirs runs out, the sampled step behind it says so: the error words read are those of the libraries listed."""
    from layover_b200.models.runtime import Runtime

    model = one_block(PartSpec("hyper_connected", STREAMS))
    assert model.takes_drafts and "attention_tree" in model.kernel_libraries(dtype, Runtime(dtype, torch.device("cpu"), None))
    sinks = one_block(PartSpec("hyper_connected", dict(STREAMS, mixer=PartSpec("attention", dict(ATTENTION, sink="s")))))
    assert "attention_tree" not in sinks.kernel_libraries(dtype, Runtime(dtype, torch.device("cpu"), None))


def test_lookup_drafts_without_width_or_depth_guess_nothing():
    import layover_b200 as lb

    text = [1, 2, 3, 1, 2, 4, 1, 2]
    assert lb.LookupDrafts(width=0, depth=3)(text, 5) == ([], []) and lb.LookupDrafts(width=2, depth=0)(text, 5) == ([], [])
    assert lb.LookupDrafts(width=1, depth=3)(text, 5) == ([4, 1, 2], [-1, 0, 1])


# ------------------------------------------------------------------------------- command line
@pytest.mark.parametrize("options, message", [
    (["--drafts", "-3"], "positive"), (["--beams", "-1"], "1 to 32"), (["--beams", "40"], "1 to 32"), (["--drafts", "4", "--beams", "2"], "exclude"),
    (["--beams", "2", "--temperature", "0.5"], "exclude"), (["--beams", "2", "--cuda-graphs"], "--cuda-graphs"), (["--drafts", "2", "--max-batch", "8"], "--max-batch"),
    (["--drafts", "2", "--pool-gib", "2.0"], "--pool-gib"), (["--beams", "2", "--max-batched-tokens", "64"], "--max-batched-tokens"),
])
def test_command_line_refuses_what_beams_and_drafts_do_not_take(options, message, capsys):
    from layover_b200.__main__ import parse_args

    with pytest.raises(SystemExit):
        parse_args(["--preset", "tiny-b", "--random-weights", "--prompt-lens", "9", *options])
    assert message in capsys.readouterr().err


def test_command_line_keeps_its_defaults():
    from layover_b200.__main__ import parse_args

    args = parse_args(["--preset", "tiny-b"])
    assert (args.pool_gib, args.max_batch, args.max_batched_tokens, args.cuda_graphs, args.beams, args.drafts) == (2.0, 32, None, False, 0, 0)
    assert parse_args(["--preset", "tiny-b", "--max-batch", "4", "--pool-gib", "0.5"]).max_batch == 4
    assert parse_args(["--preset", "tiny-b", "--beams", "32", "--num-blocks", "9"]).beams == 32


# ------------------------------------------------------------------------------- trees behind a window
def test_windows_over_trees_and_over_long_portions():
    """Itself and the nearest ancestors; a portion of thousands of tokens beside drafts takes no memory for every pair of them."""
    import random
    import tracemalloc

    from layover_b200.engine.batch import tree_rows, tree_rows_in_window

    rng = random.Random(5)
    for n in (1, 2, 40, 130):
        parents = [-1 if i == 0 or rng.random() < 0.1 else rng.randint(max(0, i - 4), i - 1) for i in range(n)]
        for window in (1, 2, 5, 8, 1000):
            want = []
            for i in range(n):
                bits, at = 0, i
                for _ in range(window):
                    if at >= 0:
                        bits, at = bits | 1 << at, parents[at]
                want.append(bits)
            assert tree_rows_in_window(parents, tree_rows(parents)[0], window) == want
    chain = list(range(-1, 8191))
    seen, _ = tree_rows(chain)
    tracemalloc.start()
    rows = tree_rows_in_window(chain, seen, 4096)
    peak = tracemalloc.get_traced_memory()[1]
    tracemalloc.stop()
    assert rows[8191] == ((1 << 4096) - 1) << 4096 and peak < 32 << 20
