"""Operators and searches over several hypotheses of a request, at calls that their documentation allows and that are easily got wrong:
sinks of -inf, drafts and held tokens that are not finite, very many rows and requests, moves right ahead of decode attention, small pools."""

import math

import pytest
import torch

from test_gpu_hypotheses import INF, NAN, Trees, feed, fresh, ops

pytestmark = pytest.mark.gpu
BOTH = [torch.bfloat16, torch.float32]


def attend(o, pool, table, ctx, q, out, splits):
    n = ctx.numel()
    o.attention_decode_bf16(q, pool[-2], pool[-1], out, table, torch.arange(n + 1, dtype=torch.int32, device="cuda"), ctx, None, n, 32, 8, 128, 16,
                            128 ** -0.5, splits=splits)


@pytest.mark.parametrize("splits", [1, 4])
@pytest.mark.parametrize("move", ["copy", "compact"])
def test_decode_attention_right_behind_a_move_sees_the_moved_rows(move, splits):
    """One graph of a move in all planes of a large pool and the attention over the last two of them, which reads earlier keys ahead of
    its wait: the bits of a call that was waited for, and the formula's."""
    o, gen = ops(), torch.Generator(device="cuda").manual_seed(splits)
    put = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    seqs, width, planes = 8, 100, 12
    pages = 2 * seqs * width
    fresh_pool = torch.randn(planes, pages, 8, 16, 128, generator=gen, device="cuda", dtype=torch.bfloat16)
    pool = fresh_pool.clone()
    q, outs = torch.randn(seqs, 32 * 128, generator=gen, device="cuda").to(torch.bfloat16), [torch.empty(seqs, 32 * 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    table = torch.arange(seqs * width, dtype=torch.int32, device="cuda").view(seqs, width)
    if move == "copy":
        src, dst = torch.arange(seqs * width, pages, dtype=torch.int32, device="cuda"), table.flatten()
        ctx = put([width * 16 - i for i in range(seqs)])
        moved = lambda: o.copy_pages(pool, src, dst)
    else:                                                  # 700 of 1,500 drafts behind ten tokens
        picks = [sorted(torch.randperm(1500, generator=torch.Generator().manual_seed(s))[:700].tolist()) for s in range(seqs)]
        first, picked, cu = put([10] * seqs), put([p for row in picks for p in row]), put([700 * s for s in range(seqs + 1)])
        ctx = put([710] * seqs)
        moved = lambda: o.compact_tokens(pool, table, first, picked, cu)
    moved(); attend(o, pool, table, ctx, q, outs[0], splits)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moved(); attend(o, pool, table, ctx, q, outs[0], splits)
    for _ in range(5):
        pool.copy_(fresh_pool); outs[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        attend(o, pool, table, ctx, q, outs[1], splits)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
    # the formula, from the rows as they were before the move
    for s in (0, seqs - 1):
        n = int(ctx[s])
        rows = fresh_pool[-2:, src.view(seqs, width)[s].long()] if move == "copy" else fresh_pool[-2:, table[s].long()]
        rows = rows.transpose(2, 3).reshape(2, -1, 8, 128).double()
        keep = torch.arange(n, device="cuda") if move == "copy" else torch.tensor(list(range(10)) + [10 + p for p in picks[s]], device="cuda")
        k, v = rows[0][keep], rows[1][keep]
        heads = q[s].double().view(8, 4, 128)
        z = torch.einsum("hgd,khd->hgk", heads, k) * 128 ** -0.5
        p = torch.softmax(z, 2)
        want, sums = (torch.einsum("hgk,khd->hgd", p, x).flatten() for x in (v, v.abs()))
        # weights and result round to bfloat16; scores, exponentials and sums in 32 bits
        size = float((torch.einsum("hgd,khd->hgk", heads.abs(), k.abs()) * 128 ** -0.5).max())
        bound = (2 * (132 * 2.0 ** -24 * size + 2.0 ** -18) + 2 * (n + 64) * 2.0 ** -24) * sums
        bound = bound + 2.0 ** -8 * sums + 2.0 ** -8 * (want.abs() + bound)
        assert ((outs[0][s].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("held, window", [(0, 0), (100, 1), (3000, 2000)])
def test_a_row_that_sees_nothing_is_zero_also_where_its_sink_is_minus_infinity(held, window, dim, dtype):
    """One part of the keys and several; a row that sees one key has its value, as without a sink."""
    empty = torch.zeros(10, 10, dtype=torch.bool)
    empty[3, 3] = True
    case = Trees([(held, 10)], 4, 2, dim, dtype=dtype, sinks=True, window=window, seen=[empty], seed=dim).fill()
    case.sinks[1:3] = -INF
    case.positions[:10] = held + 5000                      # behind the window nothing held is seen
    got = case.run()[:10].view(10, 4, dim)
    assert (got[[0, 1, 2, 4, 5, 6, 7, 8, 9]] == 0).all()
    assert torch.equal(got[3, 1], case.v[0][held + 3, 0]) and torch.equal(got[3, 2], case.v[0][held + 3, 1])


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("q_heads, kv_heads, dim, nodes, held", [(4, 1, 128, 3, 40), (8, 2, 128, 20, 61), (4, 2, 128, 70, 1500), (32, 8, 128, 40, 900),
                                                                (8, 2, 128, 30, 9000), (8, 2, 64, 20, 700), (4, 2, 128, 200, 300)])
def test_a_draft_that_is_not_finite_changes_no_bit_of_who_does_not_see_it(q_heads, kv_heads, dim, nodes, held, dtype):
    """Neither of other requests, nor of its own request's drafts, nor of heads whose values are finite; who sees it has what the formula says."""
    lengths = [(held, nodes), (held // 2, nodes), (5, 2)]
    case = Trees(lengths, q_heads, kv_heads, dim, dtype=dtype, seed=nodes).fill()
    finite = case.run()
    case.check(finite)
    odd = (nodes // 2, nodes - 1)
    for i, (place, value) in enumerate(zip(odd, (NAN, -INF))):
        case.v[0][held + place, 0, 7 + i] = value          # the first key/value head's alone
    got = case.fill().run()
    case.check(got)
    sees = case.seen[0][:, list(odd)].any(1)
    group = q_heads // kv_heads * dim
    assert torch.equal(got[:nodes, group:], finite[:nodes, group:])
    assert torch.equal(got[:nodes][~sees], finite[:nodes][~sees])
    assert torch.equal(got[nodes:], finite[nodes:])


@pytest.mark.parametrize("dtype", BOTH)
def test_drafts_that_are_not_finite_in_many_requests(dtype):
    """Requests of several row tiles and parts of the keys, each with drafts that are not finite; the bits of two calls are the same."""
    case = Trees([(700 + 300 * i, 5 + 9 * i) for i in range(7)], 8, 2, 128, dtype=dtype, seed=3)
    for i in range(7):
        case.v[i][-1 - i, i % 2, 11 * i] = (NAN, INF, -INF)[i % 3]
    got = case.fill().run()
    case.check(got)
    assert torch.equal(torch.nan_to_num(got, 99.0), torch.nan_to_num(case.run(), 99.0))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("q_heads, kv_heads, dim", [(8, 2, 64), (8, 2, 128), (2, 1, 16)])
@pytest.mark.parametrize("window", [30, 64, 700])
def test_a_held_value_behind_a_window_reaches_only_who_sees_it(window, q_heads, kv_heads, dim, dtype):
    """Held tokens at the window's edge, which the first drafts see and the deeper ones do not, may be anything."""
    n, held = 20, 900
    case = Trees([(held, n), (held, n)], q_heads, kv_heads, dim, dtype=dtype, window=window, seen=[torch.ones(n, n).tril().bool()] * 2, seed=window)
    case.v[0][held - window + 6, :, 3], case.v[0][held - window + 11, :, dim - 1] = NAN, INF      # seen by the first 6 and 11 drafts
    got = case.fill().run()
    case.check(got)
    assert torch.isnan(got[:6].float()).any(1).all() and torch.isfinite(got[11:n]).all()


def few_keys(q, keys, values, scale):
    """(outputs, sums of weight times |value|, the largest sum of |q k|) of rows that see the same few keys each: q [R, heads, dim],
    keys and values [R, keys, dim], in 64 bits."""
    q, keys, values = q.double(), keys.double(), values.double()
    z = torch.einsum("rhd,rkd->rhk", q, keys) * scale
    p = torch.softmax(z, 2)
    return (torch.einsum("rhk,rkd->rhd", p, values), torch.einsum("rhk,rkd->rhd", p, values.abs()),
            float((torch.einsum("rhd,rkd->rhk", q.abs(), keys.abs()) * scale).max()))


def few_keys_bound(want, sums, size, dim, dtype, n_keys):
    """As `Trees.check`: a score's dim + 4 roundings, the exponential's 2^-18, a rounding of the sums for each of the keys seen and for each of the tiles
    (whose other keys add zeros); in bfloat16 the weights' and the result's."""
    step = 2.0 ** -24
    bound = (2 * ((dim + 4) * step * size + 2.0 ** -18) + 2 * (n_keys + 300) * step) * sums + 1e-30
    return bound + 2.0 ** -8 * sums + 2.0 ** -8 * (want.abs() + bound) if dtype == torch.bfloat16 else bound + step * want.abs()


@pytest.mark.parametrize("dtype, dim, heads", [(torch.bfloat16, 16, 8), (torch.bfloat16, 128, 8), (torch.float32, 16, 8)])
def test_tree_attention_of_more_than_65535_rows(dtype, dim, heads):
    """A long portion beside drafts: its last row is far behind the 65,535th. Each draft sees itself and the one before it."""
    o, n, page = ops(), 8300, 16
    gen = torch.Generator().manual_seed(dim)
    q, k, v = (torch.randn(n, h * dim, generator=gen).to(dtype) for h in (heads, 1, 1))
    words = -(-n // 32)
    tree = torch.zeros(n, words, dtype=torch.int64)
    at = torch.arange(n)
    tree[at, at // 32] |= 1 << at % 32
    tree[at[1:], at[:-1] // 32] |= 1 << at[:-1] % 32
    tree = torch.where(tree >= 1 << 31, tree - (1 << 32), tree).to(torch.int32).cuda()
    pages = -(-n // page)
    pools = [torch.zeros(pages * page, dim, dtype=dtype).index_copy_(0, at, x).view(pages, 1, page, dim).cuda() for x in (k, v)]
    put = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    out = torch.empty(n, heads * dim, dtype=dtype, device="cuda")
    o.attention_tree(q.cuda(), *pools, out, torch.arange(pages, dtype=torch.int32).view(1, -1).cuda(), put([0, n]), put([n]), None, tree, 1, heads, 1, dim,
                     page, dim ** -0.5, n, n)
    assert o.attention_tree_status() == 0
    pair = torch.stack((at[1:], at[:-1]), 1)
    want, sums, size = few_keys(q.view(n, heads, dim)[1:], k[pair], v[pair], dim ** -0.5)
    got = out.cpu().view(n, heads, dim)
    assert torch.equal(got[0], v[0].expand(heads, dim))
    assert ((got[1:].double() - want).abs() <= few_keys_bound(want, sums, size, dim, dtype, 2)).all()


@pytest.mark.parametrize("dtype, dim", [(torch.bfloat16, 16), (torch.bfloat16, 128), (torch.float32, 16)])
def test_tree_attention_of_more_than_65535_requests(dtype, dim):
    """Each holds one token and brings a draft that sees both."""
    o, n, page = ops(), 66_000, 8
    gen = torch.Generator().manual_seed(dim)
    q = torch.randn(n, 2 * dim, generator=gen).to(dtype)
    pools = [torch.randn(n, 1, page, dim, generator=gen).to(dtype) for _ in range(2)]
    order = torch.randperm(n, generator=gen)
    out = torch.empty(n, 2 * dim, dtype=dtype, device="cuda")
    o.attention_tree(q.cuda(), pools[0].cuda(), pools[1].cuda(), out, order.to(torch.int32).view(n, 1).cuda(), torch.arange(n + 1, dtype=torch.int32).cuda(),
                     torch.full((n,), 2, dtype=torch.int32, device="cuda"), None, torch.ones(n, 1, dtype=torch.int32, device="cuda"), n, 2, 1, dim, page,
                     dim ** -0.5, 1, 2)
    assert o.attention_tree_status() == 0
    want, sums, size = few_keys(q.view(n, 2, dim), pools[0][order, 0, :2], pools[1][order, 0, :2], dim ** -0.5)
    assert ((out.cpu().view(n, 2, dim).double() - want).abs() <= few_keys_bound(want, sums, size, dim, dtype, 2)).all()


def test_beam_selection_of_more_than_65535_rows():
    gen = torch.Generator().manual_seed(8)
    requests, beams, vocab, keep = 17_000, 4, 40, 5
    logits, scores = torch.randn(requests * beams, vocab, generator=gen), -3 * torch.rand(requests, beams, generator=gen)
    outs = torch.empty(requests, keep).cuda(), *(torch.empty(requests, keep, dtype=torch.int32).cuda() for _ in range(2))
    ops().beam_select(logits.cuda(), scores.cuda(), *outs)
    values, places = (scores.double()[:, :, None] + torch.log_softmax(logits.double(), 1).view(requests, beams, vocab)).flatten(1).topk(keep + 1)
    got = outs[1].cpu().long() * vocab + outs[2].cpu()
    # where two lie within 1e-7 either may come first
    apart = (values[:, :-1] - values[:, 1:]).amin(1) > 1e-6
    values, places = values[:, :keep], places[:, :keep]
    assert apart.sum() > 16_000 and torch.equal(got[apart], places[apart])
    assert ((outs[0].cpu().double() - values).abs() <= 2.0 ** -24 * values.abs() + 2.0 ** -18).all()


def test_only_a_path_down_the_last_steps_drafts_is_accepted(tiny_folders):
    """Rows that no step wrote, or that are not a branch, do not become part of a request; neither do drafts of a step before the last."""
    import layover_b200 as lb
    from conftest import random_prompt
    model = lb.load_model(str(tiny_folders["a"][0]), device="cuda", dtype="fp32")
    cache, step = fresh(model)
    seq, _ = feed(cache, step, "x", random_prompt(256, 9, 1))
    with pytest.raises(ValueError, match="last step"):
        cache.accept([(seq, [0])])                         # a step without drafts
    step([lb.StepEntry(seq, [1, 2, 3, 4], [0], [-1, 0, 0, 2])])
    (child,) = cache.fork([(seq, "child")])
    for path in ([0, 5], [1], [0, 1, 2], [0, 3], [2, 3]):
        with pytest.raises(ValueError, match="last step"):
            cache.accept([(seq, path)])
    with pytest.raises(ValueError, match="last step"):
        cache.accept([(child, [0])])                       # a fork holds what is held, and no drafts
    cache.accept([(seq, [0, 2, 3])])
    assert seq.num_tokens == 12
    with pytest.raises(ValueError, match="last step"):
        cache.accept([(seq, [0])])
    step([lb.StepEntry(seq, [1, 2], [0], [-1, 0])])
    step([lb.StepEntry(seq, [5], [0])])
    with pytest.raises(ValueError, match="last step"):
        cache.accept([(seq, [0])])
    cache.accept([(seq, []), (child, [])])
    cache.check()


def test_a_search_forks_nothing_after_its_last_step(tiny_folders):
    """A pool with room for every step, but for no fork behind the last, has all beams."""
    import layover_b200 as lb
    model = lb.load_model(str(tiny_folders["a"][0]), device="cuda", dtype="fp32")
    roomy = lb.beam_search(model, [[7]], 4, 1, block_tokens=4)
    tight = lb.beam_search(model, [[7]], 4, 1, block_tokens=4, num_blocks=1)
    assert tight == roomy and len(tight[0]) == 4


def test_more_guesses_than_there_is_room_for(tiny_folders):
    """A callable may guess as much as it likes: what the default pool has no pages for is not checked, and the text is that of fewer guesses."""
    import layover_b200 as lb
    model = lb.load_model(str(tiny_folders["a"][0]), device="cuda", dtype="fp32")
    prompts = [[5, 6, 7], [9]]
    want, _ = lb.generate_with_drafts(model, prompts, 12, lambda tokens, room: ([], []), block_tokens=4)
    every = lambda tokens, room: (list(range(256)), [-1] * 256) if room else ([], [])
    got, counts = lb.generate_with_drafts(model, prompts, 12, every, block_tokens=4)
    assert got == want and counts["drafted"] > 0


def spelled_out(cache, step, prompt, beams, new):
    """Beam search that feeds every beam's whole text anew."""
    held = [(0.0, [])]
    for _ in range(new):
        rows = []
        for score, tokens in held:
            seq, logits = feed(cache, step, "t", prompt + tokens)
            cache.close(seq)
            rows += [(score + p, tokens + [t]) for t, p in enumerate(torch.log_softmax(logits.double(), 0).tolist())]
        held = sorted(rows, key=lambda x: -x[0])[:beams]
    return held


def test_beam_search_of_a_model_whose_states_move_with_the_beams():
    import layover_b200 as lb
    model = lb.random_model(lb.preset("topidra-tiny"), seed=0, device="cuda", dtype="fp32")
    vocab = model.spec.vocab_size
    prompt = [int(t) for t in torch.randint(0, vocab, (21,), generator=torch.Generator().manual_seed(5))]
    found = lb.beam_search(model, [prompt], 3, 6, block_tokens=8, prefill_chunk=8)[0]
    cache, step = fresh(model, 400, 8)
    held = spelled_out(cache, step, prompt, 3, 6)
    assert [s for s, _ in found] == pytest.approx([s for s, _ in held], abs=2e-3)
    for (score, tokens), (want, text) in zip(found, held):
        assert tokens == text or min(abs(want - s) for s, t in held if t != text) < 1e-3


@pytest.mark.parametrize("name", ["a", "c"])
def test_beam_search_in_bfloat16_gives_the_sums_of_its_texts(tiny_folders, name):
    """Every beam's score is the sum of its tokens' log probabilities, each within the logits' tolerance on both sides of the softmax."""
    import layover_b200 as lb
    from conftest import random_prompt, tolerance
    model = lb.load_model(str(tiny_folders[name][0]), device="cuda", dtype="bf16")
    prompt = random_prompt(model.spec.vocab_size, 19, 4)
    found = lb.beam_search(model, [prompt], 4, 8, block_tokens=8)[0]
    assert len(found) == 4 and len({tuple(t) for _, t in found}) == 4 and [s for s, _ in found] == sorted((s for s, _ in found), reverse=True)
    cache, step = fresh(model)
    for i, (score, tokens) in enumerate(found):
        text = prompt + tokens
        logits = step([lb.StepEntry(cache.open(f"{i}"), text, list(range(len(prompt) - 1, len(text) - 1)))])
        sums = torch.log_softmax(logits.double(), 1).gather(1, torch.tensor(tokens, device="cuda")[:, None]).sum()
        assert abs(score - float(sums)) <= len(tokens) * 2 * tolerance(logits, model.dtype)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("sinks, softcap, window", [(True, 0.0, 0), (False, 20.0, 0), (True, 20.0, 0), (False, 0.0, 300), (True, 20.0, 40)])
@pytest.mark.parametrize("nodes, group", [(12, 4), (75, 4), (9, 1)])
def test_drafts_that_are_not_finite_with_sinks_caps_and_windows(nodes, group, sinks, softcap, window, dim, dtype):
    """Many small requests (whole row tiles in a block's share), long ones (parts of their keys), some of them with drafts that are not finite."""
    lengths = [(7 * i % 90, 1 + i % nodes) for i in range(40)] + [(2600, nodes), (1300, nodes)]
    case = Trees(lengths, 2 * group, 2, dim, dtype=dtype, sinks=sinks, softcap=softcap, window=window, seed=nodes + dim).fill()
    if sinks:
        case.sinks[0] = -INF
    finite = case.run()
    odd = {3: 0, 11: lengths[11][1] - 1, 30: lengths[30][1] // 2, 40: nodes // 2, 41: nodes - 1}
    sees = torch.zeros(sum(n for _, n in lengths), dtype=torch.bool)
    for i, place in odd.items():
        case.v[i][lengths[i][0] + place, i % 2, 5 + i % 7] = (NAN, INF, -INF)[i % 3]
        first = int(case.cu_q[i])
        sees[first: first + lengths[i][1]] = case.seen[i][:, place]
    got = case.fill().run()
    assert ops().attention_tree_status() == 0
    rows = len(sees)
    assert torch.equal(got[:rows][~sees], finite[:rows][~sees]) and (got[rows:] == 7.0).all()
    if sinks:                       # a sink of -inf beside rows that see something is no sink: heads of a finite one are compared
        case.sinks[0] = -1e30
        case.check(case.run())
    else:
        case.check(got)


def test_a_captured_call_with_drafts_that_are_not_finite():
    """Replayed on finite values, on others, and on finite ones again: the bits of calls that were not captured."""
    o = ops()
    case = Trees([(900, 6), (41, 20), (2000, 40)], 8, 2, 128, seed=11, extra_rows=0).fill()
    d = {name: getattr(case, name).cuda() for name in ("q", "k_pool", "v_pool", "table", "cu_q", "ctx", "positions", "tree")}
    out = torch.empty_like(d["q"])
    call = lambda: o.attention_tree(d["q"], d["k_pool"], d["v_pool"], out, d["table"], d["cu_q"], d["ctx"], None, d["tree"], 3, 8, 2, 128, 16, case.scale, 40, 2040)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    finite = case.v_pool.clone()
    case.v[2][2000 + 13, 1, 9], case.v[1][41, 0, 100] = NAN, INF
    odd = case.fill().v_pool
    for values in (finite, odd, finite):
        d["v_pool"].copy_(values)
        out.zero_()
        graph.replay()
        got = out.cpu()
        call()
        assert torch.equal(torch.nan_to_num(got, 99.0), torch.nan_to_num(out.cpu(), 99.0))
        if values is odd:
            case.check(got)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("held, nodes", [(256, 3), (128, 40), (1280, 3), (2560, 70)])
def test_a_draft_whose_key_is_nan_alone_in_its_part_of_the_keys(held, nodes, dim, dtype):
    """Drafts that see themselves alone begin a key tile, whose scores are one part: where its only one is NaN the row is NaN, and no other."""
    case = Trees([(held, nodes), (40, 2)], 4, 2, dim, dtype=dtype, seen=[torch.eye(nodes, dtype=torch.bool), torch.eye(2, dtype=torch.bool)], seed=held).fill()
    finite = case.run()
    case.check(finite)
    for place in (1, nodes - 1):
        case.k[0][held + place] = NAN
    got = case.fill().run()
    odd = torch.zeros(nodes + 2, dtype=torch.bool)
    odd[[1, nodes - 1]] = True
    assert torch.isnan(got[:nodes + 2][odd]).all() and torch.equal(got[:nodes + 2][~odd], finite[:nodes + 2][~odd])
