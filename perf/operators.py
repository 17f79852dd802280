"""Operators of decoding with several hypotheses per request, as cases to time.

  tree      `ops.attention_tree`: drafted tokens that form a tree attend over a request's paged cache and over their own ancestors
  compact   `ops.compact_tokens`: the rows of the accepted drafts move to the places right behind what the request holds, in all layers
  copy      `ops.copy_pages`: pages of a cache (or state slots) are copied for a request that is forked, in all layers
  beam      `ops.beam_select`: the best continuations of every request's beams over the whole vocabulary

Sizes are those of the package's presets and of `bench.py`: 36 layers of 32 heads over 8 of 128 channels, 16 over 4, 4 over 2 of 16 and
6 over 1 of 32 (the tiny ones), pages of 16 tokens, states of 32 x 128 x 128, vocabularies of 151,936 and 32,768.
"""

import math

import numpy as np
import torch

own = False

PAGE = 16
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
LOWEST = torch.finfo(torch.float32).min


# ------------------------------------------------------------------------------------------- the cases
def _tree(dtype="bf16", seqs=1, nodes=8, context=700, uneven=False, q_heads=32, kv_heads=8, dim=128, window=0, sinks=False, softcap=0.0, **name):
    return {**name, "kind": "tree", "dtype": dtype, "seqs": seqs, "nodes": nodes, "context": context, "uneven": uneven, "q_heads": q_heads,
            "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks, "softcap": softcap}


def _compact(dtype="bf16", seqs=8, nodes=16, accepted=4, layers=36, kv_heads=8, dim=128, **name):
    return {**name, "kind": "compact", "dtype": dtype, "seqs": seqs, "nodes": nodes, "accepted": accepted, "layers": layers, "kv_heads": kv_heads,
            "dim": dim}


def _copy(dtype="bf16", planes=72, pages=64, elements=8 * PAGE * 128, pairs=7, **name):
    return {**name, "kind": "copy", "dtype": dtype, "planes": planes, "pages": pages, "elements": elements, "pairs": pairs}


def _beam(requests=1, beams=4, keep=4, vocab=151936, room=0, masked=0.0, first=False, ended=False, **name):
    return {**name, "kind": "beam", "requests": requests, "beams": beams, "keep": keep, "vocab": vocab, "room": room, "masked": masked,
            "first": first, "ended": ended}


def listed():
    return [
        # one chat whose next tokens are guessed: few rows over a short cache, launches count
        _tree(name="tree 1 x 8 over 700", seqs=1, nodes=8, context=700),
        # the benchmark's headline batch with drafts: eight requests in the middle of their answers, 32 drafts each
        _tree(name="tree 8 x 32 over 3000", seqs=8, nodes=32, context=3000),
        # a full server, requests of all lengths with trees of all sizes: the bytes of the cache count
        _tree(name="tree 40 x 25 over 8000 uneven", seqs=40, nodes=25, context=8000, uneven=True),
        # wide trees of one long document: many rows for every key
        _tree(name="tree 2 x 64 over 12345 16/4", seqs=2, nodes=64, context=12345, q_heads=16, kv_heads=4),
        # a windowed, capped design with sinks and smaller heads, odd sizes
        _tree(name="tree 5 x 13 window 12/2 of 64", seqs=5, nodes=13, context=1531, uneven=True, q_heads=12, kv_heads=2, dim=64, window=1024,
              sinks=True, softcap=30.0),
        # the true 32-bit path, in which users compare logits
        _tree(name="fp32 tree 4 x 13 over 900", dtype="fp32", seqs=4, nodes=13, context=900),
        # one request's accepted drafts move into place after a step
        _compact(name="compact 1", seqs=1, nodes=8, accepted=4),
        # a full server's
        _compact(name="compact 64", seqs=64, nodes=25, accepted=5),
        # eight requests whose beams are forked: the page that is still being written is copied in all layers
        _copy(name="copy 56 pages", pairs=56, pages=160),
        # states of a recurrent design move with their beams
        _copy(name="copy 24 states", dtype="fp32", planes=3, pages=64, elements=32 * 128 * 128, pairs=24),
        # one request's four beams, latency
        _beam(name="beam 1 x 4", requests=1, beams=4, keep=4),
        # a server of 16 requests, twice as many candidates as beams, some of them ended, tokens banned
        _beam(name="beam 16 x 8 keep 16", requests=16, beams=8, keep=16, masked=0.02, ended=True),
    ]


def draw(rng):
    def spread(low, high):                      # an odd size as likely as an even one, even over the logarithm
        return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))

    kind = rng.choice(("tree", "tree", "tree", "compact", "copy", "beam", "beam"))
    if kind == "tree":
        fp32 = rng.random() < 0.25
        q_heads, kv_heads, dim = rng.choice(((32, 8, 128), (32, 8, 128), (16, 4, 128), (64, 8, 128), (12, 2, 64), (6, 1, 32), (4, 2, 16), (8, 8, 128)))
        seqs, nodes = spread(1, 8 if fp32 else 40), spread(1, 24 if fp32 else 64)
        context = spread(1, min(2000, 6000 // seqs) if fp32 else min(16000, 160_000 // seqs))
        extra = rng.random() < 0.3
        return _tree("fp32" if fp32 else "bf16", seqs, nodes, context, rng.random() < 0.5, q_heads, kv_heads, dim,
                     spread(16, 2048) if extra and rng.random() < 0.7 else 0, extra and rng.random() < 0.5, 30.0 if extra and rng.random() < 0.5 else 0.0)
    if kind == "compact":
        nodes = spread(2, 64)
        dtype, dim = rng.choice((("bf16", 128), ("bf16", 128), ("bf16", 64), ("fp32", 128), ("fp32", 20)))
        return _compact(dtype, spread(1, 48), nodes, spread(1, min(8, nodes)), rng.choice((2, 4, 24, 36)), rng.choice((1, 2, 4, 8)), dim)
    if kind == "copy":
        dtype, elements, planes = rng.choice((("bf16", 8 * PAGE * 128, 72), ("bf16", 4 * PAGE * 128, 8), ("fp32", PAGE * 20, 4), ("fp32", 32 * 128 * 128, 3),
                                              ("fp32", spread(1, 5000), 5)))
        return _copy(dtype, planes, 100, elements, spread(1, 24 if elements > 100_000 else 48))
    beams = spread(1, 16)
    requests = spread(1, max(1, 64 // beams))
    vocab = rng.choice((151936, 32768, spread(300, 160_000), spread(300, 160_000)))
    return _beam(requests, beams, min(32, beams * rng.choice((1, 1, 2))), vocab, rng.choice((0, 0, 5)), rng.choice((0.0, 0.02, 0.5)),
                 beams > 1 and rng.random() < 0.3, rng.random() < 0.4)


# ------------------------------------------------------------------------------------------- inputs
class _State:
    pass


def _lengths(case):
    """(tokens a request holds, its drafts), in the order of the batch."""
    n = case["seqs"]
    if not case["uneven"] or n == 1:
        return [(case["context"], case["nodes"])] * n
    share = [(i * 7919) % n / (n - 1) for i in range(n)]
    return [(round(case["context"] * (0.1 + 0.9 * s)), max(1, round(case["nodes"] * (1 - 0.7 * s)))) for s in share]


def _parents(rng, nodes):
    """A tree as a drafter makes it: a few first guesses, then continuations of what came before; -1 hangs on the request's last token."""
    return [-1 if i < 2 or rng.random() < 0.1 else int(rng.integers(max(0, i - 6), i)) for i in range(nodes)]


def _tables(rng, needed, pages):
    order = rng.permutation(pages)[:sum(needed)].tolist()
    table = np.full((len(needed), max(needed)), pages, dtype=np.int32)          # behind a request's pages: the scratch page
    for i, n in enumerate(needed):
        table[i, :n] = [order.pop() for _ in range(n)]
    return table


def _prepare_tree(s, case, seed):
    rng, gen, dtype = np.random.default_rng(seed), torch.Generator(device="cuda").manual_seed(seed), TYPES[case["dtype"]]
    lengths = _lengths(case)
    words = -(-max(n for _, n in lengths) // 32)
    bits, positions = [], []
    for held, n in lengths:
        rows, depth = [], []
        for i, p in enumerate(_parents(rng, n)):
            rows.append((rows[p] if p >= 0 else 0) | 1 << i)
            depth.append(depth[p] + 1 if p >= 0 else 0)
        if case["window"]:                      # an ancestor may lie behind the window too
            rows = [sum(1 << j for j in range(n) if r >> j & 1 and depth[i] - depth[j] < case["window"]) for i, r in enumerate(rows)]
        bits += [[(r >> 32 * w) & 0xFFFFFFFF for w in range(words)] for r in rows]
        positions += [held + d for d in depth]
    s.n_seqs, s.max_nodes, s.max_ctx = len(lengths), max(n for _, n in lengths), max(h + n for h, n in lengths)
    tokens = sum(n for _, n in lengths)
    put = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    s.tree = torch.from_numpy(np.array(bits, dtype=np.uint32).view(np.int32)).cuda()
    s.positions, s.cu_q = put(positions), put(np.cumsum([0] + [n for _, n in lengths]))
    s.ctx_len = put([h + n for h, n in lengths])
    needed = [-(-(h + n) // PAGE) for h, n in lengths]
    pages = sum(needed) + 3
    s.block_table = torch.from_numpy(_tables(rng, needed, pages)).cuda()
    q_heads, kv_heads, dim = case["q_heads"], case["kv_heads"], case["dim"]
    s.q = torch.randn((tokens, q_heads * dim), generator=gen, device="cuda").to(dtype)
    s.pool = torch.full((2, pages + 1, kv_heads, PAGE, dim), float("nan"), dtype=dtype, device="cuda")      # what no request wrote may be anything
    for i, (h, n) in enumerate(lengths):
        at = torch.arange(h + n, device="cuda")
        page, slot = s.block_table[i].long()[at // PAGE], at % PAGE
        s.pool[0][page, :, slot] = torch.randn((h + n, kv_heads, dim), generator=gen, device="cuda").to(dtype)
        s.pool[1][page, :, slot] = torch.randn((h + n, kv_heads, dim), generator=gen, device="cuda").to(dtype)
    s.sinks = torch.randn(q_heads, generator=gen, device="cuda") if case["sinks"] else None
    s.scale = dim ** -0.5
    s.out = torch.empty_like(s.q)


def _accepted(case):
    """How many of its drafts every request keeps."""
    return [1 + (i * 7919 + case["accepted"] - 1) % case["accepted"] for i in range(case["seqs"])]


def _prepare_compact(s, case, seed):
    rng, gen, dtype = np.random.default_rng(seed), torch.Generator(device="cuda").manual_seed(seed), TYPES[case["dtype"]]
    held = rng.integers(1, 5 * PAGE, case["seqs"])
    needed = [-(-int(h + case["nodes"]) // PAGE) for h in held]
    pages = case["seqs"] * -(-(5 * PAGE + case["nodes"]) // PAGE) + 2
    s.block_table = torch.from_numpy(_tables(rng, needed, pages)).cuda()
    paths = [sorted(rng.choice(case["nodes"], count, replace=False).tolist()) for count in _accepted(case)]       # a path down a tree
    put = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    s.first, s.picked = put(held), put([p for path in paths for p in path])
    s.cu_picked = put(np.cumsum([0] + [len(p) for p in paths]))
    s.pool = torch.empty((case["layers"] * 2, pages + 1, case["kv_heads"], PAGE, case["dim"]), dtype=dtype, device="cuda").normal_(generator=gen)


def _prepare_copy(s, case, seed):
    rng, gen = np.random.default_rng(seed), torch.Generator(device="cuda").manual_seed(seed)
    free = max(1, min(case["pairs"], case["pages"] - 1))
    order = rng.permutation(case["pages"])
    s.dst = torch.tensor(order[:free], dtype=torch.int32, device="cuda")
    s.src = torch.tensor(rng.choice(order[free:], free), dtype=torch.int32, device="cuda")      # several may have one source
    s.pool = torch.empty((case["planes"], case["pages"], case["elements"]), dtype=TYPES[case["dtype"]], device="cuda").normal_(generator=gen)


def _prepare_beam(s, case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab = case["requests"] * case["beams"], case["vocab"]
    logits = torch.randn((rows, vocab + case["room"]), generator=gen, device="cuda") * 2.5
    logits += torch.randn(vocab + case["room"], generator=gen, device="cuda") * 1.5             # some tokens are frequent whatever came before
    if case["masked"]:
        banned = torch.rand((rows, vocab + case["room"]), generator=gen, device="cuda")
        logits.masked_fill_(banned < case["masked"], -math.inf)
        logits.masked_fill_((banned > 0.9) & (banned < 0.9 + 0.01), LOWEST)
    s.logits = logits[:, :vocab]
    s.scores = -8 * torch.rand((case["requests"], case["beams"]), generator=gen, device="cuda").sort(dim=1).values - 3
    if case["first"]:                                             # a request's first step: one beam alone holds its prompt
        s.scores[::2, 0], s.scores[::2, 1:] = 0.0, -math.inf
    s.ended = (torch.rand((case["requests"], case["beams"]), generator=gen, device="cuda") < 0.2).int() if case["ended"] else None
    s.pad = 1
    shape = (case["requests"], case["keep"])
    s.next_scores = torch.empty(shape, device="cuda")
    s.parents, s.tokens = (torch.empty(shape, dtype=torch.int32, device="cuda") for _ in range(2))


def prepare(case, seed):
    s = _State()
    s.case = case
    {"tree": _prepare_tree, "compact": _prepare_compact, "copy": _prepare_copy, "beam": _prepare_beam}[case["kind"]](s, case, seed)
    return s


# ------------------------------------------------------------------------------------------- the plain forms
def _plain_tree(s):
    c = s.case
    q_heads, kv_heads, dim = c["q_heads"], c["kv_heads"], c["dim"]
    group, device = q_heads // kv_heads, s.q.device
    n = (s.cu_q[1:] - s.cu_q[:-1]).long()
    first = s.ctx_len.long() - n
    at = torch.arange(s.max_ctx, device=device)
    there = at < s.ctx_len[:, None]                                                              # [S, keys]
    page = s.block_table.long()[:, at // PAGE]
    k, v = (torch.where(there[..., None, None], x[page, :, at % PAGE].float(), 0.0) for x in s.pool)         # [S, keys, kv_heads, dim]
    node = torch.arange(s.max_nodes, device=device)
    row = torch.minimum(s.cu_q[:-1, None].long() + node, s.cu_q[1:, None].long() - 1)           # [S, nodes], the last node again behind the last
    q = s.q.float().view(-1, kv_heads, group, dim)[row]                                         # [S, nodes, kv_heads, group, dim]
    scores = torch.einsum("snhgd,skhd->shgnk", q, k) * s.scale
    if c["softcap"]:
        scores = c["softcap"] * torch.tanh(scores / c["softcap"])
    own_place = at - first[:, None]                                                              # the draft that a key belongs to
    word = s.tree[row].gather(2, (own_place.clamp(0, s.max_nodes - 1) // 32)[:, None, :].expand(-1, s.max_nodes, -1))
    drafted = (word >> (own_place.clamp(min=0) % 32)[:, None, :]) & 1 == 1
    held = torch.ones_like(drafted)
    if c["window"]:
        held = s.positions.long()[row][:, :, None] - at < c["window"]
    seen = (torch.where((own_place < 0)[:, None, :], held, drafted) & there[:, None, :])[:, None, None]
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    if s.sinks is not None:
        sink = s.sinks.view(1, kv_heads, group, 1, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    weights = torch.exp(scores - top)
    total = weights.sum(dim=-1, keepdim=True)
    if s.sinks is not None:
        total = total + torch.exp(sink - top)
    out = torch.einsum("shgnk,skhd->snhgd", weights / torch.where(total == 0, 1.0, total), v)
    return out[node < n[:, None]].reshape(-1, q_heads * dim).to(s.q.dtype)


def _plain_compact(s):
    count = (s.cu_picked[1:] - s.cu_picked[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(count.numel(), device=count.device), count, output_size=s.picked.numel())
    place = torch.arange(s.picked.numel(), device=count.device) - s.cu_picked.long()[seq]
    source, target = s.first.long()[seq] + s.picked, s.first.long()[seq] + place
    table = s.block_table.long()
    rows = s.pool[:, table[seq, source // PAGE], :, source % PAGE]
    s.pool[:, table[seq, target // PAGE], :, target % PAGE] = rows
    return s.pool


def _plain_copy(s):
    s.pool[:, s.dst.long()] = s.pool[:, s.src.long()]
    return s.pool


def _plain_beam(s):
    c = s.case
    requests, beams, keep, vocab = c["requests"], c["beams"], c["keep"], c["vocab"]
    x = s.logits.double().view(requests, beams, vocab)
    top = x.amax(dim=2, keepdim=True)
    logp = x - top - (x - top).exp().sum(dim=2, keepdim=True).log()
    found = s.scores.double()[:, :, None] + logp
    found = torch.where(s.scores[:, :, None] == -math.inf, -math.inf, found)
    if s.ended is not None:                                       # an ended beam goes on as it is
        stays = torch.arange(vocab, device=x.device) == s.pad
        found = torch.where(s.ended[:, :, None] != 0, torch.where(stays, s.scores.double()[:, :, None], -math.inf), found)
    values, places = found.view(requests, -1).sort(dim=1, descending=True, stable=True)
    values, places = values[:, :keep], places[:, :keep]
    none = values == -math.inf
    return values.float(), torch.where(none, -1, places // vocab).int(), torch.where(none, -1, places % vocab).int()


def run(s):
    kind = s.case["kind"]
    if not own:
        return {"tree": _plain_tree, "compact": _plain_compact, "copy": _plain_copy, "beam": _plain_beam}[kind](s)
    from layover_b200 import ops

    c = s.case
    if kind == "tree":
        return ops.attention_tree(s.q, s.pool[0], s.pool[1], s.out, s.block_table, s.cu_q, s.ctx_len, s.positions, s.tree, s.n_seqs, c["q_heads"],
                                  c["kv_heads"], c["dim"], PAGE, s.scale, s.max_nodes, s.max_ctx, window=c["window"], sinks=s.sinks,
                                  softcap=c["softcap"])
    if kind == "compact":
        return ops.compact_tokens(s.pool, s.block_table, s.first, s.picked, s.cu_picked)
    if kind == "copy":
        return ops.copy_pages(s.pool, s.src, s.dst)
    ops.beam_select(s.logits, s.scores, s.next_scores, s.parents, s.tokens, ended=s.ended, pad=s.pad)
    return s.next_scores, s.parents, s.tokens


# ------------------------------------------------------------------------------------------- the definitions, in 64 bits
def _exact_tree(s):
    c = s.case
    kv_heads, group = c["kv_heads"], c["q_heads"] // c["kv_heads"]
    outs, cu, ctx = [], s.cu_q.tolist(), s.ctx_len.tolist()
    tree, positions = s.tree.cpu().numpy().view(np.uint32), s.positions.tolist()
    for i, (lo, hi) in enumerate(zip(cu, cu[1:])):
        n, held = hi - lo, ctx[i] - (hi - lo)
        pages = s.block_table[i, : -(-ctx[i] // PAGE)].long()
        keys, values = (x[pages].transpose(1, 2).reshape(-1, kv_heads, c["dim"])[: ctx[i]].double() for x in s.pool)
        seen = torch.zeros((n, ctx[i]), dtype=torch.bool)
        for t in range(n):
            seen[t, max(0, positions[lo + t] - c["window"] + 1) if c["window"] else 0: held] = True
            for j in range(n):
                seen[t, held + j] = bool(tree[lo + t, j // 32] >> np.uint32(j % 32) & np.uint32(1))
        seen = seen.cuda()
        heads = []
        for h in range(c["q_heads"]):
            z = s.q[lo:hi, h * c["dim"]: (h + 1) * c["dim"]].double() @ keys[:, h // group].T * s.scale
            if c["softcap"]:
                z = c["softcap"] * torch.tanh(z / c["softcap"])
            z = z.masked_fill(~seen, -math.inf)
            if s.sinks is not None:
                z = torch.cat((z, s.sinks[h].double().expand(n, 1)), dim=1)
            heads.append(torch.softmax(z, dim=1)[:, : ctx[i]] @ values[:, h // group])
        outs.append(torch.cat(heads, dim=1))
    return torch.cat(outs)


def _exact_moves(s):
    before = s.pool.clone()
    if s.case["kind"] == "copy":
        for a, b in zip(s.src.tolist(), s.dst.tolist()):
            s.pool[:, b] = before[:, a]
        return s.pool
    cu, table, picked = s.cu_picked.tolist(), s.block_table.tolist(), s.picked.tolist()
    for i, held in enumerate(s.first.tolist()):
        for place, node in enumerate(picked[cu[i]: cu[i + 1]]):
            a, b = held + node, held + place
            s.pool[:, table[i][b // PAGE], :, b % PAGE] = before[:, table[i][a // PAGE], :, a % PAGE]
    return s.pool


def _exact_beam(s):
    c = s.case
    logits, scores = s.logits.cpu().numpy().astype(np.float64), s.scores.cpu().numpy().astype(np.float64)
    ended = s.ended.cpu().numpy() if s.ended is not None else np.zeros(scores.shape, dtype=np.int32)
    outs = []
    for r in range(c["requests"]):
        found = np.full((c["beams"], c["vocab"]), -np.inf)
        for b in range(c["beams"]):
            z = logits[r * c["beams"] + b]
            if ended[r, b]:
                found[b, s.pad] = scores[r, b]
            elif scores[r, b] > -np.inf:
                found[b] = scores[r, b] + (z - (z.max() + math.log(np.exp(z - z.max()).sum())))
        best = np.argsort(-found.reshape(-1), kind="stable")[: c["keep"]]
        outs.append([(found.flat[p], p // c["vocab"], p % c["vocab"]) if found.flat[p] > -np.inf else (-np.inf, -1, -1) for p in best])
    return tuple(torch.tensor([[x[k] for x in row] for row in outs], dtype=t) for k, t in ((0, torch.float64), (1, torch.int32), (2, torch.int32)))


def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "compact": _exact_moves, "copy": _exact_moves, "beam": _exact_beam}[case["kind"]](s)


# ------------------------------------------------------------------------------------------- work
def work(case):
    size = {"bf16": 2, "fp32": 4}.get(case.get("dtype"), 4)
    if case["kind"] == "tree":
        lengths, window = _lengths(case), case["window"]
        keys = sum(n + (min(h, window) if window else h) for h, n in lengths)
        pairs = sum(n * ((min(h, window) if window else h) + 4) for h, n in lengths)            # a draft has about four ancestors
        tokens = sum(n for _, n in lengths)
        return {"bytes": size * case["dim"] * (2 * keys * case["kv_heads"] + 2 * tokens * case["q_heads"]),
                "flops": 4 * case["dim"] * case["q_heads"] * pairs}
    if case["kind"] == "compact":
        # the drafts kept, but for those that stand at their place already (all before them are kept too)
        moved = sum(1 - math.comb(case["nodes"] - i - 1, n - i - 1) / math.comb(case["nodes"], n) for n in _accepted(case) for i in range(n))
        return {"bytes": 2 * moved * 2 * case["layers"] * case["kv_heads"] * case["dim"] * size, "flops": 0}
    if case["kind"] == "copy":
        pairs = max(1, min(case["pairs"], case["pages"] - 1))
        sources = min(pairs, case["pages"] - pairs)
        return {"bytes": (pairs + sources * (1 - (1 - 1 / sources) ** pairs)) * case["planes"] * case["elements"] * size, "flops": 0}
    rows = case["requests"] * case["beams"]
    return {"bytes": 4 * rows * case["vocab"] + 12 * case["requests"] * case["keep"], "flops": 3 * rows * case["vocab"]}
