"""Beam search over the paged cache: every request follows its `beams` most likely continuations.

A beam is a request of the cache. After each step the best continuations of a request's beams over the whole
vocabulary are chosen on the device (`ops.beam_select`); a beam with several of them is forked for all but one
(`CacheManager.fork`: its full pages are shared, the page that is being written and the states are copied), a beam with none
is closed. Nothing is moved for a beam that goes on alone. The reference has no beam search (it samples greedily,
layover/engine.py:139-141).
"""

from __future__ import annotations

import torch

from .. import ops
from .batch import StepEntry


def beam_search(model, prompts: list[list[int]], beams: int = 4, max_new_tokens: int = 16, stop_tokens=frozenset(), num_blocks: int | None = None,
                block_tokens: int = 16, prefill_chunk: int = 512) -> list[list[tuple[float, list[int]]]]:
    """For every prompt its `beams` best continuations, best first, as (log probability, new tokens). A continuation that ends with a
    stop token stays as it is, and keeps its place as long as no other has a larger sum."""
    from .. import PagedKVCache
    from .step import StepFunction

    if not 1 <= beams <= ops.BEAM_MAX_KEEP:
        raise ValueError(f"beams is 1..{ops.BEAM_MAX_KEEP}")
    if any(not p for p in prompts) or max_new_tokens < 1:
        raise ValueError("a prompt needs tokens, and max_new_tokens is at least 1")
    longest = max((len(p) for p in prompts), default=0) + max_new_tokens
    if longest > model.spec.max_position:
        raise ValueError(f"{longest} tokens are more than the model's {model.spec.max_position} positions")
    if num_blocks is None:           # every beam's own pages, and as many again while some are forked and others not closed yet
        own = -(-max_new_tokens // block_tokens) + 2
        num_blocks = sum(-(-len(p) // block_tokens) + 2 * beams * own for p in prompts)
    cache = PagedKVCache(model, max(1, num_blocks), block_tokens=block_tokens, max_requests=max(1, 2 * beams * len(prompts)))
    step, device = StepFunction(model, cache), model.device
    status, names = ops.status_words(device, model.kernel_libraries(model.dtype))
    count, made = len(prompts), 0
    if not count:
        return []
    heads = [cache.open(f"{r}") for r in range(count)]
    for seq, prompt in zip(heads, prompts):                 # all but the last token of the prompts
        for at in range(0, len(prompt) - 1, prefill_chunk):
            step([StepEntry(seq, prompt[at: min(at + prefill_chunk, len(prompt) - 1)])])
    # a request's beams in the order of its rows; None: not there. Its first step is of one beam alone
    rows = [[seq] + [None] * (beams - 1) for seq in heads]
    texts = [[list(p[-1:])] + [None] * (beams - 1) for p in prompts]
    ended = torch.zeros((count, beams), dtype=torch.int32)
    scores = torch.full((count, beams), float("-inf"), device=device)
    scores[:, 0] = 0.0
    logits = torch.zeros((count * beams, model.spec.vocab_size), device=device)
    found_before = None
    parents, tokens = (torch.empty((count, beams), dtype=torch.int32, device=device) for _ in range(2))
    for left in range(max_new_tokens - 1, -1, -1):
        places = [(r, b) for r in range(count) for b in range(beams) if rows[r][b] is not None]
        if not places:
            break
        found = step([StepEntry(rows[r][b], [texts[r][b][-1]], [0]) for r, b in places])
        if len(places) == count * beams:
            logits = found
        else:                                                # rows of beams that are not there are not looked at
            if logits is found_before:
                logits = torch.zeros_like(logits)
            logits[torch.tensor([r * beams + b for r, b in places], device=device)] = found
        found_before = found
        chosen = torch.empty_like(scores)
        ops.beam_select(logits, scores, chosen, parents, tokens, ended=ended.to(device))
        if status is not None:
            check = torch.empty(1 + status.shape[0], dtype=torch.int32, device=device)
            codes = ops.sample(logits[:1], check, status=status)[1:].tolist()
            if any(codes):
                ops.reset_after_error(device)
                raise ops.KernelError("a kernel gave up waiting: " + ", ".join(f"{n}: code {c}" for n, c in zip(names, codes) if c))
        scores = chosen
        from_beam, next_token = parents.tolist(), tokens.tolist()
        forks, keeps, next_rows, next_texts, next_ended = [], set(), [], [], torch.zeros_like(ended)
        for r in range(count):
            row, text = [None] * beams, [None] * beams
            for k, (b, token) in enumerate(zip(from_beam[r], next_token[r])):
                if b < 0:
                    continue
                if ended[r, b]:
                    text[k], next_ended[r, k] = texts[r][b], 1
                    continue
                text[k] = texts[r][b] + [token]
                if token in stop_tokens:
                    next_ended[r, k] = 1
                elif id(rows[r][b]) not in keeps:
                    keeps.add(id(rows[r][b]))
                    row[k] = rows[r][b]
                else:
                    forks.append((rows[r][b], f"{r}.{made}", r, k))
                    made += 1
            next_rows.append(row)
            next_texts.append(text)
        texts = next_texts
        if not left:                                         # nobody goes on: the texts are all that is wanted
            break
        for r in range(count):                               # beams that nobody continues give their pages back first
            for seq in rows[r]:
                if seq is not None and id(seq) not in keeps:
                    cache.close(seq)
        for (_, _, r, k), child in zip(forks, cache.fork([(seq, name) for seq, name, _, _ in forks])):
            next_rows[r][k] = child
        rows, ended = next_rows, next_ended
    values = scores.tolist()
    for row in rows:
        for seq in row:
            if seq is not None:
                cache.close(seq)
    return [[(values[r][b], texts[r][b][1:]) for b in range(beams) if texts[r][b] is not None] for r in range(count)]
