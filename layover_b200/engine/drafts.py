"""Greedy generation with drafted tokens: several guessed continuations of a request are checked in one step.

Every step feeds the request's newest token and, hanging under it, a tree of guesses (`StepEntry.parents`). The greedy
choice after each of them is made on the device; the walk from the newest token down the guesses that were chosen is
what the request would have generated token by token, so its result is that of plain greedy generation and only the
number of steps differs. The rows of the tokens walked through stay in the cache (`CacheManager.accept`), the others'
are given back. The reference decodes one token a request and step (layover/engine.py:176-189).

`LookupDrafts` guesses from the request's own tokens: what followed the latest earlier occurrences of its last ones.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import ops
from .batch import StepEntry


@dataclass(frozen=True)
class LookupDrafts:
    """Up to `width` continuations of up to `depth` tokens, each what followed an earlier occurrence (the latest first) of the last
    `context` tokens; common beginnings are one branch."""
    width: int = 2
    depth: int = 6
    context: int = 2

    def __call__(self, tokens: list[int], room: int) -> tuple[list[int], list[int]]:
        """(guesses, the place of each one's parent among them or -1), at most `room` of them on any branch."""
        depth, n = min(self.depth, room), self.context
        guesses, parents, children = [], [], {}
        if depth < 1 or self.width < 1 or len(tokens) <= n:
            return guesses, parents
        key, found = tokens[-n:], 0
        for at in range(len(tokens) - n - 1, -1, -1):
            if tokens[at:at + n] != key:
                continue
            node = -1
            for token in tokens[at + n: at + n + depth]:
                if (node, token) not in children:
                    children[node, token] = len(guesses)
                    guesses.append(token)
                    parents.append(node)
                node = children[node, token]
            found += 1
            if found == self.width:
                break
        return guesses, parents


def walk(tokens: list[int], parents: list[int], chosen: list[int]) -> list[int]:
    """The path from token 0 down the tree on which each token is the one chosen after its parent: places, 0 first."""
    path, children = [0], {}
    for place in range(len(tokens) - 1, 0, -1):          # the first of equal siblings
        children[parents[place], tokens[place]] = place
    while (path[-1], chosen[path[-1]]) in children:
        path.append(children[path[-1], chosen[path[-1]]])
    return path


def generate_with_drafts(model, prompts: list[list[int]], max_new_tokens: int = 16, drafts=LookupDrafts(), stop_tokens=frozenset(),
                         num_blocks: int | None = None, block_tokens: int = 16, prefill_chunk: int = 512) -> tuple[list[list[int]], dict]:
    """Greedy continuations of `prompts`, the tokens that `generate` gives at temperature 0 up to the roundings of the kernels that
    compute them, and the counts {"steps", "drafted", "accepted"}. `drafts(tokens, room)` guesses, see `LookupDrafts`; without `num_blocks`
    the pool has room for twice its `width` x `depth` guesses a request (of a callable without those 8 x 8), and of more the first are taken."""
    from .. import PagedKVCache
    from .step import StepFunction

    if any(not p for p in prompts) or max_new_tokens < 1:
        raise ValueError("a prompt needs tokens, and max_new_tokens is at least 1")
    if not model.takes_drafts:
        raise ValueError("this model's mixers have no form for a tree of drafts")
    spare = 2 * max(0, getattr(drafts, "width", 8)) * max(0, getattr(drafts, "depth", 8)) + 2
    most_guesses = spare if num_blocks is None else model.spec.max_position
    if num_blocks is None:
        num_blocks = sum(-(-(len(p) + max_new_tokens + spare) // block_tokens) for p in prompts)
    cache = PagedKVCache(model, max(1, num_blocks), block_tokens=block_tokens, max_requests=max(1, len(prompts)))
    step = StepFunction(model, cache)
    status, names = ops.status_words(model.device, model.kernel_libraries(model.dtype))
    counts = {"steps": 0, "drafted": 0, "accepted": 0}

    def choose(logits: torch.Tensor) -> list[int]:
        """The first index of the maximum of every row; raises if a kernel of this step gave up waiting."""
        rows, words = logits.shape[0], 0 if status is None else status.shape[0]
        tokens = torch.empty(rows + words, dtype=torch.int32, device=logits.device)
        values = ops.sample(logits, tokens, status=status).tolist()
        counts["steps"] += 1
        if any(values[rows:]):
            ops.reset_after_error(model.device)
            raise ops.KernelError("a kernel gave up waiting: " + ", ".join(f"{n}: code {c}" for n, c in zip(names, values[rows:]) if c))
        return values[:rows]

    texts = [list(p) for p in prompts]
    seqs = [cache.open(str(i)) for i in range(len(prompts))]
    for text, seq in zip(texts, seqs):                     # the prompts, portion by portion
        for at in range(0, len(text), prefill_chunk):
            part = text[at: at + prefill_chunk]
            last = at + len(part) == len(text)
            logits = step([StepEntry(seq, part, [len(part) - 1] if last else [])])
        text.append(choose(logits)[0])

    def open_ends(i: int) -> int:
        return 0 if texts[i][-1] in stop_tokens else len(prompts[i]) + max_new_tokens - len(texts[i])

    while True:
        active = [i for i in range(len(prompts)) if open_ends(i) > 0]
        if not active:
            break
        entries = []
        for i in active:
            room = min(open_ends(i) - 1, step.max_position - seqs[i].num_tokens - 1)
            guesses, parents = drafts(texts[i], room)
            most = max(0, min(most_guesses, step.max_position - seqs[i].num_tokens - 1))      # parents come first: the first guesses are a tree
            guesses, parents = guesses[:most], parents[:most]
            counts["drafted"] += len(guesses)
            tokens = [texts[i][-1], *guesses]
            entries.append(StepEntry(seqs[i], tokens, list(range(len(tokens))), [-1, *(p + 1 for p in parents)]))
        chosen = choose(step(entries))
        accepted, at = [], 0
        for i, entry in zip(active, entries):
            mine = chosen[at: at + len(entry.tokens)]
            at += len(entry.tokens)
            path = walk(entry.tokens, entry.parents, mine)[: open_ends(i)]
            for k, place in enumerate(path):
                texts[i].append(mine[place])
                if mine[place] in stop_tokens:
                    path = path[: k + 1]
                    break
            counts["accepted"] += len(path) - 1
            accepted.append((entry.seq, path))
        cache.accept(accepted)
    for seq in seqs:
        cache.close(seq)
    return [text[len(p):] for text, p in zip(texts, prompts)], counts
