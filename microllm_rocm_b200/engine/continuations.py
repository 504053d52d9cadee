"""Several continuations of a request over the paged cache: a step that brings a tree of drafted tokens, the branch of it that the
model's choices accept, and beam search.

A draft step (`draft_step`) runs the nodes of each entry's tree as one flat batch: node i's keys and values go behind the request's tokens in
the order of the nodes, its position is its depth in the tree, and it attends to the request's tokens and to the nodes above it.  The request's
length does not change: `accept_drafts` then walks each tree along the given choices, moves the accepted branch's keys and values into place in
every layer and commits its length, after which the cache is what decoding these tokens one by one would have left.

Beam search (`beam_search`) holds a request per beam.  The prompt is computed once and copied; after each selection every beam's cache becomes its
parent's, all layers in a launch.
"""
from __future__ import annotations

import itertools
from dataclasses import dataclass
from typing import Hashable, List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..kernels import beams, cache_moves, drafts, ops
from .step import Engine, OutOfPages, StepEntry, StepError


@dataclass
class DraftEntry:
    """A tree of tokens for one request: `parents[i]` is the index of the node that node i continues, an earlier one; node 0, whose parent is -1,
    is the token that the last step chose and every other node continues."""
    request: Hashable
    tokens: Sequence[int]
    parents: Sequence[int]


@dataclass
class DraftStep:
    """A draft step that ran: `logits` [nodes of all entries, vocab], in the order of the entries and their nodes."""
    entries: List[DraftEntry]
    logits: torch.Tensor
    ctx: object
    held: List[Tuple[object, int]]          # the requests' books, and which of their writing steps this one is


@dataclass
class Accepted:
    nodes: List[int]              # the accepted branch, node 0 first
    tokens: List[int]             # its tokens
    following: int                # the choice behind its last node: the next step's node 0


def check_tree(entry: DraftEntry) -> None:
    n = len(entry.tokens)
    if n != len(entry.parents):
        raise StepError(f"request {entry.request!r} brings {n} drafted tokens and {len(entry.parents)} parents")
    if n > drafts.MAX_NODES:
        raise StepError(f"request {entry.request!r} brings {n} drafted tokens (at most {drafts.MAX_NODES})")
    for i, p in enumerate(entry.parents):
        if (p != -1) if i == 0 else not 0 <= p < i:
            raise StepError(f"request {entry.request!r}: node {i} cannot continue node {p} (node 0 continues the request, every other an earlier node)")


def _check_model(engine: Engine) -> None:
    for block in engine.model.blocks:
        mixer = getattr(block, "mixer", None)
        if not getattr(mixer, "takes_drafts", False):
            raise StepError(f"{type(mixer).__name__} layers take no drafted trees: a step's tokens are one sequence to them")
    if engine.model.embedding_cache is not None:
        raise StepError("an embedding that looks at the token in front takes no drafted trees")


def draft_step(engine: Engine, entries: Sequence[DraftEntry]) -> DraftStep:
    """Run the trees; the logits of every node.  The requests keep their lengths until `accept_drafts`."""
    entries = list(entries)
    _check_model(engine)
    for e in entries:
        check_tree(e)
    plain = [StepEntry(e.request, e.tokens, range(len(e.tokens))) for e in entries]
    depths = []
    for e in entries:
        depth = np.zeros(len(e.tokens), dtype=np.int32)
        for i, p in enumerate(e.parents):
            depth[i] = 0 if p < 0 else depth[p] + 1
        depths.append(depth)
    ctx = engine.build_context(plain)                  # (its positions are the places: length + index)
    lengths = np.asarray(ctx.seq_pos0_host)
    most = max(len(e.tokens) for e in entries)
    # one upload: parents, then the positions that the rotation and the attention take
    flat = np.concatenate([np.concatenate([np.asarray(e.parents, dtype=np.int32) for e in entries])]
                          + [(d + n).astype(np.int32) for d, n in zip(depths, lengths)])
    both = ops.upload(flat, "int32", engine.device)
    T = ctx.num_tokens
    parents, positions = both[:T], both[T:]
    masks = torch.empty((T, -(-most // 32)), dtype=torch.int32, device=engine.device)
    drafts.draft_masks(parents, ctx.seq_starts, ctx.seq_pos0, masks, torch.empty_like(parents), None, engine.error_flag)
    ctx.places, ctx.positions = ctx.positions, positions
    ctx.tree = (masks, parents, most)
    logits = engine.model.forward(ctx, engine.cache_views(ctx))
    engine.steps_run += 1
    engine.tokens_run += T
    return DraftStep(entries, logits, ctx, [(book, book.writes) for book in (engine.cache.requests[e.request] for e in entries)])


def accept_drafts(engine: Engine, step: DraftStep, choices: torch.Tensor) -> List[Accepted]:
    """Walk each tree of `step` along `choices` ([nodes] int32 on the device: the model's own token behind every node), keep the branch in the
    cache and commit it.  Refused when one of the requests has taken another step since, a draft step too: its rows lie where this step's were."""
    ctx, cache = step.ctx, engine.cache
    for e, n, (book, writes) in zip(step.entries, ctx.seq_pos0_host, step.held):
        if cache.requests.get(e.request) is not book or book.length != n or book.writes != writes:
            raise StepError(f"request {e.request!r} went on since its draft step")
    A, most = ctx.num_seqs, ctx.tree[2]
    result = torch.empty(A * (most + 2), dtype=torch.int32, device=engine.device)
    path, counts, following = result[:A * most].view(A, most), result[A * most:A * most + A], result[A * most + A:]
    for group in cache.groups:
        drafts.accept_drafts(ctx.token_ids, ctx.tree[1], choices, ctx.seq_starts, ctx.seq_pos0, path, counts, following, cache.page_moves(group),
                             ctx.block_tables[group], engine.error_flag)
    host = result.tolist()
    engine.check_device_errors()
    out = []
    for a, (e, n) in enumerate(zip(step.entries, ctx.seq_pos0_host)):
        nodes = host[a * most:a * most + host[A * most + a]]
        cache.commit(e.request, n + len(nodes))
        out.append(Accepted(nodes, [int(e.tokens[i]) for i in nodes], host[A * most + A + a]))
    return out


_searches = itertools.count()


def beam_search(engine: Engine, prompt: Sequence[int], num_beams: int, max_new_tokens: int, end_token: Optional[int] = None) -> List[Tuple[List[int], float]]:
    """The `num_beams` best continuations of `prompt` by the sum of their tokens' log probabilities that a search with so many beams finds: (tokens, score),
    best first.  A beam that has chosen `end_token` goes no further and keeps its place by its score.  Continuations end after `max_new_tokens`.
    Needs a free state slot and pages for every beam; raises OutOfPages (and gives everything back) where they are missing."""
    cache, device = engine.cache, engine.device
    if not 0 < num_beams <= min(beams.MAX_BEAMS, beams.MAX_WANTED):
        raise ValueError(f"beam search takes 1 to {min(beams.MAX_BEAMS, beams.MAX_WANTED)} beams")
    if max_new_tokens < 0:
        raise ValueError("max_new_tokens must be non-negative")
    vocab = engine.model.spec.vocab_size
    if end_token is not None and not 0 <= end_token < vocab:
        raise ValueError("the end token is outside the vocabulary")
    prompt = [int(t) for t in prompt]
    if not prompt:
        raise ValueError("beam search wants a prompt of at least one token")
    if not all(0 <= t < vocab for t in prompt):
        raise ValueError("prompt token is outside the vocabulary")
    if len(prompt) + max_new_tokens > engine.model.spec.max_position:
        raise ValueError("prompt plus generated tokens exceeds model context")
    if max_new_tokens == 0:
        return [([], 0.0)]
    search, B = next(_searches), num_beams
    names = [("beam", search, b) for b in range(B)]
    made = []
    try:
        for name in names:
            if not cache.add(name):
                raise OutOfPages(f"no state slot is free for beam {len(made)} of {B}")
            made.append(name)
        return _search(engine, names, prompt, max_new_tokens, end_token, device, vocab)
    finally:
        for name in made:
            cache.release(name)


def _search(engine, names, prompt, max_new_tokens, end_token, device, vocab):
    cache, B = engine.cache, len(names)
    slots = ops.upload([[cache.slot(n) for n in names]], "int32", device)
    portion = engine.max_step_tokens or len(prompt)

    def follow(parents: torch.Tensor, first: int, last: int, lagging) -> None:
        """Beams take their parents' tokens [first, last) and state; `lagging`: the beams whose books do not say `last` yet."""
        for name in lagging:
            # (a portion at a time, as its parent's came: a window's pool holds no more)
            for at in range(cache.length(name), last, portion):
                to = min(at + portion, last)
                if not cache.reserve(name, to):
                    raise OutOfPages(f"no pages left for a beam to hold {to} tokens")
                cache.commit(name, to)
        if last > first:
            bounds = ops.upload([first, last], "int32", device)
            for group in cache.groups:
                table = ops.upload(cache.block_table(group, names), "int32", device)
                cache_moves.reorder_pages(cache.page_moves(group), table, parents, bounds[:1], bounds[1:], last - first, engine.error_flag)
        cache_moves.reorder_slots(cache.slot_moves(), slots, parents, engine.error_flag)

    for at in range(0, len(prompt), portion):
        some = prompt[at:at + portion]
        logits = engine.step([StepEntry(names[0], some, [len(some) - 1] if at + portion >= len(prompt) else [])])
    n = len(prompt)
    if B > 1:
        follow(ops.upload([[0] * B], "int32", device), 0, n, names[1:])
    scores = ops.upload([[0.0] + [-float("inf")] * (B - 1)], "float32", device)      # one beam so far
    rows = torch.zeros((B, vocab), dtype=torch.float32, device=device)
    rows[0] = logits[0]
    tokens: List[List[int]] = [[] for _ in range(B)]
    ended = [False] * B
    lengths = [n] * B                                  # of the beams' caches
    while True:
        out_scores = torch.empty((1, B), dtype=torch.float32, device=device)
        chosen = torch.empty((2, 1, B), dtype=torch.int32, device=device)
        flags = ops.upload([[int(x) for x in ended]], "int32", device) if end_token is not None else None
        beams.beam_select(rows, scores, out_scores, chosen[0], chosen[1], ended=flags, end_token=-1 if end_token is None else end_token)
        parents, picks = (x[0] for x in chosen.tolist())
        values = out_scores[0].tolist()
        engine.check_device_errors()
        if any(v != v for v in values):
            raise StepError("a beam's logits are not finite")
        tokens = [tokens[p] + ([] if ended[p] else [t]) if p >= 0 else None for p, t in zip(parents, picks)]
        ended = [p < 0 or (end_token is not None and t == end_token) for p, t in zip(parents, picks)]
        scores = out_scores
        if all(ended) or max(len(t) for t in tokens if t is not None) >= max_new_tokens:
            return [(t, v) for t, v in zip(tokens, values) if t is not None]
        # beams that go on take their parents' cache, which holds every token of theirs but the one just chosen
        now = max(lengths)
        keep = [p if not e and p != b else -1 for b, (p, e) in enumerate(zip(parents, ended))]
        if any(p >= 0 for p in keep):
            lagging = [names[b] for b, p in enumerate(keep) if p >= 0 and lengths[b] < now]
            follow(ops.upload([keep], "int32", device), n, now, lagging)
            lengths = [now if keep[b] >= 0 else lengths[b] for b in range(B)]
        live = [b for b in range(B) if not ended[b]]
        logits = engine.step([StepEntry(names[b], [picks[b]], [0]) for b in live])
        for b in live:
            lengths[b] += 1
        if len(live) == B:
            rows = logits
        else:
            rows.index_copy_(0, ops.upload(live, "int64", device), logits)
