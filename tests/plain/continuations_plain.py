"""Drafted trees and beams in 64 bits, element by element, from their definitions."""
import math

import torch


def chain(parents, i):
    found = []
    while i >= 0:
        found.append(i)
        i = parents[i]
    return found


def masks(trees, lengths, words):
    """(rows of words as signed 32-bit numbers, positions, places) of all nodes."""
    rows, positions, places = [], [], []
    for tree, length in zip(trees, lengths):
        for i in range(len(tree)):
            up = chain(tree, i)
            bits = [sum(1 << (j % 32) for j in up if j // 32 == w) for w in range(words)]
            rows.append([b - (1 << 32) if b >> 31 else b for b in bits])
            positions.append(length + len(up) - 1)
            places.append(length + i)
    return rows, positions, places


def seen_bits(row):
    """The node indices of a row of mask words."""
    return [w * 32 + b for w, word in enumerate(row) for b in range(32) if (word >> b) & 1]


def attention(q, pages, starts, lengths, positions, mask_rows, table, heads, kv_heads, dim, scale, window=None):
    """[T, heads, dim] float64; all arguments on the CPU, starts .. table as lists."""
    page = pages.shape[3]
    q, pages = q.double().view(-1, heads, dim), pages.double()
    out = torch.zeros(q.shape, dtype=torch.float64)
    for a, length in enumerate(lengths):
        for t in range(starts[a], starts[a + 1]):
            n = starts[a + 1] - starts[a]
            keys = [j for j in range(length) if not window or j > positions[t] - window]
            keys += [length + j for j in seen_bits(mask_rows[t]) if j < n and (not window or positions[starts[a] + j] > positions[t] - window)]
            if not keys:
                continue
            where = torch.tensor([table[a][j // page] for j in keys])
            inside = torch.tensor([j % page for j in keys])
            for h in range(heads):
                kvh = h // (heads // kv_heads)
                k, v = pages[where, 0, kvh, inside], pages[where, 1, kvh, inside]
                w = torch.softmax(k @ q[t, h] * scale, 0)
                out[t, h] = w @ v
    return out


def accept(tokens, parents, choices):
    """(path, the token behind it) of one tree."""
    if not tokens:
        return [], -1
    path = [0]
    while True:
        fits = [i for i in range(path[-1] + 1, len(tokens)) if parents[i] == path[-1] and tokens[i] == choices[path[-1]]]
        if not fits:
            return path, choices[path[-1]]
        path.append(fits[0])


def select(logits, scores, wanted, ended=None, end_token=-1):
    """(scores, parents, tokens) lists of one request: logits [beams, vocab], scores [beams]."""
    found = []
    for b in range(logits.shape[0]):
        score = float(scores[b])
        if score == -math.inf:
            continue
        if ended is not None and int(ended[b]):
            if math.isnan(score) or score == math.inf:
                return [math.nan] * wanted, [-1] * wanted, [-1] * wanted
            found.append((-score, b, end_token))
            continue
        row = logits[b].double()
        if math.isnan(score) or score == math.inf or bool((~(row < math.inf)).any()):
            return [math.nan] * wanted, [-1] * wanted, [-1] * wanted
        row = row - row.max().clamp(min=torch.finfo(torch.float32).min)      # first, so that a row of the type's lowest values keeps its normaliser
        row = row - row.exp().sum().log()
        found += [(-(score + x), b, t) for t, x in enumerate(row.tolist()) if x > -math.inf]
    found = sorted(found)[:wanted]
    found += [(math.inf, -1, -1)] * (wanted - len(found))
    return [-f[0] for f in found], [f[1] for f in found], [f[2] for f in found]
