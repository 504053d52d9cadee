"""Decoding several continuations of a request over the paged cache: drafted trees and beams, as their users call them.

Four operators, each a kind of case:

  drafts   one step's attention of trees of drafted tokens: masks and positions from the trees' parents once, then the
           attention of every layer over that layer's pages (`draft_masks`, `draft_attention`)
  accept   the branch that the model's own choices confirm, and its keys and values moved into place in every layer
           (`accept_drafts`)
  select   the best continuations of a request's beams over the vocabulary (`beam_select`)
  reorder  every beam continues from its parent's cache: tokens in pages, or slots of recurrent state (`reorder_pages`,
           `reorder_slots`)
"""
import math
import random
import zlib

import torch

own = False

BF16, FP32 = "bfloat16", "float32"
_TYPES = {BF16: torch.bfloat16, FP32: torch.float32}


# ------------------------------------------------------------------------------------------------------ the cases
def _drafts(dtype, heads, kv_heads, dim, seqs, low, high, nodes_low, nodes, layers=1, page=64, window=0):
    """Trees of nodes_low..nodes drafted tokens behind low..high cached ones."""
    return {"kind": "drafts", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "seqs": seqs, "low": low, "high": high,
            "nodes_low": nodes_low, "nodes": nodes, "layers": layers, "page": page, "window": window}


def _accept(dtype, kv_heads, dim, layers, seqs, low, high, nodes, page=64):
    return {"kind": "accept", "dtype": dtype, "kv_heads": kv_heads, "dim": dim, "layers": layers, "seqs": seqs, "low": low, "high": high,
            "nodes": nodes, "page": page}


def _select(requests, beams, vocab, wanted, dtype=FP32, ended=False):
    return {"kind": "select", "requests": requests, "beams": beams, "vocab": vocab, "wanted": wanted, "dtype": dtype, "ended": ended}


def _pages(dtype, kv_heads, dim, layers, requests, beams, prompt, low, high, page=64):
    """Beams that have made low..high tokens behind a prompt (which all beams of a request hold alike)."""
    return {"kind": "reorder", "what": "pages", "dtype": dtype, "kv_heads": kv_heads, "dim": dim, "layers": layers, "requests": requests,
            "beams": beams, "prompt": prompt, "low": low, "high": high, "page": page}


def _slots(layers, requests, beams, width):
    return {"kind": "reorder", "what": "slots", "layers": layers, "requests": requests, "beams": beams, "width": width}


def listed():
    named = {
        # the tiny windowed configuration: the shortest call there is, latency alone
        "drafts tiny float32": _drafts(FP32, 6, 2, 32, 1, 40, 40, 5, 5, layers=2, page=16, window=32),
        # one person at a chat, a tree of 26 nodes on the 1.5B shapes
        "drafts one 2048": _drafts(BF16, 12, 2, 128, 1, 2048, 2048, 26, 26, layers=4, page=16),
        # a server in the middle of its day: sequences of all lengths, trees of all sizes (7B shapes)
        "drafts 16 ragged": _drafts(BF16, 28, 4, 128, 16, 128, 2048, 1, 64, layers=2),
        # long conversations with large trees (14B shapes): the cache streams, the products count
        "drafts long": _drafts(BF16, 40, 8, 128, 4, 8192, 8192, 64, 64, layers=2),
        # the 32-bit path, with which people check a model
        "drafts float32": _drafts(FP32, 12, 2, 128, 3, 100, 700, 3, 13, layers=1, page=16),
        # one small tree accepted on the 1.5B shapes
        "accept one": _accept(BF16, 2, 128, 28, 1, 317, 317, 12, page=16),
        # large trees of a whole batch on the 7B shapes
        "accept 16": _accept(BF16, 4, 128, 28, 16, 128, 2048, 64),
        # the tiny vocabulary: latency alone
        "select tiny": _select(1, 4, 384, 8),
        # one request of eight beams over the benchmark model's vocabulary
        "select one": _select(1, 8, 151936, 16),
        # many requests, some of whose beams have ended
        "select 32 ended": _select(32, 5, 152064, 10, ended=True),
        # four beams' generated tokens in the pages of 28 layers (1.5B shapes)
        "reorder pages": _pages(BF16, 2, 128, 28, 1, 4, 317, 40, 100, page=16),
        # recurrent state of 16 heads of 128 x 128 in 12 layers, eight requests
        "reorder slots": _slots(12, 8, 4, 16 * 128 * 128),
    }
    return [dict(case, name=name) for name, case in named.items()]


def _spread(rng, low, high):
    """An integer of low..high, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng):
    kind = rng.choice(("drafts", "drafts", "drafts", "accept", "select", "select", "reorder"))
    if kind == "drafts":
        dtype, heads, kv_heads, dim = rng.choice(((BF16, 12, 2, 128), (BF16, 28, 4, 128), (BF16, 40, 8, 128), (BF16, 8, 8, 64), (BF16, 6, 2, 32),
                                                  (FP32, 6, 2, 32), (FP32, 12, 2, 128), (FP32, 4, 1, 16)))
        nodes, high = _spread(rng, 1, 64 if dtype == BF16 else 24), _spread(rng, 1, 16384 if dtype == BF16 and dim >= 64 else 2000)
        case = _drafts(dtype, heads, kv_heads, dim, _spread(rng, 1, 32), rng.choice((high, max(1, high // 7))), high, rng.choice((1, nodes)), nodes,
                       rng.choice((1, 2)), rng.choice((16, 64)), rng.choice((0, 0, _spread(rng, 8, 4096))))
        most = 4 * 64 * 40 * 128 * 8256 * 4 * 2 // (1 if dtype == BF16 and dim >= 64 else 64)
        while case["seqs"] > 1 and 4 * nodes * heads * dim * (high + nodes) * case["seqs"] * case["layers"] > most:
            case["seqs"] = max(1, case["seqs"] // 2)
        return case
    if kind == "accept":
        dtype, kv_heads, dim, layers = rng.choice(((BF16, 2, 128, 28), (BF16, 4, 128, 28), (FP32, 2, 32, 3), (BF16, 8, 64, 12)))
        high = _spread(rng, 1, 2048)
        return _accept(dtype, kv_heads, dim, layers, _spread(rng, 1, 16), max(1, high // 3), high, _spread(rng, 1, 64), rng.choice((16, 64)))
    if kind == "select":
        beams, requests, vocab = rng.randint(1, 12), _spread(rng, 1, 32), _spread(rng, 300, 152064)
        while requests > 1 and requests * beams * vocab > 160 * 152064:
            requests //= 2
        return _select(requests, beams, vocab, rng.randint(1, 2 * beams), rng.choice((FP32, FP32, BF16)), rng.random() < 0.5)
    if rng.random() < 0.5:
        dtype, kv_heads, dim, layers = rng.choice(((BF16, 2, 128, 28), (BF16, 4, 128, 28), (FP32, 2, 32, 3)))
        high = _spread(rng, 1, 300)
        return _pages(dtype, kv_heads, dim, layers, rng.randint(1, 4), rng.randint(2, 8), rng.randint(1, 400), max(1, high // 2), high, rng.choice((16, 64)))
    return _slots(rng.randint(1, 12), rng.randint(1, 6), rng.randint(2, 6), 4 * _spread(rng, 16, 65536))


# ------------------------------------------------------------------------------------------------------ inputs
def _sizes(case, what, low, high, count):
    """`count` sizes of low..high; the first is the largest.  They belong to the case: only the values come from the seed."""
    r = random.Random(zlib.crc32(repr((what, sorted((k, v) for k, v in case.items() if k != "name"))).encode()))
    return [high] + [r.randint(low, high) for _ in range(count - 1)]


def _ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _tables(r, blocks, spare, device):
    """Block tables [rows, widest] of rows that hold blocks[row] pages each, drawn without repetition; -1 behind."""
    order = list(range(sum(blocks)))
    r.shuffle(order)
    rows, at = [], 0
    for n in blocks:
        rows.append(order[at:at + n] + [-1] * (max(blocks) + spare - n))
        at += n
    return _ints(rows, device), at


def _parents(r, n):
    """A tree as drafts make it: the last accepted token, a few likely tokens behind it, and so on, breadth first."""
    return [-1] + [r.randint(max(0, (i - 1) // 4), min(i - 1, (i + 1) // 2)) for i in range(1, n)]


def _trees(r, case, device):
    A = case["seqs"]
    lengths = _sizes(case, "lengths", case["low"], case["high"], A)
    counts = _sizes(case, "nodes", case.get("nodes_low", 1), case["nodes"], A)
    trees = [_parents(r, n) for n in counts]
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    page = case["page"]
    table, pages = _tables(r, [-(-(n + k) // page) for n, k in zip(lengths, counts)], 0, device)
    return {"trees": trees, "counts": counts, "lengths_host": lengths, "pages": pages, "table": table, "T": starts[-1], "most": max(counts),
            "longest": max(n + k for n, k in zip(lengths, counts)), "starts": _ints(starts, device), "lengths": _ints(lengths, device),
            "parents": _ints([p for t in trees for p in t], device), "seq": _ints([a for a, t in enumerate(trees) for _ in t], device),
            "node": _ints([i for t in trees for i in range(len(t))], device)}


def prepare(case, seed):
    device = torch.device("cuda")
    r = random.Random(seed * 7919 + 17)
    g = torch.Generator(device=device)
    g.manual_seed(seed * 104729 + 5)

    def normal(shape, dtype=torch.float32, scale=1.0):
        out = torch.empty(shape, dtype=dtype, device=device)
        out.normal_(generator=g)
        return out.mul_(scale) if scale != 1.0 else out

    s = {"case": case}
    if case["kind"] == "drafts":
        s.update(_trees(r, case, device))
        dtype, NKV, D, L = _TYPES[case["dtype"]], case["kv_heads"], case["dim"], case["layers"]
        s["kv"] = normal((L, s["pages"], 2, NKV, case["page"], D), dtype)
        s["q"] = normal((L, s["T"], case["heads"] * D), dtype, 1.5)
        s["error"] = torch.zeros(1, dtype=torch.int32, device=device)
    elif case["kind"] == "accept":
        s.update(_trees(r, case, device))
        s["kv"] = normal((case["layers"], s["pages"], 2, case["kv_heads"], case["page"], case["dim"]), _TYPES[case["dtype"]])
        tokens, choices = [], []
        for tree in s["trees"]:
            mine = [r.randrange(50) for _ in tree]
            picks = [r.randrange(50) for _ in tree]
            at = 0                                  # a branch that the model confirms, as deep as a draft's usually is
            while True:
                children = [i for i, p in enumerate(tree) if p == at]
                if not children or r.random() < 0.2:
                    break
                child = r.choice(children)
                picks[at] = mine[child]
                at = child
            tokens += mine
            choices += picks
        s["tokens"], s["choices"] = _ints(tokens, device), _ints(choices, device)
        s["error"] = torch.zeros(1, dtype=torch.int32, device=device)
    elif case["kind"] == "select":
        R, B, V = case["requests"], case["beams"], case["vocab"]
        s["logits"] = normal((R * B, V), _TYPES[case["dtype"]], 2.5)
        s["scores"] = -torch.rand((R, B), generator=g, device=device) * 4.0
        s["ended"] = (torch.rand((R, B), generator=g, device=device) < 0.2).to(torch.int32) if case["ended"] else None
        s["end_token"] = V - 1
    else:
        R, B, L = case["requests"], case["beams"], case["layers"]
        # about what a selection gives: good beams have several children, poor ones none
        s["parents"] = _ints([sorted(min(r.randrange(B), r.randrange(B)) for _ in range(B)) for _ in range(R)], device)
        if case["what"] == "pages":
            page = case["page"]
            made = _sizes(case, "made", case["low"], case["high"], R)
            last = [case["prompt"] + n for n in made]
            s["table"], s["pages"] = _tables(r, [-(-last[i] // page) for i in range(R) for _ in range(B)], 0, device)
            s["first"], s["last"], s["most"] = _ints([case["prompt"]] * R, device), _ints(last, device), max(made)
            s["kv"] = normal((L, s["pages"] + 1, 2, case["kv_heads"], page, case["dim"]), _TYPES[case["dtype"]])
            s["error"] = torch.zeros(1, dtype=torch.int32, device=device)
        else:
            order = list(range(R * B))
            r.shuffle(order)
            s["slots"] = _ints([order[i * B:(i + 1) * B] for i in range(R)], device)
            s["state"] = normal((L, R * B + 1, case["width"]))
    return s


# ------------------------------------------------------------------------------------------------------ one pass
def run(s):
    return {"drafts": _run_drafts, "accept": _run_accept, "select": _run_select, "reorder": _run_reorder}[s["case"]["kind"]](s)


def _ancestors(s):
    """[A, N, N] truth values: node j is node i or one of those above it; and the depths [A, N]."""
    A, N, dev = s["lengths"].shape[0], s["most"], s["parents"].device
    seq, node, parent = s["seq"].long(), s["node"].long(), s["parents"].long()
    up = torch.zeros((A, N, N), dtype=torch.float32, device=dev)
    up[seq, node, parent.clamp(min=0)] = (parent >= 0).float()
    reach = up + torch.eye(N, device=dev)
    twice = lambda m: ((m @ m) > 0).float()                                             # 2, 4, 8 .. 256 steps up
    reach = twice(twice(twice(twice(twice(twice(twice(twice(reach))))))))
    return reach > 0, reach.sum(-1).long() - 1


def _plain_masks(reach, depth, s):
    seq, node, words = s["seq"].long(), s["node"].long(), -(-s["most"] // 32)
    bits = torch.zeros((s["T"], words * 32), dtype=torch.int64, device=reach.device)
    bits[:, :s["most"]] = reach[seq, node].long()
    bits = (bits.view(-1, words, 32) << torch.arange(32, device=bits.device)).sum(-1)
    return torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32), (s["lengths"][seq] + depth[seq, node]).to(torch.int32)


def _run_drafts(s):
    case = s["case"]
    NH, NKV, D, window = case["heads"], case["kv_heads"], case["dim"], case["window"]
    if own:
        from microllm_rocm_b200.kernels import drafts
        masks = torch.empty((s["T"], -(-s["most"] // 32)), dtype=torch.int32, device=s["q"].device)
        positions, places = torch.empty_like(s["parents"]), torch.empty_like(s["parents"])
        out = torch.empty_like(s["q"])
        drafts.draft_masks(s["parents"], s["starts"], s["lengths"], masks, positions, places, s["error"])
        for layer in range(case["layers"]):
            drafts.draft_attention(s["q"][layer], s["kv"][layer], out[layer], s["starts"], s["lengths"], positions, masks, s["table"], NH, NKV, D,
                                   D ** -0.5, window or None, max_nodes=s["most"], max_length=s["longest"], error_flag=s["error"])
        return {"out": out, "masks": masks, "positions": positions}
    reach, depth = _ancestors(s)
    masks, positions = _plain_masks(reach, depth, s)
    A, N, L, page, dev = s["lengths"].shape[0], s["most"], case["layers"], case["page"], s["q"].device
    rows = (s["starts"][:-1, None].long() + torch.arange(N, device=dev)).clamp(max=s["T"] - 1)
    q = s["q"][:, rows].float().view(L, A, N, NKV, NH // NKV, D).permute(0, 1, 3, 4, 2, 5)
    blocks = s["kv"][:, s["table"].clamp(min=0).long()].float()                          # [L, A, blocks, 2, NKV, page, D]
    keys, values = (blocks[:, :, :, i].transpose(2, 3).reshape(L, A, NKV, 1, -1, D) for i in (0, 1))
    del blocks
    place = torch.arange(keys.shape[-2], device=dev)
    length, n = s["lengths"].long()[:, None, None], (s["starts"][1:] - s["starts"][:-1]).long()[:, None, None]
    inner = (place - length).clamp(min=0, max=N - 1)                                     # the node at a place behind the cached tokens
    at = torch.where(place < length, place, length + depth.gather(1, inner[:, 0]).unsqueeze(1))
    seen = torch.where(place < length, True, reach.gather(2, inner.expand(-1, N, -1)) & (place - length < n))
    if window:
        seen = seen & (at > length + depth[:, :, None] - window)
    scores = (q @ keys.transpose(-1, -2)) * D ** -0.5
    scores.masked_fill_(~seen[None, :, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = scores.sum(-1, keepdim=True)
    out = (scores @ values) / torch.where(total == 0, 1.0, total)
    out = out.permute(0, 1, 4, 2, 3, 5).reshape(L, A, N, NH * D)[:, s["seq"].long(), s["node"].long()]
    return {"out": out.to(s["q"].dtype), "masks": masks, "positions": positions}


def _run_accept(s):
    A, N, kv, page = s["lengths"].shape[0], s["most"], s["kv"], s["case"]["page"]
    path, counts, following = (torch.empty(shape, dtype=torch.int32, device=kv.device) for shape in ((A, N), (A,), (A,)))
    if own:
        from microllm_rocm_b200.kernels import cache_moves, drafts
        if "moves" not in s:                          # made once, when a program makes its cache
            s["moves"] = cache_moves.PageMoves([kv[layer] for layer in range(kv.shape[0])], page)
        drafts.accept_drafts(s["tokens"], s["parents"], s["choices"], s["starts"], s["lengths"], path, counts, following, s["moves"], s["table"],
                             error_flag=s["error"])
        return {"path": path, "counts": counts, "following": following, "pages": kv}
    reach, depth = _ancestors(s)
    seq, node, parent = s["seq"].long(), s["node"].long(), s["parents"].long()
    token = torch.full((A, N), -1, dtype=torch.long, device=kv.device)
    above = torch.full((A, N), -2, dtype=torch.long, device=kv.device)
    choice = torch.full((A, N), -3, dtype=torch.long, device=kv.device)
    token[seq, node], above[seq, node], choice[seq, node] = s["tokens"].long(), parent, s["choices"].long()
    earlier = torch.ones((N, N), dtype=torch.bool, device=kv.device).tril(-1)
    again = ((token[:, :, None] == token[:, None]) & (above[:, :, None] == above[:, None]) & earlier).any(-1)     # an earlier sibling's token
    fits = (above >= 0) & (token == choice.gather(1, above.clamp(min=0))) & ~again
    fits[:, 0] = True
    taken = ((~fits)[:, None, :] & reach).sum(-1) == 0                                   # the node and all above it fit
    taken &= above > -2
    counts = taken.sum(-1)
    order = torch.where(taken, torch.arange(N, device=kv.device), N).sort(-1).values
    path = torch.where(order < N, order, -1)
    following = choice.gather(1, path.gather(1, (counts - 1)[:, None]).clamp(min=0))[:, 0]
    source = s["lengths"].long()[:, None] + path.clamp(min=0)
    target = torch.where(path >= 0, s["lengths"].long()[:, None] + torch.arange(N, device=kv.device), source[:, :1])
    rows = torch.arange(A, device=kv.device)[:, None]
    table = s["table"].long()
    new = kv[:, table[rows, source // page], :, :, source % page]
    kv[:, table[rows, target // page], :, :, target % page] = new
    return {"path": path.to(torch.int32), "counts": counts.to(torch.int32), "following": following.to(torch.int32), "pages": kv}


def _run_select(s):
    case = s["case"]
    R, B, V, n = case["requests"], case["beams"], case["vocab"], case["wanted"]
    if own:
        from microllm_rocm_b200.kernels import beams
        scores = torch.empty((R, n), dtype=torch.float32, device=s["logits"].device)
        parents, tokens = (torch.empty((R, n), dtype=torch.int32, device=s["logits"].device) for _ in range(2))
        beams.beam_select(s["logits"], s["scores"], scores, parents, tokens, ended=s["ended"], end_token=s["end_token"])
        return {"scores": scores, "parents": parents, "tokens": tokens}
    x = s["logits"].view(R, B, V).double()                                               # 64 bits: candidates of different beams are compared
    x = x - x.amax(-1, keepdim=True)
    x = x - x.exp().sum(-1, keepdim=True).log() + s["scores"].double()[:, :, None]
    if s["ended"] is not None:
        held = torch.full((V,), -math.inf, dtype=torch.float64, device=x.device)
        held[s["end_token"]] = 0.0
        x = torch.where((s["ended"] != 0)[:, :, None], held + s["scores"].double()[:, :, None], x)
    best, at = (v[:, :n] for v in x.view(R, B * V).sort(dim=-1, descending=True, stable=True))
    none = best == -math.inf
    return {"scores": best.float(), "parents": torch.where(none, -1, at // V).to(torch.int32), "tokens": torch.where(none, -1, at % V).to(torch.int32)}


def _run_reorder(s):
    case = s["case"]
    if case["what"] == "slots":
        state = s["state"]
        if own:
            from microllm_rocm_b200.kernels import cache_moves
            if "moves" not in s:
                s["moves"] = cache_moves.SlotMoves([state[layer] for layer in range(state.shape[0])])
            cache_moves.reorder_slots(s["moves"], s["slots"], s["parents"])
            return state
        slots = s["slots"].long()
        state[:, slots.view(-1)] = state[:, slots.gather(1, s["parents"].long()).view(-1)]
        return state
    kv, page, B = s["kv"], case["page"], case["beams"]
    if own:
        from microllm_rocm_b200.kernels import cache_moves
        if "moves" not in s:
            s["moves"] = cache_moves.PageMoves([kv[layer] for layer in range(kv.shape[0])], page)
        cache_moves.reorder_pages(s["moves"], s["table"], s["parents"], s["first"], s["last"], max_tokens=s["most"], error_flag=s["error"])
        return kv
    R = case["requests"]
    place = s["first"].long()[:, None] + torch.arange(s["most"], device=kv.device)       # [R, most]
    live = place < s["last"].long()[:, None]
    block = torch.where(live, place // page, 0)[:, None].expand(-1, B, -1)
    table = s["table"].long().view(R, B, -1)
    mine = table.gather(2, block)
    theirs = table.gather(1, s["parents"].long()[:, :, None].expand(-1, -1, table.shape[2])).gather(2, block)
    pad = kv.shape[1] - 1                                                                # the page behind the pool: nobody's
    live, offset = live[:, None].expand(-1, B, -1), (place % page)[:, None].expand(-1, B, -1)
    new = kv[:, torch.where(live, theirs, pad), :, :, torch.where(live, offset, 0)]
    kv[:, torch.where(live, mine, pad), :, :, torch.where(live, offset, 0)] = new
    return kv


# ------------------------------------------------------------------------------------------------------ what a pass needs
def _size(dtype):
    return 2 if dtype == BF16 else 4


def work(case):
    """Sizes as `prepare` draws them, averaged where they are drawn."""
    mean = lambda low, high, count: (high + (count - 1) * (low + high) / 2) / count
    if case["kind"] == "drafts":
        A, L, NH, NKV, D, es = case["seqs"], case["layers"], case["heads"], case["kv_heads"], case["dim"], _size(case["dtype"])
        n = mean(case["nodes_low"], case["nodes"], A)
        keys = mean(case["low"], case["high"], A)
        keys = (min(keys, case["window"]) if case["window"] else keys) + n
        return {"bytes": A * L * (2 * keys * NKV * D + 2 * n * NH * D) * es, "flops": 4 * A * L * n * keys * NH * D}
    if case["kind"] == "accept":
        # about half of an accepted branch stands out of place; branches are a few nodes deep
        moved = min(2.0, case["nodes"] / 4)
        n = mean(1, case["nodes"], case["seqs"])
        return {"bytes": case["seqs"] * (12 * n + 4 * case["nodes"] + 2 * moved * 2 * case["layers"] * case["kv_heads"] * case["dim"] * _size(case["dtype"])), "flops": 0}
    if case["kind"] == "select":
        n = case["requests"] * case["beams"] * case["vocab"]
        return {"bytes": n * _size(case["dtype"]) * (0.8 if case["ended"] else 1.0) + 12 * case["requests"] * case["wanted"], "flops": 4 * n}
    B = case["beams"]
    # the share of beams whose parent is another one, and of beams that are another one's parent
    r = random.Random(1)
    trials = [sorted(min(r.randrange(B), r.randrange(B)) for _ in range(B)) for _ in range(400)]
    moved = sum(sum(p != b for b, p in enumerate(t)) for t in trials) / 400
    read = sum(len({p for b, p in enumerate(t) if p != b}) for t in trials) / 400
    if case["what"] == "slots":
        return {"bytes": max(16.0, (moved + read) * case["requests"] * case["layers"] * case["width"] * 4), "flops": 0}
    tokens = mean(case["low"], case["high"], case["requests"])
    return {"bytes": max(16.0, (moved + read) * case["requests"] * case["layers"] * tokens * 2 * case["kv_heads"] * case["dim"] * _size(case["dtype"])), "flops": 0}


# ------------------------------------------------------------------------------------------------------ the definition in 64 bits
def _chain(tree, i):
    """Node i and those above it, from the bottom up."""
    found = []
    while i >= 0:
        found.append(i)
        i = tree[i]
    return found


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "drafts":
        L, NH, NKV, D, page, window = case["layers"], case["heads"], case["kv_heads"], case["dim"], case["page"], case["window"]
        out = torch.zeros((L, s["T"], NH, D), dtype=torch.float64, device="cuda")
        masks, positions, row = [], [], 0
        for a, tree in enumerate(s["trees"]):
            n, length = len(tree), s["lengths_host"][a]
            chains = [_chain(tree, i) for i in range(n)]
            depth = [len(c) - 1 for c in chains]
            for c in chains:
                words = [sum(1 << (j % 32) for j in c if j // 32 == w) for w in range(-(-s["most"] // 32))]
                masks.append([w - (1 << 32) if w >> 31 else w for w in words])
                positions.append(length + len(c) - 1)
            hidden = torch.ones((n, length + n), dtype=torch.bool)
            for i, c in enumerate(chains):
                first = max(0, length + depth[i] - window + 1) if window else 0
                hidden[i, first:length] = False
                for j in c:
                    hidden[i, length + j] = bool(window) and depth[i] - depth[j] >= window
            hidden = hidden.to("cuda")
            index = torch.arange(length + n, device="cuda")
            where = s["table"][a].long()[index // page]
            for layer in range(L):
                kv = s["kv"][layer].permute(0, 3, 1, 2, 4)[where, index % page].double()  # [keys, 2, NKV, D]
                for h in range(NH):
                    w = torch.einsum("nd,kd->nk", s["q"][layer, row:row + n, h * D:(h + 1) * D].double(), kv[:, 0, h * NKV // NH]) / math.sqrt(D)
                    w = w.masked_fill(hidden, -math.inf)
                    out[layer, row:row + n, h] = torch.nan_to_num(torch.softmax(w, -1)) @ kv[:, 1, h * NKV // NH]
            row += n
        return {"out": out.view(L, s["T"], NH * D), "masks": _ints(masks, "cuda"), "positions": _ints(positions, "cuda")}
    if case["kind"] == "accept":
        paths, counts, following, row = [], [], [], 0
        kv, page, table = s["kv"], case["page"], s["table"].tolist()
        tokens, choices = s["tokens"].tolist(), s["choices"].tolist()
        before = kv.clone()
        for a, tree in enumerate(s["trees"]):
            path = [0]
            while True:
                found = [i for i, p in enumerate(tree) if p == path[-1] and tokens[row + i] == choices[row + path[-1]]]
                if not found:
                    break
                path.append(found[0])
            for i, j in enumerate(path):
                to, of = s["lengths_host"][a] + i, s["lengths_host"][a] + j
                kv[:, table[a][to // page], :, :, to % page] = before[:, table[a][of // page], :, :, of % page]
            paths.append(path + [-1] * (s["most"] - len(path)))
            counts.append(len(path))
            following.append(choices[row + path[-1]])
            row += len(tree)
        return {"path": _ints(paths, "cuda"), "counts": _ints(counts, "cuda"), "following": _ints(following, "cuda"), "pages": kv}
    if case["kind"] == "select":
        B, V, n = case["beams"], case["vocab"], case["wanted"]
        all_scores, all_parents, all_tokens = [], [], []
        for q in range(case["requests"]):
            found = []
            for b in range(B):
                score = float(s["scores"][q, b])
                if s["ended"] is not None and int(s["ended"][q, b]):
                    found.append((-score, b, s["end_token"]))
                    continue
                row = s["logits"][q * B + b].double()
                row = (row - torch.logsumexp(row, 0)).cpu()
                border = float(torch.topk(row, min(n, V)).values[-1])
                found += [(-(score + float(row[t])), b, t) for t in torch.nonzero(row >= border)[:, 0].tolist()]
            found = sorted(found)[:n] + [(math.inf, -1, -1)] * max(0, n - len(found))
            all_scores.append([-f[0] for f in found])
            all_parents.append([f[1] for f in found])
            all_tokens.append([f[2] for f in found])
        return {"scores": torch.tensor(all_scores, dtype=torch.float64), "parents": _ints(all_parents, "cpu"), "tokens": _ints(all_tokens, "cpu")}
    parents = s["parents"].tolist()
    if case["what"] == "slots":
        before, slots = s["state"].clone(), s["slots"].tolist()
        for mine, of in zip(slots, parents):
            for b, p in enumerate(of):
                s["state"][:, mine[b]] = before[:, mine[p]]
        return s["state"]
    before, page, B, table = s["kv"].clone(), case["page"], case["beams"], s["table"].tolist()
    for q, of in enumerate(parents):
        for b, p in enumerate(of):
            for t in range(int(s["first"][q]), int(s["last"][q])):
                s["kv"][:, table[q * B + b][t // page], :, :, t % page] = before[:, table[q * B + p][t // page], :, :, t % page]
    return s["kv"]
