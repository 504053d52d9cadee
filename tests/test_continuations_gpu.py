"""Drafted trees and beams on the GPU against plain implementations in 64 bits.

Tolerances, before any run.  u = 2^-24 is half a step of fp32.  A score is a sum of D products, off by at most (D + 2) u times the sum of their sizes
<= (D + 2) u |q| |k| scale = d; exponentials and the sums over S keys add (S + 16) u relative; the weights are then off by 2 d + (S + 16) u relative, and
an output, an average of values, by that times the largest value.  bf16: the output's rounding adds half a step, 2^-8 of its size, and a kernel that rounds the
weights for the tensor core another 2^-8 of the largest value.  A selected score is one fp32 rounding, and the normaliser's fp32 exponentials are off by 16 u
at most (argument and function), so 2 u of the score's size and 32 u."""
import math
import random

import pytest
import torch

from microllm_rocm_b200.kernels import beams, cache_moves, drafts, ops
from tests.plain import continuations_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def dev_ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def random_tree(rng, n):
    return [-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, n)]


class Step:
    """A cache with drafted nodes in it, and the plain answer."""

    def __init__(self, dtype, heads, kv_heads, dim, page, lengths, trees, seed=0, window=None, released=False, poison=False):
        rng = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.window, self.dtype = heads, kv_heads, dim, window, dtype
        self.lengths, self.trees = lengths, trees
        self.starts = [0]
        for t in trees:
            self.starts.append(self.starts[-1] + len(t))
        T = self.starts[-1]
        blocks = [-(-(n + len(t)) // page) for n, t in zip(lengths, trees)]
        pool = sum(blocks) + 3
        order = list(range(pool))
        rng.shuffle(order)
        self.pages = torch.randn((pool, 2, kv_heads, page, dim), generator=g).to(dtype)
        self.q = (torch.randn((T, heads * dim), generator=g) * 1.5).to(dtype)
        self.table, at = [], 0
        width = max(blocks + [1]) + 1
        for n in blocks:
            self.table.append(order[at:at + n] + [-1] * (width - n))
            at += n
        words = max(1, -(-max([len(t) for t in trees] + [1]) // 32))
        self.rows, self.positions, self.places = plain.masks(trees, lengths, words)
        self.max_nodes = max([len(t) for t in trees] + [1])
        self.max_length = max(max((n + len(t) for n, t in zip(lengths, trees)), default=1), self.max_nodes)
        self.poisoned = None
        if poison:                         # what no token of a sequence occupies: unused places and pages of nobody
            used = torch.zeros((pool, page), dtype=torch.bool)
            for a, n in enumerate(lengths):
                for j in range(n + len(trees[a])):
                    used[self.table[a][j // page], j % page] = True
            self.poisoned = self.pages.permute(0, 3, 1, 2, 4).clone()
            self.poisoned[~used] = float("nan")
            self.poisoned = self.poisoned.permute(0, 2, 3, 1, 4).contiguous()
        if released and window:            # blocks that no query can reach were given back
            for a, n in enumerate(lengths):
                for b in range(max(0, n - window + 1) // page):
                    self.table[a][b] = -1

    def want(self):
        return plain.attention(self.q, self.pages, self.starts, self.lengths, self.positions, self.rows, self.table, self.heads, self.kv_heads, self.dim,
                               self.dim ** -0.5, self.window)

    def run(self, out=None, max_length=None, max_nodes=None):
        self.error = torch.zeros(1, dtype=torch.int32, device=DEV)
        q = self.q.to(DEV)
        out = torch.full_like(q, 7.0) if out is None else out
        drafts.draft_attention(q, (self.pages if self.poisoned is None else self.poisoned).to(DEV), out, dev_ints(self.starts), dev_ints(self.lengths),
                               dev_ints(self.positions), dev_ints(self.rows).view(len(self.rows), -1), dev_ints(self.table), self.heads, self.kv_heads, self.dim,
                               self.dim ** -0.5, self.window, max_nodes=max_nodes or self.max_nodes, max_length=max_length or self.max_length, error_flag=self.error)
        return out

    def check(self, got, want=None, error=0):
        want = self.want() if want is None else want
        got = got.cpu().double().view(want.shape)
        q, k = self.q.double().view(-1, self.heads, self.dim), self.pages[:, 0].double()
        d = (self.dim + 2) * U * float(q.norm(dim=-1).max()) * float(k.norm(dim=-1).max()) * self.dim ** -0.5
        largest = float(self.pages[:, 1].double().abs().max())
        tolerance = (2 * d + (self.max_length + 16) * U) * largest
        bound = tolerance + want.abs() * 2 * U
        if self.dtype == torch.bfloat16:
            bound = tolerance + 2.0 ** -8 * want.abs() + 2.0 ** -8 * largest
        off = (got - want).abs()
        assert torch.isfinite(got).all()
        assert (off <= bound).all(), f"off by {float((off - bound).max())} more than {float(bound.max())}"
        if self.dtype == torch.bfloat16:           # and near as a whole: the roundings of many weights do not add up in one direction
            assert float((got - want).norm()) <= 2.0 ** -7 * float(want.norm()) + 1e-12
        assert int(self.error) == error


F32, BF16 = torch.float32, torch.bfloat16
SHAPES = [
    # dtype, heads, kv heads, dim, page, lengths, nodes, window
    (F32, 4, 1, 16, 16, [5], [1], None),
    (F32, 6, 2, 32, 16, [40], [5], 32),
    (F32, 6, 2, 32, 7, [0, 33, 64], [3, 1, 9], None),
    (F32, 4, 4, 6, 5, [11, 1], [4, 33], None),            # rows that are no pieces of four elements
    (F32, 12, 2, 128, 16, [100, 700, 31], [13, 3, 13], None),
    (F32, 2, 1, 200, 16, [90], [20], 17),
    (F32, 3, 1, 256, 64, [130], [40], None),
    (BF16, 4, 2, 32, 16, [50, 3], [7, 40], None),
    (BF16, 4, 1, 18, 3, [20], [6], 9),
    (BF16, 8, 8, 64, 16, [129, 0, 500], [1, 2, 65], None),
    (BF16, 8, 2, 64, 64, [700], [33], 100),
    (BF16, 12, 2, 128, 16, [2048], [26], None),
    (BF16, 28, 4, 128, 64, [128, 1000, 517], [64, 1, 17], None),
    (BF16, 28, 4, 128, 64, [640, 127], [40, 19], 300),
    (BF16, 5, 1, 128, 128, [383], [100], None),
    (BF16, 40, 8, 128, 8, [255, 256, 257], [5, 5, 5], None),
    (BF16, 6, 1, 128, 12, [77], [9], None),                # a page size that tiles of 128 keys are no multiple of
    (BF16, 3, 1, 256, 16, [200], [10], 64),
    (BF16, 32, 1, 128, 32, [300], [16], None),             # many heads of one kv head
    (BF16, 130, 1, 64, 16, [64], [3], None),               # more heads of one kv head than a tile has rows
]


@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_attention_against_64_bits(case):
    dtype, heads, kv_heads, dim, page, lengths, nodes, window = SHAPES[case]
    rng = random.Random(case)
    step = Step(dtype, heads, kv_heads, dim, page, lengths, [random_tree(rng, n) for n in nodes], case, window)
    step.check(step.run())


@pytest.mark.parametrize("dtype, dim, page", [(F32, 32, 16), (BF16, 128, 16), (BF16, 64, 64)])
def test_what_nobody_sees_reaches_no_output(dtype, dim, page):
    """Unused places of pages and pages of nobody hold NaN; blocks in front of the window were given back."""
    rng = random.Random(3)
    step = Step(dtype, 6, 2, dim, page, [300, 17, 140], [random_tree(rng, n) for n in (9, 20, 1)], 5, 50, released=True, poison=True)
    step.check(step.run())


@pytest.mark.parametrize("dtype, dim", [(F32, 32), (BF16, 128), (BF16, 64), (F32, 128)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_node_that_is_not_finite_reaches_only_those_below_it(dtype, dim, value):
    step = Step(dtype, 4, 2, dim, 16, [30, 200], [[-1, 0, 0, 1, 2, 2], [-1, 0, 1]], 1)
    want = step.want()
    place = 30 + 2
    step.pages[step.table[0][place // 16], :, :, place % 16] = value           # keys and values of node 2 of the first sequence
    got = step.run().cpu().double().view(want.shape)
    below = [2, 4, 5]
    assert not torch.isfinite(got[below]).any(-1).all(-1).any()
    rest = [t for t in range(9) if t not in below]
    largest = float(want.abs().max())
    assert (got[rest] - want[rest]).abs().max() <= (2.0 ** -6 if dtype == BF16 else 1e-4) * max(4.0, largest)


@pytest.mark.parametrize("dtype, dim", [(F32, 16), (BF16, 128)])
def test_masks_of_any_kind_and_rows_that_see_nothing(dtype, dim):
    rng = random.Random(2)
    step = Step(dtype, 4, 2, dim, 16, [0, 60], [random_tree(rng, 12), random_tree(rng, 40)], 3, None)
    for t in range(len(step.rows)):
        step.rows[t] = [rng.getrandbits(32) - (1 << 31) if rng.random() < 0.8 else 0 for _ in step.rows[t]]
    step.rows[0] = [0, 0]
    step.rows[5] = [0, 0]
    want = step.want()
    assert float(want[0].abs().max()) == 0.0
    got = step.run()
    step.check(got, want)
    assert float(got[0].abs().max()) == 0.0 and float(got[5].abs().max()) == 0.0


@pytest.mark.parametrize("dtype, dim", [(F32, 32), (BF16, 128)])
def test_rows_of_nobody_stay_and_hints_only_cut_the_work(dtype, dim):
    rng = random.Random(4)
    step = Step(dtype, 6, 2, dim, 16, [900, 40, 0], [random_tree(rng, 5), [], random_tree(rng, 2)], 6)
    want = step.want()
    for hint in (step.max_nodes, 64, step.max_length, 5000):
        step.check(step.run(max_length=max(hint, step.max_nodes)), want)
    rows = torch.full((9, 6 * dim), 7.0, dtype=dtype, device=DEV)
    q = torch.cat([step.q, torch.ones(2, 6 * dim, dtype=dtype)])
    step.q = q
    step.rows += [[1], [1]]
    step.positions += [3, 3]
    step.run(out=rows)
    assert (rows[7:] == 7.0).all()                # behind the last sequence
    step.q = q[:7]
    step.check(rows[:7], want)


@pytest.mark.parametrize("dtype, dim", [(F32, 32), (BF16, 128)])
def test_bad_pages_and_too_many_nodes_raise_the_flag(dtype, dim):
    rng = random.Random(4)
    trees = [random_tree(rng, 5), random_tree(rng, 9)]
    for wrong in (-1, 1 << 20):
        step = Step(dtype, 6, 2, dim, 16, [90, 40], trees, 6)
        step.table[0][2] = wrong
        step.run()
        assert int(step.error) == 2
    step = Step(dtype, 6, 2, dim, 16, [90, 40], trees, 6)
    step.run(max_nodes=5)
    assert int(step.error) == 3


@pytest.mark.parametrize("dtype, heads, kv_heads, dim, length", [(F32, 12, 2, 128, 500), (BF16, 12, 2, 128, 3000), (BF16, 28, 4, 128, 400)])
def test_attention_repeats_its_bits_and_captures(dtype, heads, kv_heads, dim, length):
    rng = random.Random(1)
    step = Step(dtype, heads, kv_heads, dim, 16, [length, length // 3], [random_tree(rng, 20), random_tree(rng, 31)], 2)
    first = step.run()
    assert all(torch.equal(first, step.run()) for _ in range(3))
    error = torch.zeros(1, dtype=torch.int32, device=DEV)
    pages, starts, lengths = step.pages.to(DEV), dev_ints(step.starts), dev_ints(step.lengths)
    parents = dev_ints([p for t in step.trees for p in t])
    T = step.starts[-1]
    q, table = step.q.to(DEV), dev_ints(step.table)
    out, masks, positions, places = torch.zeros_like(q), dev_ints([[0]] * T), dev_ints([0] * T), dev_ints([0] * T)

    def both():
        drafts.draft_masks(parents, starts, lengths, masks, positions, places, error)
        drafts.draft_attention(q, pages, out, starts, lengths, positions, masks, table, heads, kv_heads, dim, dim ** -0.5, max_nodes=31, max_length=step.max_length,
                               error_flag=error)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                  # another stream than the tensors'
        both()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    out.zero_()
    graph.replay()
    assert torch.equal(out, first) and int(error) == 0
    # the graph reads the lengths and trees as they are when it is replayed
    shorter = Step(dtype, heads, kv_heads, dim, 16, [length - 50, 11], step.trees, 2)
    shorter.pages, shorter.q, shorter.table = step.pages, step.q, step.table
    lengths.copy_(dev_ints(shorter.lengths))
    graph.replay()
    shorter.error = error
    shorter.check(out)


@pytest.mark.parametrize("sizes, words", [([1], 1), ([5, 0, 32], 1), ([33, 7], 2), ([256], 8), ([64, 1, 100, 3], 8)])
def test_masks(sizes, words):
    rng = random.Random(len(sizes))
    trees = [random_tree(rng, n) if n else [] for n in sizes]
    if sizes == [256]:
        trees = [list(range(-1, 255))]             # a chain
    lengths = [rng.randrange(5000) for _ in sizes]
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    T = starts[-1]
    masks, positions, places, error = dev_ints([[9] * words] * T), dev_ints([9] * T), dev_ints([9] * T), dev_ints([0])
    drafts.draft_masks(dev_ints([p for t in trees for p in t]), dev_ints(starts), dev_ints(lengths), masks, positions, places, error)
    rows, at, where = plain.masks(trees, lengths, words)
    assert masks.tolist() == rows and positions.tolist() == at and places.tolist() == where and int(error) == 0


def test_masks_of_what_is_no_tree_raise_the_flag():
    for parents in ([0, 0], [-1, 1], [-1, 5], [-2, 0]):
        masks, positions, error = dev_ints([[0], [0]]), dev_ints([0, 0]), dev_ints([0])
        drafts.draft_masks(dev_ints(parents), dev_ints([0, 2]), dev_ints([4]), masks, positions, None, error)
        assert int(error) == 3
    error = dev_ints([0])
    masks = dev_ints([[5]] * 40)
    drafts.draft_masks(dev_ints([-1] * 40), dev_ints([0, 40]), dev_ints([4]), masks, dev_ints([0] * 40), None, error)
    assert int(error) == 3 and (masks == 5).all()


# ------------------------------------------------------------------------------ the accepted branch
LAYOUTS = {
    "heads bf16": lambda pool, page: [torch.randn(pool, 2, 3, page, 8, device=DEV).to(BF16) for _ in range(3)],
    "heads fp32": lambda pool, page: [torch.randn(pool, 2, 2, page, 128, device=DEV) for _ in range(5)],
    "rows": lambda pool, page: [torch.randn(pool, page, 9, device=DEV) for _ in range(2)],
    "odd bf16 rows": lambda pool, page: [torch.randn(pool, page, 9, device=DEV).to(BF16)],
    "two widths": lambda pool, page: [(torch.randn(pool, 2 * page * 7, device=DEV), (2, 3, 4)) for _ in range(2)],
    "many layers and kinds": lambda pool, page: [torch.randn(pool, 2, 1, page, 4, device=DEV) for _ in range(130)] + [torch.randn(pool, page, 2, device=DEV)],
}


def token_view(storage, page):
    """[pages, page, elements of a token] of a pool."""
    t, widths = storage if isinstance(storage, tuple) else (storage, None)
    if widths:
        heads, dk, dv = widths
        k = t[:, :heads * page * dk].view(-1, heads, page, dk).transpose(1, 2).flatten(2)
        v = t[:, heads * page * dk:].view(-1, heads, page, dv).transpose(1, 2).flatten(2)
        return torch.cat([k, v], 2)
    return t.permute(0, 3, 1, 2, 4).flatten(2) if t.dim() == 5 else t


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("page, seed", [(5, 0), (16, 1), (64, 2)])
def test_accepted_branches_move_into_place(layout, page, seed):
    rng = random.Random(seed)
    sizes = [12, 1, 0, 64, 7]
    lengths = [rng.randrange(0, 3 * page) for _ in sizes]
    trees = [random_tree(rng, n) if n else [] for n in sizes]
    trees[4] = [-1, 0, 0, 1, 2, 4, 5]                      # 0 2 4 5 6: every node of it moves
    tokens = [[rng.randrange(4) for _ in t] for t in trees]
    choices = [[rng.randrange(4) for _ in t] for t in trees]
    tokens[4], choices[4] = [9, 1, 2, 3, 4, 5, 6], [2, 0, 4, 0, 5, 6, 8]
    wanted = [plain.accept(*x) for x in zip(tokens, trees, choices)]
    assert wanted[4] == ([0, 2, 4, 5, 6], 8)
    blocks = [-(-(n + s) // page) for n, s in zip(lengths, sizes)]
    order = list(range(sum(blocks) + 2))
    rng.shuffle(order)
    table, at = [], 0
    for n in blocks:
        table.append(order[at:at + n] + [-1] * (max(blocks) - n))
        at += n
    storages = LAYOUTS[layout](len(order), page)
    before = [token_view(s, page).clone() for s in storages]
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    flat = lambda lists: dev_ints([x for one in lists for x in one])
    path, counts, following, error = dev_ints([[7] * 70] * 5), dev_ints([7] * 5), dev_ints([7] * 5), dev_ints([0])
    moves = cache_moves.PageMoves(storages, page)
    drafts.accept_drafts(flat(tokens), flat(trees), flat(choices), dev_ints(starts), dev_ints(lengths), path, counts, following, moves, dev_ints(table), error)
    assert int(error) == 0
    assert [p[:c] for p, c in zip(path.tolist(), counts.tolist())] == [w[0] for w in wanted]
    assert following.tolist() == [w[1] for w in wanted]
    assert all(x == -1 for p, c in zip(path.tolist(), counts.tolist()) for x in p[c:])
    for s, old in zip(storages, before):
        want = old.clone()
        for a, (branch, _) in enumerate(wanted):
            for i, j in enumerate(branch):
                to, of = lengths[a] + i, lengths[a] + j
                want[table[a][to // page], to % page] = old[table[a][of // page], of % page]
        assert torch.equal(token_view(s, page), want)


def test_acceptance_alone_and_what_it_refuses_on_the_device():
    tokens, parents, choices = dev_ints([1, 2, 2, 3]), dev_ints([-1, 0, 0, 2]), dev_ints([2, 3, 3, 9])
    path, counts, following, error = dev_ints([[0] * 4]), dev_ints([0]), dev_ints([0]), dev_ints([0])
    drafts.accept_drafts(tokens, parents, choices, dev_ints([0, 4]), dev_ints([5]), path, counts, following)
    assert path.tolist() == [[0, 1, -1, -1]] and counts.tolist() == [2] and following.tolist() == [3]      # the lower of two equal children
    narrow = dev_ints([[0] * 3])
    drafts.accept_drafts(tokens, parents, choices, dev_ints([0, 4]), dev_ints([5]), narrow, counts, following, error_flag=error)
    assert int(error) == 3 and counts.tolist() == [0] and narrow.tolist() == [[-1] * 3]
    pool = torch.randn(3, 4, 8, device=DEV)
    kept = pool.clone()
    error.zero_()
    choices = dev_ints([2, 7, 3, 9])
    drafts.accept_drafts(dev_ints([1, 5, 2, 3]), parents, choices, dev_ints([0, 4]), dev_ints([6]), path, counts, following, cache_moves.PageMoves([pool], 4),
                         dev_ints([[0, 1, 99]]), error)
    assert path.tolist() == [[0, 2, 3, -1]] and int(error) == 2 and torch.equal(pool, kept)      # places 8, 9 lie in a page that is not there


# ------------------------------------------------------------------------------ beams
def check_select(logits, scores, wanted, ended=None, end_token=-1, got=None):
    requests, count = scores.shape
    out = got or (torch.zeros(requests, wanted, device=DEV), torch.zeros(requests, wanted, dtype=torch.int32, device=DEV),
                  torch.zeros(requests, wanted, dtype=torch.int32, device=DEV))
    beams.beam_select(logits, scores, *out, ended=ended, end_token=end_token)
    rows = logits.float().cpu().view(requests, count, -1)
    for r in range(requests):
        want_scores, want_parents, want_tokens = plain.select(rows[r], scores[r].cpu(), wanted, None if ended is None else ended[r].cpu(), end_token)
        assert out[1][r].tolist() == want_parents and out[2][r].tolist() == want_tokens, r
        for x, y in zip(out[0][r].tolist(), want_scores):
            assert x == y or (math.isnan(x) and math.isnan(y)) or abs(x - y) <= 2 * U * abs(y) + 32 * U, (r, x, y)
    return out


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("requests, count, vocab, wanted", [(1, 1, 1, 1), (1, 4, 384, 8), (3, 5, 8192, 10), (2, 3, 8193, 64), (1, 2, 32003, 4), (7, 32, 500, 64),
                                                            (2, 8, 20000, 16), (40, 1, 97, 2)])
def test_selection_against_64_bits(dtype, requests, count, vocab, wanted):
    g = torch.Generator().manual_seed(vocab + wanted)
    logits = (torch.randn(requests * count, vocab, generator=g) * 2.5).to(dtype).to(DEV)
    scores = (-torch.rand(requests, count, generator=g) * 4).to(DEV)
    check_select(logits, scores, wanted)
    ended = (torch.rand(requests, count, generator=g) < 0.4).int().to(DEV)
    check_select(logits, scores, wanted, ended, vocab // 2)
    scores[:, 1:] = -math.inf                              # the first step of a search
    check_select(logits, scores, wanted)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_selection_of_equal_and_masked_logits(dtype):
    V = 20000
    same = torch.zeros(6, V, dtype=dtype, device=DEV)      # every continuation equal: the lowest beams and tokens
    check_select(same, torch.zeros(2, 3, device=DEV), 64)
    few = torch.full((6, V), -math.inf, dtype=dtype, device=DEV)
    few[0, 17], few[1, 19999], few[1, 3], few[5, 0] = 1.0, 2.0, 2.0, -3.0
    check_select(few, torch.zeros(2, 3, device=DEV), 6)    # fewer continuations than wanted, beams without any
    coarse = (torch.randn(6, V, generator=torch.Generator().manual_seed(1)) * 2).round().to(dtype).to(DEV)
    check_select(coarse, torch.tensor([[0.0, 0.0, -1.0], [0.0, -2.0, 0.0]], device=DEV), 33)
    lowest = torch.full((2, 300), torch.finfo(dtype).min, dtype=dtype, device=DEV)
    lowest[0, 5] = 0.0
    check_select(lowest, torch.zeros(1, 2, device=DEV), 5)


def test_selection_of_what_cannot_be_ranked():
    logits = torch.randn(9, 9000, device=DEV)
    scores = torch.zeros(3, 3, device=DEV)
    logits[1, 8999] = math.nan
    logits[4, 2] = math.inf
    check_select(logits, scores, 5)
    scores[0, 1], scores[1, 1] = -math.inf, -math.inf      # dead beams are not looked at
    check_select(logits, scores, 5)
    ended = dev_ints([[0, 1, 0], [0, 1, 0], [0, 0, 0]])    # ended ones neither
    check_select(logits, torch.zeros(3, 3, device=DEV), 5, ended, 7)
    scores.zero_()
    scores[2, 0] = math.nan
    check_select(logits, scores, 5)


def test_selection_of_rows_in_a_wider_matrix_on_another_stream_and_captured():
    wide = torch.randn(8, 10000, device=DEV)
    scores = -torch.rand(2, 4, device=DEV)
    check_select(wide[:, :9001], scores, 8)
    check_select(wide[:, 1:9000], scores, 8)
    logits = wide[:, :9001].contiguous()
    want = check_select(logits, scores, 8)
    got = [torch.zeros_like(t) for t in want]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beams.beam_select(logits, scores, *got)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    outs = []
    for _ in range(2):                                     # two captured calls, whose scratch is their own
        outs.append([torch.zeros_like(t) for t in want])
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            beams.beam_select(logits, scores, *outs[-1])
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    graphs[0].replay()
    with torch.cuda.stream(other):
        graphs[1].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for out in outs for a, b in zip(out, want))


@pytest.mark.parametrize("requests, count", [(1, 1), (1, 2), (2, 4), (3, 5), (1, 8), (2, 13), (1, 32)])
@pytest.mark.parametrize("shape, dtype", [((16,), F32), ((3, 7), F32), ((5,), BF16), ((2, 64, 33), F32), ((1,), torch.int32)])
def test_slots_take_their_parents_state(requests, count, shape, dtype):
    rng = random.Random(count)
    slots = requests * count + 2
    order = list(range(slots))
    rng.shuffle(order)
    mine = [order[r * count:(r + 1) * count] for r in range(requests)]
    parents = [[rng.randrange(-1, count) for _ in range(count)] for _ in range(requests)]
    if count == 5:
        parents[0] = [1, 2, 3, 4, 0]                       # a cycle
    storages = [(torch.randn(slots, *shape, device=DEV) * 100).to(dtype) for _ in range(3)]
    before = [s.clone() for s in storages]
    error = dev_ints([0])
    cache_moves.reorder_slots(cache_moves.SlotMoves(storages), dev_ints(mine), dev_ints(parents), error)
    for s, old in zip(storages, before):
        want = old.clone()
        for own, of in zip(mine, parents):
            for slot, p in zip(own, of):
                if p >= 0:
                    want[slot] = old[own[p]]
        assert torch.equal(s, want)
    assert int(error) == 0


def test_slots_and_parents_out_of_range_stay_as_they_are():
    state = torch.randn(4, 8, device=DEV)
    kept = state.clone()
    for slots, parents in (([[0, 9]], [[0, 0]]), ([[0, 1]], [[0, 2]]), ([[0, -1]], [[1, 1]])):
        error = dev_ints([0])
        cache_moves.reorder_slots(cache_moves.SlotMoves([state]), dev_ints(slots), dev_ints(parents), error)
        assert int(error) == 4 and torch.equal(state, kept)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("requests, count, page", [(1, 2, 16), (2, 4, 5), (1, 9, 64), (2, 17, 16), (1, 32, 4)])
def test_pages_take_their_parents_tokens(layout, requests, count, page):
    rng = random.Random(count)
    first = [rng.randrange(0, 40) for _ in range(requests)]
    last = [f + rng.randrange(0, 50) for f in first]
    parents = [[rng.randrange(-1, count) for _ in range(count)] for _ in range(requests)]
    blocks = [-(-(last[r] + 1) // page) for r in range(requests) for _ in range(count)]
    order = list(range(sum(blocks) + 2))
    rng.shuffle(order)
    table, at = [], 0
    for n in blocks:
        table.append(order[at:at + n] + [-1] * (max(blocks) - n))
        at += n
    storages = LAYOUTS[layout](len(order), page)
    before = [token_view(s, page).clone() for s in storages]
    error = dev_ints([0])
    moves = cache_moves.PageMoves(storages, page)
    cache_moves.reorder_pages(moves, dev_ints(table), dev_ints(parents), dev_ints(first), dev_ints(last), max(1, max(last[r] - first[r] for r in range(requests))), error)
    for s, old in zip(storages, before):
        want = old.clone()
        for r in range(requests):
            for b, p in enumerate(parents[r]):
                for t in range(first[r], last[r]):
                    if p >= 0:
                        want[table[r * count + b][t // page], t % page] = old[table[r * count + p][t // page], t % page]
        assert torch.equal(token_view(s, page), want)
    assert int(error) == 0


def test_pages_skip_released_blocks_and_refuse_bad_ones():
    pool = torch.randn(6, 4, 8, device=DEV)
    kept = pool.clone()
    error = dev_ints([0])
    moves = cache_moves.PageMoves([pool], 4)
    cache_moves.reorder_pages(moves, dev_ints([[-1, 0], [-1, 1]]), dev_ints([[1, 0]]), dev_ints([1]), dev_ints([7]), 6, error)
    want = kept.clone()
    want[0, :3], want[1, :3] = kept[1, :3], kept[0, :3]
    assert int(error) == 0 and torch.equal(pool, want)
    kept = pool.clone()
    cache_moves.reorder_pages(moves, dev_ints([[6], [1]]), dev_ints([[0, 0]]), dev_ints([0]), dev_ints([4]), 4, error)
    assert int(error) == 2 and torch.equal(pool, kept)
    error.zero_()
    cache_moves.reorder_pages(moves, dev_ints([[0], [1]]), dev_ints([[0, 2]]), dev_ints([0]), dev_ints([4]), 4, error)
    assert int(error) == 4 and torch.equal(pool, kept)
    error.zero_()
    cache_moves.reorder_pages(moves, dev_ints([[0], [1]]), dev_ints([[0, 0]]), dev_ints([4]), dev_ints([9]), 4, error)      # behind the table
    assert int(error) == 2 and torch.equal(pool, kept)


def test_a_search_by_hand_beside_the_kernels():
    """Beams over a toy model whose next token depends on the tokens in the cache: selection, reordering and the next logits, step after step, against lists."""
    V, B, page, steps = 40, 4, 4, 9
    weights = torch.randn(V, V, generator=torch.Generator().manual_seed(5)).to(DEV)
    pool = torch.zeros(B * 4, page, 2, device=DEV)         # a "cache" that holds each token and its number
    table = dev_ints([[b * 4 + i for i in range(4)] for b in range(B)])
    state = torch.zeros(B, 4, device=DEV)
    moves, slots = cache_moves.PageMoves([pool], page), cache_moves.SlotMoves([state])
    scores = torch.tensor([[0.0] + [-math.inf] * (B - 1)], device=DEV)
    error = dev_ints([0])
    lists = [[] for _ in range(B)]
    logits = weights[:1].expand(B, V).contiguous()
    for step in range(steps):
        out = (torch.zeros(1, B, device=DEV), dev_ints([[0] * B]), dev_ints([[0] * B]))
        check_select(logits, scores, B, got=out)
        cache_moves.reorder_pages(moves, table, out[1], dev_ints([0]), dev_ints([step]), steps, error)
        cache_moves.reorder_slots(slots, dev_ints([list(range(B))]), out[1], error)
        chosen, parents = out[2][0], out[1][0].tolist()
        lists = [lists[p] + [int(t)] for p, t in zip(parents, chosen)]
        for b in range(B):
            pool[int(table[b, step // page]), step % page] = torch.tensor([float(chosen[b]), float(step)], device=DEV)
        state[:, 0] += chosen
        scores = out[0]
        logits = weights[(state[:, 0].long() * 7 + chosen.long()) % V].contiguous()
    held = pool[table.long()].reshape(B, -1, 2)[:, :steps]
    assert held[..., 0].long().tolist() == lists and state[:, 0].long().tolist() == [sum(x) for x in lists] and int(error) == 0


@pytest.mark.parametrize("lag", range(4))
def test_attention_does_not_depend_on_which_warp_is_late(lag, monkeypatch):
    """One warp of the tensor-core kernel sleeps at every turn of its loop: same bits, for streams that share the rows and for a row tile a stream."""
    rng = random.Random(9)
    steps = [Step(BF16, 6, 1, 128, 16, [900, 64], [random_tree(rng, 20), random_tree(rng, 3)], 1), Step(BF16, 6, 1, 128, 16, [700, 130], [random_tree(rng, 40), random_tree(rng, 64)], 2, 60)]
    want = [s.run() for s in steps]
    for s, w in zip(steps, want):
        s.check(w)
    source, defines = ops.lagged_draft_sources()[lag]
    monkeypatch.setitem(ops.TEST_DEFINES, source, {k: v for k, v in defines.items() if k != "HEAD_DIM"})
    for s, w in zip(steps, want):
        assert torch.equal(s.run(), w) and int(s.error) == 0


@pytest.mark.parametrize("dtype, dim", [(F32, 32), (BF16, 128)])
def test_starts_beyond_the_rows_raise_the_flag(dtype, dim):
    """A list of starts that names rows that are not there: nothing is read or written for that sequence."""
    step = Step(dtype, 6, 2, dim, 16, [40, 90], [[-1, 0, 0], [-1, 0, 1, 1]], 3)
    want = step.want()
    step.starts = [0, 3, 9]
    got = step.run()
    assert int(step.error) == 3 and (got[3:] == 7.0).all()
    step.check(got[:3], want[:3], error=3)
    masks, positions, error = dev_ints([[5]] * 7), dev_ints([5] * 7), dev_ints([0])
    drafts.draft_masks(dev_ints([-1, 0, 0, -1, 0, 1, 1]), dev_ints([0, 3, 9]), dev_ints([40, 90]), masks, positions, None, error)
    assert int(error) == 3 and masks[3:].tolist() == [[5]] * 4 and masks[:3].tolist() == [[1], [3], [5]]
    path, counts, following, error = dev_ints([[7] * 6] * 2), dev_ints([7, 7]), dev_ints([7, 7]), dev_ints([0])
    drafts.accept_drafts(dev_ints([1] * 7), dev_ints([-1, 0, 0, -1, 0, 1, 1]), dev_ints([1] * 7), dev_ints([0, 3, 9]), dev_ints([40, 90]), path, counts, following,
                         error_flag=error)
    assert int(error) == 3 and counts.tolist() == [2, 0] and path[1].tolist() == [-1] * 6


def test_a_chain_of_the_most_nodes_and_the_widest_masks():
    step = Step(BF16, 4, 2, 128, 16, [70, 3], [list(range(-1, 255)), [-1]], 5)
    step.check(step.run())
    step = Step(F32, 2, 1, 32, 16, [70], [[-1] + [0] * 255], 5, window=20)
    step.check(step.run())


@pytest.mark.parametrize("dtype, dim", [(F32, 64), (BF16, 64)])
def test_many_sequences_and_whole_items(dtype, dim):
    """More sequences than a warp looks at in one go, most of them in one CTA as a whole."""
    rng = random.Random(8)
    sizes = [rng.choice((0, 1, 2, 7)) for _ in range(75)]
    step = Step(dtype, 2, 1, dim, 16, [rng.randrange(0, 90) for _ in sizes], [random_tree(rng, n) if n else [] for n in sizes], 4)
    step.check(step.run())


@pytest.mark.parametrize("dtype, dim", [(F32, 32), (BF16, 128)])
@pytest.mark.parametrize("wrong", [-1, -500, 2 ** 31 - 1, 2000])
def test_lengths_that_no_table_row_holds_raise_the_flag(dtype, dim, wrong):
    """The sequence is left out; the others are as they were."""
    step = Step(dtype, 6, 2, dim, 16, [40, 90, 7], [[-1, 0, 0], [-1, 0, 1, 1], [-1]], 3)
    want = step.want()
    step.lengths = [40, wrong, 7]
    got = step.run()
    assert int(step.error) == 2 and (got[3:7] == 7.0).all()
    rest = [0, 1, 2, 7]
    step.check(got[rest], want[rest], error=2)


@pytest.mark.parametrize("dtype, dim", [(F32, 32), (BF16, 128)])
def test_scores_of_minus_infinity_weigh_nothing(dtype, dim):
    """Two whole tiles of keys that every row scores -inf, in front of and among finite ones; and a sequence that has no others: zeros."""
    step = Step(dtype, 4, 2, dim, 16, [600, 40], [[-1, 0, 0], [-1, 0]], 4)
    step.q = step.q.abs()
    clean = step.pages.clone()
    for a, places in ((0, [*range(256), 300, 555]), (1, range(42))):
        for j in places:
            step.pages[step.table[a][j // 16], 0, :, j % 16, 1] = -math.inf
    want = step.want()
    assert torch.isnan(want[3:]).all() and torch.isfinite(want[:3]).all()
    got = step.run()
    step.pages = clean                             # (the bound goes by the sizes of the finite keys)
    step.check(got[:3], want[:3])
    assert (got[3:] == 0.0).all()


@pytest.mark.parametrize("dtype, dim", [(F32, 32), (BF16, 128)])
def test_a_window_wider_than_any_sequence_is_none(dtype, dim):
    step = Step(dtype, 4, 2, dim, 16, [200], [[-1, 0, 0, 2]], 4)
    first = step.run()
    for window in (204, 2 ** 31, 2 ** 40):
        step.window = window
        assert torch.equal(step.run(), first)


def test_pages_want_a_page_wherever_the_parent_has_one():
    pool = torch.randn(6, 4, 8, device=DEV)
    kept = pool.clone()
    error = dev_ints([0])
    moves = cache_moves.PageMoves([pool], 4)
    cache_moves.reorder_pages(moves, dev_ints([[2, 0], [-1, 1]]), dev_ints([[0, 0]]), dev_ints([0]), dev_ints([6]), 6, error)
    kept[1, :2] = kept[0, :2]                      # the block that both have moves all the same
    assert int(error) == 2 and torch.equal(pool, kept)
    error.zero_()
    cache_moves.reorder_pages(moves, dev_ints([[2, 0], [3, 1]]), dev_ints([[0, 0]]), dev_ints([0]), dev_ints([2 ** 31 - 1]), 8, error)
    kept[3], kept[1] = kept[2], kept[0]            # as far as the table goes
    assert int(error) == 2 and torch.equal(pool, kept)


@pytest.mark.parametrize("dtype, dim", [(F32, 128), (BF16, 128), (BF16, 64)])
def test_pages_beyond_32_bits(dtype, dim):
    """A pool of more than 2^31 elements (and 2^32 bytes): what its last pages hold is read and moved as if they were the first."""
    rng = random.Random(9)
    step = Step(dtype, 4, 2, dim, 16, [300, 40], [random_tree(rng, 9), random_tree(rng, 5)], 7)
    want = step.run()
    step.check(want)
    near = step.pages.to(DEV)
    each = near[0].numel()
    far = torch.empty((2 ** 31 // each + 1 + len(near), *near.shape[1:]), dtype=dtype, device=DEV)
    shift = len(far) - len(near)
    far[shift:] = near
    tables = [dev_ints([[page if page < 0 else page + by for page in row] for row in step.table]) for by in (0, shift)]
    error, starts, lengths, positions, rows = dev_ints([0]), dev_ints(step.starts), dev_ints(step.lengths), dev_ints(step.positions), dev_ints(step.rows)
    out = torch.zeros_like(want)
    drafts.draft_attention(step.q.to(DEV), far, out, starts, lengths, positions, rows, tables[1], 4, 2, dim, dim ** -0.5, max_nodes=9, max_length=step.max_length,
                           error_flag=error)
    assert torch.equal(out, want)
    parents, tokens = dev_ints([p for t in step.trees for p in t]), dev_ints([3] * 14)
    for pool, table in ((near, tables[0]), (far, tables[1])):
        path, counts, following = dev_ints([[0] * 9] * 2), dev_ints([0, 0]), dev_ints([0, 0])
        moves = cache_moves.PageMoves([pool], 16)
        drafts.accept_drafts(tokens, parents, tokens, starts, lengths, path, counts, following, moves, table, error)
        cache_moves.reorder_pages(moves, table, dev_ints([[1, 0]]), dev_ints([0]), dev_ints([33]), 33, error)
    assert int(counts[0]) > 1 and torch.equal(far[shift:], near) and not torch.equal(near.cpu(), step.pages) and int(error) == 0


def test_slots_beyond_32_bits():
    state = torch.empty((5, 2 ** 30), dtype=torch.uint8, device=DEV)
    state[3, -64:], state[4, -64:] = 7, 9
    error = dev_ints([0])
    cache_moves.reorder_slots(cache_moves.SlotMoves([state]), dev_ints([[3, 4]]), dev_ints([[1, 0]]), error)
    assert (state[3, -64:] == 9).all() and (state[4, -64:] == 7).all() and int(error) == 0


def test_calls_at_once_and_graphs_replayed_in_turn():
    """Two streams with calls of their own, and two captured graphs: nothing of one call is another's."""
    rng = random.Random(12)
    steps = [Step(BF16, 12, 2, 128, 16, [900, 77], [random_tree(rng, 20), random_tree(rng, 31)], 5), Step(F32, 6, 2, 32, 16, [800, 500], [random_tree(rng, 9), random_tree(rng, 4)], 6)]
    calls = []
    for step in steps:
        step.check(step.run())
        q, pages, starts, lengths, positions, rows, table = (step.q.to(DEV), step.pages.to(DEV), dev_ints(step.starts), dev_ints(step.lengths), dev_ints(step.positions),
                                                             dev_ints(step.rows), dev_ints(step.table))
        logits, scores = torch.randn(8, 40000, device=DEV), -torch.rand(2, 4, device=DEV)
        out, best = torch.zeros_like(q), [torch.zeros(2, 8, dtype=t, device=DEV) for t in (F32, torch.int32, torch.int32)]

        def call(step=step, q=q, pages=pages, starts=starts, lengths=lengths, positions=positions, rows=rows, table=table, logits=logits, scores=scores, out=out, best=best):
            drafts.draft_attention(q, pages, out, starts, lengths, positions, rows, table, step.heads, step.kv_heads, step.dim, step.dim ** -0.5,
                                   max_nodes=step.max_nodes, max_length=step.max_length)
            beams.beam_select(logits, scores, *best)
        call()
        calls.append((call, [out, *best], [x.clone() for x in (out, *best)]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(20):
        for (call, outputs, _), stream in zip(calls, streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                for x in outputs:
                    x.zero_()
                call()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for _, outputs, wants in calls for a, b in zip(outputs, wants))
    graphs = []
    for call, outputs, _ in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graphs.append(graph)
    for turn in range(6):
        for (call, outputs, wants), graph, stream in zip(calls, graphs, streams):
            with torch.cuda.stream(stream if turn % 2 else torch.cuda.current_stream()):
                for x in outputs:
                    x.zero_()
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for _, outputs, wants in calls for a, b in zip(outputs, wants))
