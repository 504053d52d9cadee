"""Drafted trees and beams at their edges.  Attention is held against 64 bits with the bounds of test_continuations_gpu.py (Step.check)."""
import dataclasses
import math
import random

import pytest
import torch

from microllm_rocm_b200.engine import DraftEntry, OutOfPages, StepEntry, StepError
from microllm_rocm_b200.engine.loading import load_engine
from microllm_rocm_b200.kernels import beams, ops
from tests.helpers import FP32_ATOL, make_folder, random_tokens, tiny_config
from tests.test_continuations_gpu import BF16, DEV, F32, Step, check_select, dev_ints, random_tree

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    return {key: make_folder(tmp_path_factory, key) for key in "ab"}


def argmax(logits):
    out = torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device)
    ops.argmax_rows(logits, out)
    return out


# ------------------------------------------------------------------------------ steps that overtake one another
def started(folder, *names, max_tokens=64):
    engine = load_engine(folder, dtype="float32", page_size=8, max_tokens=max_tokens)
    for name in names:
        assert engine.cache.add(name)
        engine.step([StepEntry(name, [1, 2, 3])])
    return engine


def test_of_two_draft_steps_of_a_request_only_the_later_can_be_accepted(folders):
    """The second one's keys and values lie where the first one's were."""
    engine = started(folders["a"], "r", "s")
    first = engine.draft_step([DraftEntry("s", [9], [-1]), DraftEntry("r", [4, 5, 6], [-1, 0, 0])])
    choices = argmax(first.logits)
    second = engine.draft_step([DraftEntry("r", [7, 8], [-1, 0])])
    with pytest.raises(StepError, match="went on"):
        engine.accept_drafts(first, choices)
    assert engine.cache.length("r") == engine.cache.length("s") == 3          # nothing of the refused call happened
    accepted, = engine.accept_drafts(second, argmax(second.logits))
    assert accepted.tokens[0] == 7 and engine.cache.length("r") == 3 + len(accepted.tokens)
    with pytest.raises(StepError, match="went on"):
        engine.accept_drafts(second, argmax(second.logits))
    engine.cache.check()


def test_a_step_that_did_not_run_overtakes_nothing(folders):
    engine = started(folders["a"], "r", "s")
    step = engine.draft_step([DraftEntry("r", [4, 5, 6], [-1, 0, 0])])
    with pytest.raises(OutOfPages):
        engine.step([StepEntry("r", [4]), StepEntry("s", [4] * 200)])
    with pytest.raises(StepError, match="vocabulary"):
        engine.step([StepEntry("r", [4]), StepEntry("s", [256])])
    with pytest.raises(OutOfPages):
        engine.draft_step([DraftEntry("r", [4], [-1]), DraftEntry("s", [1] * 200, list(range(-1, 199)))])
    other = engine.draft_step([DraftEntry("s", [4], [-1])])                   # another request's
    accepted, = engine.accept_drafts(step, argmax(step.logits))
    assert accepted.nodes[0] == 0 and engine.cache.length("r") == 3 + len(accepted.nodes)
    assert len(engine.accept_drafts(other, argmax(other.logits))) == 1


# ------------------------------------------------------------------------------ memory that is not aligned
@pytest.mark.parametrize("what", ["bias", "angles", "both"])
def test_trees_are_rotated_by_depth_wherever_the_weights_lie(folders, what):
    """A bias and frequencies that begin 4 bytes off the 16 that wide loads want: the positions of a tree's nodes are still their depths."""
    prompt, vocab = random_tokens(20, 384, 1), tiny_config("b").vocab_size
    rng = random.Random(4)
    entry = DraftEntry("r", [rng.randrange(vocab) for _ in range(12)], random_tree(rng, 12))
    found = []
    for moved in (False, True):
        engine = load_engine(folders["b"], dtype="float32", page_size=16, max_tokens=256)
        for block in engine.model.blocks if moved else ():
            mixer = block.mixer

            def off(t):
                room = torch.empty(t.numel() + 4, dtype=t.dtype, device=t.device)
                at = (20 - room.data_ptr() % 16) // 4 % 4
                room[at:at + t.numel()] = t
                assert room[at:].data_ptr() % 16 == 4
                return room[at:at + t.numel()]
            if what != "angles":
                assert mixer.b_qkv is not None
                mixer.b_qkv = off(mixer.b_qkv)
            if what != "bias":
                mixer.rotary = dataclasses.replace(mixer.rotary, inv_freq=off(mixer.rotary.inv_freq))
        assert engine.cache.add("r")
        engine.step([StepEntry("r", prompt)])
        step = engine.draft_step([entry])
        found.append(step.logits.float().cpu())
        engine.check_device_errors()
    assert float((found[0] - found[1]).abs().max()) <= 2 * FP32_ATOL


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d, rot, interleaved, table, off", [(64, 64, False, True, 0), (64, 64, False, False, 0), (64, 64, False, True, 1), (64, 64, True, False, 0), (64, 32, False, False, 0),
                                                             (40, 40, False, True, 0), (6, 6, False, False, 0), (32, 0, False, False, 0)])
def test_tokens_are_rotated_by_position_and_stored_by_place(dtype, d, rot, interleaved, table, off):
    """Every token alone, at its position, has the bits that all of them together have at their places."""
    nh, nkv, page, T = 4, 2, 8, 21
    rng = random.Random(d + rot)
    g = torch.Generator().manual_seed(d)
    width = (nh + 2 * nkv) * d
    qkv = torch.randn(T, width, generator=g).to(DEV)
    bias = torch.randn(width + off, generator=g).to(DEV)[off:]
    freq = torch.rand(rot // 2, generator=g).to(DEV)
    positions = [rng.randrange(40) for _ in range(T)]      # they repeat
    places = rng.sample(range(40), T)
    blocks, error = dev_ints([[3, 0, 4, 1, 2]]), dev_ints([0])

    def write(rows, where, at):
        q, pages = torch.full((len(rows), nh * d), 7.0, dtype=dtype, device=DEV), torch.full((5, 2, nkv, page, d), 7.0, dtype=dtype, device=DEV)
        ops.rope_kv_write(qkv[rows].contiguous(), bias, dev_ints(where), dev_ints([0] * len(rows)), blocks, freq, rot, interleaved, q, pages, nh, nkv, d, error,
                          ops.rope_table(dev_ints(where), freq) if table else None, at)
        return q, pages[blocks[0].long()].permute(0, 3, 1, 2, 4).reshape(40, 2 * nkv * d)
    q, rows = write(list(range(T)), positions, dev_ints(places))
    for t in range(T):
        alone, kept = write([t], [positions[t]], None)
        assert torch.equal(q[t], alone[0]) and torch.equal(rows[places[t]], kept[positions[t]])
    nobodys = [i for i in range(40) if i not in places]
    assert (rows[nobodys] == 7.0).all() and int(error) == 0
    write([0], [0], dev_ints([40]))                        # a place that no block holds
    assert int(error) == 1


# ------------------------------------------------------------------------------ values that are not finite
SPOILED = [
    # dtype, heads, kv heads, dim, lengths, nodes, window
    (F32, 4, 2, 32, [300, 200], [6, 3], None),
    (F32, 4, 2, 200, [300, 200], [6, 3], 60),
    (BF16, 4, 2, 128, [300, 20], [6, 3], None),            # one row tile, whose two streams share the rows
    (BF16, 4, 2, 64, [90, 20], [6, 3], 60),                # the same with one key tile
    (BF16, 12, 2, 64, [300, 200], [40, 50], 100),          # a row tile a stream
    (BF16, 12, 2, 128, [5000, 3000], [50, 3], None),       # items that lie in several CTAs
    (BF16, 28, 4, 128, [5000, 3000, 40], [60, 3, 64], 700),
]


def poison(step, seq, place, column, value, kv_head=1, which=1):
    step.pages[step.table[seq][place // 16], which, kv_head, place % 16, column] = value


@pytest.mark.parametrize("case", range(len(SPOILED)))
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_a_value_that_is_not_finite_stays_in_its_column(case, value):
    """Of a cached key in a tile that all rows see alike, of the last cached one, of one at a window's start, and of nodes; one column each of one kv head, and
    one column where +inf and -inf meet.  The row that 64 bits say, in every column and head."""
    dtype, heads, kv_heads, dim, lengths, nodes, window = SPOILED[case]
    rng = random.Random(case)
    step = Step(dtype, heads, kv_heads, dim, 16, lengths, [random_tree(rng, n) for n in nodes], case, window)
    clean = step.pages.clone()
    n = lengths[0]
    for column, place in enumerate((5, n // 2, n - 1, max(0, n - (window or n) + 2), n, n + 2)):
        poison(step, 0, place, 3 * column, value)
    poison(step, 0, n - 2, 20, math.inf)
    poison(step, 0, n + 1, 20, -math.inf)
    poison(step, 1, lengths[1] + 1, 21, value)
    want = step.want()
    got = step.run()
    there = torch.isfinite(want)
    assert 0 < int((~there).sum()) < want.numel() / 2
    seen = got.cpu().double().view(want.shape)
    assert torch.equal(torch.isfinite(seen), there)
    assert torch.equal(seen[~there].nan_to_num(5.0, 6.0, 7.0), want[~there].nan_to_num(5.0, 6.0, 7.0))
    step.pages = clean                                     # (the bound goes by the sizes of the finite values)
    step.check(torch.where(there, seen, 0.0).view(got.shape), torch.where(there, want, 0.0))


@pytest.mark.parametrize("case", range(len(SPOILED)))
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_a_node_of_one_kv_head_that_is_not_finite_reaches_every_head_of_its_group(case, value):
    """Its key (queries of mixed sign make every score NaN) and its value, in all columns: every element of the rows below it in that group's heads, and no other."""
    dtype, heads, kv_heads, dim, lengths, nodes, window = SPOILED[case]
    rng = random.Random(case)
    step = Step(dtype, heads, kv_heads, dim, 16, lengths, [random_tree(rng, n) for n in nodes], case, window)
    want = step.want()
    clean = step.pages.clone()
    below = torch.zeros(want.shape, dtype=torch.bool)
    group = heads // kv_heads
    for t in range(nodes[0]):
        if (step.rows[t][0] >> 2) & 1:
            below[t, group:2 * group] = True
    assert 0 < int(below.any(-1).any(-1).sum()) < nodes[0]
    for which in (0, 1, None):
        step.pages = clean.clone()
        for half in (0, 1) if which is None else (which,):
            poison(step, 0, lengths[0] + 2, slice(None), value, which=half)
        got = step.run()
        seen = got.cpu().double().view(want.shape)
        assert torch.equal(~torch.isfinite(seen), below), which
        step.pages = clean
        step.check(torch.where(below, 0.0, seen).view(got.shape), torch.where(below, 0.0, want))


# ------------------------------------------------------------------------------ equal scores of different beams
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("far", [-80.0, -33.25, -20.5])
def test_equal_scores_of_different_beams_go_to_the_lower_one(far, dtype):
    """A beam whose score is `far` and that has one continuation, beside one whose second continuation lies that far below its first: 64 bits say equal or nearly so, and
    a distance that was scaled by a rounded constant would put the higher beam first."""
    V = 9000
    logits = torch.full((2, V), -math.inf, dtype=dtype, device=DEV)
    logits[0, 7] = 3.0
    logits[1, 11], logits[1, 12] = 0.0, far
    check_select(logits, torch.tensor([[far, 0.0]], device=DEV), 3)
    flipped, scores = logits.flip(0).contiguous(), torch.tensor([[0.0, far]], device=DEV)
    if far == -20.5 and dtype == BF16:
        # One thread has both terms: 1 + e^-20.5 = 1 + 1.25e-9 is 1 in fp32, whose half step is 2^-25 = 3.0e-8 below and 6.0e-8 above 1, so a normaliser of 0 where 64 bits
        # have 1.25e-9.  The candidates 1.25e-9 apart are equal then, and the lower beam's comes first.
        got = torch.zeros(1, 3, device=DEV), dev_ints([[0] * 3]), dev_ints([[0] * 3])
        beams.beam_select(flipped, scores, *got)
        assert got[1].tolist() == [[0, 0, 1]] and got[2].tolist() == [[11, 12, 7]] and got[0].tolist() == [[0.0, far, far]]
    else:
        check_select(flipped, scores, 3)
    logits[1, 11], logits[1, 12] = 1000.0, 1000.0 + far if dtype == F32 else 920.0
    check_select(logits, torch.tensor([[far if dtype == F32 else -80.0, 0.0]], device=DEV), 3)


def test_scores_are_the_logarithms_of_the_softmax_nearly_in_64_bits():
    """Scores that come out near 0, where fp32 shows what the normaliser is worth.  A term of the row's sum, 2^-a of the largest, is off by 2^-22 of the function (its
    documented error) and by its argument's rounding, (a + 1) 2^-24 log 2 at most.  Weighted by its share of the sum these are 2^-22 and 2^-24 times the entropy and one (12 at
    most for 50,000 tokens), log2 e's rounding is 2^-26 of the entropy, and sums of 32 terms add 5 x 2^-24: 2^-24 (4 + 13 + 3 + 5) = 1.5e-6, if all went one way."""
    g = torch.Generator().manual_seed(3)
    for scale, V in ((0.1, 50000), (1.0, 9000), (2.5, 50000), (6.0, 50000)):
        rows = torch.randn(8, V, generator=g) * scale
        top = rows.max(1).values.double()
        start = (torch.logsumexp(rows.double(), 1) - top).float()              # the best continuation comes out within 1e-6 of 0
        out = (torch.zeros(8, 1, device=DEV), torch.zeros(8, 1, dtype=torch.int32, device=DEV), torch.zeros(8, 1, dtype=torch.int32, device=DEV))
        beams.beam_select(rows.to(DEV), start.view(8, 1).to(DEV), *out)
        want = start.double() + top - torch.logsumexp(rows.double(), 1)
        off = (out[0].cpu().double().view(8) - want).abs().max()
        print(f"scale {scale}, {V} tokens: off by {float(off):.2e}")
        assert float(off) <= 1.5e-6


# ------------------------------------------------------------------------------ warps that are late, waits that run out
def cut_steps(dim):
    """Streams that share the rows, a row tile a stream, and CTAs that walk through many items, whose queries follow one another into the same place."""
    rng = random.Random(9)
    sizes = [1 + rng.randrange(40) for _ in range(70)]
    return [Step(BF16, 6, 1, dim, 16, [900, 64], [random_tree(rng, 20), random_tree(rng, 3)], 1), Step(BF16, 6, 1, dim, 16, [700, 130], [random_tree(rng, 40), random_tree(rng, 64)], 2, 60),
            Step(BF16, 6, 6, dim, 16, [rng.randrange(300) for _ in sizes], [random_tree(rng, n) for n in sizes], 3)]


def with_defines(monkeypatch, defines):
    monkeypatch.setitem(ops.TEST_DEFINES, "drafts_tc.cu", {k: v for k, v in defines.items() if k != "HEAD_DIM"})


@pytest.mark.parametrize("which", [i for i, (_, d) in enumerate(ops.lagged_draft_sources()) if "MLB_LAG_WARP" in d])
def test_items_that_follow_one_another_do_not_depend_on_which_warp_is_late(which, monkeypatch):
    _, defines = ops.lagged_draft_sources()[which]
    steps = cut_steps(defines["HEAD_DIM"])
    want = [s.run() for s in steps]
    for s, w in zip(steps, want):
        s.check(w)
    with_defines(monkeypatch, defines)
    for s, w in zip(steps, want):
        assert torch.equal(s.run(), w) and int(s.error) == 0


@pytest.mark.parametrize("polls", [0, 1, 4])
def test_a_wait_that_runs_out_is_reported_and_leaves_nothing_behind(polls, monkeypatch):
    """Every wait gives up after a few polls: the error flag says so (or, where none ran out, the rows are right), the kernel ends, and the next launch is as ever."""
    steps = cut_steps(128)
    want = [s.run() for s in steps]
    with_defines(monkeypatch, {"MLB_SPIN_LIMIT": polls})
    for s, w in zip(steps, want):
        for _ in range(3):
            got = s.run()
            code = int(s.error)
            assert 40 <= code <= 54 if polls == 0 else code == 0 or 40 <= code <= 54
            assert code != 0 or torch.equal(got, w)
    monkeypatch.undo()
    for s, w in zip(steps, want):
        assert torch.equal(s.run(), w) and int(s.error) == 0
