"""Draft steps and beam search through the engine: against the engine's own one-sequence steps, against generation token by token and against a search in plain
arithmetic."""
import math
import random

import pytest
import torch

from microllm_rocm_b200.config import find_preset
from microllm_rocm_b200.engine import DraftEntry, OutOfPages, StepEntry, StepError
from microllm_rocm_b200.engine.llm import LLM
from microllm_rocm_b200.engine.loading import load_engine, random_engine
from microllm_rocm_b200.kernels import ops
from microllm_rocm_b200.sampling import GenerationConfig
from tests.helpers import BF16_REL, FP32_ATOL, make_folder, plain_logits, random_tokens, tiny_config
from tests.plain import continuations_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    return {key: make_folder(tmp_path_factory, key) for key in "abcd"}


def random_tree(rng, n):
    return [-1] + [rng.randrange(max(0, i - 4), i) for i in range(1, n)]


def argmax(logits):
    out = torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device)
    ops.argmax_rows(logits, out)
    return out


@pytest.mark.parametrize("key, dtype, page", [("a", "float32", 16), ("b", "float32", 16), ("b", "bfloat16", 16), ("c", "bfloat16", 64), ("d", "bfloat16", 16), ("d", "float32", 8)])
def test_every_node_gets_the_logits_of_its_branch(folders, key, dtype, page):
    """Both sides round at the same places, so they differ by the order of sums (fp32: the engine tests' bound twice, once for each side)."""
    engine = load_engine(folders[key], dtype=dtype, page_size=page, max_tokens=2048)
    vocab = tiny_config(key).vocab_size
    rng = random.Random(3)
    prompts = {"x": random_tokens(45, vocab, 1), "y": random_tokens(130, vocab, 2), "z": random_tokens(1, vocab, 3)}
    for name, prompt in prompts.items():
        assert engine.cache.add(name)
        engine.step([StepEntry(name, prompt)])
    entries = [DraftEntry(name, [rng.randrange(vocab) for _ in range(n)], random_tree(rng, n)) for name, n in (("x", 13), ("y", 1), ("z", 34))]
    step = engine.draft_step(entries)
    assert all(engine.cache.length(n) == len(p) for n, p in prompts.items())
    got = step.logits.float().cpu()
    row = 0
    for e in entries:
        for i in range(len(e.tokens)):
            branch = [e.tokens[j] for j in reversed(plain.chain(e.parents, i))]
            assert engine.cache.add("one")
            want = engine.step([StepEntry("one", prompts[e.request] + branch, [len(prompts[e.request]) + len(branch) - 1])])[0].float().cpu()
            engine.cache.release("one")
            limit = 2 * FP32_ATOL if dtype == "float32" else BF16_REL * float(want.abs().max())
            assert float((got[row] - want).abs().max()) <= limit, (e.request, i)
            row += 1
    engine.check_device_errors()


@pytest.mark.parametrize("key, page", [("a", 16), ("b", 16), ("b", 5), ("d", 16)])
def test_drafting_gives_the_tokens_of_decoding(folders, key, page):
    """Greedy decoding with trees of guesses, most of them wrong and some right, several requests at a time; a request goes on by plain steps in between."""
    vocab = tiny_config(key).vocab_size
    prompts = [random_tokens(n, vocab, n) for n in (7, 60, 33)]
    new = 30
    want = LLM(folders[key], dtype="float32", page_size=page, max_tokens=2048).generate(prompts, GenerationConfig(max_new_tokens=new, temperature=0.0))
    engine = load_engine(folders[key], dtype="float32", page_size=page, max_tokens=2048, guard_pages=True)
    rng = random.Random(9)
    got, root = [[] for _ in prompts], []
    for r, prompt in enumerate(prompts):
        assert engine.cache.add(r)
        root.append(int(argmax(engine.step([StepEntry(r, prompt, [len(prompt) - 1])]))[0]))
    steps = 0
    while any(len(g) < new for g in got):
        steps += 1
        entries = []
        for r, g in enumerate(got):
            if len(g) >= new:
                continue
            n = rng.randrange(1, 20)
            parents = random_tree(rng, n)
            depth = [len(plain.chain(parents, i)) - 1 for i in range(n)]
            right = want[r][len(g):] + [0] * n               # the guesses: the true token half of the time
            tokens = [root[r]] + [right[depth[i]] if rng.random() < 0.5 else rng.randrange(vocab) for i in range(1, n)]
            entries.append(DraftEntry(r, tokens, parents))
        step = engine.draft_step(entries)
        for e, a in zip(entries, engine.accept_drafts(step, argmax(step.logits))):
            got[e.request] += a.tokens
            root[e.request] = a.following
            assert engine.cache.length(e.request) == len(prompts[e.request]) + len(got[e.request])
        engine.cache.check()
        if steps % 3 == 0:                                    # a step of one token each
            live = [r for r, g in enumerate(got) if len(g) < new]
            if live:
                logits = engine.step([StepEntry(r, [root[r]], [0]) for r in live])
                for r, t in zip(live, argmax(logits).tolist()):
                    got[r].append(root[r])
                    root[r] = t
    assert [g[:new] for g in got] == want and steps < 25
    engine.check_device_errors()


def plain_search(next_logprobs, prompt, beams, new, end=None):
    """Beam search from a function tokens -> log probabilities [vocab] in 64 bits."""
    held = [([], 0.0, False)]
    for _ in range(new):
        found = []
        for b, (tokens, score, ended) in enumerate(held):
            if ended:
                found.append((-score, b, end))
                continue
            row = next_logprobs(prompt + tokens)
            top = torch.topk(row, min(beams, row.shape[0]))
            found += [(-(score + float(v)), b, int(t)) for v, t in zip(top.values, top.indices)]
        found = sorted(found)[:beams]
        held = [(held[b][0] + ([] if held[b][2] else [t]), -s, t == end if end is not None else False) for s, b, t in found]
        if all(e for _, _, e in held):
            break
    return [(t, s) for t, s, _ in held]


@pytest.mark.parametrize("key, beams, end", [("a", 4, None), ("a", 1, None), ("b", 5, None), ("b", 8, "some"), ("d", 3, "some")])
def test_beam_search_against_plain_arithmetic(folders, key, beams, end):
    llm = LLM(folders[key], dtype="float32", page_size=8, max_tokens=2048)
    vocab, new = tiny_config(key).vocab_size, 9
    prompt = random_tokens(37, vocab, 4)

    def next_logprobs(tokens):
        return torch.log_softmax(plain_logits(folders[key], tokens)[-1].double(), -1)
    if end == "some":                                      # a token that the search without an end chooses third: some beams end early
        end = plain_search(next_logprobs, prompt, beams, new)[beams // 2][0][2]
    want = plain_search(next_logprobs, prompt, beams, new, end)
    used = llm.engine.cache.stats()
    got = llm.beam_search(prompt, beams, new, end)
    assert [t for t, _ in got] == [t for t, _ in want]
    assert all(abs(a - b) <= len(t) * 4 * FP32_ATOL + 2e-6 * abs(b) for (t, a), (_, b) in zip(got, want))
    assert llm.engine.cache.stats()["live_requests"] == used["live_requests"] == 0
    llm.engine.cache.check()
    assert llm.generate([prompt], GenerationConfig(max_new_tokens=3, temperature=0.0))[0] == plain_search(next_logprobs, prompt, 1, 3)[0][0]


@pytest.mark.parametrize("preset", ["gedalix-tiny", "matidra-tiny", "fonuvik-tiny", "lozepel-tiny", "gubidra-tiny", "naburax-tiny"])
def test_beam_search_moves_every_kind_of_state(preset):
    """The same search without moving anything: every beam's whole sequence in a step of its own."""
    arch, config = find_preset(preset)
    engine = random_engine(config, seed=5, dtype="float32", page_size=4, max_tokens=1024, architecture=arch.name)
    vocab = engine.model.spec.vocab_size
    prompt = random_tokens(21, vocab, 8)
    rows = {}

    def next_logprobs(tokens):
        if tuple(tokens) not in rows:
            assert engine.cache.add("whole")
            rows[tuple(tokens)] = torch.log_softmax(engine.step([StepEntry("whole", tokens, [len(tokens) - 1])])[0].double().cpu(), -1)
            engine.cache.release("whole")
        return rows[tuple(tokens)]
    from microllm_rocm_b200.engine.continuations import beam_search
    want = plain_search(next_logprobs, prompt, 4, 8)
    got = beam_search(engine, prompt, 4, 8)
    assert [t for t, _ in got] == [t for t, _ in want]
    assert all(abs(a - b) <= 1e-4 for (_, a), (_, b) in zip(got, want))
    engine.cache.check()


def test_models_that_take_no_trees_say_so():
    arch, config = find_preset("matidra-tiny")
    engine = random_engine(config, seed=1, dtype="float32", page_size=16, max_tokens=256, architecture=arch.name)
    assert engine.cache.add("r")
    with pytest.raises(StepError, match="no drafted trees"):
        engine.draft_step([DraftEntry("r", [1, 2], [-1, 0])])


def test_draft_steps_refuse_and_leave_the_books(folders):
    engine = load_engine(folders["a"], dtype="float32", page_size=8, max_tokens=64)
    assert engine.cache.add("r")
    engine.step([StepEntry("r", [1, 2, 3])])
    with pytest.raises(StepError, match="node 1"):
        engine.draft_step([DraftEntry("r", [1, 2], [-1, 1])])
    with pytest.raises(OutOfPages):
        engine.draft_step([DraftEntry("r", [1] * 70, list(range(-1, 69)))])
    step = engine.draft_step([DraftEntry("r", [4, 5], [-1, 0])])
    engine.step([StepEntry("r", [4])])
    with pytest.raises(StepError, match="went on"):
        engine.accept_drafts(step, argmax(step.logits))
    engine.cache.check()


def test_beam_search_refuses_and_gives_everything_back(folders):
    llm = LLM(folders["a"], dtype="float32", page_size=8, max_tokens=64, max_seqs=4)
    with pytest.raises(OutOfPages, match="state slot"):
        llm.beam_search([1, 2, 3], 5, 4)
    with pytest.raises(OutOfPages):
        llm.beam_search(list(range(1, 31)), 4, 4)
    for bad in (dict(num_beams=0), dict(num_beams=33), dict(end_token=256), dict(max_new_tokens=-1)):
        with pytest.raises(ValueError):
            llm.beam_search([1, 2, 3], **bad)
    with pytest.raises(ValueError):
        llm.beam_search([], 2, 2)
    assert llm.beam_search([1, 2], 2, 0) == [([], 0.0)]
    llm.engine.cache.check()
    assert llm.engine.cache.stats()["live_requests"] == 0
    got = llm.beam_search([1, 2, 3], 2, 5)
    assert len(got) == 2 and all(len(t) == 5 and math.isfinite(s) for t, s in got)


def test_beam_search_in_windows_that_the_prompt_does_not_fit(folders):
    """Windowed layers' pools are sized for a window and a portion of the prompt, and a prompt of many such portions goes through them beam by beam."""
    config = tiny_config("b")
    prompt = random_tokens(250, config.vocab_size, 6)
    whole = LLM(folders["b"], dtype="float32", page_size=8, max_tokens=4096).beam_search(prompt, 4, 6)
    engine = load_engine(folders["b"], dtype="float32", page_size=8, max_tokens=4 * 264, max_requests=4, max_step_tokens=16)
    windowed = [g for g in engine.cache.groups.values() if g.window is not None]
    assert windowed and all(g.pool.num_pages < 4 * 32 for g in windowed)          # fewer than four prompts take
    from microllm_rocm_b200.engine.continuations import beam_search
    got = beam_search(engine, prompt, 4, 6)
    assert [t for t, _ in got] == [t for t, _ in whole]
    assert all(abs(a - b) <= 6 * 4 * FP32_ATOL for (_, a), (_, b) in zip(got, whole))
    engine.cache.check()


def test_a_request_that_was_released_and_added_again_is_another_one(folders):
    engine = load_engine(folders["a"], dtype="float32", page_size=8, max_tokens=64)
    assert engine.cache.add("r")
    engine.step([StepEntry("r", [1, 2, 3])])
    step = engine.draft_step([DraftEntry("r", [4, 5], [-1, 0])])
    engine.cache.release("r")
    assert engine.cache.add("r")
    engine.step([StepEntry("r", [6, 7, 8])])
    with pytest.raises(StepError, match="went on"):
        engine.accept_drafts(step, argmax(step.logits))
    with pytest.raises(StepError):
        engine.draft_step([])
    with pytest.raises(StepError, match="no tokens"):
        engine.draft_step([DraftEntry("r", [], [])])


@pytest.mark.parametrize("steps", [1, 2, 4, 7])
def test_a_search_beside_requests_that_the_scheduler_holds(folders, steps):
    config = GenerationConfig(max_new_tokens=12, temperature=0.0)
    prompts = [random_tokens(n, 384, n) for n in (5, 40, 17)]
    alone = LLM(folders["b"], dtype="float32", page_size=8, max_tokens=2048)
    want = alone.generate(prompts, config)
    found = alone.beam_search(prompts[1], 3, 5)
    llm = LLM(folders["b"], dtype="float32", page_size=8, max_tokens=2048)
    names = [llm.submit(p, config) for p in prompts]
    for _ in range(steps):
        llm.step()
    got = llm.beam_search(prompts[1], 3, 5)
    assert [t for t, _ in got] == [t for t, _ in found]
    assert all(abs(a - b) <= 5 * 4 * FP32_ATOL for (_, a), (_, b) in zip(got, found))
    while llm.has_work():
        llm.step()
    llm.engine.cache.check()
    assert [list(llm.poll(name).generated) for name in names] == want


def test_beam_search_refuses_what_generation_refuses(folders):
    llm = LLM(folders["a"], dtype="float32", page_size=8, max_tokens=1024)
    with pytest.raises(ValueError, match="vocabulary"):
        llm.beam_search([1, 256], 2, 2)
    with pytest.raises(ValueError, match="context"):
        llm.beam_search([1] * 500, 2, 13)
    got = llm.beam_search([1] * 500, 2, 12)                # as far as the model goes
    assert all(len(t) == 12 for t, _ in got)
    llm.engine.cache.check()
