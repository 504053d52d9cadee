"""Drafted trees and beams at their edges."""
import pytest
import torch

from microllm_rocm_b200.engine import DraftEntry, OutOfPages, StepEntry, StepError
from microllm_rocm_b200.engine.loading import load_engine
from microllm_rocm_b200.kernels import ops
from tests.helpers import make_folder

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
