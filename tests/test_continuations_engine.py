"""Trees and books of draft steps and beams, without a GPU."""
import pytest
import torch

from microllm_rocm_b200.cache.manager import CacheManager
from microllm_rocm_b200.engine.continuations import DraftEntry, check_tree
from microllm_rocm_b200.engine.step import StepError
from microllm_rocm_b200.parts.base import FixedStateNeed, PagedKVNeed, PagedRowsNeed


@pytest.mark.parametrize("parents, message", [
    ([0, 0], "node 0"), ([-1, -1], "node 1 cannot continue node -1"), ([-1, 1], "node 1 cannot continue node 1"), ([-1, 2, 0], "node 1"), ([-1], "2 drafted tokens and 1 parents"),
])
def test_what_is_no_tree_is_refused(parents, message):
    with pytest.raises(StepError, match=message):
        check_tree(DraftEntry("r", [1] * max(2, len(parents)), parents))


def test_trees_have_a_most():
    with pytest.raises(StepError, match="at most 256"):
        check_tree(DraftEntry("r", [1] * 257, list(range(-1, 256))))
    check_tree(DraftEntry("r", [1] * 256, list(range(-1, 255))))


def test_the_caches_moves_name_every_storage_of_a_group():
    entries = {"a": PagedKVNeed(2, 16), "b": PagedKVNeed(2, 16, window=32), "c": PagedRowsNeed(24), "d": PagedKVNeed(2, 8, value_dim=4),
               "s": FixedStateNeed((3, 5)), "t": FixedStateNeed((1,), torch.int32)}
    cache = CacheManager(entries, 4, 8, 2, device=torch.device("cpu"))
    full, window = cache.page_moves("full"), cache.page_moves("window32")
    assert cache.page_moves("full") is full
    assert sorted(layout for _, _, layout, _ in full.groups) == sorted([(9, 4, 4, 64, 0, 0), (9, 4, 1, 96, 0, 0), (9, 4, 2, 32, 2, 16)])
    assert [layout for _, _, layout, _ in window.groups] == [(9, 4, 4, 64, 0, 0)]
    assert sorted(layout for _, _, layout, _ in cache.slot_moves().groups) == [(3, 4), (3, 60)]
