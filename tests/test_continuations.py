"""What the calls for drafted trees and beams refuse, and how they cut their work: no GPU."""
import pytest
import torch

from microllm_rocm_b200.engine.step import device_error_text
from microllm_rocm_b200.kernels import beams, cache_moves, drafts, ops
from microllm_rocm_b200.kernels.build import KernelError
from tests.plain import continuations_plain as plain

I = torch.int32


def ints(*shape):
    return torch.zeros(shape, dtype=I)


def masks_arguments(**change):
    a = dict(parents=ints(5), starts=ints(3), lengths=ints(2), masks=ints(5, 1), positions=ints(5), places=ints(5), error_flag=ints(1))
    a.update(change)
    return a


@pytest.mark.parametrize("change, message", [
    ({}, "no CPU path"),
    ({"parents": torch.zeros(5)}, "parents"),
    ({"starts": ints(2)}, "one entry per sequence and one more"),
    ({"masks": ints(5, 9)}, "1 to 8 words"),
    ({"masks": ints(4, 1)}, "1 to 8 words"),
    ({"positions": ints(6)}, "one position per node"),
    ({"positions": ints(10)[::2]}, "contiguous"),
    ({"places": ints(4)}, "one place per node"),
    ({"error_flag": torch.zeros(1)}, "error_flag"),
])
def test_draft_masks_refuses(change, message):
    with pytest.raises(KernelError, match=message):
        drafts.draft_masks(**masks_arguments(**change))


def attention_arguments(**change):
    a = dict(q=torch.zeros(5, 64), pages=torch.zeros(4, 2, 2, 16, 16), out=torch.zeros(5, 64), starts=ints(3), lengths=ints(2), positions=ints(5),
             masks=ints(5, 1), block_table=ints(2, 3), num_heads=4, num_kv_heads=2, head_dim=16, scale=0.25, window=None, max_nodes=5, max_length=40)
    a.update(change)
    return a


@pytest.mark.parametrize("change, message", [
    ({}, "no CPU path"),
    ({"q": torch.zeros(5, 64, dtype=torch.float16)}, "unsupported tensor dtype"),
    ({"pages": torch.zeros(4, 2, 2, 16, 16, dtype=torch.bfloat16)}, "pages"),
    ({"out": torch.zeros(5, 64, dtype=torch.bfloat16)}, "out"),
    ({"out": torch.zeros(5, 128)[:, ::2]}, "out"),
    ({"pages": torch.zeros(4, 2, 4, 16, 16)}, "head geometry"),
    ({"num_heads": 3}, "heads 3/2"),
    ({"positions": ints(4)}, "shapes do not agree"),
    ({"block_table": ints(3, 3)}, "shapes do not agree"),
    ({"max_nodes": 33, "max_length": 80}, "33 nodes"),
    ({"max_nodes": 0}, "0 nodes"),
    ({"max_length": 4}, "5 nodes among 4 keys"),
    ({"window": 0}, "at least one key"),
])
def test_draft_attention_refuses(change, message):
    with pytest.raises(KernelError, match=message):
        drafts.draft_attention(**attention_arguments(**change))


def accept_arguments(**change):
    a = dict(tokens=ints(5), parents=ints(5), choices=ints(5), starts=ints(3), lengths=ints(2), path=ints(2, 5), counts=ints(2), following=ints(2))
    a.update(change)
    return a


@pytest.mark.parametrize("change, message", [
    ({}, "no CPU path"),
    ({"choices": ints(4)}, "one token, parent and choice per node"),
    ({"path": ints(2, 0)}, "one path"),
    ({"counts": ints(3)}, "one path"),
    ({"moves": cache_moves.PageMoves([torch.zeros(4, 2, 2, 16, 16)], 16)}, "block table"),
    ({"moves": cache_moves.PageMoves([torch.zeros(4, 2, 2, 16, 16)], 16), "block_table": ints(3, 2)}, "one row of the block table"),
    ({"moves": cache_moves.SlotMoves([torch.zeros(4, 2)]), "block_table": ints(2, 2)}, "PageMoves"),
])
def test_accept_drafts_refuses(change, message):
    with pytest.raises(KernelError, match=message):
        drafts.accept_drafts(**accept_arguments(**change))


def select_arguments(**change):
    a = dict(logits=torch.zeros(6, 50), scores=torch.zeros(2, 3), out_scores=torch.zeros(2, 4), out_parents=ints(2, 4), out_tokens=ints(2, 4))
    a.update(change)
    return a


@pytest.mark.parametrize("change, message", [
    ({}, "no CPU path"),
    ({"logits": torch.zeros(6, 50, dtype=torch.float16)}, "unsupported tensor dtype"),
    ({"logits": torch.zeros(50, 6).t()}, "rows of neighbouring elements"),
    ({"logits": torch.zeros(1, 50).expand(6, 50)}, "do not overlap"),
    ({"logits": torch.zeros(5, 50)}, "one row of logits per beam"),
    ({"out_tokens": ints(2, 5)}, "one row of outputs"),
    ({"scores": torch.zeros(1, 33), "logits": torch.zeros(33, 50), "out_scores": torch.zeros(1, 4), "out_parents": ints(1, 4), "out_tokens": ints(1, 4)}, "33 beams"),
    ({"out_scores": torch.zeros(2, 65), "out_parents": ints(2, 65), "out_tokens": ints(2, 65)}, "65 continuations"),
    ({"ended": ints(2, 3)}, "end token -1"),
    ({"ended": ints(2, 3), "end_token": 50}, "end token 50"),
    ({"ended": ints(3, 2), "end_token": 1}, "one `ended` per beam"),
])
def test_beam_select_refuses(change, message):
    with pytest.raises(KernelError, match=message):
        beams.beam_select(**select_arguments(**change))


@pytest.mark.parametrize("call, message", [
    (lambda: cache_moves.PageMoves([torch.zeros(4, 2, 2, 16, 16)], 8), "pages of 8 tokens"),
    (lambda: cache_moves.PageMoves([(torch.zeros(4, 100), (2, 3, 4))], 16), "2 heads of 3 \\+ 4"),
    (lambda: cache_moves.PageMoves([torch.zeros(4, 16, 8).transpose(0, 1)], 4), "contiguous"),
    (lambda: cache_moves.SlotMoves([torch.zeros(4)]), "slots, ..."),
    (lambda: cache_moves.reorder_slots(cache_moves.SlotMoves([torch.zeros(4, 6)]), ints(1, 3), ints(1, 2)), "one slot and one parent"),
    (lambda: cache_moves.reorder_slots(cache_moves.SlotMoves([torch.zeros(4, 6)]), ints(1, 33), ints(1, 33)), "33 beams"),
    (lambda: cache_moves.reorder_slots(cache_moves.SlotMoves([torch.zeros(4, 6)]), ints(1, 3), ints(1, 3)), "no CPU path"),
    (lambda: cache_moves.reorder_slots(cache_moves.PageMoves([torch.zeros(4, 4, 6)], 4), ints(1, 3), ints(1, 3)), "SlotMoves"),
    (lambda: cache_moves.reorder_pages(cache_moves.PageMoves([torch.zeros(4, 4, 6)], 4), ints(3, 2), ints(1, 3), ints(1), ints(1), 8), "no CPU path"),
    (lambda: cache_moves.reorder_pages(cache_moves.PageMoves([torch.zeros(4, 4, 6)], 4), ints(3, 2), ints(1, 3), ints(1), ints(1), 9), "9 tokens do not fit"),
    (lambda: cache_moves.reorder_pages(cache_moves.PageMoves([torch.zeros(4, 4, 6)], 4), ints(2, 2), ints(1, 3), ints(1), ints(1), 8), "one row of the block table"),
    (lambda: cache_moves.reorder_pages(cache_moves.PageMoves([torch.zeros(4, 4, 6)], 4), ints(3, 2), ints(1, 3), ints(2), ints(1), 8), "one first and last"),
])
def test_moves_refuse(call, message):
    with pytest.raises(KernelError, match=message):
        call()


def test_storages_of_one_layout_share_a_launch():
    kv, rows = [torch.zeros(5, 2, 2, 8, 4) for _ in range(130)], [torch.zeros(5, 8, 12) for _ in range(3)]
    moves = cache_moves.PageMoves(kv + rows + [(torch.zeros(5, 2 * 8 * 7), (2, 3, 4))], 8)
    assert [(count, layout) for _, count, layout, _ in moves.groups] == [(128, (5, 8, 4, 16, 0, 0)), (2, (5, 8, 4, 16, 0, 0)), (3, (5, 8, 1, 48, 0, 0)),
                                                                        (1, (5, 8, 2, 12, 2, 16))]


@pytest.mark.parametrize("ctas, keys", [(1, 1), (1, 63), (1, 64), (1, 5000), (3, 131072), (148, 1000), (200, 5000), (297, 64), (5000, 100000)])
def test_shares_cover_the_keys(ctas, keys):
    share, shares = drafts._shares(ctas, keys, 148)
    assert share % drafts.SHARE_KEYS == 0 and shares >= 1 and share * shares >= keys and share * (shares - 1) < keys
    assert ctas * shares <= max((4 if ctas > 148 else 2) * 148, ctas)


def test_tensor_core_attention_takes_a_cta_a_multiprocessor_at_most():
    assert [drafts._ctas(*x, 148) for x in ((1, 1, 1), (2, 2, 17), (64, 4, 17), (1, 1, 2))] == [1, 34, 148, 1]


def test_scratch_on_the_second_stream_is_the_steps(monkeypatch):
    monkeypatch.setattr(ops._launch_on, "side", 7, raising=False)
    with pytest.raises(KernelError, match="second stream"):
        ops.scratch(64, torch.empty(1), "beam_select")
    kept = torch.empty(64, dtype=torch.uint8)
    monkeypatch.setattr(ops._launch_on, "scratch", lambda n: kept[:n], raising=False)
    assert ops.scratch(32, torch.empty(1), "beam_select").data_ptr() == kept.data_ptr()


def test_error_texts():
    assert "tree" in device_error_text(3) and "beam" in device_error_text(4) and "page" in device_error_text(2)


def test_plain_definitions():
    tree = [-1, 0, 0, 1, 1, 2]
    rows, positions, places = plain.masks([tree], [7], 1)
    assert rows == [[1], [3], [5], [11], [19], [37]] and positions == [7, 8, 8, 9, 9, 9] and places == [7, 8, 9, 10, 11, 12]
    assert plain.accept([5, 6, 6, 8, 9, 8], tree, [6, 8, 8, 1, 2, 3]) == ([0, 1, 3], 1)
    scores, parents, tokens = plain.select(torch.zeros(2, 3), torch.tensor([0.0, 0.0]), 7)
    assert parents == [0, 0, 0, 1, 1, 1, -1] and tokens == [0, 1, 2, 0, 1, 2, -1]


def test_memory_of_the_callers_own_is_looked_at():
    q, room = torch.zeros(4, 8), torch.zeros(256, dtype=torch.uint8)
    at = -room.data_ptr() % 16
    assert drafts._memory(lambda n: room[at:at + n], q, 64).numel() == 64
    for bad in (lambda n: room[at:at + n - 1], lambda n: room[at + 8:at + 8 + n], lambda n: room[at:at + 2 * n:2]):
        with pytest.raises(KernelError, match="64 bytes"):
            drafts._memory(bad, q, 64)
