"""Trees of drafted tokens over the paged cache (`csrc/drafts.cu`, `csrc/cache_moves.cu`): masks and positions from the trees, their
attention, and the branch that the model's choices accept.

A step brings A sequences; sequence a has `lengths[a]` cached tokens and the nodes `starts[a] .. starts[a + 1]` of the step's T
drafted ones.  Node i's `parents` entry is the index within the sequence of the node it continues, an earlier one, or -1; node 0
is the token that the last step chose, which every other node continues.  Node i's keys and values go to place lengths[a] + i of
the sequence's pages (`places`), while its position, which the rotation takes, is lengths[a] plus its depth.
"""
from __future__ import annotations

from ctypes import c_float, c_int, c_void_p
from typing import Callable, Optional

import torch

from . import build, ops
from .build import KernelError
from .cache_moves import INT, PageMoves, _address, need_current, need_on
from .device import sm_count

MAX_NODES = 256             # csrc/drafts.cu: nodes of a sequence
ROWS, KEYS = 16, 32         # csrc/drafts.cu: rows (node, head of a group) and keys a CTA works on at a time
SHARE_KEYS = 128            # a share is whole rounds of a CTA's groups, a tile of keys each (one of 724 keys: in shares of 128 18.8 us, of 256 25.9)
MAX_WINDOW = 1 << 30        # keys of a sequence at most
TC_HEAD_DIMS, TC_KEYS, TC_ROWS = (64, 128), 128, 128        # csrc/drafts_tc.cu: keys a tile, rows of a stream (a CTA has two)
TC_STRETCH = 2              # units (row tile x key tile) a CTA takes at least: a turn of both streams (one sequence of 2,074 keys 14.8 us a layer; 1: 16.3, 4: 19.7)

ops.register_signatures("drafts.cu", {
    "mlb_draft_masks": [c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p],
    "mlb_draft_attention": [c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_int, c_int, c_int, c_int, c_int,
                            c_int, c_int, c_int, c_int, c_float, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p],
})
ops.register_signatures("drafts_tc.cu", {
    "mlb_draft_attention_tc": [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_int, c_int, c_int, c_int, c_int,
                               c_int, c_int, c_int, c_float, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p],
})


_TC_DEFINES = {d: {"HEAD_DIM": d} for d in TC_HEAD_DIMS}
_sms = {}


def _sm_count(device_index: int) -> int:
    got = _sms.get(device_index)
    if got is None:
        got = _sms[device_index] = sm_count(torch.device("cuda", device_index))
    return got


def sources(head_dim: int, fp32: bool):
    """(source, defines) of what steps with drafted trees launch for layers of this head size."""
    tc = [("drafts_tc.cu", {"HEAD_DIM": head_dim})] if head_dim in TC_HEAD_DIMS and not fp32 else []
    return [("drafts.cu", {}), ("cache_moves.cu", {})] + tc


def tc_supported(head_dim: int, page_size: int, group: int, scale: float) -> bool:
    """What the tensor-core kernel takes (csrc/drafts_tc.cu): pages that divide a tile of keys, a group of heads that fits its rows."""
    return (head_dim in TC_HEAD_DIMS and page_size >= 8 and page_size % 8 == 0 and TC_KEYS % page_size == 0 and group <= TC_ROWS and scale > 0.0)


def _need_trees(device: int, starts: torch.Tensor, lengths: torch.Tensor) -> int:
    need_on(device, (starts, "starts", INT, 1), (lengths, "lengths", INT, 1))
    if starts.shape[0] != lengths.shape[0] + 1:
        raise KernelError("drafts: `starts` has one entry per sequence and one more")
    return lengths.shape[0]


def draft_masks(parents: torch.Tensor, starts: torch.Tensor, lengths: torch.Tensor, masks: torch.Tensor, positions: torch.Tensor,
                places: Optional[torch.Tensor] = None, error_flag: Optional[torch.Tensor] = None) -> None:
    """What a step's layers share: `masks` [T, words] int32, bit j of node i's row set for node i and every node above it (node
    j of the same sequence), `positions` [T] = length + depth and `places` [T] = length + index.  `words` = ceil(most nodes of a sequence / 32), at
    most 8.  A parent that is not an earlier node counts as none and raises the error flag; a sequence of more nodes than the masks hold
    raises it too and is left out."""
    device = parents.get_device()
    need_on(device, (parents, "parents", INT, 1), (masks, "masks", INT, 2), (positions, "positions", INT, 1))
    sequences = _need_trees(device, starts, lengths)
    T = parents.shape[0]
    if masks.shape[0] != T or positions.shape[0] != T or not 0 < masks.shape[1] <= MAX_NODES // 32:
        raise KernelError(f"draft_masks: one row of 1 to {MAX_NODES // 32} words and one position per node")
    if places is not None:
        need_on(device, (places, "places", INT, 1))
        if places.shape[0] != T:
            raise KernelError("draft_masks: one place per node")
    if error_flag is not None:
        need_on(device, (error_flag, "error_flag", INT, 1))
    need_current(device, "draft_masks")
    L = ops.lib("drafts.cu")
    build.check(L, L.mlb_draft_masks(parents.data_ptr(), starts.data_ptr(), lengths.data_ptr(), T, sequences, masks.shape[1], masks.data_ptr(), positions.data_ptr(),
                                     _address(places), _address(error_flag), ops._stream()))


def _shares(ctas: int, keys: int, sms: int):
    """(keys a share, shares): the keys are split until two CTAs a multiprocessor have work, down to a round of a CTA's groups, always into whole rounds; where there are
    more CTAs than multiprocessors already, until there are four, down to four rounds.  (us a layer: 4 sequences of 500 to 2,000 keys, 6 heads of 32, 12 shares of 168 keys
    22.4, 8 of 256 15.0; 4 of 1,000, 24 nodes, 12 heads of 128, 8 shares of 128 keys 59.4, 4 of 256 49.9; 16 of up to 2,000, 1 share 177, 2 of 1,024 160.)"""
    most, least = 2 * sms // max(1, ctas), SHARE_KEYS
    if ctas > sms:
        most, least = 4 * sms // ctas, 4 * SHARE_KEYS
    shares = max(1, min(-(-keys // least), most))
    share = -(-(-(-keys // shares)) // SHARE_KEYS) * SHARE_KEYS
    return share, -(-keys // share)


def _ctas(heads: int, row_tiles: int, key_tiles: int, sms: int) -> int:
    """CTAs of the tensor-core kernel: one a multiprocessor, as long as each finds TC_STRETCH units of heads x row tiles x key tiles."""
    return max(1, min(sms, -(-heads * row_tiles * key_tiles // TC_STRETCH)))


def _memory(alloc, q: torch.Tensor, nbytes: int) -> torch.Tensor:
    if alloc is None:
        return ops.scratch(nbytes, q, "draft_attention")
    got = alloc(nbytes)
    if got.get_device() != q.get_device() or not got.is_contiguous() or got.numel() * got.element_size() < nbytes or got.data_ptr() % 16:
        raise KernelError(f"draft_attention: `alloc` gave no {nbytes} bytes of the call's device that begin at a multiple of 16")
    return got


def draft_attention(q: torch.Tensor, pages: torch.Tensor, out: torch.Tensor, starts: torch.Tensor, lengths: torch.Tensor, positions: torch.Tensor,
                    masks: torch.Tensor, block_table: torch.Tensor, num_heads: int, num_kv_heads: int, head_dim: int, scale: float,
                    window: Optional[int] = None, *, max_nodes: int, max_length: int, error_flag: Optional[torch.Tensor] = None,
                    alloc: Optional[Callable[[int], torch.Tensor]] = None) -> None:
    """out[t, h] = softmax(scale q[t, h] . k) v over what node t sees: its sequence's cached tokens and the nodes of its mask, of both only
    those of the last `window` positions where one is given.  A node that sees nothing gets zeros.  A key that scores NaN or +inf makes its row NaN, one that
    scores -inf weighs nothing; a value that is not finite makes its column inf or NaN, as the sum has it, in the rows that see its key with a weight above zero
    (in fp32), and no other.

    `q` and `out` [T, heads * D], `pages` [pages, 2, kv heads, page, D] of the same type (fp32 or bf16); `positions` and `masks` as `draft_masks`
    makes them (any other mask over a sequence's nodes will do); `block_table` [sequences, blocks] int32.
    `max_nodes`: the most nodes of a sequence, which the launch is sized for (a sequence of more raises the error flag).  `max_length`: the most keys
    of a sequence, its nodes among them (how the work is cut; a longer sequence costs time only).  A sequence that its row of `block_table` has no blocks for,
    or whose `starts` name rows that are not there, raises the flag and is left out; a page that is not there raises it.  `alloc(bytes)` -> uint8 tensor: the step's own memory
    for partial results, for a caller whose launches are recorded and issued again; else it is taken and given back in the current stream's order."""
    device = q.get_device()
    tag, dtype = ops.dtype_tag(q), q.dtype
    need_on(device, (q, "q", dtype, 2), (pages, "pages", dtype, 5), (out, "out", dtype, 2), (positions, "positions", INT, 1), (masks, "masks", INT, 2),
            (block_table, "block_table", INT, 2), (starts, "starts", INT, 1), (lengths, "lengths", INT, 1))
    (T, width), (rows, words), (sequences, max_blocks) = q.shape, masks.shape, block_table.shape
    num_pages, two, nkv, page_size, d = pages.shape
    if two != 2 or nkv != num_kv_heads or d != head_dim:
        raise KernelError(f"draft_attention: pages {tuple(pages.shape)} do not match the head geometry")
    if num_kv_heads <= 0 or num_heads % num_kv_heads or not 0 < head_dim <= 256:
        raise KernelError(f"draft_attention: heads {num_heads}/{num_kv_heads} of {head_dim}")
    if (width != num_heads * head_dim or rows != T or out.shape != q.shape or positions.shape[0] != T or lengths.shape[0] != sequences
            or starts.shape[0] != sequences + 1):
        raise KernelError("draft_attention: shapes do not agree")
    if not 0 < words <= MAX_NODES // 32 or not 0 < max_nodes <= words * 32 or max_length < max_nodes:
        raise KernelError(f"draft_attention: {max_nodes} nodes among {max_length} keys in masks of {words} words (at most {MAX_NODES // 32})")
    if window is not None and window <= 0:
        raise KernelError("draft_attention: a window has at least one key")
    window = min(int(window), MAX_WINDOW) if window is not None else 0
    if error_flag is not None:
        need_on(device, (error_flag, "error_flag", INT, 1))
    if T == 0 or sequences == 0:
        return
    need_current(device, "draft_attention")
    group = num_heads // num_kv_heads
    q_at, pages_at, out_at = q.data_ptr(), pages.data_ptr(), out.data_ptr()
    if dtype is torch.bfloat16 and tc_supported(head_dim, page_size, group, scale) and not (q_at | pages_at | out_at) & 15:
        keys = min(max_length, window + max_nodes + TC_KEYS) if window else max_length
        ctas = _ctas(sequences * num_kv_heads, -(-max_nodes // (TC_ROWS // group)), -(-keys // TC_KEYS), _sm_count(device))
        scratch = _memory(alloc, q, ctas * 4 * TC_ROWS * (head_dim + 2) * 4 + 8 + 4 * sequences) if ctas > 1 else None
        L = ops.lib("drafts_tc.cu", _TC_DEFINES[head_dim])
        build.check(L, L.mlb_draft_attention_tc(q_at, pages_at, out_at, starts.data_ptr(), lengths.data_ptr(), positions.data_ptr(),
                                                masks.data_ptr(), words, block_table.data_ptr(), max_blocks, num_pages, page_size, T, sequences,
                                                int(max_nodes), num_heads, num_kv_heads, float(scale), window, TC_STRETCH, ctas, _address(scratch),
                                                _address(error_flag), ops._stream()))
        return
    keys = min(max_length, window + max_nodes + KEYS) if window else max_length
    row_tiles = -(-max_nodes * group // ROWS)
    share, shares = _shares(sequences * num_kv_heads * row_tiles, keys, _sm_count(device))
    scratch = _memory(alloc, q, shares * T * num_heads * (head_dim + 2) * 4) if shares > 1 else None
    L = ops.lib("drafts.cu")
    build.check(L, L.mlb_draft_attention(q_at, pages_at, out_at, tag, starts.data_ptr(), lengths.data_ptr(), positions.data_ptr(),
                                         masks.data_ptr(), words, block_table.data_ptr(), max_blocks, num_pages, page_size, T, sequences, int(max_nodes),
                                         num_heads, num_kv_heads, head_dim, float(scale), window, share, shares, _address(scratch),
                                         _address(error_flag), ops._stream()))


def accept_drafts(tokens: torch.Tensor, parents: torch.Tensor, choices: torch.Tensor, starts: torch.Tensor, lengths: torch.Tensor, path: torch.Tensor,
                  counts: torch.Tensor, following: torch.Tensor, moves: Optional[PageMoves] = None, block_table: Optional[torch.Tensor] = None,
                  error_flag: Optional[torch.Tensor] = None) -> None:
    """The branch of each tree that the model confirms: from node 0, the lowest child whose token is the model's choice (`choices`, e.g.
    `argmax_rows` of the nodes' logits) at its parent, and so on.  `path` [sequences, width >= most nodes] gets the nodes' indices (-1 behind them), `counts`
    how many they are, `following` the model's choice behind the last one, which the next step's node 0 is.  With `moves` their rows of every pool
    move from place lengths[a] + path[a, i] to lengths[a] + i, so that the cache holds the branch as if it had been decoded token by
    token.  All int32.  A sequence without nodes gets a count of 0; one of more than `width` or 256 nodes raises the error flag."""
    device = tokens.get_device()
    need_on(device, (tokens, "tokens", INT, 1), (parents, "parents", INT, 1), (choices, "choices", INT, 1), (path, "path", INT, 2), (counts, "counts", INT, 1),
            (following, "following", INT, 1))
    sequences, T = _need_trees(device, starts, lengths), tokens.shape
    if parents.shape != T or choices.shape != T:
        raise KernelError("accept_drafts: one token, parent and choice per node")
    if path.shape[0] != sequences or path.shape[1] == 0 or counts.shape[0] != sequences or following.shape[0] != sequences:
        raise KernelError("accept_drafts: one path, count and following token per sequence")
    if error_flag is not None:
        need_on(device, (error_flag, "error_flag", INT, 1))
    groups = []
    if moves is not None:
        if not isinstance(moves, PageMoves):
            raise KernelError("accept_drafts moves the storages of a PageMoves")
        if block_table is None:
            raise KernelError("accept_drafts: moving rows takes a block table")
        need_on(device, (block_table, "block_table", INT, 2))
        if block_table.shape[0] != sequences or (moves.groups and moves.device_index != device):
            raise KernelError("accept_drafts: one row of the block table per sequence, and pools on the same device")
        groups = moves.groups
    if sequences == 0:
        return
    need_current(device, "accept_drafts")
    L = ops.lib("cache_moves.cu")
    trees = (tokens.data_ptr(), parents.data_ptr(), choices.data_ptr(), starts.data_ptr(), lengths.data_ptr(), T[0], sequences)
    for i, (address, count, layout, _) in enumerate(groups or [(0, 0, (1, 1, 1, 1, 0, 0), None)]):
        build.check(L, L.mlb_accept_drafts(address, count, *layout, *trees, _address(block_table), block_table.shape[1] if block_table is not None else 0,
                                           path.data_ptr(), path.shape[1], counts.data_ptr(), following.data_ptr(), 1 if i == 0 else 0,
                                           _address(error_flag), ops._stream()))
