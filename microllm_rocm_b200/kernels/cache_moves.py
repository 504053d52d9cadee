"""Moving what requests hold in the cache (`csrc/cache_moves.cu`): beams continue from their parents' cache, in place and for
all layers in one launch.

`PageMoves` and `SlotMoves` name the storages once (a program makes them when it makes its cache; `CacheManager.page_moves` and
`slot_moves` do); they hold the tensors, whose memory the kernels write.
"""
from __future__ import annotations

import ctypes
from ctypes import c_int, c_longlong, c_void_p
from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import build, ops
from .build import KernelError

MAX_STORAGES = 128          # csrc/cache_moves.cu: MAX_STORAGES
MAX_BEAMS = 32              # csrc/cache_moves.cu: MAX_BEAMS
INT = torch.int32

_PAGES = [c_void_p, c_int, c_longlong, c_int, c_int, c_int, c_int, c_int]          # bases, count, pages, page size, planes, row, planes2, row2

ops.register_signatures("cache_moves.cu", {
    "mlb_reorder_slots": [c_void_p, c_int, c_longlong, c_longlong, c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p],
    "mlb_reorder_pages": [*_PAGES, c_void_p, c_int, c_void_p, c_int, c_int, c_void_p, c_void_p, c_int, c_void_p, c_void_p],
    "mlb_accept_drafts": [*_PAGES, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_void_p, c_int, c_void_p, c_int, c_void_p, c_void_p,
                          c_int, c_void_p, c_void_p],
})


def _check_storages(storages, what: str) -> None:
    device = storages[0].device if storages else None
    for t in storages:
        if not t.is_contiguous() or t.device != device:
            raise KernelError(f"{what}: storages are contiguous tensors of one device")


class _Storages:
    """Groups of storages of one shape and type, at most MAX_STORAGES each: (addresses as a C array, count, layout)."""

    def _gather(self, storages: Sequence[torch.Tensor], layouts) -> None:
        self.tensors = list(storages)
        self.device_index = storages[0].get_device() if storages else -1
        found = {}
        for t, layout in zip(storages, layouts):
            found.setdefault(layout, []).append(t.data_ptr())
        self.groups = []
        for layout, addresses in found.items():
            for i in range(0, len(addresses), MAX_STORAGES):
                some = addresses[i:i + MAX_STORAGES]
                array = (c_void_p * len(some))(*some)
                self.groups.append((ctypes.addressof(array), len(some), layout, array))


class SlotMoves(_Storages):
    """Storages [slots, ...] of fixed-size state, one row a slot."""

    def __init__(self, storages: Sequence[torch.Tensor]):
        storages = list(storages)
        _check_storages(storages, "SlotMoves")
        for t in storages:
            if t.dim() < 2 or t.numel() == 0:
                raise KernelError("SlotMoves: a storage is [slots, ...]")
        self._gather(storages, [(t.shape[0], t.numel() // t.shape[0] * t.element_size()) for t in storages])


class PageMoves(_Storages):
    """Page pools of one page size: keys and values [pages, 2, kv heads, page, D], rows [pages, page, width], or, as
    `(tensor, (kv heads, key width, value width))`, pools [pages, elements] whose pages hold the keys of all kv heads and then the values."""

    def __init__(self, storages: Sequence[Union[torch.Tensor, Tuple[torch.Tensor, Tuple[int, int, int]]]], page_size: int):
        tensors: List[torch.Tensor] = []
        layouts = []
        for entry in storages:
            t, widths = entry if isinstance(entry, tuple) else (entry, None)
            size = t.element_size()
            if widths is not None:
                heads, dk, dv = widths
                if t.dim() != 2 or t.shape[1] != heads * page_size * (dk + dv):
                    raise KernelError(f"PageMoves: pool {tuple(t.shape)} does not hold pages of {page_size} tokens of {heads} heads of {dk} + {dv}")
                layout = (t.shape[0], page_size, heads, dk * size, heads, dv * size)
            elif t.dim() == 5 and t.shape[3] == page_size:
                layout = (t.shape[0], page_size, t.shape[1] * t.shape[2], t.shape[4] * size, 0, 0)
            elif t.dim() == 3 and t.shape[1] == page_size:
                layout = (t.shape[0], page_size, 1, t.shape[2] * size, 0, 0)
            else:
                raise KernelError(f"PageMoves: pool {tuple(t.shape)} does not hold pages of {page_size} tokens")
            if t.numel() == 0:
                raise KernelError("PageMoves: an empty pool")
            tensors.append(t)
            layouts.append(layout)
        _check_storages(tensors, "PageMoves")
        self.page_size = int(page_size)
        self._gather(tensors, layouts)


def need_on(device_index: int, *tensors) -> None:
    """Each of the (tensor, name, type, dimensions) is a contiguous tensor of that type on the device of the call's other tensors."""
    for t, name, dtype, dims in tensors:
        if t.dtype is not dtype or t.get_device() != device_index or t.dim() != dims or not t.is_contiguous():
            raise KernelError(f"{name} must be a contiguous {dtype} tensor of {dims} dimensions on the call's device, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _address(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def need_current(device_index: int, what: str) -> None:
    """Launches go to the current device's stream: the tensors have to lie there."""
    if device_index < 0:
        raise KernelError(f"{what} wants CUDA tensors (there is no CPU path)")
    current = ops._current_device() if ops._current_device is not None else torch.cuda.current_device()
    if device_index != current:
        raise KernelError(f"{what}: the tensors lie on device {device_index}, the current device is {current}")


def _need_beams(device: int, parents: torch.Tensor, what: str) -> Tuple[int, int]:
    need_on(device, (parents, "parents", INT, 2))
    requests, beams = parents.shape
    if not 0 < beams <= MAX_BEAMS:
        raise KernelError(f"{what}: {beams} beams (1 to {MAX_BEAMS})")
    return requests, beams


def reorder_slots(moves: SlotMoves, slots: torch.Tensor, parents: torch.Tensor, error_flag: Optional[torch.Tensor] = None) -> None:
    """In every storage: row slots[r, b] <- what row slots[r, parents[r, b]] held before the call, for all beams b of request r at
    once.  `slots` and `parents` [requests, beams] int32; the slots of a call are all different; a negative parent leaves
    a beam as it is.  A slot or parent out of range raises the error flag and leaves its beam as it is."""
    if not isinstance(moves, SlotMoves):
        raise KernelError("reorder_slots moves the storages of a SlotMoves")
    if not moves.groups:
        return
    device = moves.device_index
    requests, beams = _need_beams(device, parents, "reorder_slots")
    need_on(device, (slots, "slots", INT, 2))
    if slots.shape != parents.shape:
        raise KernelError("reorder_slots: one slot and one parent per beam")
    if error_flag is not None:
        need_on(device, (error_flag, "error_flag", INT, 1))
    need_current(device, "reorder_slots")
    L = ops.lib("cache_moves.cu")
    for address, count, layout, _ in moves.groups:
        build.check(L, L.mlb_reorder_slots(address, count, *layout, slots.data_ptr(), parents.data_ptr(), requests, beams, _address(error_flag), ops._stream()))


def reorder_pages(moves: PageMoves, block_table: torch.Tensor, parents: torch.Tensor, first: torch.Tensor, last: torch.Tensor, max_tokens: int,
                  error_flag: Optional[torch.Tensor] = None) -> None:
    """In every pool: tokens first[r] .. last[r] - 1 of beam b (row r * beams + b of `block_table`) <- what its parent's pages held at these places
    before the call.  `parents` [requests, beams], `first` and `last` [requests], `block_table` [requests * beams, blocks], all int32.
    Beams have pages of their own for these tokens.  Blocks of the parent that a window gave back (negative entries) are skipped; an entry
    beyond the pool, a beam without a page where its parent has one, a block beyond the table or a parent out of range raises the error flag and is skipped.
    `max_tokens`: the most tokens of a request (what the launch is sized for; more are moved all the same)."""
    if not isinstance(moves, PageMoves):
        raise KernelError("reorder_pages moves the storages of a PageMoves")
    if not moves.groups:
        return
    device = moves.device_index
    requests, beams = _need_beams(device, parents, "reorder_pages")
    need_on(device, (block_table, "block_table", INT, 2), (first, "first", INT, 1), (last, "last", INT, 1))
    if block_table.shape[0] != requests * beams or first.shape[0] != requests or last.shape[0] != requests:
        raise KernelError("reorder_pages: one row of the block table per beam, one first and last token per request")
    if max_tokens < 0 or max_tokens > block_table.shape[1] * moves.page_size:
        raise KernelError(f"reorder_pages: {max_tokens} tokens do not fit {block_table.shape[1]} blocks of {moves.page_size}")
    if error_flag is not None:
        need_on(device, (error_flag, "error_flag", INT, 1))
    if requests == 0 or max_tokens == 0:
        return
    need_current(device, "reorder_pages")
    L = ops.lib("cache_moves.cu")
    for address, count, layout, _ in moves.groups:
        build.check(L, L.mlb_reorder_pages(address, count, *layout, block_table.data_ptr(), block_table.shape[1], parents.data_ptr(), requests, beams,
                                           first.data_ptr(), last.data_ptr(), int(max_tokens), _address(error_flag), ops._stream()))
