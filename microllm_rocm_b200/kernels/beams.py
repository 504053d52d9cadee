"""Beam search's selection (`csrc/beams.cu`): the best continuations of every request's beams over the whole vocabulary."""
from __future__ import annotations

from ctypes import c_int, c_longlong, c_void_p
from typing import Optional

import torch

from . import build, ops
from .build import KernelError
from .cache_moves import INT, _address, need_current, need_on

MAX_BEAMS = 32              # csrc/beams.cu
MAX_WANTED = 64
SLICE = 8192                # csrc/beams.cu: logits of a slice (a CTA takes one or more of a row)

ops.register_signatures("beams.cu", {
    "mlb_beam_select": [c_void_p, c_int, c_longlong, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p, c_void_p,
                        c_longlong, c_void_p],
})


def _scratch_bytes(rows: int, vocab: int, wanted: int) -> int:
    slots = rows * -(-vocab // SLICE)
    up = lambda n: -(-n // 16) * 16
    return 2 * up(slots * 8) + up(slots * 4) + 2 * up(slots * wanted * 4)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, out_scores: torch.Tensor, out_parents: torch.Tensor, out_tokens: torch.Tensor,
                ended: Optional[torch.Tensor] = None, end_token: int = -1) -> None:
    """The best continuations of each request: of all (beam b, token t), score[b] + log softmax(logits[b])[t], the `wanted`
    largest in falling order; equal ones by the lower beam, then the lower token.

    `logits` [requests * beams, vocab] fp32 or bf16 (rows may be further apart than vocab), `scores` [requests, beams] fp32; out_scores
    fp32, out_parents (the beam within its request) and out_tokens int32, all [requests, wanted], wanted at most 64, beams at most 32.
    `ended` [requests, beams] int32: a beam with a non-zero entry has one continuation, `end_token`, which leaves its score as it is;
    its logits are not read.  A score of -inf is a beam that is not there (the first step of a search has one beam).
    Logits of -inf are never chosen; with fewer continuations than `wanted` the last ones have score -inf, parent and token -1.
    A live beam with a logit that is NaN or +inf, or a score that is, makes its request's scores NaN and its parents and tokens -1."""
    device = logits.get_device()
    if logits.dim() != 2 or logits.stride(1) != 1 or (logits.shape[0] > 1 and logits.stride(0) < logits.shape[1]):
        raise KernelError("beam_select: logits are rows of neighbouring elements that do not overlap")
    tag = ops.dtype_tag(logits)
    need_on(device, (scores, "scores", torch.float32, 2), (out_scores, "out_scores", torch.float32, 2), (out_parents, "out_parents", INT, 2),
            (out_tokens, "out_tokens", INT, 2))
    (requests, beams), (rows, vocab), wanted = scores.shape, logits.shape, out_scores.shape[1]
    if rows != requests * beams or out_scores.shape[0] != requests or out_parents.shape != out_scores.shape or out_tokens.shape != out_scores.shape:
        raise KernelError("beam_select: one row of logits per beam, one row of outputs per request")
    if not 0 < beams <= MAX_BEAMS or not 0 < wanted <= MAX_WANTED or vocab == 0:
        raise KernelError(f"beam_select: {beams} beams and {wanted} continuations of {vocab} tokens (1 to {MAX_BEAMS} and 1 to {MAX_WANTED})")
    if ended is not None:
        need_on(device, (ended, "ended", INT, 2))
        if ended.shape != scores.shape:
            raise KernelError("beam_select: one `ended` per beam")
        if not 0 <= end_token < vocab:
            raise KernelError(f"beam_select: end token {end_token} outside the vocabulary")
    if requests == 0:
        return
    need_current(device, "beam_select")
    L = ops.lib("beams.cu")
    nbytes = _scratch_bytes(rows, vocab, wanted)
    scratch = ops.scratch(nbytes, logits, "beam_select")
    build.check(L, L.mlb_beam_select(logits.data_ptr(), tag, logits.stride(0) if rows > 1 else vocab, scores.data_ptr(), _address(ended), int(end_token) if ended is not None else -1,
                                     requests, beams, vocab, wanted, out_scores.data_ptr(), out_parents.data_ptr(), out_tokens.data_ptr(),
                                     scratch.data_ptr(), nbytes, ops._stream()))
