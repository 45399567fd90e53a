"""Beam search behind the logits (``csrc/beam.cu``): the choice of the next beams and the cached states that follow them."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from ..runtime.kv import PAGE
from ._lib import check, cuda
from .decode import sm_count

MAX_BEAMS = 64
_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_float
_entries: dict = {}


def _fn(name, *args):
    fn = _entries.get(name)
    if fn is None:
        fn = getattr(cuda(), name)
        fn.argtypes = args
        _entries[name] = fn
    return fn


def _ptr(t: Optional[torch.Tensor]):
    return t.data_ptr() if t is not None else None


class BeamScratch:
    """Scratch of :func:`beam_select` for ``groups`` searches of ``beams`` over ``vocab`` ids; the calls that use one follow each
    other on one stream."""

    def __init__(self, groups: int, beams: int, vocab: int, device):
        if groups < 1 or vocab < 1 or not 1 <= beams <= MAX_BEAMS:
            raise ValueError(f"searches of 1 to {MAX_BEAMS} beams")
        self.groups, self.beams, self.vocab = groups, beams, vocab
        self.device = torch.device(device)
        if groups * beams > 65535:
            raise ValueError("at most 65,535 beams in all")
        self.sms = sm_count(self.device) if self.device.type == "cuda" else 1
        size = _fn("bl_beam_work_bytes", _I, _I, _I, _I)
        size.restype = _L
        self.work = torch.zeros(size(vocab, groups, beams, self.sms), dtype=torch.uint8, device=self.device)


def _same(name: str, t: torch.Tensor, dtype, n: int) -> None:
    if t.dtype != dtype or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous {dtype}, {n} values")


def beam_select(logits: torch.Tensor, scores: torch.Tensor, scratch: BeamScratch, parent: torch.Tensor, token: torch.Tensor,
                out_scores: torch.Tensor, *, done: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                out_done: Optional[torch.Tensor] = None, out_lengths: Optional[torch.Tensor] = None, eos: int = -1,
                alpha: float = 0.0, fault: Optional[torch.Tensor] = None) -> None:
    """The next beams of every search, best first: ``parent`` (a beam of the search), ``token`` and ``out_scores`` [groups, beams].

    ``logits`` fp32 [groups * beams, vocab] (rows may be strided), ``scores`` fp32 [groups, beams]; a score of -inf is no beam (the
    first step has one beam a search) and its logits are not read.  ``done`` int32: a finished beam continues as itself, with
    token ``eos``.  ``lengths`` int32: tokens of each beam; candidates are ranked by score / length ** alpha, the new token
    counted.  ``out_done`` / ``out_lengths``: the same of the next beams.  Ties go to the lower beam, then to the lower id.  Ids with
    a logit of -inf are no candidates; where a search has too few, the last places get parent = their own index, token ``eos`` (0
    without one), score -inf and done.  A search with a NaN or +inf among its logits or scores gets NaN scores and raises
    ``fault``."""
    G, B = scratch.groups, scratch.beams
    n = G * B
    if logits.dtype != torch.float32 or logits.dim() != 2 or logits.shape[0] != n or logits.shape[1] != scratch.vocab or \
            (logits.stride(1) != 1 and scratch.vocab > 1):
        raise ValueError(f"logits: fp32 [{n}, {scratch.vocab}], ids next to each other")
    _same("scores", scores, torch.float32, n)
    _same("out_scores", out_scores, torch.float32, n)
    _same("parent", parent, torch.int32, n)
    _same("token", token, torch.int32, n)
    for name, t in (("done", done), ("lengths", lengths), ("out_done", out_done), ("out_lengths", out_lengths)):
        if t is not None:
            _same(name, t, torch.int32, n)
    if eos >= scratch.vocab or (done is not None and eos < 0):
        raise ValueError("finished beams need the id of the end")
    if lengths is None and (alpha != 0.0 or out_lengths is not None):
        raise ValueError("a rank by length needs the lengths")
    fn = _fn("bl_beam_select", _P, _L, _I, _I, _I, _P, _P, _P, _I, _F, _P, _I, _P, _P, _P, _P, _P, _P, _P)
    check(fn(logits.data_ptr(), max(logits.stride(0), scratch.vocab), scratch.vocab, G, B, scores.data_ptr(), _ptr(done), _ptr(lengths), eos,
             alpha, scratch.work.data_ptr(), scratch.sms, parent.data_ptr(), token.data_ptr(), out_scores.data_ptr(), _ptr(out_done),
             _ptr(out_lengths), _ptr(fault), torch.cuda.current_stream(scratch.device).cuda_stream), "bl_beam_select")


def beam_reorder(k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, table_out: torch.Tensor, slots: torch.Tensor,
                 parent: torch.Tensor, held: torch.Tensor, fault: Optional[torch.Tensor] = None) -> None:
    """Cached states behind a choice: the beam in place i of a search (slot ``slots[g, i]``) continues the history of
    ``parent[g, i]``, of which ``held[g]`` positions are cached.

    ``k``, ``v``: the pools of all layers, [layers, pages, heads, 64, row] of any type (a latent cache has a ``v`` without
    values).  ``table_out``, another table than ``table``, gets the rows of these slots: full pages are the parent's, pages behind the
    one being filled stay the slot's.  In the page being filled a parent's first child goes on; each further child takes
    over the page of a beam that has none and a copy of the positions in it.  The pages from the one being filled on must belong
    to one slot each.  A search whose parents, slots or positions are out of range stays as it is and raises ``fault``."""
    G, B = parent.shape
    for name, t, n in (("slots", slots, G * B), ("parent", parent, G * B), ("held", held, G)):
        _same(name, t, torch.int32, n)
    if k.dim() != 5 or v.dim() != 5 or k.shape[:4] != v.shape[:4] or k.shape[3] != PAGE or not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError(f"pools: contiguous [layers, pages, heads, {PAGE}, row], alike but for the row")
    for t in (table, table_out):
        if t.dtype != torch.int32 or t.dim() != 2 or not t.is_contiguous() or t.shape != table.shape:
            raise ValueError("tables: contiguous int32 [slots, pages]")
    if table.data_ptr() == table_out.data_ptr():
        raise ValueError("the new table is written while the old one is read: another tensor")
    if B > MAX_BEAMS:
        raise ValueError(f"at most {MAX_BEAMS} beams a search")
    fn = _fn("bl_beam_reorder", _P, _P, _L, _L, _I, _I, _I, _P, _P, _I, _I, _P, _P, _P, _I, _I, _P, _P)
    check(fn(k.data_ptr(), v.data_ptr(), k.shape[4] * k.element_size(), v.shape[4] * v.element_size(), k.shape[0], k.shape[1],
             k.shape[2], table.data_ptr(), table_out.data_ptr(), table.shape[0], table.shape[1], slots.data_ptr(), parent.data_ptr(),
             held.data_ptr(), G, B, _ptr(fault), torch.cuda.current_stream(parent.device).cuda_stream), "bl_beam_reorder")
