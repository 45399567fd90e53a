"""Beam search behind the logits (``csrc/beam.cu``): the choice of the next beams and the cached states that follow them."""
from __future__ import annotations

import ctypes
import struct
from typing import Optional

import torch

from ..runtime.kv import PAGE
from ._lib import I, check, cuda, fault_ptr, p, raw_stream
from .decode import sm_count

MAX_BEAMS = 64
MAX_ALPHA = 16              # length ** alpha and a score times it stay in range of 64 bits for any length of 32
_SELECT, _REORDER = struct.Struct("P1l11P5if"), struct.Struct("2P2l7P7i4x")      # BeamSelectCall, BeamReorderCall in the source
_entries: dict = {}


def _fn(name):
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(cuda(), name)
        fn.argtypes = [ctypes.c_char_p]
    return fn


def _same(name: str, t: torch.Tensor, dtype, n: int, index: int) -> int:
    if t.dtype is not dtype or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous {dtype}, {n} values")
    if t.get_device() != index:
        raise ValueError(f"{name}: on another device than the rest")
    return t.data_ptr()


class BeamScratch:
    """Scratch of :func:`beam_select` for ``groups`` searches of ``beams`` over ``vocab`` ids; the calls that use one follow each
    other on one stream."""

    def __init__(self, groups: int, beams: int, vocab: int, device):
        if groups < 1 or vocab < 1 or not 1 <= beams <= MAX_BEAMS:
            raise ValueError(f"searches of 1 to {MAX_BEAMS} beams")
        self.groups, self.beams, self.vocab = groups, beams, vocab
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        if groups * beams > 65535:
            raise ValueError("at most 65,535 beams in all")
        sms = sm_count(self.device) if self.device.type == "cuda" else 1
        self.chunks = cuda().bl_beam_chunks(I(vocab), I(groups * beams), I(beams), I(sms))
        self.index = self.device.index if self.device.type == "cuda" else -1      # as Tensor.get_device() says it
        size = cuda().bl_beam_work_bytes
        size.restype = ctypes.c_long
        self.work = torch.zeros(size(groups, beams, self.chunks), dtype=torch.uint8, device=self.device)
        self.work_ptr = self.work.data_ptr()


def beam_select(logits: torch.Tensor, scores: torch.Tensor, scratch: BeamScratch, parent: torch.Tensor, token: torch.Tensor,
                out_scores: torch.Tensor, *, done: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                out_done: Optional[torch.Tensor] = None, out_lengths: Optional[torch.Tensor] = None, eos: int = -1,
                alpha: float = 0.0, fault: Optional[torch.Tensor] = None) -> None:
    """The next beams of every search, best first: ``parent`` (a beam of the search), ``token`` and ``out_scores`` [groups, beams].

    ``logits`` fp32 [groups * beams, vocab] (rows may be strided), ``scores`` fp32 [groups, beams]; a score of -inf is no beam (the
    first step has one beam a search) and its logits are not read.  ``done`` int32: a finished beam continues as itself, with
    token ``eos``.  ``lengths`` int32: tokens of each beam; candidates are ranked by score / length ** alpha (``alpha`` of -16 to 16), the new
    token counted.  ``out_done`` / ``out_lengths``: the same of the next beams.  Ties go to the lower beam, then to the lower id.  Ids with
    a logit of -inf are no candidates; where a search has too few, the last places get parent = their own index, token ``eos`` (0
    without one), score -inf and done.  A search with a NaN or +inf among its logits or scores gets NaN scores and raises
    ``fault``.  The outputs are tensors of their own: blocks that start late still read the inputs when the first places of a
    search are written."""
    G, B, V, index = scratch.groups, scratch.beams, scratch.vocab, scratch.index
    n = G * B
    if logits.dtype is not torch.float32 or logits.shape != (n, V) or (logits.stride(1) != 1 and V > 1):
        raise ValueError(f"logits: fp32 [{n}, {V}], ids next to each other")
    if logits.get_device() != index:
        raise ValueError("logits: on another device than the scratch")
    i32 = torch.int32
    at = (_same("scores", scores, torch.float32, n, index), _same("done", done, i32, n, index) if done is not None else 0,
          _same("lengths", lengths, i32, n, index) if lengths is not None else 0, scratch.work_ptr,
          _same("parent", parent, i32, n, index), _same("token", token, i32, n, index),
          _same("out_scores", out_scores, torch.float32, n, index),
          _same("out_done", out_done, i32, n, index) if out_done is not None else 0,
          _same("out_lengths", out_lengths, i32, n, index) if out_lengths is not None else 0,
          0 if fault is None else fault_ptr(fault, index))
    old_scores, old_done, old_lengths = at[:3]
    out = at[4:9]
    if old_scores in out or (old_done and old_done in out) or (old_lengths and old_lengths in out):
        raise ValueError("the next beams are written while the old ones are read: other tensors")
    if eos >= V or (done is not None and eos < 0):
        raise ValueError("finished beams need the id of the end")
    if not -MAX_ALPHA <= alpha <= MAX_ALPHA:
        raise ValueError(f"alpha: -{MAX_ALPHA} to {MAX_ALPHA}")
    if lengths is None and (alpha != 0.0 or out_lengths is not None):
        raise ValueError("a rank by length needs the lengths")
    if index < 0:
        raise ValueError("the kernels need a CUDA device")
    code = _fn("bl_beam_select")(_SELECT.pack(logits.data_ptr(), max(logits.stride(0), V), *at, raw_stream(index), V, G, B, max(eos, -1),
                                              scratch.chunks, alpha))
    if code:
        check(code, "bl_beam_select")


def beam_reorder(k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, table_out: torch.Tensor, slots: torch.Tensor,
                 parent: torch.Tensor, held: torch.Tensor, fault: Optional[torch.Tensor] = None) -> None:
    """Cached states behind a choice: the beam in place i of a search (slot ``slots[g, i]``) continues the history of
    ``parent[g, i]``, of which ``held[g]`` positions are cached.

    ``k``, ``v``: the pools of all layers, [layers, pages, heads, 64, row] of any type (a latent cache has a ``v`` without
    values).  ``table_out``, another table than ``table``, gets the rows of these slots: full pages are the parent's, pages behind the
    one being filled stay the slot's.  In the page being filled a parent's first child goes on; each further child takes
    over the page of a beam that has none and a copy of the positions in it.  The pages from the one being filled on must belong
    to one slot each.  A search whose parents, slots or positions are out of range stays as it is and raises ``fault``;
    so does a child whose page being filled, its parent's or the one it takes over, is none of the pools'."""
    G, B = parent.shape
    index = k.get_device()
    at = (_same("slots", slots, torch.int32, G * B, index), _same("parent", parent, torch.int32, G * B, index),
          _same("held", held, torch.int32, G, index), 0 if fault is None else fault_ptr(fault, index))
    shape, v_shape, tables = k.shape, v.shape, table.shape
    if len(shape) != 5 or len(v_shape) != 5 or shape[:4] != v_shape[:4] or shape[3] != PAGE or not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError(f"pools: contiguous [layers, pages, heads, {PAGE}, row], alike but for the row")
    for t in (table, table_out):
        if t.dtype is not torch.int32 or len(tables) != 2 or t.shape != tables or not t.is_contiguous() or t.get_device() != index:
            raise ValueError("tables: contiguous int32 [slots, pages]")
    if table.data_ptr() == table_out.data_ptr():
        raise ValueError("the new table is written while the old one is read: another tensor")
    if B > MAX_BEAMS:
        raise ValueError(f"at most {MAX_BEAMS} beams a search")
    if index < 0 or v.get_device() != index:
        raise ValueError("the kernels need the pools on one CUDA device")
    code = _fn("bl_beam_reorder")(_REORDER.pack(k.data_ptr(), v.data_ptr(), shape[4] * k.element_size(), v_shape[4] * v.element_size(),
                                                table.data_ptr(), table_out.data_ptr(), *at, raw_stream(index), shape[0], shape[1],
                                                shape[2], tables[0], tables[1], G, B))
    if code:
        check(code, "bl_beam_reorder")


def beam_advance(tokens, row_pos, row_seq, held, hist, count, slots, parent, token, done, scores, G: int, B: int) -> None:
    """The rows of the next pass out of a choice: tokens, positions one further, sequences (-1 for finished and missing beams);
    ``held`` [G] one more; ``hist`` int32 [cap, 2, G * B] takes the parents and tokens of step ``count``."""
    index, n, i32 = tokens.get_device(), G * B, torch.int32
    if G < 1 or B < 1 or n > 65535:
        raise ValueError("1 to 65,535 beams in all")
    for name, t in (("tokens", tokens), ("row_pos", row_pos), ("row_seq", row_seq)):
        if t.dtype is not i32 or t.dim() != 1 or t.numel() < n or not t.is_contiguous() or t.get_device() != index:
            raise ValueError(f"{name}: contiguous int32, {n} rows at least, on one device")
    if hist.dim() != 3 or tuple(hist.shape[1:]) != (2, n):
        raise ValueError(f"hist: int32 [steps, 2, {n}]")
    _same("hist", hist, i32, hist.shape[0] * 2 * n, index)
    for name, t, size in (("held", held, G), ("count", count, 1), ("slots", slots, n), ("parent", parent, n), ("token", token, n),
                          ("done", done, n)):
        _same(name, t, i32, size, index)
    _same("scores", scores, torch.float32, n, index)
    if index < 0:
        raise ValueError("the kernels need a CUDA device")
    check(cuda().bl_beam_advance(p(tokens), p(row_pos), p(row_seq), p(held), p(hist), I(hist.shape[0]), p(count), p(slots), p(parent),
                                 p(token), p(done), p(scores), I(G), I(B), ctypes.c_void_p(raw_stream(index))), "bl_beam_advance")
