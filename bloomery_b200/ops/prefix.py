"""Decode attention of rows that share a prefix (``csrc/prefix_attn.cu``): the shared keys are read once for all rows.

A group is a run of consecutive rows of a pass whose sequences hold the same first positions in the same pages (beams of a
prompt, answers to one question, chats behind one system prompt: :meth:`KvPool.share_prefix` maps such pages).  Behind the
shared pages every row has keys of its own.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from ..runtime.kv import PAGE
from ._lib import check, cuda
from .decode import sm_count

_entry = None


def _fn():
    global _entry
    if _entry is None:
        fn = cuda().bl_prefix_attention
        P, I = ctypes.c_void_p, ctypes.c_int
        fn.argtypes = [P, P, P, P, P, P, I, I, I, I, I, I, I, P, I, P, I, P, I, P, I, P]
        _entry = fn
    return _entry


class PrefixPlan:
    """The groups of a pass with the scratch of its launches: rows of each group (consecutive, in order) and positions that
    each group shares, whole pages.  A row that shares nothing is a group with prefix 0.  Lengths behind the prefix are read
    from ``row_pos`` by every call, so a plan, and a captured graph, serve for as long as the groups stay; the calls that use
    one plan follow each other on one stream."""

    def __init__(self, group_rows: Sequence[int], prefix_len: Sequence[int], n_q: int, n_kv: int, head: int, device):
        if len(group_rows) != len(prefix_len) or not group_rows:
            raise ValueError("a prefix length for every group, and one group at least")
        if any(r < 1 for r in group_rows):
            raise ValueError("a group has one row at least")
        if any(n < 0 or n % PAGE for n in prefix_len):
            raise ValueError(f"shared positions are whole pages of {PAGE}")
        if head not in (64, 128):
            raise ValueError(f"heads of 64 or 128 values, not {head}")
        if n_kv < 1 or n_q < 1 or n_q % n_kv or n_q // n_kv > 16:
            raise ValueError(f"{n_q} query heads over {n_kv} key heads: 1 to 16 each")
        self.n_q, self.n_kv, self.head = n_q, n_kv, head
        self.group_rows, self.prefix_len = list(group_rows), list(prefix_len)
        self.rows = sum(group_rows)
        self.max_prefix = max(prefix_len)
        self.device = torch.device(device)
        if self.rows > 512:
            raise ValueError("at most 512 rows")
        # units: rows of a group that read all of their keys together, as many as two tiles of 128 (row, head) pairs of a key
        # head hold
        G = n_q // n_kv
        per = 128 // G
        rows, units, first = [], [], 0
        for n, p in zip(group_rows, prefix_len):
            rows += [(first, n, p, len(units) + i // (2 * per), i % (2 * per) // per * 128 + i % per * G) for i in range(n)]
            units += [(first + i, min(2 * per, n - i), p, first, n) for i in range(0, n, 2 * per)]
            first += n
        self.n_units = len(units)
        self.meta = torch.tensor(rows + units, dtype=torch.int32).to(self.device)
        self.n_cta = min(160, sm_count(self.device)) if self.device.type == "cuda" else 1
        fn = cuda().bl_prefix_work_bytes
        fn.restype = ctypes.c_long
        self.work = torch.empty(fn(head, n_kv, self.n_units, self.n_cta), dtype=torch.uint8, device=self.device)


def prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, row_pos: torch.Tensor, row_seq: torch.Tensor,
                     block_table: torch.Tensor, plan: PrefixPlan, out: torch.Tensor, fault: Optional[torch.Tensor] = None,
                     layer: int = 0) -> None:
    """``out`` bf16 [M, n_q * head] = attention of ``q`` fp32 [M, n_q, head] (scaled as the softmax wants it) over keys
    0 .. row_pos of each row's sequence ``row_seq`` in the paged caches of one layer, f16 [pages, n_kv, 64, head] or q8_0 rows as
    uint8.  The first positions of a row come from the pages of its group's first live row.  Rows with a negative sequence get
    zeros; a row without keys, past its table or with a page that the pool does not have gets NaN and raises ``fault``."""
    n_kv, head = plan.n_kv, plan.head
    if q.dtype != torch.float32 or not q.is_contiguous() or q.shape != (plan.rows, plan.n_q, head):
        raise ValueError(f"q: contiguous fp32 [{plan.rows}, {plan.n_q}, {head}]")
    q8 = k_cache.dtype == torch.uint8
    width = head // 32 * 34 if q8 else head
    for c in (k_cache, v_cache):
        if c.dtype != (torch.uint8 if q8 else torch.float16) or not c.is_contiguous() or c.dim() != 4 or c.shape[1:] != (n_kv, PAGE, width) \
                or c.shape[0] != k_cache.shape[0]:
            raise ValueError(f"caches: contiguous [pages, {n_kv}, {PAGE}, {width}], both f16 or both q8_0 bytes")
    if out.dtype != torch.bfloat16 or not out.is_contiguous() or out.shape != (plan.rows, plan.n_q * head):
        raise ValueError(f"out: contiguous bf16 [{plan.rows}, {plan.n_q * head}]")
    for t in (row_pos, row_seq):
        if t.dtype != torch.int32 or not t.is_contiguous() or t.numel() < plan.rows:
            raise ValueError(f"row_pos and row_seq: int32, {plan.rows} rows")
    if block_table.dtype != torch.int32 or not block_table.is_contiguous() or block_table.dim() != 2:
        raise ValueError("block_table: contiguous int32 [slots, pages]")
    if plan.max_prefix > block_table.shape[1] * PAGE:
        raise ValueError("the prefix is longer than a table row")
    rc = _fn()(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), row_pos.data_ptr(), row_seq.data_ptr(), block_table.data_ptr(),
               block_table.shape[0], block_table.shape[1], k_cache.shape[0], head, plan.n_q, n_kv, plan.rows, plan.meta.data_ptr(), plan.n_units, plan.work.data_ptr(),
               1 if q8 else 0, out.data_ptr(), plan.n_cta, fault.data_ptr() if fault is not None else None, layer,
               torch.cuda.current_stream(plan.device).cuda_stream)
    check(rc, "bl_prefix_attention")
