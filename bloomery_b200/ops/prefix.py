"""Decode attention of rows that share a prefix (``csrc/prefix_attn.cu``): the shared keys are read once for up to 256 (row, query
head) pairs of a key head.

A group is a run of consecutive rows of a pass whose sequences hold the same first positions in the same pages (beams of a
prompt, answers to one question, chats behind one system prompt: :meth:`KvPool.share_prefix` maps such pages).  Behind the
shared pages every row has keys of its own.  ``BatchDecode.prefix`` takes a plan for its passes; beam search sets one.

Queries, probabilities and expanded q8_0 rows are held in the 11 bits of f16, which the bf16 output hardly shows at scores of a few
nats and by some percent where scores are in the hundreds; ``flash_decode_bf16`` keeps 22 bits or more.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Sequence

import torch

from ..runtime.kv import PAGE
from ._lib import check, cuda, fault_ptr, raw_stream
from .decode import sm_count

_entry = None
_CALL = struct.Struct("11P12i")                       # PrefixCall in the source


class PrefixPlan:
    """The groups of a pass with the scratch of its launches: rows of each group (consecutive, in order) and positions that
    each group shares, whole pages.  A row that shares nothing is a group with prefix 0.  Lengths behind the prefix are read
    from ``row_pos`` by every call, so a plan, and a captured graph, serve for as long as the groups stay; the calls that use
    one plan follow each other on one stream."""

    def __init__(self, group_rows: Sequence[int], prefix_len: Sequence[int], n_q: int, n_kv: int, head: int, device):
        if not group_rows or any(r < 1 for r in group_rows):
            raise ValueError("one group at least, and one row in each")
        if head not in (64, 128):
            raise ValueError(f"heads of 64 or 128 values, not {head}")
        if n_kv < 1 or n_q < 1 or n_q % n_kv or n_q // n_kv > 16:
            raise ValueError(f"{n_q} query heads over {n_kv} key heads: 1 to 16 each")
        self.n_q, self.n_kv, self.head = n_q, n_kv, head
        self.group_rows = list(group_rows)
        self.rows = sum(group_rows)
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.index = self.device.index if self.device.type == "cuda" else -1      # as Tensor.get_device() says it
        self.q_shape, self.out_shape = (sum(group_rows), n_q, head), (sum(group_rows), n_q * head)
        if self.rows > 512:
            raise ValueError("at most 512 rows")
        self.max_pages = 1 << 24                          # of the narrowest table that a call of the plan came with
        rows = self._meta(prefix_len)
        self.n_units, self.unit_rows = len(rows) - self.rows, max(u[1] for u in rows[self.rows:])
        self.meta = torch.tensor(rows, dtype=torch.int32).to(self.device)
        self.n_cta = min(160, sm_count(self.device)) if self.device.type == "cuda" else 1
        fn = cuda().bl_prefix_work_bytes
        fn.restype = ctypes.c_long
        self.work = torch.empty(fn(head, n_q, n_kv, self.n_units, self.unit_rows, self.n_cta), dtype=torch.uint8, device=self.device)
        self.meta_ptr, self.work_ptr = self.meta.data_ptr(), self.work.data_ptr()

    def _meta(self, prefix_len: Sequence[int]):
        if len(prefix_len) != len(self.group_rows):
            raise ValueError("a prefix length for every group")
        if any(n < 0 or n % PAGE for n in prefix_len):
            raise ValueError(f"shared positions are whole pages of {PAGE}")
        if max(prefix_len) > self.max_pages * PAGE:
            raise ValueError(f"the prefix is longer than a table row of {self.max_pages} pages")
        self.prefix_len, self.max_prefix = list(prefix_len), max(prefix_len)
        # units: rows of a group that read all of their keys together, as many as two tiles of 128 (row, head) pairs of a key
        # head hold
        G = self.n_q // self.n_kv
        per = 128 // G
        rows, units, first = [], [], 0
        for n, p in zip(self.group_rows, prefix_len):
            rows += [(first, n, p, len(units) + i // (2 * per), i % (2 * per) // per * 128 + i % per * G) for i in range(n)]
            units += [(first + i, min(2 * per, n - i), p, first, n) for i in range(0, n, 2 * per)]
            first += n
        return rows + units

    def set_prefix(self, prefix_len: Sequence[int]) -> None:
        """Other shared positions for the same groups, within the table rows that the plan was called with; graphs captured with
        the plan take them up."""
        self.meta.copy_(torch.tensor(self._meta(prefix_len), dtype=torch.int32))


def prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, row_pos: torch.Tensor, row_seq: torch.Tensor,
                     block_table: torch.Tensor, plan: PrefixPlan, out: torch.Tensor, fault: Optional[torch.Tensor] = None,
                     layer: int = 0) -> None:
    """``out`` bf16 [M, n_q * head] = attention of ``q`` fp32 [M, n_q, head] (scaled as the softmax wants it) over keys
    0 .. row_pos of each row's sequence ``row_seq`` in the paged caches of one layer, f16 [pages, n_kv, 64, head] or q8_0 rows as
    uint8.  The first positions of a row come from the pages of its group's first live row.  Rows with a negative sequence get
    zeros; a row without keys, past its table or with a page that the pool does not have gets NaN and raises ``fault``."""
    global _entry
    rows, n_kv, head = plan.rows, plan.n_kv, plan.head
    if q.dtype is not torch.float32 or q.shape != plan.q_shape or not q.is_contiguous():
        raise ValueError(f"q: contiguous fp32 {list(plan.q_shape)}")
    q8 = k_cache.dtype is torch.uint8
    shape = k_cache.shape
    width = head // 32 * 34 if q8 else head
    if shape != v_cache.shape or len(shape) != 4 or shape[1] != n_kv or shape[2] != PAGE or shape[3] != width or \
            (not q8 and k_cache.dtype is not torch.float16) or v_cache.dtype is not k_cache.dtype or \
            not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError(f"caches: contiguous [pages, {n_kv}, {PAGE}, {width}], both f16 or both q8_0 bytes")
    if out.dtype is not torch.bfloat16 or out.shape != plan.out_shape or not out.is_contiguous():
        raise ValueError(f"out: contiguous bf16 {list(plan.out_shape)}")
    i32 = torch.int32
    if row_pos.dtype is not i32 or row_pos.numel() < rows or not row_pos.is_contiguous() or \
            row_seq.dtype is not i32 or row_seq.numel() < rows or not row_seq.is_contiguous():
        raise ValueError(f"row_pos and row_seq: int32, {rows} rows")
    table = block_table.shape
    if block_table.dtype is not i32 or len(table) != 2 or not block_table.is_contiguous():
        raise ValueError("block_table: contiguous int32 [slots, pages]")
    if plan.max_prefix > table[1] * PAGE:
        raise ValueError("the prefix is longer than a table row")
    if table[1] < plan.max_pages:
        plan.max_pages = table[1]                        # a graph captured with this call goes on with this table
    index = plan.index
    if not (index == q.get_device() == k_cache.get_device() == v_cache.get_device() == row_pos.get_device() == row_seq.get_device()
            == block_table.get_device() == out.get_device()):
        raise ValueError("the tensors are on the plan's device")
    fault_at = 0 if fault is None else fault_ptr(fault, index)
    if index < 0:
        raise ValueError("the kernels need a CUDA device")
    if _entry is None:
        _entry = cuda().bl_prefix_attention
        _entry.argtypes = [ctypes.c_char_p]
    code = _entry(_CALL.pack(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), row_pos.data_ptr(), row_seq.data_ptr(),
                             block_table.data_ptr(), plan.meta_ptr, plan.work_ptr, out.data_ptr(),
                             fault_at, raw_stream(index), table[0], table[1], shape[0], head,
                             plan.n_q, n_kv, rows, plan.n_units, plan.unit_rows, q8, plan.n_cta, layer))
    if code:
        check(code, "bl_prefix_attention")
