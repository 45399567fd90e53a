"""NVFP4 activations and their products with NVFP4 weights (``csrc/fp4_rows.cu``, ``csrc/fp4_gemm.cu``, ``csrc/fp4_moe.cu``).

A row of K values is K / 2 bytes of E2M1 codes, K / 16 E4M3 scales and one fp32 scale, padded to 16 bytes: the layout of resident
NVFP4 weights.  :func:`fp4_rows` makes such rows of activations, :func:`fp4_gemm` multiplies them with NVFP4 weights on the four-bit
tensor cores, :func:`fp4_moe` runs the routed experts of a few tokens in two launches.  ``BatchDecode`` and ``GemmPrefill`` take them
for NVFP4 weights where ``BLOOMERY_FP4_NATIVE`` is on.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional

import torch

from ..formats.resident import resident_row_bytes
from ._lib import check, cuda, fault_ptr, raw_stream
from .decode import QWeight, sm_count
from .gemm import TileTable

_ROWS, _GEMM, _MOE = struct.Struct("6P2ld4i"), struct.Struct("12P3l8i"), struct.Struct("13P3ld8i")      # Fp4RowsCall, Fp4GemmCall, Fp4MoeCall
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_K = 32768                                             # values of a row that fp4_rows holds in registers
_entries: dict = {}
_processors: dict = {}


def _fn(name):
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(cuda(), name)
        fn.argtypes = [ctypes.c_char_p]
    return fn


def _sms(index: int) -> int:
    n = _processors.get(index)
    if n is None:
        n = _processors[index] = sm_count(torch.device("cuda", index))
    return n


class RowsAsWeight(QWeight):
    """Rows that a launch in flight may still be writing, where weights are there before: a product waits before it reads them."""


class Fp4Rows:
    """Buffer of ``rows`` NVFP4 rows of ``k`` values."""

    def __init__(self, rows: int, k: int, device):
        if rows < 1 or k < 64 or k % 64 or k > MAX_K:
            raise ValueError(f"rows of 64 to {MAX_K} values, a multiple of 64")
        self.rows, self.k = rows, k
        self.data = torch.zeros(rows, resident_row_bytes("NVFP4", k), dtype=torch.uint8, device=device)
        self.ptr, self.index = self.data.data_ptr(), self.data.get_device()

    @property
    def weight(self) -> QWeight:
        """The rows as a resident NVFP4 matrix (what expands or dots one takes them too)."""
        return RowsAsWeight(self.data, "NVFP4", self.k)


def fp4_tile_rows(rows: int, groups: int = 1, gated: bool = False) -> int:
    """Rows of a tile of :func:`fp4_gemm` for ``rows`` rows dealt to ``groups`` matrices; ``gated``: with a second matrix.

    The smallest tile that holds a group's rows: a second tile of a group reads its weights again.  us, gate and up of 128 experts of
    768 x 2,048: 32 rows each in tiles of 32 / 64: 44.3 / 45.7, 33 rows 61.6 / 45.8; 64 rows in tiles of 64 / 128: 47.7 / 51.8, 65 rows 71.2 /
    55.5.  256 rows a tile halve what many rows ask of the weights and pad ragged groups more.  Tiles of 128 / 256: 4,096 x 8,192 for 512
    rows 19.3 / 16.2, for 4,096 rows 119 / 101, but for 256 rows 11.1 / 15.4; 16 matrices of 512 x 512 with 256 rows each 6.2 / 8.1, with 1,024
    11.4 / 10.8, with 1,100 11.5 / 14.1, with 1,500 15.4 / 14.2; eight of 4,096 x 4,096 with 512 rows each 63.9 / 61.4, with 1,100 149 / 137, with
    2,048 263 / 223.  (Two limits could lie closer: a single matrix gains from 256 rows a tile past some 300 rows, wide groups past 128.)"""
    per = -(-rows // groups)
    return 32 if per <= 32 else 64 if per <= 64 else 128 if per <= (128 if groups == 1 else 1024) or gated else 256


def fp4_tiles(rows: int, device) -> TileTable:
    """The table of a product of ``rows`` rows with one matrix."""
    if rows == 0:
        return TileTable(0, 1, device, 32)
    return TileTable.dense(rows, device, fp4_tile_rows(rows), host=True)


def fp4_rows(x: torch.Tensor, out: Fp4Rows, *, gain: Optional[torch.Tensor] = None, eps: float = 0.0,
             tensor_scale: Optional[torch.Tensor] = None, pos_of: Optional[torch.Tensor] = None) -> None:
    """NVFP4 rows of ``x`` [M, k] (bf16, f16 or fp32; rows may be strided) in the first M rows of ``out``.

    A row's scale takes its largest magnitude to 6 x 448, or is ``tensor_scale``, one fp32 on the device (values too large for it
    saturate; 2^-100 where it is below that, and with one that is no finite number all rows' products are NaN); a
    block's scale takes its own to 6; scales and codes are the nearest, ties go to the even code.  A row with a NaN or an
    infinity becomes one whose products are all NaN.  ``gain`` fp32 [k] (fp32 rows): RMSNorm first, with 1 / sqrt(mean square + eps)
    in fp32 (rows that are all zeros, or too small for that, need an ``eps``).  ``pos_of`` int32 [M * copies]:
    row m goes to the rows ``pos_of[m * copies + j]`` of ``out`` (none where that is negative or past the end; no place twice), as
    ``moe_plan`` deals the slots of M tokens."""
    kind = _TYPES.get(x.dtype)
    index = out.index
    if kind is None or x.dim() != 2 or x.shape[1] != out.k or x.stride(1) != 1:
        raise ValueError(f"x: bf16, f16 or fp32 [rows, {out.k}], values next to each other")
    M = x.shape[0]
    copies, at = 1, 0
    if pos_of is not None:
        copies, rest = divmod(pos_of.numel(), M) if M else (1, pos_of.numel())
        if pos_of.dtype is not torch.int32 or not pos_of.is_contiguous() or rest or copies < 1 or pos_of.get_device() != index:
            raise ValueError("pos_of: contiguous int32, as many places for every row, on the device of the rest")
        at = pos_of.data_ptr()
    elif M > out.rows:
        raise ValueError(f"{M} rows into {out.rows}")
    gain_at = scale_at = 0
    if gain is not None:
        if kind != 2 or gain.dtype is not torch.float32 or gain.numel() != out.k or not gain.is_contiguous() or gain.get_device() != index:
            raise ValueError(f"gain: contiguous fp32 [{out.k}] beside fp32 rows, on the device of the rest")
        gain_at = gain.data_ptr()
    if tensor_scale is not None:
        if tensor_scale.dtype is not torch.float32 or tensor_scale.numel() != 1 or tensor_scale.get_device() != index:
            raise ValueError("tensor_scale: one fp32 on the device of the rest")
        scale_at = tensor_scale.data_ptr()
    if x.get_device() != index:
        raise ValueError("x: on another device than the rows")
    if index < 0:
        raise ValueError("the kernels need a CUDA device")
    if M == 0:
        return
    ldx = x.stride(0) if M > 1 else out.k
    code = _fn("bl_fp4_rows")(_ROWS.pack(x.data_ptr(), gain_at, scale_at, at, out.ptr, raw_stream(index), ldx, out.rows, eps, kind, M, out.k,
                                         copies))
    if code:
        check(code, "bl_fp4_rows")


def fp4_supports(w: QWeight) -> bool:
    """Whether the products here take a matrix or stack: NVFP4 whose block scales are without a sign, as checkpoints have them (looks at
    all of them and waits for the answer: once, when a model is set up)."""
    if w.qtype != "NVFP4" or w.k % 64 or w.k > MAX_K or not _rows_of(w.data, w.k):
        return False
    return not bool((w.data[..., w.k // 2:w.k // 2 + w.k // 16] >= 0x80).any())


class Fp4Work:
    """What a program keeps for the dense products of one stream.  Products with few tiles take narrower ones instead of sharing their depth, so
    there is nothing in it yet; it is part of the call so that a program that keeps one per stream stays as it is."""

    def __init__(self, device):
        self.device = device


def _rows_of(data: torch.Tensor, k: int) -> bool:
    """Whether these are one matrix, or a stack, of NVFP4 rows of k values."""
    shape = data.shape
    return 2 <= len(shape) <= 3 and shape[-1] == (k // 2 + k // 16 + 19) // 16 * 16 and 0 not in shape and data.dtype is torch.uint8


def _matrix(name: str, w: QWeight, k: int, index: int) -> int:
    data = w.data
    if w.qtype != "NVFP4" or w.k != k or not _rows_of(data, k) or not data.is_contiguous() or data.get_device() != index:
        raise ValueError(f"{name}: contiguous NVFP4 rows of {k} values on the device of the rest")
    return data.data_ptr()


def _of_rows(name: str, t: torch.Tensor, dtype, rows: int, index: int) -> int:
    if t.dtype is not dtype or t.numel() < rows or not t.is_contiguous() or t.get_device() != index:
        raise ValueError(f"{name}: contiguous {dtype}, {rows} values at least, on the device of the rest")
    return t.data_ptr()


def fp4_gemm(X: Fp4Rows, W: QWeight, tiles: TileTable, *, out_f32: Optional[torch.Tensor] = None,
             out_bf16: Optional[torch.Tensor] = None, W2: Optional[QWeight] = None, dst_row=None, row_scale=None, resid=None,
             status: Optional[torch.Tensor] = None, work: Optional[Fp4Work] = None) -> None:
    """C = X @ W[g].T per token tile, codes by codes on tcgen05 ``kind::mxf4nvf4`` with fp32 sums: ``X`` NVFP4 rows, W (and W2)
    resident NVFP4 matrices [N, bytes] or stacks [G, N, bytes]; tiles of 32, 64 or 128 rows, without W2 of 256 too
    (:func:`fp4_tile_rows`; :func:`fp4_tiles` for one matrix).  With W2 the output is silu(X W^T) * (X W2^T).  Epilogue options as :func:`gemm.qgemm`; a row
    that ``dst_row`` sends below 0 or past the output goes nowhere, and no two go to one place.  Block scales are
    taken without their sign, which no checkpoint sets (:func:`fp4_supports`)."""
    index, k = X.index, X.k
    wp = _matrix("W", W, k, index)
    shape = W.data.shape
    G, N = (shape[0] if len(shape) == 3 else 1), shape[-2]
    w2p = 0
    if W2 is not None:
        w2p = _matrix("W2", W2, k, index)
        if W2.data.shape != shape:
            raise ValueError("W and W2 are alike")
    f32 = out_f32 is not None
    out = out_f32 if f32 else out_bf16
    if (out_f32 is None) == (out_bf16 is None) or out.dtype is not (torch.float32 if f32 else torch.bfloat16) or out.dim() != 2 or \
            out.shape[1] != N or (out.stride(1) != 1 and N > 1) or out.get_device() != index:
        raise ValueError(f"one output, fp32 or bf16 [rows, {N}], on the device of the rest")
    rp = ldr = 0
    if resid is not None:
        if resid.dtype is not torch.float32 or resid.shape != out.shape or (resid.stride(1) != 1 and N > 1) or resid.get_device() != index:
            raise ValueError("resid: fp32, shaped like the output")
        rp, ldr = resid.data_ptr(), resid.stride(0)
    rows = tiles.rows
    if out.shape[0] > 1 and out.stride(0) < N:
        raise ValueError("the output's rows lie over each other")
    if tiles.n_groups > G or tiles.tile_rows not in (32, 64, 128, 256) or (w2p and tiles.tile_rows == 256) or tiles.index != index:
        raise ValueError(f"tiles: of 32, 64 or 128 rows (256 without W2) over at most {G} matrices, on the device of the rest")
    if rows > X.rows or (dst_row is None and rows > out.shape[0]):
        raise ValueError(f"the tiles reach {rows} rows")
    dp = _of_rows("dst_row", dst_row, torch.int32, rows, index) if dst_row is not None else 0
    fp = _of_rows("row_scale", row_scale, torch.float32, rows, index) if row_scale is not None else 0
    sp = fault_ptr(status, index) if status is not None else 0
    if index < 0:
        raise ValueError("the kernels need a CUDA device")
    if out.shape[0] == 0:
        return                                   # no row of it to write
    code = _fn("bl_fp4_gemm")(_GEMM.pack(
        X.ptr, wp, w2p, tiles.mtiles_ptr, tiles.n_mtiles_ptr, out.data_ptr() if f32 else 0, 0 if f32 else out.data_ptr(),
        dp, fp, rp, sp, raw_stream(index), X.rows, out.stride(0), ldr, G, N, k,
        tiles.fixed or tiles.max_mtiles, tiles.tile_rows, _sms(index),
        tiles.fixed != 0 and type(W) is QWeight and (W2 is None or type(W2) is QWeight), min(out.shape[0], 2 ** 31 - 1)))
    if code:
        check(code, "bl_fp4_gemm")


MOE_TOKENS, MOE_USED, MOE_EXPERTS, MOE_WIDTH = 64, 16, 512, 8192


class Fp4MoeWork:
    """Scratch of :func:`fp4_moe` for up to ``rows`` tokens of ``used`` experts each, of ``n_expert``, ``hidden`` and ``inter`` values wide:
    one per stream that runs them.  After a call that raised its status word make another."""

    def __init__(self, rows: int, used: int, hidden: int, inter: int, n_expert: int, device):
        if not 1 <= rows <= MOE_TOKENS or not 1 <= used <= MOE_USED or not 1 <= n_expert <= MOE_EXPERTS:
            raise ValueError(f"1 to {MOE_TOKENS} tokens, 1 to {MOE_USED} of up to {MOE_EXPERTS} experts each")
        if any(n < 64 or n % 64 or n > MOE_WIDTH for n in (hidden, inter)):
            raise ValueError(f"widths of 64 to {MOE_WIDTH}, multiples of 64")
        self.rows, self.used, self.hidden, self.inter, self.n_expert = rows, used, hidden, inter, n_expert
        size = cuda().bl_fp4_moe_work_bytes
        size.restype = ctypes.c_long
        self.data = torch.zeros(size(rows, used, n_expert, hidden, inter, sm_count(device) if torch.device(device).type == "cuda" else 1), dtype=torch.uint8, device=device)
        self.ptr, self.index = self.data.data_ptr(), self.data.get_device()


def fp4_moe(x: torch.Tensor, ids: torch.Tensor, wts: torch.Tensor, gate: QWeight, up: QWeight, down: QWeight, work: Fp4MoeWork, *,
            out_f32: Optional[torch.Tensor] = None, out_bf16: Optional[torch.Tensor] = None, gain: Optional[torch.Tensor] = None,
            eps: float = 0.0, resid: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> None:
    """out[t] = resid[t] + sum_j wts[t, j] down_e(silu(gate_e(x_t)) * up_e(x_t)), e = ids[t, j], for 1 to 64 tokens in two launches:
    tokens ``x`` [T, hidden] (fp32 or bf16; ``gain`` fp32: RMSNorm of fp32 rows first) and the products in between go through NVFP4 rows
    as :func:`fp4_rows` makes them.  ``ids`` int32 and ``wts`` fp32 [T, used]; a slot whose id is not in 0 .. experts - 1 is another
    tier's and adds nothing.  ``out`` may be ``resid`` and, in fp32, ``x``."""
    T = x.shape[0] if x.dim() == 2 else 0
    kind, index = _TYPES.get(x.dtype), work.index
    H, I_, E, k = work.hidden, work.inter, work.n_expert, work.used
    if kind not in (0, 2) or not 1 <= T <= work.rows or x.shape[1] != H or x.stride(1) != 1 or x.get_device() != index:
        raise ValueError(f"x: fp32 or bf16 [1 to {work.rows}, {H}], values next to each other, on the scratch's device")
    if ids.dtype is not torch.int32 or ids.numel() != T * k or not ids.is_contiguous() or ids.get_device() != index:
        raise ValueError(f"ids: contiguous int32 [{T}, {k}] on the scratch's device")
    if wts.dtype is not torch.float32 or wts.numel() != T * k or not wts.is_contiguous() or wts.get_device() != index:
        raise ValueError(f"wts: contiguous fp32 [{T}, {k}] on the scratch's device")
    at = [_matrix(n, w, d, index) for n, w, d in (("gate", gate, H), ("up", up, H), ("down", down, I_))]
    if gate.data.shape[:-1] != (E, I_) or up.data.shape[:-1] != (E, I_) or down.data.shape[:-1] != (E, H):
        raise ValueError(f"gate and up: stacks of {E} x {I_} rows, down of {E} x {H}")
    f32 = out_f32 is not None
    out = out_f32 if f32 else out_bf16
    if (out_f32 is None) == (out_bf16 is None) or out.dtype is not (torch.float32 if f32 else torch.bfloat16) or out.shape != (T, H) or \
            out.stride(1) != 1 or out.get_device() != index:
        raise ValueError(f"one output, fp32 or bf16 [{T}, {H}], on the scratch's device")
    rp = ldr = gain_at = 0
    if resid is not None:
        if resid.dtype is not torch.float32 or resid.shape != out.shape or resid.stride(1) != 1 or resid.get_device() != index:
            raise ValueError("resid: fp32, shaped like the output")
        rp, ldr = resid.data_ptr(), resid.stride(0)
    if gain is not None:
        if kind != 2 or gain.dtype is not torch.float32 or gain.numel() != H or not gain.is_contiguous() or gain.get_device() != index:
            raise ValueError(f"gain: contiguous fp32 [{H}] beside fp32 rows")
        gain_at = gain.data_ptr()
    sp = fault_ptr(status, index) if status is not None else 0
    if T > 1 and (out.stride(0) < H or (resid is not None and resid.stride(0) < H)):
        raise ValueError("rows lie over each other")
    if index < 0:
        raise ValueError("the kernels need a CUDA device")
    ldx = x.stride(0) if T > 1 else H
    code = _fn("bl_fp4_moe")(_MOE.pack(x.data_ptr(), gain_at, ids.data_ptr(), wts.data_ptr(), *at, work.ptr, rp, out.data_ptr() if f32 else 0,
                                       0 if f32 else out.data_ptr(), sp, raw_stream(index), ldx, ldr,
                                       out.stride(0), eps, kind, T, k, E, H, I_, work.rows, _sms(index)))
    if code:
        check(code, "bl_fp4_moe")
