"""What the NVFP4 calls refuse, without a card: the entries of the library answer a code before they touch the device, the Python face raises
ValueError, and tensors of the CPU get as far as the last check."""
import ctypes

import pytest
import torch

from bloomery_b200.ops import fp4 as Q
from bloomery_b200.ops._lib import cuda
from bloomery_b200.ops.decode import QWeight
from bloomery_b200.ops.gemm import TileTable

SHAPE, TYPE, ALIGN, LIMIT = -2, -3, -4, -5
A = 0x10000          # an aligned address that nothing reads


def call(name, packed):
    fn = getattr(cuda(), name)
    return fn(packed)


def rows(x=A, gain=0, tensor=0, pos=0, out=A, ldx=1024, rows_out=8, eps=0.0, kind=0, M=4, K=1024, copies=1):
    return call("bl_fp4_rows", Q._ROWS.pack(x, gain, tensor, pos, out, 0, ldx, rows_out, eps, kind, M, K, copies))


def test_rows_are_refused_before_they_are_launched():
    assert rows(K=1000) == SHAPE and rows(K=0) == SHAPE and rows(M=0) == SHAPE and rows(copies=0) == SHAPE
    assert rows(K=32768 + 64, ldx=40000) == LIMIT
    assert rows(kind=3) == TYPE and rows(kind=-1) == TYPE
    assert rows(gain=A, kind=0) == TYPE                           # the norm reads fp32 rows
    assert rows(x=A + 8) == ALIGN and rows(out=A + 4) == ALIGN and rows(ldx=1028) == ALIGN and rows(ldx=512) == ALIGN
    assert rows(gain=A + 4, kind=2) == ALIGN
    assert rows(rows_out=3) == SHAPE                              # four rows into three, without places
    assert rows(copies=2) == SHAPE


def gemm(x=A, w=A, w2=0, f32=A, bf16=0, rows_x=64, ldc=256, groups=1, N=256, K=1024, tiles=4, tile_rows=32, sms=148):
    return call("bl_fp4_gemm", Q._GEMM.pack(x, w, w2, A, A, f32, bf16, 0, 0, 0, 0, 0, rows_x, ldc, 0, groups, N, K, tiles, tile_rows, sms, 0, 0))


def test_products_are_refused_before_they_are_launched():
    assert gemm(K=1000) == SHAPE and gemm(K=0) == SHAPE and gemm(N=0) == SHAPE and gemm(rows_x=0) == SHAPE and gemm(tiles=0) == SHAPE
    assert gemm(tile_rows=48) == SHAPE and gemm(tile_rows=256, w2=A) == SHAPE and gemm(groups=0) == SHAPE
    assert gemm(f32=A, bf16=A) == SHAPE and gemm(f32=0) == SHAPE and gemm(ldc=1 << 30) == SHAPE
    assert gemm(x=A + 8) == ALIGN and gemm(w=A + 4) == ALIGN and gemm(w2=A + 4) == ALIGN
    assert gemm(N=1 << 30, tiles=1 << 10) == LIMIT


def moe(x=A, gain=0, work=A, f32=A, bf16=0, ldx=512, kind=2, T=4, k=4, E=16, H=512, I=256, cap=8, sms=148, wd=A):
    return call("bl_fp4_moe", Q._MOE.pack(x, gain, A, A, A, A, wd, work, 0, f32, bf16, 0, 0, ldx, 0, H, 1e-6, kind, T, k, E, H, I, cap, sms))


def test_experts_are_refused_before_they_are_launched():
    assert moe(T=0) == SHAPE and moe(T=9) == SHAPE and moe(k=0) == SHAPE and moe(E=0) == SHAPE
    assert moe(H=500, ldx=512) == SHAPE and moe(I=100) == SHAPE
    assert moe(T=65, cap=65) == LIMIT and moe(k=17) == LIMIT and moe(E=513) == LIMIT and moe(H=8256, ldx=8256) == LIMIT and moe(I=8256) == LIMIT
    assert moe(kind=1) == TYPE and moe(kind=0, gain=A) == TYPE
    assert moe(x=A + 4) == ALIGN and moe(work=A + 16) == ALIGN and moe(wd=A + 8) == ALIGN and moe(ldx=510) == ALIGN
    assert moe(bf16=A) == SHAPE and moe(f32=0) == SHAPE


def test_scratch_grows_with_what_it_holds():
    size = cuda().bl_fp4_moe_work_bytes
    size.restype = ctypes.c_long
    base = size(8, 8, 128, 2048, 768, 148)
    assert base < size(16, 8, 128, 2048, 768, 148) < size(64, 8, 128, 2048, 768, 148)
    assert base < size(8, 8, 512, 2048, 768, 148) and base < size(8, 8, 128, 4096, 768, 148) and base < size(8, 8, 128, 2048, 2048, 148)


def w(N, K, groups=0, qtype="NVFP4"):
    from bloomery_b200.formats.resident import resident_row_bytes
    shape = ([groups] if groups else []) + [N, resident_row_bytes("NVFP4", K)]
    return QWeight(torch.zeros(*shape, dtype=torch.uint8), qtype, K)


@pytest.mark.parametrize("rows_,k", [(0, 64), (1, 0), (1, 96), (1, 32), (4, 32768 + 64)])
def test_buffers_of_rows(rows_, k):
    with pytest.raises(ValueError):
        Q.Fp4Rows(rows_, k, "cpu")


def test_buffers_are_nvfp4_matrices():
    r = Q.Fp4Rows(3, 192, "cpu")
    assert r.weight.qtype == "NVFP4" and r.weight.k == 192 and r.weight.rows == 3 and r.data.shape[1] % 16 == 0


BAD_ROWS = {
    "type": dict(x=torch.zeros(2, 128, dtype=torch.float64)),
    "width": dict(x=torch.zeros(2, 64)),
    "one dimension": dict(x=torch.zeros(128)),
    "columns apart": dict(x=torch.zeros(2, 256)[:, ::2]),
    "too many rows": dict(x=torch.zeros(5, 128)),
    "gain beside 16 bits": dict(x=torch.zeros(2, 128, dtype=torch.bfloat16), gain=torch.zeros(128)),
    "gain's width": dict(gain=torch.zeros(64)),
    "gain's type": dict(gain=torch.zeros(128, dtype=torch.bfloat16)),
    "scale": dict(tensor_scale=torch.zeros(2)),
    "scale's type": dict(tensor_scale=torch.zeros(1, dtype=torch.float64)),
    "places' type": dict(pos_of=torch.zeros(4, dtype=torch.int64)),
    "places of half a row": dict(pos_of=torch.zeros(3, dtype=torch.int32)),
    "no place": dict(pos_of=torch.zeros(0, dtype=torch.int32)),
}


@pytest.mark.parametrize("what", sorted(BAD_ROWS))
def test_rows_that_are_none(what):
    kw = dict(BAD_ROWS[what])
    x = kw.pop("x", torch.zeros(2, 128))
    with pytest.raises(ValueError) as e:
        Q.fp4_rows(x, Q.Fp4Rows(4, 128, "cpu"), **kw)
    assert "CUDA" not in str(e.value)


def test_the_last_check_is_the_device():
    r, t = Q.Fp4Rows(4, 128, "cpu"), Q.fp4_tiles(4, "cpu")
    with pytest.raises(ValueError, match="CUDA"):
        Q.fp4_rows(torch.zeros(2, 128), r)
    with pytest.raises(ValueError, match="CUDA"):
        Q.fp4_gemm(r, w(16, 128), t, out_f32=torch.zeros(4, 16))
    with pytest.raises(ValueError, match="CUDA"):
        Q.fp4_moe(torch.zeros(2, 128), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2), w(64, 128, 3), w(64, 128, 3), w(128, 64, 3),
                  Q.Fp4MoeWork(2, 2, 128, 64, 3, "cpu"), out_f32=torch.zeros(2, 128))


BAD_GEMM = {
    "weights' type": dict(W=w(16, 128, qtype="Q8_0")),
    "depth": dict(W=w(16, 192)),
    "second matrix": dict(W2=w(32, 128)),
    "no output": dict(out_f32=None),
    "two outputs": dict(out_bf16=torch.zeros(4, 16, dtype=torch.bfloat16)),
    "output's type": dict(out_f32=torch.zeros(4, 16, dtype=torch.float64)),
    "output's width": dict(out_f32=torch.zeros(4, 17)),
    "output's rows": dict(out_f32=torch.zeros(3, 16)),
    "output over itself": dict(out_f32=torch.zeros(1, 16).expand(4, 16)),
    "columns apart": dict(out_f32=torch.zeros(4, 32)[:, ::2]),
    "residual": dict(resid=torch.zeros(3, 16)),
    "residual's type": dict(resid=torch.zeros(4, 16, dtype=torch.bfloat16)),
    "more rows than there are": dict(tiles=Q.fp4_tiles(5, "cpu"), out_f32=torch.zeros(5, 16)),
    "more matrices than there are": dict(tiles=TileTable(4, 2, "cpu", 32)),
    "tiles of 48": dict(tiles=TileTable(4, 1, "cpu", 48)),
    "wide tiles of pairs": dict(tiles=TileTable(4, 1, "cpu", 256), W2=w(16, 128)),
    "scatter's type": dict(dst_row=torch.zeros(4, dtype=torch.int64)),
    "scatter's length": dict(dst_row=torch.zeros(3, dtype=torch.int32)),
    "factors": dict(row_scale=torch.zeros(4, dtype=torch.float64)),
    "status": dict(status=torch.zeros(1)),
}


@pytest.mark.parametrize("what", sorted(BAD_GEMM))
def test_products_that_are_none(what):
    kw = dict(W=w(16, 128), tiles=Q.fp4_tiles(4, "cpu"), out_f32=torch.zeros(4, 16))
    kw.update(BAD_GEMM[what])
    with pytest.raises(ValueError) as e:
        Q.fp4_gemm(Q.Fp4Rows(4, 128, "cpu"), kw.pop("W"), kw.pop("tiles"), **kw)
    assert "CUDA" not in str(e.value)


BAD_MOE = {
    "no token": dict(x=torch.zeros(0, 128)),
    "more tokens than the scratch has": dict(x=torch.zeros(3, 128)),
    "width": dict(x=torch.zeros(2, 64)),
    "type": dict(x=torch.zeros(2, 128, dtype=torch.float16)),
    "ids' type": dict(ids=torch.zeros(2, 2, dtype=torch.int64)),
    "ids' number": dict(ids=torch.zeros(2, 3, dtype=torch.int32)),
    "weights of the router": dict(wts=torch.zeros(2, 2, dtype=torch.float16)),
    "gate": dict(gate=w(64, 128, 2)),
    "up": dict(up=w(32, 128, 3)),
    "down": dict(down=w(128, 128, 3)),
    "one matrix": dict(down=w(128, 64)),
    "two outputs": dict(out_bf16=torch.zeros(2, 128, dtype=torch.bfloat16)),
    "output's rows": dict(out_f32=torch.zeros(1, 128)),
    "output over itself": dict(out_f32=torch.zeros(1, 128).expand(2, 128)),
    "residual": dict(resid=torch.zeros(2, 64)),
    "gain beside 16 bits": dict(x=torch.zeros(2, 128, dtype=torch.bfloat16), gain=torch.zeros(128)),
    "gain": dict(gain=torch.zeros(64)),
    "status": dict(status=torch.zeros(1, dtype=torch.int64)),
}


@pytest.mark.parametrize("what", sorted(BAD_MOE))
def test_experts_that_are_none(what):
    kw = dict(x=torch.zeros(2, 128), ids=torch.zeros(2, 2, dtype=torch.int32), wts=torch.zeros(2, 2), gate=w(64, 128, 3), up=w(64, 128, 3),
              down=w(128, 64, 3), out_f32=torch.zeros(2, 128))
    kw.update(BAD_MOE[what])
    args = [kw.pop(n) for n in ("x", "ids", "wts", "gate", "up", "down")]
    with pytest.raises(ValueError) as e:
        Q.fp4_moe(*args, Q.Fp4MoeWork(2, 2, 128, 64, 3, "cpu"), **kw)
    assert "CUDA" not in str(e.value)


@pytest.mark.parametrize("what", [(0, 2, 128, 64, 3), (65, 2, 128, 64, 3), (2, 17, 128, 64, 3), (2, 2, 100, 64, 3), (2, 2, 128, 8256, 3), (2, 2, 128, 64, 513)])
def test_scratch_that_is_none(what):
    with pytest.raises(ValueError):
        Q.Fp4MoeWork(*what, "cpu")


def test_tiles_by_the_rows_they_hold():
    assert [Q.fp4_tile_rows(n) for n in (1, 32, 33, 64, 65, 128, 129, 5000)] == [32, 32, 64, 64, 128, 128, 256, 256]
    assert [Q.fp4_tile_rows(n, 8) for n in (8, 300, 512, 700, 8192, 9000)] == [32, 64, 64, 128, 128, 256]
    assert Q.fp4_tile_rows(9000, 8, gated=True) == 128 and Q.fp4_tile_rows(5000, gated=True) == 128
    t = Q.fp4_tiles(70, "cpu")
    assert t.fixed == 1 and t.tile_rows == 128 and t.rows == 70


def test_weights_with_signs_in_their_scales_are_not_taken():
    m = w(16, 128)
    assert Q.fp4_supports(m)
    m.data[3, 64 + 2] = 0x80
    assert not Q.fp4_supports(m)
    assert not Q.fp4_supports(w(16, 128, qtype="Q8_0"))


def test_the_lever_is_off_unless_it_is_set():
    from bloomery_b200.utils import levers
    assert levers.at_main({})["BLOOMERY_FP4_NATIVE"] is False
    assert levers.at_main({"BLOOMERY_FP4_NATIVE": "1"})["BLOOMERY_FP4_NATIVE"] is True
    levers.at_main()
