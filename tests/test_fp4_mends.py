"""What the NVFP4 calls took, or kept, wrongly once; without a card."""
import pytest
import torch

from bloomery_b200.ops import fp4 as Q
from bloomery_b200.ops.decode import QWeight
from test_fp4_contracts import w


@pytest.mark.parametrize("data", [torch.zeros(16, 48, dtype=torch.uint8), torch.zeros(16, 96, dtype=torch.uint8), torch.zeros(2, 2, 16, 80, dtype=torch.uint8),
                                  torch.zeros(80, dtype=torch.uint8), torch.zeros(16, 80, dtype=torch.int8), torch.zeros(0, 80, dtype=torch.uint8), torch.zeros((), dtype=torch.uint8)],
                         ids=["short rows", "long rows", "four dimensions", "one row", "signed", "no rows", "one byte"])
def test_weights_that_are_not_rows_of_their_width(data):
    """Rows of 128 values are 80 bytes: others would be read past their end."""
    bad, rows = QWeight(data, "NVFP4", 128), Q.Fp4Rows(4, 128, "cpu")
    for kw in (dict(W=bad), dict(W=w(16, 128), W2=bad)):
        with pytest.raises(ValueError, match="W2?: "):
            Q.fp4_gemm(rows, kw.pop("W"), Q.fp4_tiles(4, "cpu"), out_f32=torch.zeros(4, 16), **kw)
    assert not Q.fp4_supports(bad)


def test_stacks_that_are_not_rows_of_their_width():
    good = dict(gate=w(64, 128, 3), up=w(64, 128, 3), down=w(128, 64, 3))
    for name, k in (("gate", 128), ("up", 128), ("down", 64)):
        q = good[name]
        bad = QWeight(q.data[..., :-16].contiguous(), "NVFP4", k)
        with pytest.raises(ValueError, match=name + ": "):
            Q.fp4_moe(torch.zeros(2, 128), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2), *{**good, name: bad}.values(),
                      Q.Fp4MoeWork(2, 2, 128, 64, 3, "cpu"), out_f32=torch.zeros(2, 128))


def test_what_was_said_of_a_matrix_is_not_said_of_the_next_one():
    """A matrix that took the place of another, address and all, is looked at itself."""
    from types import SimpleNamespace
    from bloomery_b200.runtime.batch_decode import BatchDecode
    asks = SimpleNamespace(fp4_native=True, _fp4_ok={})
    native = lambda q: BatchDecode._native_fp4(asks, q)                                          # noqa: E731
    signed = w(16, 128).data
    signed[3, 64 + 2] = 0x80
    for _ in range(200):
        good = QWeight(w(1, 128).data, "NVFP4", 128)
        assert native(good)
        del good
        assert not native(QWeight(signed, "NVFP4", 128))


def test_tables_of_no_rows():
    t = Q.fp4_tiles(0, "cpu")
    assert t.rows == 0 and t.fixed == 0 and int(t.n_mtiles) == 0
    with pytest.raises(ValueError, match="CUDA"):                 # the last check
        Q.fp4_gemm(Q.Fp4Rows(1, 128, "cpu"), w(16, 128), t, out_f32=torch.zeros(0, 16))


def test_plans_of_more_slots_than_their_table_has_rows():
    """A product trusts the rows that the table was made for."""
    from bloomery_b200.ops import gemm as G
    ids, i32 = torch.zeros(65, dtype=torch.int32), torch.zeros(200, dtype=torch.int32)
    with pytest.raises(ValueError, match="65 slots"):
        G.moe_plan(ids, ids.float(), 4, G.TileTable(64, 4, "cpu", 32), i32, i32, i32.float())
    with pytest.raises(ValueError, match="5 experts"):
        G.moe_plan(ids[:64], ids.float()[:64], 5, G.TileTable(64, 4, "cpu", 32), i32, i32, i32.float())
