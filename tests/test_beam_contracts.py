"""Launch contracts of the shared-prefix attention and of the beam entries, without a card: each refuses before it touches the
device.  The pointers are never dereferenced."""
import ctypes
import struct

import pytest
import torch

from bloomery_b200.ops import beam, prefix
from bloomery_b200.ops._lib import KernelError, check, cuda
from bloomery_b200.ops.beam import BeamScratch
from bloomery_b200.ops.prefix import PrefixPlan

SHAPE, ALIGN, LIMIT = -2, -4, -5
A = 0x10000          # an aligned address nothing reads


def _call(name, packing, values):
    fn = getattr(cuda(), name)
    fn.argtypes = [ctypes.c_char_p]
    return fn(packing.pack(*values.values()))


def _attention(**kw):
    call = dict(q=A, k=A, v=A, row_pos=A, row_seq=A, table=A, meta=A, work=A, out=A, fault=A, stream=0, n_slots=8, max_pages=16,
                n_pages=64, head=128, n_q=32, n_kv=4, M=8, n_units=1, unit_rows=8, kv_q8=0, n_cta=148, layer=0)
    assert set(kw) <= set(call)
    return _call("bl_prefix_attention", prefix._CALL, call | kw)


@pytest.mark.parametrize("code, kw", [
    (SHAPE, dict(head=96)), (SHAPE, dict(n_kv=0)), (SHAPE, dict(n_q=30)), (SHAPE, dict(n_q=128)), (SHAPE, dict(M=0)), (SHAPE, dict(M=513)),
    (SHAPE, dict(n_units=0)), (SHAPE, dict(n_units=9)), (SHAPE, dict(unit_rows=0)), (SHAPE, dict(unit_rows=33)), (SHAPE, dict(n_cta=0)),
    (SHAPE, dict(n_cta=161)), (SHAPE, dict(n_slots=0)), (SHAPE, dict(max_pages=0)), (SHAPE, dict(n_pages=0)),
    (LIMIT, dict(n_pages=1 << 23)), (LIMIT, dict(max_pages=1 << 19)), (LIMIT, dict(M=512, max_pages=1 << 13)),
    (ALIGN, dict(q=A + 4)), (ALIGN, dict(k=A + 8)), (ALIGN, dict(v=A + 2)), (ALIGN, dict(out=A + 2)), (ALIGN, dict(work=A + 8)),
])
def test_shared_prefix_attention_refuses_before_it_launches(code, kw):
    assert _attention(**kw) == code


def _select(**kw):
    call = dict(logits=A, stride=1000, scores=A, done=0, lengths=0, work=A, parent=A, token=A, out_scores=A, out_done=0, out_lengths=0,
                fault=0, stream=0, V=1000, G=2, B=4, eos=-1, chunks=1, alpha=0.0)
    assert set(kw) <= set(call)
    return _call("bl_beam_select", beam._SELECT, call | kw)


@pytest.mark.parametrize("code, kw", [
    (SHAPE, dict(V=0)), (SHAPE, dict(G=0)), (SHAPE, dict(B=0)), (SHAPE, dict(stride=999)), (SHAPE, dict(chunks=0)), (SHAPE, dict(chunks=1001)),
    (SHAPE, dict(eos=1000)), (SHAPE, dict(done=A)), (SHAPE, dict(alpha=0.5)), (SHAPE, dict(out_lengths=A)),
    (LIMIT, dict(B=65)), (LIMIT, dict(G=16384)), (LIMIT, dict(chunks=65)),
    (ALIGN, dict(logits=A + 2)), (ALIGN, dict(work=A + 4)),
])
def test_choice_of_beams_refuses_before_it_launches(code, kw):
    assert _select(**kw) == code


def _reorder(**kw):
    call = dict(k=A, v=A, k_row=256, v_row=256, table=A, table_out=A + 4096, slots=A, parent=A, held=A, fault=0, stream=0, n_layer=2,
                n_pages=64, n_kv=4, n_slots=8, max_pages=16, G=2, B=4)
    assert set(kw) <= set(call)
    return _call("bl_beam_reorder", beam._REORDER, call | kw)


@pytest.mark.parametrize("code, kw", [
    (SHAPE, dict(n_layer=0)), (SHAPE, dict(n_layer=65536)), (SHAPE, dict(n_pages=0)), (SHAPE, dict(n_kv=0)), (SHAPE, dict(G=0)),
    (SHAPE, dict(B=0)), (SHAPE, dict(n_slots=0)), (SHAPE, dict(max_pages=0)), (SHAPE, dict(table_out=A)), (SHAPE, dict(k_row=0)),
    (LIMIT, dict(B=65)), (LIMIT, dict(n_kv=1 << 17)),
    (ALIGN, dict(k_row=34)), (ALIGN, dict(v_row=34)), (ALIGN, dict(k=A + 8)), (ALIGN, dict(v=A + 4)),
])
def test_states_of_beams_refuse_before_they_launch(code, kw):
    assert _reorder(**kw) == code


@pytest.mark.parametrize("G, B, cap", [(0, 4, 8), (2, 0, 8), (2, 4, -1), (16384, 4, 8)])
def test_bookkeeping_of_beams_refuses_before_it_launches(G, B, cap):
    I, P = ctypes.c_int, ctypes.c_void_p
    p = P(A)
    assert cuda().bl_beam_advance(p, p, p, p, p, I(cap), p, p, p, p, p, p, I(G), I(B), P(0)) == SHAPE


def test_blocks_of_memory_are_as_long_as_the_sources_say():
    assert prefix._CALL.size == 11 * 8 + 12 * 4
    assert beam._SELECT.size == 13 * 8 + 6 * 4 and beam._REORDER.size == 11 * 8 + 8 * 4
    with pytest.raises(KernelError, match=r"bl_beam_select: .* \(code -5\)"):
        check(_select(B=65), "bl_beam_select")


@pytest.mark.parametrize("vocab", [1, 3, 4096, 4097, 32000, 151936, 1 << 20])
@pytest.mark.parametrize("rows", [1, 4, 15, 64, 593, 65535])
@pytest.mark.parametrize("beams", [1, 5, 16, 64])
def test_chunks_of_a_row_are_of_4096_ids_and_merge_in_one_block(vocab, rows, beams):
    n = cuda().bl_beam_chunks(ctypes.c_int(vocab), ctypes.c_int(rows), ctypes.c_int(beams), ctypes.c_int(148))
    assert 1 <= n <= max(1, (vocab + 4095) // 4096)
    assert n * beams <= 256 and (n == 1 or n * rows <= 4 * 148)


def test_scratch_and_plans_refuse_what_no_kernel_takes():
    for groups, beams, vocab in ((0, 4, 100), (1, 0, 100), (1, 65, 100), (1, 4, 0), (16384, 4, 100)):
        with pytest.raises(ValueError):
            BeamScratch(groups, beams, vocab, "cpu")
    for rows, shared, n_q, n_kv, head in (([], [], 32, 4, 128), ([0], [64], 32, 4, 128), ([4], [63], 32, 4, 128), ([4], [-64], 32, 4, 128),
                                          ([4], [64, 64], 32, 4, 128), ([513], [64], 32, 4, 128), ([4], [64], 30, 4, 128),
                                          ([4], [64], 68, 4, 128), ([4], [64], 32, 4, 96)):
        with pytest.raises(ValueError):
            PrefixPlan(rows, shared, n_q, n_kv, head, torch.device("cpu"))
