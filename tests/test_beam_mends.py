"""Calls of the beam operators that were taken although no kernel can serve them, without a card."""
import ctypes

import pytest
import torch

from bloomery_b200.ops import beam
from bloomery_b200.ops._lib import cuda

SHAPE = -2
A = 0x1000000        # an aligned address nothing reads


def _cells(dtype=torch.int32):
    return torch.zeros(2, 3, dtype=dtype)


def _select(**kw):
    a = dict(logits=torch.zeros(6, 10), scores=_cells(torch.float32), scratch=beam.BeamScratch(2, 3, 10, "cpu"), parent=_cells(),
             token=_cells(), out_scores=_cells(torch.float32), done=_cells(), lengths=_cells(), out_done=_cells(), out_lengths=_cells(),
             eos=1)
    a.update(kw)
    beam.beam_select(**a)


def test_a_choice_in_place_is_refused():
    with pytest.raises(ValueError, match="CUDA device"):
        _select()                                          # everything else is in order
    x, i = _cells(torch.float32), _cells()
    for kw in (dict(scores=x, out_scores=x), dict(done=i, out_done=i), dict(lengths=i, out_lengths=i), dict(done=i, out_lengths=i),
               dict(done=i, parent=i)):
        with pytest.raises(ValueError, match="other tensors"):
            _select(**kw)


@pytest.mark.parametrize("out", ["parent", "token", "out_scores", "out_done", "out_lengths"])
@pytest.mark.parametrize("over", ["scores", "done", "lengths", "logits", "parent"])
@pytest.mark.parametrize("off", [-28, 0, 28])
def test_outputs_over_what_is_read_are_refused_before_the_launch(out, over, off):
    """Two searches of four: 32 bytes a tensor; the logits are 28,000 bytes before their last row."""
    if out == over:
        return
    names = ["logits", "scores", "done", "lengths", "work", "parent", "token", "out_scores", "out_done", "out_lengths"]
    call = dict(logits=A, stride=1000, scores=0, done=0, lengths=0, work=0, parent=0, token=0, out_scores=0, out_done=0, out_lengths=0,
                fault=0, stream=0, V=1000, G=2, B=4, eos=5, chunks=1, alpha=0.5)
    call |= {n: A + (i << 16) for i, n in enumerate(names)}
    call[out] = call[over] + (31000 if over == "logits" else 0) + off
    fn = cuda().bl_beam_select
    fn.argtypes = [ctypes.c_char_p]
    assert fn(beam._SELECT.pack(*call.values())) == SHAPE


def test_a_plan_takes_no_prefix_that_its_tables_cannot_hold():
    """A replayed graph checks nothing: the lengths that it will find are checked where they are set."""
    from bloomery_b200.ops.prefix import PrefixPlan, prefix_attention
    plan = PrefixPlan([2], [64], 4, 2, 64, "cpu")
    plan.set_prefix([640])                                 # no call so far
    plan.set_prefix([64])
    cache = torch.zeros(3, 2, 64, 64, dtype=torch.float16)
    rows = torch.zeros(2, dtype=torch.int32)
    for pages in (9, 4, 6):
        with pytest.raises(ValueError, match="CUDA device"):
            prefix_attention(torch.zeros(2, 4, 64), cache, cache, rows, rows, torch.zeros(2, pages, dtype=torch.int32), plan,
                             torch.zeros(2, 256, dtype=torch.bfloat16))
    plan.set_prefix([256])
    with pytest.raises(ValueError, match="longer than a table row of 4"):
        plan.set_prefix([320])
    assert plan.prefix_len == [256] and plan.meta[0, 2] == 256


def test_launches_for_another_device_than_the_current_one_are_refused(monkeypatch):
    from bloomery_b200.ops import _lib, prefix
    from bloomery_b200.ops._lib import raw_stream
    monkeypatch.setattr(_lib, "_device", lambda: 0)
    monkeypatch.setattr(_lib, "_stream", lambda index: 40 + index)
    assert raw_stream(0) == 40
    with pytest.raises(ValueError, match="not the current device"):
        raw_stream(1)

    # the calls take their stream from there: tensors that say they are on the second card
    class Far(torch.Tensor):
        def get_device(self):
            return 1

    def far(*shape, dtype=torch.int32):
        return torch.zeros(*shape, dtype=dtype).as_subclass(Far)
    scratch = beam.BeamScratch(2, 3, 10, "cpu")
    scratch.index = 1
    with pytest.raises(ValueError, match="not the current device"):
        beam.beam_select(far(6, 10, dtype=torch.float32), far(2, 3, dtype=torch.float32), scratch, far(2, 3), far(2, 3),
                         far(2, 3, dtype=torch.float32))
    with pytest.raises(ValueError, match="not the current device"):
        beam.beam_reorder(far(1, 4, 1, 64, 8), far(1, 4, 1, 64, 8), far(2, 4), far(2, 4), far(2), far(1, 2), far(1))
    plan = prefix.PrefixPlan([2], [64], 4, 2, 64, "cpu")
    plan.index = 1
    cache = far(3, 2, 64, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="not the current device"):
        prefix.prefix_attention(far(2, 4, 64, dtype=torch.float32), cache, cache, far(2), far(2), far(2, 4), plan,
                                far(2, 256, dtype=torch.bfloat16))


@pytest.mark.parametrize("fault", [torch.zeros(1, dtype=torch.int64), torch.zeros(0, dtype=torch.int32), torch.zeros(1),
                                   torch.zeros(1, dtype=torch.int32, device="meta")])
def test_a_fault_word_is_an_int32_on_the_device_of_the_rest(fault):
    from bloomery_b200.ops.prefix import PrefixPlan, prefix_attention
    if fault.device.type == "meta":                        # a tensor of some other device
        fault = fault.as_subclass(type("Far", (torch.Tensor,), {"get_device": lambda self: 0}))
    cache, rows = torch.zeros(3, 2, 64, 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    calls = [
        lambda f: _select(fault=f),
        lambda f: beam.beam_reorder(torch.zeros(1, 4, 1, 64, 8), torch.zeros(1, 4, 1, 64, 8), torch.zeros(2, 4, dtype=torch.int32),
                                    torch.zeros(2, 4, dtype=torch.int32), rows, rows.view(1, 2), rows[:1], f),
        lambda f: prefix_attention(torch.zeros(2, 4, 64), cache, cache, rows, rows, torch.zeros(2, 4, dtype=torch.int32),
                                   PrefixPlan([2], [64], 4, 2, 64, "cpu"), torch.zeros(2, 256, dtype=torch.bfloat16), f),
    ]
    for call in calls:
        with pytest.raises(ValueError, match="CUDA device"):
            call(torch.zeros(1, dtype=torch.int32))        # everything else is in order
        with pytest.raises(ValueError, match="fault"):
            call(fault)


def _advance(**kw):
    G, B, i32 = 2, 3, dict(dtype=torch.int32)
    a = dict(tokens=torch.zeros(16, **i32), row_pos=torch.zeros(16, **i32), row_seq=torch.zeros(16, **i32), held=torch.zeros(G, **i32),
             hist=torch.zeros(8, 2, G * B, **i32), count=torch.zeros(1, **i32), slots=torch.zeros(G * B, **i32),
             parent=torch.zeros(G * B, **i32), token=torch.zeros(G * B, **i32), done=torch.zeros(G, B, **i32), scores=torch.zeros(G, B),
             G=G, B=B)
    a.update(kw)
    beam.beam_advance(**a)


@pytest.mark.parametrize("kw", [
    dict(tokens=torch.zeros(5, dtype=torch.int32)), dict(row_pos=torch.zeros(16, dtype=torch.int64)),
    dict(row_seq=torch.zeros(32, dtype=torch.int32)[::2]), dict(held=torch.zeros(3, dtype=torch.int32)),
    dict(hist=torch.zeros(8, 2, 5, dtype=torch.int32)), dict(hist=torch.zeros(8, 12, dtype=torch.int32)), dict(hist=torch.zeros(8, 2, 6)),
    dict(count=torch.zeros(0, dtype=torch.int32)), dict(slots=torch.zeros(5, dtype=torch.int32)),
    dict(parent=torch.zeros(6, dtype=torch.int64)), dict(token=torch.zeros(6)), dict(done=torch.zeros(2, 3, dtype=torch.bool)),
    dict(scores=torch.zeros(2, 3, dtype=torch.float64)), dict(G=0), dict(B=0)])
def test_arguments_of_the_bookkeeping_are_checked(kw):
    with pytest.raises(ValueError, match="CUDA device"):
        _advance()                                         # everything else is in order
    with pytest.raises(ValueError) as e:
        _advance(**kw)
    assert "CUDA device" not in str(e.value)


@pytest.mark.parametrize("alpha", [float("nan"), float("inf"), float("-inf"), 17.0, -17.0])
def test_an_exponent_that_leaves_no_order_is_refused(alpha):
    """Ranks of NaN found no candidate at all, an infinite exponent made all of them equal."""
    with pytest.raises(ValueError, match="CUDA device"):
        _select(alpha=16.0)
    with pytest.raises(ValueError, match="alpha"):
        _select(alpha=alpha)
    call = dict(logits=A, stride=1000, scores=A + 0x10000, done=0, lengths=A + 0x20000, work=A + 0x30000, parent=A + 0x40000,
                token=A + 0x50000, out_scores=A + 0x60000, out_done=0, out_lengths=0, fault=0, stream=0, V=1000, G=2, B=4, eos=-1,
                chunks=1, alpha=alpha)
    fn = cuda().bl_beam_select
    fn.argtypes = [ctypes.c_char_p]
    assert fn(beam._SELECT.pack(*call.values())) == SHAPE
