"""What a beam search does to the engine around it, without a card: pages, their protection, and the order of streams.  The engine
is a page pool with the bookkeeping of :class:`DecodeEngine`; the launches of a search are left out."""
import contextlib
import threading
from types import SimpleNamespace

import pytest
import torch

from bloomery_b200.runtime.batch_decode import BatchDecode
from bloomery_b200.runtime.beam import BeamSearch
from bloomery_b200.runtime.kv import PAGE, KvPool, OutOfPages


class Reached(Exception):
    """The launches of the first step would come next."""


class FakeStream:
    def __init__(self, name, log):
        self.name, self.log = name, log

    def wait_stream(self, other):
        self.log.append((self.name, "waits for", other.name))


class FakeEngine:
    def __init__(self, n_pages, n_slots, max_pages, log):
        self.kv = KvPool(1, 1, 4, n_pages, n_slots, max_pages, "cpu")
        self.n_slots, self.slot_ctx, self.device = n_slots, max_pages * PAGE, "cpu"
        self._lock, self.log, self.kv_q8 = threading.Lock(), log, False

    def reset(self, slot):
        self.kv.truncate(slot, 0)

    def prefill(self, slot, tokens):
        with self._lock:
            for i in range(0, len(tokens), 8):             # the 8-row pass: set_rows
                self.kv.protect = {slot}
                for pos in range(i, min(i + 8, len(tokens))):
                    self.kv.ensure(slot, pos + 1)
                    self.kv.own(slot, pos)


@pytest.fixture
def make(monkeypatch):
    log = []
    caller, current = FakeStream("caller", log), []
    current.append(caller)

    @contextlib.contextmanager
    def stream(s):
        current.append(s)
        try:
            yield
        finally:
            current.pop()

    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: current[-1])

    def build(n_pages, n_slots, max_pages, beams, groups, first_slot=0):
        e = FakeEngine(n_pages, n_slots, max_pages, log)
        s = object.__new__(BeamSearch)
        s.e, s.B, s.G, s.max_new, s.alpha, s.eos = e, beams, groups, 128, 0.0, -1
        s.shared_attention = True
        s.R = s.M = beams * groups
        s.slots = list(range(first_slot, first_slot + s.R))
        s.bd = SimpleNamespace(_stream=FakeStream("steps", log))

        def first_step(shared):
            log.append((current[-1].name, "first step", None))
            assert all(e.kv.pages[x] for x in s.slots), "a beam without pages"
            raise Reached
        s.plan = SimpleNamespace(set_prefix=first_step)
        for name in ("snapshot", "sync_table"):
            def traced(*a, _f=getattr(e.kv, name), _n=name, **kw):
                log.append((current[-1].name, _n, a[0] if a else None))
                return _f(*a, **kw)
            monkeypatch.setattr(e.kv, name, traced)
        return s, e, log
    return build


def test_a_later_prompt_does_not_take_an_earlier_ones_pages(make):
    """Nine pages; two searches of two beams whose prompts end in their first page, three pages a beam.  A prompt's passes
    protect its own slot alone."""
    s, e, log = make(9, 6, 4, beams=2, groups=2)
    with pytest.raises(OutOfPages):
        s.search([[1] * 21, [2] * 21], 110)
    assert not e.kv.spilled and e.kv.n_spills == 0 and ("steps", "first step", None) not in log
    assert e.kv.free_pages() == 9 and not e.kv.pinned


def test_an_idle_sequence_makes_room_and_beams_keep_theirs(make):
    s, e, log = make(9, 6, 4, beams=2, groups=2, first_slot=1)
    e.prefill(0, [7] * 70)                                 # two pages that nobody needs now
    with pytest.raises(Reached):
        s.search([[1] * 21, [2] * 21], 80)                 # two pages a beam
    assert set(e.kv.spilled) == {0} and e.kv.n_spills == 1
    assert e.kv.free_pages() == 9 and not e.kv.pinned


def test_steps_wait_for_what_made_room_and_the_caller_for_the_steps(make):
    """The copy of a sequence that makes room runs on the caller's stream: the steps that write its pages come behind it, and
    the caller's next work, the table first, behind the steps."""
    s, e, log = make(9, 6, 4, beams=2, groups=2, first_slot=1)
    e.prefill(0, [7] * 70)
    e.kv.protect = {5}                                     # as after a pass over another slot
    with pytest.raises(Reached):
        s.search([[1], [2]], 100)                          # two pages a beam, no prompt pass that the host waits for
    spill, step = log.index(("caller", "snapshot", 0)), log.index(("steps", "first step", None))
    assert ("steps", "waits for", "caller") in log[spill:step]
    behind = log.index(("caller", "waits for", "steps"), step)
    assert log.index(("caller", "sync_table", None), step) > behind
    assert ("steps", "sync_table", None) not in log[step:]


def test_pages_change_hands_under_the_engines_lock(make, monkeypatch):
    s, e, log = make(9, 6, 4, beams=2, groups=2)
    for name in ("ensure", "share_prefix", "truncate"):
        def held(*a, _f=getattr(e.kv, name), _n=name, **kw):
            assert e._lock.locked(), _n
            return _f(*a, **kw)
        monkeypatch.setattr(e.kv, name, held)
    with pytest.raises(Reached):
        s.search([[1] * 70, [2] * 5], 20)
    assert not e._lock.locked()


def test_engines_whose_experts_are_elsewhere_are_refused():
    """The batched pass would hand host stacks, or a rank's share of them, to the kernels."""
    from bloomery_b200.parallel.sharded import ShardedEngine
    from bloomery_b200.runtime.tiered import TieredEngine
    for kind in (TieredEngine, ShardedEngine):
        e = object.__new__(kind)
        e.spec, e.n_slots = SimpleNamespace(mla=False, eos_id=2), 8
        with pytest.raises(NotImplementedError):
            BeamSearch(e, 4)


def _batched(e):
    bd = object.__new__(BatchDecode)
    bd.e, bd._stream = e, FakeStream("steps", e.log)
    bd.params, bd.params_host = torch.zeros(3, 16, dtype=torch.int32), torch.zeros(3, 16, dtype=torch.int32)
    bd._params_np = bd.params_host.numpy()
    e.slot_len = [0] * e.n_slots
    return bd


def test_rows_of_a_batched_pass_do_not_take_each_others_pages(make):
    """Twelve sequences of a page each, a pool of twelve: the last row's second page has to come from nobody in the pass."""
    _, e, _ = make(12, 12, 4, beams=2, groups=2)
    bd = _batched(e)
    bd.set_rows([(i, 1, 40) for i in range(12)])
    with pytest.raises(OutOfPages):
        bd.set_rows([(i, 1, 64 if i == 11 else 41) for i in range(12)])
    assert not e.kv.spilled
    bd.set_rows([(i, 1, 64 if i == 11 else 41) for i in range(3, 12)])      # three idle ones: the oldest makes room
    assert set(e.kv.spilled) == {0}


def test_a_batched_pass_waits_for_the_table_and_for_what_made_room(make):
    _, e, log = make(12, 13, 4, beams=2, groups=2)
    bd = _batched(e)
    bd.set_rows([(i, 1, 40) for i in range(12)])
    del log[:]
    bd.set_rows([(12, 1, 0)])
    spill, table = log.index(("caller", "snapshot", 0)), log.index(("caller", "sync_table", None))
    assert spill < table < log.index(("steps", "waits for", "caller"))


@pytest.mark.parametrize("asked,q8,lengths,shared", [
    (None, False, [21, 9], False), (None, False, [64, 9], False), (None, False, [21, 65], True), (None, True, [21, 9], True),
    (True, False, [21, 9], True), (False, False, [130, 130], False), (False, True, [130, 130], False)])
def test_which_attention_a_search_takes(make, monkeypatch, asked, q8, lengths, shared):
    s, e, log = make(16, 6, 4, beams=2, groups=2)
    s.shared_attention, e.kv_q8 = asked, q8
    if asked is False:
        s.plan = None
    zeros = torch.zeros
    s.tables, s.scores, s.done, s.lengths = [None, zeros(1)], [zeros(2, 2)], [zeros(2, 2)], [zeros(2, 2)]
    monkeypatch.setattr(e.kv, "sync_table", lambda: (_ for _ in ()).throw(Reached) if s.bd.prefix is None else None)
    with pytest.raises(Reached):
        s.search([[1] * n for n in lengths], 20)
    assert (s.bd.prefix is s.plan and s.plan is not None) is shared
