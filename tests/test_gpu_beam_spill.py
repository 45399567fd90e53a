"""A beam search that needs the pages of an idle sequence: what comes back for that sequence is what it had."""
import dataclasses

import pytest
import torch

gpu = pytest.mark.gpu
DEV = "cuda:0"


@gpu
@pytest.mark.parametrize("busy", [False, True])
def test_a_sequence_that_made_room_comes_back_bit_for_bit(busy):
    """``busy``: the caller's stream still has work in front, so that the copies out start long after the call."""
    from bloomery_b200.models.spec import tiny_qwen3moe
    from bloomery_b200.models.weights import Weights, synth_tensors
    from bloomery_b200.runtime.beam import BeamSearch
    from bloomery_b200.runtime.engine import DecodeEngine
    spec = dataclasses.replace(tiny_qwen3moe(), eos_id=-1)
    w = Weights.from_items(spec, synth_tensors(spec, DEV, seed=3), DEV)
    eng = DecodeEngine(w, n_slots=6, slot_ctx=512, kv_pages=14)
    g = torch.Generator().manual_seed(1)
    prompt = torch.randint(0, spec.vocab, (390,), generator=g).tolist()
    search = BeamSearch(eng, 4, max_new=70, first_slot=1)
    want = [h.tokens for h in search.search([[5]], 66)[0]]      # two pages a beam; warms the launches up
    eng.prefill(0, prompt)                                      # seven pages
    eng.step([(5, 3, 0)])                                       # the pass that comes last is another sequence's
    n = len(prompt)
    pages = torch.tensor(eng.kv.pages[0], device=DEV)
    had = [c[:, pages].clone() for c in (eng.kv.k, eng.kv.v)]
    torch.cuda.synchronize()
    spills = eng.kv.n_spills
    if busy:
        torch.cuda._sleep(200_000_000)                          # a tenth of a second
    got = [h.tokens for h in search.search([[5]], 66)[0]]
    assert eng.kv.n_spills == spills + 1 and 0 in eng.kv.spilled
    assert got == want
    eng.kv.ensure(0, n)
    back = torch.tensor(eng.kv.pages[0], device=DEV)
    for c, before in zip((eng.kv.k, eng.kv.v), had):
        assert torch.equal(c[:, back].view(torch.int16), before.view(torch.int16))
