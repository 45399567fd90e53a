"""Beam search on the engine: what it returns is scored again, token by token, through the ordinary batched pass of a slot of its own;
a search of one beam is the greedy chain; wider searches find no worse sequences; a finished beam stays as it is."""
import dataclasses

import pytest
import torch

gpu = pytest.mark.gpu
DEV = "cuda:0"


def _engine(n_slots, slot_ctx=512, **kw):
    from bloomery_b200.models.spec import tiny_qwen3moe
    from bloomery_b200.models.weights import Weights, synth_tensors
    from bloomery_b200.runtime.engine import DecodeEngine
    spec = dataclasses.replace(tiny_qwen3moe(), eos_id=-1)
    return spec, DecodeEngine(Weights.from_items(spec, synth_tensors(spec, DEV, seed=3), DEV), n_slots=n_slots, slot_ctx=slot_ctx, **kw)


def _prompts(spec, lengths, seed=5):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, spec.vocab, (n,), generator=g).tolist() for n in lengths]


def _score(eng, bd, slot, prompt, tokens):
    """The log-probability of ``tokens`` behind ``prompt``, every position from a pass that appends it as the search does."""
    eng.reset(slot)
    if len(prompt) > 1:
        eng.prefill(slot, prompt[:-1])
    total, ids = 0.0, [prompt[-1]] + tokens
    for i in range(len(tokens)):
        bd.step([(slot, ids[i], len(prompt) - 1 + i)])
        total += float(torch.log_softmax(bd.logits[0].double(), 0)[ids[i + 1]])
    eng.reset(slot)
    return total


@gpu
@pytest.mark.parametrize("beams,lengths,kv", [(4, [130], "f16"), (5, [70, 9, 200], "f16"), (3, [64, 65], "f16"), (2, [1], "f16"),
                                              (4, [150, 20], "q8_0")])
def test_scores_are_those_of_the_returned_sequences(beams, lengths, kv):
    """70 new tokens: the page being filled ends once at least, so that states move within a page and over its end.  The band is
    the batched pass's own: bf16 rows through four layers put a log-probability within 0.05 of another route's."""
    from bloomery_b200.runtime.batch_decode import BatchDecode
    from bloomery_b200.runtime.beam import BeamSearch
    G = len(lengths)
    spec, eng = _engine(beams * G + 1, kv_type=kv)
    search = BeamSearch(eng, beams, groups=G, max_new=80)
    bd = BatchDecode(eng, max_rows=16)
    prompts = _prompts(spec, lengths)
    free = eng.kv.free_pages()
    got = search.search(prompts, 70)
    assert eng.kv.free_pages() == free
    for g, prompt in enumerate(prompts):
        assert len(got[g]) == beams and len({tuple(h.tokens) for h in got[g]}) == beams
        assert [h.score for h in got[g]] == sorted((h.score for h in got[g]), reverse=True)
        for h in (got[g][0], got[g][-1]):
            assert len(h.tokens) == 70
            want = _score(eng, bd, beams * G, prompt, h.tokens)
            assert abs(h.score - want) < 0.05 * 70 ** 0.5, (g, h.score, want)
    again = search.search(prompts, 70)                     # the captured steps, from the first on
    assert [[h.tokens for h in hs] for hs in again] == [[h.tokens for h in hs] for hs in got]


@gpu
def test_one_beam_is_the_greedy_chain_and_more_find_no_less():
    from bloomery_b200.runtime.beam import BeamSearch
    spec, eng = _engine(8)
    prompt = _prompts(spec, [90])[0]
    best = {}
    for beams in (1, 2, 8):
        best[beams] = BeamSearch(eng, beams, max_new=24).search([prompt], 24)[0][0]
    eng.prefill(0, prompt[:-1])
    tok, greedy = prompt[-1], []
    from bloomery_b200.runtime.batch_decode import BatchDecode
    bd = BatchDecode(eng, max_rows=16)
    for i in range(24):
        tok = bd.step([(0, tok, len(prompt) - 1 + i)])[0]
        greedy.append(tok)
    same = sum(a == b for a, b in zip(best[1].tokens, greedy))
    assert best[1].tokens[:4] == greedy[:4] and same >= 4   # random weights: a near tie may part them later
    assert best[8].score >= best[1].score - 0.5


@gpu
def test_a_beam_that_ends_stays_and_is_ranked_by_length():
    from bloomery_b200.runtime.beam import BeamSearch
    spec, eng = _engine(12)
    prompt = _prompts(spec, [77])[0]
    plain = BeamSearch(eng, 4, max_new=20).search([prompt], 20)[0]
    eos = plain[0].tokens[6]                                # an id that the best beam comes to
    first = plain[0].tokens.index(eos)
    got = BeamSearch(eng, 4, groups=3, eos=eos, alpha=0.7, max_new=40).search([prompt] * 3, 40)
    assert [h.tokens for h in got[0]] == [h.tokens for h in got[1]] == [h.tokens for h in got[2]]
    ended = [h for h in got[0] if h.finished]
    assert ended and all(eos not in h.tokens for h in got[0])
    assert any(h.tokens == plain[0].tokens[:first] for h in ended) or min(h.rank for h in got[0]) > plain[0].score / 20 ** 0.7
    assert [h.rank for h in got[0]] == sorted((h.rank for h in got[0]), reverse=True)


@gpu
def test_without_graphs_and_with_other_sequences_beside_it():
    """The slots of other sequences keep theirs, and launches one by one give what the graphs give."""
    from bloomery_b200.runtime.beam import BeamSearch
    spec, eng = _engine(6)
    a, b = _prompts(spec, [100, 40], seed=8)
    eng.prefill(0, b)
    before = eng.step([(0, 7, 40)])
    eng.cut(0, 40)
    want = BeamSearch(eng, 4, max_new=12, first_slot=2).search([a], 12)
    eng.use_graphs = False
    got = BeamSearch(eng, 4, max_new=12, first_slot=2).search([a], 12)
    eng.use_graphs = True
    assert [h.tokens for h in got[0]] == [h.tokens for h in want[0]]
    assert eng.step([(0, 7, 40)]) == before


@gpu
def test_what_cannot_be_searched_is_refused():
    from bloomery_b200.runtime.beam import BeamSearch
    spec, eng = _engine(4)
    for kw in (dict(beams=5), dict(beams=0), dict(beams=2, groups=3), dict(beams=2, first_slot=3), dict(beams=33, groups=2)):
        with pytest.raises(ValueError):
            BeamSearch(eng, **kw)
    search = BeamSearch(eng, 2, max_new=8)
    for prompts, n in (([], 4), ([[1], [2]], 4), ([[]], 4), ([[1]], 9), ([[1]], 0), ([[1] * 510], 8)):
        with pytest.raises(ValueError):
            search.search(prompts, n)


@gpu
def test_the_example_runs(capsys):
    from bloomery_b200.runtime.beam import main
    assert main(["--beams", "3", "--new", "6"]) == 0
    assert len(capsys.readouterr().out.strip().splitlines()) == 3
