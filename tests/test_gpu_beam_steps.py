"""A beam search step by step: what it chose from its own beams, beside the candidates that the ordinary batched pass gives for the same
sequences, and captured steps under prompts of other lengths."""
import pytest
import torch

from test_gpu_beam_search import _engine, _prompts

gpu = pytest.mark.gpu


class Plain:
    """Beams in slots ``first`` and on, a pass of the ordinary attention a step; a child gets a copy of its parent's positions."""

    def __init__(self, eng, beams, first, prompt, n_new):
        from bloomery_b200.runtime.batch_decode import BatchDecode
        self.e, self.B, self.slots = eng, beams, list(range(first, first + beams))
        self.bd = BatchDecode(eng, max_rows=16)
        for slot in self.slots:
            eng.reset(slot)
            if len(prompt) > 1:
                eng.prefill(slot, prompt[:-1])
            eng.kv.ensure(slot, len(prompt) + n_new)
        self.ids, self.pos = [prompt[-1]] * beams, len(prompt) - 1
        self.scores = [0.0] + [float("-inf")] * (beams - 1)

    def candidates(self):
        """[beams, vocab] in 64 bits: the scores of all continuations."""
        self.bd.step([(s, t, self.pos) for s, t in zip(self.slots, self.ids)])
        lp = torch.log_softmax(self.bd.logits[:self.B].double(), -1)
        return lp + torch.tensor(self.scores, dtype=torch.float64, device=lp.device).unsqueeze(1)

    def follow(self, cand, parent, token):
        kv = self.e.kv
        torch.cuda.synchronize()
        for pool in (kv.k, kv.v):
            was = [pool[:, torch.tensor(kv.pages[s], device=pool.device)].clone() for s in self.slots]
            for i, p in enumerate(parent):
                pool[:, torch.tensor(kv.pages[self.slots[i]], device=pool.device)] = was[p]
        torch.cuda.synchronize()
        self.scores = [float(cand[p, t]) for p, t in zip(parent, token)]
        self.ids, self.pos = list(token), self.pos + 1


@gpu
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("beams,length,kv", [(4, 130, "f16"), (3, 40, "f16"), (6, 64, "f16"), (4, 90, "q8_0")])
def test_every_step_takes_the_best_candidates_of_its_beams(shared, beams, length, kv):
    """30 steps.  The plain side follows the search's choices and says after each what they were worth among all candidates of
    the same beams.  With the ordinary attention both sides compute the same rows, and the search adds its scores in 32 bits
    (2^-24 of 300 nats a step at most); behind shared pages a log-probability is within 0.05 of the other route's, sums of t
    within 0.05 sqrt(t), and a candidate that is taken within two of those of one that is not."""
    from bloomery_b200.runtime.beam import BeamSearch
    n = 30
    spec, eng = _engine(2 * beams, kv_type=kv)
    prompt = _prompts(spec, [length], seed=length)[0]
    search = BeamSearch(eng, beams, max_new=n, shared_attention=shared)
    best = search.search([prompt], n)[0]
    hist = search.hist[:n].cpu()
    plain = Plain(eng, beams, beams, prompt, n)
    for t in range(n):
        cand = plain.candidates()
        band = 2 * 0.05 * (t + 1) ** 0.5 if shared else (t + 1) * 300 * 2.0 ** -23
        parent, token = hist[t, 0].tolist(), hist[t, 1].tolist()
        taken = [float(cand[p, k]) for p, k in zip(parent, token)]
        order = cand.flatten().topk(beams).values.tolist()
        assert len(set(zip(parent, token))) == beams, t
        for i in range(beams):                             # place i is worth what the i-th best candidate is
            assert abs(taken[i] - order[i]) <= band, (t, i, taken, order)
        plain.follow(cand, parent, token)
    for h, score in zip(best, plain.scores):
        assert abs(h.score - score) <= (0.05 * n ** 0.5 if shared else n * 300 * 2.0 ** -23)


@gpu
def test_one_beam_is_the_greedy_chain_to_its_end():
    """The same pass, row for row: 40 ids, all of them."""
    from bloomery_b200.runtime.batch_decode import BatchDecode
    from bloomery_b200.runtime.beam import BeamSearch
    spec, eng = _engine(2)
    prompt = _prompts(spec, [90])[0]
    got = BeamSearch(eng, 1, max_new=40).search([prompt], 40)[0][0].tokens
    eng.prefill(1, prompt[:-1])
    bd, tok, greedy = BatchDecode(eng, max_rows=16), prompt[-1], []
    for i in range(40):
        tok = bd.step([(1, tok, len(prompt) - 1 + i)])[0]
        greedy.append(tok)
    assert got == greedy


@gpu
def test_captured_steps_take_up_other_prompts():
    """Graphs of the first search serve prompts of other lengths, with more shared pages and fewer, and searches that share
    nothing; a search of launches, made for each of them, gives the same."""
    from bloomery_b200.runtime.beam import BeamSearch
    spec, eng = _engine(8)
    search = BeamSearch(eng, 4, groups=2, max_new=20)
    search.search(_prompts(spec, [130, 70], seed=1), 20)
    assert len(search.graphs) == 2
    for lengths in ([300, 20], [20, 300], [65, 66], [20, 9], [200, 333], [9, 64]):
        prompts = _prompts(spec, lengths, seed=sum(lengths))
        got = search.search(prompts, 20)
        eng.use_graphs = False
        want = BeamSearch(eng, 4, groups=2, max_new=20).search(prompts, 20)
        eng.use_graphs = True
        assert got == want, lengths
    assert len(search.graphs) == 4


@gpu
def test_the_example_takes_either_attention(capsys):
    from bloomery_b200.runtime.beam import main
    assert main(["--beams", "3", "--new", "6", "--separate"]) == 0
    assert len(capsys.readouterr().out.strip().splitlines()) == 3
