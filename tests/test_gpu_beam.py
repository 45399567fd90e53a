"""The choice of the next beams against a sort of all candidates in 64 bits, and the states that follow them against copies made one
by one."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
DEV = "cuda:0"
PAGE = 64
INF = math.inf


def _reference(logits, scores, done=None, lengths=None, eos=-1, alpha=0.0):
    """[groups][beams] of (parent, token, score, done, length), candidates in 64 bits, ties to the lowest beam and id."""
    G, B = scores.shape
    V = logits.shape[1]
    out = []
    for g in range(G):
        cand = []
        for b in range(B):
            s = float(scores[g, b])
            n = int(lengths[g, b]) if lengths is not None else 0
            if s == -INF:
                continue
            if done is not None and done[g, b]:
                cand.append((s * max(1, n) ** -alpha, b, eos, s, 1, n))
                continue
            x = logits[g * B + b].double()
            c = x - torch.logsumexp(x, 0) + s
            at = torch.sort(c, descending=True, stable=True).indices[:B].tolist()
            cand += [(float(c[t]) * max(1, n + 1) ** -alpha, b, t, float(c[t]), int(t == eos), n + 1) for t in at if c[t] > -INF]
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        row = [c[1:] for c in cand[:B]]
        row += [(i, max(eos, 0), -INF, 1, int(lengths[g, i]) if lengths is not None else 0) for i in range(len(row), B)]
        out.append(row)
    return out


def _run(logits, scores, done=None, lengths=None, eos=-1, alpha=0.0, scratch=None, fault=None):
    from bloomery_b200.ops.beam import BeamScratch, beam_select
    G, B = scores.shape
    i32 = dict(dtype=torch.int32, device=DEV)
    o = dict(parent=torch.full((G, B), -9, **i32), token=torch.full((G, B), -9, **i32), scores=torch.full((G, B), 9.0, device=DEV),
             done=torch.full((G, B), -9, **i32), length=torch.full((G, B), -9, **i32))
    f = torch.full((1,), -1, **i32) if fault is None else fault
    beam_select(logits, scores, scratch or BeamScratch(G, B, logits.shape[1], DEV), o["parent"], o["token"], o["scores"], done=done,
                lengths=lengths, out_done=o["done"], out_lengths=o["length"] if lengths is not None else None, eos=eos, alpha=alpha, fault=f)
    if fault is None:
        assert int(f) == -1
    return o


def _check(o, want):
    """Picks are equal; a score is the sum of a 32-bit logit, its log-sum (64-bit sums of 32-bit exponentials, within 2^-20 of
    itself) and a 32-bit score, rounded once."""
    G, B = o["parent"].shape
    for g in range(G):
        for i, (p, t, s, d, n) in enumerate(want[g]):
            assert (int(o["parent"][g, i]), int(o["token"][g, i])) == (p, t), (g, i, want[g][i])
            assert int(o["done"][g, i]) == d
            if int(o["length"][g, i]) != -9:
                assert int(o["length"][g, i]) == n
            got = float(o["scores"][g, i])
            assert got == s or abs(got - s) <= 2.0 ** -23 * abs(s) + 2.0 ** -19, (g, i, got, s)


def _logits(rows, V, seed, stride=None, grid=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, stride or V, generator=g, device=DEV) * 3
    if grid:
        x = (x / grid).round() * grid                  # many equal logits
    return x[:, :V]


@gpu
@pytest.mark.parametrize("G,B", [(1, 1), (1, 4), (3, 5), (2, 16), (8, 8), (1, 33), (2, 64)])
@pytest.mark.parametrize("V", [64, 1000, 32000, 151936])
def test_picks_match_a_sort_of_all_candidates(G, B, V):
    x = _logits(G * B, V, seed=V + B)
    scores = -5 * torch.rand(G, B, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    _check(_run(x, scores), _reference(x, scores))


@gpu
@pytest.mark.parametrize("V,stride", [(1, 1), (2, 5), (3, 3), (31, 33), (4097, 4099), (8191, 8200)])
def test_odd_vocabularies_and_strided_rows(V, stride):
    B = min(V, 5)
    x = _logits(2 * B, V, seed=V, stride=stride)
    scores = torch.linspace(0, -1, 2 * B, device=DEV).view(2, B).contiguous()
    _check(_run(x, scores), _reference(x, scores))


@gpu
@pytest.mark.parametrize("B", [2, 7, 16, 64])
def test_ties_go_to_the_lowest_beam_and_id(B):
    """Logits on a coarse grid, every beam with the same row and score: nearly all candidates have equals."""
    row = _logits(1, 32000, seed=3, grid=1.0)
    x = row.expand(B, -1).contiguous()
    scores = torch.zeros(1, B, device=DEV)
    _check(_run(x, scores), _reference(x, scores))
    x.zero_()                                          # all equal: the first B ids of the first beam
    o = _run(x, scores)
    assert o["parent"].flatten().tolist() == [0] * B and o["token"].flatten().tolist() == list(range(B))


@gpu
@pytest.mark.parametrize("order", ["ascending", "descending", "one block", "zeros of both signs"])
def test_orders_that_let_many_candidates_through(order):
    """Rows whose blocks cannot tell their best from a few values, and zeros whose sign is no order."""
    V, B = 30000, 7
    row = torch.linspace(-3, 3, V, device=DEV)
    if order == "descending":
        row = row.flip(0)
    elif order == "one block":
        row = torch.full((V,), -INF, device=DEV)
        row[8000:12000] = torch.linspace(-3, 3, 4000, device=DEV)
    elif order == "zeros of both signs":
        row = torch.where(torch.arange(V, device=DEV) % 3 == 0, -0.0, 0.0)
    x = row.expand(B, -1).contiguous()
    scores = torch.linspace(0, -0.5, B, device=DEV).view(1, B).contiguous()
    scores[0, 3:] = 0
    _check(_run(x, scores), _reference(x, scores))


@gpu
@pytest.mark.parametrize("G,B,V,stride", [(1, 4, 40000, 40000), (8, 8, 151936, 151936), (2, 64, 151936, 151936), (2, 40, 50001, 50003), (16, 16, 32768, 32769)])
@pytest.mark.parametrize("equal", [False, True])
def test_large_logits_that_sit_in_a_few_lanes(G, B, V, stride, equal):
    """Every 1,024 ids eight of large logits: the same few threads hold all of the best, so that the maxima of the others say little.
    Equal ones among them are more than a list holds."""
    x = _logits(G * B, V, seed=V, stride=stride)
    x.clamp_(max=8.0)
    for j in range(8):
        part = x[:, j::1024]
        part.copy_(torch.full_like(part, 12.0) if equal else 12 + part.abs())
    scores = -2 * torch.rand(G, B, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    _check(_run(x, scores), _reference(x, scores))


@gpu
def test_logits_that_a_32_bit_sum_would_merge_keep_their_order():
    x = torch.full((2, 5000), -30.0, device=DEV)
    x[0, 4000], x[0, 7] = 1.0 + 2.0 ** -23, 1.0        # the larger one has the higher id
    x[1, 4], x[1, 3] = 1.0, 1.0 - 2.0 ** -24
    scores = torch.tensor([[-4000.0, -9000.0]], device=DEV)
    o = _run(x, scores)
    assert o["token"].flatten().tolist() == [4000, 7] and o["parent"].flatten().tolist() == [0, 0]


@gpu
def test_the_first_step_has_one_beam():
    """Scores of -inf are no beams and their rows are not read."""
    x = _logits(12, 5000, seed=4)
    scores = torch.full((3, 4), -INF, device=DEV)
    scores[:, 0] = 0
    scores[1] = -INF
    scores[1, 2] = -1.5
    x[1:4] = float("nan")
    x[4:6] = INF
    _check(_run(x, scores), _reference(x, scores))


@gpu
@pytest.mark.parametrize("left", [0, 1, 3, 7])
def test_masked_ids_are_no_candidates_and_short_searches_have_empty_places(left):
    x = torch.full((8, 3000), -INF, device=DEV)
    x[::2, :2990].fill_(-torch.finfo(torch.float32).max)   # a mask of the lowest value keeps its ids as candidates of no weight
    x[4:] = -INF
    if left:
        x[5, 100:100 + left] = torch.linspace(1, 2, left, device=DEV)
    scores = torch.zeros(2, 4, device=DEV)
    _check(_run(x, scores, eos=9), _reference(x, scores, eos=9))


@gpu
@pytest.mark.parametrize("alpha", [0.0, 0.6, 1.0, -0.5])
def test_finished_beams_and_ranks_by_length(alpha):
    G, B, V, eos = 4, 6, 9000, 17
    x = _logits(G * B, V, seed=6)
    x[:, eos] += 8
    g = torch.Generator(device=DEV).manual_seed(7)
    lengths = torch.randint(0, 40, (G, B), generator=g, device=DEV, dtype=torch.int32)
    scores = -3 * torch.rand(G, B, generator=g, device=DEV) - 0.2 * lengths
    done = (torch.rand(G, B, generator=g, device=DEV) < 0.4).int()
    done[1] = 1                                        # nothing left to do
    scores[2, 1] = -INF
    x[done.flatten().bool()] = float("nan")            # rows of finished beams are not read
    o = _run(x, scores, done, lengths, eos, alpha)
    _check(o, _reference(x, scores, done, lengths, eos, alpha))
    assert sorted(o["parent"][1].tolist()) == list(range(B))


@gpu
@pytest.mark.parametrize("bad", [float("nan"), INF])
@pytest.mark.parametrize("where", ["logits", "scores"])
def test_a_search_that_is_not_finite_gets_nan_and_a_fault(bad, where):
    x = _logits(10, 4000, seed=8)
    scores = torch.zeros(2, 5, device=DEV)
    fine = _reference(x, scores)[1]
    if where == "logits":
        x[3, 3999] = bad
    else:
        scores[0, 4] = bad
    fault = torch.full((1,), -1, dtype=torch.int32, device=DEV)
    o = _run(x, scores, fault=fault)
    assert int(fault) == 8 and torch.isnan(o["scores"][0]).all()
    assert o["parent"][0].tolist() == list(range(5))
    assert [(int(p), int(t)) for p, t in zip(o["parent"][1], o["token"][1])] == [c[:2] for c in fine]


@gpu
def test_one_scratch_serves_call_after_call():
    from bloomery_b200.ops.beam import BeamScratch
    scratch = BeamScratch(2, 8, 20000, DEV)
    for seed in range(5):
        x = _logits(16, 20000, seed=seed, grid=0.25)
        scores = (-seed * torch.rand(2, 8, device=DEV)).contiguous()
        first = _run(x, scores, scratch=scratch)
        _check(first, _reference(x, scores))
        again = _run(x, scores, scratch=scratch)
        assert all(torch.equal(first[k], again[k]) for k in first)


# ---- states -------------------------------------------------------------------------------------------------------
def _states(G, B, held, n_layer=3, n_kv=2, k_row=64, v_row=64, dtype=torch.float16, seed=0, extra=2):
    g = torch.Generator().manual_seed(seed)
    col = held // PAGE
    max_pages = col + extra
    n_pages = G * (col + extra * B) + 1
    perm = torch.randperm(n_pages, generator=g).tolist()
    table = torch.full((G * B + 3, max_pages), -1, dtype=torch.int32)
    slots = torch.randperm(G * B + 3, generator=g)[:G * B]
    for s in range(G):
        shared = [perm.pop() for _ in range(col)]
        for b in range(B):
            table[slots[s * B + b]] = torch.tensor(shared + [perm.pop() for _ in range(extra)], dtype=torch.int32)
    make = lambda row: (torch.randint(0, 255, (n_layer, n_pages, n_kv, PAGE, row), generator=g, dtype=torch.uint8)  # noqa: E731
                        if dtype == torch.uint8 else torch.randn(n_layer, n_pages, n_kv, PAGE, row, generator=g).to(dtype))
    return make(k_row), make(v_row), table, slots.int()


def _follow(k, v, table, slots, parent, held):
    """The same on the CPU, a beam after the other, out of copies of the old state."""
    G, B = parent.shape
    new, old = table.clone(), (k.clone(), v.clone())
    for g in range(G):
        col, part = int(held[g]) // PAGE, int(held[g]) % PAGE
        mine = [int(s) for s in slots[g * B:(g + 1) * B]]
        ps = parent[g].tolist()
        bare = [b for b in range(B) if b not in ps]
        for i, p in enumerate(ps):
            new[mine[i], :col] = table[mine[p], :col]
            if part:
                src = int(table[mine[p], col])
                if p in ps[:i]:
                    dst = int(table[mine[bare.pop(0)], col])
                    for pool, was in zip((k, v), old):
                        pool[:, dst, :, :part] = was[:, src, :, :part]
                    src = dst
                new[mine[i], col] = src
    return new


@gpu
@pytest.mark.parametrize("held", [0, 1, 63, 64, 65, 191, 200])
@pytest.mark.parametrize("rows", [(64, 64, torch.float16), (68, 68, torch.uint8), (136, 136, torch.uint8), (576, 0, torch.float16),
                                  (128, 128, torch.bfloat16)])
def test_states_follow_their_beams(held, rows):
    from bloomery_b200.ops.beam import beam_reorder
    for seed, (G, B) in enumerate([(1, 1), (1, 2), (3, 5), (2, 33), (1, 64)]):
        k, v, table, slots = _states(G, B, held, k_row=rows[0], v_row=rows[1], dtype=rows[2], seed=seed)
        parent = torch.randint(0, B, (G, B), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)
        if seed == 3:
            parent[0] = 7                              # everybody follows one beam
        at = torch.full((G,), held, dtype=torch.int32)
        on = [t.to(DEV) for t in (k, v, table, slots, parent, at)]
        new = on[2].clone()
        fault = torch.full((1,), -1, dtype=torch.int32, device=DEV)
        for _ in range(2):                             # the old state leads to the new one however often it is asked
            beam_reorder(on[0], on[1], on[2], new, on[3], on[4], on[5], fault)
        want = _follow(k, v, table, slots, parent, at)
        assert torch.equal(new.cpu(), want) and torch.equal(on[2].cpu(), table)
        assert torch.equal(on[0].cpu().view(torch.uint8), k.view(torch.uint8))
        assert torch.equal(on[1].cpu().view(torch.uint8), v.view(torch.uint8))
        assert int(fault) == -1


@gpu
def test_searches_of_unequal_length():
    from bloomery_b200.ops.beam import beam_reorder
    k, v, table, slots = _states(3, 4, 128, seed=9, extra=3)
    parent = torch.tensor([[1, 1, 3, 0], [0, 0, 0, 0], [3, 2, 1, 0]], dtype=torch.int32)
    held = torch.tensor([130, 191, 128], dtype=torch.int32)
    on = [t.to(DEV) for t in (k, v, table, slots, parent, held)]
    new = on[2].clone()
    beam_reorder(on[0], on[1], on[2], new, *on[3:])
    assert torch.equal(new.cpu(), _follow(k, v, table, slots, parent, held))
    assert torch.equal(on[0].cpu(), k) and torch.equal(on[1].cpu(), v)


@gpu
@pytest.mark.parametrize("what", ["parent", "slot", "held", "page"])
def test_what_is_out_of_range_moves_nothing_and_raises_the_fault(what):
    from bloomery_b200.ops.beam import beam_reorder
    k, v, table, slots = _states(2, 4, 100, seed=10)
    parent = torch.tensor([[1, 1, 3, 0], [0, 1, 2, 3]], dtype=torch.int32)
    held = torch.tensor([100, 100], dtype=torch.int32)
    if what == "parent":
        parent[0, 2] = 4
    elif what == "slot":
        slots[1] = table.shape[0]
    elif what == "held":
        held[0] = table.shape[1] * PAGE + 1
    else:
        table[slots[2], 1] = k.shape[1]                # the childless beam's page, where the second child of 1 would go
    on = [t.to(DEV) for t in (k, v, table, slots, parent, held)]
    new = on[2].clone()
    fault = torch.full((1,), -1, dtype=torch.int32, device=DEV)
    beam_reorder(on[0], on[1], on[2], new, on[3], on[4], on[5], fault)
    assert int(fault) == (6 if what == "page" else 9)
    assert torch.equal(on[0].cpu(), k) and torch.equal(on[1].cpu(), v)
    if what != "page":
        assert torch.equal(new.cpu(), table)


# ---- refusals (CPU) -------------------------------------------------------------------------------------------------
def _select(**kw):
    from bloomery_b200.ops.beam import BeamScratch, beam_select
    i32 = dict(dtype=torch.int32)
    a = dict(logits=torch.zeros(6, 10), scores=torch.zeros(2, 3), scratch=BeamScratch(2, 3, 10, "cpu"), parent=torch.zeros(2, 3, **i32),
             token=torch.zeros(2, 3, **i32), out_scores=torch.zeros(2, 3))
    a.update(kw)
    beam_select(**a)


@pytest.mark.parametrize("kw", [
    dict(logits=torch.zeros(6, 10).bfloat16()), dict(logits=torch.zeros(5, 10)), dict(logits=torch.zeros(6, 11)),
    dict(logits=torch.zeros(10, 6).t()), dict(scores=torch.zeros(2, 4)), dict(parent=torch.zeros(2, 3)),
    dict(done=torch.zeros(2, 3, dtype=torch.int32)), dict(eos=10), dict(alpha=1.0), dict(out_lengths=torch.zeros(2, 3, dtype=torch.int32)),
    dict(lengths=torch.zeros(2, 3, dtype=torch.int64))])
def test_arguments_of_a_choice_are_checked(kw):
    with pytest.raises(ValueError):
        _select(**kw)


def test_searches_wider_than_the_limit_are_refused():
    from bloomery_b200.ops.beam import MAX_BEAMS, BeamScratch
    for beams in (0, MAX_BEAMS + 1):
        with pytest.raises(ValueError):
            BeamScratch(1, beams, 10, "cpu")


def _reorder(**kw):
    from bloomery_b200.ops.beam import beam_reorder
    k, v, table, slots = _states(1, 2, 10)
    a = dict(k=k, v=v, table=table, table_out=table.clone(), slots=slots, parent=torch.zeros(1, 2, dtype=torch.int32),
             held=torch.zeros(1, dtype=torch.int32))
    a.update({n: f(a) for n, f in kw.items()})
    beam_reorder(**a)


@pytest.mark.parametrize("kw", [
    dict(table_out=lambda a: a["table"]), dict(table=lambda a: a["table"].long()), dict(table_out=lambda a: a["table"][:, :1].contiguous()),
    dict(k=lambda a: a["k"][:, :, :, :32].contiguous()), dict(v=lambda a: a["v"].transpose(1, 2)), dict(held=lambda a: a["slots"]),
    dict(slots=lambda a: a["slots"][:1]), dict(parent=lambda a: torch.zeros(1, 2))])
def test_arguments_of_a_reordering_are_checked(kw):
    with pytest.raises(ValueError):
        _reorder(**kw)
