"""Shared-prefix attention where it once read, rounded or reported what it should not have."""
import pytest
import torch

from test_gpu_prefix_attention import DEV, Case

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("rows", [5, 40])                  # schedules of one warp's registers and of the whole block
@pytest.mark.parametrize("q8", [False, True])
def test_a_prefix_longer_than_a_table_row_ends_with_the_row(rows, q8):
    """Lengths that a captured call finds on the card: every key of these rows is in their table, and nothing behind it is read."""
    c = Case([(192, [1 + i * 191 // (rows - 1) for i in range(rows)])], 32, 4, 128, q8, seed=21, max_pages=3)
    c.table = c.table.contiguous()
    plan = c.plan()
    first = c.run(plan)
    c.check(first)
    out = torch.zeros_like(first)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            c.run(plan, out)
    with pytest.raises(ValueError):
        plan.set_prefix([640])
    plan.max_pages = 1 << 24                                # past the host's check, as another holder of the lengths could
    for longer in (640, 1 << 28):
        plan.set_prefix([longer])
        torch.cuda.synchronize()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    assert int(c.fault) == -1


@gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("n_q,n_kv,head", [(32, 4, 128), (8, 2, 64)])
@pytest.mark.parametrize("gap", [5.0, 12.0, 14.5, 16.3])
@pytest.mark.parametrize("first", [True, False])
def test_what_lies_far_below_the_largest_score_keeps_its_bits(gap, first, n_q, n_kv, head, q8):
    """One key takes nearly all of the weight and its value is zero: the output is the sum over all others, which score ``gap``
    nats less, all the same.  The band is that of any other case: rounded probabilities are off by 2^-11 of themselves.  No
    value is negative, so that what all of the probabilities lose is not lost among values that cancel; there are groups enough
    that a processor has most of a row's pages behind one maximum."""
    from test_gpu_prefix_attention import _q8
    c = Case([(512, [520])] * (40 * 4 // n_kv), n_q, n_kv, head, q8, seed=22)
    G = n_q // n_kv
    for r, (_, ids) in enumerate(c.rows):
        top, at = (ids[0], 3) if first else (ids[-1], 5)
        q = c.q[r].double().view(n_kv, G, head)
        k0 = (torch.linalg.pinv(q) @ torch.full((n_kv, G, 1), gap, dtype=torch.float64, device=DEV)).squeeze(-1)   # q . k0 = gap
        for page in ids:
            n = c.keys[page].shape[1]
            c.keys[page].zero_()
            c.k[page, :, :n] = 0
            c.values[page].abs_()
            if q8:
                codes = c.v[page, :, :n, head // 16:]
                codes.copy_(codes.contiguous().view(torch.int8).abs().view(torch.uint8))
            else:
                c.v[page, :, :n].abs_()
        if q8:
            d, codes = _q8(k0.float())
            c.k[top, :, at] = torch.cat([d.view(torch.uint8), codes.view(torch.uint8)], -1)
            c.keys[top][:, at] = codes.double() * d.double().repeat_interleave(32, -1)
        else:
            c.k[top, :, at] = k0.half()
            c.keys[top][:, at] = k0.half().double()
        c.v[top, :, at] = 0
        c.values[top][:, at] = 0
    c.check(c.run())


@gpu
@pytest.mark.parametrize("n_q,n_kv,head", [(32, 4, 128), (8, 2, 64)])
@pytest.mark.parametrize("at", [3, 130])                   # in the shared pages, in a row's own
def test_q8_0_keys_past_the_range_of_f16(at, n_q, n_kv, head):
    """-127 * 520 is no f16, the sum with 127 * 508 and 3 * 508 is 0: a key like all others, not one of weight 0.  Scores are exact
    and equal, so that the output is the mean of the values, summed in 32 bits and rounded to 8."""
    c = Case([(128, [140, 150])], n_q, n_kv, head, True, seed=23)
    c.q.zero_()
    c.q[:, :, [0, 32, 33]] = 1.0
    for pages in (c.rows[0][1], c.rows[1][1]):
        for page in pages:
            c.keys[page].zero_()
            c.k[page, :, :c.keys[page].shape[1]] = 0
    page, i = c.rows[0][1][at // 64], at % 64
    d = torch.zeros(n_kv, head // 32, dtype=torch.float16, device=DEV)
    d[:, 0], d[:, 1] = 520.0, 508.0
    codes = torch.zeros(n_kv, head, dtype=torch.int8, device=DEV)
    codes[:, 0], codes[:, 32], codes[:, 33] = -127, 127, 3
    c.k[page, :, i] = torch.cat([d.view(torch.uint8), codes.view(torch.uint8)], -1)
    c.keys[page][:, i] = codes.double() * d.double().repeat_interleave(32, -1)
    wide = torch.full((n_kv, head), 100, dtype=torch.int8, device=DEV)          # a value that is missed if the key is
    c.v[page, :, i] = torch.cat([torch.ones_like(d).view(torch.uint8), wide.view(torch.uint8)], -1)
    c.values[page][:, i] = 100.0
    out = c.run()
    want, _ = c.reference()
    assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4).all()
    assert int(c.fault) == -1
