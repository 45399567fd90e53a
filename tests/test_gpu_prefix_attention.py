"""Attention of rows that share a prefix against the same sums in 64 bits, over f16 and q8_0 caches whose every other position
holds NaN: rows of one position, of none of their own, that end inside the prefix, dead rows, odd groups and odd pages."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
DEV = "cuda:0"
PAGE = 64
NAN = float("nan")


def _q8(x):
    b = x.unflatten(-1, (-1, 32))
    d = (b.abs().amax(-1) / 127).half()
    c = (b / d.float().clamp_min(1e-8).unsqueeze(-1)).round().clamp(-127, 127)
    return d, c.to(torch.int8).flatten(-2)


class Case:
    """``rows``: for each group (prefix, [positions of each row, None: dead])."""

    def __init__(self, groups, n_q, n_kv, head, q8=False, seed=0, n_pages=None, q_scale=1.4, max_pages=None, q_powers=False):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.n_q, self.n_kv, self.head, self.q8 = n_q, n_kv, head, q8
        rows = [(gi, p, n) for gi, (p, ns) in enumerate(groups) for n in ns]
        self.M = len(rows)
        longest = max([p for p, _ in groups] + [n or 0 for _, _, n in rows])
        max_pages = max_pages or (longest + PAGE - 1) // PAGE + 1
        total = sum(p // PAGE for p, _ in groups) + sum(max(0, (n or 0) - p + PAGE - 1) // PAGE + 1 for _, p, n in rows)
        n_pages = n_pages or total + 3
        free = [n_pages - 1 - i for i in torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()]
        table = torch.full((self.M + 2, max_pages), -1, dtype=torch.int32)
        seqs = torch.randperm(self.M + 2, generator=torch.Generator().manual_seed(seed + 1))[:self.M].tolist()
        shared = [[free.pop() for _ in range(p // PAGE)] for p, _ in groups]
        width = head // 32 * 34 if q8 else head
        self.k = torch.empty(n_pages, n_kv, PAGE, width, dtype=torch.uint8 if q8 else torch.float16, device=DEV)
        self.v = torch.empty_like(self.k)
        for pg in sorted(set(range(n_pages - total, n_pages)) | {0}):
            for c in (self.k, self.v):
                c[pg] = 255 if q8 else NAN             # an f16 of 0xffff is NaN
        self.keys, self.values = {}, {}               # page -> fp64 [n_kv, 64, head]

        def fill(page, n):
            for c, kept in ((self.k, self.keys), (self.v, self.values)):
                x = torch.randn(n_kv, n, head, generator=g, device=DEV)
                if q8:
                    d, codes = _q8(x)
                    c[page, :, :n] = torch.cat([d.view(torch.uint8), codes.view(torch.uint8)], -1)
                    x = codes.double() * d.double().repeat_interleave(32, -1)
                else:
                    c[page, :, :n] = x.half()
                    x = x.half().double()
                kept[page] = x
        for (p, ns), pages in zip(groups, shared):
            for pg in pages:
                fill(pg, PAGE)
        self.rows = []
        pos, seq = [], []
        for r, (gi, p, n) in enumerate(rows):
            ids = list(shared[gi])
            for at in range(p, n or 0, PAGE):
                pg = free.pop()
                fill(pg, min(PAGE, n - at))
                ids.append(pg)
            table[seqs[r], :len(ids)] = torch.tensor(ids, dtype=torch.int32)
            pos.append((n or 1) - 1)
            seq.append(-1 if n is None else seqs[r])
            self.rows.append((n, ids))
        self.q = torch.randn(self.M, n_q, head, generator=g, device=DEV) * (q_scale / math.sqrt(head))
        if q_powers:                                   # rows of very different size: none may lose its bits or run over
            self.q *= (2.0 ** torch.linspace(-24, 3, self.M, device=DEV)).view(-1, 1, 1)
        self.pos = torch.tensor(pos, dtype=torch.int32, device=DEV)
        self.seq = torch.tensor(seq, dtype=torch.int32, device=DEV)
        self.table = table.to(DEV)
        self.group_rows, self.prefix = [len(ns) for _, ns in groups], [p for p, _ in groups]
        self.fault = torch.full((1,), -1, dtype=torch.int32, device=DEV)

    def plan(self):
        from bloomery_b200.ops.prefix import PrefixPlan
        return PrefixPlan(self.group_rows, self.prefix, self.n_q, self.n_kv, self.head, DEV)

    def run(self, plan=None, out=None):
        from bloomery_b200.ops.prefix import prefix_attention
        out = torch.full((self.M, self.n_q * self.head), 7.0, dtype=torch.bfloat16, device=DEV) if out is None else out
        prefix_attention(self.q, self.k, self.v, self.pos, self.seq, self.table, plan or self.plan(), out, self.fault, 3)
        return out

    def reference(self):
        """Rows in 64 bits and how far 16-bit operands may be off: queries, keys (q8_0) and probabilities are rounded to 11
        bits each.  A score's error is a sum of independent roundings, within 6 standard deviations of 2^-12 |q k| (root
        of the sum of squares) for each rounded operand; probabilities and values (q8_0) add 2^-11 at most; an error of d in
        every probability moves the output by 2 d sum p |v| at most (numerator and sum); the output is rounded to 8 bits."""
        out = torch.zeros(self.M, self.n_q, self.head, dtype=torch.float64, device=DEV)
        tol = torch.zeros_like(out)
        G = self.n_q // self.n_kv
        for r, (n, ids) in enumerate(self.rows):
            if n is None:
                continue
            k = torch.cat([self.keys[p] for p in ids[:(n + PAGE - 1) // PAGE]], 1)[:, :n]
            v = torch.cat([self.values[p] for p in ids[:(n + PAGE - 1) // PAGE]], 1)[:, :n]
            q = self.q[r].double().view(self.n_kv, G, self.head)
            p = torch.softmax(q @ k.transpose(1, 2), -1)
            o = p @ v
            off = 6 * 2.0 ** -12 * (q.square() @ k.square().transpose(1, 2)).sqrt().amax(-1, keepdim=True) * (2 if self.q8 else 1) \
                + 2.0 ** -11 * (2 if self.q8 else 1)
            out[r] = o.reshape(self.n_q, self.head)
            tol[r] = (2.0 ** -8 * o.abs() + 2 * off * (p @ v.abs())).reshape(self.n_q, self.head) + 1e-6
        return out.view(self.M, -1), tol.view(self.M, -1)

    def check(self, out):
        want, tol = self.reference()
        over = (out.double() - want).abs() - tol
        assert not torch.isnan(out).any(), "NaN from a position that no row has"
        assert over.max().item() <= 0, (over.max().item(), over.argmax().item() // out.shape[1])
        assert int(self.fault) == -1


SHAPES = [(32, 4, 128), (8, 2, 64), (16, 1, 128), (6, 6, 64), (10, 2, 128), (24, 8, 64), (9, 3, 128)]
GROUPS = {
    "one row, one position": [(0, [1])],
    "one row, a page and one": [(64, [65])],
    "two rows, nothing of their own": [(64, [64, 64])],
    "a row in the prefix": [(192, [1, 63, 64, 65, 130, 192, 193, 320])],
    "dead rows, leading and all": [(128, [None, 140, None, 200]), (64, [None, None]), (0, [None]), (0, [17])],
    "odd groups": [(64, [70] * 3), (320, [321, 340, 383, 384, 385]), (0, [5, 64, 129]), (960, [1000])],
    "tails of several pages": [(256, [256 + i * 37 for i in range(17)])],
}


@gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("n_q,n_kv,head", SHAPES)
@pytest.mark.parametrize("name", list(GROUPS))
def test_rows_match_their_sums_in_64_bits(name, n_q, n_kv, head, q8):
    c = Case(GROUPS[name], n_q, n_kv, head, q8, seed=n_q + head)
    c.check(c.run())


@gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("n_q,n_kv,head,rows,prefix,tail", [(32, 4, 128, 64, 4096, 300), (64, 4, 128, 40, 2112, 5), (8, 2, 64, 33, 8256, 70),
                                                            (8, 2, 64, 200, 640, 30)])
def test_many_rows_behind_a_long_prefix(n_q, n_kv, head, rows, prefix, tail, q8):
    c = Case([(prefix, [prefix + 1 + i * (tail - 1) // (rows - 1) for i in range(rows)])], n_q, n_kv, head, q8, seed=rows)
    c.check(c.run())


@gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("n_q,n_kv,head,rows,prefix,tail", [(32, 4, 128, 64, 16448, 300), (8, 2, 64, 33, 39936, 70), (32, 4, 128, 5, 20480, 140),
                                                            (48, 8, 128, 7, 16384, 1)])
def test_prefixes_that_take_the_long_form(n_q, n_kv, head, rows, prefix, tail, q8):
    """Four tiles of shared keys or more for every processor."""
    c = Case([(prefix, [prefix + 1 + i * (tail - 1) // (rows - 1) for i in range(rows)]), (64, [70])], n_q, n_kv, head, q8, seed=rows)
    c.check(c.run())


@gpu
@pytest.mark.parametrize("q8", [False, True])
def test_tails_longer_than_the_prefix(q8):
    c = Case([(64, [3000, 70, 2500]), (128, [129, 1999])], 32, 4, 128, q8, seed=5)
    c.check(c.run())


@gpu
@pytest.mark.parametrize("scale", [1e-6, 40.0])
def test_scores_from_flat_to_peaked(scale):
    """A scale of 40 makes scores of some hundreds: one key takes all, and the running maximum moves often."""
    c = Case([(512, [512 + i for i in range(1, 12)])], 32, 4, 128, seed=11, q_scale=scale)
    c.check(c.run())


@gpu
def test_rows_of_very_different_size_keep_their_bits():
    c = Case([(256, [256 + i for i in range(1, 28)])], 32, 4, 128, seed=12, q_powers=True)
    c.check(c.run())


@gpu
def test_pages_behind_the_first_four_gigabytes():
    """70,000 pages of 4 heads of 128: 4.6 GB a cache, offsets past 32 bits; only the last pages are touched."""
    c = Case([(192, [200, 300])], 32, 4, 128, seed=13, n_pages=70000)
    c.check(c.run())


@gpu
def test_calls_repeat_bit_for_bit_and_follow_the_lengths():
    """One plan for a growing search: the same call again gives the same bits, other lengths need no other plan, and a
    captured call reads the lengths of its replay."""
    c = Case([(640, [640 + 200] * 9), (64, [300, 100])], 32, 4, 128, seed=14)
    plan = c.plan()
    first = c.run(plan)
    assert torch.equal(first, c.run(plan))
    c.check(first)
    full = list(c.rows)
    c.rows = [(n - 60 - r, ids) for r, (n, ids) in enumerate(full)]
    c.pos -= torch.arange(60, 60 + c.M, dtype=torch.int32, device=DEV)
    c.check(c.run(plan))
    out = torch.zeros_like(first)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c.run(plan, out)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            c.run(plan, out)
    torch.cuda.synchronize()
    c.rows = full
    c.pos += torch.arange(60, 60 + c.M, dtype=torch.int32, device=DEV)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)


@gpu
def test_rows_that_cannot_be_served_get_nan_and_a_fault():
    rows = [300, 310, 320, 330]
    c = Case([(256, rows)], 32, 4, 128, seed=15)
    want, _ = c.reference()
    for change in ("no keys", "past the table", "page", "slot"):
        c = Case([(256, rows)], 32, 4, 128, seed=15)
        if change == "no keys":
            c.pos[2] = -1
        elif change == "past the table":
            c.pos[2] = c.table.shape[1] * PAGE
        elif change == "slot":
            c.seq[2] = c.table.shape[0]
        else:
            c.table[c.seq[2].long(), 4] = c.k.shape[0]
        out = c.run()
        assert torch.isnan(out[2]).all(), change
        assert (out[[0, 1, 3]].double() - want[[0, 1, 3]]).abs().max() < 0.05, change
        assert int(c.fault) == (3 << 8 | (6 if change == "page" else 5)), change


@gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("bad", [NAN, math.inf, -math.inf])
def test_what_one_row_holds_does_not_reach_another(bad, q8):
    """Values and keys that are not finite, in one row's own pages and behind the end of a row inside the prefix."""
    c = Case([(128, [100, 200, 150, 128, 260])], 32, 4, 128, q8, seed=16)
    c.check(c.run())
    want, tol = c.reference()
    own, shared = c.rows[1][1][2], c.rows[1][1][1]
    raw = torch.tensor([bad], dtype=torch.float16, device=DEV).view(torch.uint8) if q8 else bad
    for cache in (c.k, c.v):
        if q8:
            cache[own, :, 3, :2] = raw
            cache[own, :, 3, 8:40] = 1
        else:
            cache[own, :, 3] = raw
    out = c.run()
    fine = [0, 2, 3, 4]
    assert ((out.double() - want).abs() - tol)[fine].max() <= 0
    assert not torch.isfinite(out[1]).all()
    if q8:
        c.v[shared, :, 50, :2] = raw
        c.v[shared, :, 50, 8:40] = 1
    else:
        c.v[shared, :, 50] = raw                       # position 114: behind row 0's end, seen by all others
    out = c.run()
    assert ((out.double() - want).abs() - tol)[0].max() <= 0
    assert not torch.isfinite(out[2]).all()


def _cpu_call(**kw):
    from bloomery_b200.ops.prefix import PrefixPlan, prefix_attention
    plan = PrefixPlan([2], [64], 4, 2, 64, "cpu")
    a = dict(q=torch.zeros(2, 4, 64), k_cache=torch.zeros(3, 2, 64, 64, dtype=torch.float16),
             v_cache=torch.zeros(3, 2, 64, 64, dtype=torch.float16), row_pos=torch.zeros(2, dtype=torch.int32),
             row_seq=torch.zeros(2, dtype=torch.int32), block_table=torch.zeros(2, 4, dtype=torch.int32), plan=plan,
             out=torch.zeros(2, 256, dtype=torch.bfloat16))
    a.update(kw)
    return prefix_attention(**a)


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(2, 4, 64, dtype=torch.float16)), dict(q=torch.zeros(3, 4, 64)), dict(q=torch.zeros(2, 64, 4).transpose(1, 2)),
    dict(k_cache=torch.zeros(3, 2, 32, 64, dtype=torch.float16)), dict(v_cache=torch.zeros(4, 2, 64, 64, dtype=torch.float16)),
    dict(k_cache=torch.zeros(3, 2, 64, 64, dtype=torch.uint8)), dict(v_cache=torch.zeros(3, 2, 64, 68, dtype=torch.uint8)),
    dict(out=torch.zeros(2, 256)), dict(row_pos=torch.zeros(2, dtype=torch.int64)), dict(row_seq=torch.zeros(1, dtype=torch.int32)),
    dict(block_table=torch.zeros(4, dtype=torch.int32)), dict(block_table=torch.zeros(2, 0, dtype=torch.int32))])
def test_arguments_are_checked(kw):
    with pytest.raises(ValueError):
        _cpu_call(**kw)


@pytest.mark.parametrize("args", [([], [], 4, 2, 64), ([2], [64, 0], 4, 2, 64), ([0], [64], 4, 2, 64), ([2], [63], 4, 2, 64),
                                  ([2], [-64], 4, 2, 64), ([2], [64], 4, 3, 64), ([2], [64], 4, 2, 96), ([2], [64], 34, 2, 64),
                                  ([1025], [64], 4, 2, 64)])
def test_plans_are_checked(args):
    from bloomery_b200.ops.prefix import PrefixPlan
    with pytest.raises(ValueError):
        PrefixPlan(*args, "cpu")
