"""The calls by which the operators of beam search are measured: attention of rows that share a prefix, the choice of the
next beams, and the cached states that follow their beams.

A server that keeps several answers to one prompt (the beams of a search, the samples of one request, chats behind one
system prompt) asks these of one layer, one pass or one model.  Shapes are the framework's own: the Qwen3-30B-A3B layer (32
query heads over 4 key heads of 128, 151,936 ids, 48 layers), the 235B one (64 over 4) and the tiny one (8 over 2 of 64, 32,000
ids, 4 layers); caches are its pages of 64 positions in f16 or in q8_0 rows.
"""
import math
import random

import torch

own = False

PAGE = 64
MAX_PAGES = 640                 # pages that a slot's table row holds: the 40,960 positions that the models were trained for
LAYERS = {"30b": (48, 32, 4, 128, 151936), "235b": (94, 64, 4, 128, 151936), "tiny": (4, 8, 2, 64, 32000)}
APART = 5e-5                    # candidates around the last place lie further apart than 32-bit sums of their size round


def listed():
    return [
        # the smallest call: four beams a few ids behind a short prompt; launches and latency are all it costs
        attention("4 beams behind 512", "30b", 4, 1, 512, 12),
        # eight answers to one question over a page of context, half of them long
        attention("8 answers behind 2048", "30b", 8, 1, 2048, 400),
        # a bucket of 24 chats behind one system prompt, each with a conversation of its own; three rows fill the bucket
        attention("21 chats behind 4096", "30b", 21, 1, 4096, 1100, dead=3),
        # three documents with their readers, keys and values in q8_0 rows
        attention("24 readers of 3 documents, q8_0", "30b", 24, 3, 9024, 300, cache="q8_0"),
        # odd everywhere: heads of 64, five prompts of unequal length, 13 rows
        attention("13 rows of 5 prompts, tiny", "tiny", 13, 5, 960, 70),
        # the largest call: 64 beams over a long document
        attention("64 beams behind 32768", "30b", 64, 1, 32768, 256),
        # one search of four beams; most of it latency
        selection("the best of 4 beams", "30b", 1, 4),
        # odd: three searches of five beams over a small vocabulary, some finished, ranked by length
        selection("the best of 3 searches of 5, some finished", "tiny", 3, 5, finished=2, alpha=0.6),
        # a full bucket: eight searches of eight beams
        selection("the best of 8 searches of 8", "30b", 8, 8),
        # wide searches next to each other
        selection("the best of 16 searches of 16, by length", "30b", 16, 16, finished=3, alpha=1.0),
        # two of four beams move, few positions are in the page
        reorder("states of 4 beams, tiny", "tiny", 1, 4, 2, 137),
        # a full bucket of the 30B shape: half of the beams follow another one
        reorder("states of 8 searches of 8", "30b", 8, 8, 4, 240),
    ]


def attention(name, model, rows, groups, prefix, tail, cache="f16", dead=0):
    return {"name": name, "op": "attention", "model": model, "rows": rows, "groups": groups, "prefix": prefix, "tail": tail,
            "cache": cache, "dead": dead}


def selection(name, model, groups, beams, finished=0, alpha=0.0):
    return {"name": name, "op": "select", "model": model, "groups": groups, "beams": beams, "finished": finished, "alpha": alpha}


def reorder(name, model, groups, beams, moved, held):
    return {"name": name, "op": "reorder", "model": model, "groups": groups, "beams": beams, "moved": moved, "held": held}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Attention of 1 to 64 rows in 1 to 5 groups behind 64 to 32,768 shared positions, up to 2,000 of their own; selections of
    1 to 16 searches of 2 to 16 beams; reorderings of 1 to 8 searches of 2 to 8 beams."""
    kind = rng.choice(["attention", "attention", "select", "reorder"])
    while True:
        model = rng.choice(["30b", "30b", "30b", "235b", "tiny"])
        if kind == "attention":
            rows = _log(rng, 1, 64)
            case = attention("", model, rows, min(rows, rng.choice([1, 1, 1, 2, 3, 5])), PAGE * _log(rng, 1, 512),
                             _log(rng, 1, 2000), rng.choice(["f16", "f16", "q8_0"]), rng.choice([0, 0, 1, 3]))
        elif kind == "select":
            beams = _log(rng, 2, 16)
            case = selection("", "tiny" if model == "tiny" else "30b", _log(rng, 1, 16), beams, rng.choice([0, 0, beams // 3]),
                             rng.choice([0.0, 0.6, 1.0]))
        else:
            beams = rng.randint(2, 8)
            case = reorder("", "tiny" if model == "tiny" else "30b", rng.randint(1, 8), beams, rng.randint(0, beams - 1),
                           rng.randint(1, 400))
        cost = work(case)
        if all(cost[k] <= max(work(c)[k] for c in listed() if c["op"] == kind) for k in cost):
            del case["name"]
            return case


# ---- what a case is made of -----------------------------------------------------------------------------------------
def _split(n, parts):
    """``n`` things in ``parts`` unequal shares of one at least."""
    w = [2 + i % 3 for i in range(parts)]
    got = [1 + (n - parts) * x // sum(w) for x in w]
    got[0] += n - sum(got)
    return got


def _lengths(case):
    """Rows and shared positions of each group, own positions of each row (in the order before the seed mixes them)."""
    rows, groups = case["rows"], case["groups"]
    prefix = [max(1, case["prefix"] // PAGE * (groups - g) // groups) * PAGE for g in range(groups)]
    tail = [1 + (case["tail"] - 1) * i // max(1, rows - 1) for i in range(rows)]
    return _split(rows, groups), prefix, tail


def work(case):
    n_layer, n_q, n_kv, head, vocab = LAYERS[case["model"]]
    if case["op"] == "attention":
        group_rows, prefix, tail = _lengths(case)
        row = head * 2 if case["cache"] == "f16" else head // 32 * 34
        keys = sum(r * n for r, n in zip(group_rows, prefix)) + sum(tail)
        return {"bytes": 2 * n_kv * row * (sum(prefix) + sum(tail)) + (case["rows"] * 4 + (case["rows"] + case["dead"]) * 2) * n_q * head,
                "flops": 4 * n_q * head * keys}
    if case["op"] == "select":
        rows = case["groups"] * case["beams"]
        return {"bytes": 4 * vocab * case["groups"] * (case["beams"] - case["finished"]) + 28 * rows, "flops": 0}
    part = case["held"] % PAGE
    return {"bytes": 2 * case["groups"] * case["moved"] * n_layer * n_kv * part * head * 2 * 2 + 8 * case["groups"] * case["beams"] * MAX_PAGES,
            "flops": 0}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng = random.Random(seed)
    with torch.no_grad():
        return {"attention": _prepare_attention, "select": _prepare_select, "reorder": _prepare_reorder}[case["op"]](case, gen, rng)


def run(state):
    with torch.no_grad():
        return {"attention": _run_attention, "select": _run_select, "reorder": _run_reorder}[state["case"]["op"]](state)


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = kept
    with torch.no_grad():
        return {"attention": _exact_attention, "select": _exact_select, "reorder": lambda s: None}[case["op"]](state)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- attention of rows that share a prefix --------------------------------------------------------------------------
def _q8_rows(x):
    """q8_0 rows of the last dimension: f16 scales of its blocks of 32, then the codes."""
    blocks = x.unflatten(-1, (-1, 32))
    d = (blocks.abs().amax(-1) / 127).half()
    codes = (blocks / d.float().clamp_min(1e-8).unsqueeze(-1)).round().clamp(-127, 127).to(torch.int8)
    return torch.cat([d.contiguous().view(torch.uint8), codes.flatten(-2).view(torch.uint8)], -1).contiguous()


def _prepare_attention(case, gen, rng):
    _, n_q, n_kv, head, _ = LAYERS[case["model"]]
    group_rows, prefix, tail = _lengths(case)
    rows, dead = case["rows"], case["dead"]
    rng.shuffle(tail)
    need = [[(n + PAGE - 1) // PAGE for n in tail[sum(group_rows[:g]):sum(group_rows[:g + 1])]] for g in range(len(prefix))]
    n_pages = sum(prefix) // PAGE + sum(map(sum, need)) + 8
    free = list(range(n_pages))
    rng.shuffle(free)
    slots = list(range(rows))
    rng.shuffle(slots)
    table = torch.full((rows, MAX_PAGES), -1, dtype=torch.int32)
    row_pos, row = [], 0
    for g, own_pages in enumerate(need):
        shared = [free.pop() for _ in range(prefix[g] // PAGE)]
        for pages in own_pages:
            ids = shared + [free.pop() for _ in range(pages)]
            table[slots[row], :len(ids)] = torch.tensor(ids, dtype=torch.int32)
            row_pos.append(prefix[g] + tail[row] - 1)
            row += 1
    # keys with a direction that queries share and a few positions hold more of, as trained heads have them
    u = torch.randn(n_kv, 1, head, generator=gen, device="cuda")
    k = torch.randn(n_pages, n_kv, PAGE, head, generator=gen, device="cuda")
    k += u * (torch.rand(n_pages, n_kv, PAGE, 1, generator=gen, device="cuda") < 0.02) * 0.5
    v = torch.randn(n_pages, n_kv, PAGE, head, generator=gen, device="cuda") + 0.25 * u
    q = torch.randn(rows + dead, n_q, head, generator=gen, device="cuda") + 0.5 * u[:, 0].repeat_interleave(n_q // n_kv, 0)
    pack = _q8_rows if case["cache"] == "q8_0" else torch.Tensor.half
    state = {"case": case, "q": q * (1.4 / math.sqrt(head)), "k": pack(k), "v": pack(v), "row_pos": _ints(row_pos + [0] * dead),
             "row_seq": _ints(slots + [-1] * dead), "table": table.cuda()}
    if own:
        from bloomery_b200.ops.prefix import PrefixPlan
        # the rows that fill a bucket are a group without a prefix
        state["plan"] = PrefixPlan(group_rows + [dead] * (dead > 0), prefix + [0] * (dead > 0), n_q, n_kv, head, "cuda")
        state["out"] = torch.empty(rows + dead, n_q * head, dtype=torch.bfloat16, device="cuda")
    return state


def _run_attention(s):
    if own:
        from bloomery_b200.ops.prefix import prefix_attention
        prefix_attention(s["q"], s["k"], s["v"], s["row_pos"], s["row_seq"], s["table"], s["plan"], s["out"])
        return s["out"]
    case = s["case"]
    _, n_q, n_kv, head, _ = LAYERS[case["model"]]
    group_rows, prefix, _ = _lengths(case)
    group = n_q // n_kv
    q = s["q"].view(-1, n_kv, group, head)
    out = torch.zeros_like(q)
    values = _f16_rows if case["cache"] == "f16" else _q8_values
    row = 0
    for n_rows, n in zip(group_rows, prefix):
        rows = slice(row, row + n_rows)
        seq, pos = s["row_seq"][rows].long(), s["row_pos"][rows].long()
        mine = s["table"][seq]
        shared = mine[0, :n // PAGE].long()
        k, v = (values(x[shared]).transpose(0, 1).reshape(n_kv, n, head) for x in (s["k"], s["v"]))
        ahead = torch.einsum("rhgd,hnd->rhgn", q[rows], k)
        # every row's own keys, up to the longest of the group
        pages = (case["tail"] + PAGE - 1) // PAGE
        ids = mine[:, n // PAGE:n // PAGE + pages].long().clamp_min(0)
        ko, vo = (values(x[ids]).transpose(1, 2).reshape(n_rows, n_kv, pages * PAGE, head) for x in (s["k"], s["v"]))
        behind = torch.einsum("rhgd,rhnd->rhgn", q[rows], ko)
        there = n + torch.arange(pages * PAGE, device="cuda") <= pos[:, None]
        behind = behind.masked_fill(~there[:, None, None], -math.inf)
        top = torch.maximum(ahead.amax(-1), behind.amax(-1)).unsqueeze(-1)
        pa, pb = torch.exp(ahead - top), torch.exp(behind - top)
        out[rows] = torch.einsum("rhgn,hnd->rhgd", pa, v) + torch.einsum("rhgn,rhnd->rhgd", pb, vo)
        out[rows] /= pa.sum(-1, keepdim=True) + pb.sum(-1, keepdim=True)
        row += n_rows
    return out.view(out.shape[0], -1).bfloat16()


def _f16_rows(x):
    return x.float()


def _q8_values(x):
    blocks = x.shape[-1] // 34
    d = x[..., :2 * blocks].contiguous().view(torch.float16).float()
    return (x[..., 2 * blocks:].contiguous().view(torch.int8).float().unflatten(-1, (blocks, 32)) * d.unsqueeze(-1)).flatten(-2)


def _exact_attention(s):
    """Row by row over all its keys in 64 bits."""
    _, n_q, n_kv, head, _ = LAYERS[s["case"]["model"]]
    q = s["q"].double()
    out = torch.zeros_like(q)
    for r, (seq, pos) in enumerate(zip(s["row_seq"].tolist(), s["row_pos"].tolist())):
        if seq < 0:
            continue
        ids = s["table"][seq, :pos // PAGE + 1].long()

        def cached(x):
            x = x[ids]
            if x.dtype == torch.uint8:
                d, codes = x[..., :head // 16].contiguous().view(torch.float16), x[..., head // 16:].contiguous().view(torch.int8)
                x = d.double().repeat_interleave(32, -1) * codes.double()
            return x.double().permute(1, 0, 2, 3).reshape(n_kv, -1, head)[:, :pos + 1]
        k, v = cached(s["k"]), cached(s["v"])
        for h in range(n_kv):
            mine = slice(h * (n_q // n_kv), (h + 1) * (n_q // n_kv))
            out[r, mine] = torch.softmax(q[r, mine] @ k[h].T, -1) @ v[h]
    return out.view(out.shape[0], -1)


# ---- the next beams -------------------------------------------------------------------------------------------------
def _prepare_select(case, gen, rng):
    G, B, V = case["groups"], case["beams"], LAYERS[case["model"]][4]
    eos = V - 7
    done = torch.zeros(G, B, dtype=torch.int32)
    length = torch.full((G, B), rng.randint(4, 60), dtype=torch.int32)
    for g in range(G):
        for b in rng.sample(range(B), case["finished"]):
            done[g, b], length[g, b] = 1, rng.randint(3, int(length.max()))
    done, length = done.cuda(), length.cuda()
    state = {"case": case, "eos": eos, "done": done, "length": length,
             "logits": torch.empty(G * B, V, device="cuda"), "scores": torch.empty(G, B, device="cuda")}
    left = torch.arange(G, device="cuda")
    while len(left):
        # a bulk of unlikely ids and some 30 that the model considers, as logits of trained models have them
        n = len(left)
        x = torch.randn(n * B, V, generator=gen, device="cuda") * 1.5
        likely = torch.randint(0, V, (n * B, 30), generator=gen, device="cuda")
        x.scatter_add_(1, likely, 4 + 6 * torch.rand(n * B, 30, generator=gen, device="cuda"))
        state["logits"].view(G, B, V)[left] = x.view(n, B, V)
        # beams of one search lie a few nats apart; those that ended did so earlier
        state["scores"][left] = length[left].float() * -0.9 - 3 * torch.rand(n, B, generator=gen, device="cuda")
        rank = _ranks(state, left, torch.float64)
        best = rank.flatten(1).topk(B + 1).values
        # a search whose last places are decided by rounding has no one answer: it is made again
        left = left[((best[:, :-1] - best[:, 1:]).amin(-1) < APART)]
    if own:
        from bloomery_b200.ops.beam import BeamScratch
        state["scratch"] = BeamScratch(G, B, V, "cuda")
        state["out"] = {"parent": torch.empty_like(done), "token": torch.empty_like(done), "scores": torch.empty_like(state["scores"]),
                        "done": torch.empty_like(done), "length": torch.empty_like(length)}
    return state


def _candidates(s, groups, dtype):
    case = s["case"]
    B, V = case["beams"], s["logits"].shape[1]
    x = s["logits"].view(-1, B, V)[groups].to(dtype)
    top = x.amax(-1, keepdim=True)
    x = s["scores"][groups].to(dtype).unsqueeze(-1) + (x - (top + torch.exp(x - top).sum(-1, keepdim=True).log()))
    if case["finished"]:
        done = s["done"][groups].bool()
        x[done] = -math.inf
        x[..., s["eos"]] = torch.where(done, s["scores"][groups].to(dtype), x[..., s["eos"]])
    return x


def _ranks(s, groups, dtype):
    x = _candidates(s, groups, dtype)
    if s["case"]["alpha"]:
        x = x * (s["length"] + 1 - s["done"])[groups].to(dtype).pow(-s["case"]["alpha"]).unsqueeze(-1)
    return x


def _run_select(s):
    case = s["case"]
    if own:
        from bloomery_b200.ops.beam import beam_select
        o = s["out"]
        beam_select(s["logits"], s["scores"], s["scratch"], o["parent"], o["token"], o["scores"], done=s["done"], lengths=s["length"],
                    out_done=o["done"], out_lengths=o["length"], eos=s["eos"], alpha=case["alpha"])
        return o
    every = slice(None)
    x = _candidates(s, every, torch.float32)
    rank = x
    if case["alpha"]:
        rank = x * (s["length"] + 1 - s["done"]).float().pow(-case["alpha"]).unsqueeze(-1)
    at = rank.flatten(1).topk(case["beams"]).indices             # no two are equal: see _prepare_select
    parent, token = at // x.shape[-1], at % x.shape[-1]
    over = s["done"].gather(1, parent)
    return {"parent": parent.int(), "token": token.int(), "scores": x.flatten(1).gather(1, at),
            "done": (over.bool() | (token == s["eos"])).int(), "length": s["length"].gather(1, parent) + 1 - over}


def _exact_select(s):
    """Search by search in 64 bits: the log-probabilities of each beam, then a stable sort of all candidates."""
    case, V = s["case"], s["logits"].shape[1]
    out = {"parent": [], "token": [], "scores": [], "done": [], "length": []}
    for g in range(case["groups"]):
        rank, value = [], []
        for b in range(case["beams"]):
            score, done, length = float(s["scores"][g, b]), int(s["done"][g, b]), int(s["length"][g, b])
            if done:
                c = torch.full((V,), -math.inf, dtype=torch.float64, device="cuda")
                c[s["eos"]] = score
            else:
                c = torch.log_softmax(s["logits"][g * case["beams"] + b].double(), 0) + score
            value.append(c)
            rank.append(c / float(length + 1 - done) ** case["alpha"])
        at = torch.sort(torch.cat(rank), descending=True, stable=True).indices[:case["beams"]].tolist()
        value = torch.cat(value)
        out["parent"].append([i // V for i in at])
        out["token"].append([i % V for i in at])
        out["scores"].append([float(value[i]) for i in at])
        out["done"].append([int(int(s["done"][g, i // V]) or i % V == s["eos"]) for i in at])
        out["length"].append([int(s["length"][g, i // V]) + 1 - int(s["done"][g, i // V]) for i in at])
    return {k: torch.tensor(x, dtype=torch.float64 if k == "scores" else torch.int32, device="cuda") for k, x in out.items()}


# ---- states that follow their beams ---------------------------------------------------------------------------------
def _prepare_reorder(case, gen, rng):
    n_layer, _, n_kv, head, _ = LAYERS[case["model"]]
    G, B, col = case["groups"], case["beams"], case["held"] // PAGE
    # whole pages are shared within a search; the page being filled and the next one belong to each beam
    n_pages = G * (col + 2 * B)
    free = list(range(n_pages))
    rng.shuffle(free)
    slots = list(range(G * B))
    rng.shuffle(slots)
    table = torch.full((G * B, MAX_PAGES), -1, dtype=torch.int32)
    parent = []
    for g in range(G):
        shared = [free.pop() for _ in range(col)]
        for b in range(B):
            ids = shared + [free.pop(), free.pop()]
            table[slots[g * B + b], :col + 2] = torch.tensor(ids, dtype=torch.int32)
        # `moved` beams end; others have more than one child
        kept = sorted(rng.sample(range(B), B - case["moved"]))
        row = kept + [rng.choice(kept) for _ in range(case["moved"])]
        rng.shuffle(row)
        parent.append(row)
    shape = (n_layer, n_pages, n_kv, PAGE, head)
    k = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(generator=gen)
    v = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(generator=gen)
    table = table.cuda()
    return {"case": case, "k": k, "v": v, "table": table, "table_out": torch.full_like(table, -1), "slots": _ints(slots),
            "parent": _ints(parent), "held": _ints([case["held"]] * G)}


def _run_reorder(s):
    """The tables of all slots behind the choice, and the caches.  A pass leaves the old tables and every page that they lead
    a surviving beam to as they are, so it may be made again."""
    if own:
        from bloomery_b200.ops.beam import beam_reorder
        beam_reorder(s["k"], s["v"], s["table"], s["table_out"], s["slots"], s["parent"], s["held"])
        return {"k": s["k"], "v": s["v"], "table": s["table_out"]}
    G, B = s["parent"].shape
    slots, col = s["slots"].long().view(G, B), s["held"].long() // PAGE
    part = s["case"]["held"] % PAGE
    rows = s["table"][slots]                                     # [G, B, pages]
    parent = s["parent"].long()
    mine = torch.arange(MAX_PAGES, device="cuda") >= col[:, None, None]
    new = torch.where(mine, rows, rows.gather(1, parent.unsqueeze(-1).expand_as(rows)))
    if part:
        # a beam's first child goes on in its page, other children take the pages of beams without one, in order
        same = parent.unsqueeze(-1) == parent.unsqueeze(-2)
        first = ~(same & torch.ones(B, B, dtype=torch.bool, device="cuda").tril(-1)).any(-1)
        bare = ~(parent.unsqueeze(-2) == torch.arange(B, device="cuda").unsqueeze(-1)).any(-1)
        page = rows.gather(2, col.view(G, 1, 1).expand(G, B, 1)).squeeze(-1)
        source = page.gather(1, parent)
        place = torch.where(first, source, 0)
        place[~first] = page[bare]
        new.scatter_(2, col.view(G, 1, 1).expand(G, B, 1), place.unsqueeze(-1))
        src, dst = source[~first].long(), place[~first].long()
        for pool in (s["k"], s["v"]):
            pool[:, dst, :, :part] = pool[:, src, :, :part]
    s["table_out"][slots] = new
    return {"k": s["k"], "v": s["v"], "table": s["table_out"]}
