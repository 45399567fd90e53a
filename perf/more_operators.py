"""The calls by which the operators of NVFP4 products are measured: rows of activations in four bits, their products with NVFP4
weights as they are, and the routed experts of a few tokens.

NVFP4 is blocks of 16 E2M1 codes with an E4M3 scale each and one 32-bit scale over them, of a tensor (weights) or of a row
(activations).  A checkpoint that stores its weights so is served with activations in the same form: every product of a layer
quantises its input rows and multiplies codes by codes.  Shapes are the framework's own: the Qwen3-30B-A3B layer (2,048 wide, 32
heads of 128, 128 experts of 768, 8 of them for a token, 4 key heads), the 235B one (4,096 wide, 64 heads, experts of 1,536) and the
tiny one (512 wide, 16 experts of 256, 4 for a token, 32,000 ids).
"""
import math
import random

import torch

own = False

#         hidden, rows of Q, experts, experts of a token, width of an expert, vocabulary
MODELS = {"30b": (2048, 4096, 128, 8, 768, 151936), "235b": (4096, 8192, 128, 8, 1536, 151936), "tiny": (512, 512, 16, 4, 256, 32000)}
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # the smallest call: the input of a round's products; launches are all it costs
        rows("rows of a round", 24, 2048, "bf16"),
        # the input of a prompt's projections, with the norm in front of them
        rows("rows of a prompt behind their norm", 4096, 4096, "f32", norm=True),
        # the projection behind attention in a round of 16 sequences: few rows, few tiles
        linear("output projection of a round", 16, 4096, 2048, "bf16", "f32", resid=True),
        # odd: 37 rows in f16 on the vocabulary of the tiny model
        linear("37 rows on a vocabulary", 37, 512, 32000, "f16", "f32"),
        # the widest product of a long prompt
        linear("queries of a prompt of 4096, 235b", 4096, 4096, 8192, "bf16", "bf16"),
        # experts with some six rows each, tiny
        experts("gate and up of 100 ids, tiny", "gated", "tiny", 100, 16),
        # a prompt's gate and up: 125 rows an expert, ragged
        experts("gate and up of 2000 ids", "gated", "30b", 2000, 128),
        # a long prompt's down products, back in the order of the ids, with the router's weights
        experts("down of 4096 ids", "down", "30b", 4096, 128),
        # one token: eight experts, most of it latency
        experts("experts of 1 token", "moe", "30b", 1, 8),
        # a round of 24 sequences that hits 95 experts
        experts("experts of 24 tokens", "moe", "30b", 24, 95),
        # odd: five tokens, six slots that another tier serves
        experts("experts of 5 tokens, some elsewhere, tiny", "moe", "tiny", 5, 11, away=6),
        # the largest round of the largest model: every expert is hit
        experts("experts of 64 tokens, 235b", "moe", "235b", 64, 128),
    ]


def rows(name, T, K, dtype, norm=False):
    return {"name": name, "op": "rows", "T": T, "K": K, "dtype": dtype, "norm": norm}


def linear(name, T, K, N, dtype, out, resid=False):
    return {"name": name, "op": "linear", "T": T, "K": K, "N": N, "dtype": dtype, "out": out, "resid": resid}


def experts(name, op, model, T, hit, away=0):
    return {"name": name, "op": op, "model": model, "T": T, "hit": hit, "away": away}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Rows of 1 to 4,096 by 64 to 7,168 values; products of 1 to 4,096 rows, 64 to 7,168 deep, with 1 to 32,000 rows of weights;
    prompts of 1 to 4,096 ids through gate and up or down; rounds of 1 to 64 tokens through the routed experts."""
    kind = rng.choice(["rows", "linear", "linear", "gated", "down", "moe", "moe"])
    while True:
        T, K = _log(rng, 1, 4096), 64 * _log(rng, 1, 112)
        if kind == "rows":
            norm = rng.random() < 0.5
            case = rows("", T, K, "f32" if norm else rng.choice(["bf16", "f16", "f32"]), norm)
        elif kind == "linear":
            case = linear("", T, K, _log(rng, 1, 32000), rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice(["f32", "bf16"]),
                          rng.random() < 0.5)
        else:
            model = rng.choice(["30b", "30b", "tiny"] if kind != "moe" else ["30b", "235b", "tiny"])
            E, k = MODELS[model][2:4]
            T = _log(rng, 1, 4096 if kind != "moe" else 64)
            most = min(E, T * k)
            hit = rng.randint(min(k, most), most)
            case = experts("", kind, model, T, hit, rng.choice([0, 0, T * k // 5]) if kind == "moe" else 0)
        cost = work(case)
        if all(cost[key] <= max(work(c)[key] for c in listed() if c["op"] == kind) for key in cost):
            del case["name"]
            return case


def work(case):
    """Bytes and operations of a pass: inputs once, the weights of the experts that are hit once, outputs once."""
    T = case["T"]
    if case["op"] == "rows":
        K = case["K"]
        return {"bytes": T * K * (4 if case["dtype"] == "f32" else 2) + T * _row_bytes(K) + 2 * T * K, "flops": 0}
    if case["op"] == "linear":
        K, N = case["K"], case["N"]
        size = 4 if case["out"] == "f32" else 2
        return {"bytes": T * K * (4 if case["dtype"] == "f32" else 2) + N * _row_bytes(K) + T * N * (size + 4 * case["resid"]),
                "flops": 2 * T * N * K}
    H, _, E, k, inter, _ = MODELS[case["model"]]
    slots, hit = T * k - case["away"], case["hit"]
    gate, down = 2 * hit * inter * _row_bytes(H), hit * H * _row_bytes(inter)
    if case["op"] == "gated":
        return {"bytes": 2 * T * H + gate + 2 * slots * inter, "flops": 4 * slots * inter * H}
    if case["op"] == "down":
        return {"bytes": 2 * slots * inter + down + 4 * slots * H, "flops": 2 * slots * inter * H}
    return {"bytes": 4 * T * H + gate + down + 2 * T * H, "flops": 6 * slots * inter * H}


def _row_bytes(K):
    return (K // 2 + K // 16 + 4 + 15) // 16 * 16


# ---- what a case is made of -----------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng = random.Random(seed)
    with torch.no_grad():
        s = _prepare(case, gen, rng)
        if own:
            _keep(case, s)
    return s


def _activations(gen, T, K, dtype):
    """Rows with a few channels far above the others and a size of their own, as the inputs of trained layers have them."""
    size = torch.exp(0.4 * torch.randn(K, generator=gen, device="cuda"))
    size[torch.randint(0, K, (max(1, K // 256),), generator=gen, device="cuda")] *= 12
    x = torch.randn(T, K, generator=gen, device="cuda") * size * torch.exp(0.5 * torch.randn(T, 1, generator=gen, device="cuda"))
    return x.to(TYPES[dtype])


def _weights(gen, *shape):
    """NVFP4 rows [..., N, K]: K / 2 bytes of codes (the even value in the low half), K / 16 scales, the tensor's scale, padding.
    Codes are those of normal values."""
    *lead, K = shape
    z = torch.erfinv((2 * torch.arange(256, device="cuda") + 1) / 256 - 1) * math.sqrt(2) * 2.9
    code = _nearest_code(z.abs().double(), torch.ones_like(z, dtype=torch.float64))
    lut = (torch.tensor([0, 1, 2, 3, 4, 0, 5, 0, 6, 0, 0, 0, 7], device="cuda")[(2 * code).long()] + 8 * (z < 0)).to(torch.uint8)
    out = torch.zeros(*lead, _row_bytes(K), dtype=torch.uint8, device="cuda")
    half = torch.empty(*lead, K // 2, dtype=torch.uint8, device="cuda")
    for shift in (1, 16):
        half.random_(0, 256, generator=gen)
        out[..., :K // 2] += lut[half.int()] * shift
    out[..., K // 2:K // 2 + K // 16].random_(0x6b, 0x7a, generator=gen)
    scale = 4e-5 * (0.5 + torch.rand(1, generator=gen, device="cuda"))
    out[..., K // 2 + K // 16:K // 2 + K // 16 + 4] = scale.view(torch.uint8)
    return out


def _routed(case, gen, rng):
    """Which experts each id goes to: ``hit`` of them in all, the first ids see to that; ``away`` slots belong to another tier."""
    _, _, E, k, _, _ = MODELS[case["model"]]
    T, hit = case["T"], case["hit"]
    some = rng.sample(range(E), hit)
    ids = [rng.sample(some, k) if hit > k else list(some) for _ in range(T)]
    for t in range(-(-hit // k)):
        ids[t] = [some[(t * k + j) % hit] for j in range(k)]
    ids = torch.tensor(ids, dtype=torch.int32)
    for i in rng.sample(range(T * k), case["away"]):
        ids.view(-1)[i] = -1
    w = torch.softmax(torch.randn(T, k, generator=gen, device="cuda"), -1)
    return ids.cuda(), w, torch.tensor(sorted(some), device="cuda")


def _prepare(case, gen, rng):
    s = {"case": case}
    T = case["T"]
    if case["op"] in ("rows", "linear"):
        s["x"] = _activations(gen, T, case["K"], case["dtype"])
        if case["op"] == "rows":
            s["gain"] = 1 + 0.2 * torch.randn(case["K"], generator=gen, device="cuda") if case["norm"] else None
            return s
        s["w"] = _weights(gen, case["N"], case["K"])
        s["resid"] = torch.randn(T, case["N"], generator=gen, device="cuda") if case["resid"] else None
        return s
    H, _, E, k, inter, _ = MODELS[case["model"]]
    s["ids"], s["wts"], s["some"] = _routed(case, gen, rng)
    if case["op"] == "down":
        s["x"] = _activations(gen, T * k, inter, "bf16")
        s["w"] = _weights(gen, E, H, inter)
    else:
        s["x"] = _activations(gen, T, H, "f32" if case["op"] == "moe" else "bf16")
        s["gate"], s["up"] = _weights(gen, E, inter, H), _weights(gen, E, inter, H)
    if case["op"] == "moe":
        s["w"] = _weights(gen, E, H, inter)
        s["gain"] = (1 + 0.2 * torch.randn(H, generator=gen, device="cuda"))
    else:
        # slots in the order of their experts, for products that read an expert's rows next to each other
        flat = s["ids"].view(-1).long()
        order = torch.argsort(flat, stable=True)
        count = torch.bincount(flat, minlength=E)
        s["most"] = int(count.max())
        s["slot"], s["expert"] = order, flat[order]
        s["place"] = torch.arange(T * k, device="cuda") - (count.cumsum(0) - count)[flat[order]]
    return s


def _keep(case, s):
    """What a program keeps beside its data: weights under their type, tables of tiles, buffers."""
    from bloomery_b200.ops import fp4 as Q
    from bloomery_b200.ops import gemm as G
    from bloomery_b200.ops.decode import QWeight
    T = case["T"]
    for name, width in (("w", 4), ("gate", 0), ("up", 0)):
        if name in s:
            s[name] = QWeight(s[name], "NVFP4", case["K"] if "K" in case else MODELS[case["model"]][width])
    bf, f32, i32 = (dict(dtype=t, device="cuda") for t in (torch.bfloat16, torch.float32, torch.int32))
    if case["op"] in ("rows", "linear"):
        s["rows"] = Q.Fp4Rows(T, case["K"], "cuda")
    if case["op"] == "rows":
        s["out"] = torch.empty(T, case["K"], **bf)
    elif case["op"] == "linear":
        s["tiles"] = Q.fp4_tiles(T, "cuda")
        s["work"] = Q.Fp4Work("cuda")
        s["out"] = torch.empty(T, case["N"], **(f32 if case["out"] == "f32" else bf))
    else:
        H, _, E, k, inter, _ = MODELS[case["model"]]
        if case["op"] == "moe":
            s["work"] = Q.Fp4MoeWork(T, k, H, inter, E, "cuda")
            s["out"] = torch.empty(T, H, **bf)
            return
        n = T * k
        s["rows"] = Q.Fp4Rows(n, H if case["op"] == "gated" else inter, "cuda")
        s["tiles"] = G.TileTable(n, E, "cuda", Q.fp4_tile_rows(n, E, case["op"] == "gated"))
        s["pos_of"], s["dst_row"] = torch.zeros(n, **i32), torch.zeros(n + 128, **i32)
        s["row_scale"] = torch.zeros(n + 128, **f32)
        G.moe_plan(s["ids"], s["wts"], E, s["tiles"], s["pos_of"], s["dst_row"], s["row_scale"])
        s["out"] = torch.empty(n, inter, **bf) if case["op"] == "gated" else torch.empty(n, H, **f32)


# ---- the operators --------------------------------------------------------------------------------------------------
def run(state):
    with torch.no_grad():
        return {"rows": _rows, "linear": _linear, "gated": _gated, "down": _down, "moe": _moe}[state["case"]["op"]](state)


def _nearest_scale(q):
    """Values of E4M3 next to q >= 0 (64 bits), the even one of two as near, 448 at most."""
    e = torch.frexp(q)[1].clamp_min(-5) - 4
    return torch.ldexp(torch.round(torch.ldexp(q, -e)), e).clamp_max(448.0)


def _nearest_code(a, d):
    """Values of E2M1 next to a / d (64 bits), the even one of two as near, 6 at most; 0 where d is."""
    y = (a / torch.where(d > 0, d, 1.0)).clamp_max(7.0) * (d > 0)
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    return (torch.round(y / step) * step).clamp_max(6.0)


def _quantised(x):
    """The values that rows are in four bits: a scale of the row that takes the largest of it to 6 x 448, E4M3 scales of blocks of
    16 that take theirs to 6, codes.  Which value is nearest is looked at in 64 bits; values in 32."""
    x = x.float()
    g = (x.abs().amax(-1, keepdim=True).double() / 2688).float().clamp_min(2.0 ** -100).unsqueeze(-1)      # rounded once
    b = x.unflatten(-1, (-1, 16))
    s = _nearest_scale(b.abs().amax(-1, keepdim=True).double() / (6.0 * g.double())).float()
    d = s * g
    return (torch.copysign(_nearest_code(b.abs().double(), d.double()).float(), b) * d).flatten(-2)


def _normed(x, gain):
    mean = x.double().square().mean(-1, keepdim=True)
    return x * (1.0 / (mean + EPS).sqrt()).float() * gain


def _values(w, K):
    """32-bit values of NVFP4 rows."""
    code, sc = w[..., :K // 2], w[..., K // 2:K // 2 + K // 16].int()
    scale = w[..., K // 2 + K // 16:K // 2 + K // 16 + 4].contiguous().view(torch.float32)
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=w.device)
    pairs = torch.stack([lut[torch.arange(256, device=w.device) % 16], lut[torch.arange(256, device=w.device) // 16]], -1)
    v = pairs[code.int()].flatten(-2).unflatten(-1, (-1, 16))
    size = torch.where(sc >= 8, torch.ldexp(1 + (sc % 8) / 8, sc // 8 - 7), sc * 2.0 ** -9)
    v *= (size * scale).unsqueeze(-1)
    return v.flatten(-2)


def _silu_times(g, u):
    return g / (1 + torch.exp(-g)) * u


def _rows(s):
    """The values that the rows have become, in bf16."""
    if own:
        from bloomery_b200.ops.fp4 import fp4_rows
        from bloomery_b200.ops.gemm import dequant_bf16
        fp4_rows(s["x"], s["rows"], gain=s["gain"], eps=EPS)
        return dequant_bf16(s["rows"].weight, s["out"])
    x = _normed(s["x"], s["gain"]) if s["case"]["norm"] else s["x"]
    return _quantised(x).bfloat16()


def _linear(s):
    if own:
        from bloomery_b200.ops.fp4 import fp4_gemm, fp4_rows
        fp4_rows(s["x"], s["rows"])
        f32 = s["out"].dtype is torch.float32
        fp4_gemm(s["rows"], s["w"], s["tiles"], out_f32=s["out"] if f32 else None, out_bf16=None if f32 else s["out"],
                 resid=s["resid"], work=s["work"])
        return s["out"]
    y = _quantised(s["x"]) @ _values(s["w"], s["case"]["K"]).mT
    if s["case"]["resid"]:
        y = y + s["resid"]
    return y.to(TYPES[s["case"]["out"]])


def _dealt(s, x):
    """Rows of the slots, expert by expert, [experts, most rows of one, values]."""
    out = torch.zeros(MODELS[s["case"]["model"]][2], s["most"], x.shape[-1], device="cuda")
    out[s["expert"], s["place"]] = x
    return out


def _gated(s):
    """silu(x gate) * (x up) of every slot, in the order of the slots."""
    H, _, E, k, inter, _ = MODELS[s["case"]["model"]]
    if own:
        from bloomery_b200.ops.fp4 import fp4_gemm, fp4_rows
        fp4_rows(s["x"], s["rows"], pos_of=s["pos_of"])
        fp4_gemm(s["rows"], s["gate"], s["tiles"], W2=s["up"], out_bf16=s["out"], dst_row=s["dst_row"])
        return s["out"]
    x = _dealt(s, _quantised(s["x"])[s["slot"] // k])
    y = _silu_times(x @ _values(s["gate"], H).mT, x @ _values(s["up"], H).mT)
    out = torch.empty(s["slot"].numel(), inter, device="cuda")
    out[s["slot"]] = y[s["expert"], s["place"]]
    return out.bfloat16()


def _down(s):
    """Router weight times (x down) of every slot, in the order of the slots."""
    H, _, E, k, inter, _ = MODELS[s["case"]["model"]]
    if own:
        from bloomery_b200.ops.fp4 import fp4_gemm, fp4_rows
        fp4_rows(s["x"], s["rows"], pos_of=s["pos_of"])
        fp4_gemm(s["rows"], s["w"], s["tiles"], out_f32=s["out"], dst_row=s["dst_row"], row_scale=s["row_scale"])
        return s["out"]
    y = _dealt(s, _quantised(s["x"])[s["slot"]]) @ _values(s["w"], inter).mT
    out = torch.empty(s["slot"].numel(), H, device="cuda")
    out[s["slot"]] = y[s["expert"], s["place"]]
    return out * s["wts"].view(-1, 1)


def _moe(s):
    """What the routed experts add to every token: the norm, gate and up of its experts, their products in four bits again, down, and the
    sum by the router's weights."""
    H, _, E, k, inter, _ = MODELS[s["case"]["model"]]
    if own:
        from bloomery_b200.ops.fp4 import fp4_moe
        fp4_moe(s["x"], s["ids"], s["wts"], s["gate"], s["up"], s["w"], s["work"], gain=s["gain"], eps=EPS, out_bf16=s["out"])
        return s["out"]
    x, some = _quantised(_normed(s["x"], s["gain"])), s["some"]
    y = _silu_times(x @ _values(s["gate"][some], H).mT, x @ _values(s["up"][some], H).mT)             # [experts, tokens, inter]
    y = _quantised(y) @ _values(s["w"][some], inter).mT
    mine = (s["ids"].unsqueeze(-1) == some) * s["wts"].unsqueeze(-1)
    return torch.einsum("te,eth->th", mine.sum(1), y).bfloat16()


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------
def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    with torch.no_grad():
        return {"rows": _exact_rows, "linear": _exact_linear, "gated": _exact_gated, "down": _exact_down, "moe": _exact_moe}[case["op"]](s)


def _exact_quantised(x):
    """Row by row of the definition: the nearest of the listed values of each type, by bisection between their midpoints."""
    f64 = dict(dtype=torch.float64, device="cuda")
    e4m3 = torch.tensor([m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1], **f64)
    e2m1 = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], **f64)

    def nearest(v, table):
        mid = (table[1:] + table[:-1]) / 2
        lo, hi = torch.searchsorted(mid, v), torch.searchsorted(mid, v, right=True)
        return table[torch.where(lo % 2 == 0, lo, hi)]           # they differ on a midpoint alone: the even one
    out = torch.empty(x.shape, **f64)
    for i in range(0, x.shape[0], 4096):
        v = x[i:i + 4096].double()
        g = (v.abs().amax(1) / 2688).float().double().clamp_min(2.0 ** -100)
        b = v.view(v.shape[0], -1, 16)
        s = nearest((b.abs().amax(2) / (6 * g[:, None])).contiguous(), e4m3)
        d = (s.float() * g.float()[:, None]).double()             # the step is a product in 32 bits
        c = nearest((b.abs() / d.clamp_min(1e-300).unsqueeze(-1)).contiguous(), e2m1) * (s > 0).unsqueeze(-1)
        out[i:i + 4096] = (torch.sign(b) * c * (s * g[:, None]).unsqueeze(-1)).flatten(1)
    return out


def _exact_normed(x, gain):
    r = (x.double().square().sum(1) / x.shape[1] + EPS).rsqrt().float()
    return x * r[:, None] * gain                                  # two products in 32 bits


def _exact_values(w, K):
    code = w[:, :K // 2].long()
    code = torch.stack([code & 15, code >> 4], 2).flatten(1)
    v = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")[code & 7] * (1 - 2.0 * (code > 7))
    sc = w[:, K // 2:K // 2 + K // 16].contiguous().view(torch.float8_e4m3fn).double().repeat_interleave(16, 1)
    return v * sc * w[:, K // 2 + K // 16:K // 2 + K // 16 + 4].contiguous().view(torch.float32).double()


def _exact_silu(g):
    return g * torch.sigmoid(g)


def _exact_rows(s):
    x = s["x"]
    return _exact_quantised(_exact_normed(x, s["gain"]) if s["case"]["norm"] else x)


def _exact_linear(s):
    w = _exact_values(s["w"], s["case"]["K"])
    y = torch.cat([x @ w.T for x in _exact_quantised(s["x"]).split(1024)])
    return y + s["resid"].double() if s["case"]["resid"] else y


def _exact_gated(s):
    H, _, E, k, inter, _ = MODELS[s["case"]["model"]]
    x, flat = _exact_quantised(s["x"]), s["ids"].view(-1)
    out = torch.empty(flat.numel(), inter, dtype=torch.float64, device="cuda")
    for e in range(E):
        at = (flat == e).nonzero().squeeze(1)
        g, u = (x[at // k] @ _exact_values(s[name][e], H).T for name in ("gate", "up"))
        out[at] = _exact_silu(g) * u
    return out


def _exact_down(s):
    H, _, E, k, inter, _ = MODELS[s["case"]["model"]]
    x, flat = _exact_quantised(s["x"]), s["ids"].view(-1)
    out = torch.empty(flat.numel(), H, dtype=torch.float64, device="cuda")
    for e in range(E):
        at = (flat == e).nonzero().squeeze(1)
        out[at] = s["wts"].view(-1)[at, None].double() * (x[at] @ _exact_values(s["w"][e], inter).T)
    return out


def _exact_moe(s):
    H, _, E, k, inter, _ = MODELS[s["case"]["model"]]
    x, flat = _exact_quantised(_exact_normed(s["x"], s["gain"])), s["ids"].view(-1)
    out = torch.zeros(s["case"]["T"], H, dtype=torch.float64, device="cuda")
    for e in flat.unique().tolist():
        if e < 0:
            continue
        at = (flat == e).nonzero().squeeze(1)
        g, u = (x[at // k] @ _exact_values(s[name][e], H).T for name in ("gate", "up"))
        y = _exact_quantised((_exact_silu(g) * u).float()) @ _exact_values(s["w"][e], inter).T
        out.index_add_(0, at // k, s["wts"].view(-1)[at, None].double() * y)
    return out
