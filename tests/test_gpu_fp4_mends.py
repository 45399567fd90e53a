"""Calls of the NVFP4 operators that were answered wrongly once, or could be."""
import gc
import math

import pytest
import torch

from bloomery_b200.formats import planes
from test_gpu_fp4 import DEV, allowed, make, parts, quantised, same, weight
from test_gpu_fp4_moe import case, oracle, run

gpu = pytest.mark.gpu


# ---- rows of a few tokens one behind the other ----------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("T,k,dtype", [(2, 4, torch.bfloat16), (3, 4, torch.float32), (4, 4, torch.bfloat16), (4, 8, torch.float32)])
def test_few_tokens_without_a_norm_keep_their_own_scales(T, k, dtype):
    """Rows of very different sizes: a maximum of the row behind taken for a row's own would be far off.  Every row as if it were alone,
    bit for bit and every time."""
    c = case(T, 16, k, 256, 2048, seed=40 + T, dtype=dtype)
    x = c[0]
    x *= torch.tensor([2.0 ** (9 * (t % 2) - 3 * t) for t in range(T)], device=DEV)[:, None]
    want, tol = oracle(*c[:3], *(w[1] for w in c[3:]))
    tol = tol + (k + 1) * 2.0 ** -24 * want.abs()
    alone = torch.empty(T, 2048, device=DEV)
    for t in range(T):
        run(x[t:t + 1], c[1][t:t + 1], c[2][t:t + 1], *c[3:], out_f32=alone[t:t + 1])
    assert bool(((alone.double().cpu() - want).abs() <= tol).all())
    out, work = torch.empty(T, 2048, device=DEV), None
    for _ in range(40):
        work = run(*c, work=work, out_f32=out)
        assert torch.equal(out, alone)


# ---- products of one input on several streams -----------------------------------------------------------------------
def engine(kind, n_slots=12):
    """Tiny models: every matrix NVFP4, but the v projections in Q8_0 (``mixed``) or one projection of a layer with signs in its block
    scales (``signs``); latent attention with a shared expert and a dense layer (``latent``)."""
    from bloomery_b200.models.spec import tiny_deepseek, tiny_qwen3moe
    from bloomery_b200.models.weights import Weights, synth_tensors
    from bloomery_b200.runtime.engine import DecodeEngine
    spec = tiny_deepseek() if kind == "latent" else tiny_qwen3moe()
    items = list(synth_tensors(spec, DEV, seed=3, mix="NVFP4"))
    if kind == "mixed":
        items = [b if a[0].endswith("attn_v.weight") else a for a, b in zip(items, synth_tensors(spec, DEV, seed=3, mix="Q8_0"))]
    w = Weights.from_items(spec, iter(items), DEV)
    if kind == "signs":
        q = w.q["blk.0.attn_k.weight"]
        q.data[3, q.k // 2 + 1] |= 0x80
    eng = DecodeEngine(w, n_slots=n_slots, slot_ctx=256)
    g = torch.Generator().manual_seed(7)
    prompts = [torch.randint(0, spec.vocab, (5 + 3 * (i % 7),), generator=g).tolist() for i in range(n_slots)]
    return spec, eng, [(slot, eng.prefill(slot, p, gemm=False), len(p)) for slot, p in enumerate(prompts)]


@pytest.fixture(autouse=True)
def no_engine_left():
    """Engines hold their prompt paths and those the engines: their graphs must not be taken down while a later test captures one."""
    yield
    gc.collect()


def values(q):
    flat = q.data.reshape(-1, q.data.shape[-1]).cpu()
    ts = flat[:, q.k // 2 + q.k // 16:q.k // 2 + q.k // 16 + 4].contiguous().view(torch.float32).double()
    return planes.nvfp4_dequantize(flat[:, :q.k // 2], flat[:, q.k // 2:q.k // 2 + q.k // 16], 1.0).double() * ts


@gpu
@pytest.mark.parametrize("kind", ["mixed", "signs", "latent"])
def test_rows_of_one_input_are_made_on_one_stream(kind, monkeypatch):
    """Two streams that fill one buffer while either reads it have no order between them.  The first pass, of plain launches, gives the
    bits of the captured one."""
    from bloomery_b200.ops import fp4 as Q
    from bloomery_b200.runtime.batch_decode import BatchDecode
    spec, eng, rows = engine(kind)
    bd = BatchDecode(eng, max_rows=16)
    bd.fp4_native = True
    streams, plain = {}, Q.fp4_rows

    def recorded(x, out, **kw):
        streams.setdefault(out.ptr, set()).add(torch.cuda.current_stream().cuda_stream)
        plain(x, out, **kw)
    monkeypatch.setattr(Q, "fp4_rows", recorded)
    M = bd.set_rows(rows)
    with torch.cuda.stream(bd._stream):
        bd.enqueue(M)
    torch.cuda.synchronize()
    first = bd.logits[:len(rows)].clone()
    assert streams and all(s == {bd._stream.cuda_stream} for s in streams.values())
    monkeypatch.setattr(Q, "fp4_rows", plain)
    for _ in range(3):
        bd.step(rows)
        assert torch.equal(bd.logits[:len(rows)], first)
    assert first.isfinite().all()


@gpu
@pytest.mark.parametrize("kind", ["mixed", "signs", "latent"])
def test_projections_beside_others_of_another_type(kind):
    """Those that take NVFP4 rows against the definition, the others as without."""
    from bloomery_b200.ops import gemm as G
    from bloomery_b200.runtime.batch_decode import BatchDecode
    spec, eng, rows = engine(kind)
    bd = BatchDecode(eng, max_rows=16)
    M = bd.set_rows(rows)
    x = torch.randn(M, spec.hidden, generator=torch.Generator().manual_seed(1)).to(DEV)
    names = ("attn_q_a", "attn_kv_a_mqa") if spec.mla else ("attn_q", "attn_k", "attn_v")
    got = {}
    for native in (False, True):
        bd.fp4_native = native
        with torch.cuda.stream(bd._stream):
            bd.x[:M].copy_(x)
            G.rmsnorm_bf16(bd.x[:M], eng.w.f["blk.0.attn_norm.weight"], spec.rms_eps, bd.xn[:M])
            (bd._attn_mla if spec.mla else bd._attn_gqa)(0, M, bd.xn[:M], bd.dense_tiles[M])
        torch.cuda.synchronize()
        got[native] = bd.qkv[:M].clone()
    xv, lo, taken = quantised(bd.xn[:M])[3], 0, 0
    for n in names:
        q = eng.w.q[f"blk.0.{n}.weight"]
        a, b = got[False][:, lo:lo + q.rows], got[True][:, lo:lo + q.rows]
        if kind == "mixed" and n == "attn_v" or kind == "signs" and n == "attn_k":
            assert torch.equal(a, b)
        else:
            w = values(q)
            off = (b.double().cpu() - xv @ w.T).abs()
            assert bool((off <= allowed(xv, w, q.k)).all()), n
            taken += 1
        lo += q.rows
    assert taken == 2


# ---- norms of large and of small rows -------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("K", [64, 512, 1024, 2048, 4096, 16384])
def test_norms_of_rows_whose_squares_pass_32_bits(K):
    """Squares of 2^70 and of 2^-80 are no fp32 numbers, their norm is.  One large value among ordinary ones, and blocks that vanish beside
    others, too."""
    from bloomery_b200.ops.fp4 import Fp4Rows, fp4_rows
    x = make(7, K, torch.float32, seed=K)
    x[1] *= 2.0 ** 70
    x[2] *= 2.0 ** -80
    x[3, K // 2] = 3e38
    x[4, :K // 2] *= 2.0 ** -75
    x[5] = x[5].sign() * 2.0 ** -62
    x[6] = 2.0 ** 127
    gain = (1 + 0.3 * torch.randn(K, generator=torch.Generator().manual_seed(1))).to(DEV)
    out = Fp4Rows(7, K, DEV)
    fp4_rows(x, out, gain=gain)
    r = (1 / x.double().square().mean(1, keepdim=True).sqrt()).float()
    want = quantised(x * r * gain)
    # ordinary rows (0, 4): their root may be the next fp32 number, 2^-23 away; behind it two products and a quotient round on either side,
    # 2^-24 each
    g = parts(out.data, K)[2].double()
    assert bool(((g - want[2].double()).abs() <= 2.0 ** -21 * want[2].double()).all())
    odd = [1, 2, 3, 5, 6]
    same(out.data[odd], K, tuple(t[odd] for t in want))


@gpu
@pytest.mark.parametrize("T", [3, 9])
def test_experts_of_tokens_whose_squares_pass_32_bits(T):
    c = case(T, 16, 4, 256, 512, seed=70 + T)
    x, rest = c[0], c[1:]
    x[1] *= 2.0 ** 70
    x[2] *= 2.0 ** -80
    gain = (1 + 0.3 * torch.randn(512, generator=torch.Generator().manual_seed(1))).to(DEV)
    r = (1 / x.double().square().mean(1, keepdim=True).sqrt()).float()
    want, tol = oracle(x * r * gain, *rest[:2], *(w[1] for w in rest[2:]))
    out = torch.empty(T, 512, device=DEV)
    run(x, *rest, out_f32=out, gain=gain)
    off = (out.double().cpu() - want).abs()
    assert bool((off <= tol + 5 * 2.0 ** -24 * want.abs()).all())


# ---- one scale for all rows -----------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_given_scales_over_the_whole_range(dtype):
    """Six times a scale past 5.6e37 is no fp32 number."""
    from bloomery_b200.ops.fp4 import Fp4Rows, fp4_rows
    K = 256
    x = make(24, K, torch.float32, seed=4)
    x *= torch.exp2(torch.linspace(-40, 125, 24)).to(DEV)[:, None] / x.abs().amax(1, keepdim=True)
    x = x.to(dtype)
    for scale in (2.0 ** -100, 1e-20, 1.0, 5e37, 5.7e37, 1e38, 2.0 ** 127, 3.4e38):
        out, s = Fp4Rows(24, K, DEV), torch.tensor([scale], device=DEV)
        fp4_rows(x, out, tensor_scale=s)
        same(out.data, K, quantised(x, s.item()))


@gpu
def test_given_scales_that_are_no_number():
    """Every row becomes one whose products are NaN, as one with a value that is none."""
    from bloomery_b200.ops.fp4 import Fp4Rows, fp4_rows
    x = make(5, 128, torch.float32)
    for scale in (math.nan, math.inf):
        out = Fp4Rows(5, 128, DEV)
        out.data.fill_(0x55)
        fp4_rows(x, out, tensor_scale=torch.tensor([scale], device=DEV))
        codes, scales, g = parts(out.data, 128)
        assert g.isnan().all() and not codes.any() and not scales.any()


# ---- stacks of a type of their own behind a layer of bf16 ones ------------------------------------------------------
@gpu
def test_grouped_products_keep_their_tiles():
    """A first routed layer in bf16 makes token tiles of 128 rows; the NVFP4 gate and up of the next one, whose down is Q8_0, run on the
    experts' tiles all the same."""
    from bloomery_b200.models.spec import tiny_qwen3moe
    from bloomery_b200.models.weights import Weights, synth_tensors
    from bloomery_b200.runtime.batch_decode import BatchDecode
    from bloomery_b200.runtime.engine import DecodeEngine
    spec = tiny_qwen3moe()
    kinds = {m: list(synth_tensors(spec, DEV, seed=3, mix=m)) for m in ("NVFP4", "BF16", "Q8_0")}

    def kind(name):
        return "NVFP4" if "_exps" not in name else "BF16" if name.startswith("blk.0.") else "Q8_0" if "down" in name else "NVFP4"
    items = (kinds[kind(a[0])][i] for i, a in enumerate(kinds["NVFP4"]))
    eng = DecodeEngine(Weights.from_items(spec, items, DEV), n_slots=1, slot_ctx=256)
    bd = BatchDecode(eng, max_rows=64)
    assert bd.moe_tiles.tile_rows == 128
    bd.fp4_native = True
    M, k, gen = 64, spec.n_used, torch.Generator().manual_seed(5)
    xn = torch.randn(M, spec.hidden, generator=gen).bfloat16().to(DEV)
    ids = torch.stack([torch.randperm(spec.n_expert, generator=gen)[:k] for _ in range(M)]).to(torch.int32)
    bd.x.zero_()
    for _ in bd.experts(1, M, bd.x[:M], xn.clone(), ids.to(DEV), torch.rand(M, k, generator=gen).to(DEV), bd.dense_tiles[M]):
        pass
    act, slot = bd.act[:M * k].double().cpu(), bd.dst_row[:M * k].cpu()
    xv, H = quantised(xn)[3], spec.hidden
    g_, u_ = (values(eng.w.q[f"blk.1.ffn_{n}_exps.weight"]).view(spec.n_expert, -1, H) for n in ("gate", "up"))
    assert slot.sort().values.tolist() == list(range(M * k))
    for i, s in enumerate(slot.tolist()):
        v, e = xv[s // k:s // k + 1], int(ids[s // k, s % k])
        g, u = v @ g_[e].T, v @ u_[e].T
        want = g * torch.sigmoid(g) * u
        # the factor's slope is at most 1.1; the exponential and the quotient are off by a few units of 2^-22
        tg, tu = allowed(v, g_[e], H), allowed(v, u_[e], H)
        tol = 1.1 * tg * (u.abs() + tu) + (g.abs() + tg) * tu + (2.0 ** -8 + 2.0 ** -19) * want.abs() + 1e-30
        assert bool(((act[i] - want[0]).abs() <= tol[0]).all()), i


@gpu
def test_grouped_fp8_products_keep_their_tiles():
    """The same layers with FP8 gate and up: tiles of 128 rows are no case of the E4M3 kernel, so they run as without it."""
    from bloomery_b200.models.spec import tiny_qwen3moe
    from bloomery_b200.models.weights import Weights, synth_tensors
    from bloomery_b200.runtime.batch_decode import BatchDecode
    from bloomery_b200.runtime.engine import DecodeEngine
    spec = tiny_qwen3moe()
    kinds = {m: list(synth_tensors(spec, DEV, seed=3, mix=m)) for m in ("FP8_B128", "BF16")}
    items = (kinds["BF16" if "_exps" in a[0] and a[0].startswith("blk.0.") else "FP8_B128"][i] for i, a in enumerate(kinds["BF16"]))
    eng = DecodeEngine(Weights.from_items(spec, items, DEV), n_slots=1, slot_ctx=256)
    bd = BatchDecode(eng, max_rows=64)
    assert bd.moe_tiles.tile_rows == 128
    M, k, gen = 64, spec.n_used, torch.Generator().manual_seed(5)
    xn = torch.randn(M, spec.hidden, generator=gen).bfloat16().to(DEV)
    ids = torch.stack([torch.randperm(spec.n_expert, generator=gen)[:k] for _ in range(M)]).to(torch.int32).to(DEV)
    wts = torch.rand(M, k, generator=gen).to(DEV)
    got = []
    for native in (False, True):
        bd.fp8_native = native
        bd.x.zero_()
        for _ in bd.experts(1, M, bd.x[:M], xn.clone(), ids, wts, bd.dense_tiles[M]):
            pass
        got.append(bd.x[:M].clone())
    assert bool((got[0] != 0).any()) and torch.equal(*got)


@gpu
def test_bf16_stacks_behind_a_quantised_layer():
    """A second routed layer in bf16 gives what it gives behind a bf16 one."""
    from bloomery_b200.models.spec import tiny_qwen3moe
    from bloomery_b200.models.weights import Weights, synth_tensors
    from bloomery_b200.runtime.batch_decode import BatchDecode
    from bloomery_b200.runtime.engine import DecodeEngine
    spec = tiny_qwen3moe()
    kinds = {m: list(synth_tensors(spec, DEV, seed=3, mix=m)) for m in ("Q8_0", "BF16")}
    M, k, gen = 64, spec.n_used, torch.Generator().manual_seed(5)
    xn = torch.randn(M, spec.hidden, generator=gen).bfloat16().to(DEV)
    ids = torch.stack([torch.randperm(spec.n_expert, generator=gen)[:k] for _ in range(M)]).to(torch.int32).to(DEV)
    wts = torch.rand(M, k, generator=gen).to(DEV)
    got = []
    for first in ("Q8_0", "BF16"):
        items = (kinds[first if a[0].startswith("blk.0.") else "BF16"][i] for i, a in enumerate(kinds["BF16"]))
        eng = DecodeEngine(Weights.from_items(spec, items, DEV), n_slots=1, slot_ctx=256)
        bd = BatchDecode(eng, max_rows=64)
        bd.x.zero_()
        for _ in bd.experts(1, M, bd.x[:M], xn.clone(), ids, wts, bd.dense_tiles[M]):
            pass
        got.append(bd.x[:M].clone())
    assert bool((got[0] != 0).any()) and torch.equal(*got)


# ---- no rows --------------------------------------------------------------------------------------------------------
@gpu
def test_products_of_no_rows():
    from bloomery_b200.ops.fp4 import Fp4Rows, fp4_gemm, fp4_rows, fp4_tiles
    rows, (q, _) = Fp4Rows(4, 128, DEV), weight(16, 128)
    fp4_rows(torch.zeros(0, 128, device=DEV), rows)
    fp4_gemm(rows, q, fp4_tiles(0, DEV), out_f32=torch.empty(0, 16, device=DEV))
    out = torch.full((3, 16), 7.0, device=DEV)
    fp4_gemm(rows, q, fp4_tiles(0, DEV), out_f32=out)
    assert (out == 7).all()


# ---- the lever ------------------------------------------------------------------------------------------------------
@gpu
def test_the_pass_over_ranks_keeps_16_bits():
    from bloomery_b200.models.spec import tiny_qwen3moe
    from bloomery_b200.models.weights import Weights, synth_tensors
    from bloomery_b200.parallel.batch_dist import ShardedBatchDecode
    from bloomery_b200.runtime.batch_decode import BatchDecode
    from bloomery_b200.runtime.engine import DecodeEngine
    from bloomery_b200.utils import levers
    spec = tiny_qwen3moe()
    eng = DecodeEngine(Weights.from_items(spec, synth_tensors(spec, DEV, seed=3, mix="NVFP4"), DEV), n_slots=1, slot_ctx=256)
    try:
        levers.at_main({"BLOOMERY_FP4_NATIVE": "1"})
        assert BatchDecode(eng, max_rows=16).fp4_native
        assert not ShardedBatchDecode(eng, 0, 1, max_rows=16, local_only=True).fp4_native
    finally:
        levers.at_main()


def by_definition(X, W):
    """(X [rows, K] in NVFP4) W^T in 64 bits, and how far fp32 sums may be off."""
    xv = quantised(X)[3]
    return xv @ W.T, allowed(xv, W, W.shape[1])


@gpu
@pytest.mark.parametrize("T,experts", [(64, 16), (131, 16), (300, 16), (131, 32)])
def test_a_layer_of_a_prompt_is_the_sum_of_its_parts(T, experts):
    """A model of one layer: every product of a prompt against the definition, of the rows that the path itself has in front of it."""
    from dataclasses import replace
    from bloomery_b200.models.spec import tiny_qwen3moe
    from bloomery_b200.models.weights import Weights, synth_tensors
    from bloomery_b200.runtime.engine import DecodeEngine
    from bloomery_b200.runtime.prefill import GemmPrefill
    spec = replace(tiny_qwen3moe(), n_layer=1, n_expert=experts)
    eng = DecodeEngine(Weights.from_items(spec, synth_tensors(spec, DEV, seed=3, mix="NVFP4"), DEV), n_slots=1, slot_ctx=1024)
    pf = GemmPrefill(eng)
    pf.fp4_native = True
    ids = torch.randint(0, spec.vocab, (T,), generator=torch.Generator().manual_seed(T)).tolist()
    pf.run(0, ids)
    torch.cuda.synchronize()
    eng.check_fault()
    assert "Ap" not in pf._buf and not pf._resident               # nothing is laid out, or kept, that this path does not read
    w, H, E, k, n = eng.w, spec.hidden, spec.n_expert, spec.n_used, T * spec.n_used
    get = lambda name, *shape: pf._buf[name][:math.prod(shape)].view(*shape).double().cpu()       # noqa: E731
    normed = lambda v, gain: v * (1 / (v.double().square().mean(1, keepdim=True) + spec.rms_eps).sqrt()).float() * gain      # noqa: E731
    from bloomery_b200.ops import decode as K
    x0 = torch.empty(T, H, device=DEV)
    K.embed_rows(torch.tensor(ids, dtype=torch.int32, device=DEV), T, w.q["token_embd.weight"], spec.vocab, x0, eng.fault)
    # the projections, of the embeddings behind their norm: its root may be the next fp32 number
    W = torch.cat([values(w.q[f"blk.0.attn_{m}.weight"]) for m in "qkv"])
    want, tol = by_definition(normed(x0, w.f["blk.0.attn_norm.weight"]), W)
    off = (get("qkv", T, W.shape[0]) - want).abs()
    assert bool((off <= tol + 2.0 ** -21 * want.abs()).all())
    # the o projection, seen behind the experts: x = embeddings + o + experts
    attn = pf._buf["attn"][:T * spec.q_rows].view(T, spec.q_rows)
    o, tol_o = by_definition(attn, values(w.q["blk.0.attn_output.weight"]))
    x1 = x0.double().cpu() + o
    # the experts' rows: the router's input, in bf16
    split = T >= 128 and E % 32 == 0                              # the router's product in two halves: the rows are the high ones
    rows = (pf._buf["xn3"][:T * 3 * H].view(T, 3 * H)[:, :H] if split else pf._buf["xn"][:T * H].view(T, H)).contiguous()
    ref = normed(x1.float().to(DEV), w.f["blk.0.ffn_norm.weight"]).double().cpu()
    assert bool(((rows.double().cpu() - ref).abs() <= (2.0 ** -8 + 2.0 ** -12) * ref.abs() + 1e-4).all())
    sel, wts, slot = get("ids", T, k).long(), get("wts", T, k), get("dst_row", n).long()
    act, out = get("act", n, spec.moe_inter), get("slot_out", n, H)
    gate, up, down = (values(w.q[f"blk.0.ffn_{m}_exps.weight"]).view(E, -1, kk) for m, kk in (("gate", H), ("up", H), ("down", spec.moe_inter)))
    xv, av = quantised(rows)[3], quantised(act.bfloat16())[3]
    for e in range(E):
        at = (sel.view(-1)[slot] == e).nonzero().flatten()       # places of this expert's slots
        if not len(at):
            continue
        v = xv[slot[at] // k]
        g, u = v @ gate[e].T, v @ up[e].T
        tg, tu, a = allowed(v, gate[e], H), allowed(v, up[e], H), g * torch.sigmoid(g) * u
        # the factor's slope is at most 1.1; the exponential and the quotient are off by a few units of 2^-22
        tol = 1.1 * tg * (u.abs() + tu) + (g.abs() + tg) * tu + (2.0 ** -8 + 2.0 ** -19) * a.abs() + 1e-30
        assert bool(((act[at] - a).abs() <= tol).all()), e
        f = wts.view(-1)[slot[at], None]
        d = f * (av[at] @ down[e].T)
        assert bool(((out[slot[at]] - d).abs() <= f * allowed(av[at], down[e], spec.moe_inter) + 2.0 ** -23 * d.abs() + 1e-30).all()), e
    x2 = x1 + out.view(T, k, H).sum(1)
    tol = tol_o + (k + 2) * 2.0 ** -23 * (x1.abs() + out.view(T, k, H).abs().sum(1))
    assert bool(((get("x", T, H) - x2).abs() <= tol).all())


# ---- every form of the kernels --------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("N", [2040, 4096, 8200, 20000])
@pytest.mark.parametrize("M", [20, 60, 100, 200])
def test_products_in_every_tile(M, N, gated):
    """Tiles of 16 to 128 weight rows, by how many find a processor at once, and of 32 to 256 tokens."""
    from bloomery_b200.ops.fp4 import Fp4Rows, fp4_gemm, fp4_rows, fp4_tile_rows
    from bloomery_b200.ops.gemm import TileTable
    K = 192
    x, rows, status = make(M, K, seed=N), Fp4Rows(M, K, DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    fp4_rows(x, rows)
    (w1, v1), (w2, v2) = weight(N, K, 1), weight(N, K, 2)
    out = torch.empty(M, N, dtype=torch.bfloat16, device=DEV)
    tiles = TileTable.dense(M, DEV, fp4_tile_rows(M, gated=gated), host=True)
    fp4_gemm(rows, w1, tiles, W2=w2 if gated else None, out_bf16=out, status=status)
    xv = quantised(x)[3]
    g, tg = xv @ v1.T, allowed(xv, v1, K)
    want, tol = g, tg
    if gated:
        u, tu = xv @ v2.T, allowed(xv, v2, K)
        want = g * torch.sigmoid(g) * u
        # the factor's slope is at most 1.1; the exponential and the quotient are off by a few units of 2^-22
        tol = 1.1 * tg * (u.abs() + tu) + (g.abs() + tg) * tu + 2.0 ** -19 * want.abs()
    assert int(status) == 0
    assert bool(((out.double().cpu() - want).abs() <= tol + 2.0 ** -8 * (want.abs() + tol)).all())


@gpu
@pytest.mark.parametrize("T,E,k,inter,H", [(1, 4, 2, 256, 512), (2, 4, 2, 256, 2048), (1, 16, 8, 768, 2048), (4, 32, 8, 768, 512), (3, 5, 3, 2048, 4096),
                                           (3, 20, 16, 128, 512), (4, 40, 16, 64, 4096), (5, 9, 4, 320, 4096)])
def test_few_tokens_behind_their_norm(T, E, k, inter, H):
    """Every height of a tile of one to four tokens, and more slots than that form has room for."""
    c = case(T, E, k, inter, H, seed=20 + T)
    gain = (1 + 0.3 * torch.randn(H, generator=torch.Generator().manual_seed(1))).to(DEV)
    x, rest = c[0], c[1:]
    r = (1 / (x.double().square().mean(1, keepdim=True) + 1e-6).sqrt()).float()
    want, tol = oracle(x * r * gain, *rest[:2], *(w[1] for w in rest[2:]))
    want = want + x.double().cpu()
    out = x.clone()
    work = run(out, *rest, out_f32=out, resid=out, gain=gain, eps=1e-6)
    # twice the oracle's: its rows may differ by a unit of the root's last place (and a code on the edge with it)
    off = (out.double().cpu() - want).abs()
    assert bool((off <= 2 * tol + (k + 1) * 2.0 ** -24 * (want.abs() + x.double().cpu().abs())).all()), float((off / tol).max())
    again = torch.empty(T, H, device=DEV)
    for _ in range(3):
        run(x, *rest, work=work, out_f32=again, resid=x, gain=gain, eps=1e-6)
        assert torch.equal(again, out)


@gpu
def test_the_dense_layers_and_the_shared_expert():
    """Both halves of a SwiGLU pair against the definition, in a model with latent attention."""
    from bloomery_b200.runtime.batch_decode import BatchDecode
    spec, eng, rows = engine("latent")
    bd = BatchDecode(eng, max_rows=16)
    bd.fp4_native = True
    M, gen = 16, torch.Generator().manual_seed(5)
    xn = torch.randn(M, spec.hidden, generator=gen).bfloat16().to(DEV)
    x = torch.randn(M, spec.hidden, generator=gen).to(DEV)
    q = lambda name: values(eng.w.q[name + ".weight"])                                            # noqa: E731
    for stem, suffix, act in (("blk.0.ffn_", "", bd.dact), ("blk.1.ffn_", "_shexp", bd.sh_act)):
        bd.x[:M].copy_(x)
        if suffix:
            bd.shared_expert(1, M, xn, bd.dense_tiles[M], bd.x[:M], bd.x[:M])
        else:
            for _ in bd.dense_ffn(0, M, bd.x[:M], xn, bd.dense_tiles[M]):
                pass
        torch.cuda.synchronize()
        (g, tg), (u, tu) = (by_definition(xn, q(stem + n + suffix)) for n in ("gate", "up"))
        a = g * torch.sigmoid(g) * u
        tol = 1.1 * tg * (u.abs() + tu) + (g.abs() + tg) * tu + (2.0 ** -8 + 2.0 ** -19) * a.abs() + 1e-30
        assert bool(((act[:M].double().cpu() - a).abs() <= tol).all())
        y, tol = by_definition(act[:M], q(stem + "down" + suffix))
        want = y + x.double().cpu()
        assert bool(((bd.x[:M].double().cpu() - want).abs() <= tol + 2.0 ** -23 * want.abs()).all())


# ---- tables built from rows a group ---------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("tile_rows", [32, 64, 128, 256])
def test_tables_have_tiles_of_their_own_rows(tile_rows):
    """Every row of ragged groups is in one tile, and the product over the table has them all."""
    from bloomery_b200.ops.fp4 import Fp4Rows, fp4_gemm, fp4_rows
    from bloomery_b200.ops.gemm import TileTable
    groups, K, N = [0, 1, 300, 33, 128, 64, 0, 7], 128, 72
    M = sum(groups)
    t = TileTable(M, len(groups), DEV, tile_rows)
    t.build(torch.tensor(groups, dtype=torch.int32, device=DEV))
    want, lo = [], 0
    for g, n in enumerate(groups):
        want += [[g, lo + r, lo + n, 0] for r in range(0, n, tile_rows)]
        lo += n
    assert t.mtiles[:int(t.n_mtiles)].tolist() == want
    x, rows, (q, v) = make(M, K, seed=2), Fp4Rows(M, K, DEV), weight(N, K, 3, len(groups))
    fp4_rows(x, rows)
    out = torch.empty(M, N, device=DEV)
    fp4_gemm(rows, q, t, out_f32=out)
    xv, lo = quantised(x)[3], 0
    for g, n in enumerate(groups):
        a = xv[lo:lo + n]
        assert bool(((out[lo:lo + n].double().cpu() - a @ v[g].T).abs() <= allowed(a, v[g], K)).all())
        lo += n
