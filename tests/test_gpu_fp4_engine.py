"""Passes and prompts of an NVFP4 model with its activations in NVFP4 too.

A value in four bits is off by a tenth of itself or so (a step is half of the value next to 1, a fifth next to 5, evenly spread: 0.09 of
the block's rms).  A pass of the tiny model has 16 such products on the way of the residual stream, whose errors add up like
noise: 0.4 of the logits' own size at most, a cosine of 0.92.  The bits of the operators are tested elsewhere; here the passes are
held to themselves, and to the 16-bit ones within that."""
import gc

import pytest
import torch

from test_gpu_fp4 import DEV
from test_gpu_fp4_moe import oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_engine_left():
    """Engines hold their prompt paths and those the engines: their graphs must not be taken down while a later test captures one."""
    yield
    gc.collect()


def engine(n_slots, native=True, seed=3, spec=None):
    from bloomery_b200.models.spec import tiny_qwen3moe
    from bloomery_b200.models.weights import Weights, synth_tensors
    from bloomery_b200.runtime.engine import DecodeEngine
    spec = spec or tiny_qwen3moe()
    w = Weights.from_items(spec, synth_tensors(spec, DEV, seed=seed, mix="NVFP4"), DEV)
    return spec, DecodeEngine(w, n_slots=n_slots, slot_ctx=1024)


def prompts(spec, n, seed=7):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, spec.vocab, (5 + 3 * (i % 7),), generator=g).tolist() for i in range(n)]


def cosine(a, b):
    a, b = a.double(), b.double()
    return (a * b).sum(-1) / (a.norm(dim=-1) * b.norm(dim=-1))


@pytest.mark.parametrize("n_rows", [2, 13, 40, 64])
def test_a_pass_on_four_bits(n_rows):
    from bloomery_b200.runtime.batch_decode import BatchDecode
    spec, eng = engine(n_rows)
    rows = [(slot, eng.prefill(slot, p, gemm=False), len(p)) for slot, p in enumerate(prompts(spec, n_rows))]
    got = {}
    for native in (False, True):
        bd = BatchDecode(eng, max_rows=64)
        assert not bd.fp4_native                                  # off unless asked for
        bd.fp4_native = native
        tok = bd.step(rows)
        got[native] = bd.logits[:n_rows].clone()
        assert bd.step(rows) == tok                               # the captured pass again
        assert torch.equal(bd.logits[:n_rows], got[native])
        if native:
            assert bd._moe_work is not None
    assert got[True].isfinite().all()
    assert float(cosine(got[False], got[True]).min()) > 0.92


def test_a_row_does_not_depend_on_the_bucket_around_it():
    """Three rows alone, among 13 and, behind passes that were captured before, among 40: the same bits."""
    from bloomery_b200.runtime.batch_decode import BatchDecode
    spec, eng = engine(40)
    rows = [(slot, eng.prefill(slot, p, gemm=False), len(p)) for slot, p in enumerate(prompts(spec, 40))]
    bd = BatchDecode(eng, max_rows=64)
    bd.fp4_native = True
    seen = []
    for n in (3, 13, 40, 3):
        bd.step(rows[:n])
        seen.append(bd.logits[:3].clone())
    assert torch.equal(seen[0], seen[1]) and torch.equal(seen[0], seen[3])
    # in the bucket of 64 attention walks other key segments: rounding in front of a quantiser
    assert float(cosine(seen[0], seen[2]).min()) > 0.92


def test_the_expert_half_of_a_layer_is_the_sum_of_its_parts():
    """The rows that a pass leaves behind a layer's experts, against the definition: norm, rows in four bits, both products."""
    from bloomery_b200.formats import planes
    from bloomery_b200.ops import decode as K
    from bloomery_b200.runtime.batch_decode import BatchDecode
    spec, eng = engine(4)
    bd = BatchDecode(eng, max_rows=16)
    bd.fp4_native = True
    g = torch.Generator().manual_seed(5)
    M = 16
    x = torch.randn(M, spec.hidden, generator=g).to(DEV)
    ids = torch.stack([torch.randperm(spec.n_expert, generator=g)[:spec.n_used] for _ in range(M)]).to(torch.int32)
    wts = torch.rand(M, spec.n_used, generator=g)
    bd.x[:M].copy_(x)
    for _ in bd.experts(0, M, bd.x[:M], bd.xn[:M], ids.to(DEV), wts.to(DEV), bd.dense_tiles[M]):
        pass
    w = eng.w
    gain = w.f["blk.0.ffn_norm.weight"]
    r = (1 / (x.double().square().mean(1, keepdim=True) + spec.rms_eps).sqrt()).float()

    def values(name):
        q = w.q[f"blk.0.{name}.weight"]
        flat = q.data.reshape(-1, q.data.shape[-1]).cpu()
        ts = flat[:, q.k // 2 + q.k // 16:q.k // 2 + q.k // 16 + 4].contiguous().view(torch.float32).double()
        v = planes.nvfp4_dequantize(flat[:, :q.k // 2], flat[:, q.k // 2:q.k // 2 + q.k // 16], 1.0).double() * ts
        return v.view(*q.data.shape[:-1], q.k)
    want, tol = oracle((x * r * gain).cpu(), ids, wts, *(values(n) for n in ("ffn_gate_exps", "ffn_up_exps", "ffn_down_exps")))
    want = want + x.double().cpu()
    # the root of the mean square may be the next fp32 number: a code on the edge moves as one of the oracle's does
    tol = tol * 2 + 8 * 2.0 ** -24 * (want.abs() + x.double().cpu().abs())
    off = (bd.x[:M].double().cpu() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("T", [70, 200, 700])
def test_prompts_on_four_bits(T):
    spec, eng = engine(2)
    g = torch.Generator().manual_seed(T)
    prompt = torch.randint(0, spec.vocab, (T,), generator=g).tolist()
    got = {}
    for slot, native in enumerate((False, True)):
        eng._gemm_prefill = None
        eng.prefill(slot, prompt[:1], gemm=False)
        eng.cut(slot, 0)
        from bloomery_b200.runtime.prefill import GemmPrefill
        eng._gemm_prefill = GemmPrefill(eng)
        assert not eng._gemm_prefill.fp4_native
        eng._gemm_prefill.fp4_native = native
        eng.prefill(slot, prompt, gemm=True)
        got[native] = eng.logits[0].clone()
        if native:
            assert eng._gemm_prefill._native_fp4() and not eng._gemm_prefill._resident       # nothing was expanded
        eng.check_fault()
    assert got[True].isfinite().all()
    assert float(cosine(got[False], got[True])) > 0.92


def test_models_that_have_no_place_for_it_go_on_as_they_were():
    """Other weight types, and block scales with a sign."""
    from bloomery_b200.ops.fp4 import fp4_supports
    from bloomery_b200.models.spec import tiny_qwen3moe
    from bloomery_b200.models.weights import Weights, synth_tensors
    from bloomery_b200.runtime.batch_decode import BatchDecode
    from bloomery_b200.runtime.engine import DecodeEngine
    spec = tiny_qwen3moe()
    eng = DecodeEngine(Weights.from_items(spec, synth_tensors(spec, DEV, seed=3, mix="Q8_0"), DEV), n_slots=16, slot_ctx=256)
    rows = [(slot, eng.prefill(slot, p, gemm=False), len(p)) for slot, p in enumerate(prompts(spec, 16))]
    seen = []
    for native in (False, True):
        bd = BatchDecode(eng, max_rows=16)
        bd.fp4_native = native
        bd.step(rows)
        seen.append(bd.logits[:16].clone())
    assert torch.equal(*seen)
    spec, eng = engine(1)
    q = eng.w.q["blk.0.attn_q.weight"]
    assert fp4_supports(q)
    q.data[3, q.k // 2 + 1] |= 0x80
    assert not fp4_supports(q)
