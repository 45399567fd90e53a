"""The routed experts of a few tokens in NVFP4 against the definition in 64 bits.

Between the two products the activations are quantised again.  fp32 sums and exponentials in front of that differ from the exact ones by
a relative 2^-17 at most at these depths, so a value next to a midpoint may become the other neighbour: a step of a code is at most
a third of its value (2 to 3 and the like; half of a step next to zero, of 0.5 / 6 of the block's largest).  The oracle counts them:
outputs are compared with the products of its own quantised activations, and every activation within 2^-16 of a midpoint may move its
weight's share."""
import pytest
import torch

from test_gpu_fp4 import DEV, allowed, make, quantised, weight

gpu = pytest.mark.gpu


def oracle(x, ids, wts, gv, uv, dv):
    """(values fp64 [T, H], how far fp32 sums and codes on the edge may move them)."""
    T, H = x.shape[0], dv[0].shape[0]
    xv = quantised(x)[3]
    out, tol = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    for t in range(T):
        for j, e in enumerate(ids[t].tolist()):
            if not 0 <= e < len(gv):
                continue
            v = xv[t:t + 1]
            g, u = v @ gv[e].T, v @ uv[e].T
            a = g * torch.sigmoid(g) * u
            ta = 1.1 * allowed(v, gv[e], v.shape[1]) * u.abs() + g.abs() * allowed(v, uv[e], v.shape[1]) + 2.0 ** -19 * a.abs()
            av = quantised(a.float())[3]
            # a code may change where the value, its block's scale or the row's moves across a midpoint
            lo, hi = (quantised((a.sign() * (a.abs() + s * (ta + 2.0 ** -18 * a.abs())).clamp_min(0)).float())[3] for s in (-1, 1))
            move = torch.maximum((lo - av).abs(), (hi - av).abs()) + 2.0 ** -17 * av.abs()
            w = float(wts[t, j])
            out[t] += w * (av @ dv[e].T)[0]
            tol[t] += abs(w) * (allowed(av, dv[e], av.shape[1]) + move @ dv[e].abs().T)[0]
    return out, tol


def case(T, E, k, inter, H, seed, away=0, dtype=torch.float32, same=False):
    gen = torch.Generator().manual_seed(seed)
    x = make(T, H, dtype, seed=seed)
    ids = torch.stack([torch.randperm(E, generator=gen)[:k] for _ in range(T)]).to(torch.int32)
    if same:
        ids[:] = 1                                                # every slot of every token: one expert
    for i in torch.randperm(T * k, generator=gen)[:away].tolist():
        ids.view(-1)[i] = (-1, E, -7, 1 << 30)[i % 4]             # another tier's
    wts = torch.rand(T, k, generator=gen)
    return x, ids, wts, weight(inter, H, seed, E), weight(inter, H, seed + 1, E), weight(H, inter, seed + 2, E)


def run(x, ids, wts, g, u, d, work=None, **kw):
    from bloomery_b200.ops.fp4 import Fp4MoeWork, fp4_moe
    T, k = ids.shape
    work = work or Fp4MoeWork(T, k, x.shape[1], g[0].rows, len(g[1]), DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    fp4_moe(x, ids.to(DEV), wts.to(DEV), g[0], u[0], d[0], work, status=status, **kw)
    assert int(status) == 0
    return work


@gpu
@pytest.mark.parametrize("T,E,k,inter,H,away", [(1, 16, 4, 256, 512, 0), (5, 16, 4, 256, 512, 6), (32, 16, 4, 192, 320, 0), (33, 7, 3, 128, 1024, 20),
                                                (64, 24, 8, 320, 576, 0), (64, 3, 2, 64, 64, 5), (2, 130, 16, 64, 192, 0), (9, 4, 1, 2112, 2048, 1),
                                                (3, 4, 2, 64, 192, 6), (64, 512, 16, 64, 64, 100), (7, 2, 2, 64, 8192, 0), (4, 3, 1, 8192, 64, 0)])
def test_tokens_through_their_experts(T, E, k, inter, H, away):
    c = case(T, E, k, inter, H, seed=T, away=away)
    out = torch.full((T + 1, H + 4), 5.0, device=DEV)
    resid = torch.randn(T, H, device=DEV)
    work = run(*c, out_f32=out[:T, :H], resid=resid)
    want, tol = oracle(*c[:3], *(w[1] for w in c[3:]))
    want = want + resid.double().cpu()
    tol = tol + (k + 1) * 2.0 ** -24 * (want.abs() + resid.double().cpu().abs())
    off = (out[:T, :H].double().cpu() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    assert (out[T] == 5).all() and (out[:, H:] == 5).all()
    first = out[:T, :H].clone()
    for _ in range(3):                                            # the scratch is ready again, and the bits are the same
        out.fill_(5.0)
        run(*c, work=work, out_f32=out[:T, :H], resid=resid)
        assert torch.equal(out[:T, :H], first)


@gpu
def test_one_expert_for_every_slot():
    c = case(64, 5, 4, 128, 256, seed=3, same=True)
    out = torch.empty(64, 256, device=DEV)
    run(*c, out_f32=out)
    want, tol = oracle(*c[:3], *(w[1] for w in c[3:]))
    off = (out.double().cpu() - want).abs()
    assert bool((off <= tol + 5 * 2.0 ** -24 * want.abs()).all())


@gpu
def test_norm_bf16_rows_and_output_in_place():
    T, E, k, inter, H = 12, 16, 4, 256, 512
    c = case(T, E, k, inter, H, seed=8)
    x, rest = c[0], c[1:]
    gain = (1 + 0.3 * torch.randn(H, generator=torch.Generator().manual_seed(1))).to(DEV)
    r = (1 / (x.double().square().mean(1, keepdim=True) + 1e-6).sqrt()).float()
    want, tol = oracle(x * r * gain, *rest[:2], *(w[1] for w in rest[2:]))
    want = want + x.double().cpu()
    y = x.clone()
    run(y, *rest, out_f32=y, resid=y, gain=gain, eps=1e-6)        # the residual stream in its place
    off = (y.double().cpu() - want).abs()
    assert bool((off <= tol + 5 * 2.0 ** -24 * (want.abs() + x.double().cpu().abs())).all())
    xb = x.bfloat16()
    out = torch.empty(T, H, dtype=torch.bfloat16, device=DEV)
    run(xb, *rest, out_bf16=out)
    want, tol = oracle(xb, *rest[:2], *(w[1] for w in rest[2:]))
    off = (out.double().cpu() - want).abs()
    assert bool((off <= tol + 2.0 ** -8 * (want.abs() + tol)).all())


@gpu
def test_a_row_that_is_not_finite_stays_alone():
    c = case(6, 16, 4, 128, 256, seed=5)
    out, ref = torch.empty(6, 256, device=DEV), torch.empty(6, 256, device=DEV)
    run(*c, out_f32=ref)
    c[0][2, 100] = float("nan")
    c[0][4, 3] = float("inf")
    run(*c, out_f32=out)
    assert out[[2, 4]].isnan().all()
    assert torch.equal(out[[0, 1, 3, 5]], ref[[0, 1, 3, 5]])


@gpu
def test_calls_on_two_streams_and_in_graphs():
    """Two calls at once, more CTAs than processors between them; a captured call replayed with other tokens and other experts."""
    from bloomery_b200.ops.fp4 import Fp4MoeWork, fp4_moe
    cs = [case(40, 64, 8, 256, 512, seed=s) for s in (1, 2)]
    outs = [torch.empty(40, 512, device=DEV) for _ in cs]
    works = [run(*c, out_f32=o) for c, o in zip(cs, outs)]
    want = [o.clone() for o in outs]
    on = [(c[0], c[1].to(DEV), c[2].to(DEV), c[3][0], c[4][0], c[5][0]) for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, a, w, o in zip(streams, on, works, outs):
            with torch.cuda.stream(s):
                fp4_moe(*a, w, out_f32=o)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    x, ids, wts = (t.clone() for t in on[0][:3])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fp4_moe(x, ids, wts, *on[0][3:], works[0], out_f32=outs[0])
        fp4_moe(x, ids, wts, *on[0][3:], works[0], out_f32=outs[1])
    other = case(40, 64, 8, 256, 512, seed=7, away=50)
    x.copy_(other[0]); ids.copy_(other[1]); wts.copy_(other[2])
    graph.replay()
    torch.cuda.synchronize()
    ref = torch.empty(40, 512, device=DEV)
    fp4_moe(x, ids, wts, *on[0][3:], Fp4MoeWork(40, 8, 512, 256, 64, DEV), out_f32=ref)
    assert torch.equal(outs[0], ref) and torch.equal(outs[1], ref)


@gpu
def test_a_wait_that_runs_out_is_reported():
    """Rows that are said to be taken and never come: the launch gives up after its limit, says so and leaves the card as it was."""
    from bloomery_b200.ops.fp4 import Fp4MoeWork, fp4_moe
    c = case(8, 16, 4, 256, 512, seed=4)
    args = (c[0], c[1].to(DEV), c[2].to(DEV), c[3][0], c[4][0], c[5][0])
    want, out = torch.empty(8, 512, device=DEV), torch.empty(8, 512, device=DEV)
    work, status = Fp4MoeWork(8, 4, 512, 256, 16, DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    fp4_moe(*args, work, out_f32=want, status=status)
    assert int(status) == 0
    work.data[:4].view(torch.int32).fill_(8)
    fp4_moe(*args, work, out_f32=out, status=status)
    assert int(status) == 1
    status.zero_()
    fp4_moe(*args, Fp4MoeWork(8, 4, 512, 256, 16, DEV), out_f32=out, status=status)
    assert int(status) == 0 and torch.equal(out, want)
