"""NVFP4 rows and their products against the definitions in 64 bits.

Codes and scales are decided exactly, so they are compared bit by bit.  A product's sum runs in fp32 on the tensor cores: K / 64 steps that
each lose at most one unit of their partial sum's last place (2^-23, should they cut instead of round), a few more inside a step
and in the two scales behind it, all relative to the sum of magnitudes."""
import math

import pytest
import torch

from bloomery_b200.formats import planes
from bloomery_b200.ops.decode import QWeight

gpu = pytest.mark.gpu
DEV = "cuda"
E2M1 = [0, .5, 1, 1.5, 2, 3, 4, 6]


def nearest(v, table):
    """Index of the value of a table next to v >= 0 (fp64), the even index of two as near."""
    mid = (table[1:] + table[:-1]) / 2
    lo, hi = torch.searchsorted(mid, v.contiguous()), torch.searchsorted(mid, v.contiguous(), right=True)
    return torch.where(lo % 2 == 0, lo, hi)


def quantised(x, tensor_scale=None):
    """(codes [M, K] 0..15, scale codes [M, K / 16], row scales fp32 [M], values fp64) of finite rows."""
    x = x.double().cpu()
    e4m3 = planes.e4m3_decode(torch.arange(0, 127, dtype=torch.uint8)).double()
    e2m1 = torch.tensor(E2M1, dtype=torch.float64)
    g = (x.abs().amax(1) / 2688).float() if tensor_scale is None else torch.full((len(x),), float(tensor_scale))
    g = g.clamp_min(2.0 ** -100)
    b = x.view(len(x), -1, 16)
    sc = nearest((b.abs().amax(2) / (6 * g.double()[:, None])).clamp_max(448), e4m3)
    d = (e4m3[sc].float() * g[:, None]).double().unsqueeze(-1)
    c = nearest((b.abs() / d.clamp_min(1e-300)).clamp_max(6), e2m1) * (sc > 0).unsqueeze(-1)
    values = torch.sign(b) * e2m1[c] * (e4m3[sc] * g.double()[:, None]).unsqueeze(-1)
    codes = c + 8 * ((b < 0) & (sc > 0).unsqueeze(-1))
    return codes.flatten(1), sc, g, values.flatten(1)


def parts(data, k):
    data = data.cpu()
    lo, hi = data[:, :k // 2] & 15, data[:, :k // 2] >> 4
    g = data[:, k // 2 + k // 16:k // 2 + k // 16 + 4].contiguous().view(torch.float32).flatten()
    return torch.stack([lo, hi], -1).flatten(1).long(), data[:, k // 2:k // 2 + k // 16].long(), g


def same(data, k, want):
    codes, sc, g = parts(data, k)
    assert torch.equal(g, want[2])
    assert torch.equal(sc, want[1])
    zero = (codes % 8 == 0) & (want[0] % 8 == 0)                 # a zero may keep its sign
    assert torch.equal(codes[~zero], want[0][~zero])


def make(M, K, dtype=torch.bfloat16, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=gen) * torch.exp(0.5 * torch.randn(K, generator=gen)) * torch.exp(torch.randn(M, 1, generator=gen))
    return x.to(dtype).to(DEV)


def weight(N, K, seed=0, groups=0):
    gen = torch.Generator().manual_seed(1000 + seed)
    w = torch.randn(max(1, groups) * N, K, generator=gen)
    packed, sc, ts = planes.nvfp4_quantize(w)
    data = planes.nvfp4_resident(packed, sc, ts * 0.01)
    v = planes.nvfp4_dequantize(packed, sc, 1.0).double() * float((ts * 0.01).float())
    if groups:
        data, v = data.view(groups, N, -1), v.view(groups, N, K)
    return QWeight(data.to(DEV).contiguous(), "NVFP4", K), v


def allowed(x, w, K):
    """fp32 sums of K products: see the module's text."""
    return (K / 64 + 8) * 2.0 ** -23 * (x.abs() @ w.abs().T) + 1e-30


@gpu
@pytest.mark.parametrize("M,K,dtype", [(1, 64, torch.bfloat16), (3, 192, torch.float16), (24, 2048, torch.bfloat16), (37, 4096 + 64, torch.float32),
                                       (5, 18432, torch.bfloat16), (2, 32768, torch.float16), (300, 512, torch.bfloat16)])
def test_rows_hold_the_nearest_codes(M, K, dtype):
    from bloomery_b200.ops.fp4 import Fp4Rows, fp4_rows
    x = make(M, K, dtype, seed=M)
    out = Fp4Rows(M + 2, K, DEV)
    out.data.fill_(0x55)
    fp4_rows(x, out)
    same(out.data[:M], K, quantised(x))
    assert bool((out.data[M:] == 0x55).all())                     # rows behind the last one stay


@gpu
def test_values_on_the_midpoints_go_to_the_even_code():
    """A block whose scale is a power of two, with values on every midpoint and one step to either side; a scale on a midpoint."""
    from bloomery_b200.ops.fp4 import Fp4Rows, fp4_rows
    mids = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.])
    up, down = (torch.nextafter(mids, torch.full_like(mids, s)) for s in (9., 0.))
    rows = []
    for size in (1.0, 2.0 ** -20, 2.0 ** 30, 1.0 / 3):
        for m in (mids, up, down):
            x = torch.zeros(64)
            x[:7], x[7] = m, 6.0
            x[16:23], x[23] = -m, 6.0
            x[32] = 6 * 448                                       # the row's scale is one
            x[48:64] = torch.linspace(0, 6 * (1 + 1 / 16), 16)    # its scale lies on a midpoint between 1 and 1.125
            rows.append(x * size)
    x = torch.stack(rows).to(DEV)
    out = Fp4Rows(len(rows), 64, DEV)
    fp4_rows(x, out)
    same(out.data, 64, quantised(x))


@gpu
def test_every_scale_and_step_is_met():
    """Blocks over forty powers of two, many of them a ratio away from a midpoint, under a row scale of 24 bits."""
    from bloomery_b200.ops.fp4 import Fp4Rows, fp4_rows
    gen = torch.Generator().manual_seed(3)
    x = torch.randint(-200, 201, (512, 128, 16), generator=gen).float() * torch.exp2(torch.randint(-24, 17, (512, 128, 1), generator=gen).float())
    x = x.view(512, 2048).bfloat16().to(DEV)
    out = Fp4Rows(512, 2048, DEV)
    fp4_rows(x, out)
    same(out.data, 2048, quantised(x))
    ts = torch.tensor([0.0123], device=DEV)
    fp4_rows(x, out, tensor_scale=ts)                             # most of it saturates, or vanishes
    same(out.data, 2048, quantised(x, ts.item()))


@gpu
def test_rows_of_zeros_and_rows_that_are_not_finite():
    from bloomery_b200.ops.fp4 import Fp4Rows, fp4_gemm, fp4_rows, fp4_tiles
    x = make(6, 256, torch.float32)
    x[1] = 0
    x[2, 17], x[3, 200], x[4, 0] = math.nan, math.inf, -math.inf
    x[5] = 1e-44                                                  # denormal throughout
    out = Fp4Rows(6, 256, DEV)
    fp4_rows(x, out)
    good = [0, 1, 5]
    same(out.data[good], 256, quantised(x[good]))
    w, wv = weight(130, 256)
    y = torch.empty(6, 130, device=DEV)
    fp4_gemm(out, w, fp4_tiles(6, DEV), out_f32=y)
    assert y[2:5].isnan().all() and y[good].isfinite().all() and (y[1] == 0).all()


@gpu
def test_norm_strides_and_scatter():
    from bloomery_b200.ops.fp4 import Fp4Rows, fp4_rows
    M, K = 19, 2048
    wide = make(M, K + 64, torch.float32, seed=2)
    x = wide[:, 32:32 + K]
    gain = (1 + 0.3 * torch.randn(K, generator=torch.Generator().manual_seed(1))).to(DEV)
    out = Fp4Rows(M, K, DEV)
    fp4_rows(x, out, gain=gain, eps=1e-6)
    r = (1 / (x.double().square().mean(1, keepdim=True) + 1e-6).sqrt()).float()
    want = quantised(x * r * gain)
    same(out.data, K, want)
    places = torch.randperm(64, generator=torch.Generator().manual_seed(5))[:M * 3].to(torch.int32)
    places[4], places[30] = -1, 64                                # nowhere
    out = Fp4Rows(64, K, DEV)
    out.data.fill_(0x55)
    fp4_rows(x, out, gain=gain, eps=1e-6, pos_of=places.to(DEV))
    hit = [i for i in range(M * 3) if 0 <= places[i] < 64]
    same(out.data[places[hit].long().to(DEV)], K, tuple(t[[i // 3 for i in hit]] for t in want))
    free = sorted(set(range(64)) - {int(places[i]) for i in hit})
    assert bool((out.data[free] == 0x55).all())


@gpu
@pytest.mark.parametrize("M,N,K", [(1, 1, 64), (5, 130, 192), (16, 2048, 4096), (32, 256, 256), (37, 1000, 512), (64, 384, 768), (65, 129, 320),
                                   (128, 512, 2048), (129, 640, 1024), (300, 257, 576), (700, 512, 4096 + 128)])
@pytest.mark.parametrize("f32", [True, False])
def test_dense_products(M, N, K, f32):
    from bloomery_b200.ops.fp4 import Fp4Rows, Fp4Work, fp4_gemm, fp4_rows, fp4_tiles
    x = make(M, K, seed=N)
    rows = Fp4Rows(M, K, DEV)
    fp4_rows(x, rows)
    w, wv = weight(N, K, seed=M)
    xv = quantised(x)[3]
    want, tol = xv @ wv.T, allowed(xv, wv, K)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    if f32:
        resid = torch.randn(M, N, device=DEV)
        y = torch.full((M + 1, N + 3), 7.0, device=DEV)
        fp4_gemm(rows, w, fp4_tiles(M, DEV), out_f32=y[:M, :N], resid=resid, status=status, work=Fp4Work(DEV))
        assert (y[M] == 7).all() and (y[:, N:] == 7).all()
        want = want + resid.double().cpu()
        got = y[:M, :N]
        tol = tol + 2.0 ** -23 * want.abs()
    else:
        got = torch.empty(M, N, dtype=torch.bfloat16, device=DEV)
        fp4_gemm(rows, w, fp4_tiles(M, DEV), out_bf16=got, status=status)
        tol = tol + 2.0 ** -8 * want.abs()
    assert int(status) == 0
    off = (got.double().cpu() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


def plan(T, E, k, tile_rows, seed, elsewhere=0):
    from bloomery_b200.ops import gemm as G
    gen = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(E, generator=gen)[:k] for _ in range(T)]).to(torch.int32)
    for i in torch.randperm(T * k, generator=gen)[:elsewhere].tolist():
        ids.view(-1)[i] = -1
    wts = torch.rand(T, k, generator=gen)
    n = T * k
    i32 = dict(dtype=torch.int32, device=DEV)
    tiles = G.TileTable(n, E, DEV, tile_rows)
    pos_of, dst_row, row_scale = torch.zeros(n, **i32), torch.zeros(n + 128, **i32), torch.zeros(n + 128, device=DEV)
    G.moe_plan(ids.to(DEV), wts.to(DEV), E, tiles, pos_of, dst_row, row_scale)
    return ids, wts, tiles, pos_of, dst_row, row_scale


@gpu
@pytest.mark.parametrize("T,E,k,inter,H,tile_rows", [(1, 16, 4, 256, 512, 32), (24, 16, 4, 256, 512, 32), (100, 16, 4, 256, 512, 64),
                                                     (333, 16, 4, 192, 320, 128), (40, 5, 2, 130, 192, 128), (600, 7, 3, 256, 512, 256)])
def test_gated_and_scattered_products_of_experts(T, E, k, inter, H, tile_rows):
    from bloomery_b200.ops.fp4 import Fp4Rows, fp4_gemm, fp4_rows
    ids, wts, tiles, pos_of, dst_row, row_scale = plan(T, E, k, tile_rows, T, elsewhere=T // 3)
    x = make(T, H, seed=9)
    rows = Fp4Rows(T * k, H, DEV)
    fp4_rows(x, rows, pos_of=pos_of)
    (wg, gv), (wu, uv) = weight(inter, H, 1, E), weight(inter, H, 2, E)
    act = torch.full((T * k, inter), 3.0, dtype=torch.bfloat16, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    if tile_rows <= 128:
        fp4_gemm(rows, wg, tiles, W2=wu, out_bf16=act, dst_row=dst_row, status=status)
        xv = quantised(x)[3]
        flat = ids.view(-1)
        for i in range(T * k):
            e = int(flat[i])
            if e < 0:
                assert (act[i] == 3).all()
                continue
            v = xv[i // k:i // k + 1]
            g, u = v @ gv[e].T, v @ uv[e].T
            want = g * torch.sigmoid(g) * u
            # the factor's slope is at most 1.1; the exponential and the quotient are off by a few units of 2^-22
            tg, tu = allowed(v, gv[e], H), allowed(v, uv[e], H)
            tol = 1.1 * tg * (u.abs() + tu) + (g.abs() + tg) * tu + (2.0 ** -8 + 2.0 ** -19) * want.abs() + 1e-30
            off = (act[i].double().cpu() - want[0]).abs()
            assert bool((off <= tol[0]).all()), (i, float((off / tol[0]).max()))
    down, dv = weight(H, H, 3, E)
    out = torch.full((T * k, H), 3.0, device=DEV)
    fp4_gemm(rows, down, tiles, out_f32=out, dst_row=dst_row, row_scale=row_scale, status=status)
    xv = quantised(x)[3]
    for i in range(T * k):
        e = int(ids.view(-1)[i])
        if e < 0:
            assert (out[i] == 3).all()
            continue
        f = float(wts.view(-1)[i])
        v = xv[i // k:i // k + 1]
        off = (out[i].double().cpu() - f * (v @ dv[e].T)[0]).abs()
        assert bool((off <= f * allowed(v, dv[e], H)[0] + 1e-30).all())
    assert int(status) == 0


@gpu
def test_rows_times_rows_made_right_before():
    """Both sides of a product out of the launches in front of it, again and again: it reads none of them before they are written."""
    from bloomery_b200.ops.fp4 import Fp4Rows, fp4_gemm, fp4_rows, fp4_tiles
    M, N, K = 20, 300, 2048
    tiles, a, b = fp4_tiles(M, DEV), Fp4Rows(M, K, DEV), Fp4Rows(N, K, DEV)
    xs = [make(M, K, seed=s) for s in range(3)]
    ys = [make(N, K, seed=10 + s) for s in range(3)]
    outs = [torch.empty(M, N, device=DEV) for _ in range(12)]
    for i, out in enumerate(outs):
        fp4_rows(xs[i % 3], a)
        fp4_rows(ys[(i * 2) % 3], b)
        fp4_gemm(a, b.weight, tiles, out_f32=out)
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        xv, yv = quantised(xs[i % 3])[3], quantised(ys[(i * 2) % 3])[3]
        off = (out.double().cpu() - xv @ yv.T).abs()
        assert bool((off <= allowed(xv, yv, K)).all()), i


@gpu
def test_no_rows_and_no_tiles():
    from bloomery_b200.ops.fp4 import Fp4Rows, fp4_gemm, fp4_rows
    rows = Fp4Rows(8, 128, DEV)
    rows.data.fill_(0x55)
    fp4_rows(torch.zeros(0, 128, device=DEV), rows)
    fp4_rows(torch.zeros(0, 128, device=DEV), rows, pos_of=torch.zeros(0, dtype=torch.int32, device=DEV))
    assert bool((rows.data == 0x55).all())
    ids, wts, tiles, pos_of, dst_row, row_scale = plan(4, 5, 2, 32, 1, elsewhere=8)          # every slot is another tier's
    fp4_rows(make(4, 128), rows, pos_of=pos_of)
    assert bool((rows.data == 0x55).all())
    w, _ = weight(64, 128, 1, 5)
    out = torch.full((8, 64), 3.0, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    fp4_gemm(rows, w, tiles, out_f32=out, dst_row=dst_row, status=status)
    assert (out == 3).all() and int(status) == 0


@gpu
def test_products_in_place_on_streams_and_in_graphs():
    """The residual stream as addend and output; a captured pair replayed with other rows; two streams at once."""
    from bloomery_b200.ops.fp4 import Fp4Rows, fp4_gemm, fp4_rows, fp4_tiles
    M, N, K = 48, 512, 1024
    w, wv = weight(N, K, seed=4)
    x, tiles = make(M, K, seed=6), fp4_tiles(M, DEV)
    rows, y = Fp4Rows(M, K, DEV), torch.randn(M, N, device=DEV)
    y0 = y.clone()
    fp4_rows(x, rows)
    fp4_gemm(rows, w, tiles, out_f32=y, resid=y)
    xv = quantised(x)[3]
    off = (y.double().cpu() - (xv @ wv.T + y0.double().cpu())).abs()
    assert bool((off <= allowed(xv, wv, K) + 2.0 ** -23 * y.double().cpu().abs()).all())
    out = torch.empty(M, N, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fp4_rows(x, rows)
        fp4_gemm(rows, w, tiles, out_f32=out)
    other = make(M, K, seed=7)
    x.copy_(other)
    graph.replay()
    ref, rows2 = torch.empty(M, N, device=DEV), Fp4Rows(M, K, DEV)
    fp4_rows(other, rows2)
    fp4_gemm(rows2, w, tiles, out_f32=ref)
    torch.cuda.synchronize()
    assert torch.equal(out, ref)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs, bufs = [torch.empty(M, N, device=DEV) for _ in streams], [Fp4Rows(M, K, DEV) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, o, b in zip(streams, outs, bufs):
            with torch.cuda.stream(s):
                fp4_rows(other, b)
                fp4_gemm(b, w, tiles, out_f32=o)
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs)


@gpu
@pytest.mark.parametrize("rows,K", [(1, 64), (37, 320), (9, 4096)])
def test_expansion_of_every_code_and_scale(rows, K):
    """Exact: fp32(E4M3 * g / 2) times the doubled code, rounded once; negative, zero, infinite and NaN scales among them.  The halving takes
    no rounding of its own (E4M3 * g / 2 has 28 bits, exact in 64): twice as much may pass fp32's largest value where the half does not."""
    from bloomery_b200.ops.gemm import dequant_bf16

    gen = torch.Generator().manual_seed(K)
    codes = torch.randint(0, 16, (rows, K), generator=gen)
    sc = torch.randint(0, 256, (rows, K // 16), generator=gen, dtype=torch.uint8)
    g = torch.randn(rows, generator=gen) * 1e-3
    odd = torch.tensor([0.0, -0.0, 1e-40, 3e38, math.inf, -math.inf, math.nan, -1.0])
    g[:min(rows - 1, 8)] = odd[:min(rows - 1, 8)]
    data = torch.zeros(rows, (K // 2 + K // 16 + 4 + 15) // 16 * 16, dtype=torch.uint8)
    data[:, :K // 2] = (codes[:, ::2] | codes[:, 1::2] << 4).to(torch.uint8)
    data[:, K // 2:K // 2 + K // 16] = sc
    data[:, K // 2 + K // 16:K // 2 + K // 16 + 4] = g.view(rows, 1).view(torch.uint8)
    out = torch.empty(rows, K, dtype=torch.bfloat16, device=DEV)
    dequant_bf16(QWeight(data.to(DEV), "NVFP4", K), out)
    doubled = torch.tensor([int(2 * v) for v in E2M1] + [-int(2 * v) for v in E2M1]).float()
    step = (planes.e4m3_decode(sc).double() * g[:, None].double() * 0.5).float()
    want = (step.repeat_interleave(16, 1) * doubled[codes]).to(torch.bfloat16)
    nan = want.isnan()
    assert torch.equal(out.cpu().isnan(), nan)
    assert torch.equal(out.cpu()[~nan].view(torch.int16), want[~nan].view(torch.int16))


@gpu
@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("M,N,K", [(5, 24, 128), (40, 130, 320), (300, 136, 64)])
def test_rows_sent_past_the_output_go_nowhere(M, N, K, f32):
    """A third of the rows below 0, a third past the end; the rest as without the sending, bit for bit."""
    from bloomery_b200.ops.fp4 import Fp4Rows, fp4_gemm, fp4_rows, fp4_tiles
    rows, (w, _) = Fp4Rows(M, K, DEV), weight(N, K, 4)
    fp4_rows(make(M, K, seed=3), rows)
    dtype = torch.float32 if f32 else torch.bfloat16
    kw = lambda t: dict(out_f32=t) if f32 else dict(out_bf16=t)
    plain, whole = torch.empty(M, N, dtype=dtype, device=DEV), torch.full((2 * M, N), 3.0, dtype=dtype, device=DEV)
    fp4_gemm(rows, w, fp4_tiles(M, DEV), **kw(plain))
    dst = torch.arange(M, dtype=torch.int32)
    dst[1::3], dst[2::3] = -1 - dst[1::3], M + dst[2::3] % 7
    dst[2] = 2 ** 31 - 1
    resid = torch.zeros(M, N, device=DEV)
    fp4_gemm(rows, w, fp4_tiles(M, DEV), **kw(whole[:M]), dst_row=dst.to(DEV))
    assert torch.equal(whole[0:M:3], plain[::3])
    whole[0:M:3] = 3.0
    assert (whole == 3).all()
    fp4_gemm(rows, w, fp4_tiles(M, DEV), **kw(whole[:M]), dst_row=dst.to(DEV), resid=resid)
    assert torch.equal(whole[0:M:3], plain[::3])
    whole[0:M:3] = 3.0
    assert (whole == 3).all()
