"""MXFP4 Block-ELL on the B200 against the float64 definition.

Tolerances, derived: Q is exact (every code and scale is compared).  A product
of two quantised values is exact in fp32, so a linear's error is that of its
sum: at most 64 additions inside an MMA and one per MMA after it, each losing
at most one unit of 2^-23 of the running sum of magnitudes, plus one rounding
of the output (half a step: bf16 2^-8, fp32 2^-24 of the value).
"""

import numpy as np
import pytest
import torch

from gpu_util import rand_cols
from oracle import mxfp4_oracle as M

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def _K():
    from looped_blockell import kernels
    return kernels


def f64(t):
    return t.detach().double().cpu().numpy()


def rows(rng, T, n, dtype=BF16, spread=2.0):
    """Rows whose magnitudes spread over several octaves."""
    x = rng.standard_normal((T, n)) * np.exp2(rng.uniform(-spread, spread, (T, n)))
    return torch.from_numpy(x.astype(np.float32)).to(dtype).cuda()


def weight(rng, R, C, K, B, dead=0, dtype=BF16, layout=0, dup=False, dead_row=None):
    cols = rand_cols(rng, R, C, K, dead, dup)
    if dead_row is not None:
        cols[dead_row] = -1
    v = torch.from_numpy((rng.standard_normal((R, K, B, B)) * 0.02).astype(np.float32)).to(dtype).cuda()
    ct = torch.from_numpy(cols).cuda()
    return v, ct, M.dense(M.quantize_tiles(f64(v), layout), cols, C, layout)


def sum_bound(xq, w, n_mma):
    return (64 + n_mma) * 2.0 ** -23 * (np.abs(xq) @ np.abs(w).T)


def check_linear(y, xq, w, n_mma, res=None):
    ref = xq @ w.T
    bound = sum_bound(xq, w, n_mma)
    if res is not None:
        bound = bound + 2.0 ** -23 * (np.abs(ref) + np.abs(res))
        ref = ref + res
    err = np.abs(f64(y) - ref)
    assert (err <= bound + HALF_STEP[y.dtype] * (np.abs(ref) + bound)).all(), float((err - bound).max())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,n,tile", [(1, 128, 128), (1, 64, 64), (7, 192, 64), (128, 256, 128), (130, 320, 64),
                                      (333, 1152, 128)])
def test_quantize_rows_equals_the_definition(T, n, tile, dtype):
    K = _K()
    x = rows(np.random.default_rng(T + n), T, n, dtype)
    q = K.mxfp4_quantize(x, tile=tile)
    ref = M.quantize(f64(x))
    for out_dtype in (BF16, F32):  # Q(x) is exact in either
        np.testing.assert_array_equal(f64(K.mxfp4_dequantize(q, out_dtype)), ref)


def test_quantize_every_rounding_case_and_extreme_scales():
    K = _K()
    # every tie, both neighbours of each, both signs, at scales over the whole fp32 range
    edges = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9375])
    vals = np.concatenate([edges, np.nextafter(edges.astype(np.float32), np.float32(0)),
                           np.nextafter(edges.astype(np.float32), np.float32(8)), -edges]).astype(np.float32)
    lead = np.float32(4.0)  # the block's largest magnitude is in [4, 8): s = 1
    blocks = [np.concatenate([[lead], vals[i:i + 31], np.zeros(31 - len(vals[i:i + 31]))]) for i in range(0, len(vals), 31)]
    base = np.stack(blocks).astype(np.float32)
    out = []
    for e in (-145, -130, -128, -126, -100, -1, 0, 1, 90, 124):
        with np.errstate(over="ignore"):
            out.append(np.ldexp(base, e).astype(np.float32))
    out.append(np.zeros((2, 32), np.float32))
    x = np.concatenate([o for o in out if np.isfinite(o).all()])
    x = np.concatenate([x, np.zeros((-len(x) % 2, 32), np.float32)]).reshape(-1, 64)
    q = K.mxfp4_quantize(torch.from_numpy(x).cuda(), tile=64)
    np.testing.assert_array_equal(f64(q.dequantize(F32)), M.quantize(x))


def test_quantize_non_finite_blocks_only():
    K = _K()
    x = np.random.default_rng(0).standard_normal((3, 128)).astype(np.float32)
    x[0, 5], x[1, 40], x[2, 127] = np.nan, np.inf, -np.inf
    got = f64(K.mxfp4_quantize(torch.from_numpy(x).cuda()).dequantize(F32))
    bad = np.zeros((3, 4), bool)
    bad[0, 0] = bad[1, 1] = bad[2, 3] = True
    np.testing.assert_array_equal(np.isnan(got).reshape(3, 4, 32), np.repeat(bad[..., None], 32, -1))
    ok = ~np.isnan(got)
    np.testing.assert_array_equal(got[ok], M.quantize(x)[ok])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quantize_strided_and_misaligned_rows(dtype):
    K = _K()
    wide = rows(np.random.default_rng(3), 40, 512, dtype)
    for x in (wide[:, 128:384], wide[::3, :256], wide[:, 1:257], wide.t()[:128, :].t()[:, :128], wide[5:6, 64:192]):
        np.testing.assert_array_equal(f64(K.mxfp4_quantize(x).dequantize(F32)), M.quantize(f64(x)))


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B", [64, 128])
def test_make_mxfp4_tiles(B, dtype, layout):
    K = _K()
    rng = np.random.default_rng(B + layout)
    v, cols, _ = weight(rng, 3, 4, 2, B, dead=1, dtype=dtype)
    w = K.make_mxfp4(v, cols, 4, layout)
    for back in (0, 1):
        ref = M.quantize_tiles(f64(v), layout)
        np.testing.assert_array_equal(f64(w.dequantize(back)), ref if back == layout else np.swapaxes(ref, -1, -2))


@pytest.mark.parametrize("T,R,C,Kk,B,dead", [
    (1, 1, 1, 1, 128, 0), (1, 1, 1, 1, 64, 0), (5, 3, 4, 2, 64, 1), (128, 2, 3, 3, 128, 0), (129, 2, 40, 35, 64, 3),
    (257, 5, 36, 33, 128, 7), (300, 160, 2, 2, 64, 11), (1000, 40, 9, 4, 128, 5),
    (1, 32, 128, 32, 128, 0), (2, 70, 20, 17, 64, 9), (130, 9, 32, 32, 128, 20), (33, 1, 64, 61, 64, 3),
    (8, 3, 5, 5, 128, 2), (9, 6, 9, 9, 64, 4), (25, 2, 17, 13, 128, 0), (32, 4, 3, 2, 64, 0), (17, 170, 40, 39, 64, 9)])
@pytest.mark.parametrize("dtype,residual", [(BF16, False), (BF16, True), (F32, True)])
def test_linear(T, R, C, Kk, B, dead, dtype, residual):
    K = _K()
    rng = np.random.default_rng(T + R)
    v, cols, w = weight(rng, R, C, Kk, B, dead, dead_row=R - 1 if dead else None)
    x = rows(rng, T, C * B, dtype)
    res = rows(rng, T, R * B, dtype) if residual else None
    mw = K.make_mxfp4(v, cols, C)
    y = K.mxfp4_linear(x, mw, residual=res)
    assert y.dtype == dtype and y.shape == (T, R * B)
    check_linear(y, M.quantize(f64(x)), w, Kk * B // 64, None if res is None else f64(res))
    y2 = K.mxfp4_linear(K.mxfp4_quantize(x, tile=B), mw, residual=res, out_dtype=dtype)
    assert torch.equal(y, y2)  # quantised before or on the way: the same bits
    assert K.read_status() == 0


def check_ffn(K, x, g, u, d, wg, wu, wd, residual):
    """Every stage against the definition at the GPU's own operands of that stage."""
    B = g.B
    out, ws = K.mxfp4_swiglu_fwd(x, g, u, d, add_residual=residual, return_intermediates=True)
    xq, hq = f64(ws["q_x"].dequantize(F32)), f64(ws["q_h"].dequantize(F32))
    np.testing.assert_array_equal(xq, M.quantize(f64(x)))
    n = g.K * B // 64
    bg, bu = sum_bound(xq, wg, n), sum_bound(xq, wu, u.K * B // 64)
    gd, ud = xq @ wg.T, xq @ wu.T
    for name, ref, bound in (("gate", gd, bg), ("up", ud, bu)):
        assert (np.abs(f64(ws[name]) - ref) <= bound + HALF_STEP[BF16] * (np.abs(ref) + bound)).all(), name
    # h's codes: those of some h within the fp32 error of g, u, e^-g and the divide (2^-18)
    h = M.silu_mul(gd, ud)
    sig = 1 / (1 + np.exp(-gd))
    tol = 1.1 * np.abs(ud) * bg + np.abs(gd * sig) * bu + 2.0 ** -18 * np.abs(h) + 1.1 * bg * bu
    T, F = h.shape
    lo, hi = h - tol, h + tol
    mag = np.abs(h).reshape(T, -1, 32)
    top_lo, top_hi = (np.maximum(mag + s * tol.reshape(T, -1, 32), 0).max(-1, keepdims=True) for s in (-1, 1))
    s_lo, s_hi = (M.scales(np.repeat(t, 32, -1)) for t in (top_lo, top_hi))
    q = hq.reshape(T, -1, 32)
    fits = np.zeros((T, F // 32), bool)
    for s in (s_lo, s_hi):  # the block's scale may be either, where its largest value is next to a power of two
        a, b = (M.e2m1(v.reshape(T, -1, 32) / s[..., :1]) * s[..., :1] for v in (lo, hi))
        fits |= ((q >= a) & (q <= b)).all(-1)
    assert fits.all(), int((~fits).sum())
    check_linear(out, hq, wd, d.K * B // 64, f64(x) if residual else None)
    assert K.read_status() == 0
    return out


@pytest.mark.parametrize("T,d,F,B,Kg,Kd,dead", [
    (1, 128, 256, 64, 1, 1, 0), (1, 256, 512, 128, 2, 4, 0), (3, 192, 320, 64, 2, 3, 2), (8, 1280, 1536, 128, 9, 11, 3),
    (17, 640, 896, 64, 9, 13, 5), (32, 512, 20480, 128, 3, 2, 0), (33, 384, 512, 128, 3, 3, 1), (2, 1280, 20480, 64, 18, 40, 30), (128, 256, 512, 64, 4, 8, 3),
    (131, 384, 640, 128, 2, 5, 2), (700, 512, 2560, 64, 3, 20, 9), (515, 640, 3200, 128, 3, 12, 4)])
@pytest.mark.parametrize("residual", [False, True])
def test_swiglu_stages(T, d, F, B, Kg, Kd, dead, residual):
    K = _K()
    rng = np.random.default_rng(T + d)
    vg, cg, wg = weight(rng, F // B, d // B, Kg, B, dead, dead_row=0 if dead else None)
    vu, cu, wu = weight(rng, F // B, d // B, Kg, B, dead)
    vd, cd, wd = weight(rng, d // B, F // B, Kd, B, dead, dead_row=0 if dead > 2 else None)
    x = rows(rng, T, d, spread=1.0)
    out = check_ffn(K, x, K.make_mxfp4(vg, cg, d // B), K.make_mxfp4(vu, cu, d // B), K.make_mxfp4(vd, cd, F // B), wg,
                    wu, wd, residual)
    out2 = K.mxfp4_swiglu_fwd(x, K.make_mxfp4(vg, cg, d // B), K.make_mxfp4(vu, cu, d // B),
                              K.make_mxfp4(vd, cd, F // B), add_residual=residual)
    assert torch.equal(out, out2)


def rel(a, b):
    return np.linalg.norm(a - b) / np.linalg.norm(b)


# Counted for the backward: bf16 roundings (2^-8 of a value each) of d_g or d_u and of the result; what is left (fp32
# products and sums, the exponential's 2^-18) stays below a tenth of one: at most 2.1 x 2^-8 of the norm.
GRAD_TOL = 2.1 * 2.0 ** -8


@pytest.mark.parametrize("T,R,C,Kk,B,dead,layout,dtype", [
    (1, 2, 3, 2, 64, 0, 0, BF16), (130, 4, 6, 3, 64, 2, 1, BF16), (257, 3, 4, 2, 128, 1, 0, F32), (64, 3, 4, 3, 128, 0, 1, BF16)])
def test_linear_gradients(T, R, C, Kk, B, dead, layout, dtype):
    K = _K()
    rng = np.random.default_rng(T)
    v, cols, w = weight(rng, R, C, Kk, B, dead, dtype=dtype, layout=layout)
    x, dy = rows(rng, T, C * B), rows(rng, T, R * B)
    res = rows(rng, T, R * B)
    for t in (x, v, res):
        t.requires_grad_(True)
    y = K.mxfp4_linear_ad(x, v, cols, residual=res, layout=layout)
    y.backward(dy)
    xq = M.quantize(f64(x))
    check_linear(y, xq, w, Kk * B // 64, f64(res))
    assert x.grad.dtype == BF16 and v.grad.dtype == dtype
    assert rel(f64(x.grad), f64(dy) @ w) <= GRAD_TOL
    assert rel(f64(v.grad), M.tile_grads(f64(dy).T @ xq, f64(cols).astype(int), B, layout)) <= GRAD_TOL
    assert torch.equal(res.grad, dy)
    if dead:
        assert (v.grad[cols < 0] == 0).all()


@pytest.mark.parametrize("T,d,F,B,Kg,Kd,dead,layout,dtype", [
    (1, 128, 256, 64, 1, 2, 0, 0, BF16), (200, 256, 512, 64, 2, 4, 3, 0, BF16), (257, 256, 512, 128, 2, 3, 1, 1, BF16),
    (130, 384, 640, 128, 2, 4, 0, 0, F32)])
def test_swiglu_gradients(T, d, F, B, Kg, Kd, dead, layout, dtype):
    K = _K()
    rng = np.random.default_rng(T + 1)
    mats = [weight(rng, F // B, d // B, Kg, B, dead, dtype, layout), weight(rng, F // B, d // B, Kg, B, dead, dtype, layout),
            weight(rng, d // B, F // B, Kd, B, dead, dtype, layout)]
    x, dy = rows(rng, T, d, spread=1.0), rows(rng, T, d)
    leaves = [x] + [m[0] for m in mats]
    for t in leaves:
        t.requires_grad_(True)
    args = [a for v, c, _ in mats for a in (v, c)]
    y = K.mxfp4_swiglu(x, *args, add_residual=True, layout=layout)
    y.backward(dy)
    packed = [K.make_mxfp4(v.detach(), c, n, layout) for (v, c, _), n in zip(mats, (d // B, d // B, F // B))]
    out, ws = K.mxfp4_swiglu_fwd(x.detach(), *packed, add_residual=True, return_intermediates=True)
    assert torch.equal(out, y)
    refs = M.swiglu_backward(M.quantize(f64(x)), *(m[2] for m in mats), f64(ws["q_h"].dequantize(F32)), f64(dy), True)
    assert rel(f64(x.grad), refs[0]) <= GRAD_TOL
    for (v, c, _), ref in zip(mats, refs[1:]):
        assert v.grad.dtype == dtype
        assert rel(f64(v.grad), M.tile_grads(ref, f64(c).astype(int), B, layout)) <= GRAD_TOL
    assert K.read_status() == 0


# ------------------------------------------------------------ ways of calling


def _ffn(rng, d=256, F=512, B=64, Kg=2, Kd=4, dead=0):
    mats = [weight(rng, F // B, d // B, Kg, B, dead), weight(rng, F // B, d // B, Kg, B, dead),
            weight(rng, d // B, F // B, Kd, B, dead)]
    K = _K()
    return mats, [K.make_mxfp4(v, c, n) for (v, c, _), n in zip(mats, (d // B, d // B, F // B))]


@pytest.mark.parametrize("T", [3, 200])
@pytest.mark.parametrize("B", [64, 128])
def test_a_token_gets_the_same_result_in_any_batch(T, B):
    """Sums run over the slots in one order whatever the batch (up to the number of CTAs sharing a row)."""
    K = _K()
    rng = np.random.default_rng(T)
    _, packed = _ffn(rng, 512, 40960, B, 2, 3)  # more units than half of the SMs: whole units
    x = rows(rng, T, 512)
    whole = K.mxfp4_swiglu_fwd(x, *packed)
    again = K.mxfp4_swiglu_fwd(x, *packed)
    assert torch.equal(whole, again)
    part = K.mxfp4_swiglu_fwd(x[1:2], *packed)
    q_whole, q_part = (K.mxfp4_swiglu_fwd(t, *packed, return_intermediates=True)[1]["q_h"].dequantize() for t in (x, x[1:2]))
    assert torch.equal(q_whole[1:2], q_part)
    np.testing.assert_allclose(f64(part), f64(whole[1:2]), rtol=2.0 ** -7, atol=1e-5)


def test_graph_replay_two_graphs_and_other_streams():
    """Captured calls own their workspaces: two graphs and an eager call run at once, each with its own result."""
    K = _K()
    rng = np.random.default_rng(7)
    _, packed = _ffn(rng)
    xs = [rows(rng, T, 256) for T in (1, 70)]
    want = [K.mxfp4_swiglu_fwd(x, *packed, add_residual=True) for x in xs]
    graphs, outs, bufs = [], [], [torch.zeros_like(x) for x in xs]
    for b in bufs:
        K.mxfp4_swiglu_fwd(b, *packed, add_residual=True)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(K.mxfp4_swiglu_fwd(b, *packed, add_residual=True))
        graphs.append(g)
    for b, x in zip(bufs, xs):
        b.copy_(x)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
        eager = K.mxfp4_swiglu_fwd(xs[1], *packed, add_residual=True)
    torch.cuda.synchronize()
    for got, ref in zip(outs + [eager], want + [want[1]]):
        assert torch.equal(got, ref)
    assert K.read_status() == 0


def test_side_stream_inputs_and_producers_ahead():
    """The call runs on the current stream, after what made its inputs there (x, weights and residual included)."""
    K = _K()
    rng = np.random.default_rng(8)
    v, cols, _ = weight(rng, 4, 4, 3, 64)
    x, res = rows(rng, 50, 256), rows(rng, 50, 256)
    want = K.mxfp4_linear(x, K.make_mxfp4(v, cols, 4), residual=res)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for T in (50, 5):
            busy = torch.randn(2000, 2000, device="cuda")
            for _ in range(20):
                busy = busy @ busy * 1e-3
            late = [t.clone() + 0 * busy[0, 0].to(t.dtype).nan_to_num() for t in (x, res)]
            w = K.make_mxfp4(v.clone(), cols.clone(), 4)
            y = K.mxfp4_linear(late[0][:T], w, residual=late[1][:T])
            q = K.mxfp4_linear(K.mxfp4_quantize(late[0][:T], 64), w, residual=late[1][:T])
            s.synchronize()
            if T == 50:
                assert torch.equal(y, want) and torch.equal(q, want)
            else:
                assert torch.equal(y, q)


@pytest.mark.parametrize("T", [2, 33, 400])
def test_nan_and_infinite_rows_stay_in_their_rows(T):
    K = _K()
    rng = np.random.default_rng(9)
    _, packed = _ffn(rng, 256, 1024, 64, 3, 6)
    x = rows(rng, T, 256)
    clean = K.mxfp4_swiglu_fwd(x, *packed)
    x[1, :] = float("nan")
    x[T - 1, 200] = float("inf")
    got = K.mxfp4_swiglu_fwd(x, *packed)
    assert got[1].isnan().all()
    keep = [t for t in range(T) if t not in (1, T - 1)]
    assert torch.equal(got[keep], clean[keep])


def test_rows_behind_the_last_token_are_left_alone():
    K = _K()
    rng = np.random.default_rng(10)
    _, packed = _ffn(rng)
    for T in (1, 37, 130):
        out = torch.full((T + 3, 256), 7.0, dtype=BF16, device="cuda")
        x = rows(rng, T, 256)
        h = rows(rng, T, 512)
        K.mxfp4_linear(h, packed[2], out=out[:T])
        assert (out[T:] == 7).all()
        dq = torch.full((T + 2, 256), 3.0, dtype=F32, device="cuda")
        K.mxfp4_dequantize(K.mxfp4_quantize(x, 64), F32, out=dq[:T])
        assert (dq[T:] == 3).all()


def test_no_tokens_dead_weights_and_bad_columns():
    K = _K()
    rng = np.random.default_rng(11)
    mats, packed = _ffn(rng)
    empty = torch.empty(0, 256, dtype=BF16, device="cuda")
    assert K.mxfp4_swiglu_fwd(empty, *packed, add_residual=True).shape == (0, 256)
    assert K.mxfp4_dequantize(K.mxfp4_quantize(empty, 64)).shape == (0, 256)
    leaves = [m[0].clone().requires_grad_(True) for m in mats]
    xe = empty.clone().requires_grad_(True)
    y = K.mxfp4_swiglu(xe, leaves[0], mats[0][1], leaves[1], mats[1][1], leaves[2], mats[2][1])
    y.sum().backward()
    assert xe.grad.shape == (0, 256) and all((t.grad == 0).all() for t in leaves)
    # every slot dead: zeros, or the residual alone
    dead = torch.full_like(mats[0][1], -1)
    x = rows(rng, 40, 256)
    w = K.make_mxfp4(mats[0][0], dead, 4)
    assert (K.mxfp4_linear(x, w) == 0).all()
    res = rows(rng, 40, 512)
    assert torch.equal(K.mxfp4_linear(x, w, residual=res), res)
    assert torch.equal(K.mxfp4_swiglu_fwd(x, w, w, packed[2], add_residual=True), x)
    assert K.read_status() == 0
    # an index outside the columns is dropped and reported
    bad = mats[0][1].clone()
    bad[1, 0] = 99
    gone = mats[0][1].clone()
    gone[1, 0] = -1
    y1, y2 = (K.mxfp4_linear(x, K.make_mxfp4(mats[0][0], c, 4)) for c in (bad, gone))
    assert torch.equal(y1, y2)
    assert K.read_status() == 1


def test_refusals_on_the_device():
    K = _K()
    rng = np.random.default_rng(12)
    mats, packed = _ffn(rng)
    x = rows(rng, 5, 256)
    for call, text in [
            (lambda: K.mxfp4_linear(x[:, :128], packed[0]), "features"),
            (lambda: K.mxfp4_linear(x.half(), packed[0]), "bf16 or fp32"),
            (lambda: K.mxfp4_linear(x[0], packed[0]), "2D"),
            (lambda: K.mxfp4_linear(x, packed[0], residual=x), "residual"),
            (lambda: K.mxfp4_linear(x, packed[0], out=torch.empty(5, 512, device="cuda")), "out must be"),
            (lambda: K.mxfp4_linear(K.mxfp4_quantize(x, 128), packed[0]), "tile"),
            (lambda: K.mxfp4_swiglu_fwd(x, packed[0], packed[1], packed[0]), "down"),
            (lambda: K.mxfp4_swiglu_fwd(K.mxfp4_quantize(x, 64), *packed, add_residual=True), "needs the residual"),
            (lambda: K.mxfp4_quantize(x, 96), "tile size"),
            (lambda: K.mxfp4_quantize(x[:, :192], 128), "multiple"),
            (lambda: K.make_mxfp4(mats[0][0][:, :, :32, :32].contiguous(), mats[0][1], 4), "tile size"),
            (lambda: K.make_mxfp4(mats[0][0], mats[0][1].long(), 4), "int32"),
            (lambda: K.make_mxfp4(mats[0][0], mats[0][1][:1], 4), "do not fit")]:
        with pytest.raises(RuntimeError, match=text):
            call()


@pytest.mark.parametrize("swiglu", [True, False])
def test_mlp_block_trains_and_serves_in_mxfp4(swiglu):
    """The layers: a training step, the packed weight followed through the update, pruned tiles, serving."""
    from looped_blockell.layers import MLPBlock
    torch.manual_seed(0)
    m = MLPBlock(256, 512, use_swiglu=swiglu, tile_size=64, density=0.5, device="cuda", weight_format="mxfp4")
    lin = m.w_gate if swiglu else m.fc1
    lin.alive_mask[0, 0] = False
    x = torch.randn(2, 65, 256, device="cuda", dtype=BF16, requires_grad=True)
    y = m(x, residual=True)
    y.backward(torch.randn_like(y))
    assert x.grad.isfinite().all() and (lin.values.grad[0, 0] == 0).all() and lin.values.grad[0, 1].abs().sum() > 0
    with torch.no_grad():
        before = m(x, residual=True)
        assert torch.equal(before, y)  # the packed weight gives what the step computed
        torch.optim.SGD(m.parameters(), lr=1.0).step()
        after = m(x, residual=True)
    assert torch.equal(after, m(x, residual=True).detach()) and not torch.equal(before, after)
    with pytest.raises(ValueError, match="tile_size"):
        MLPBlock(256, 512, tile_size=16, weight_format="mxfp4")
    with pytest.raises(ValueError, match="weight_format"):
        MLPBlock(256, 512, tile_size=64, weight_format="int3")


def test_training_captured_in_a_graph():
    """Forward and backward of one step captured, replayed on new data; no eager graph of the leaves is alive."""
    K = _K()
    rng = np.random.default_rng(13)
    mats, _ = _ffn(rng)
    x0, dy = rows(rng, 60, 256), rows(rng, 60, 256)
    leaves = [x0.clone()] + [m[0].clone() for m in mats]

    def step():
        ls = [t.detach().requires_grad_(True) for t in leaves]
        y = K.mxfp4_swiglu(ls[0], ls[1], mats[0][1], ls[2], mats[1][1], ls[3], mats[2][1], add_residual=True)
        return (y.detach(), *torch.autograd.grad(y, ls, dy))

    want = step()  # also builds the transposed topologies
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    leaves[0].copy_(rows(rng, 60, 256))
    g.replay()
    leaves[0].copy_(x0)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for a, b in zip(got[2:], want[2:]):  # tile sums meet in arrival order: fp32 sums of 60 terms, then bf16
        np.testing.assert_allclose(f64(a), f64(b), rtol=2.0 ** -7, atol=1e-4)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_buffers_aligned_to_16_bytes_only(dtype):
    """Outputs and residuals that start half a sector in: the same values as aligned ones."""
    K = _K()
    rng = np.random.default_rng(14)
    _, packed = _ffn(rng)
    per16 = 16 // torch.empty(0, dtype=dtype).element_size()
    for T in (1, 200):
        x = rows(rng, T, 512, dtype)
        flat, rflat = (torch.full((T * 256 + 2 * per16,), 5.0, dtype=dtype, device="cuda") for _ in range(2))
        out, res = (f[per16:per16 + T * 256].view(T, 256) for f in (flat, rflat))
        assert out.data_ptr() % 32 == 16
        want = K.mxfp4_linear(x, packed[2], residual=res.clone())
        assert torch.equal(K.mxfp4_linear(x, packed[2], residual=res, out=out), want)
        assert (flat[:per16] == 5).all() and (flat[per16 + T * 256:] == 5).all()


def test_gradients_of_fp32_layers_and_of_some_inputs_only():
    """fp32 rows and tiles: dy is rounded to bf16 once more (2^-8).  Inputs that need no gradient get none, and the
    others' do not change."""
    K = _K()
    rng = np.random.default_rng(15)
    mats = [weight(rng, 8, 4, 2, 64, 1, F32), weight(rng, 8, 4, 3, 64, 0, F32), weight(rng, 4, 8, 5, 64, 0, F32)]
    x, dy = rows(rng, 70, 256, F32, 1.0), rows(rng, 70, 256, F32)
    everything = None
    for which in ([0, 1, 2, 3], [0], [2], [3], [1, 3]):
        leaves = [t.detach().clone().requires_grad_(i in which) for i, t in enumerate([x] + [m[0] for m in mats])]
        y = K.mxfp4_swiglu(leaves[0], leaves[1], mats[0][1], leaves[2], mats[1][1], leaves[3], mats[2][1])
        assert y.dtype == F32
        y.backward(dy)
        if everything is None:
            everything = [t.grad for t in leaves]
            _, ws = K.mxfp4_swiglu_fwd(x, *(K.make_mxfp4(m[0], m[1], n) for m, n in zip(mats, (4, 4, 8))),
                                       return_intermediates=True)
            refs = M.swiglu_backward(M.quantize(f64(x)), *(m[2] for m in mats), f64(ws["q_h"].dequantize(F32)), f64(dy),
                                     False)
            assert rel(f64(leaves[0].grad), refs[0]) <= GRAD_TOL + 2.0 ** -8
            for t, (_, c, _), ref in zip(leaves[1:], mats, refs[1:]):
                assert t.grad.dtype == F32
                assert rel(f64(t.grad), M.tile_grads(ref, f64(c).astype(int), 64)) <= GRAD_TOL + 2.0 ** -8
        for i, t in enumerate(leaves):
            assert (t.grad is None) == (i not in which)
            if i in which:  # tile sums meet in arrival order
                np.testing.assert_allclose(f64(t.grad), f64(everything[i]), rtol=1e-4, atol=1e-4)
    with pytest.raises(RuntimeError):  # no second derivative
        xg = x.detach().requires_grad_(True)
        y = K.mxfp4_linear_ad(xg, mats[0][0], mats[0][1])
        (g,) = torch.autograd.grad(y.sum(), xg, create_graph=True)
        torch.autograd.grad(g.sum(), xg)


@pytest.mark.parametrize("T", [5, 100])
@pytest.mark.parametrize("B", [64, 128])
def test_outputs_that_overlap_inputs(T, B):
    """out may be x or the residual; a residual that starts a row later is read before it is overwritten."""
    K = _K()
    rng = np.random.default_rng(16)
    v, cols, _ = weight(rng, 512 // B, 512 // B, 2, B)
    w = K.make_mxfp4(v, cols, 512 // B)
    x, res = rows(rng, T, 512), rows(rng, T, 512)
    want, want_res = K.mxfp4_linear(x, w), K.mxfp4_linear(x, w, residual=res)
    for _ in range(5):
        buf = x.clone()
        assert K.mxfp4_linear(buf, w, out=buf) is buf and torch.equal(buf, want)
        buf = res.clone()
        K.mxfp4_linear(x, w, residual=buf, out=buf)
        assert torch.equal(buf, want_res)
        buf = torch.cat([torch.zeros_like(res[:1]), res])
        K.mxfp4_linear(x, w, residual=buf[1:], out=buf[:T])
        assert torch.equal(buf[:T], want_res)
        buf = torch.cat([x, torch.zeros_like(x[:1])])
        K.mxfp4_linear(buf[:T], w, out=buf[1:])
        assert torch.equal(buf[1:], want)


def test_a_weight_with_other_fields():
    """A weight's fields are fixed; one made from others, or copied, is checked and used as it is."""
    import copy
    from dataclasses import FrozenInstanceError, replace
    K = _K()
    rng = np.random.default_rng(17)
    v, cols, _ = weight(rng, 3, 4, 2, 64)
    w = K.make_mxfp4(v, cols, 4)
    x = rows(rng, 9, 256)
    want = K.mxfp4_linear(x, w)
    with pytest.raises(FrozenInstanceError):
        w.data = w.data.clone()
    for other in (copy.deepcopy(w), replace(w, data=w.data.clone())):
        assert torch.equal(K.mxfp4_linear(x, other), want) and torch.equal(other.dequantize(), w.dequantize())
    for bad in (dict(R=4), dict(data=w.data[:-16]), dict(data=w.data.view(torch.int8)), dict(B=32),
                dict(data=w.data.cpu())):
        broken = replace(w, **bad)
        with pytest.raises(RuntimeError):
            K.mxfp4_linear(x, broken)
        with pytest.raises(RuntimeError):
            broken.dequantize()


def _block():
    from looped_blockell.layers import MLPBlock
    torch.manual_seed(1)
    return MLPBlock(256, 512, use_swiglu=True, tile_size=64, density=0.5, device="cuda", weight_format="mxfp4")


@torch.no_grad()
def test_a_captured_layer_follows_its_parameters():
    """Captured before any eager call: replays see updates, and the eager call after it has a weight of its own."""
    m, ref = _block(), _block()
    x = torch.randn(40, 256, device="cuda", dtype=BF16)
    ref(x)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        y = m(x)
    assert torch.equal(m(x), ref(x))  # the graph has not run yet
    g.replay()
    assert torch.equal(y, ref(x))
    for b in (m, ref):
        b.w_down.values.mul_(-3)
        b.w_up.alive_mask[0, 0] = False
        b.w_up.values[0, 0] = 0  # the graph's topology is that of its capture
    g.replay()
    assert torch.equal(y, ref(x)) and torch.equal(m(x), ref(x))


@torch.no_grad()
def test_a_layer_used_on_two_streams():
    """The weight quantised on one stream is ready on the next one that uses it, and outlives its replacement there."""
    x = torch.randn(40, 256, device="cuda", dtype=BF16)
    want = [_block()(x)]
    m = _block()
    m.w_down.values.mul_(2)
    want.append(m(x))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(3):
        m = _block()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            busy = torch.randn(2000, 2000, device="cuda")
            for _ in range(20):
                busy = busy @ busy * 1e-3
            m.w_down.mxfp4_weight(), m.w_up.mxfp4_weight(), m.w_gate.mxfp4_weight()
        y0 = m(x)
        m.w_down.values.mul_(2)
        y1 = m(x)
        junk = [torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda") for _ in range(4)]
        torch.cuda.synchronize()
        assert torch.equal(y0, want[0]) and torch.equal(y1, want[1])
        del junk


def test_residual_gradient_of_fp32_rows_is_not_rounded():
    K = _K()
    rng = np.random.default_rng(18)
    mats, _ = _ffn(rng)
    x0, dy = rows(rng, 33, 256, F32), rows(rng, 33, 256, F32)
    dx = []
    for add in (False, True):
        x = x0.clone().requires_grad_(True)
        y = K.mxfp4_swiglu(x, mats[0][0], mats[0][1], mats[1][0], mats[1][1], mats[2][0], mats[2][1], add_residual=add)
        dx.append(torch.autograd.grad(y, x, dy)[0])
    assert torch.equal(dx[1], dx[0] + dy)


def test_more_slots_than_the_backward_takes():
    """A column block that 255 block-rows use: the forward and the tile gradients run, dx is refused before it starts."""
    K = _K()
    rng = np.random.default_rng(19)
    cols = torch.zeros(255, 1, dtype=torch.int32, device="cuda")
    v = torch.randn(255, 1, 64, 64, device="cuda").to(BF16).requires_grad_(True)
    x = rows(rng, 3, 64).requires_grad_(True)
    y = K.mxfp4_linear_ad(x.detach(), v, cols)
    assert torch.autograd.grad(y.sum(), v)[0].isfinite().all()
    y = K.mxfp4_linear_ad(x, v, cols)
    with pytest.raises(RuntimeError, match="254"):
        y.sum().backward()


@pytest.mark.parametrize("T", [128 * 74, 128 * 74 - 5, 128 * 73])
@pytest.mark.parametrize("B,dtype", [(64, BF16), (128, BF16), (128, F32)])
def test_many_tokens_equal_the_same_tokens_in_parts(T, B, dtype):
    """The kernels for many tokens (two token tiles to a unit, odd and even numbers of tiles) against those for few."""
    K = _K()
    rng = np.random.default_rng(20)
    v, cols, _ = weight(rng, 8, 4, 3, B, dead=5, dead_row=4)
    w = K.make_mxfp4(v, cols, 4)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(T, 4 * B, generator=g, device="cuda").to(dtype)
    res = torch.randn(T, 8 * B, generator=g, device="cuda").to(dtype)
    big = torch.full((T + 130, 8 * B), 7.0, device="cuda", dtype=dtype)
    y = K.mxfp4_linear(x, w, residual=res, out=big[:T])
    parts = torch.cat([K.mxfp4_linear(a, w, residual=b) for a, b in zip(x.split(1000), res.split(1000))])
    assert torch.equal(y, parts) and (big[T:] == 7).all()
    assert torch.equal(y[:, 4 * B:5 * B], res[:, 4 * B:5 * B])
    assert torch.equal(K.mxfp4_linear(x, w, max_ctas=5), K.mxfp4_linear(x, w))


@pytest.mark.parametrize("T", [128 * 74, 128 * 74 - 5, 128 * 73])
@pytest.mark.parametrize("B,Kg,Ku,Kd", [(64, 2, 3, 5), (128, 1, 5, 8), (128, 2, 7, 8), (128, 19, 3, 8), (128, 18, 20, 1)])
def test_many_tokens_of_a_block_equal_the_same_tokens_in_parts(T, B, Kg, Ku, Kd):
    """As above for the gated block: unequal numbers of slots, dead rows, several stages and units of each CTA."""
    K = _K()
    rng = np.random.default_rng(21)
    C = 20
    mats = [weight(rng, 8, C, Kg, B, dead=4, dead_row=3), weight(rng, 8, C, Ku, B, dead=4, dead_row=5),
            weight(rng, C, 8, Kd, B)]
    packed = [K.make_mxfp4(v, c, n) for (v, c, _), n in zip(mats, (C, C, 8))]
    x = torch.randn(T, C * B, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").to(BF16)
    y = K.mxfp4_swiglu_fwd(x, *packed, add_residual=True)
    parts = torch.cat([K.mxfp4_swiglu_fwd(a, *packed, add_residual=True) for a in x.split(1000)])
    assert torch.equal(y, parts)
    y2, ws = K.mxfp4_swiglu_fwd(x, *packed, add_residual=True, return_intermediates=True)
    assert torch.equal(y, y2) and (ws["gate"][:, 3 * B:4 * B] == 0).all() and (ws["up"][:, 5 * B:6 * B] == 0).all()
    for _ in range(3):
        assert torch.equal(K.mxfp4_swiglu_fwd(x, *packed, add_residual=True), y)
    assert K.read_status() == 0


@pytest.mark.parametrize("T", [1, 32, 33, 128, 300])
@pytest.mark.parametrize("R,C,Kk,B,dead,dtype", [
    (2, 40, 33, 128, 0, BF16), (5, 70, 64, 128, 9, F32), (1, 140, 129, 64, 3, BF16), (12, 80, 64, 64, 0, F32)])
def test_long_rows_shared_by_a_cluster(T, R, C, Kk, B, dead, dtype):
    """Few units of many slots: CTAs of a cluster share each (up to the largest cluster; fewer tokens, more of them)."""
    K = _K()
    rng = np.random.default_rng(22)
    v, cols, w = weight(rng, R, C, Kk, B, dead, dead_row=R - 1 if R > 1 else None)
    x, res = rows(rng, T, C * B, dtype), rows(rng, T, R * B, dtype)
    p = K.make_mxfp4(v, cols, C)
    xq = M.quantize(f64(x))
    check_linear(K.mxfp4_linear(x, p), xq, w, Kk * B // 64)
    y = K.mxfp4_linear(x, p, residual=res)
    check_linear(y, xq, w, Kk * B // 64, f64(res))
    assert torch.equal(y, K.mxfp4_linear(x, p, residual=res))
    assert K.read_status() == 0


@pytest.mark.parametrize("B", [64, 128])
def test_a_column_block_twice_in_a_row(B):
    """Slots of one block-row may share a column block: both count, in the sums and in each one's gradient."""
    K = _K()
    rng = np.random.default_rng(23)
    cols = torch.tensor([[1, 1, 0], [2, -1, 2], [0, 0, 0]], dtype=torch.int32, device="cuda")
    v = torch.from_numpy((rng.standard_normal((3, 3, B, B)) * 0.02).astype(np.float32)).to(BF16).cuda()
    w = M.dense(M.quantize_tiles(f64(v), 0), cols.cpu().numpy(), 3, 0)
    x, dy = rows(rng, 77, 3 * B), rows(rng, 77, 3 * B)
    xq = M.quantize(f64(x))
    leaves = [t.clone().requires_grad_(True) for t in (x, v)]
    y = K.mxfp4_linear_ad(*leaves, cols)
    check_linear(y, xq, w, 3 * B // 64)
    dx, dw = torch.autograd.grad(y, leaves, dy)
    ref = f64(dy) @ w
    assert np.linalg.norm(f64(dx) - ref) <= 2.1 * 2.0 ** -8 * np.linalg.norm(ref)
    full = f64(dy).T @ xq  # [out, in]
    for r in range(3):
        for k, c in enumerate(cols[r].tolist()):
            want = full[r * B:(r + 1) * B, c * B:(c + 1) * B].T if c >= 0 else np.zeros((B, B))
            assert np.linalg.norm(f64(dw[r, k]) - want) <= 2.1 * 2.0 ** -8 * np.linalg.norm(want), (r, k)


def test_offsets_past_32_bits():
    """Rows, chunks, hidden states and gradients of more than 2^32 values: the last tokens as in a call of their own."""
    K = _K()
    rng = np.random.default_rng(24)
    T, n, d, F, B = 270336, 1000, 2048, 16384, 128
    x = torch.zeros(T, d, dtype=BF16, device="cuda")
    dy = torch.zeros(T, d, dtype=BF16, device="cuda")
    x[:n], x[-n:], dy[-n:] = rows(rng, n, d), rows(rng, n, d), rows(rng, n, d)
    mats = [weight(rng, F // B, d // B, 1, B)[:2] for _ in range(2)] + [weight(rng, d // B, F // B, 2, B)[:2]]
    packed = [K.make_mxfp4(v, c, C) for (v, c), C in zip(mats, (d // B, d // B, F // B))]
    y, ws = K.mxfp4_swiglu_fwd(x, *packed, return_intermediates=True)
    y2, ws2 = K.mxfp4_swiglu_fwd(x[-n:].clone(), *packed, return_intermediates=True)
    assert ws["gate"].numel() > 2 ** 32 and ws["q_h"].data.numel() > 2 ** 31
    assert torch.equal(y[-n:], y2) and torch.equal(ws["gate"][-n:], ws2["gate"]) and torch.equal(ws["up"][-n:], ws2["up"])
    h = ws["q_h"].dequantize()
    assert torch.equal(h[-n:], ws2["q_h"].dequantize())
    q = K.mxfp4_quantize(h, B)  # quantising is idempotent
    assert torch.equal(K.mxfp4_dequantize(q)[-n:], h[-n:])
    assert torch.equal(K.mxfp4_linear(q, packed[2])[-n:], y2)
    del ws, h, q, y

    def grads(a, g):
        leaves = [a.requires_grad_(True)] + [v.clone().requires_grad_(True) for v, _ in mats]
        out = K.mxfp4_swiglu(leaves[0], leaves[1], mats[0][1], leaves[2], mats[1][1], leaves[3], mats[2][1])
        return torch.autograd.grad(out, leaves, g)

    many, few = grads(x, dy), grads(x[-n:].detach().clone(), dy[-n:].clone())
    # both are within one rounding and an fp32 sum's order of the same value
    for a, b in zip((many[0][-n:], *many[1:]), few):
        assert torch.linalg.norm(a.float() - b.float()) <= 2.0 ** -7 * torch.linalg.norm(b.float())
    assert (many[0][:-n] == 0).all()
    assert K.read_status() == 0


def test_two_host_threads():
    """Calls from two threads, each on a stream of its own, do not see one another's arguments or errors."""
    import threading
    K = _K()
    rng = np.random.default_rng(25)
    _, packed = _ffn(rng)
    xs = [rows(rng, T, 256) for T in (3, 150)]
    want = [K.mxfp4_swiglu_fwd(x, *packed, add_residual=True) for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(100):
                y = K.mxfp4_swiglu_fwd(xs[i], *packed, add_residual=True)
                try:
                    K.mxfp4_linear(xs[i], packed[0], out=y)
                    wrong.append("not refused")
                except RuntimeError as e:
                    if "out must be" not in str(e):
                        wrong.append(str(e))
            torch.cuda.current_stream().synchronize()
            if not torch.equal(y, want[i]):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and K.read_status() == 0


def tile_errors(grad, ref, cols, B, layout):
    """Each live tile's error norm over its reference's; ref is the dense gradient on the device, float64."""
    R, Kk = cols.shape
    dense = ref.reshape(R, B, -1, B).permute(0, 2, 3, 1)  # [R, C, B_in, B_out]
    want = dense[torch.arange(R, device="cuda")[:, None], cols.clamp(min=0).long()]
    got = grad.double() if layout == 0 else grad.double().transpose(-1, -2)
    e = (torch.linalg.vector_norm(got - want, dim=(-1, -2)) / torch.linalg.vector_norm(want, dim=(-1, -2)))
    return e[cols >= 0]


@pytest.mark.parametrize("T,R,C,Kk,B,dead,layout,dtype", [
    (64, 8, 4, 3, 64, 1, 0, BF16), (777, 16, 16, 4, 64, 3, 0, BF16), (777, 16, 16, 7, 64, 3, 1, F32),
    (5000, 128, 32, 2, 64, 9, 0, BF16), (1000, 8, 8, 3, 128, 2, 0, BF16), (1000, 8, 8, 5, 128, 2, 1, F32),
    (2600, 128, 32, 3, 128, 9, 1, BF16), (2047, 1, 2, 1, 128, 0, 0, BF16), (2047, 1, 3, 2, 64, 0, 1, BF16)])
def test_tile_gradients_repeat_exactly(T, R, C, Kk, B, dead, layout, dtype):
    K = _K()
    rng = np.random.default_rng(T + B)
    v, cols, _ = weight(rng, R, C, Kk, B, dead, dtype=dtype, layout=layout)
    x, dy = rows(rng, T, C * B), rows(rng, T, R * B)
    v.requires_grad_(True)
    y = K.mxfp4_linear_ad(x, v, cols, layout=layout)
    grads = [torch.autograd.grad(y, v, dy, retain_graph=True)[0] for _ in range(8)]
    for g in grads[1:]:
        assert torch.equal(g, grads[0])
    xq = K.mxfp4_dequantize(K.mxfp4_quantize(x, B), F32).double()
    assert tile_errors(grads[0], dy.double().T @ xq, cols, B, layout).max() <= GRAD_TOL
    assert (grads[0][cols < 0] == 0).all()
    assert K.read_status() == 0


@pytest.mark.parametrize("T,d,F,B,Kg,Kd", [(777, 1024, 4096, 64, 4, 16), (1000, 1024, 4096, 128, 3, 6)])
def test_a_training_step_repeats_exactly(T, d, F, B, Kg, Kd):
    K = _K()
    rng = np.random.default_rng(T)
    mats, _ = _ffn(rng, d, F, B, Kg, Kd, 3)
    x, dy = rows(rng, T, d), rows(rng, T, d)
    leaves = [x] + [m[0] for m in mats]
    for t in leaves:
        t.requires_grad_(True)
    first = None
    for _ in range(6):
        y = K.mxfp4_swiglu(x, *(a for m in mats for a in m[:2]), add_residual=True)
        got = (y.detach(), *torch.autograd.grad(y, leaves, dy))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


def _busy():
    a = torch.randn(4000, 4000, device="cuda")
    for _ in range(30):
        a = a @ a * 1e-3
    return a


def test_gradients_on_a_second_stream():
    """A topology that is still being written on one stream is whole on the next stream that uses it."""
    from torch.utils._python_dispatch import TorchDispatchMode
    K = _K()
    rng = np.random.default_rng(30)
    mats, _ = _ffn(rng, 1024, 2048, 64, 4, 16)
    x, dy = rows(rng, 60, 1024), rows(rng, 60, 1024)

    class BehindOtherWork(TorchDispatchMode):  # the topology's last kernels
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            if func is torch.ops.aten.index_put_.default:
                _busy()
            return func(*args, **(kwargs or {}))

    def step(cols):
        ls = [t.detach().requires_grad_(True) for t in [x] + [m[0] for m in mats]]
        y = K.mxfp4_swiglu(ls[0], ls[1], cols[0], ls[2], cols[1], ls[3], cols[2])
        return torch.autograd.grad(y, ls, dy)

    want = step([m[1] for m in mats])
    _busy()
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        cols = [m[1].clone() for m in mats]
        torch.cuda.synchronize()
        with torch.cuda.stream(s), BehindOtherWork():
            K.transposed_topology([cols[2]], 32)
            K.transposed_topology(cols[:2], 16)
        with torch.cuda.stream(t):
            got = step(cols)
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("train", [False, True])
def test_a_layers_columns_on_a_second_stream(train):
    """Masked columns made behind queued work on one stream, used on another by a layer whose weight changed."""
    x = torch.randn(40, 256, device="cuda", dtype=BF16)
    dy = torch.randn(40, 256, device="cuda", dtype=BF16)

    def run(m):
        if not train:
            with torch.no_grad():
                return [m(x)]
        y = m(x)
        return [y.detach(), *torch.autograd.grad(y, [m.w_gate.values, m.w_down.values], dy)]

    ref = _block()
    with torch.no_grad():
        ref.w_up.alive_mask[1:, 0] = False
        ref.w_gate.alive_mask[1:, 1] = False
    want = run(ref)
    s = torch.cuda.Stream()
    for _ in range(5):
        m = _block()
        with torch.no_grad():
            m.w_up.alive_mask[1:, 0] = False
            m.w_gate.alive_mask[1:, 1] = False
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            keep = _busy()
            for w in (m.w_gate, m.w_up, m.w_down):
                w.effective_col_indices()
        got = run(m)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        del keep


def test_twelve_blocks_train_from_a_graph():
    """The topologies of many blocks stay: a second step builds none, and can be captured."""
    K = _K()
    rng = np.random.default_rng(31)
    blocks = [_ffn(rng)[0] for _ in range(12)]
    x, dy = rows(rng, 40, 256, spread=0.5), rows(rng, 40, 256)
    leaves = [x] + [m[0] for b in blocks for m in b]

    def step():
        ls = [t.detach().requires_grad_(True) for t in leaves]
        y = ls[0]
        for i, b in enumerate(blocks):
            vs = ls[1 + 3 * i:4 + 3 * i]
            y = K.mxfp4_swiglu(y, vs[0], b[0][1], vs[1], b[1][1], vs[2], b[2][1], add_residual=True)
        return (y.detach(), *torch.autograd.grad(y, ls, dy))

    want = step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_only_the_wanted_gradients_build_topologies(monkeypatch):
    """d_down needs none, d_gate and d_up that of down, dx both; the gradients are the same."""
    K = _K()
    from looped_blockell.kernels import mxfp4
    rng = np.random.default_rng(38)
    mats, _ = _ffn(rng)
    x, dy = rows(rng, 70, 256), rows(rng, 70, 256)
    built = []
    real = mxfp4.transposed_topology
    monkeypatch.setattr(mxfp4, "transposed_topology", lambda m, n: built.append(len(m)) or real(m, n))
    every = None
    for which, want in (([0, 1, 2, 3], [1, 2]), ([3], []), ([1], [1]), ([2, 3], [1]), ([0], [1, 2])):
        ls = [t.detach().requires_grad_(i in which) for i, t in enumerate([x] + [m[0] for m in mats])]
        built.clear()
        y = K.mxfp4_swiglu(ls[0], ls[1], mats[0][1], ls[2], mats[1][1], ls[3], mats[2][1], add_residual=True)
        got = dict(zip(which, torch.autograd.grad(y, [ls[i] for i in which], dy)))
        every = every or got
        assert built == want and all(torch.equal(g, every[i]) for i, g in got.items())


def _junk():
    """Buffers of the sizes that a layer caches, filled, so that freed ones hold something else."""
    return [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (8, 16, 32, 64, 128) for _ in range(64)]


@torch.no_grad()
def test_a_captured_layer_follows_its_topology():
    """Captured with its caches filled: replays follow the mask, whatever the eager calls between have replaced."""
    m, ref = _block(), _block()
    x = torch.randn(40, 256, device="cuda", dtype=BF16)
    m(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = m(x)
    for b in (m, ref):
        b.w_up.alive_mask[0, 0] = False
        b.w_down.alive_mask[1, 1] = False
    assert torch.equal(m(x), ref(x))
    junk = _junk()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, ref(x))
    del junk


def test_a_captured_training_step_keeps_its_topology():
    """The columns and transposed topologies that a graph reads stay when the layer's are replaced."""
    m = _block()
    x, dy = (torch.randn(40, 256, device="cuda", dtype=BF16) for _ in range(2))
    leaf = x.clone().requires_grad_(True)

    def step():
        y = m(leaf)
        return (y.detach(), *torch.autograd.grad(y, [leaf, m.w_gate.values, m.w_up.values, m.w_down.values], dy))

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for how in range(3):
        with torch.no_grad():
            if how == 0:
                m.w_up.alive_mask[0, 0] = False
            elif how == 1:
                m.w_down.alive_mask[1, 1] = False
            else:
                for w in (m.w_gate, m.w_up, m.w_down):
                    w.refresh()
        step()
        junk = _junk()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del junk


def test_fp32_rows_get_fp32_gradients():
    K = _K()
    rng = np.random.default_rng(32)
    v, cols, w = weight(rng, 4, 6, 3, 64, 1)
    x = rows(rng, 70, 384, F32).requires_grad_(True)
    dy = rows(rng, 70, 256).float()  # bf16 values: rounding dy costs nothing
    (dx,) = torch.autograd.grad(K.mxfp4_linear_ad(x, v, cols), x, dy)
    ref = f64(dy) @ w
    bound = (16 + 4 * 64 * 4 // 16) * 2.0 ** -23 * (np.abs(f64(dy)) @ np.abs(w))
    assert (np.abs(f64(dx) - ref) <= bound + HALF_STEP[F32] * np.abs(ref)).all()


@pytest.mark.parametrize("B", [64, 128])
def test_fp32_rows_of_a_block_get_fp32_gradients(B):
    """dx is not rounded to bf16 on its way, with and without the residual; no tokens, one token."""
    K = _K()
    rng = np.random.default_rng(39)
    mats, _ = _ffn(rng, 4 * B, 8 * B, B)
    for T in (0, 1, 150):
        x, dy = rows(rng, T, 4 * B, F32, 1.0), rows(rng, T, 4 * B, F32)
        dx = []
        for dtype in (F32, BF16):
            leaf = x.to(dtype).requires_grad_(True)
            y = K.mxfp4_swiglu(leaf, *(a for m in mats for a in m[:2]))
            dx.append(torch.autograd.grad(y, leaf, dy.to(dtype))[0])
        assert dx[0].dtype == F32 and dx[1].dtype == BF16 and dx[0].shape == x.shape
        if T:  # bf16 rows of other values have other codes: only the type is compared
            assert (dx[0] != dx[0].bfloat16().float()).float().mean() > 0.9


@pytest.mark.parametrize("T,d,F,B,Kg,dtype,residual", [
    (40, 128, 8192, 64, 2, BF16, True), (1, 128, 8192, 64, 2, F32, True), (200, 64, 20480, 64, 1, BF16, False),
    (130, 256, 16640, 128, 2, F32, True)])
def test_gate_and_up_on_more_than_254_slots(T, d, F, B, Kg, dtype, residual):
    """Column blocks that 256, 640 and 260 block-rows of gate and up use: dx in several passes, also from a graph."""
    K = _K()
    rng = np.random.default_rng(33)
    mats, _ = _ffn(rng, d, F, B, Kg, 3, 2)
    x, dy = rows(rng, T, d, dtype, 1.0), rows(rng, T, d, dtype)
    leaves = [x] + [m[0] for m in mats]
    for t in leaves:
        t.requires_grad_(True)

    def step():
        y = K.mxfp4_swiglu(x, *(a for m in mats for a in m[:2]), add_residual=residual)
        return torch.autograd.grad(y, leaves, dy)

    grads = step()
    packed = [K.make_mxfp4(v.detach(), c, n) for (v, c, _), n in zip(mats, (d // B, d // B, F // B))]
    _, ws = K.mxfp4_swiglu_fwd(x.detach(), *packed, add_residual=residual, return_intermediates=True)
    refs = M.swiglu_backward(M.quantize(f64(x)), *(m[2] for m in mats), f64(ws["q_h"].dequantize(F32)), f64(dy), residual)
    tol = GRAD_TOL + (2.0 ** -8 if dtype == F32 else 0)  # fp32: dy is rounded to bf16 once more
    assert grads[0].dtype == dtype and rel(f64(grads[0]), refs[0]) <= tol
    for g, (_, c, _), ref in zip(grads[1:], mats, refs[1:]):
        assert rel(f64(g), M.tile_grads(ref, f64(c).astype(int), B)) <= tol
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, grads))
    assert K.read_status() == 0


@pytest.mark.parametrize("B", [64, 128])
def test_gates_far_below_zero(B):
    """Gates of -16 to -96.  silu's error: 1.25 |g| 2^-24 for the rounded exponent (2^-24 and 2^-26 of its constant) and
    2^-21 for ex2, rcp, the sum and the products; flushed below -87.3, |g| e^g <= 2^-119.  u adds one rounding, 2^-24."""
    K = _K()
    rng = np.random.default_rng(37)
    d, T = 4 * B, 150
    cols = torch.arange(4, dtype=torch.int32, device="cuda")[:, None].contiguous()

    def diagonal(values):  # exact in MXFP4
        t = torch.zeros(4, 1, B, B, device="cuda")
        t[:, 0] = torch.diag_embed(torch.from_numpy(values.astype(np.float32)).cuda().view(4, B))
        return K.make_mxfp4(t, cols, 4)

    wg = diagonal(np.full(d, 16.0))
    wu = diagonal(rng.choice([1.0, 1.5, 2.0, 3.0, -4.0, 6.0], d) * 2.0 ** 60)
    # a scale block has one gate: its h's differ by u alone
    x = -np.repeat(rng.choice([1.0, 1.5, 2.0, 3.0, 4.0, 6.0], (T, d // 32)), 32, 1)
    out, ws = K.mxfp4_swiglu_fwd(torch.from_numpy(x).to(BF16).cuda(), wg, wu, wg, return_intermediates=True)
    g, u = f64(ws["gate"]), f64(ws["up"])
    h = M.silu_mul(g, u)
    tol = np.abs(h) * (1.25 * np.abs(g) * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -24) + np.abs(u) * 2.0 ** -119
    lo, hi = h - tol, h + tol
    q = f64(ws["q_h"].dequantize(F32)).reshape(T, -1, 32)
    mag, t3 = np.abs(h).reshape(T, -1, 32), tol.reshape(T, -1, 32)
    fits = np.zeros(q.shape[:2], bool)
    for s in (-1, 1):
        sc = M.scales(np.repeat(np.maximum(mag + s * t3, 0).max(-1, keepdims=True), 32, -1))
        a, b = (M.e2m1(v.reshape(T, -1, 32) / sc[..., :1]) * sc[..., :1] for v in (lo, hi))
        fits |= ((q >= np.minimum(a, b)) & (q <= np.maximum(a, b))).all(-1)
    assert fits.all()
    assert K.read_status() == 0


@pytest.mark.parametrize("B,T,d,F,Kg,Ku,Kd", [(64, 777, 1024, 4096, 4, 3, 16), (128, 1000, 1024, 8192, 2, 5, 8)])
def test_backward_of_many_units_equals_the_same_tokens_in_parts(B, T, d, F, Kg, Ku, Kd):
    """Several units for each CTA of the gated backward: dx and the sums of d_gate, d_up."""
    K = _K()
    rng = np.random.default_rng(35)
    mats = [weight(rng, F // B, d // B, Kg, B, 5, dead_row=1), weight(rng, F // B, d // B, Ku, B, 2),
            weight(rng, d // B, F // B, Kd, B, 3)]
    x, dy = rows(rng, T, d, spread=1.0), rows(rng, T, d)

    def grads(a, g):
        ls = [a.detach().requires_grad_(True)] + [m[0].detach().requires_grad_(True) for m in mats]
        y = K.mxfp4_swiglu(ls[0], ls[1], mats[0][1], ls[2], mats[1][1], ls[3], mats[2][1], add_residual=True)
        return torch.autograd.grad(y, ls, g)

    whole = grads(x, dy)
    parts = [grads(x[i:i + 100], dy[i:i + 100]) for i in range(0, T, 100)]
    assert torch.equal(whole[0], torch.cat([p[0] for p in parts]))
    packed = [K.make_mxfp4(m[0], m[1], n) for m, n in zip(mats, (d // B, d // B, F // B))]
    q = K.mxfp4_quantize(x, B)
    _, ws = K.mxfp4_swiglu_fwd(q, *packed, return_intermediates=True)
    xq, hq = K.mxfp4_dequantize(q, F32).double(), ws["q_h"].dequantize(F32).double()
    wg, wu, wd = (torch.from_numpy(m[2]).cuda() for m in mats)
    g, u = xq @ wg.T, xq @ wu.T
    sig = torch.sigmoid(g)
    dh = dy.double() @ wd
    du, dg = dh * g * sig, dh * u * sig * (1 + g * (1 - sig))
    for got, ref, m in zip(whole[1:], (dg.T @ xq, du.T @ xq, dy.double().T @ hq), mats):
        e = tile_errors(got, ref, m[1], B, 0)
        assert e[e.isfinite()].max() <= GRAD_TOL
    assert K.read_status() == 0


@pytest.mark.parametrize("T", [9, 17, 32])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_direct_rows_of_several_groups(T, dtype):
    """x = NULL at tile 128 up to BELL_MX_DIRECT_ROWS rows: what rows quantised before give."""
    import ctypes as C
    K = _K()
    from looped_blockell.kernels import _lib as L
    rng = np.random.default_rng(36)
    lib = L.load()
    kind = L.BELL_DTYPE_BF16 if dtype == BF16 else L.BELL_DTYPE_F32
    mats, packed = _ffn(rng, 1024, 2560, 128, 5, 9, 2)
    x = rows(rng, T, 2560, dtype)
    stream = torch.cuda.current_stream().cuda_stream
    for w, n in ((packed[2], 1024),):
        out = torch.full((T, n), 7.0, dtype=dtype, device="cuda")
        d = L.BellMxLinearDesc(T, kind, 0, None, x.data_ptr(), 2560, kind, 0, None, out.data_ptr(), w._abi, None)
        assert lib.bell_linear_mx(C.byref(d), stream) == 0
        assert torch.equal(out, K.mxfp4_linear(K.mxfp4_quantize(x, 128), w, out_dtype=dtype))
    x = rows(rng, T, 1024, dtype)
    out = torch.full((T, 1024), 7.0, dtype=dtype, device="cuda")
    h = torch.empty(lib.bell_mx_rows_bytes(T, 2560, 128), dtype=torch.uint8, device="cuda")
    d = L.BellMxFFNDesc(T, kind, 0, None, x.data_ptr(), 1024, kind, 0, None, h.data_ptr(), None, None, out.data_ptr(),
                        *(p._abi for p in packed), None)
    assert lib.bell_swiglu_fwd_mx(C.byref(d), stream) == 0
    want = K.mxfp4_swiglu_fwd(K.mxfp4_quantize(x, 128), *packed) if dtype == BF16 else \
        K.mxfp4_swiglu_fwd(x, *packed, return_intermediates=True)[0]
    assert torch.equal(out, want)
    assert K.read_status() == 0


@pytest.mark.parametrize("T", [1, 8, 9, 32, 33, 64, 128, 129])
@pytest.mark.parametrize("R,Kk,B,dead,dtype", [
    (3, 16, 128, 5, BF16), (16, 32, 128, 0, F32), (18, 44, 128, 9, BF16), (3, 24, 64, 7, BF16), (16, 64, 64, 3, F32),
    (70, 33, 64, 0, BF16)])
def test_rows_that_begin_to_be_shared(T, R, Kk, B, dead, dtype):
    """Around the lengths from which clusters share a unit: dead slots, rows quantised before and on the way."""
    K = _K()
    rng = np.random.default_rng(T + Kk)
    v, cols, w = weight(rng, R, 2 * Kk, Kk, B, dead, dead_row=1 if dead else None)
    mw = K.make_mxfp4(v, cols, 2 * Kk)
    x, res = rows(rng, T, 2 * Kk * B, dtype), rows(rng, T, R * B, dtype)
    y = K.mxfp4_linear(x, mw, residual=res)
    check_linear(y, M.quantize(f64(x)), w, Kk * B // 64, f64(res))
    assert torch.equal(y, K.mxfp4_linear(K.mxfp4_quantize(x, B), mw, residual=res, out_dtype=dtype))
    assert torch.equal(y, K.mxfp4_linear(x, mw, residual=res)) and K.read_status() == 0


@pytest.mark.parametrize("T", [16, 17, 32])
def test_a_captured_call_gives_the_same_bits(T):
    """Captured calls may quantise their rows first where eager ones do not."""
    K = _K()
    rng = np.random.default_rng(40)
    _, packed = _ffn(rng, 512, 2048, 64, 4, 24, 3)
    x, h = rows(rng, T, 512), rows(rng, T, 2048)
    want = K.mxfp4_swiglu_fwd(x, *packed, add_residual=True), K.mxfp4_linear(h, packed[2])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = K.mxfp4_swiglu_fwd(x, *packed, add_residual=True), K.mxfp4_linear(h, packed[2])
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_gradients_that_start_anywhere():
    """The output's gradient as a slice of a larger one, at any element, and as an expanded scalar."""
    K = _K()
    rng = np.random.default_rng(41)
    mats, _ = _ffn(rng)
    x, dy = rows(rng, 9, 256).requires_grad_(True), rows(rng, 9, 256)
    vs = [m[0].requires_grad_(True) for m in mats]

    def ffn():
        return K.mxfp4_swiglu(x, vs[0], mats[0][1], vs[1], mats[1][1], vs[2], mats[2][1], add_residual=True)

    def linear():
        return K.mxfp4_linear_ad(x, vs[0], mats[0][1])[:, :256].contiguous()

    for call, leaves in ((ffn, [x] + vs), (linear, [x, vs[0]])):
        want = torch.autograd.grad(call(), leaves, dy)
        for start in (1, 3, 4, 8):
            y = torch.cat([torch.zeros(start, dtype=BF16, device="cuda"), call().reshape(-1)])
            weights = torch.cat([torch.zeros(start, dtype=BF16, device="cuda"), dy.reshape(-1)])
            got = torch.autograd.grad(y, leaves, weights)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        ones = torch.autograd.grad(call(), leaves, torch.ones_like(dy))
        got = torch.autograd.grad(call().sum(), leaves)
        assert all(torch.equal(a, b) for a, b in zip(got, ones))
    flat = torch.zeros(9 * 512 + 8, dtype=BF16, device="cuda")
    for start in (0, 1, 4, 8):
        g = flat[start:start + 9 * 512].view(9, 512).copy_(rows(np.random.default_rng(1), 9, 512))
        got = torch.autograd.grad(K.mxfp4_linear_ad(x, vs[0], mats[0][1]), [x, vs[0]], g)
        want = torch.autograd.grad(K.mxfp4_linear_ad(x, vs[0], mats[0][1]), [x, vs[0]], g.clone())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_weight_put_together_from_fields_is_checked():
    """Fields that do not fit the plan are refused before a kernel follows it; those that do are used."""
    import copy
    import pickle
    from dataclasses import replace
    K = _K()
    rng = np.random.default_rng(42)
    v, cols, _ = weight(rng, 6, 5, 3, 64, 2)
    cols[0, 0] = 4
    w = K.make_mxfp4(v, cols, 5)
    x = rows(rng, 9, 320)
    want = K.mxfp4_linear(x, w)
    for bad in (dict(C=4), dict(C=0), dict(C=1 << 16), dict(R=3, K=6), dict(R=9, K=2), dict(R=2, K=9), dict(R=1, K=18),
                dict(data=torch.zeros_like(w.data)), dict(data=torch.full_like(w.data, 255))):
        broken = replace(w, **bad)
        with pytest.raises(RuntimeError):
            K.mxfp4_linear(rows(rng, 9, 64 * max(1, min(broken.C, 16))), broken)
        with pytest.raises(RuntimeError, match="plan"):
            broken.dequantize()
    fits = replace(w, C=7)  # columns 5 and 6 are not used
    assert torch.equal(K.mxfp4_linear(torch.cat([x, x[:, :128]], 1), fits), want)
    for other in (copy.deepcopy(w), pickle.loads(pickle.dumps(w)), replace(w, data=w.data.clone())):
        assert torch.equal(K.mxfp4_linear(x, other), want)
    fresh, unused = copy.deepcopy(w), replace(w, data=w.data.clone())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = K.mxfp4_linear(x, fresh)  # a copy of a made weight needs no check
        with pytest.raises(RuntimeError, match="capture"):
            K.mxfp4_linear(x, unused)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want) and K.read_status() == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,F", [(64, 512), (128, 1024), (64, 8192)])
def test_gradients_of_no_tokens(B, F, dtype):
    """Empty dx, tile gradients that are zero whatever lay in their memory; 8192 features take dx in two passes."""
    K = _K()
    rng = np.random.default_rng(43)
    mats, _ = _ffn(rng, 2 * B, F, B, 2, 3, 1)
    x = torch.zeros(0, 2 * B, dtype=dtype, device="cuda", requires_grad=True)
    vs = [m[0].to(dtype).requires_grad_(True) for m in mats]
    for _ in range(2):
        junk = [torch.full_like(v, 7.0) for v in vs]
        del junk
        y = K.mxfp4_swiglu(x, vs[0], mats[0][1], vs[1], mats[1][1], vs[2], mats[2][1], add_residual=True)
        dx, *dws = torch.autograd.grad(y, [x] + vs, torch.zeros_like(y))
        assert dx.shape == x.shape and dx.dtype == dtype
        assert all(g.dtype == dtype and (g == 0).all() for g in dws)
        y = K.mxfp4_linear_ad(x, vs[0], mats[0][1])
        dx, dw = torch.autograd.grad(y, [x, vs[0]], torch.zeros_like(y))
        assert dx.shape == x.shape and (dw == 0).all()
    assert K.read_status() == 0
