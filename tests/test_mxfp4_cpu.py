"""MXFP4 on the host: the float64 definition itself, buffer sizes, and the
refusals of the C ABI and the Python entry points (nothing is launched)."""

import ctypes as C
import os

import numpy as np
import pytest
import torch

from oracle import mxfp4_oracle as M


def _L():
    from looped_blockell.kernels import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    return _lib


def test_e2m1_ties_go_to_the_even_code():
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    np.testing.assert_array_equal(M.e2m1(ties), [0, 1, 1, 2, 2, 4, 4])
    np.testing.assert_array_equal(M.e2m1(-ties), [0, -1, -1, -2, -2, -4, -4])
    np.testing.assert_array_equal(M.e2m1(np.nextafter(ties, 9)), [0.5, 1, 1.5, 2, 3, 4, 6])
    np.testing.assert_array_equal(M.e2m1(np.nextafter(ties, 0)), [0, 0.5, 1, 1.5, 2, 3, 4])
    assert M.e2m1(np.array([100.0]))[0] == 6


def test_quantize_is_idempotent_and_bounded():
    v = np.random.default_rng(0).standard_normal((5, 96)) * 10.0 ** np.arange(-2, 3)[:, None]
    q = M.quantize(v)
    np.testing.assert_array_equal(M.quantize(q), q)
    s = np.repeat(M.scales(v), 32, -1)
    # half a step is at most s; a value in (6, 8) s saturates, off by less than 2 s
    assert (np.abs(q - v) <= np.where(np.abs(v) <= 6 * s, 1.0, 2.0) * s).all()
    np.testing.assert_array_equal(M.scales(np.zeros((1, 32))), [[2.0 ** -127]])


def test_straight_through_gradients_against_differences():
    """The backward's formula is the derivative of the block in which Q(h) is h
    plus a constant (what straight-through means), at the quantised operands."""
    rng = np.random.default_rng(1)
    x, wg, wu, wd, dy = (rng.standard_normal(s) for s in ((3, 8), (6, 8), (6, 8), (8, 6), (3, 8)))
    hq0 = rng.standard_normal((3, 6))
    shift = hq0 - M.silu_mul(x @ wg.T, x @ wu.T)

    def loss(x, wg, wu, wd):
        return float((dy * ((M.silu_mul(x @ wg.T, x @ wu.T) + shift) @ wd.T + x)).sum())

    grads = M.swiglu_backward(x, wg, wu, wd, hq0, dy, True)
    eps = 1e-6
    for i, (t, g) in enumerate(zip((x, wg, wu, wd), grads)):
        for at in [(0, 0), (1, 3), (2, 5)]:
            args = [a.copy() for a in (x, wg, wu, wd)]
            args[i][at] += eps
            up = loss(*args)
            args[i][at] -= 2 * eps
            # a central difference of O(10) sums: 1e-16 * 1e2 / 1e-6 rounding and eps^2 truncation
            assert abs((up - loss(*args)) / (2 * eps) - g[at]) < 1e-6 * (1 + abs(g[at]))


def test_sizes():
    L = _L()
    lib = L.load()
    from looped_blockell.kernels import mxfp4
    for T, f, B in [(1, 128, 128), (128, 64, 64), (129, 192, 64), (1000, 4096, 128)]:
        assert lib.bell_mx_rows_bytes(T, f, B) == mxfp4._rows_bytes(T, f, B)
    assert lib.bell_mx_tiles_bytes(3, 2, 64) == 6 * (64 * 32 + 512)
    assert lib.bell_mx_tiles_bytes(3, 2, 128) == 6 * (128 * 64 + 512)
    assert lib.bell_mx_rows_bytes(0, 128, 128) == 0 and lib.bell_mx_rows_bytes(5, 128, 32) == 0
    assert lib.bell_mx_tiles_bytes(0, 2, 64) == 0


def test_rows_refusals():
    L = _L()
    lib = L.load()
    q = lambda *a: lib.bell_mx_quantize_rows(*a, None)  # noqa: E731
    assert q(4, 128, 32, 0, 1024, 128, 1024) == -2 and "64 or 128" in L.last_error()
    assert q(-1, 128, 128, 0, 1024, 128, 1024) == -2
    assert q(4, 192, 128, 0, 1024, 192, 1024) == -2 and "multiple of B" in L.last_error()
    assert q(4, 128, 128, 7, 1024, 128, 1024) == -1
    assert q(4, 128, 128, 0, None, 128, 1024) == -8
    assert q(4, 128, 128, 0, 1024, 64, 1024) == -3  # rows overlap
    assert q(4, 128, 128, 0, 1024, 132, 1024) == -3  # 264 bytes
    assert q(4, 128, 128, 0, 1032, 128, 1024) == -3
    assert lib.bell_mx_dequantize_rows(4, 128, 128, 1024, 0, 1028, 128, None) == -3


def test_pack_refusals():
    L = _L()
    lib = L.load()
    ok = dict(values=1024, col_indices=1024, R=2, C=2, K=2, B=64, layout=0, flags=0)

    def call(dtype=0, chunks=1024, plan=1024, n=1, **kw):
        return lib.bell_mx_pack_ell(C.byref(L.BellEll(*{**ok, **kw}.values())), n, dtype, (C.c_void_p * 1)(chunks),
                                    (C.c_void_p * 1)(plan), None, None)

    assert call(B=32) == -2 and call(K=0) == -2 and call(C=1 << 16) == -2 and call(R=1 << 24) == -2
    assert call(dtype=3) == -1 and call(layout=5) == -8 and call(values=None) == -8 and call(plan=None) == -8
    assert call(values=1032) == -3 and call(n=0) == -8 and call(n=4) == -8
    assert lib.bell_mx_unpack_tiles(1024, 2, None, 0, 64, None, 3, 1024, None) == -2
    assert lib.bell_mx_unpack_tiles(1024, 2, None, 0, 32, None, 2, 1024, None) == -2


def _mx(L, R, C_, K=2, B=64, chunks=1024, plan=1024):
    return L.BellMxEll(chunks, plan, R, C_, K, B)


def test_linear_and_ffn_refusals():
    L = _L()
    lib = L.load()
    assert lib.bell_linear_mx(None, None) == -8 and lib.bell_swiglu_fwd_mx(None, None) == -8

    def lin(**kw):
        d = L.BellMxLinearDesc()
        d.T, d.x, d.out, d.w = 5, 1024, 1024, _mx(L, 2, 3)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.bell_linear_mx(C.byref(d), None)

    assert lin(w=_mx(L, 2, 3, B=16)) == -2 and lin(w=_mx(L, 0, 3)) == -2 and lin(w=_mx(L, 2, 3, plan=None)) == -8
    assert lin(T=-1) == -2 and lin(T=1 << 31) == -2 and lin(T=(1 << 31) - 300, w=_mx(L, 64, 3)) == -2
    assert lin(out_dtype=9) == -1 and lin(x=None) == -8 and lin(out=1025) == -3 and lin(residual=1026) == -3
    assert lin(max_ctas=-1) == -8
    assert lin(x=None, x_src=1024, ld_src=192, T=L.BELL_MX_DIRECT_ROWS + 1) == -8 and "DIRECT_ROWS" in L.last_error()

    def ffn(**kw):
        d = L.BellMxFFNDesc()
        d.T, d.x, d.h, d.out = 5, 1024, 1024, 1024
        d.gate, d.up, d.down = _mx(L, 4, 2), _mx(L, 4, 2), _mx(L, 2, 4)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.bell_swiglu_fwd_mx(C.byref(d), None)

    assert ffn(up=_mx(L, 4, 3)) == -2 and "gate and up" in L.last_error()
    assert ffn(down=_mx(L, 2, 5)) == -2 and ffn(down=_mx(L, 2, 4, B=128)) == -2
    assert ffn(gate_pre=1024) == -8 and "together" in L.last_error()
    assert ffn(h=None) == -8 and ffn(out_dtype=4) == -1


def test_python_refuses_what_is_not_on_a_gpu_or_does_not_fit():
    _L()
    from looped_blockell import kernels as K
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    v, c = torch.zeros(2, 1, 64, 64), torch.zeros(2, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        K.mxfp4_quantize(x)
    with pytest.raises(RuntimeError, match="tile size"):
        K.mxfp4_quantize(x, tile=32)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        K.make_mxfp4(v, c, 2)
    with pytest.raises(RuntimeError, match="bf16 or fp32"):
        K.make_mxfp4(v.half(), c, 2)
    with pytest.raises(RuntimeError, match="4D"):
        K.mxfp4_swiglu(x, v[0], c, v, c, v, c)
    with pytest.raises(RuntimeError, match="not a multiple"):
        K.mxfp4_swiglu(x[:, :100], v, c, v, c, v, c)


def test_backward_refusals():
    L = _L()
    lib = L.load()
    assert lib.bell_linear_bwd_mx(None, None) == -8 and lib.bell_swiglu_bwd_mx(None, None) == -8
    assert lib.bell_linear_bwd_mx_workspace_bytes(None) == 0 and lib.bell_swiglu_bwd_mx_workspace_bytes(None) == 0
    d = L.BellMxLinearBwdDesc()
    d.T, d.grad_out, d.x, d.w = 4, 1024, 1024, _mx(L, 2, 3)
    d.workspace = 1024
    d.dx = 1024
    assert lib.bell_linear_bwd_mx(C.byref(d), None) == -8 and "transposed" in L.last_error()
    d.dx, d.dw, d.col_indices, d.grad_dtype = None, 1024, 1024, 5
    assert lib.bell_linear_bwd_mx(C.byref(d), None) == -8
    d.grad_dtype, d.workspace = 0, None
    assert lib.bell_linear_bwd_mx(C.byref(d), None) == -3
    d.K_t, d.dx = 1, 1024
    # unpacked transpose [3, 1] tiles + plan + Q(x) + fp32 sums of [2, 2] tiles, each padded to 256 bytes
    assert lib.bell_linear_bwd_mx_workspace_bytes(C.byref(d)) == 3 * 64 * 64 * 2 + 256 + 4 * 192 * 2 + 4 * 64 * 64 * 4
    d.cols_t = d.index_t = d.workspace = 1024
    d.K_t = 255
    assert lib.bell_linear_bwd_mx(C.byref(d), None) == -2 and "254" in L.last_error()
    f = L.BellMxFFNBwdDesc()
    f.T, f.gate, f.up, f.down = 4, _mx(L, 4, 2), _mx(L, 4, 2), _mx(L, 2, 4)
    f.grad_out = f.x = f.h = f.workspace = 1024
    assert lib.bell_swiglu_bwd_mx(C.byref(f), None) == -8 and "topologies" in L.last_error()
    assert lib.bell_swiglu_bwd_mx_workspace_bytes(C.byref(f)) == 0
    f.up = _mx(L, 4, 3)
    assert lib.bell_swiglu_bwd_mx(C.byref(f), None) == -2
    f.up, f.dx = _mx(L, 4, 2), 1024
    f.cols_t_down = f.index_t_down = f.cols_t_gate_up = f.index_t_gate_up = 1024
    for kd, kg, name in [(255, 1, "down"), (1, 255, "gate and up")]:
        f.K_t_down, f.K_t_gate_up = kd, kg
        assert lib.bell_swiglu_bwd_mx(C.byref(f), None) == -2 and "254" in L.last_error() and name in L.last_error()


def test_a_copied_layer_makes_its_own_kernel_copies():
    """A copy or a pickle holds no buffer that was derived for the original."""
    import copy
    import pickle
    from looped_blockell.layers import MLPBlock
    m = MLPBlock(128, 256, use_swiglu=True, tile_size=64, weight_format="mxfp4")
    m.w_gate.effective_col_indices()
    for other in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        assert "_kcache" not in other.w_gate.__dict__ and torch.equal(other.w_gate.values, m.w_gate.values)
    assert "_kcache" in m.w_gate.__dict__


def test_backward_refuses_misaligned_buffers():
    """Every pointer of both backwards is checked before anything is launched: the gated one's workspace for 32 bytes."""
    L = _L()
    lib = L.load()
    d = L.BellMxLinearBwdDesc()

    def lin(**kw):
        d.T, d.grad_out, d.x, d.w, d.K_t = 4, 1024, 1024, _mx(L, 2, 3), 1
        d.workspace = d.dx = d.dw = d.col_indices = d.cols_t = d.index_t = 1024
        d.layout = d.grad_dtype = 0
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.bell_linear_bwd_mx(C.byref(d), None)

    for name in ("grad_out", "x", "dx", "dw", "workspace"):
        assert lin(**{name: 1032}) == -3, name
    assert lin(w=_mx(L, 2, 3, chunks=1032)) == -3 and lin(index_t=1028) == -3
    assert lin(col_indices=1026) == -3 and lin(cols_t=1026) == -3
    assert lin(layout=2) == -8 and lin(w=_mx(L, 2, 1 << 16)) == -2
    f = L.BellMxFFNBwdDesc()

    def ffn(**kw):
        f.T, f.gate, f.up, f.down = 4, _mx(L, 4, 2), _mx(L, 4, 2), _mx(L, 2, 4)
        for n in ("grad_out", "x", "h", "workspace", "cols_gate", "cols_up", "cols_down", "cols_t_down", "index_t_down",
                  "cols_t_gate_up", "index_t_gate_up", "dx", "d_gate", "d_up", "d_down"):
            setattr(f, n, 1024)
        f.K_t_down = f.K_t_gate_up = 1
        f.layout = 0
        for k, v in kw.items():
            setattr(f, k, v)
        return lib.bell_swiglu_bwd_mx(C.byref(f), None)

    assert ffn(workspace=1024 + 16) == -3 and "32" in L.last_error()
    for name in ("grad_out", "x", "h", "dx", "d_gate", "d_up", "d_down", "workspace"):
        assert ffn(**{name: 1032}) == -3, name
    for name, m in (("gate", _mx(L, 4, 2, chunks=1032)), ("up", _mx(L, 4, 2, plan=1032)), ("down", _mx(L, 2, 4, chunks=1032))):
        assert ffn(**{name: m}) == -3, name
    for name in ("index_t_down", "index_t_gate_up"):
        assert ffn(**{name: 1028}) == -3, name
    for name in ("cols_gate", "cols_up", "cols_down", "cols_t_down", "cols_t_gate_up"):
        assert ffn(**{name: 1026}) == -3, name
    assert ffn(layout=-1) == -8


@pytest.mark.parametrize("swiglu", [True, False])
def test_a_module_pickled_without_a_weight_format(swiglu):
    """Modules from before the choice hold no such attribute: they compute as they did, in the native format."""
    import pickle
    from looped_blockell.layers import MLPBlock
    m = MLPBlock(128, 256, use_swiglu=swiglu, tile_size=64)
    for part in m.modules():
        part.__dict__.pop("weight_format", None)
    other = pickle.loads(pickle.dumps(m))
    with pytest.raises(RuntimeError, match="CUDA"):  # the forward reaches the kernels, which need a GPU
        other(torch.zeros(1, 128))


def test_a_residual_needs_add_residual():
    """It was dropped without a word."""
    _L()
    from looped_blockell import kernels as K
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="add_residual"):
        K.mxfp4_swiglu_fwd(x, None, None, None, residual=x)


def test_backward_refuses_other_types_of_dx():
    L = _L()
    lib = L.load()
    d = L.BellMxLinearBwdDesc()
    d.T, d.grad_out, d.x, d.w, d.K_t = 4, 1024, 1024, _mx(L, 2, 3), 1
    d.workspace = d.dx = d.cols_t = d.index_t = 1024
    d.dx_dtype = 2
    assert lib.bell_linear_bwd_mx(C.byref(d), None) == -1 and "dx_dtype" in L.last_error()
    f = L.BellMxFFNBwdDesc()
    f.T, f.gate, f.up, f.down = 4, _mx(L, 4, 2), _mx(L, 4, 2), _mx(L, 2, 4)
    f.grad_out = f.x = f.h = f.workspace = f.dx = 1024
    f.cols_t_down = f.index_t_down = f.cols_t_gate_up = f.index_t_gate_up = 1024
    f.K_t_down = f.K_t_gate_up = 1
    f.dx_dtype = 2
    assert lib.bell_swiglu_bwd_mx(C.byref(f), None) == -1 and "dx_dtype" in L.last_error()
