"""MXFP4 Block-ELL: microscaled 4-bit floats (OCP Microscaling Formats 1.0)
for weights and activations, products on the tensor cores' block-scaled MMA.

A block is 32 consecutive values along the contraction: for a row of
activations along its features, for a tile along ``B_in``.  With ``a`` the
largest magnitude of a block and ``s = 2**max(floor(log2 a) - 2, -127)``,

    Q(v) = s * e2m1(v / s)

where e2m1 rounds to nearest even on {0, .5, 1, 1.5, 2, 3, 4, 6} and
saturates.  A block that holds an infinity or a NaN is NaN throughout.

* ``mxfp4_quantize`` / ``mxfp4_dequantize``: activation rows (``MXRows``).
* ``make_mxfp4``: a quantised Block-ELL weight (``MXBlockELL``), once per
  weight set for serving, on every step in training.
* ``mxfp4_linear``: ``Q(x) Q(W)^T (+ residual)``.
* ``mxfp4_swiglu_fwd``: the gated feed-forward block, h quantised on its way
  from the gate/up kernel to the down projection.
* ``mxfp4_linear_ad``, ``mxfp4_swiglu``: the same, differentiable.  The
  gradient passes straight through Q: the backward is the bf16 one at the
  quantised operands (their values are exact in bf16).

Where ``ternary`` keeps 2 bits a weight and int8 activations, this keeps
4.25 bits of both, at tile sizes 64 and 128.  Stream-ordered on torch's
current stream; CUDA tensors only.
"""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional, Union

import torch

from . import _lib
from .backward import block_ell_sddmm, down_silu_bwd, silu_mul_bwd, transposed_topology
from .ops import TILE_IN_OUT, TILE_OUT_IN, _check_cuda, _check_out, _prep_ell, _stream, block_ell_linear, plan_bytes

_DTYPES = {torch.bfloat16: _lib.BELL_DTYPE_BF16, torch.float32: _lib.BELL_DTYPE_F32}
_ROWS = 128  # tokens of one chunk of quantised rows


def _check_tile(tile: int) -> None:
    if tile not in (64, 128):
        raise RuntimeError(f"MXFP4 needs tile size 64 or 128, got {tile}")


def _rows_bytes(T: int, features: int, tile: int) -> int:
    return -(-T // _ROWS) * (features // tile) * (_ROWS * tile // 2 + 512)


@dataclass
class MXRows:
    """Quantised rows ``[T, features]`` for products with weights of tile size
    ``tile``; ``data`` is in the kernels' operand layout (include/bell.h)."""
    data: torch.Tensor  # uint8
    T: int
    features: int
    tile: int

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return mxfp4_dequantize(self, dtype)


@dataclass
class MXBlockELL:
    """A quantised Block-ELL weight (``make_mxfp4``)."""
    data: torch.Tensor         # uint8: the quantised tiles, operand layout
    plan: torch.Tensor         # uint8: live slots of each block-row
    col_indices: torch.Tensor  # int32 [R, K]
    R: int
    K: int
    C: int                     # input column blocks
    B: int

    def __post_init__(self):
        self._abi = _lib.BellMxEll(self.data.data_ptr(), self.plan.data_ptr(), self.R, self.C, self.K, self.B)

    @property
    def in_features(self) -> int:
        return self.C * self.B

    @property
    def out_features(self) -> int:
        return self.R * self.B

    def dequantize(self, layout: int = TILE_IN_OUT) -> torch.Tensor:
        """The quantised values as bf16 tiles ``[R, K, B, B]`` (dead slots too)."""
        v = _unpack((self,), None, self.R * self.K).view(self.R, self.K, self.B, self.B)
        return v if layout == TILE_OUT_IN else v.transpose(-1, -2).contiguous()


def _rows_2d(name: str, x: torch.Tensor) -> torch.Tensor:
    """x as 2-D rows the kernels can read: unit stride along the features, rows
    16 bytes aligned (a copy where it is not)."""
    _check_cuda(name, x)
    if x.dim() != 2:
        raise RuntimeError(f"{name} must be 2D [N, features]")
    if x.dtype not in _DTYPES:
        raise RuntimeError(f"{name} must be bf16 or fp32")
    per16 = 16 // x.element_size()
    T, f = x.shape
    if x.is_contiguous() and f % per16 == 0:
        ok = x.data_ptr() % 16 == 0
    else:
        ok = x.stride(1) == 1 and (T < 2 or (x.stride(0) >= f and x.stride(0) % per16 == 0)) and x.data_ptr() % 16 == 0
    return x if ok else x.clone(memory_format=torch.contiguous_format)


def _ld(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def mxfp4_quantize(x: torch.Tensor, tile: int = 128) -> MXRows:
    """Quantise rows ``x [T, features]`` (bf16 or fp32, ``features`` a multiple
    of ``tile``, the tile size of the weights they will meet)."""
    _check_tile(tile)
    x = _rows_2d("x", x)
    T, f = x.shape
    if f % tile or f == 0:
        raise RuntimeError(f"features={f} is not a multiple of the tile size {tile}")
    data = torch.empty(_rows_bytes(T, f, tile), dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().bell_mx_quantize_rows(T, f, tile, _DTYPES[x.dtype], x.data_ptr(), _ld(x),
                                                     data.data_ptr(), _stream()), "mxfp4_quantize")
    return MXRows(data, T, f, tile)


def mxfp4_dequantize(q: MXRows, dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values that ``q`` holds, ``[T, features]``; exact in bf16 and fp32."""
    _check_rows(q)
    if dtype not in _DTYPES:
        raise RuntimeError("dtype must be bf16 or fp32")
    if out is None:
        out = torch.empty((q.T, q.features), dtype=dtype, device=q.data.device)
    else:
        _check_out("out", out, (q.T, q.features), dtype, q.data.device)
    with torch.cuda.device(q.data.device):
        _lib.check(_lib.load().bell_mx_dequantize_rows(q.T, q.features, q.tile, q.data.data_ptr(), _DTYPES[dtype],
                                                       out.data_ptr(), q.features, _stream()), "mxfp4_dequantize")
    return out


def _check_rows(q: MXRows) -> None:
    _check_cuda("quantised rows", q.data)
    if q.data.numel() < _rows_bytes(q.T, q.features, q.tile) or q.data.dtype != torch.uint8 or \
            not q.data.is_contiguous():
        raise RuntimeError("MXRows.data does not hold T x features quantised values")


def make_mxfp4(values: torch.Tensor, col_indices: torch.Tensor, C_blocks: int, layout: int = TILE_IN_OUT) -> MXBlockELL:
    """Quantise the tiles of a Block-ELL weight (``values [R, K, B, B]`` bf16 or
    fp32, B 64 or 128) and list its live slots.  A column index of -1 is a dead
    slot; one outside [0, C_blocks) is dropped and sets the status word."""
    if values.dtype not in _DTYPES:
        raise RuntimeError("tiles must be bf16 or fp32")
    v, cols = _prep_ell("weight", values, col_indices, values.dtype)
    R, K, B, B2 = v.shape
    _check_tile(B)
    if B2 != B or tuple(cols.shape) != (R, K):
        raise RuntimeError(f"values {tuple(v.shape)} and col_indices {tuple(cols.shape)} do not fit")
    if cols.device != v.device:
        raise RuntimeError("values and col_indices must be on one device")
    data = torch.empty(R * K * (B * B // 2 + 512), dtype=torch.uint8, device=v.device)
    plan = torch.empty(plan_bytes(0, 0, 0, R, K), dtype=torch.uint8, device=v.device)
    w = _lib.BellEll(v.data_ptr(), cols.data_ptr(), R, int(C_blocks), K, B, layout, 0)
    with torch.cuda.device(v.device):
        _lib.check(_lib.load().bell_mx_pack_ell(C.byref(w), _DTYPES[v.dtype], data.data_ptr(), plan.data_ptr(), None,
                                                _stream()), "make_mxfp4")
    return MXBlockELL(data, plan, cols, R, K, int(C_blocks), B)


def _unpack(weights, index: Optional[torch.Tensor], n: int) -> torch.Tensor:
    """bf16 tiles ``[n, B_out, B_in]`` of one or two stacked weights, gathered by ``index``."""
    w0 = weights[0]
    w1 = weights[1] if len(weights) > 1 else None
    out = torch.empty((n, w0.B, w0.B), dtype=torch.bfloat16, device=w0.data.device)
    with torch.cuda.device(w0.data.device):
        _lib.check(_lib.load().bell_mx_unpack_tiles(
            w0.data.data_ptr(), w0.R * w0.K, w1.data.data_ptr() if w1 is not None else None,
            w1.R * w1.K if w1 is not None else 0, w0.B, index.data_ptr() if index is not None else None, n,
            out.data_ptr(), _stream()), "mxfp4 unpack")
    return out


def _same_device(dev, *weights) -> None:
    for w in weights:
        if w.data.device != dev:
            raise RuntimeError(f"weight is on {w.data.device}, x on {dev}")


def _source(desc, x, tile: int, features: int):
    """Point ``desc`` at the rows of x (quantised already, or to be quantised
    into a workspace); returns (T, device, output dtype, the rows' buffer)."""
    if isinstance(x, MXRows):
        _check_rows(x)
        if x.tile != tile or x.features != features:
            raise RuntimeError(f"quantised rows of {x.features} features, tile {x.tile}; the weight needs {features}, "
                               f"tile {tile}")
        desc.x = x.data.data_ptr()
        return x.T, x.data.device, torch.bfloat16, x.data
    T, f = x.shape
    if f != features:
        raise RuntimeError(f"x has {f} features, the weight {features}")
    buf = torch.empty(_rows_bytes(T, f, tile), dtype=torch.uint8, device=x.device)
    desc.x, desc.x_src, desc.ld_src, desc.src_dtype = buf.data_ptr(), x.data_ptr(), _ld(x), _DTYPES[x.dtype]
    return T, x.device, x.dtype, buf


def _out_and_residual(desc, T, features, dtype, dev, out, out_dtype, residual):
    out_dtype = out_dtype or dtype
    if out_dtype not in _DTYPES:
        raise RuntimeError("out_dtype must be bf16 or fp32")
    if out is None:
        out = torch.empty((T, features), dtype=out_dtype, device=dev)
    else:
        _check_out("out", out, (T, features), out_dtype, dev)
    if residual is not None:
        _check_cuda("residual", residual)
        if tuple(residual.shape) != (T, features) or residual.dtype != out_dtype or residual.device != dev:
            raise RuntimeError(f"residual must be {out_dtype} {(T, features)} on {dev}, as the output")
        if not residual.is_contiguous() or residual.data_ptr() % 16:
            residual = residual.clone(memory_format=torch.contiguous_format)
        desc.residual = residual.data_ptr()
    desc.T, desc.out, desc.out_dtype = T, out.data_ptr(), _DTYPES[out_dtype]
    return out, residual


def mxfp4_linear(x: Union[torch.Tensor, MXRows], w: MXBlockELL, residual: Optional[torch.Tensor] = None,
                 out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
                 max_ctas: int = 0) -> torch.Tensor:
    """``Q(x) Q(W)^T (+ residual)`` with fp32 sums, rounded once.

    ``x`` is ``[T, in_features]`` bf16 or fp32, or rows quantised before
    (``mxfp4_quantize``).  The output has ``out_dtype`` (default: x's, bf16 for
    quantised rows); ``residual`` has the output's shape and dtype.
    ``max_ctas`` caps the persistent grid (0 = every SM)."""
    return _linear(x, w, residual, out_dtype, out, max_ctas)[0]


def _linear(x, w, residual=None, out_dtype=None, out=None, max_ctas=0):
    if not isinstance(x, MXRows):
        x = _rows_2d("x", x)
    d = _lib.BellMxLinearDesc()
    T, dev, dtype, rows = _source(d, x, w.B, w.C * w.B)
    _same_device(dev, w)
    out, residual = _out_and_residual(d, T, w.R * w.B, dtype, dev, out, out_dtype, residual)
    d.w, d.max_ctas = w._abi, int(max_ctas)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().bell_linear_mx(C.byref(d), _stream()), "mxfp4_linear")
    return out, rows


def mxfp4_swiglu_fwd(x: Union[torch.Tensor, MXRows], gate: MXBlockELL, up: MXBlockELL, down: MXBlockELL,
                     add_residual: bool = False, residual: Optional[torch.Tensor] = None,
                     return_intermediates: bool = False, max_ctas: int = 0):
    """``Q(h) Q(Wd)^T (+ x)`` with ``h = silu(Q(x) Q(Wg)^T) * (Q(x) Q(Wu)^T)``.

    ``x`` is ``[T, d_model]`` bf16 or fp32 (the output's dtype too), or
    quantised rows (bf16 output; a ``residual`` must then be given for
    ``add_residual``).  ``return_intermediates`` returns ``(out, ws)``, ``ws``
    with the quantised rows ``q_x`` and ``q_h`` (``MXRows``) and the bf16
    projections ``gate`` and ``up``."""
    if not isinstance(x, MXRows):
        x = _rows_2d("x", x)
    if gate.R != up.R or gate.C != up.C or gate.B != up.B:
        raise RuntimeError("gate and up must have the same R, C and tile size")
    if down.B != gate.B or down.C != gate.R or down.R != gate.C:
        raise RuntimeError("down must map d_ff back to d_model at the tile size of gate and up")
    d = _lib.BellMxFFNDesc()
    B, F = gate.B, gate.R * gate.B
    T, dev, dtype, rows = _source(d, x, B, gate.C * B)
    _same_device(dev, gate, up, down)
    if add_residual and residual is None:
        if isinstance(x, MXRows):
            raise RuntimeError("add_residual on quantised rows needs the residual")
        residual = x
    out, residual = _out_and_residual(d, T, down.R * B, dtype, dev, None, None, residual if add_residual else None)
    h = torch.empty(_rows_bytes(T, F, B), dtype=torch.uint8, device=dev)
    d.h = h.data_ptr()
    g = u = None
    if return_intermediates:
        g, u = (torch.empty((T, F), dtype=torch.bfloat16, device=dev) for _ in range(2))
        d.gate_pre, d.up_out = g.data_ptr(), u.data_ptr()
    d.gate, d.up, d.down, d.max_ctas = gate._abi, up._abi, down._abi, int(max_ctas)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().bell_swiglu_fwd_mx(C.byref(d), _stream()), "mxfp4_swiglu_fwd")
    if return_intermediates:
        return out, dict(q_x=MXRows(rows, T, gate.C * B, B), q_h=MXRows(h, T, F, B), gate=g, up=u)
    return out


# ----------------------------------------------------------------- training


def _transposed(weights, cols, C_blocks: int):
    """bf16 tiles and columns of the transpose of the stacked quantised weights.
    The tiles come out [B_out, B_in], which the transpose reads as [B_in, B_out]."""
    cols_t, index = transposed_topology(cols, C_blocks)
    B = weights[0].B
    return _unpack(weights, index.reshape(-1), index.numel()).view(*index.shape, B, B), cols_t


def _like_master(grad: torch.Tensor, bf16: Optional[torch.Tensor], master: torch.Tensor) -> torch.Tensor:
    return bf16 if bf16 is not None else grad.to(master.dtype)


def _tile_grad(a, b, cols, B, layout, dtype):
    """Tile gradient in the master's dtype (the bf16 copy is written by the same launch)."""
    R, K = cols.shape
    half = torch.empty((R, K, B, B), dtype=torch.bfloat16, device=a.device) if dtype == torch.bfloat16 else None
    full = block_ell_sddmm(a, b, cols, B, layout, out_bf16=half)
    return full if half is None else half


class MXLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, values, cols, residual, layout):
        w = make_mxfp4(values, cols, x.shape[1] // values.shape[2], layout)
        x2 = _rows_2d("x", x)
        y, rows = _linear(x2, w, residual)
        ctx.w, ctx.rows, ctx.layout = w, MXRows(rows, x.shape[0], x.shape[1], w.B), layout
        ctx.save_for_backward(cols)
        ctx.dtypes = (x.dtype, values.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        w, (cols,) = ctx.w, ctx.saved_tensors
        x_dtype, v_dtype = ctx.dtypes
        dyb = dy.to(torch.bfloat16).contiguous()
        dx = dw = None
        if ctx.needs_input_grad[0]:
            vt, ct = _transposed((w,), [cols], w.C)
            dx = block_ell_linear(dyb, vt, ct, layout=TILE_IN_OUT).to(x_dtype)
        if ctx.needs_input_grad[1]:
            dw = _tile_grad(ctx.rows.dequantize(), dyb, w.col_indices, w.B, ctx.layout, v_dtype)
        return dx, dw, None, dy if ctx.needs_input_grad[3] else None, None


def mxfp4_linear_ad(x: torch.Tensor, values: torch.Tensor, cols: torch.Tensor, residual: Optional[torch.Tensor] = None,
                    layout: int = TILE_IN_OUT) -> torch.Tensor:
    """Differentiable ``Q(x) Q(W)^T (+ residual)`` from the weight's own tiles
    (``values [R, K, B, B]`` bf16 or fp32, quantised on every call).

    The backward passes the gradient straight through Q:
    ``dx = dy Q(W)``, ``dW = dy^T Q(x)`` on the live tiles (zero in dead slots),
    in bf16 products with fp32 sums."""
    if x.dim() != 2 or values.dim() != 4 or x.shape[1] % values.shape[2]:
        raise RuntimeError("x must be 2D [N, C*B] and values [R, K, B, B]")
    return MXLinearFn.apply(x, values, cols, residual, layout)


class MXSwiGLUFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, v_gate, ci_gate, v_up, ci_up, v_down, ci_down, add_residual, layout):
        B = v_gate.shape[2]
        C_model, R_ff = x.shape[1] // B, v_gate.shape[0]
        gate, up = make_mxfp4(v_gate, ci_gate, C_model, layout), make_mxfp4(v_up, ci_up, C_model, layout)
        down = make_mxfp4(v_down, ci_down, R_ff, layout)
        out, ws = mxfp4_swiglu_fwd(x, gate, up, down, add_residual=add_residual, return_intermediates=True)
        ctx.weights, ctx.q = (gate, up, down), (ws["q_x"], ws["q_h"])
        ctx.save_for_backward(ws["gate"], ws["up"], ci_gate, ci_up, ci_down)
        ctx.add_residual, ctx.layout = bool(add_residual), layout
        ctx.dtypes = (x.dtype, v_gate.dtype, v_up.dtype, v_down.dtype)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        g, u, ci_gate, ci_up, ci_down = ctx.saved_tensors
        (gate, up, down), (q_x, q_h), layout = ctx.weights, ctx.q, ctx.layout
        x_dtype, *v_dtypes = ctx.dtypes
        B, F = gate.B, gate.R * gate.B
        dy = grad_out.to(torch.bfloat16).contiguous()
        T = dy.shape[0]
        need = ctx.needs_input_grad
        dx = d_gate = d_up = d_down = dgu = None
        if need[0] or need[1] or need[3]:
            if T > 0:
                vt, ct = _transposed((down,), [ci_down], gate.R)
                # as the bf16 backward: one kernel for d_h and the SiLU backward at tile 64, two at 128
                if B == 64:
                    dgu = down_silu_bwd(dy, vt, ct, TILE_IN_OUT, g, u)
                else:
                    dgu = silu_mul_bwd(block_ell_linear(dy, vt, ct, layout=TILE_IN_OUT), g, u)
            else:
                dgu = torch.empty((0, 2 * F), dtype=torch.bfloat16, device=dy.device)
        if need[0]:
            vt, ct = _transposed((gate, up), [ci_gate, ci_up], gate.C)
            dx = block_ell_linear(dgu, vt, ct, residual=dy if ctx.add_residual else None, layout=TILE_IN_OUT).to(x_dtype)
        if need[1] or need[3]:
            xq = q_x.dequantize()
            if need[1]:
                d_gate = _tile_grad(xq, dgu[:, :F], gate.col_indices, B, layout, v_dtypes[0])
            if need[3]:
                d_up = _tile_grad(xq, dgu[:, F:], up.col_indices, B, layout, v_dtypes[1])
        if need[5]:
            d_down = _tile_grad(q_h.dequantize(), dy, down.col_indices, B, layout, v_dtypes[2])
        return dx, d_gate, None, d_up, None, d_down, None, None, None


def mxfp4_swiglu(x: torch.Tensor, v_gate: torch.Tensor, ci_gate: torch.Tensor, v_up: torch.Tensor, ci_up: torch.Tensor,
                 v_down: torch.Tensor, ci_down: torch.Tensor, add_residual: bool = False,
                 layout: int = TILE_IN_OUT) -> torch.Tensor:
    """Differentiable ``mxfp4_swiglu_fwd`` from the weights' own tiles (bf16 or
    fp32, quantised on every call), with the arguments of ``block_ell_swiglu``.

    The backward is that of the bf16 block at the quantised operands Q(x),
    Q(W), Q(h), the gradient passing straight through Q; tile gradients are
    summed in fp32 and come back in the tiles' dtype."""
    if x.dim() != 2 or v_gate.dim() != 4 or v_up.dim() != 4 or v_down.dim() != 4:
        raise RuntimeError("x must be 2D [N, d_model] and the tiles 4D [R, K, B, B]")
    if x.shape[1] % v_gate.shape[2]:
        raise RuntimeError(f"d_model={x.shape[1]} is not a multiple of the tile size {v_gate.shape[2]}")
    return MXSwiGLUFn.apply(x, v_gate, ci_gate, v_up, ci_up, v_down, ci_down, add_residual, layout)
