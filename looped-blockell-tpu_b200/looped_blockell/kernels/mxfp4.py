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
  quantised operands (their values are exact in bf16).  Tile
  gradients are fp32 sums of token ranges added in a fixed order, which
  depends on the sizes and the device's SMs: they are the same on every run.
  A weight's first backward builds its
  transposed topology and waits for the device once: before a step is captured
  in a graph, run one, and let no autograd graph of the same leaves live on.

Where ``ternary`` keeps 2 bits a weight and int8 activations, this keeps
4.25 bits of both, at tile sizes 64 and 128.  Stream-ordered on torch's
current stream; CUDA tensors only.
"""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from functools import cached_property, lru_cache
from typing import Optional, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .backward import topology_in_passes, transposed_topology
from .ops import TILE_IN_OUT, TILE_OUT_IN, _check_cuda, _check_out, _prep_ell, plan_bytes

_BF16, _F32 = _lib.BELL_DTYPE_BF16, _lib.BELL_DTYPE_F32
_DTYPES = {torch.bfloat16: _BF16, torch.float32: _F32}
_SLOTS = 254  # of a row of the backward's bf16 products
_ROWS = 128  # tokens of one chunk of quantised rows
_ELLS = {n: (_lib.BellEll * n, C.c_void_p * n) for n in (1, 2, 3)}  # array types of a pack of n weights


def _call(name: str, dev: torch.device, *args) -> None:
    """Library entry point `name` on the current stream of `dev`."""
    fn = getattr(_lib.load(), name)
    if torch.cuda.current_device() == dev.index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if rc:
        _lib.check(rc, name)


def _bytes(n: int, dev: torch.device) -> torch.Tensor:
    return torch.empty(n, dtype=torch.uint8, device=dev)


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


@dataclass(frozen=True)
class MXBlockELL:
    """A quantised Block-ELL weight (``make_mxfp4``).  One put together from
    fields (``dataclasses.replace``) is checked on its first use, which waits
    for the device: the kernels follow its plan into the rows and the tiles."""
    data: torch.Tensor         # uint8: the quantised tiles, operand layout, then the plan of the live slots
    col_indices: torch.Tensor  # int32 [R, K]
    R: int
    K: int
    C: int                     # input column blocks
    B: int

    @cached_property
    def _abi(self):  # the library's view of this weight
        data = self.data
        _check_cuda("quantised weight", data)
        _check_tile(self.B)
        if self.R < 1 or self.K < 1 or data.dtype != torch.uint8 or not data.is_contiguous() or \
                data.numel() < _tiles_bytes(self.R, self.K, self.B) + _plan_bytes(self.R, self.K):
            raise RuntimeError("MXBlockELL.data does not hold R x K quantised tiles and their plan")
        if "_made" not in self.__dict__:
            self._check_plan()
        return self._view(data.data_ptr())

    def _check_plan(self):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("use an MXBlockELL made from fields once before a capture")
        R, K = self.R, self.K
        plan = self.data[_tiles_bytes(R, K, self.B):_tiles_bytes(R, K, self.B) + _plan_bytes(R, K)].clone().view(torch.int32)
        e, counts = plan[:R * K].view(R, K), plan[-(-R * K // 4) * 4:][:R]
        slots = torch.arange(K, device=e.device)
        dead = e == -1
        ok = ((e & 0xFFFF) < self.C) & ((e >> 16) & 0xFFFF < K)
        ok = torch.where(dead, slots >= counts[:, None], ok & (slots < counts[:, None])).all() & (counts >= 0).all()
        if not (0 < self.C <= 65535 and bool(ok)):
            raise RuntimeError("MXBlockELL.data's plan does not fit R, K and C")

    def _view(self, at: int):
        return _lib.BellMxEll(at, at + _tiles_bytes(self.R, self.K, self.B), self.R, self.C, self.K, self.B)

    def __getstate__(self):  # a copy has other addresses
        return {k: v for k, v in self.__dict__.items() if k != "_abi"}

    @property
    def in_features(self) -> int:
        return self.C * self.B

    @property
    def out_features(self) -> int:
        return self.R * self.B

    def dequantize(self, layout: int = TILE_IN_OUT) -> torch.Tensor:
        """The quantised values as bf16 tiles ``[R, K, B, B]`` (dead slots too)."""
        n, dev = self.R * self.K, self.data.device
        v = torch.empty((self.R, self.K, self.B, self.B), dtype=torch.bfloat16, device=dev)
        _call("bell_mx_unpack_tiles", dev, self._abi.chunks, n, None, 0, self.B, None, n, v.data_ptr())
        return v if layout == TILE_OUT_IN else v.transpose(-1, -2).contiguous()


@lru_cache(maxsize=256)
def _plan_bytes(R: int, K: int) -> int:
    return plan_bytes(0, 0, 0, R, K)


def _tiles_bytes(R: int, K: int, B: int) -> int:
    return R * K * (B * B // 2 + 512)


def _rows_2d(name: str, x: torch.Tensor) -> torch.Tensor:
    """x as 2-D rows the kernels can read: unit stride along the features, rows
    16 bytes aligned (a copy where it is not)."""
    _check_cuda(name, x)
    if x.dim() != 2:
        raise RuntimeError(f"{name} must be 2D [N, features]")
    if x.dtype not in _DTYPES:
        raise RuntimeError(f"{name} must be bf16 or fp32")
    if x.is_contiguous() and x.data_ptr() % 16 == 0 and x.shape[1] % 8 == 0:
        return x
    per16 = 16 // x.element_size()
    T, f = x.shape
    ok = x.data_ptr() % 16 == 0 and x.stride(1) == 1 and \
        (x.stride(0) >= f and x.stride(0) % per16 == 0 or T < 2 and f % per16 == 0)
    return x if ok else x.clone(memory_format=torch.contiguous_format)


def _direct(T: int, tile: int) -> bool:
    """Whether a product of T rows quantises them itself, which saves a launch
    (about 5 us of the host's time, none in a graph).  On the device alone, graph
    replays of the gated block, on the way and quantised first: tile 64, d_model
    1024: 8.5 us and 9.1 at 1 token, 8.8 and 9.0 at 16, 9.6 and 9.1 at 24, 9.7
    and 8.9 at 32; tile 128, d_model 4096: 14.6 and 15.6 at 1, 15.6 and 15.6 at
    8, 17.1 and 15.6 at 9, 20.0 and 16.5 at 24.  Either way gives the same bits."""
    if tile != 64:
        return T <= 8
    return T <= 16 or T <= _lib.BELL_MX_DIRECT_ROWS and not torch.cuda.is_current_stream_capturing()


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
    dev = x.device
    data = _bytes(_rows_bytes(T, f, tile), dev)
    _call("bell_mx_quantize_rows", dev, T, f, tile, _DTYPES[x.dtype], x.data_ptr(), _ld(x), data.data_ptr())
    return MXRows(data, T, f, tile)


def mxfp4_dequantize(q: MXRows, dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values that ``q`` holds, ``[T, features]``; exact in bf16 and fp32."""
    _check_rows(q)
    if dtype not in _DTYPES:
        raise RuntimeError("dtype must be bf16 or fp32")
    dev = q.data.device
    if out is None:
        out = q.data.new_empty((q.T, q.features), dtype=dtype)
    else:
        _check_out("out", out, (q.T, q.features), dtype, dev)
    _call("bell_mx_dequantize_rows", dev, q.T, q.features, q.tile, q.data.data_ptr(), _DTYPES[dtype], out.data_ptr(),
          q.features)
    return out


def _check_rows(q: MXRows) -> None:
    data = q.data
    _check_cuda("quantised rows", data)
    _check_tile(q.tile)
    if q.T < 0 or q.features < 1 or q.features % q.tile or data.dtype != torch.uint8 or not data.is_contiguous() or \
            data.numel() < _rows_bytes(q.T, q.features, q.tile):
        raise RuntimeError("MXRows.data does not hold T x features quantised values")


def make_mxfp4(values: torch.Tensor, col_indices: torch.Tensor, C_blocks: int, layout: int = TILE_IN_OUT) -> MXBlockELL:
    """Quantise the tiles of a Block-ELL weight (``values [R, K, B, B]`` bf16 or
    fp32, B 64 or 128) and list its live slots.  A column index of -1 is a dead
    slot; one outside [0, C_blocks) is dropped and sets the status word."""
    return _pack(((values, col_indices, C_blocks),), layout)[0]


def _pack(weights, layout: int):
    """``make_mxfp4`` of several (values, col_indices, C_blocks), one launch for
    those of one dtype."""
    dtype = weights[0][0].dtype
    if any(v.dtype != dtype for v, _, _ in weights):
        return [_pack((w,), layout)[0] for w in weights]
    if dtype not in _DTYPES:
        raise RuntimeError("tiles must be bf16 or fp32")
    n, dev, out = len(weights), weights[0][0].device, []
    ells, pointers = _ELLS[n]
    abi, chunks, plans = ells(), pointers(), pointers()
    held = []  # copies that must outlive the launch's enqueueing
    for i, (values, col_indices, C_blocks) in enumerate(weights):
        v, cols = _prep_ell("weight", values, col_indices, dtype)
        R, K, B, B2 = v.shape
        _check_tile(B)
        if B2 != B or tuple(cols.shape) != (R, K):
            raise RuntimeError(f"values {tuple(v.shape)} and col_indices {tuple(cols.shape)} do not fit")
        if v.device != dev or cols.device != dev:
            raise RuntimeError("values and col_indices must be on one device")
        if v.data_ptr() % 16:
            v = v.clone()
        data = _bytes(_tiles_bytes(R, K, B) + _plan_bytes(R, K), dev)
        w = MXBlockELL(data, cols, R, K, int(C_blocks), B)
        w.__dict__["_made"] = True
        view = w.__dict__["_abi"] = w._view(data.data_ptr())
        abi[i] = _lib.BellEll(v.data_ptr(), cols.data_ptr(), R, w.C, K, B, layout, 0)
        chunks[i], plans[i] = view.chunks, view.plan
        held.append(v)
        out.append(w)
    _call("bell_mx_pack_ell", dev, abi, n, _DTYPES[dtype], chunks, plans, None)
    return out


def _check_weight(w: MXBlockELL, dev: torch.device) -> None:
    if w.data.device != dev:
        raise RuntimeError(f"weight is on {w.data.device}, x on {dev}")


def _source(x, tile: int, features: int):
    """The rows a product reads: (T, device, output dtype, address of rows to
    quantise or None, their stride and type), for x quantised already or not."""
    if isinstance(x, MXRows):
        _check_rows(x)
        if x.tile != tile or x.features != features:
            raise RuntimeError(f"quantised rows of {x.features} features, tile {x.tile}; the weight needs {features}, "
                               f"tile {tile}")
        return x.T, x.data.device, torch.bfloat16, None, 0, 0
    if x.shape[1] != features:
        raise RuntimeError(f"x has {x.shape[1]} features, the weight {features}")
    return x.shape[0], x.device, x.dtype, x.data_ptr(), _ld(x), _DTYPES[x.dtype]


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two 2-D tensors of rows share addresses (the ranges they span)."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _check_residual(residual, shape, dtype, dev) -> torch.Tensor:
    _check_cuda("residual", residual)
    if tuple(residual.shape) != shape or residual.dtype != dtype or residual.device != dev:
        raise RuntimeError(f"residual must be {dtype} {shape} on {dev}, as the output")
    if not residual.is_contiguous() or residual.data_ptr() % 16:
        residual = residual.clone(memory_format=torch.contiguous_format)
    return residual


def mxfp4_linear(x: Union[torch.Tensor, MXRows], w: MXBlockELL, residual: Optional[torch.Tensor] = None,
                 out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
                 max_ctas: int = 0) -> torch.Tensor:
    """``Q(x) Q(W)^T (+ residual)`` with fp32 sums, rounded once.

    ``x`` is ``[T, in_features]`` bf16 or fp32, or rows quantised before
    (``mxfp4_quantize``).  The output has ``out_dtype`` (default: x's, bf16 for
    quantised rows); ``residual`` has the output's shape and dtype.
    Where there are few units of many slots, parts of a row are summed first, so
    the order of its fp32 sum may depend on the number of tokens (and on the
    device's SMs); it is the same on every run.  ``out`` may be ``residual`` or
    ``x`` itself.  ``max_ctas`` caps the
    persistent grid (0 = every SM)."""
    return _linear(x, w, residual, out_dtype, out, max_ctas)[0]


def _linear(x, w, residual=None, out_dtype=None, out=None, max_ctas=0, keep_rows=False):
    if not isinstance(x, MXRows):
        x = _rows_2d("x", x)
    in_f, out_f = w.C * w.B, w.R * w.B
    T, dev, dtype, src, ld, src_type = _source(x, w.B, in_f)
    _check_weight(w, dev)
    dtype = out_dtype or dtype
    if dtype not in _DTYPES:
        raise RuntimeError("out_dtype must be bf16 or fp32")
    if residual is not None:
        residual = _check_residual(residual, (T, out_f), dtype, dev)
    if out is None:
        out = w.data.new_empty((T, out_f), dtype=dtype)
    else:
        _check_out("out", out, (T, out_f), dtype, dev)
        # one CTA writes its outputs while others still read x (direct) or
        # residual elements other than those they replace
        keep_rows = keep_rows or src is not None and _overlap(out, x)
        if residual is not None and residual.data_ptr() != out.data_ptr() and _overlap(out, residual):
            residual = residual.clone()
    if src is None:
        rows = x.data
    else:  # a few rows are quantised by the product itself
        rows = _bytes(_rows_bytes(T, in_f, w.B), dev) if keep_rows or not _direct(T, w.B) else None
    d = _lib.BellMxLinearDesc(T, _DTYPES[dtype], int(max_ctas), None if rows is None else rows.data_ptr(), src, ld, src_type, 0,
                              None if residual is None else residual.data_ptr(), out.data_ptr(), w._abi, None)
    _call("bell_linear_mx", dev, C.byref(d))
    return out, rows


def mxfp4_swiglu_fwd(x: Union[torch.Tensor, MXRows], gate: MXBlockELL, up: MXBlockELL, down: MXBlockELL,
                     add_residual: bool = False, residual: Optional[torch.Tensor] = None,
                     return_intermediates: bool = False, max_ctas: int = 0):
    """``Q(h) Q(Wd)^T (+ x)`` with ``h = silu(Q(x) Q(Wg)^T) * (Q(x) Q(Wu)^T)``.

    ``x`` is ``[T, d_model]`` bf16 or fp32 (the output's dtype too), or
    quantised rows (bf16 output; a ``residual`` must then be given for
    ``add_residual``).  ``residual`` stands for x there and needs
    ``add_residual``.  ``return_intermediates`` returns ``(out, ws)``, ``ws``
    with the quantised rows ``q_x`` and ``q_h`` (``MXRows``) and the bf16
    projections ``gate`` and ``up``."""
    if residual is not None and not add_residual:
        raise RuntimeError("a residual needs add_residual=True")
    out, ws = _swiglu(x, gate, up, down, add_residual, residual, return_intermediates, return_intermediates, max_ctas)
    return (out, ws) if return_intermediates else out


def _swiglu(x, gate, up, down, add_residual=False, residual=None, keep_rows=False, keep_projections=False, max_ctas=0):
    """The forward; with ``keep_rows`` also its quantised rows (and projections)."""
    quantised = isinstance(x, MXRows)
    if not quantised:
        x = _rows_2d("x", x)
    B, R, Cm = gate.B, gate.R, gate.C
    if R != up.R or Cm != up.C or B != up.B:
        raise RuntimeError("gate and up must have the same R, C and tile size")
    if down.B != B or down.C != R or down.R != Cm:
        raise RuntimeError("down must map d_ff back to d_model at the tile size of gate and up")
    D, F = Cm * B, R * B
    T, dev, dtype, src, ld, src_type = _source(x, B, D)
    for w in (gate, up, down):
        _check_weight(w, dev)
    if not add_residual:
        residual = None
    elif residual is not None:
        residual = _check_residual(residual, (T, D), dtype, dev)
    elif quantised:
        raise RuntimeError("add_residual on quantised rows needs the residual")
    else:  # x is [T, D] of the output's dtype, aligned
        residual = x.contiguous()
    out = gate.data.new_empty((T, D), dtype=dtype)
    direct = not quantised and not keep_rows and _direct(T, B)
    n_x, n_h = 0 if quantised or direct else _rows_bytes(T, D, B), _rows_bytes(T, F, B)
    ws = _bytes(n_x + n_h, dev)  # the quantised rows of x, then of h
    at = ws.data_ptr()
    g = u = None
    if keep_projections:
        g, u = (ws.new_empty((T, F), dtype=torch.bfloat16) for _ in range(2))
    d = _lib.BellMxFFNDesc(T, _DTYPES[dtype], int(max_ctas), x.data.data_ptr() if quantised else None if direct else at, src, ld, src_type, 0,
                           None if residual is None else residual.data_ptr(), at + n_x,
                           None if g is None else g.data_ptr(), None if u is None else u.data_ptr(), out.data_ptr(),
                           gate._abi, up._abi, down._abi, None)
    _call("bell_swiglu_fwd_mx", dev, C.byref(d))
    if not keep_rows:
        return out, None
    return out, dict(q_x=x if quantised else MXRows(ws[:n_x], T, D, B), q_h=MXRows(ws[n_x:], T, F, B), gate=g, up=u)


# ----------------------------------------------------------------- training


def _grad_rows(dy: torch.Tensor) -> torch.Tensor:
    """An incoming gradient as the backward reads it: contiguous bf16 rows,
    16-byte aligned (that of a slice may start anywhere)."""
    dy = dy.to(torch.bfloat16).contiguous()
    return dy if dy.data_ptr() % 16 == 0 else dy.clone()


def _grad(need: bool, cols: torch.Tensor, B: int, dtype: torch.dtype):
    """Buffer of a tile gradient (bf16 for bf16 tiles, else fp32), its address and type."""
    if not need:
        return None, None, _BF16
    kind = torch.bfloat16 if dtype == torch.bfloat16 else torch.float32
    g = cols.new_empty((*cols.shape, B, B), dtype=kind)
    return g, g.data_ptr(), _DTYPES[kind]


class MXLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, values, cols, residual, layout):
        w = make_mxfp4(values, cols, x.shape[1] // values.shape[2], layout)
        y, rows = _linear(x, w, residual, keep_rows=True)
        ctx.w, ctx.layout = w, layout
        ctx.save_for_backward(cols, rows)
        ctx.dtypes = (x.dtype, values.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w, (cols, rows) = ctx.w, ctx.saved_tensors
        x_dtype, v_dtype = ctx.dtypes
        dyb = _grad_rows(dy)
        T, dev = dyb.shape[0], dyb.device
        need = ctx.needs_input_grad
        dx = dx_at = cols_t = index_t = None
        K_t = 1
        if need[0]:
            cols_t, index_t = transposed_topology([cols], w.C)
            K_t = cols_t.shape[1]
            dx = dyb.new_empty((T, w.C * w.B), dtype=x_dtype)
            dx_at = dx.data_ptr()
        dw, dw_at, kind = _grad(need[1], w.col_indices, w.B, v_dtype)
        d = _lib.BellMxLinearBwdDesc(T, dyb.data_ptr(), rows.data_ptr(), w._abi, w.col_indices.data_ptr(),
                                     None if cols_t is None else cols_t.data_ptr(),
                                     None if index_t is None else index_t.data_ptr(), K_t, ctx.layout, dx_at, dw_at,
                                     kind, _DTYPES[x_dtype], None, None)
        ws = _bytes(_lib.load().bell_linear_bwd_mx_workspace_bytes(C.byref(d)), dev)
        d.workspace = ws.data_ptr()
        _call("bell_linear_bwd_mx", dev, C.byref(d))
        return dx, dw, None, dy if need[3] else None, None


def mxfp4_linear_ad(x: torch.Tensor, values: torch.Tensor, cols: torch.Tensor, residual: Optional[torch.Tensor] = None,
                    layout: int = TILE_IN_OUT) -> torch.Tensor:
    """Differentiable ``Q(x) Q(W)^T (+ residual)`` from the weight's own tiles
    (``values [R, K, B, B]`` bf16 or fp32, quantised on every call).

    The backward passes the gradient straight through Q:
    ``dx = dy Q(W)``, ``dW = dy^T Q(x)`` on the live tiles (zero in dead slots),
    in bf16 products with fp32 sums, in the dtypes of x and values.  The
    operands are bf16: an fp32 dy is rounded to it first.  A column block of W may be used by at most
    254 block-rows."""
    if x.dim() != 2 or values.dim() != 4 or x.shape[1] % values.shape[2]:
        raise RuntimeError("x must be 2D [N, C*B] and values [R, K, B, B]")
    return MXLinearFn.apply(x, values, cols, residual, layout)


class MXSwiGLUFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, v_gate, ci_gate, v_up, ci_up, v_down, ci_down, add_residual, layout):
        C_model, R_ff = x.shape[1] // v_gate.shape[2], v_gate.shape[0]
        gate, up, down = _pack(((v_gate, ci_gate, C_model), (v_up, ci_up, C_model), (v_down, ci_down, R_ff)), layout)
        out, ws = _swiglu(x, gate, up, down, add_residual, keep_rows=True)
        ctx.weights = (gate, up, down)
        ctx.save_for_backward(ws["q_x"].data, ws["q_h"].data, ci_gate, ci_up, ci_down)
        ctx.add_residual, ctx.layout = bool(add_residual), layout
        ctx.dtypes = (x.dtype, v_gate.dtype, v_up.dtype, v_down.dtype)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        q_x, q_h, ci_gate, ci_up, ci_down = ctx.saved_tensors
        gate, up, down = ctx.weights
        dy = _grad_rows(grad_out)
        T, dev = dy.shape[0], dy.device
        need = ctx.needs_input_grad
        # transposed topologies: of down for d_gate and d_up, of gate and up for dx (the address, the address, slots)
        td = tg = (None, None, 1)
        passes = 1
        if need[0] or need[1] or need[3]:
            td_cols, td_index = transposed_topology([ci_down], gate.R)
            td = td_cols.data_ptr(), td_index.data_ptr(), td_cols.shape[1]
        if need[0]:
            tg_cols, tg_index = transposed_topology([ci_gate, ci_up], gate.C)
            if tg_cols.shape[1] > _SLOTS:
                tg_cols, tg_index = topology_in_passes([ci_gate, ci_up], gate.C, _SLOTS)
                passes = tg_cols.shape[0]
            tg = tg_cols.data_ptr(), tg_index.data_ptr(), tg_cols.shape[-1]
        dx = torch.empty_like(dy, dtype=ctx.dtypes[0]) if need[0] else None
        # fp32 rows: the residual's gradient is added to theirs in fp32
        late = ctx.add_residual and ctx.dtypes[0] == torch.float32
        cols = (gate.col_indices, up.col_indices, down.col_indices)
        grads = [_grad(n, c, gate.B, t) for n, c, t in zip((need[1], need[3], need[5]), cols, ctx.dtypes[1:])]
        d = _lib.BellMxFFNBwdDesc(
            T, int(ctx.add_residual and not late), ctx.layout, dy.data_ptr(), q_x.data_ptr(),
            q_h.data_ptr(), gate._abi, up._abi, down._abi, cols[0].data_ptr(), cols[1].data_ptr(), cols[2].data_ptr(),
            *td[:2], *tg[:2], td[2], tg[2], None if dx is None else dx.data_ptr(), grads[0][1], grads[1][1], grads[2][1], grads[0][2],
            grads[1][2], grads[2][2], _DTYPES[ctx.dtypes[0]], passes, None, None)
        ws = _bytes(_lib.load().bell_swiglu_bwd_mx_workspace_bytes(C.byref(d)), dev)
        d.workspace = ws.data_ptr()
        _call("bell_swiglu_bwd_mx", dev, C.byref(d))
        if dx is not None and late:
            dx += grad_out
        return dx, grads[0][0], None, grads[1][0], None, grads[2][0], None, None, None


def mxfp4_swiglu(x: torch.Tensor, v_gate: torch.Tensor, ci_gate: torch.Tensor, v_up: torch.Tensor, ci_up: torch.Tensor,
                 v_down: torch.Tensor, ci_down: torch.Tensor, add_residual: bool = False,
                 layout: int = TILE_IN_OUT) -> torch.Tensor:
    """Differentiable ``mxfp4_swiglu_fwd`` from the weights' own tiles (bf16 or
    fp32, quantised on every call), with the arguments of ``block_ell_swiglu``.

    The backward is that of the bf16 block at the quantised operands Q(x),
    Q(W), Q(h), the gradient passing straight through Q; the projections are
    computed again rather than kept, so a step keeps 4.25 bits a value of x
    and h.  Gradients are summed in fp32 and come back in the dtypes of x and
    the tiles; the operands of the backward's products (dy, the gradients of
    the projections) are bf16, an fp32 dy and its own are rounded to it first.
    A column block may be used by at most 254 block-rows of down; of gate and
    up together by any number (dx then takes several passes)."""
    if x.dim() != 2 or v_gate.dim() != 4 or v_up.dim() != 4 or v_down.dim() != 4:
        raise RuntimeError("x must be 2D [N, d_model] and the tiles 4D [R, K, B, B]")
    if x.shape[1] % v_gate.shape[2]:
        raise RuntimeError(f"d_model={x.shape[1]} is not a multiple of the tile size {v_gate.shape[2]}")
    return MXSwiGLUFn.apply(x, v_gate, ci_gate, v_up, ci_up, v_down, ci_down, add_residual, layout)
