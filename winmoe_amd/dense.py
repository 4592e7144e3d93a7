"""PyTorch-ROCm host API of the operators on 16-bit weights (fp16 or bf16).

The products of an expert layer that is not quantised -- a GGUF file's F16 and
BF16 tensors, or a layer in training -- for any number of rows, with their
gradients:

* ``linear`` / ``linear_backward``                  y = act(x W^T + bias) + residual
* ``grouped_matmul`` / ``grouped_matmul_backward``  the same per expert over ragged groups of rows
* ``act_backward``                                  the activation's gradient, between the two
* ``group_by_expert``                               (token, pick) pairs sorted by expert
* ``combine`` / ``combine_backward``                the weighted sum over a token's picks

``FloatMoELayer`` runs them together as a mixture-of-experts block, forward and
backward.  The gradients are functions of their own; nothing is recorded for
autograd.  Each is one call of libwinmoe_hip.so (wm_product and the entry
points after it in include/winmoe_hip.h); torch is used for device memory and
streams.  Matrices are row-major with contiguous rows; the distance of rows may
be larger than their length (a column range of a wider tensor).  Tensors must
live on the current HIP device.  Every output is rounded once from fp32.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import ACTS, ProductDesc, check, load
from .moe import _p, _stream

_TYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


def _dev(t: torch.Tensor, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA (HIP) tensor")
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f"{name} is on {t.device}, not on the current device cuda:{torch.cuda.current_device()}")
    return t


def _rows(t: torch.Tensor, shape, dtype, name: str) -> torch.Tensor:
    """A matrix of the given shape and type whose rows are contiguous and do not overlap."""
    _dev(t, name)
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != 2 or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if (shape[1] > 1 and t.stride(1) != 1) or (shape[0] > 1 and t.stride(0) < shape[1]):
        raise ValueError(f"{name} must have contiguous rows, got strides {t.stride()}")
    return t


def _dense(t: torch.Tensor, shape, dtype, name: str) -> torch.Tensor:
    _dev(t, name)
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _ld(t: torch.Tensor) -> int:
    """Distance of two rows in elements (a single row's stride means nothing)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _new(shape, dtype, device, stream) -> torch.Tensor:
    """An output or workspace for work on `stream` (None: the current stream)."""
    t = torch.empty(shape, dtype=dtype, device=device)
    if stream is not None and stream != torch.cuda.current_stream():
        t.record_stream(stream)
    return t


def _dtype16(t: torch.Tensor, name: str):
    _dev(t, name)
    if t.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"{name} must be float16 or bfloat16, got {t.dtype}")
    return t.dtype


def _act(act: str) -> int:
    if act not in ACTS:
        raise ValueError(f"act must be one of {sorted(ACTS)}, got {act!r}")
    return ACTS[act]


def _out_type(dtype, like, name: str):
    dtype = like if dtype is None else dtype
    if dtype not in (like, torch.float32):
        raise ValueError(f"{name} must be {like} or float32, got {dtype}")
    return dtype


def _desc(x, w, offsets, token) -> ProductDesc:
    """The operands of a product: w [E][out][in], or [out][in] when offsets is None."""
    dt = _dtype16(x, "x")
    grouped = offsets is not None
    if w.dim() != (3 if grouped else 2):
        raise ValueError("w must be [E][out][in]" if grouped else "W must be [out][in]")
    E, out, inn = w.shape if grouped else (1, *w.shape)
    if min(E, out, inn) < 1:
        raise ValueError(f"the weights are empty: {list(w.shape)}")
    if x.dim() != 2:
        raise ValueError(f"x must be [rows][{inn}], got {list(x.shape)}")
    _rows(x, (x.shape[0], inn), dt, "x")
    _dev(w, "w")
    m = w[0] if grouped else w
    _rows(m, (out, inn), dt, "w")
    d = ProductDesc()
    d.dtype, d.inn, d.out, d.n_groups, d.x_rows = _TYPES[dt], inn, out, E, x.shape[0]
    d.x, d.ldx, d.w, d.ldw = _p(x), _ld(x), _p(w), _ld(m)
    d.w_stride = w.stride(0) if grouped and E > 1 else out * d.ldw
    if grouped:
        d.offsets = _p(_dense(offsets, (E + 1,), torch.int32, "offsets"))
    if token is not None:
        d.token = _p(_dense(token, (token.numel(),), torch.int32, "token"))
    d.rows = x.shape[0] if token is None else token.numel()
    return d


def _product(x, w, offsets, token, bias, act, residual, out, pre, out_dtype, stream):
    d = _desc(x, w, offsets, token)
    d.act = _act(act)
    if act == "swiglu" and d.out % 2:
        raise ValueError("SwiGLU needs the gate rows and as many up rows in w")
    cols = d.out // 2 if act == "swiglu" else d.out
    if bias is not None:
        d.bias = _p(_dense(bias, w.shape[:-1], x.dtype, "bias"))
    if residual is not None:
        d.residual, d.ld_residual = _p(_rows(residual, (d.rows, cols), x.dtype, "residual")), _ld(residual)
    if out is not None and out_dtype is None:
        out_dtype = out.dtype
    yt = _out_type(out_dtype, x.dtype, "out_dtype")
    y = _new((d.rows, cols), yt, x.device, stream) if out is None else _rows(out, (d.rows, cols), yt, "out")
    d.y, d.ldy, d.y_type = _p(y), _ld(y), _TYPES[yt]
    if pre is not None:
        d.pre, d.ld_pre = _p(_rows(pre, (d.rows, d.out), x.dtype, "pre")), _ld(pre)
    L = load()
    ws, nb = _workspace(L, d, 0, x.device, stream)
    check(L.wm_product(C.byref(d), _p(ws), nb, _stream(stream)), "wm_product")
    return y


def _workspace(L, d, backward, device, stream):
    nb = L.wm_product_workspace_size(C.byref(d), backward)
    if nb < 0:
        check(_lib.WM_EINVAL, "wm_product_workspace_size")
    return (_new((nb,), torch.uint8, device, stream), nb) if nb else (None, 0)


def _product_backward(dz, x, w, offsets, token, need_dx, need_dw, need_db, dw_dtype, dx, dw, db, stream):
    d = _desc(x, w, offsets, token)
    _rows(dz, (d.rows, d.out), x.dtype, "dz")
    if dw is not None and dw_dtype is None:
        dw_dtype = dw.dtype
    wt = _out_type(dw_dtype, x.dtype, "dw_dtype")
    if need_dx or dx is not None:
        shape = (d.rows, d.inn)
        dx = _new(shape, x.dtype, x.device, stream) if dx is None else _rows(dx, shape, x.dtype, "dx")
    if need_dw or dw is not None:
        dw = _new(w.shape, wt, x.device, stream) if dw is None else _dense(dw, w.shape, wt, "dw")
    if need_db or db is not None:
        shape = w.shape[:-1]
        db = (_new(shape, torch.float32, x.device, stream) if db is None
              else _dense(db, shape, torch.float32, "db"))
    L = load()
    ws, nb = _workspace(L, d, 1, x.device, stream)
    check(L.wm_product_backward(C.byref(d), _p(dz), _ld(dz), _p(dx), _ld(dx) if dx is not None else 0, _p(dw),
                                _TYPES[wt], _p(db), _p(ws), nb, _stream(stream)), "wm_product_backward")
    return dx, dw, db


def linear(x: torch.Tensor, W: torch.Tensor, bias: Optional[torch.Tensor] = None, act: str = "none",
           residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
           pre: Optional[torch.Tensor] = None, out_dtype=None, stream=None) -> torch.Tensor:
    """act(x W^T + bias) + residual: x [T][in], W [out][in], bias [out], residual [T][columns].

    act is "none", "relu", "silu", "gelu" (exact) or "swiglu": silu(gate) * up
    with the gate rows of W before the up rows, the result half as wide.  x, W,
    bias and residual are of one 16-bit type; the result is of that type or
    float32 (out_dtype, or out's).  pre [T][out] receives x W^T + bias for the
    way back.  residual may be out itself; no other output may overlap an input."""
    return _product(x, W, None, None, bias, act, residual, out, pre, out_dtype, stream)


def linear_backward(dz: torch.Tensor, x: torch.Tensor, W: torch.Tensor, need_dx: bool = True, need_dw: bool = True,
                    need_db: bool = False, dw_dtype=None, dx: Optional[torch.Tensor] = None,
                    dw: Optional[torch.Tensor] = None, db: Optional[torch.Tensor] = None, stream=None):
    """(dx, dw, db) of z = x W^T + bias given dz [T][out]: dx [T][in] in x's type, dw [out][in] in
    x's type or float32 (dw_dtype), db [out] float32; None where not asked for.  dx, dw and db may be
    given to be written to."""
    return _product_backward(dz, x, W, None, None, need_dx, need_dw, need_db, dw_dtype, dx, dw, db, stream)


class Grouping(NamedTuple):
    """The pairs of a batch sorted by expert (``group_by_expert``)."""
    offsets: torch.Tensor   # int32 [E + 1]: rows offsets[e] .. offsets[e + 1] - 1 belong to expert e
    token: torch.Tensor     # int32 [T * K]: the token of each sorted row, -1 from offsets[E] on
    row: torch.Tensor       # int32 [T][K]: the sorted row of each pick, -1 for a pick of no expert


def group_by_expert(ids: torch.Tensor, E: int, stream=None) -> Grouping:
    """Sorts the picks ids int32 [T][K] by expert, stably.  A pick outside [0, E) (padding) belongs to none."""
    _dev(ids, "ids")
    if ids.dim() != 2 or ids.shape[1] < 1:
        raise ValueError(f"ids must be [T][K], got {list(ids.shape)}")
    _dense(ids, ids.shape, torch.int32, "ids")
    if E < 1:
        raise ValueError("there must be an expert")
    T, K = ids.shape
    g = Grouping(*(_new(s, torch.int32, ids.device, stream) for s in ((E + 1,), (T * K,), (T, K))))
    check(load().wm_group_by_expert(_p(ids), T, K, E, _p(g.offsets), _p(g.token), _p(g.row), _stream(stream)),
          "wm_group_by_expert")
    return g


def grouped_matmul(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, token: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, act: str = "none", out: Optional[torch.Tensor] = None,
                   pre: Optional[torch.Tensor] = None, out_dtype=None, stream=None) -> torch.Tensor:
    """Row r of group e is act(w[e] x[token[r]] + bias[e]): w [E][out][in], bias [E][out], offsets int32 [E + 1].

    Without token, row r takes row r of x.  A token outside x counts as zeros.
    Activations, types and pre are as for ``linear``.  Rows of no group are
    left as they are: what they hold in a new result is unspecified."""
    return _product(x, w, offsets, token, bias, act, None, out, pre, out_dtype, stream)


def grouped_matmul_backward(dz: torch.Tensor, x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor,
                            token: Optional[torch.Tensor] = None, need_dx: bool = True, need_dw: bool = True,
                            need_db: bool = False, dw_dtype=None, dx: Optional[torch.Tensor] = None,
                            dw: Optional[torch.Tensor] = None, db: Optional[torch.Tensor] = None, stream=None):
    """(dx, dw, db) of ``grouped_matmul`` without its activation, given dz [rows][out].

    dx [rows][in] has one row per row of dz: with token, ``combine(dx, row)``
    sums them per row of x.  dw [E][out][in] and db [E][out] of an empty group
    are zeros; types are as for ``linear_backward``.  Rows of no group are not
    read, and left as they are in dx."""
    return _product_backward(dz, x, w, offsets, token, need_dx, need_dw, need_db, dw_dtype, dx, dw, db, stream)


def act_backward(dy: torch.Tensor, pre: torch.Tensor, act: str, out: Optional[torch.Tensor] = None,
                 stream=None) -> torch.Tensor:
    """dz = act'(pre) * dy.  dy [T][n]; pre and the result [T][n], or [T][2 n] for "swiglu".  out may be pre."""
    dt = _dtype16(pre, "pre")
    if dy.dim() != 2 or dy.shape[1] < 1:
        raise ValueError(f"dy must be [rows][columns], got {list(dy.shape)}")
    T, n = dy.shape
    wide = (T, 2 * n if _act(act) == ACTS["swiglu"] else n)
    _rows(dy, (T, n), dt, "dy")
    _rows(pre, wide, dt, "pre")
    dz = _new(wide, dt, pre.device, stream) if out is None else _rows(out, wide, dt, "out")
    check(load().wm_act_backward(_TYPES[dt], ACTS[act], T, n, _p(dy), _ld(dy), _p(pre), _ld(pre), _p(dz), _ld(dz),
                                 _stream(stream)), "wm_act_backward")
    return dz


def _combine_args(y, row, w):
    dt = _dtype16(y, "y")
    if y.dim() != 2 or y.shape[1] < 1:
        raise ValueError(f"y must be [rows][H], got {list(y.shape)}")
    _rows(y, y.shape, dt, "y")
    _dev(row, "row")
    if row.dim() != 2:
        raise ValueError(f"row must be [T][K], got {list(row.shape)}")
    _dense(row, row.shape, torch.int32, "row")
    if w is not None:
        _dense(w, row.shape, torch.float32, "w")
    return dt, row.shape[0], row.shape[1], y.shape[1]


def combine(y: torch.Tensor, row: torch.Tensor, w: Optional[torch.Tensor] = None,
            residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, out_dtype=None,
            stream=None) -> torch.Tensor:
    """out[t] = sum_k w[t][k] * y[row[t][k]] + residual[t], k in order.

    y [rows][H] 16-bit, row int32 [T][K], w float32 [T][K] (None: ones),
    residual [T][H] of the result's type: y's or float32.  A row outside y
    (-1: padding) adds nothing, whatever its weight.  residual may be out."""
    dt, T, K, H = _combine_args(y, row, w)
    if out is not None and out_dtype is None:
        out_dtype = out.dtype
    if out is None and out_dtype is None and residual is not None:
        out_dtype = residual.dtype
    ot = _out_type(out_dtype, dt, "out_dtype")
    o = _new((T, H), ot, y.device, stream) if out is None else _rows(out, (T, H), ot, "out")
    if residual is not None:
        _rows(residual, (T, H), ot, "residual")
    check(load().wm_combine_rows(_TYPES[dt], _p(y), _ld(y), y.shape[0], _p(row), _p(w), T, K, H, _p(residual),
                                 _ld(residual) if residual is not None else 0, _p(o), _ld(o), _TYPES[ot],
                                 _stream(stream)), "wm_combine_rows")
    return o


def combine_backward(dout: torch.Tensor, y: torch.Tensor, row: torch.Tensor, w: Optional[torch.Tensor] = None,
                     need_dy: bool = True, need_dw: bool = True, dy: Optional[torch.Tensor] = None, stream=None):
    """(dy, dw) of ``combine`` given dout [T][H]: dy [rows][H] in y's type, dw float32 [T][K].

    Every row of y may be named by one pick only.  Rows that none names are
    left as they are in dy (unspecified in a new one); dw is 0 where the row
    is outside y.  The residual's gradient is dout itself."""
    dt, T, K, H = _combine_args(y, row, w)
    gt = _out_type(dout.dtype, dt, "dout's type")
    _rows(dout, (T, H), gt, "dout")
    if need_dy or dy is not None:
        dy = _new(y.shape, dt, y.device, stream) if dy is None else _rows(dy, y.shape, dt, "dy")
    dw = _new((T, K), torch.float32, y.device, stream) if need_dw else None
    check(load().wm_combine_rows_backward(_TYPES[dt], _p(dout), _ld(dout), _TYPES[gt], _p(y), _ld(y), y.shape[0],
                                          _p(row), _p(w), T, K, H, _p(dy), _ld(dy) if dy is not None else 0, _p(dw),
                                          _stream(stream)), "wm_combine_rows_backward")
    return dy, dw
