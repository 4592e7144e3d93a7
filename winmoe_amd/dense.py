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

import struct
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import ACTS, check, load

_TYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}

# wm_product_desc as a byte string: filling a ctypes structure field by field
# takes 3 us of a call whose kernel may take 5.
_DESC = struct.Struct("8i16q")


# Checks cost the host a few microseconds a call, so they are plain Python on
# what a tensor hands out at once.

# The current device's number (torch.cuda.current_device() initialises first,
# 0.2 us; whoever holds a device tensor has done that).
_current = torch._C._cuda_getDevice


def _dev(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA (HIP) tensor")
    if t.get_device() != _current():
        raise ValueError(f"{name} is on {t.device}, not on the current device cuda:{_current()}")


def _rows(t: torch.Tensor, rows: int, cols: int, dtype, name: str) -> int:
    """Distance of two rows of a [rows][cols] matrix whose rows are contiguous and do not overlap."""
    _dev(t, name)
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != (rows, cols):
        raise ValueError(f"{name} must be {[rows, cols]}, got {list(t.shape)}")
    return _distance(t, rows, cols, name)


def _distance(t: torch.Tensor, rows: int, cols: int, name: str) -> int:
    strides = t.stride()
    if (cols > 1 and strides[1] != 1) or (rows > 1 and strides[0] < cols):
        raise ValueError(f"{name} must have contiguous rows, got strides {strides}")
    return strides[0] if rows > 1 else max(cols, 1)         # a single row's stride means nothing


def _dense(t: torch.Tensor, shape, dtype, name: str) -> int:
    """Address of a contiguous tensor."""
    _dev(t, name)
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _new(like: torch.Tensor, shape, dtype, stream) -> torch.Tensor:
    """An output or workspace for work on `stream` (None: the current stream).

    Memory freed on the current stream may still be in use there, so what another
    stream writes comes from that stream's own; it is kept from reuse until the
    current stream, where the result may be read, is done with it."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(stream):
        t = like.new_empty(shape, dtype=dtype)
    t.record_stream(torch.cuda.current_stream())
    return t


def _raw(stream, t: torch.Tensor) -> int:
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(t.get_device())
    if stream.device_index != t.get_device():
        raise ValueError(f"the stream is on device {stream.device_index}, the tensors on {t.get_device()}")
    return stream.cuda_stream


def _dtype16(t: torch.Tensor, name: str):
    _dev(t, name)
    dt = t.dtype
    if dt is not torch.bfloat16 and dt is not torch.float16:
        raise ValueError(f"{name} must be float16 or bfloat16, got {dt}")
    return dt


def _act(act: str) -> int:
    if act not in ACTS:
        raise ValueError(f"act must be one of {sorted(ACTS)}, got {act!r}")
    return ACTS[act]


def _out_type(dtype, like, name: str):
    dtype = like if dtype is None else dtype
    if dtype is not like and dtype is not torch.float32:
        raise ValueError(f"{name} must be {like} or float32, got {dtype}")
    return dtype


def _operands(x, w, offsets, token):
    """(rows, in, out, E, x rows, offsets, token, x, ldx, w, ldw, w stride) of a product:
    w [E][out][in], or [out][in] when offsets is None."""
    _dev(x, "x")
    _dev(w, "w")
    dt = x.dtype
    if dt is not torch.bfloat16 and dt is not torch.float16:
        raise ValueError(f"x must be float16 or bfloat16, got {dt}")
    shape, strides = w.shape, w.stride()
    if offsets is None:
        if len(shape) != 2:
            raise ValueError("W must be [out][in]")
        E, (out, inn) = 1, shape
        off = 0
    else:
        if len(shape) != 3:
            raise ValueError("w must be [E][out][in]")
        E, out, inn = shape
        strides = strides[1:]
        off = _dense(offsets, (E + 1,), torch.int32, "offsets")
    if min(E, out, inn) < 1:
        raise ValueError(f"the weights are empty: {list(shape)}")
    if w.dtype is not dt:
        raise ValueError(f"w must be {dt}, got {w.dtype}")
    if (inn > 1 and strides[1] != 1) or (out > 1 and strides[0] < inn):
        raise ValueError(f"w must have contiguous rows, got strides {w.stride()}")
    ldw = strides[0] if out > 1 else inn
    stride = w.stride(0) if E > 1 else 0
    if E > 1 and stride < (out - 1) * ldw + inn:
        raise ValueError(f"the experts of w overlap: strides {w.stride()}")
    if x.dim() != 2 or x.shape[1] != inn:
        raise ValueError(f"x must be [rows][{inn}], got {list(x.shape)}")
    x_rows = x.shape[0]
    ldx = _distance(x, x_rows, inn, "x")
    rows, tok = x_rows, 0
    if token is not None:
        rows = token.numel()
        tok = _dense(token, (rows,), torch.int32, "token")
    return rows, inn, out, E, x_rows, off, tok, x.data_ptr(), ldx, w.data_ptr(), ldw, stride


def _workspace(L, desc, backward, like, stream):
    nb = L.wm_product_workspace_size(desc, backward)
    if nb < 0:
        check(_lib.WM_EINVAL, "wm_product_workspace_size")
    return _new(like, (nb,), torch.uint8, stream) if nb else None, nb


def _product(x, w, offsets, token, bias, act, residual, out, pre, out_dtype, stream):
    rows, inn, outs, E, x_rows, off, tok, xp, ldx, wp, ldw, stride = _operands(x, w, offsets, token)
    dt, a = x.dtype, _act(act)
    cols = outs
    if act == "swiglu":
        if outs % 2:
            raise ValueError("SwiGLU needs the gate rows and as many up rows in w")
        cols = outs // 2
    bp = rp = ldr = pp = ldp = 0
    if bias is not None:
        bp = _dense(bias, w.shape[:-1], dt, "bias")
    if residual is not None:
        rp, ldr = residual.data_ptr(), _rows(residual, rows, cols, dt, "residual")
    if out is None:
        yt = _out_type(out_dtype, dt, "out_dtype")
        out, ldy = _new(x, (rows, cols), yt, stream), cols
    else:
        yt = _out_type(out.dtype if out_dtype is None else out_dtype, dt, "out_dtype")
        ldy = _rows(out, rows, cols, yt, "out")
    if pre is not None:
        pp, ldp = pre.data_ptr(), _rows(pre, rows, outs, dt, "pre")
    desc = _DESC.pack(_TYPES[dt], rows, inn, outs, E, x_rows, a, _TYPES[yt], off, tok, xp, ldx, wp, ldw, stride, bp,
                      rp, ldr, out.data_ptr(), ldy, pp, ldp, 0, 0)
    L = load()
    ws, nb = _workspace(L, desc, 0, x, stream)
    check(L.wm_product(desc, ws.data_ptr() if nb else None, nb, _raw(stream, x)), "wm_product")
    return out


def _product_backward(dz, x, w, offsets, token, need_dx, need_dw, need_db, dw_dtype, dx, dw, db, stream):
    rows, inn, outs, E, x_rows, off, tok, xp, ldx, wp, ldw, stride = _operands(x, w, offsets, token)
    dt = x.dtype
    ldz = _rows(dz, rows, outs, dt, "dz")
    wt = _out_type(dw.dtype if dw is not None and dw_dtype is None else dw_dtype, dt, "dw_dtype")
    dxp = lddx = dwp = dbp = 0
    if need_dx or dx is not None:
        if dx is None:
            dx, lddx = _new(x, (rows, inn), dt, stream), inn
        else:
            lddx = _rows(dx, rows, inn, dt, "dx")
        dxp = dx.data_ptr()
    if need_dw or dw is not None:
        if dw is None:
            dw = _new(x, w.shape, wt, stream)
        dwp = _dense(dw, w.shape, wt, "dw")
    if need_db or db is not None:
        if db is None:
            db = _new(x, w.shape[:-1], torch.float32, stream)
        dbp = _dense(db, w.shape[:-1], torch.float32, "db")
    desc = _DESC.pack(_TYPES[dt], rows, inn, outs, E, x_rows, 0, _TYPES[dt], off, tok, xp, ldx, wp, ldw, stride,
                      0, 0, 0, 0, 0, 0, 0, dz.data_ptr(), ldz)
    L = load()
    ws, nb = _workspace(L, desc, 1, x, stream)
    check(L.wm_product_backward(desc, dxp, lddx, dwp, _TYPES[wt], dbp, ws.data_ptr() if nb else None, nb,
                                _raw(stream, x)), "wm_product_backward")
    return dx, dw, db


def linear(x: torch.Tensor, W: torch.Tensor, bias: Optional[torch.Tensor] = None, act: str = "none",
           residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
           pre: Optional[torch.Tensor] = None, out_dtype=None, stream=None) -> torch.Tensor:
    """act(x W^T + bias) + residual: x [T][in], W [out][in], bias [out], residual [T][columns].

    act is "none", "relu", "silu", "gelu" (exact), "sigmoid" or "swiglu":
    silu(gate) * up with the gate rows of W before the up rows, the result half
    as wide.  x, W,
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
    shape = ids.shape if isinstance(ids, torch.Tensor) else ()
    p = _dense(ids, shape, torch.int32, "ids")
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"ids must be [T][K], got {list(shape)}")
    if E < 1:
        raise ValueError("there must be an expert")
    T, K = shape
    offsets, token, row = _new(ids, (E + 1,), torch.int32, stream), _new(ids, (T * K,), torch.int32, stream), _new(ids, shape, torch.int32, stream)
    check(load().wm_group_by_expert(p, T, K, E, offsets.data_ptr(), token.data_ptr(), row.data_ptr(), _raw(stream, ids)),
          "wm_group_by_expert")
    return Grouping(offsets, token, row)


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
    dt, a = _dtype16(pre, "pre"), _act(act)
    if dy.dim() != 2 or dy.shape[1] < 1:
        raise ValueError(f"dy must be [rows][columns], got {list(dy.shape)}")
    T, n = dy.shape
    wide = 2 * n if act == "swiglu" else n
    ldy, ldp = _rows(dy, T, n, dt, "dy"), _rows(pre, T, wide, dt, "pre")
    if out is None:
        dz, ldz = _new(pre, (T, wide), dt, stream), wide
    else:
        dz, ldz = out, _rows(out, T, wide, dt, "out")
    check(load().wm_act_backward(_TYPES[dt], a, T, n, dy.data_ptr(), ldy, pre.data_ptr(), ldp, dz.data_ptr(), ldz,
                                 _raw(stream, pre)), "wm_act_backward")
    return dz


def _combine_args(y, row, w):
    """(type, T, K, H, distance of y's rows, row, w)."""
    dt, shape = _dtype16(y, "y"), y.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"y must be [rows][H], got {list(shape)}")
    rows, H = shape
    ldy = _distance(y, rows, H, "y")
    shape = row.shape if isinstance(row, torch.Tensor) else ()
    rp = _dense(row, shape, torch.int32, "row")
    if len(shape) != 2:
        raise ValueError(f"row must be [T][K], got {list(shape)}")
    wp = 0 if w is None else _dense(w, shape, torch.float32, "w")
    return dt, shape[0], shape[1], H, ldy, rp, wp


def combine(y: torch.Tensor, row: torch.Tensor, w: Optional[torch.Tensor] = None,
            residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, out_dtype=None,
            stream=None) -> torch.Tensor:
    """out[t] = sum_k w[t][k] * y[row[t][k]] + residual[t], k in order.

    y [rows][H] 16-bit, row int32 [T][K], w float32 [T][K] (None: ones),
    residual [T][H] of the result's type: y's or float32.  A row outside y
    (-1: padding) adds nothing, whatever its weight.  residual may be out."""
    dt, T, K, H, ldy, rp, wp = _combine_args(y, row, w)
    if out_dtype is None and (out is not None or residual is not None):
        out_dtype = (residual if out is None else out).dtype
    ot = _out_type(out_dtype, dt, "out_dtype")
    if out is None:
        o, ldo = _new(y, (T, H), ot, stream), H
    else:
        o, ldo = out, _rows(out, T, H, ot, "out")
    sp = ldr = 0
    if residual is not None:
        sp, ldr = residual.data_ptr(), _rows(residual, T, H, ot, "residual")
    check(load().wm_combine_rows(_TYPES[dt], y.data_ptr(), ldy, y.shape[0], rp, wp, T, K, H, sp, ldr, o.data_ptr(), ldo,
                                 _TYPES[ot], _raw(stream, y)), "wm_combine_rows")
    return o


def combine_backward(dout: torch.Tensor, y: torch.Tensor, row: torch.Tensor, w: Optional[torch.Tensor] = None,
                     need_dy: bool = True, need_dw: bool = True, dy: Optional[torch.Tensor] = None, stream=None):
    """(dy, dw) of ``combine`` given dout [T][H]: dy [rows][H] in y's type, dw float32 [T][K].

    Every row of y may be named by one pick only.  Rows that none names are
    left as they are in dy (unspecified in a new one); dw is 0 where the row
    is outside y.  The residual's gradient is dout itself."""
    dt, T, K, H, ldy, rp, wp = _combine_args(y, row, w)
    gt = _out_type(dout.dtype, dt, "dout's type")
    ldg = _rows(dout, T, H, gt, "dout")
    dyp = lddy = dwp = 0
    dw = None
    if need_dy or dy is not None:
        if dy is None:
            dy = _new(y, y.shape, dt, stream)
        dyp, lddy = dy.data_ptr(), _rows(dy, *y.shape, dt, "dy")
    if need_dw:
        dw = _new(y, (T, K), torch.float32, stream)
        dwp = dw.data_ptr()
    check(load().wm_combine_rows_backward(_TYPES[dt], dout.data_ptr(), ldg, _TYPES[gt], y.data_ptr(), ldy, y.shape[0],
                                          rp, wp, T, K, H, dyp, lddy, dwp, _raw(stream, y)),
          "wm_combine_rows_backward")
    return dy, dw


# ------------------------------------------------------------------ layer

class Gradients(NamedTuple):
    """What ``FloatMoELayer.backward`` returns; None for parts the layer does not have."""
    x: torch.Tensor                         # [T][H]
    w: torch.Tensor                         # routing weights, float32 [T][K]
    gate_up: torch.Tensor                   # [E][2 I][H]
    down: torch.Tensor                      # [E][H][I]
    shared_gate_up: Optional[torch.Tensor]  # [2 I_s][H]
    shared_down: Optional[torch.Tensor]     # [H][I_s]
    shared_gate: Optional[torch.Tensor]     # [1][H]


class FloatMoELayer:
    """A mixture-of-experts layer whose weights are fp16 or bf16, for any number of tokens.

    gate_up [E][2 I][H] holds each expert's gate rows, then its up rows; down
    is [E][H][I].  The optional shared expert has the same form without E, and
    an optional gate [1][H] (its output counts sigmoid(x . gate) times).  The
    mathematics is ``MoELayer``'s (winmoe_inference.c:1684-2027), which takes
    the quantised formats; here every product runs on 16-bit values with fp32
    sums, and the layer can be trained: ``forward(..., keep=True)`` hands out
    what ``backward`` needs."""

    def __init__(self, gate_up: torch.Tensor, down: torch.Tensor, K: int, router: Optional[torch.Tensor] = None,
                 shared_gate_up: Optional[torch.Tensor] = None, shared_down: Optional[torch.Tensor] = None,
                 shared_gate: Optional[torch.Tensor] = None):
        dt = _dtype16(gate_up, "gate_up")
        if gate_up.dim() != 3 or gate_up.shape[1] % 2:
            raise ValueError(f"gate_up must be [E][2 I][H], got {list(gate_up.shape)}")
        self.E, self.I, self.H, self.K, self.dtype = gate_up.shape[0], gate_up.shape[1] // 2, gate_up.shape[2], K, dt
        if not 1 <= K <= self.E:
            raise ValueError(f"K must lie in [1, {self.E}], got {K}")
        _dense(gate_up, gate_up.shape, dt, "gate_up")
        _dense(down, (self.E, self.H, self.I), dt, "down")
        if router is not None:
            _dense(router, (self.E, self.H), torch.float32, "router")
        if (shared_gate_up is None) != (shared_down is None) or (shared_gate is not None and shared_down is None):
            raise ValueError("a shared expert needs shared_gate_up and shared_down")
        if shared_down is not None:
            _dense(shared_down, (self.H, shared_down.shape[-1]), dt, "shared_down")
            _dense(shared_gate_up, (2 * shared_down.shape[1], self.H), dt, "shared_gate_up")
        if shared_gate is not None:
            _dense(shared_gate, (1, self.H), dt, "shared_gate")
        self.gate_up, self.down, self.router = gate_up, down, router
        self.shared_gate_up, self.shared_down, self.shared_gate = shared_gate_up, shared_down, shared_gate

    def route(self, x: torch.Tensor):
        """(ids int32 [T][K], weights float32 [T][K]) by the layer's router, one token after another (``router_topk``)."""
        from .moe import router_topk
        if self.router is None:
            raise ValueError("the layer has no router")
        _rows(x, x.shape[0], self.H, self.dtype, "x")
        ids = x.new_empty((x.shape[0], self.K), dtype=torch.int32)
        w = x.new_empty((x.shape[0], self.K), dtype=torch.float32)
        for t, h in enumerate(x.float()):
            ids[t], w[t] = router_topk(h, self.router, self.K)
        return ids, w

    def forward(self, x: torch.Tensor, ids: torch.Tensor, w: torch.Tensor, residual: Optional[torch.Tensor] = None,
                keep: bool = False):
        """The layer's output [T][H] for x [T][H], picks ids int32 [T][K] and weights w float32 [T][K].

        A pick outside [0, E) counts as nothing.  residual [T][H] (x's type or
        float32) is added, and the result is of its type, else of x's.  With
        keep, returns (output, what ``backward`` takes)."""
        T, K = x.shape[0], self.K
        _rows(x, T, self.H, self.dtype, "x")
        _dense(ids, (T, K), torch.int32, "ids")
        _dense(w, (T, K), torch.float32, "w")
        R = T * K
        g = group_by_expert(ids, self.E)
        shared = self.shared_down is not None
        pre = x.new_empty((R, 2 * self.I)) if keep else None
        h = grouped_matmul(x, self.gate_up, g.offsets, token=g.token, act="swiglu", pre=pre)
        # the shared expert's rows stand behind the routed ones: one more pick of every token
        y = x.new_empty((R + T if shared else R, self.H))
        grouped_matmul(h, self.down, g.offsets, out=y[:R])
        row, weight, pre_s, hs = g.row, w, None, None
        if shared:
            pre_s = x.new_empty((T, self.shared_gate_up.shape[0])) if keep else None
            hs = linear(x, self.shared_gate_up, act="swiglu", pre=pre_s)
            linear(hs, self.shared_down, out=y[R:])
            s = (linear(x, self.shared_gate, act="sigmoid", out_dtype=torch.float32) if self.shared_gate is not None
                 else w.new_ones((T, 1)))
            last = torch.arange(R, R + T, dtype=torch.int32, device=x.device).view(T, 1)
            row, weight = torch.cat([g.row, last], 1), torch.cat([w, s], 1)
        out = combine(y, row, weight, residual=residual)
        return (out, (x, g, pre, h, y, row, weight, pre_s, hs)) if keep else out

    def backward(self, dout: torch.Tensor, kept, dw_dtype=None) -> Gradients:
        """Gradients given dout [T][H] (x's type or float32) and what ``forward(..., keep=True)`` handed out.

        The matrices' gradients are of the layer's type or float32 (dw_dtype);
        the residual's gradient is dout itself."""
        x, g, pre, h, y, row, weight, pre_s, hs = kept
        T, K, R = x.shape[0], self.K, x.shape[0] * self.K
        dy, dweight = combine_backward(dout, y, row, weight)
        dh, ddown, _ = grouped_matmul_backward(dy[:R], h, self.down, g.offsets, dw_dtype=dw_dtype)
        dz = act_backward(dh, pre, "swiglu")
        # one buffer for the parts of dx, which are summed and rounded once
        extra = 0 if hs is None else 1 if self.shared_gate is None else 2       # rows per token that the shared expert adds
        parts = x.new_empty((R + extra * T, self.H))
        _, dgu, _ = grouped_matmul_backward(dz, x, self.gate_up, g.offsets, token=g.token, dw_dtype=dw_dtype, dx=parts[:R])
        dsgu = dsd = dsg = None
        rows = [g.row]
        if hs is not None:
            dhs, dsd, _ = linear_backward(dy[R:], hs, self.shared_down, dw_dtype=dw_dtype)
            dzs = act_backward(dhs, pre_s, "swiglu")
            _, dsgu, _ = linear_backward(dzs, x, self.shared_gate_up, dw_dtype=dw_dtype, dx=parts[R:R + T])
            if self.shared_gate is not None:
                s = weight[:, K:]
                ds = (dweight[:, K:] * s * (1.0 - s)).to(self.dtype)
                _, dsg, _ = linear_backward(ds, x, self.shared_gate, dw_dtype=dw_dtype, dx=parts[R + T:])
            rows.append(torch.arange(R, parts.shape[0], dtype=torch.int32, device=x.device).view(extra, T).T)
        dx = combine(parts, torch.cat(rows, 1) if len(rows) > 1 else g.row)
        return Gradients(dx, dweight[:, :K], dgu, ddown, dsgu, dsd, dsg)
