"""The feed-forward half of a block on plain row-major matrices, forward and backward: :func:`layer_norm` with its tables, :func:`linear` with bias,
activation, gate and residual in its epilogue, and :func:`feed_forward`, two products with an activation (and, gated, a product of two projections)
between them.  Tensor-level front end of ``include/pkh3_rows.h``; as in :mod:`.ops`, PyTorch is memory and streams only.

The layers are the reference's ``ff.net.0.proj`` and ``ff.net.2`` (src/pika_h3/core/loader.py:9); the norm in front of them is modulated by tables of a few
rows (patches/0001-h3-adaln-fp32.patch:34-40).

Rows are ``[rows, width]`` with unit column stride, other strides and widths multiples of 8 elements, 16-byte aligned.  Where gradients are recorded and an
input needs them, the three calls take part in torch's differentiation (backwards; not while a stream is captured; ``out``, ``save`` and ``gate`` are refused
then); the ``*_backward`` functions are the same passes by themselves, which a graph may hold.

What lies between two products is rounded to bfloat16: h of a block, dz of its backward pass, and a norm's result in front of a product.  They are operands of bfloat16 MFMAs;
with float32's bits each would be two operands and the product behind it twice the work (three times, where both of its operands are split).  That rounding makes a result's relative
error 0.0021 to 0.0024 where its own rounding alone makes 0.0017.  Gradients of weights and biases come in one type, bfloat16, whatever a bias's own: their sums are float32 until then.
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _lib
from .ops import _raw_stream

ACTIVATIONS = {"none": _lib.ACT_NONE, "silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU, "gelu_tanh": _lib.ACT_GELU_TANH}

_BF16, _F32 = torch.bfloat16, torch.float32
_pack_product = _lib.PRODUCT_ARGS_FORMAT.pack
_pack_norm = _lib.NORM_ARGS_FORMAT.pack


@lru_cache(maxsize=None)
def _entry(name: str):
    """A C entry that takes the packed bytes of its arguments."""
    call = _lib.load()[name]
    call.argtypes = [C.c_char_p, C.c_void_p]
    call.restype = C.c_int
    return call


def _call(name: str, args: bytes, index: int) -> None:
    if index == torch.cuda.current_device():
        rc = _entry(name)(args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = _entry(name)(args, _raw_stream(index))
    if rc:
        _lib.check(rc)


def _place(x: torch.Tensor) -> int:
    """The device of a call, that of its rows."""
    index = x.get_device()
    if index < 0:
        raise ValueError(f"x must live in device memory (got {x.device}); the HIP library is the only compute path")
    return index


def _matrix(name: str, t: torch.Tensor, rows: int, cols: int, index: int, dtype=_BF16) -> Tuple[int, int]:
    """Raises unless ``t`` is a ``[rows, cols]`` matrix (-1: any) that the kernels can read or write; its address and row stride."""
    shape = t.shape
    if len(shape) != 2 or (rows >= 0 and shape[0] != rows) or (cols >= 0 and shape[1] != cols):
        raise ValueError(f"{name} must be [{rows if rows >= 0 else 'rows'}, {cols if cols >= 0 else 'columns'}], got {tuple(shape)}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    row, column = t.stride()
    if column != 1 and shape[1] > 1:
        raise ValueError(f"{name}: column stride must be 1, got {column}")
    if t.get_device() != index:
        raise ValueError(f"{name} must live in device memory, with x (got {t.device})")
    return t.data_ptr(), (row if shape[0] > 1 else shape[1])


def _vector(name: str, t: torch.Tensor, n: int, index: int) -> Tuple[int, bool]:
    """Address of a bias and whether it is bfloat16."""
    if t.dtype not in (_BF16, _F32) or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous float32 or bfloat16 [{n}], got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != index:
        raise ValueError(f"{name} must live in device memory, with x (got {t.device})")
    return t.data_ptr(), t.dtype is _BF16


def _index(name: str, t: torch.Tensor, rows: int, index: int) -> int:
    if t.dtype is not torch.int32 or t.shape != (rows,) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 [{rows}], got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != index:
        raise ValueError(f"{name} must live in device memory, with x (got {t.device})")
    return t.data_ptr()


def _activation(name: str) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {name!r}")
    return ACTIVATIONS[name]


def _refuse_tangents(*tensors) -> None:
    """The passes carry no tangents of forward-mode differentiation (inside a dual level a tensor may have one): raises where one would be lost."""
    if _forward_ad._current_level >= 0 and any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("forward-mode tangents are not carried through these calls")


def _wants_grad(x, *tensors) -> bool:
    """Whether a call is recorded for torch's differentiation.  Not while a stream is captured: the nodes that add up the leaves' gradients may live already, with the
    stream of an eager pass, and running them on it inside a capture ends the process."""
    _refuse_tangents(x, *tensors)
    if not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in (x, *tensors)):
        return False
    if x.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("gradients are not recorded while a stream is captured: call the forward and the *_backward functions under torch.no_grad()")
    return True


def _written(out: torch.Tensor) -> torch.Tensor:
    """A caller's ``out`` after the launch that fills it.  The kernels know addresses only; torch's version counter tells whoever holds the tensor's earlier contents (a recorded
    call that saved it, a cache that goes by it) that they are gone."""
    torch.autograd.graph.increment_version(out)
    return out


def _scratch_bytes(entry: str, args) -> int:
    lib = _lib.load()
    n = int(getattr(lib, entry)(C.byref(args)))
    if n == 0 and lib.pkh3_last_error():
        raise _lib.Pkh3Error(_lib.PKH3_EARG, lib.pkh3_last_error().decode())
    return n


# ---- layer norm ----

@lru_cache(maxsize=4096)
def _norm_scratch(rows: int, width: int, tables: int) -> int:
    return _scratch_bytes("pkh3_norm_workspace_bytes", _lib.NormArgs(rows=rows, width=width, tables=tables))


def _norm_tables(weight, bias, row_index, rows: int, width: int, index: int) -> Tuple[int, int, int, int, int]:
    """Addresses of weight, bias and index, the number of table rows, and the flag of the tables' type."""
    tables, kind = 1, None
    at = [0, 0]
    for i, (name, t) in enumerate((("weight", weight), ("bias", bias))):
        if t is None:
            continue
        shape = t.shape
        n = shape[0] if len(shape) == 2 else 1
        if len(shape) not in (1, 2) or shape[-1] != width or n < 1 or t.dtype not in (_BF16, _F32) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous float32 or bfloat16 [{width}] or [tables, {width}], got {t.dtype} {tuple(shape)}")
        if t.get_device() != index:
            raise ValueError(f"{name} must live in device memory, with x (got {t.device})")
        if kind is not None and (n != tables or t.dtype is not kind):
            raise ValueError(f"weight and bias must have one type and the same number of table rows, got {weight.dtype} {tuple(weight.shape)} and {t.dtype} {tuple(shape)}")
        tables, kind = n, t.dtype
        at[i] = t.data_ptr()
    if tables > 1 and row_index is None:
        raise ValueError(f"{tables} table rows need a row_index")
    where = 0 if row_index is None else _index("row_index", row_index, rows, index)
    return at[0], at[1], where, tables, _lib.LAYER_NORM_TABLES_BF16 if kind is _BF16 else 0


def _rows_type(x: torch.Tensor) -> int:
    if x.dtype not in (_BF16, _F32):
        raise TypeError(f"x must be bfloat16 or float32, got {x.dtype}")
    return _lib.LAYER_NORM_F32 if x.dtype is _F32 else 0


def _layer_norm(x, weight, bias, row_index, eps, out=None):
    index = _place(x)
    flags = _rows_type(x)
    x_at, x_row = _matrix("x", x, -1, -1, index, x.dtype)
    rows, width = x.shape
    w, b, where, tables, tables_type = _norm_tables(weight, bias, row_index, rows, width, index)
    given = out
    if out is None:
        out = torch.empty(rows, width, dtype=x.dtype, device=x.device)
    o_at, o_row = _matrix("out", out, rows, width, index, x.dtype)
    _call("pkh3_layer_norm", _pack_norm(x_at, w, b, where, o_at, 0, 0, 0, 0, 0, 0, x_row, o_row, 0, 0, rows, width, tables, eps, flags | tables_type), index)
    return out if given is None else _written(out)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               row_index: Optional[torch.Tensor] = None, eps: float = 1e-6, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` for the rows of ``x``, bfloat16 or float32 ``[rows, width]``, as ``x``'s type.  ``weight`` and
    ``bias``: float32 or bfloat16 ``[width]``, or ``[tables, width]`` with ``row_index`` int32 ``[rows]`` saying which table row a row takes (values are
    brought into range); a modulation ``norm(x) * (1 + scale) + shift`` is the tables ``1 + scale`` and ``shift``.  Width up to 16,384.  ``out`` may be ``x``."""
    if _wants_grad(x, weight, bias, out):
        if out is not None:
            raise ValueError("out cannot be given where gradients are recorded")
        for t in (weight, bias):
            if t is not None and t.requires_grad and t.dim() == 2 and t.shape[0] > _lib.LAYER_NORM_MAX_TABLES:
                raise ValueError(f"gradients of at most {_lib.LAYER_NORM_MAX_TABLES} table rows, got {t.shape[0]}")
        return _LayerNorm.apply(x, weight, bias, row_index, eps)
    return _layer_norm(x, weight, bias, row_index, eps, out)


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
                        row_index: Optional[torch.Tensor] = None, eps: float = 1e-6, weight_grad: bool = True, bias_grad: bool = True):
    """The backward pass of :func:`layer_norm` from the gradient ``dy`` of its result and the arguments of the call: ``(dx, dweight, dbias)``, ``dx`` as
    ``x``, the others float32 in the shape of ``weight`` and ``bias`` (None where these are, or are not asked for).  Tables that gradients are asked of have up to 64 rows."""
    _refuse_tangents(dy, x, weight, bias)
    index = _place(x)
    flags = _rows_type(x)
    x_at, x_row = _matrix("x", x, -1, -1, index, x.dtype)
    rows, width = x.shape
    dy_at, dy_row = _matrix("dy", dy, rows, width, index, x.dtype)
    w, b, where, tables, tables_type = _norm_tables(weight, bias, row_index, rows, width, index)
    dx = torch.empty(rows, width, dtype=x.dtype, device=x.device)
    make = torch.empty if rows else torch.zeros
    dw = make(weight.shape, dtype=_F32, device=x.device) if weight is not None and weight_grad else None
    db = make(bias.shape, dtype=_F32, device=x.device) if bias is not None and bias_grad else None
    if not rows:
        return dx, dw, db
    scratch, need = None, 0
    if dw is not None or db is not None:
        need = _norm_scratch(rows, width, tables)
        scratch = torch.empty(need, dtype=torch.uint8, device=x.device)
    _call("pkh3_layer_norm_backward",
          _pack_norm(x_at, w, 0, where, 0, dy_at, dx.data_ptr(), 0 if dw is None else dw.data_ptr(), 0 if db is None else db.data_ptr(),
                     0 if scratch is None else scratch.data_ptr(), need, x_row, 0, dy_row, width, rows, width, tables, eps, flags | tables_type), index)
    return dx, dw, db


# ---- products ----

@lru_cache(maxsize=8192)
def _product_scratch(M: int, N: int, K: int, flags: int, sums: bool) -> int:
    return _scratch_bytes("pkh3_product_workspace_bytes", _lib.ProductArgs(M=M, N=N, K=K, flags=flags, sums=256 if sums else None))


@lru_cache(maxsize=4096)
def _activation_scratch(M: int, N: int) -> int:
    return _scratch_bytes("pkh3_activation_grad_workspace_bytes", _lib.ProductArgs(M=M, N=N, sums=256))


def _product(a, b, out, M: int, N: int, K: int, flags: int, index: int, *, bias: int = 0, gate=(0, 0, 0, 0), residual=(0, 0), pre=(0, 0), sums: int = 0,
             act: int = 0) -> None:
    """One call of pkh3_product; ``a``, ``b``, ``out``, ``residual`` and ``pre`` as (address, row stride), ``gate`` as (address, index, row stride, rows)."""
    need = _product_scratch(M, N, K, flags & ~_lib.PRODUCT_BIAS_BF16, sums != 0)
    scratch = torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", index)) if need else None
    _call("pkh3_product", _pack_product(a[0], b[0], bias, gate[0], gate[1], residual[0], pre[0], out[0], sums, 0 if scratch is None else scratch.data_ptr(), need,
                                        a[1], b[1], gate[2], residual[1], pre[1], out[1], M, N, K, gate[3], act, flags), index)


def _finish(gate, row_index, residual, rows: int, N: int, index: int):
    """The fields gate and residual of a product."""
    g, r = (0, 0, 0, 0), (0, 0)
    if gate is not None:
        at, stride = _matrix("gate", gate, -1, N, index)
        if gate.shape[0] < 1:                             # (without rows it has no address either, and would be taken for none)
            raise ValueError("gate must have a row")
        if gate.shape[0] > 1 and row_index is None:
            raise ValueError(f"{gate.shape[0]} gate rows need a row_index")
        g = (at, 0 if row_index is None else _index("row_index", row_index, rows, index), stride, gate.shape[0])
    elif row_index is not None:
        raise ValueError("row_index goes with a gate")
    if residual is not None:
        r = _matrix("residual", residual, rows, N, index)
    return g, r


def _linear(x, weight, bias, activation, gate, row_index, residual, out, save):
    index = _place(x)
    act = _activation(activation)
    a = _matrix("x", x, -1, -1, index)
    rows, K = x.shape
    b = _matrix("weight", weight, -1, K, index)
    N = weight.shape[0]
    bias_at, flags = 0, 0
    if bias is not None:
        bias_at, narrow = _vector("bias", bias, N, index)
        flags = _lib.PRODUCT_BIAS_BF16 if narrow else 0
    g, r = _finish(gate, row_index, residual, rows, N, index)
    given = out
    if out is None:
        out = torch.empty(rows, N, dtype=_BF16, device=x.device)
    o = _matrix("out", out, rows, N, index)
    pre, p = None, (0, 0)
    if save and act:
        pre = torch.empty(rows, N, dtype=_F32, device=x.device)
        p = (pre.data_ptr(), N)
    _product(a, b, o, rows, N, K, flags, index, bias=bias_at, gate=g, residual=r, pre=p, act=act)
    return out if given is None else _written(out), pre


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: str = "none", gate: Optional[torch.Tensor] = None,
           row_index: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, save: bool = False):
    """``residual + gate[row_index] * act(x weight^T + bias)``, as far as given, in one pass: ``x`` bfloat16 ``[rows, K]``, ``weight`` ``[N, K]`` as a
    ``torch.nn.Linear`` has it, ``bias`` float32 or bfloat16, ``activation`` one of :data:`ACTIVATIONS`, ``gate`` bfloat16 ``[table rows, N]`` with
    ``row_index`` int32 ``[rows]`` (as :func:`.projections.out_proj` takes them), ``residual`` bfloat16 ``[rows, N]``; ``out`` may be ``residual``.
    ``save``: also returns what :func:`linear_backward` takes as ``pre`` (``x weight^T + bias`` in float32; None without an activation).  Where gradients are recorded, ``gate``,
    ``out`` and ``save`` are refused: the gate has no gradient here, so multiply by it behind the call, or call under no_grad."""
    if _wants_grad(x, weight, bias, gate, residual, out):
        if out is not None or save or gate is not None or row_index is not None:
            raise ValueError("out, save and gate (and its row_index) cannot be given where gradients are recorded")
        return _Linear.apply(x, weight, bias, residual, activation)
    y, pre = _linear(x, weight, bias, activation, gate, row_index, residual, out, save)
    return (y, pre) if save else y


def _column_sums(dy, at, rows: int, N: int, index: int) -> torch.Tensor:
    """Sums of dy's columns, bfloat16."""
    sums = torch.empty(N, dtype=_BF16, device=dy.device)
    _activation_grad(at, (0, 0), (0, 0), sums.data_ptr(), rows, N, 0, index)
    return sums


def _activation_grad(a, pre, out, sums: int, M: int, N: int, act: int, index: int) -> None:
    need = _activation_scratch(M, N) if sums else 0
    scratch = torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", index)) if need else None
    _call("pkh3_activation_grad", _pack_product(a[0], 0, 0, 0, 0, 0, pre[0], out[0], sums, 0 if scratch is None else scratch.data_ptr(), need,
                                                a[1], 0, 0, 0, pre[1], out[1], M, N, 0, 0, act, 0), index)


def _input_grad(dz, at, weight, w, rows: int, N: int, K: int, index: int) -> torch.Tensor:
    """dz weight, [rows, K]."""
    dx = torch.empty(rows, K, dtype=_BF16, device=dz.device)
    _product(at, w, (dx.data_ptr(), K), rows, K, N, _lib.PRODUCT_B_ACROSS, index)
    return dx


def _weight_grad(at, x, device, rows: int, N: int, K: int, index: int) -> torch.Tensor:
    """dz^T x, [N, K]."""
    dw = torch.empty(N, K, dtype=_BF16, device=device)
    _product(at, x, (dw.data_ptr(), K), N, K, rows, _lib.PRODUCT_A_ACROSS | _lib.PRODUCT_B_ACROSS, index)
    return dw


def _zeros(device, *shape):
    return torch.zeros(shape, dtype=_BF16, device=device)


def linear_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, pre: Optional[torch.Tensor] = None, *, activation: str = "none",
                    x_grad: bool = True, weight_grad: bool = True, bias_grad: bool = True):
    """``(dx, dweight, dbias)`` of ``act(x weight^T + bias)`` from the gradient ``dy`` of that (a residual's gradient is ``dy`` itself; that of a gated result
    is multiplied by the gate first), bfloat16 all; None for what is not asked for.  ``pre``: what :func:`linear` returned with ``save``."""
    _refuse_tangents(dy, x, weight, pre)
    index = _place(x)
    act = _activation(activation)
    xa = _matrix("x", x, -1, -1, index)
    rows, K = x.shape
    w = _matrix("weight", weight, -1, K, index)
    N = weight.shape[0]
    at = _matrix("dy", dy, rows, N, index)
    p = (0, 0)
    if act:
        if pre is None:
            raise ValueError(f"activation {activation!r} needs pre")
        p = _matrix("pre", pre, rows, N, index, _F32)
    dev = x.device
    if not rows:
        return (torch.empty_like(x) if x_grad else None, _zeros(dev, N, K) if weight_grad else None, _zeros(dev, N) if bias_grad else None)
    db = torch.empty(N, dtype=_BF16, device=dev) if bias_grad else None
    if act and (x_grad or weight_grad or bias_grad):
        dz = torch.empty(rows, N, dtype=_BF16, device=dev)
        z = (dz.data_ptr(), N)
        _activation_grad(at, p, z, db.data_ptr() if bias_grad else 0, rows, N, act, index)
    else:
        dz, z = dy, at
        if bias_grad:
            _activation_grad(at, p, (0, 0), db.data_ptr(), rows, N, 0, index)
    dx = _input_grad(dz, z, weight, w, rows, N, K, index) if x_grad else None
    dw = _weight_grad(z, xa, dev, rows, N, K, index) if weight_grad else None
    return dx, dw, db


# ---- the two products of a block ----

class Saved(NamedTuple):
    """What the backward pass of :func:`feed_forward` takes of the forward one: the first product with its bias, float32 (``[rows, 2 inner]`` gated: values
    and gates), and what the second product took, bfloat16."""

    pre: torch.Tensor
    hidden: torch.Tensor


def _block(x, w_in, w_out, gated: bool, index: int):
    """Checks of x and the weights: addresses, rows, width, inner features, features of the first product, outputs."""
    a = _matrix("x", x, -1, -1, index)
    rows, K = x.shape
    w1 = _matrix("w_in", w_in, -1, K, index)
    first = w_in.shape[0]
    if gated and first % 16:
        raise ValueError(f"w_in of a gated block has twice a multiple of 8 rows, got {first}")
    inner = first // 2 if gated else first
    w2 = _matrix("w_out", w_out, -1, inner, index)
    return a, w1, w2, rows, K, inner, first, w_out.shape[0]


def _feed_forward(x, w_in, w_out, b_in, b_out, activation, gated, gate, row_index, residual, out, save):
    index = _place(x)
    act = _activation(activation)
    a, w1, w2, rows, K, inner, first, N = _block(x, w_in, w_out, gated, index)
    b1 = b2 = 0
    f1 = _lib.PRODUCT_GATED if gated else 0
    f2 = 0
    if b_in is not None:
        b1, narrow = _vector("b_in", b_in, first, index)
        f1 |= _lib.PRODUCT_BIAS_BF16 if narrow else 0
    if b_out is not None:
        b2, narrow = _vector("b_out", b_out, N, index)
        f2 |= _lib.PRODUCT_BIAS_BF16 if narrow else 0
    g, r = _finish(gate, row_index, residual, rows, N, index)
    given = out
    if out is None:
        out = torch.empty(rows, N, dtype=_BF16, device=x.device)
    o = _matrix("out", out, rows, N, index)
    hidden = torch.empty(rows, inner, dtype=_BF16, device=x.device)
    h = (hidden.data_ptr(), inner)
    pre, p = None, (0, 0)
    if save:
        pre = torch.empty(rows, first, dtype=_F32, device=x.device)
        p = (pre.data_ptr(), first)
    _product(a, w1, h, rows, inner, K, f1, index, bias=b1, pre=p, act=act)
    _product(h, w2, o, rows, N, inner, f2, index, bias=b2, gate=g, residual=r)
    return out if given is None else _written(out), Saved(pre, hidden) if save else None


def feed_forward(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, b_in: Optional[torch.Tensor] = None, b_out: Optional[torch.Tensor] = None, *,
                 activation: str = "silu", gated: bool = True, gate: Optional[torch.Tensor] = None, row_index: Optional[torch.Tensor] = None,
                 residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, save: bool = False):
    """``residual + gate[row_index] * (h w_out^T + b_out)`` with ``h = act(x w_in^T + b_in)``, or, ``gated``, ``h = a * act(b)`` where the first half of
    ``w_in``'s rows (and of ``b_in``) makes a and the second b.  ``x`` bfloat16 ``[rows, width]``, ``w_in`` ``[inner or 2 inner, width]``, ``w_out``
    ``[outputs, inner]``; the rest as :func:`linear` takes it, and refuses it where gradients are recorded.  h is rounded to bfloat16 between the products.  ``save``: also
    returns :class:`Saved`."""
    if _wants_grad(x, w_in, w_out, b_in, b_out, gate, residual, out):
        if out is not None or save or gate is not None or row_index is not None:
            raise ValueError("out, save and gate (and its row_index) cannot be given where gradients are recorded")
        return _FeedForward.apply(x, w_in, w_out, b_in, b_out, residual, activation, gated)
    y, saved = _feed_forward(x, w_in, w_out, b_in, b_out, activation, gated, gate, row_index, residual, out, save)
    return (y, saved) if save else y


def feed_forward_backward(dy: torch.Tensor, x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, saved: Saved, *, activation: str = "silu",
                          gated: bool = True, x_grad: bool = True, weight_grad: bool = True, bias_grad: bool = True):
    """``(dx, dw_in, dw_out, db_in, db_out)`` of :func:`feed_forward` without its gate and residual (see :func:`linear_backward`), bfloat16; None for what is not
    asked for."""
    _refuse_tangents(dy, x, w_in, w_out, saved.pre, saved.hidden)
    return _feed_forward_backward(dy, x, w_in, w_out, saved, activation, gated, (x_grad, weight_grad, weight_grad, bias_grad, bias_grad))


def _feed_forward_backward(dy, x, w_in, w_out, saved: Saved, activation: str, gated: bool, wanted):
    """``wanted``: for each of the five gradients whether it is."""
    index = _place(x)
    act = _activation(activation)
    a, w1, w2, rows, K, inner, first, N = _block(x, w_in, w_out, gated, index)
    at = _matrix("dy", dy, rows, N, index)
    p = _matrix("saved.pre", saved.pre, rows, first, index, _F32)
    h = _matrix("saved.hidden", saved.hidden, rows, inner, index)
    dev = x.device
    if not rows:
        shapes = (first, K), (N, inner), (first,), (N,)
        return (torch.empty_like(x) if wanted[0] else None, *(_zeros(dev, *shape) if want else None for shape, want in zip(shapes, wanted[1:])))
    dx = dw_in = db_in = None
    if wanted[0] or wanted[1] or wanted[3]:
        dz = torch.empty(rows, first, dtype=_BF16, device=dev)
        z = (dz.data_ptr(), first)
        db_in = torch.empty(first, dtype=_BF16, device=dev) if wanted[3] else None
        flags = _lib.PRODUCT_B_ACROSS | _lib.PRODUCT_GRAD | (_lib.PRODUCT_GATED if gated else 0)
        _product(at, w2, z, rows, inner, N, flags, index, pre=p, sums=db_in.data_ptr() if wanted[3] else 0, act=act)
        dx = _input_grad(dz, z, w_in, w1, rows, first, K, index) if wanted[0] else None
        dw_in = _weight_grad(z, a, dev, rows, first, K, index) if wanted[1] else None
    dw_out = _weight_grad(at, h, dev, rows, N, inner, index) if wanted[2] else None
    db_out = _column_sums(dy, at, rows, N, index) if wanted[4] else None
    return dx, dw_in, dw_out, db_in, db_out


# ---- torch's differentiation ----

def _usable(dy: torch.Tensor, dtype) -> torch.Tensor:
    """The gradient that torch hands back, as rows that the kernels take (a sum's is one value in all places)."""
    if dy.dtype is not dtype:
        dy = dy.to(dtype)
    if dy.dim() == 2 and dy.stride(1) == 1 and dy.stride(0) % 8 == 0 and dy.stride(0) >= dy.shape[1] and dy.data_ptr() % 16 == 0:
        return dy
    return dy.clone(memory_format=torch.contiguous_format)


def _as(grad: Optional[torch.Tensor], like: Optional[torch.Tensor], wanted: bool):
    return grad.to(like.dtype) if wanted and grad is not None else None


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, row_index, eps):
        ctx.save_for_backward(x, weight, bias, row_index)
        ctx.eps = eps
        return _layer_norm(x, weight, bias, row_index, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, row_index = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = layer_norm_backward(_usable(dy, x.dtype), x, weight, bias, row_index=row_index, eps=ctx.eps, weight_grad=need[1], bias_grad=need[2])
        return dx if need[0] else None, _as(dw, weight, need[1]), _as(db, bias, need[2]), None, None


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        y, pre = _linear(x, weight, bias, activation, None, None, residual, None, True)
        ctx.save_for_backward(x, weight, bias, pre)
        ctx.activation = activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        dy = _usable(dy, _BF16)
        dx, dw, db = linear_backward(dy, x, weight, pre, activation=ctx.activation, x_grad=need[0], weight_grad=need[1], bias_grad=need[2])
        return dx, dw, _as(db, bias, need[2]), dy if need[3] else None, None


class _FeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, w_out, b_in, b_out, residual, activation, gated):
        y, saved = _feed_forward(x, w_in, w_out, b_in, b_out, activation, gated, None, None, residual, None, True)
        ctx.save_for_backward(x, w_in, w_out, b_in, b_out, *saved)
        ctx.kind = activation, gated
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w_in, w_out, b_in, b_out, *saved = ctx.saved_tensors
        need = ctx.needs_input_grad
        dy = _usable(dy, _BF16)
        activation, gated = ctx.kind
        dx, dw1, dw2, db1, db2 = _feed_forward_backward(dy, x, w_in, w_out, Saved(*saved), activation, gated, need[:5])
        return dx, dw1, dw2, _as(db1, b_in, need[3]), _as(db2, b_out, need[4]), dy if need[5] else None, None, None
