"""A K/V cache in pages, shared by sequences of unequal length that grow as rows arrive: tensor-level front end of
``include/pkh3_paged.h``.  Keys and values go in through :func:`paged_write` (norm, rotation, and for a cache in 8 bits the
rounding, in one pass), :func:`paged_attention` attends to them, single tokens and chunks alike, and :func:`paged_read` gives them
back as rows.  As in :mod:`.ops`, PyTorch is memory and streams only.

The reference keeps nothing between two model calls (its document is one packed sequence, src/pika_h3/core/wrapper.py:192-204);
the rows are those of its attention module (src/pika_h3/core/loader.py:9).
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass, field
from functools import lru_cache
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from .ops import HEAD_DIM, _raw_stream

PAGE_KEYS = _lib.PAGE_KEYS
_F32 = C.c_float


# Where the elements of a pool's or a batch's tensors lie: what resizing one of them, setting it or giving it other data changes.  (A type of another width
# changes the shape over the same memory, another device the address.)

def _pool_state(t: torch.Tensor) -> tuple:
    return t.data_ptr(), t.shape, t.stride()


def _batch_state(s: torch.Tensor, n: torch.Tensor, t: torch.Tensor) -> tuple:
    return s.data_ptr(), s.shape, s.stride(), n.data_ptr(), n.shape, n.stride(), t.data_ptr(), t.shape, t.stride()


class PagedKV:
    """A pool of pages: 64 keys and values of ``heads`` heads each, head dim 128, in bf16 or (``fp8``) in e4m3 with a power-of-two
    scale per key, head and side.  ``data`` is uint8 ``[pages, heads, record]`` in the layout of the attention kernel;
    which page holds what is the caller's business (:class:`PagedBatch`).  A pool needs no clearing before pages are used again."""

    def __init__(self, pages: int, heads: int, *, fp8: bool = False, device=None, data: Optional[torch.Tensor] = None):
        self.pages, self.heads, self.fp8 = int(pages), int(heads), bool(fp8)
        if self.pages < 1 or self.heads < 1:
            raise ValueError(f"a pool has at least one page and one head, got {pages} and {heads}")
        self.flags = _lib.PAGED_FP8 if self.fp8 else 0
        self.record_bytes = int(_lib.load().pkh3_paged_record_bytes(self.flags))
        if data is None:
            shape = (self.pages, self.heads, self.record_bytes)
            data = torch.empty(shape, dtype=torch.uint8, device=device if device is not None else "cuda")
        self._data = data
        self._take()

    def _take(self) -> None:
        """Checks the tensor and keeps what a call needs of it."""
        data, shape = self._data, (self.pages, self.heads, self.record_bytes)
        state = _pool_state(data)
        if data.dtype != torch.uint8 or not data.is_contiguous() or data.shape != shape:
            raise ValueError(f"data must be contiguous uint8 {shape}, got {data.dtype} {tuple(data.shape)}")
        self._head = (data.data_ptr(), self.pages)
        self._index = data.get_device()
        self._seen = state

    def __reduce__(self):
        # copies and pickles are made anew: what is kept beside the tensor holds its address
        return _pool_of, (self.pages, self.heads, self.fp8, self._data)

    @property
    def data(self) -> torch.Tensor:
        return self._data

    @property
    def device(self):
        return self._data.device


def _pool_of(pages: int, heads: int, fp8: bool, data: torch.Tensor) -> PagedKV:
    return PagedKV(pages, heads, fp8=fp8, data=data)


@dataclass(frozen=True)
class PagedBatch:
    """The sequences of a call: int32 device tensors ``starts [B + 1]`` (sequence b owns the call's rows ``starts[b] ..
    starts[b+1]-1``, its newest), ``lengths [B]`` (its keys, these rows among them where they are written) and ``table [B, P]``
    (key j lies in page ``table[b, j // 64]``).  ``rows``: the rows of the call where the host knows that they all are
    the sequences'; without it rows in front of the first sequence and behind the last may be nobody's, and are zeros in new outputs.  What the tensors hold may be
    changed in place between calls, replays of a captured graph among them (a graph goes on with the memory it was captured with);
    include/pkh3_paged.h says what out-of-range values do."""

    starts: torch.Tensor
    lengths: torch.Tensor
    table: torch.Tensor
    rows: Optional[int] = None
    _arrays: tuple = field(init=False, repr=False, compare=False)
    _sizes: tuple = field(init=False, repr=False, compare=False)
    _index: int = field(init=False, repr=False, compare=False)
    _seen: tuple = field(init=False, repr=False, compare=False)

    def __post_init__(self):
        # checked here, and again by the call that finds a tensor moved: small calls wait for the host, and a batch is the handle of many
        seen = _batch_state(self.starts, self.lengths, self.table)
        index = self.table.get_device()
        for name, t, dim in (("starts", self.starts, 1), ("lengths", self.lengths, 1), ("table", self.table, 2)):
            if t.dtype != torch.int32 or t.dim() != dim or (t.stride(dim - 1) != 1 and t.shape[dim - 1] > 1):
                raise ValueError(f"batch {name} must be int32 with {dim} dimension(s) and unit stride, got {t.dtype} {tuple(t.shape)}")
            if t.get_device() != index:
                raise ValueError(f"batch {name} must live with the table on {self.table.device} (got {t.device})")
        B = self.lengths.shape[0]
        if self.starts.shape[0] != B + 1 or self.table.shape[0] != B:
            raise ValueError(f"batch of {B} lengths has {self.starts.shape[0]} starts (need {B + 1}) and {self.table.shape[0]} rows of pages")
        object.__setattr__(self, "_arrays", (self.starts.data_ptr(), self.lengths.data_ptr(), self.table.data_ptr(), self.table.stride(0)))
        object.__setattr__(self, "_sizes", (B, self.table.shape[1]))
        object.__setattr__(self, "_index", index)
        object.__setattr__(self, "_seen", seen)

    def __reduce__(self):
        return PagedBatch, (self.starts, self.lengths, self.table, self.rows)

    @staticmethod
    def build(new_rows: Sequence[int], lengths: Sequence[int], pages: Sequence[Sequence[int]], *, device=None) -> "PagedBatch":
        """From host lists, checked: sequence b brings ``new_rows[b]`` rows, then has ``lengths[b]`` keys in ``pages[b]``."""
        B = len(new_rows)
        if B < 1 or len(lengths) != B or len(pages) != B:
            raise ValueError(f"one entry per sequence: got {B}, {len(lengths)} and {len(pages)}")
        if B > _lib.PAGED_MAX_SEQUENCES:
            raise ValueError(f"at most {_lib.PAGED_MAX_SEQUENCES} sequences a call, got {B}")
        for b in range(B):
            if new_rows[b] < 0 or lengths[b] < 0:
                raise ValueError(f"sequence {b}: negative rows or keys")
            if len(pages[b]) * PAGE_KEYS < lengths[b]:
                raise ValueError(f"sequence {b}: {lengths[b]} keys do not fit {len(pages[b])} pages of {PAGE_KEYS}")
            if any(page < 0 for page in pages[b]):
                raise ValueError(f"sequence {b}: negative page")
        P = max(1, max(len(x) for x in pages))
        starts = [0]
        for n in new_rows:
            starts.append(starts[-1] + int(n))
        table = [list(x) + [-1] * (P - len(x)) for x in pages]
        as_int = lambda x: torch.tensor(x, dtype=torch.int32).to(device if device is not None else "cuda")  # noqa: E731
        return PagedBatch(as_int(starts), as_int([int(n) for n in lengths]), as_int(table), starts[-1])


def _rows_of(name: str, t: torch.Tensor, heads: int, index: int) -> Tuple[int, int, int]:
    """Raises unless the kernels can read (or write) ``t`` as [rows, heads, 128] on device ``index``; its strides and rows.  ``heads`` 0: any."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != HEAD_DIM or (heads and shape[1] != heads):
        raise ValueError(f"{name} must be [rows, {heads or 'heads'}, {HEAD_DIM}], got {tuple(shape)}")
    if t.dtype is not torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    strides = t.stride()
    if strides[2] != 1:
        raise ValueError(f"{name}: head-dim stride must be 1, got {strides[2]}")
    on = t.get_device()
    if on != index or on < 0:
        raise ValueError(f"{name} must live in device memory, with the cache (got {t.device}); the HIP library is the only compute path")
    return strides[0], strides[1], shape[0]


def _f32(name: str, t: torch.Tensor, shape: tuple, index: int) -> int:
    if t.dtype is not torch.float32 or not t.is_contiguous() or t.shape != shape:
        raise ValueError(f"{name} must be contiguous float32 {shape}, got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != index:
        raise ValueError(f"{name} must live in device memory, with the cache (got {t.device})")
    return t.data_ptr()


def _norm_rope(norm_w, rope_mode, rope, rows: int, index: int) -> tuple:
    """The fields norm_w, rope_cos, rope_sin, rope_mode."""
    w = 0 if norm_w is None else _f32("norm weight", norm_w, (HEAD_DIM,), index)
    rope_mode = int(rope_mode)
    if rope_mode == _lib.ROPE_NONE:
        return w, 0, 0, rope_mode
    if rope is None:
        raise ValueError("rope_mode set but its tables are missing")
    shape = (rows, HEAD_DIM // 2)
    return w, _f32("rope cos", rope[0], shape, index), _f32("rope sin", rope[1], shape, index), rope_mode


def _place(cache: PagedKV, batch: PagedBatch) -> int:
    """The device of a call: that of the cache and the batch, whose tensors are looked for first where they were at their last check."""
    if _batch_state(batch.starts, batch.lengths, batch.table) != batch._seen:
        batch.__post_init__()
    if _pool_state(cache._data) != cache._seen:
        cache._take()
    if batch._index != cache._index:
        raise ValueError(f"the batch must live with the cache on {cache.device} (got {batch.table.device})")
    return cache._index


def _check_rows(batch: PagedBatch, rows: int) -> None:
    if batch.rows is not None and batch.rows != rows:
        raise ValueError(f"the batch has {batch.rows} rows, the call {rows}")


_pack = _lib.PAGED_ARGS_FORMAT.pack


@lru_cache(maxsize=None)
def _entry(name: str):
    """A C entry that takes the packed bytes of its arguments."""
    call = _lib.load()[name]
    call.argtypes = [C.c_char_p, C.c_void_p]
    call.restype = C.c_int
    return call


@lru_cache(maxsize=4096)
def _workspace_bytes(rows: int, B: int, table_pages: int, kv_heads: int, heads: int, flags: int) -> int:
    """Scratch of an attention call: a matter of its sizes alone."""
    args = _lib.PagedArgs(n_pages=1, B=B, table_pages=table_pages, rows=rows, kv_heads=kv_heads, heads=heads, D=HEAD_DIM, flags=flags)
    lib = _lib.load()
    n = int(lib.pkh3_paged_workspace_bytes(C.byref(args)))
    if n == 0:
        raise _lib.Pkh3Error(_lib.PKH3_EARG, lib.pkh3_last_error().decode())
    return n


def _call(name: str, args: bytes, index: int) -> None:
    if index == torch.cuda.current_device():
        rc = _entry(name)(args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = _entry(name)(args, _raw_stream(index))
    if rc:
        _lib.check(rc)


def paged_write(cache: PagedKV, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor, *, k_norm_weight: Optional[torch.Tensor] = None,
                norm_eps: float = 1e-6, rope_mode: int = _lib.ROPE_NONE, rope_k=None) -> None:
    """Keys (through RMSNorm and rotation, as given) and values of the call's rows, bf16 ``[rows, heads, 128]``, into their pages.
    ``rope_k``: cos/sin tables ``[rows, 64]``, a row per row of the call.  Runs asynchronously on the current stream."""
    index, H = _place(cache, batch), cache.heads
    k_ss, k_sh, rows = _rows_of("k", k, H, index)
    v_ss, v_sh, v_rows = _rows_of("v", v, H, index)
    if rows != v_rows:
        raise ValueError(f"k has {rows} rows, v {v_rows}")
    _check_rows(batch, rows)
    prep = _norm_rope(k_norm_weight, rope_mode, rope_k, rows, index)
    if rows:
        _call("pkh3_paged_write", _pack(*cache._head, *batch._arrays, 0, k.data_ptr(), v.data_ptr(), 0, 0, 0, k_ss, k_sh, v_ss, v_sh, 0, 0,
                                        *batch._sizes, rows, H, 0, HEAD_DIM, 0.0, _F32(norm_eps).value, *prep, cache.flags, 0, 0), index)


def paged_read(cache: PagedKV, batch: PagedBatch, rows: Optional[int] = None, *, out=None) -> List[torch.Tensor]:
    """Keys and values of the call's rows as the cache holds them: ``[k, v]``, bf16 ``[rows, heads, 128]`` (``out``: two tensors
    to put them in, apart from each other).  ``rows``: as ``batch.rows`` where the batch does not know.  Rows of no sequence stay as
    they are in given tensors; in new ones they are zeros, or where ``batch.rows`` says that there are none may hold anything."""
    index, H = _place(cache, batch), cache.heads
    if rows is None:
        rows = batch.rows if out is None else out[0].shape[0]
    if rows is None:
        raise ValueError("the batch does not know its rows: say how many")
    if out is None:
        make = torch.zeros if batch.rows is None else torch.empty             # (the kernels leave rows of no sequence alone)
        out = [make(rows, H, HEAD_DIM, dtype=torch.bfloat16, device=cache.device) for _ in range(2)]
    k, v = out
    k_ss, k_sh, k_rows = _rows_of("k", k, H, index)
    v_ss, v_sh, v_rows = _rows_of("v", v, H, index)
    if k_rows != rows or v_rows != rows:
        raise ValueError(f"out has {k_rows} and {v_rows} rows, the call {rows}")
    _check_rows(batch, rows)
    if rows:
        _call("pkh3_paged_read", _pack(*cache._head, *batch._arrays, 0, k.data_ptr(), v.data_ptr(), 0, 0, 0, k_ss, k_sh, v_ss, v_sh, 0, 0,
                                       *batch._sizes, rows, H, 0, HEAD_DIM, 0.0, 0.0, 0, 0, 0, 0, cache.flags, 0, 0), index)
    return [k, v]


def paged_attention(q: torch.Tensor, cache: PagedKV, batch: PagedBatch, *, causal: bool = False, q_norm_weight: Optional[torch.Tensor] = None,
                    norm_eps: float = 1e-6, rope_mode: int = _lib.ROPE_NONE, rope_q=None, softmax_scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, workspace=None) -> torch.Tensor:
    """softmax(norm_rope(q) K^T * scale) V of the call's rows ``q``, bf16 ``[rows, heads, 128]`` with ``heads`` a multiple of the
    cache's, over all keys of their sequence, or with ``causal`` over those up to their own position.  A row that sees no key gets
    zeros.  ``workspace``: a uint8 device tensor, or a callable ``(device, nbytes) -> tensor``, as :func:`.ops.attention` takes it; two calls
    that may overlap need one each.  Returns ``out`` (may be ``q``, and must not overlap it otherwise); rows of no sequence are as those of :func:`paged_read`.
    For inference: gradients do not flow through it, as through none of the package's calls."""
    index = _place(cache, batch)
    q_ss, q_sh, rows = _rows_of("q", q, 0, index)
    heads = q.shape[1]
    if heads == 0 or heads % cache.heads:
        raise ValueError(f"{heads} query heads are no multiple of the cache's {cache.heads}")
    if out is None:
        out = (torch.zeros_like if batch.rows is None else torch.empty_like)(q, memory_format=torch.contiguous_format)
        o_ss, o_sh = heads * HEAD_DIM, HEAD_DIM
    else:
        o_ss, o_sh, o_rows = _rows_of("out", out, heads, index)
        if o_rows != rows:
            raise ValueError(f"out has {o_rows} rows, q {rows}")
    _check_rows(batch, rows)
    prep = _norm_rope(q_norm_weight, rope_mode, rope_q, rows, index)
    if not rows:
        return out
    need = _workspace_bytes(rows, *batch._sizes, cache.heads, heads, cache.flags)
    if callable(workspace):
        workspace = workspace(cache.device, need)
    own = workspace is None or workspace.numel() * workspace.element_size() < need
    if own:
        workspace = torch.empty(need, dtype=torch.uint8, device=cache.device)
    elif workspace.get_device() != index or not workspace.is_contiguous():
        raise ValueError(f"workspace must be contiguous and live on {cache.device} (got {workspace.device}, strides {workspace.stride()})")
    _call("pkh3_paged_attn", _pack(*cache._head, *batch._arrays, q.data_ptr(), 0, 0, out.data_ptr(), q_ss, q_sh, 0, 0, 0, 0, o_ss, o_sh,
                                   *batch._sizes, rows, cache.heads, heads, HEAD_DIM, 0.0 if softmax_scale is None else _F32(softmax_scale).value,
                                   _F32(norm_eps).value, *prep, cache.flags | (_lib.PAGED_CAUSAL if causal else 0), workspace.data_ptr(),
                                   workspace.numel() * workspace.element_size()), index)
    if not own:
        workspace.record_stream(torch.cuda.current_stream(index))
    return out
