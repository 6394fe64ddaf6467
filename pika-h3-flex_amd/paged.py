"""A K/V cache in pages, shared by sequences of unequal length that grow as rows arrive: tensor-level front end of
``include/pkh3_paged.h``.  Keys and values go in through :func:`paged_write` (norm, rotation, and for a cache in 8 bits the
rounding, in one pass), :func:`paged_attention` attends to them, single tokens and chunks alike, and :func:`paged_read` gives them
back as rows.  As in :mod:`.ops`, PyTorch is memory and streams only.

The reference keeps nothing between two model calls (its document is one packed sequence, src/pika_h3/core/wrapper.py:192-204);
the rows are those of its attention module (src/pika_h3/core/loader.py:9).
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from .ops import HEAD_DIM, _f32, _on_device, _raw_stream

PAGE_KEYS = _lib.PAGE_KEYS


class PagedKV:
    """A pool of pages: 64 keys and values of ``heads`` heads each, head dim 128, in bf16 or (``fp8``) in e4m3 with a power-of-two
    scale per key, head and side.  ``data`` is uint8 ``[pages, heads, record]`` in the layout of the attention kernel;
    which page holds what is the caller's business (:class:`PagedBatch`).  A pool needs no clearing before pages are used again."""

    def __init__(self, pages: int, heads: int, *, fp8: bool = False, device=None, data: Optional[torch.Tensor] = None):
        self.pages, self.heads, self.fp8 = int(pages), int(heads), bool(fp8)
        if self.pages < 1 or self.heads < 1:
            raise ValueError(f"a pool has at least one page and one head, got {pages} and {heads}")
        self.record_bytes = int(_lib.load().pkh3_paged_record_bytes(_lib.PAGED_FP8 if self.fp8 else 0))
        shape = (self.pages, self.heads, self.record_bytes)
        if data is None:
            data = torch.empty(shape, dtype=torch.uint8, device=device if device is not None else "cuda")
        elif data.dtype != torch.uint8 or not data.is_contiguous() or data.shape != shape:
            raise ValueError(f"data must be contiguous uint8 {shape}, got {data.dtype} {tuple(data.shape)}")
        self.data = data

    @property
    def device(self):
        return self.data.device


@dataclass
class PagedBatch:
    """The sequences of a call: int32 device tensors ``starts [B + 1]`` (sequence b owns the call's rows ``starts[b] ..
    starts[b+1]-1``, its newest), ``lengths [B]`` (its keys, these rows among them where they are written) and ``table [B, P]``
    (key j lies in page ``table[b, j // 64]``).  ``rows``: the rows of the call where the host knows them.  The tensors may be changed in
    place between calls, replays of a captured graph among them; include/pkh3_paged.h says what out-of-range values do."""

    starts: torch.Tensor
    lengths: torch.Tensor
    table: torch.Tensor
    rows: Optional[int] = None

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


def _rows_of(name: str, t: torch.Tensor, heads: Optional[int], device) -> Tuple[int, int]:
    """Raises unless the kernels can read (or write) ``t`` as [rows, heads, 128]; its strides."""
    if t.dim() != 3 or t.shape[2] != HEAD_DIM or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be [rows, {'heads' if heads is None else heads}, {HEAD_DIM}], got {tuple(t.shape)}")
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    if t.stride(2) != 1:
        raise ValueError(f"{name}: head-dim stride must be 1, got {t.stride(2)}")
    if not t.is_cuda:
        raise ValueError(f"{name} must live in device memory (got {t.device}); the HIP library is the only compute path")
    _on_device(name, t, device)
    return t.stride(0), t.stride(1)


def _args(cache: PagedKV, batch: PagedBatch, rows: int, *, q=None, k=None, v=None, o=None, strides=(0,) * 8, heads=0, softmax_scale=None,
          norm_w=None, norm_eps=1e-6, rope_mode=_lib.ROPE_NONE, rope=None, flags=0) -> _lib.PagedArgs:
    dev = cache.data.device
    for name, t, dim in (("starts", batch.starts, 1), ("lengths", batch.lengths, 1), ("table", batch.table, 2)):
        if t.dtype != torch.int32 or t.dim() != dim or (t.stride(dim - 1) != 1 and t.shape[dim - 1] > 1):
            raise ValueError(f"batch {name} must be int32 with {dim} dimension(s) and unit stride, got {t.dtype} {tuple(t.shape)}")
        _on_device(f"batch {name}", t, dev)
    B = batch.lengths.shape[0]
    if batch.starts.shape[0] != B + 1 or batch.table.shape[0] != B:
        raise ValueError(f"batch of {B} lengths has {batch.starts.shape[0]} starts (need {B + 1}) and {batch.table.shape[0]} rows of pages")
    if batch.rows is not None and batch.rows != rows:
        raise ValueError(f"the batch has {batch.rows} rows, the call {rows}")
    norm_w = _f32("norm weight", norm_w, (HEAD_DIM,), dev)
    rope_mode = int(rope_mode)
    cos = sin = None
    if rope_mode != _lib.ROPE_NONE:
        if rope is None:
            raise ValueError("rope_mode set but its tables are missing")
        cos, sin = (_f32(f"rope {n}", t, (rows, HEAD_DIM // 2), dev) for n, t in zip(("cos", "sin"), rope))
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    return _lib.PagedArgs.from_buffer_copy(_lib.PAGED_ARGS_FORMAT.pack(
        cache.data.data_ptr(), cache.pages, batch.starts.data_ptr(), batch.lengths.data_ptr(), batch.table.data_ptr(), batch.table.stride(0),
        ptr(q), ptr(k), ptr(v), ptr(o), *strides, B, batch.table.shape[1], rows, cache.heads, heads, HEAD_DIM,
        0.0 if softmax_scale is None else C.c_float(softmax_scale).value, C.c_float(norm_eps).value, ptr(norm_w), ptr(cos), ptr(sin), rope_mode,
        flags | (_lib.PAGED_FP8 if cache.fp8 else 0), 0, 0))


def _call(entry, args: _lib.PagedArgs, device) -> None:
    if device.index == torch.cuda.current_device():
        _lib.check(entry(C.byref(args), _raw_stream(device.index)))
    else:
        with torch.cuda.device(device):
            _lib.check(entry(C.byref(args), _raw_stream(device.index)))


def paged_write(cache: PagedKV, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor, *, k_norm_weight: Optional[torch.Tensor] = None,
                norm_eps: float = 1e-6, rope_mode: int = _lib.ROPE_NONE, rope_k=None) -> None:
    """Keys (through RMSNorm and rotation, as given) and values of the call's rows, bf16 ``[rows, heads, 128]``, into their pages.
    ``rope_k``: cos/sin tables ``[rows, 64]``, a row per row of the call.  Runs asynchronously on the current stream."""
    dev = cache.data.device
    strides = _rows_of("k", k, cache.heads, dev) + _rows_of("v", v, cache.heads, dev)
    if k.shape[0] != v.shape[0]:
        raise ValueError(f"k has {k.shape[0]} rows, v {v.shape[0]}")
    args = _args(cache, batch, k.shape[0], k=k, v=v, strides=(0, 0) + strides + (0, 0), norm_w=k_norm_weight, norm_eps=norm_eps,
                 rope_mode=rope_mode, rope=rope_k)
    if k.shape[0]:
        _call(_lib.load().pkh3_paged_write, args, dev)


def paged_read(cache: PagedKV, batch: PagedBatch, rows: Optional[int] = None, *, out=None) -> List[torch.Tensor]:
    """Keys and values of the call's rows as the cache holds them: ``[k, v]``, bf16 ``[rows, heads, 128]`` (``out``: two tensors
    to put them in).  ``rows``: as ``batch.rows`` where the batch does not know.  Rows of no sequence, in given tensors, stay as they are;
    in new ones they hold anything."""
    dev = cache.data.device
    if rows is None:
        rows = batch.rows if out is None else out[0].shape[0]
    if rows is None:
        raise ValueError("the batch does not know its rows: say how many")
    if out is None:
        out = [torch.empty((rows, cache.heads, HEAD_DIM), dtype=torch.bfloat16, device=dev) for _ in range(2)]
    k, v = out
    strides = _rows_of("k", k, cache.heads, dev) + _rows_of("v", v, cache.heads, dev)
    if k.shape[0] != rows or v.shape[0] != rows:
        raise ValueError(f"out has {k.shape[0]} and {v.shape[0]} rows, the call {rows}")
    args = _args(cache, batch, rows, k=k, v=v, strides=(0, 0) + strides + (0, 0))
    if rows:
        _call(_lib.load().pkh3_paged_read, args, dev)
    return [k, v]


def paged_attention(q: torch.Tensor, cache: PagedKV, batch: PagedBatch, *, causal: bool = False, q_norm_weight: Optional[torch.Tensor] = None,
                    norm_eps: float = 1e-6, rope_mode: int = _lib.ROPE_NONE, rope_q=None, softmax_scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, workspace=None) -> torch.Tensor:
    """softmax(norm_rope(q) K^T * scale) V of the call's rows ``q``, bf16 ``[rows, heads, 128]`` with ``heads`` a multiple of the
    cache's, over all keys of their sequence, or with ``causal`` over those up to their own position.  A row that sees no key gets
    zeros.  ``workspace``: a uint8 device tensor, or a callable ``(device, nbytes) -> tensor``, as :func:`.ops.attention` takes it; two calls
    that may overlap need one each.  Returns ``out`` (may be ``q``)."""
    dev = cache.data.device
    lib = _lib.load()
    q_strides = _rows_of("q", q, None, dev)
    heads = q.shape[1]
    if heads == 0 or heads % cache.heads:
        raise ValueError(f"{heads} query heads are no multiple of the cache's {cache.heads}")
    if out is None:
        out = torch.empty(q.shape, dtype=torch.bfloat16, device=dev)
    o_strides = _rows_of("out", out, heads, dev)
    if out.shape[0] != q.shape[0]:
        raise ValueError(f"out has {out.shape[0]} rows, q {q.shape[0]}")
    args = _args(cache, batch, q.shape[0], q=q, o=out, strides=q_strides + (0,) * 4 + o_strides, heads=heads, softmax_scale=softmax_scale,
                 norm_w=q_norm_weight, norm_eps=norm_eps, rope_mode=rope_mode, rope=rope_q, flags=_lib.PAGED_CAUSAL if causal else 0)
    if not q.shape[0]:
        return out
    need = int(lib.pkh3_paged_workspace_bytes(C.byref(args)))
    if need == 0:
        raise _lib.Pkh3Error(_lib.PKH3_EARG, lib.pkh3_last_error().decode())
    if callable(workspace):
        workspace = workspace(dev, need)
    own = workspace is None or workspace.numel() * workspace.element_size() < need
    if own:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    elif workspace.device != dev:
        raise ValueError(f"workspace must live on {dev} (got {workspace.device})")
    args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    _call(lib.pkh3_paged_attn, args, dev)
    if not own:
        workspace.record_stream(torch.cuda.current_stream(dev))
    return out
