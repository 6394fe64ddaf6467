"""Float64 restatement of the paged K/V cache: what it holds of rows, and attention over it (test infrastructure only)."""
from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple

import torch

from .attention_oracle import apply_rope, rms_norm

PAGE = 64


def norm_rope(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float, rope=None, mode: int = 0) -> torch.Tensor:
    """Rows ``[n, heads, 128]`` through RMSNorm (``weight`` None: none) and rotation by tables ``[n, 64]``, in float64."""
    y = x.double()
    if weight is not None:
        y = rms_norm(y, weight.double(), eps)
    if mode:
        y = apply_rope(y[None], rope[0].double(), rope[1].double(), mode)[0]
    return y


def key_scales(x: torch.Tensor) -> torch.Tensor:
    """Scale of every row: the smallest power of two that is at least max|x| / 448 as float32 forms it, 2^-126 at least; 1 for zeros."""
    amax = x.abs().amax(-1, keepdim=True).float()
    ratio = (amax * torch.tensor(1.0 / 448.0, dtype=torch.float32)).double()
    exponent = torch.ceil(torch.log2(torch.where(ratio > 0, ratio, torch.full_like(ratio, 2.0 ** -126)))).clamp(min=-126)
    return torch.where(amax.double() > 0, torch.exp2(exponent), torch.ones_like(exponent))


def stored(x: torch.Tensor, fp8: bool) -> torch.Tensor:
    """What the cache gives back for rows ``x`` (float64): bf16 values, or e4m3 values times their scale."""
    if not fp8:
        return x.to(torch.bfloat16).double()
    scale = key_scales(x)
    y = x / scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)   # below the smallest normal number the step stays
    return torch.round(y / step) * step * scale                                    # (torch.round: ties to even)


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool, scale: Optional[float] = None,
           gone: Sequence[int] = ()) -> Tuple[torch.Tensor, torch.Tensor]:
    """One sequence in float64: queries ``[n, Hq, 128]``, its keys and values ``[m, H, 128]``.  Returns the output and sum_j p_j |v_j|, what an
    error of the weights is measured by; rows without a key give zeros in both.  ``gone``: pages whose keys nobody sees."""
    n, Hq, D = q.shape
    m, H, _ = k.shape
    out = torch.zeros((n, Hq, D), dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    if n == 0 or m == 0:
        return out, size
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    seen = torch.ones((n, m), dtype=torch.bool, device=q.device)
    if causal:
        seen = torch.arange(m, device=q.device)[None] <= (m - n + torch.arange(n, device=q.device))[:, None]
    for page in gone:
        seen = seen.clone()
        seen[:, PAGE * page:PAGE * (page + 1)] = False
    for h in range(Hq):
        s = q[:, h].double() @ k[:, h * H // Hq].double().t() * scale
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top > -math.inf, top, torch.zeros_like(top)))
        total = p.sum(-1, keepdim=True)
        p = torch.where(total > 0, p / torch.where(total > 0, total, torch.ones_like(total)), torch.zeros_like(p))
        out[:, h] = p @ v[:, h * H // Hq].double()
        size[:, h] = p @ v[:, h * H // Hq].double().abs()
    return out, size


def page_lists(lengths: List[int], spare: int, gen: torch.Generator) -> Tuple[int, List[List[int]]]:
    """A pool of shuffled pages that holds these sequences and ``spare`` pages besides: its size and the pages of every sequence."""
    counts = [(n + PAGE - 1) // PAGE for n in lengths]
    order = torch.randperm(sum(counts) + spare, generator=gen).tolist()
    lists, at = [], 0
    for c in counts:
        lists.append(order[at:at + c])
        at += c
    return len(order), lists
