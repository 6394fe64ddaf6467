"""What is timed of the operators on a paged K/V cache: writing it (norm, rotation, 8-bit rounding), reading it back, and the attention of new rows
over it, single tokens and chunks, each as a program that serves several sequences calls it.

``own`` selects the side: False the plain form in elementary torch operations, True the calls of this package.  A case is a dict of plain values:

  kind      "write"   new rows go into the cache and are read back (what the cache holds of them)
            "read"    the whole context of every sequence is read back
            "attend"  attention of the new rows over the cache
            "step"    the new rows' keys and values are written, then the new rows attend to everything; what the cache holds of them is read back
  seqs      sequences of the batch
  heads, kv_heads     query heads and the cache's (a divisor of them)
  new, new_min        new rows of a sequence: spread evenly between the two
  keys, keys_min      keys of a sequence, the new rows among them where they are written: spread evenly between the two
  fp8       the cache holds e4m3 with a power-of-two scale per key and head, else bf16
  causal    row i of n new ones sees the keys up to position keys - n + i, else all of its sequence
  norm      RMSNorm over the head dim of the rows that come in (queries; keys that are written)
  rope      0 none, 1 interleaved pairs, 2 half-split pairs: rotation of the same rows by tables
  empty     one sequence more without new rows and, where nothing is written, one with new rows and no keys
"""
import math
from types import SimpleNamespace

import torch

own = False

D = 128
PAGE = 64
EPS = 1e-6
FP8_MAX = 448.0
MOST_SCORES = 1 << 28     # scores that the plain form holds at once


def _case(kind, **kw):
    c = dict(kind=kind, seqs=1, heads=24, kv_heads=24, new=1, new_min=0, keys=64, keys_min=0, fp8=False, causal=False, norm=False, rope=0,
             empty=False)
    c.update(kw)
    c["new_min"] = c["new_min"] or c["new"]
    c["keys_min"] = c["keys_min"] or c["keys"]
    return c


def _named(name, kind, **kw):
    return dict(_case(kind, **kw), name=name)


def listed():
    return [
        # single tokens of a few short sequences: the smallest write there is, launches and host time
        _named("token-write", "write", seqs=4, heads=8, kv_heads=8, new=1, keys=333, keys_min=65, norm=True, rope=2),
        # keys and values of a whole document (480p, five seconds of video, audio and prompt) in 8 bits
        _named("clip-write-fp8", "write", new=15342, keys=15342, fp8=True, norm=True, rope=1),
        # contexts handed on to calls that take rows: three documents of unequal length out of 8 bits
        _named("context-read-fp8", "read", seqs=3, new=15342, new_min=2001, keys=15342, keys_min=2001, fp8=True),
        # one token of one small sequence
        _named("token", "attend", heads=4, kv_heads=4, keys=1024, causal=True, norm=True, rope=1),
        # a batch of single tokens, query heads sharing the cache's in groups of six, contexts of unequal length
        _named("tokens-grouped", "attend", seqs=16, kv_heads=4, keys=8000, keys_min=300, causal=True),
        # the same without groups, out of 8 bits and up to the length of the longest document
        _named("tokens-fp8", "attend", seqs=8, keys=48360, keys_min=1000, fp8=True, causal=True, norm=True, rope=2),
        # one token over the longest clip at the larger size
        _named("token-long", "attend", keys=124992, causal=True),
        # a new latent frame (30 x 52 rows) over the 480p clip before it, all of whose keys it sees
        _named("frame", "attend", new=1560, keys=48360, norm=True, rope=1),
        # the same step at the smaller patch grid (15 x 26), the frame's own keys written first, cache in 8 bits
        _named("frame-step-fp8", "step", new=390, keys=14830, fp8=True, norm=True, rope=1),
        # prompts of several requests in chunks: ragged, causal, grouped heads, written and attended to in 8 bits
        _named("prompt-step-fp8", "step", seqs=5, kv_heads=4, new=700, new_min=33, keys=2048, keys_min=700, fp8=True, causal=True, norm=True, rope=2),
        # text cross-attention of several requests at once: many video rows against prompts of other lengths kept in pages
        _named("cross-prompts", "attend", seqs=3, new=14430, new_min=5773, keys=512, keys_min=77, norm=True),
        # a long causal chunk over a longer context, grouped heads
        _named("chunk-long", "attend", kv_heads=4, new=8192, keys=32768, causal=True),
    ]


def _pairs(case):
    """(new rows, keys) of every sequence."""
    n = case["seqs"]
    spread = lambda lo, hi, i: hi if n == 1 else lo + (hi - lo) * i // (n - 1)   # noqa: E731
    # the longest context does not belong to the longest chunk
    got = [(spread(case["new_min"], case["new"], i), spread(case["keys_min"], case["keys"], (i * 7 + 3) % n if n % 7 else i)) for i in range(n)]
    if case["kind"] in ("write", "step"):
        got = [(min(a, b), b) for a, b in got]
    if case["kind"] == "read":
        got = [(b, b) for _, b in got]
    if case["empty"]:
        got.insert(n // 2, (0, case["keys_min"]))
        if case["kind"] == "attend" and not case["causal"]:
            got.append((case["new_min"], 0))
    return got


def _visible(case, new, keys):
    """Pairs of a new row and a key that it sees."""
    if not case["causal"]:
        return new * keys
    return sum(max(0, keys - new + i + 1) for i in range(new)) if new < 64 else _triangle(new, keys)


def _triangle(new, keys):
    short = max(0, new - keys)          # rows that stand before the first key
    rows = new - short
    return rows * (keys - new + short + 1) + rows * (rows - 1) // 2


def work(case):
    pairs = _pairs(case)
    rows, keys = sum(a for a, _ in pairs), sum(b for _, b in pairs)
    key_bytes = case["kv_heads"] * (2 * (D + 1) if case["fp8"] else 4 * D)     # one key as the cache holds it
    row_bytes = case["kv_heads"] * 4 * D                                       # ... and as rows of K and V
    tables = rows * D * 4 if case["rope"] else 0
    queries = 2 * rows * case["heads"] * D * 2
    if case["kind"] == "read":
        return {"bytes": keys * (key_bytes + row_bytes), "flops": 0}
    if case["kind"] == "write":
        return {"bytes": rows * (2 * row_bytes + key_bytes) + tables, "flops": 0}
    flops = sum(4 * D * case["heads"] * _visible(case, a, b) for a, b in pairs)
    moved = queries + keys * key_bytes + tables
    if case["kind"] == "step":
        moved += 2 * rows * row_bytes
    return {"bytes": moved, "flops": flops}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges, no dearer than the dearest listed one."""
    while True:
        kind = rng.choice(["write", "read", "attend", "attend", "attend", "step"])
        kv = rng.choice([1, 2, 3, 4, 8, 24])
        c = dict(kv_heads=kv, heads=kv * rng.choice([1, 1, 2, 3, 6, 8]), seqs=_log(rng, 1, 24), fp8=rng.random() < 0.5, rope=rng.choice([0, 1, 2]),
                 norm=rng.random() < 0.6, causal=rng.random() < 0.5, empty=rng.random() < 0.3)
        if kind == "write":
            c["heads"] = kv
            c["new"] = _log(rng, 1, 15000)
            c["keys"] = c["new"] + _log(rng, 1, 3000)
            c["causal"] = False
        elif kind == "read":
            c["heads"] = kv
            c["keys"] = _log(rng, 1, 15000)
            c["new"] = c["keys"]
            c.update(rope=0, norm=False, causal=False)
        else:
            c["new"] = rng.choice([1, _log(rng, 1, 40), _log(rng, 1, 8000)])
            c["keys"] = _log(rng, 1, 60000)
            if kind == "step" or c["causal"]:
                c["keys"] += c["new"]
        c["new_min"] = _log(rng, 1, c["new"])
        c["keys_min"] = _log(rng, min(c["keys"], c["new"] if kind == "step" else 1), c["keys"])
        case = _case(kind, **c)
        w = work(case)
        if w["flops"] <= 1.5e12 and w["bytes"] <= 6e8:
            return case


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=gen.device, dtype=torch.float32)


def _quantised(x):
    """(e4m3 values as float32, scales [..., 1]) of rows: the scale is the smallest power of two that is at least max|x| / 448, 1 for a row of zeros."""
    amax = x.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(amax * (1.0 / FP8_MAX))
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent).clamp(-126, 127)
    scale = torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), exponent), torch.ones_like(amax))
    return (x / scale).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    """The cache with what was written before, the batch, and the rows of the call."""
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    pairs = _pairs(case)
    rows = sum(a for a, _ in pairs)
    H, Hq = case["kv_heads"], case["heads"]
    counts = [(b + PAGE - 1) // PAGE for _, b in pairs]
    pages = sum(counts) + 3                                   # a pool has pages that nobody holds
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed))).tolist()
    lists, at = [], 0
    for c in counts:
        lists.append(order[at:at + c])
        at += c
    s = SimpleNamespace(case=case, pairs=pairs, rows=rows, pages=lists, dev=dev, norm_w=None, rope=None)
    if case["norm"]:
        s.norm_w = (1.0 + 0.2 * _randn(gen, D)).contiguous()
    if case["rope"]:
        where = torch.cat([torch.arange(b - a, b, device=dev, dtype=torch.float64) for a, b in pairs] or [torch.zeros(0, device=dev, dtype=torch.float64)])
        angle = where[:, None] * (10000.0 ** (-torch.arange(D // 2, device=dev, dtype=torch.float64) / (D // 2)))
        s.rope = (angle.cos().float().contiguous(), angle.sin().float().contiguous())
    s.k = s.v = s.q = None
    if case["kind"] in ("write", "step"):
        s.k = (_randn(gen, rows, H, D) * (0.5 + 1.5 * torch.rand((rows, H, 1), generator=gen, device=dev))).to(torch.bfloat16)
        s.v = (_randn(gen, rows, H, D) * (0.5 + 1.5 * torch.rand((rows, H, 1), generator=gen, device=dev))).to(torch.bfloat16)
    if case["kind"] in ("attend", "step"):
        s.q = (_randn(gen, rows, Hq, D) * (1.5 if case["norm"] else 1.2)).to(torch.bfloat16)
    # what the cache held before the call: rows as they are stored, in the order of the sequences
    held = [b if case["kind"] in ("read", "attend") else b - a for a, b in pairs]
    n = sum(held)
    k0 = _randn(gen, n, H, D).to(torch.bfloat16)
    v0 = _randn(gen, n, H, D).to(torch.bfloat16)
    if own:
        import pika_h3_flex_amd as pk

        s.cache = pk.PagedKV(pages, H, fp8=case["fp8"], device=dev)
        if n:
            pk.paged_write(s.cache, pk.PagedBatch.build(held, held, lists, device=dev), k0, v0)
        s.batch = pk.PagedBatch.build([a for a, _ in pairs], [b for _, b in pairs], lists, device=dev)
        return s
    s.kind = torch.float8_e4m3fn if case["fp8"] else torch.bfloat16
    s.k_pages = torch.zeros((pages * PAGE, H, D), dtype=torch.bfloat16, device=dev).to(s.kind)
    s.v_pages = s.k_pages.clone()
    s.k_scale = torch.ones((pages * PAGE, H, 1), device=dev)
    s.v_scale = s.k_scale.clone()
    s.slots = []                                              # place in the pool of every key of a sequence
    for (a, b), own_pages in zip(pairs, lists):
        t = torch.tensor(own_pages, dtype=torch.int64, device=dev)
        s.slots.append((t[:, None] * PAGE + torch.arange(PAGE, device=dev)).reshape(-1)[:b])
    if n:
        _store(s, torch.cat([at[:h] for at, h in zip(s.slots, held)]), k0.float(), v0.float())
    if rows:
        s.new_slots = torch.cat([at[b - a:b] for at, (a, b) in zip(s.slots, pairs)])
    return s


def _put(pool, at, x):
    # (index assignment of 8-bit floats goes by their bytes)
    if pool.dtype == torch.float8_e4m3fn:
        pool.view(torch.uint8)[at] = x.view(torch.uint8)
    else:
        pool[at] = x


def _take(pool, at):
    if pool.dtype == torch.float8_e4m3fn:
        return pool.view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
    return pool[at].float()


def _store(s, at, k, v):
    for x, pool, scales in ((k, s.k_pages, s.k_scale), (v, s.v_pages, s.v_scale)):
        if s.case["fp8"]:
            values, scale = _quantised(x)
            _put(pool, at, values)
            scales[at] = scale
        else:
            _put(pool, at, x.to(torch.bfloat16))


def _held(s, at):
    """Keys and values of these places, float32 [n, H, D]."""
    k, v = _take(s.k_pages, at), _take(s.v_pages, at)
    return (k * s.k_scale[at], v * s.v_scale[at]) if s.case["fp8"] else (k, v)


def _norm_rope(x, w, rope, mode):
    """Rows [n, heads, D] in the precision of ``x``: RMSNorm with weight ``w`` (None: no norm), then the rotation."""
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.to(x.dtype)
    if mode:
        c, t = rope[0].to(x.dtype)[:, None], rope[1].to(x.dtype)[:, None]
        if mode == 1:
            a, b = x[..., 0::2], x[..., 1::2]
            x = torch.stack([a * c - b * t, b * c + a * t], -1).reshape(x.shape)
        else:
            a, b = x[..., : D // 2], x[..., D // 2:]
            x = torch.cat([a * c - b * t, b * c + a * t], -1)
    return x


def _attend(s):
    case = s.case
    H, G = case["kv_heads"], case["heads"] // case["kv_heads"]
    q = _norm_rope(s.q.float(), s.norm_w, s.rope, case["rope"]) * (1.0 / math.sqrt(D))
    out = torch.zeros_like(s.q)
    at = 0
    for (a, b), slots in zip(s.pairs, s.slots):
        if a and b:
            k, v = _held(s, slots)
            kt = k.permute(1, 2, 0).contiguous()              # [H, D, keys]
            vh = v.permute(1, 0, 2).contiguous()              # [H, keys, D]
            step = max(1, MOST_SCORES // (case["heads"] * b))
            for i in range(0, a, step):
                n = min(step, a - i)
                qs = q[at + i:at + i + n].view(n, H, G, D).permute(1, 0, 2, 3).reshape(H, n * G, D).contiguous()
                scores = torch.matmul(qs, kt)
                if case["causal"]:
                    last = (b - a + i + torch.arange(n, device=s.dev)).repeat_interleave(G)
                    hidden = torch.arange(b, device=s.dev)[None] > last[:, None]
                    scores.masked_fill_(hidden, -math.inf)
                top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
                p = torch.exp(scores.sub_(top))
                o = torch.matmul(p, vh) / p.sum(-1, keepdim=True).clamp(min=1e-30)
                out[at + i:at + i + n] = o.view(H, n, G, D).permute(1, 0, 2, 3).reshape(n, H * G, D).to(torch.bfloat16)
        at += a
    return out


def run(s):
    case = s.case
    kind = case["kind"]
    got = []
    if own:
        import pika_h3_flex_amd as pk

        if kind in ("write", "step"):
            pk.paged_write(s.cache, s.batch, s.k, s.v, k_norm_weight=s.norm_w, norm_eps=EPS, rope_mode=case["rope"], rope_k=s.rope)
        if kind in ("attend", "step"):
            got.append(pk.paged_attention(s.q, s.cache, s.batch, causal=case["causal"], q_norm_weight=s.norm_w, norm_eps=EPS,
                                          rope_mode=case["rope"], rope_q=s.rope))
        if kind != "attend":
            got += pk.paged_read(s.cache, s.batch, s.rows)
        return got
    if kind in ("write", "step"):
        k = _norm_rope(s.k.float(), s.norm_w, s.rope, case["rope"])
        _store(s, s.new_slots, k, s.v.float())
    if kind in ("attend", "step"):
        got.append(_attend(s))
    if kind != "attend":
        k, v = _held(s, s.new_slots)
        got += [k.to(torch.bfloat16), v.to(torch.bfloat16)]
    return got


# ---- the same from the definition, in 64 bits ----

def _stored64(x, fp8):
    """What the cache holds of rows in float64, written out from the rule: every value to the nearest multiple of its own step, ties to even."""
    if not fp8:
        return x.to(torch.bfloat16).double()
    top = x.abs().amax(-1, keepdim=True)
    ratio = (top.float() * (1.0 / FP8_MAX)).double()
    scale = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, ratio, torch.ones_like(ratio)))))
    y = x / scale
    size = y.abs().clamp(min=2.0 ** -6)                       # below the smallest normal number the step stays
    step = torch.exp2(torch.floor(torch.log2(size)) - 3)
    return torch.round(y / step) * step * scale


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    kind, H, Hq = case["kind"], case["kv_heads"], case["heads"]
    G = Hq // H
    new = None
    if s.k is not None:
        k = _norm_rope(s.k.double(), s.norm_w, s.rope, case["rope"])
        new = (_stored64(k, case["fp8"]), _stored64(s.v.double(), case["fp8"]))
    got = []
    if kind in ("attend", "step"):
        q = _norm_rope(s.q.double(), s.norm_w, s.rope, case["rope"])
        o = torch.zeros((s.rows, Hq, D), dtype=torch.float64, device=s.dev)
        at = 0
        for (a, b), slots in zip(s.pairs, s.slots):
            if a and b:
                k, v = (t.double() for t in _held(s, slots))
                if new is not None:
                    k[b - a:], v[b - a:] = new[0][at:at + a], new[1][at:at + a]
                for h in range(Hq):
                    kh, vh = k[:, h // G].t().contiguous(), v[:, h // G].contiguous()
                    for i in range(0, a, 2048):
                        n = min(2048, a - i)
                        logits = q[at + i:at + i + n, h].contiguous() @ kh / math.sqrt(D)
                        if case["causal"]:
                            row = torch.arange(b - a + i, b - a + i + n, device=s.dev)[:, None]
                            logits = torch.where(torch.arange(b, device=s.dev)[None] <= row, logits, -math.inf)
                        p = torch.softmax(logits, -1).nan_to_num(0.0)
                        o[at + i:at + i + n, h] = p @ vh
            at += a
        got.append(o)
    if kind == "read":
        got += [t.double() for t in _held(s, s.new_slots)]
    elif new is not None:
        got += list(new)
    return got
