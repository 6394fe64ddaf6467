"""What is timed of the feed-forward half of a block: layer norm with its tables, the matrix product with bias, activation, gate and residual, and the
feed-forward block of two products, plain or gated, each forward as in serving and forward and backward as in a training step.

``own`` selects the side: False the plain form in elementary torch operations, True the calls of this package.  A case is a dict of plain values:

  kind      "norm"    layer norm of rows                 "norm-train"    and its gradients
            "linear"  one product                        "linear-train"  and its gradients
            "ff"      two products, activation between   "ff-train"      and its gradients
            "half"    layer norm, feed-forward, gate and residual, one behind the other
  rows      tokens of the call
  width     elements of a row that comes in
  inner     features of the product ("linear"), of the block's middle ("ff", "half")
  act       "none", "silu", "gelu" (erf), "gelu_tanh"
  gated     the first product has 2 * inner features: values, and gates that the activation goes to
  bias      0 none, 1 float32, 2 bfloat16; of the norm: its tables' type, 0 none
  residual  a residual is added to the output;  gate: the output is multiplied by the row's table row first (forward kinds)
  tables    rows of the norm's tables and of the gate's: above 1 a row of the call takes the one that its index names
  wide      the norm's rows are float32, else bfloat16
"""
import math
from types import SimpleNamespace

import torch

own = False

EPS = 1e-6
DENSE_FLOPS, DENSE_BYTES = 5.2e12, 2.5e9      # what the dearest listed cases take


def _case(kind, **kw):
    c = dict(kind=kind, rows=1, width=1024, inner=1024, act="silu", gated=False, bias=0, residual=False, gate=False, tables=1, wide=False)
    c.update(kw)
    return c


def _named(name, kind, **kw):
    return dict(_case(kind, **kw), name=name)


def listed():
    return [
        # a few rows' norm in a small model: launches and host time
        _named("norm-rows", "norm", rows=4, width=1024, bias=1),
        # the modulated norm of a 480p clip: rows of three timestep groups take their shift and scale from bf16 tables
        _named("norm-clip", "norm", rows=48360, width=2048, bias=2, tables=3),
        # a training step's norm, plain weights, float32 rows of a small clip
        _named("norm-train", "norm-train", rows=15342, width=1536, bias=1, wide=True),
        # one row through a projection: the weight is read for it alone
        _named("linear-row", "linear", rows=1, width=2048, inner=8192, act="gelu_tanh", bias=2),
        # the output projection of one image, with gate and residual
        _named("linear-image", "linear", rows=1085, width=2048, inner=2048, act="none", bias=1, residual=True, gate=True, tables=3),
        # one projection of a training step over prompts, widths that are no powers of two
        _named("linear-train", "linear-train", rows=2003, width=1400, inner=5160, act="gelu", bias=1),
        # eight rows through a gated block: both weights are read for them
        _named("ff-rows", "ff", rows=8, width=2048, inner=5504, act="silu", gated=True),
        # the prompts of a batch through a plain block
        _named("ff-prompts", "ff", rows=302, width=4096, inner=11008, act="gelu_tanh", bias=1, residual=True),
        # the smallest training step of a gated block
        _named("ff-image-train", "ff-train", rows=1085, width=1536, inner=4096, act="gelu", gated=True, bias=2),
        # a training step of a gated block over a short clip
        _named("ff-clip-train", "ff-train", rows=15342, width=2048, inner=5504, act="silu", gated=True, residual=True),
        # half a block as a sampler calls it: modulated norm, gated block, gate, residual
        _named("half-clip", "half", rows=15342, width=2048, inner=8192, act="silu", gated=True, bias=2, tables=3),
        # a plain block over a whole 480p document
        _named("ff-document", "ff", rows=48360, width=2048, inner=8192, act="gelu_tanh", bias=2, residual=True),
    ]


def work(case):
    T, C, F = case["rows"], case["width"], case["inner"]
    kind = case["kind"]
    train = kind.endswith("-train")
    element = 4 if case["wide"] else 2
    tables = 2 * case["tables"] * C * (4 if case["bias"] == 1 else 2) if case["bias"] else 0
    if kind.startswith("norm"):
        # forward: rows in and out; backward: the gradient in, the rows' gradient out (the rows themselves are read once)
        grads = 2 * case["tables"] * C * 4 if train and case["bias"] else 0
        return {"bytes": (4 if train else 2) * T * C * element + tables + grads, "flops": 0}
    out = T * (F if kind.startswith("linear") else C)
    weights = C * F if kind.startswith("linear") else C * F * (3 if case["gated"] else 2)
    moved = 2 * (T * C + weights + out) + (2 * out if case["residual"] or kind == "half" else 0)
    flops = 2 * T * weights
    if train:
        moved += 2 * (out + T * C + weights)
        flops *= 3
    return {"bytes": moved + (tables if kind == "half" else 0), "flops": flops}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Rows of whole 16-byte pieces."""
    return max(8, _log(rng, lo, hi) // 8 * 8)


def draw(rng):
    """One more case of the same ranges, no dearer than the dearest listed one."""
    while True:
        kind = rng.choice(["norm", "norm-train", "linear", "linear", "linear-train", "ff", "ff", "ff-train", "half"])
        c = dict(rows=_log(rng, 1, 48360), width=_width(rng, 256, 4096), inner=_width(rng, 256, 12000), bias=rng.choice([0, 1, 2]),
                 act=rng.choice(["silu", "gelu", "gelu_tanh"]), tables=rng.choice([1, 1, 2, 3, 7]))
        if kind.startswith("norm"):
            c.update(wide=rng.random() < 0.5, act="none", inner=c["width"])
        else:
            c["gated"] = not kind.startswith("linear") and rng.random() < 0.6
            if kind.startswith("linear") and rng.random() < 0.4:
                c["act"] = "none"
            c["residual"] = kind != "half" and rng.random() < 0.5
            c["gate"] = kind in ("linear", "ff") and rng.random() < 0.4
            if kind in ("linear-train", "ff-train"):
                c["tables"] = 1
        case = _case(kind, **c)
        w = work(case)
        if w["flops"] <= DENSE_FLOPS and w["bytes"] <= DENSE_BYTES:
            return case


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=gen.device, dtype=torch.float32)


def prepare(case, seed):
    """Rows, weights, tables, and the gradient that comes back from what follows."""
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    T, C, F, kind = case["rows"], case["width"], case["inner"], case["kind"]
    table_type = torch.bfloat16 if case["bias"] == 2 else torch.float32
    s = SimpleNamespace(case=case, dev=dev, w=None, b=None, index=None, w_in=None, w_out=None, b_in=None, b_out=None, residual=None, gate=None, dy=None)
    # rows have sizes of their own and a mean beside zero, as a residual stream has
    x = _randn(gen, T, C) * (0.5 + 1.5 * torch.rand((T, 1), generator=gen, device=dev))
    if kind.startswith("norm") or kind == "half":
        x += 0.3 * _randn(gen, T, 1)
        if case["bias"]:
            shape = (case["tables"], C) if case["tables"] > 1 else (C,)
            s.w = (1.0 + 0.2 * _randn(gen, *shape)).to(table_type)
            s.b = (0.2 * _randn(gen, *shape)).to(table_type)
    if case["tables"] > 1:
        # a document's rows come in runs of one group (its frames, its sound, its condition)
        cuts = torch.randint(0, T + 1, (2 * case["tables"],), generator=gen, device=dev).sort().values
        run = torch.bucketize(torch.arange(T, device=dev), cuts, right=True)
        s.index = (run % case["tables"]).to(torch.int32)
    s.x = x.to(torch.float32 if case["wide"] else torch.bfloat16)
    out = C
    if not kind.startswith("norm"):
        first = F * (2 if case["gated"] else 1)
        s.w_in = (_randn(gen, first, C) / math.sqrt(C)).to(torch.bfloat16)
        if case["bias"]:
            s.b_in = (0.2 * _randn(gen, first)).to(table_type)
        if kind.startswith("linear"):
            out = F
        else:
            s.w_out = (_randn(gen, C, F) * (1.5 / math.sqrt(F))).to(torch.bfloat16)
            if case["bias"]:
                s.b_out = (0.2 * _randn(gen, C)).to(table_type)
        if case["residual"]:
            s.residual = _randn(gen, T, out).to(torch.bfloat16)
        if case["gate"] or kind == "half":
            s.gate = (0.5 * _randn(gen, case["tables"], out)).to(torch.bfloat16)
    if kind.endswith("-train"):
        s.dy = _randn(gen, T, out).to(s.x.dtype)
    return s


# ---- the plain form: elementary operations in 32 bits, rounded at the end ----

def _phi(v):
    return 0.5 * (1.0 + torch.erf(v * (1.0 / math.sqrt(2.0))))


_TANH = math.sqrt(2.0 / math.pi)


def _act(name, v):
    if name == "none":
        return v
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    if name == "gelu":
        return v * _phi(v)
    return 0.5 * v * (1.0 + torch.tanh(_TANH * (v + 0.044715 * v * v * v)))


def _act_slope(name, v):
    if name == "silu":
        q = 1.0 / (1.0 + torch.exp(-v))
        return q * (1.0 + v * (1.0 - q))
    if name == "gelu":
        return _phi(v) + v * torch.exp(-0.5 * v * v) * (1.0 / math.sqrt(2.0 * math.pi))
    t = torch.tanh(_TANH * (v + 0.044715 * v * v * v))
    return 0.5 * (1.0 + t) + 0.5 * v * (1.0 - t * t) * _TANH * (1.0 + 3 * 0.044715 * v * v)


def _rows_of(table, index):
    """What each row takes of a table, float32."""
    if table is None:
        return None
    t = table.float().view(-1, table.shape[-1])
    return t if index is None or t.shape[0] == 1 else t[index.long()]


def _standard(x):
    x = x.float()
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    rstd = torch.rsqrt(d.square().mean(-1, keepdim=True) + EPS)
    return d * rstd, rstd


def _norm(s):
    xh, _ = _standard(s.x)
    w, b = _rows_of(s.w, s.index), _rows_of(s.b, s.index)
    return xh if w is None else xh * w + b


def _table_sums(s, rows):
    """Sums of the rows that take the same table row."""
    n = s.case["tables"]
    if n == 1:
        return rows.sum(0)
    return torch.stack([rows[s.index == i].sum(0) for i in range(n)])


def _norm_gradients(s):
    xh, rstd = _standard(s.x)
    dy, w = s.dy.float(), _rows_of(s.w, s.index)
    g = dy if w is None else dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    got = [dx.to(s.x.dtype)]
    if w is not None:
        got += [_table_sums(s, dy * xh), _table_sums(s, dy)]
    return got


def _product(x, w, b):
    z = torch.matmul(x, w.float().t())
    return z if b is None else z + b.float()


def _finish(s, y):
    if s.gate is not None:
        y = y * _rows_of(s.gate, s.index)
    if s.residual is not None:
        y = y + s.residual.float()
    return y.to(torch.bfloat16)


def _middle(s, z):
    if not s.case["gated"]:
        return _act(s.case["act"], z)
    F = s.case["inner"]
    return z[:, :F] * _act(s.case["act"], z[:, F:])


def _forward(s, x):
    """(output, first product, what the second one takes)"""
    z = _product(x, s.w_in, s.b_in)
    if s.w_out is None:
        return _finish(s, _act(s.case["act"], z)), z, None
    h = _middle(s, z)
    return _finish(s, _product(h, s.w_out, s.b_out)), z, h


def _gradients(s, x, z, h):
    act, F = s.case["act"], s.case["inner"]
    dy = s.dy.float()
    got = []
    if s.w_out is None:
        dz = dy if act == "none" else dy * _act_slope(act, z)
    else:
        dh = torch.matmul(dy, s.w_out.float())
        if s.case["gated"]:
            a, b = z[:, :F], z[:, F:]
            dz = torch.cat([dh * _act(act, b), dh * a * _act_slope(act, b)], 1)
        else:
            dz = dh * _act_slope(act, z)
    got += [torch.matmul(dz, s.w_in.float()).to(torch.bfloat16), torch.matmul(dz.t(), x).to(torch.bfloat16)]
    if s.w_out is not None:
        got.append(torch.matmul(dy.t(), h).to(torch.bfloat16))
    if s.b_in is not None:
        # (in the type of the weights' gradients)
        got.append(dz.sum(0).to(torch.bfloat16))
        if s.w_out is not None:
            got.append(dy.sum(0).to(torch.bfloat16))
    return got


def _run_own(s):
    import pika_h3_flex_amd as pk

    case, kind = s.case, s.case["kind"]
    act, gated = case["act"], case["gated"]
    if kind.startswith("norm"):
        y = pk.layer_norm(s.x, s.w, s.b, row_index=s.index, eps=EPS)
        if kind == "norm":
            return [y]
        return [y] + [t for t in pk.layer_norm_backward(s.dy, s.x, s.w, s.b, row_index=s.index, eps=EPS) if t is not None]
    bias = s.b_in is not None
    if kind == "linear":
        return [pk.linear(s.x, s.w_in, s.b_in, activation=act, gate=s.gate, row_index=s.index if s.gate is not None else None, residual=s.residual)]
    if kind == "linear-train":
        y, pre = pk.linear(s.x, s.w_in, s.b_in, activation=act, residual=s.residual, save=True)
        return [y] + [t for t in pk.linear_backward(s.dy, s.x, s.w_in, pre, activation=act, bias_grad=bias) if t is not None]
    if kind == "ff-train":
        y, saved = pk.feed_forward(s.x, s.w_in, s.w_out, s.b_in, s.b_out, activation=act, gated=gated, residual=s.residual, save=True)
        return [y] + [t for t in pk.feed_forward_backward(s.dy, s.x, s.w_in, s.w_out, saved, activation=act, gated=gated, bias_grad=bias) if t is not None]
    x, residual = s.x, s.residual
    if kind == "half":
        x, residual = pk.layer_norm(s.x, s.w, s.b, row_index=s.index, eps=EPS), s.x
    return [pk.feed_forward(x, s.w_in, s.w_out, s.b_in, s.b_out, activation=act, gated=gated, gate=s.gate,
                            row_index=s.index if s.gate is not None else None, residual=residual)]


def run(s):
    if own:
        return _run_own(s)
    kind = s.case["kind"]
    if kind.startswith("norm"):
        y = [_norm(s).to(s.x.dtype)]
        return y + _norm_gradients(s) if kind == "norm-train" else y
    x = s.x.float()
    if kind == "half":
        s.residual = s.x
        return [_forward(s, _norm(s))[0]]
    y, z, h = _forward(s, x)
    return [y] + _gradients(s, x, z, h) if s.dy is not None else [y]


# ---- the same from the definition, in 64 bits, gradients by torch's own differentiation ----

def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    kind, act = case["kind"], case["act"]
    F = torch.nn.functional
    train = kind.endswith("-train")
    wide = lambda t: None if t is None else t.double().requires_grad_(train)   # noqa: E731
    x, w, b, w_in, w_out, b_in, b_out = (wide(t) for t in (s.x, s.w, s.b, s.w_in, s.w_out, s.b_in, s.b_out))
    apply = {"none": lambda v: v, "silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda v: F.gelu(v, approximate="tanh")}[act]
    take = lambda t: t if s.index is None or t.dim() == 1 or t.shape[0] == 1 else t.index_select(0, s.index.long())   # noqa: E731
    y, leaves = x, [x]
    if kind.startswith("norm") or kind == "half":
        y = F.layer_norm(x, (case["width"],), eps=EPS)
        if w is not None:
            y = y * take(w) + take(b)
            leaves += [w, b]
    if not kind.startswith("norm"):
        y = F.linear(y, w_in, b_in)
        leaves = [x, w_in]
        if case["gated"]:
            value, gate = y.chunk(2, 1)
            y = value * apply(gate)
        else:
            y = apply(y)
        if w_out is not None:
            y = F.linear(y, w_out, b_out)
            leaves.append(w_out)
        leaves += [t for t in (b_in, b_out) if t is not None]
        if s.gate is not None:
            y = y * take(s.gate.double())
        residual = s.x if kind == "half" else s.residual
        if residual is not None:
            y = y + residual.double()
    got = [y.detach()]
    if train:
        got += list(torch.autograd.grad(y, leaves, s.dy.double()))
    return got
