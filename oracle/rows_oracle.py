"""Layer norm with tables, products with their epilogues and the feed-forward block in float64, forward and backward, written out from the formulas; beside
every result how far a computation may be off that sums in float32 and rounds to bfloat16 where the operators do (``bound``: per element)."""
import math

import torch

HALF_BF16 = 2.0 ** -8      # largest relative error of a rounding to bfloat16
HALF_F32 = 2.0 ** -24
# largest |f''| of the activations, for what an error of a saved value does to f'(v): |silu''| <= 1/2 (at 0), |gelu''| = (2 - v^2) phi(v) <= 2 phi(0) < 0.8, and its
# tanh form's is within 0.03 of that
CURVATURE = {"none": 0.0, "silu": 0.5, "gelu": 0.8, "gelu_tanh": 0.83}
SLOPE = {"none": 1.0, "silu": 1.1, "gelu": 1.13, "gelu_tanh": 1.13}      # largest |f'|
_TANH = math.sqrt(2.0 / math.pi)


def act(name, v):
    if name == "none":
        return v
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * torch.special.erfc(-v / math.sqrt(2.0))
    return v * torch.sigmoid(2.0 * _TANH * (v + 0.044715 * v ** 3))


def act_slope(name, v):
    if name == "none":
        return torch.ones_like(v)
    if name == "silu":
        s = torch.sigmoid(v)
        return s * (1.0 + v * (1.0 - s))
    if name == "gelu":
        return 0.5 * torch.special.erfc(-v / math.sqrt(2.0)) + v * torch.exp(-0.5 * v * v) / math.sqrt(2.0 * math.pi)
    s = torch.sigmoid(2.0 * _TANH * (v + 0.044715 * v ** 3))
    return s + v * s * (1.0 - s) * 2.0 * _TANH * (1.0 + 3 * 0.044715 * v * v)


def take(table, index, rows):
    """[rows, n]: each row's table row (indexes brought into range)."""
    t = table.double().reshape(-1, table.shape[-1])
    i = torch.zeros(rows, dtype=torch.int64, device=t.device) if index is None else index.long().clamp(0, t.shape[0] - 1)
    return t[i]


def standard(x, eps):
    x = x.double()
    d = x - x.mean(-1, keepdim=True)
    rstd = (d.square().mean(-1, keepdim=True) + eps).rsqrt()
    return d * rstd, rstd


def layer_norm(x, weight=None, bias=None, index=None, eps=1e-6):
    y, _ = standard(x, eps)
    if weight is not None:
        y = y * take(weight, index, x.shape[0])
    return y if bias is None else y + take(bias, index, x.shape[0])


def table_sums(rows, index, like):
    """Sums of the rows of each table row, in the shape of the table."""
    n = like.numel() // like.shape[-1]
    i = torch.zeros(rows.shape[0], dtype=torch.int64, device=rows.device) if index is None else index.long().clamp(0, n - 1)
    return torch.zeros(n, rows.shape[-1], dtype=rows.dtype, device=rows.device).index_add_(0, i, rows).reshape(like.shape)


def layer_norm_backward(dy, x, weight=None, bias=None, index=None, eps=1e-6):
    xh, rstd = standard(x, eps)
    dy = dy.double()
    g = dy if weight is None else dy * take(weight, index, x.shape[0])
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return dx, None if weight is None else table_sums(dy * xh, index, weight), None if bias is None else table_sums(dy, index, bias)


def product(a, b):
    """(a b^T, bound): sums of K products in float32, in whatever order, are off by at most K + 1 roundings of the sum of magnitudes."""
    a, b = a.double(), b.double()
    return a @ b.t(), (a.shape[1] + 1) * 2 * HALF_F32 * (a.abs() @ b.abs().t())


def rounded(y, bound):
    return y, bound + HALF_BF16 * (y.abs() + bound) + 1e-30


def act_error(name, v):
    """How far an activation in float32 is off: 2e-6 of the value and, far out, 1e-37.  On the negative side it is exp(-E) in the main, E = |v|, v^2 / 2 or 2 |u| (u the tanh form's), and
    an exponent with up to five roundings on its way (constants, squares, products, the difference) is off by 5 * 2^-24 E, and so is the value, relative to itself."""
    if name == "none":
        return torch.zeros_like(v)
    far = {"silu": -v, "gelu": 0.5 * v * v, "gelu_tanh": -2.0 * _TANH * (v + 0.044715 * v ** 3)}[name]
    return act(name, v).abs() * (2e-6 + 5 * HALF_F32 * torch.where(v < 0, far, torch.zeros_like(v)).clamp(max=90.0)) + 1e-37


def finish(z, bound, name, gate=None, index=None, residual=None):
    """Activation (its own error: act_error), gate and residual; rounded."""
    y = act(name, z)
    bound = bound * SLOPE[name] + act_error(name, z)
    if gate is not None:
        g = take(gate, index, z.shape[0])
        y, bound = y * g, bound * g.abs() + 2 * HALF_F32 * (y * g).abs()
    if residual is not None:
        y, bound = y + residual.double(), bound + 2 * HALF_F32 * (y.abs() + residual.double().abs())
    return rounded(y, bound)


def first_product(x, w, b):
    z, e = product(x, w)
    if b is not None:
        z = z + b.double()
        e = e + 2 * HALF_F32 * z.abs()
    return z, e


def linear(x, w, b=None, name="none", gate=None, index=None, residual=None):
    """(result, bound)"""
    return finish(*first_product(x, w, b), name, gate, index, residual)


def middle(x, w_in, b_in, name, gated):
    """(h, its bound, the first product, its bound), h rounded to bfloat16."""
    z, e = first_product(x, w_in, b_in)
    if not gated:
        h, eh = finish(z, e, name)
        return h, eh, z, e
    a, b = z.chunk(2, 1)
    ea, eb = e.chunk(2, 1)
    f = act(name, b)
    ef = eb * SLOPE[name] + act_error(name, b)
    h, eh = rounded(a * f, ea * f.abs() + (a.abs() + ea) * ef + 2 * HALF_F32 * (a * f).abs())
    return h, eh, z, e


def feed_forward(x, w_in, w_out, b_in=None, b_out=None, name="silu", gated=True, gate=None, index=None, residual=None):
    h, eh, _, _ = middle(x, w_in, b_in, name, gated)
    y, _ = first_product(h, w_out, b_out)
    w = w_out.double().abs()
    e = eh @ w.t() + (h.shape[1] + 2) * 2 * HALF_F32 * ((h.abs() + eh) @ w.t()) + 2 * HALF_F32 * y.abs()
    return finish(y, e, "none", gate, index, residual)


def _grad(sum_, e, z, ez, name):
    """sum * act'(z) from a saved z: (value, bound) before its own rounding."""
    slope = act_slope(name, z)
    es = CURVATURE[name] * ez + (4e-6 * (1 + z.abs()) if name != "none" else 0.0)
    v = sum_ * slope
    return v, e * (slope.abs() + es) + sum_.abs() * es + 2 * HALF_F32 * v.abs()


def _times(a, ea, b, eb=None):
    """(a^T b, bound) of values that are off by ea and eb already."""
    k = a.shape[0]
    b = b.double()
    eb = torch.zeros_like(b) if eb is None else eb
    y = a.t() @ b
    big_a, big_b = a.abs() + ea, b.abs() + eb
    return rounded(y, ea.t() @ big_b + a.abs().t() @ eb + (k + 1) * 2 * HALF_F32 * (big_a.t() @ big_b))


def _sums(v, e):
    return rounded(v.sum(0), e.sum(0) + (v.shape[0] + 1) * 2 * HALF_F32 * (v.abs() + e).sum(0))


def linear_backward(dy, x, w, b=None, name="none"):
    """[(dx, bound), (dw, bound), (db, bound)]"""
    z, ez = first_product(x, w, b)
    dz, e = _grad(dy.double(), torch.zeros_like(z), z, ez, name)
    db = _sums(dz, e)
    if name != "none":
        dz, e = rounded(dz, e)
    dx = _times(dz.t().contiguous(), e.t().contiguous(), w)
    return [dx, _times(dz, e, x), db]


def feed_forward_backward(dy, x, w_in, w_out, b_in=None, b_out=None, name="silu", gated=True):
    """[(dx, bound), (dw_in, bound), (dw_out, bound), (db_in, bound), (db_out, bound)]"""
    h, eh, z, ez = middle(x, w_in, b_in, name, gated)
    dy = dy.double()
    zero = torch.zeros_like(dy)
    dh, e = product(dy, w_out.t().contiguous())
    if gated:
        a, b = z.chunk(2, 1)
        ea, eb = ez.chunk(2, 1)
        f = act(name, b)
        ef = SLOPE[name] * eb + 2 * act_error(name, b)
        da, e_da = dh * f, e * (f.abs() + ef) + dh.abs() * ef + 2 * HALF_F32 * (dh * f).abs()
        p = dh * a
        ep = e * (a.abs() + ea) + dh.abs() * ea
        slope = act_slope(name, b)
        es = CURVATURE[name] * eb + (4e-6 * (1 + b.abs()) if name != "none" else 0.0)
        db, e_db = p * slope, ep * (slope.abs() + es) + p.abs() * es + 4 * HALF_F32 * (p * slope).abs()
        dz, e = torch.cat([da, db], 1), torch.cat([e_da, e_db], 1)
    else:
        dz, e = _grad(dh, e, z, ez, name)
    db_in = _sums(dz, e)
    dz, e = rounded(dz, e)
    dx = _times(dz.t().contiguous(), e.t().contiguous(), w_in)
    return [dx, _times(dz, e, x), _times(dy, zero, h, eh), db_in, _sums(dy, zero)]
