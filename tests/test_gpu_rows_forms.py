"""Every form of the products on plain rows against its formula (tests/rows_cases.py names them; tests/test_rows_forms_cpu.py holds that list against the plan).

The operands are small whole numbers times a power of two, so that every sum of their products is exact in float32, in whatever order: at most 4 * 12,000 < 2^24 of its units.  What is saved before
an activation, and results without one, then have to be equal to the last bit; behind an activation the bound counts its own error and the roundings.  Every matrix lies in
a larger one full of NaN, which must reach no result and stay as it is."""
import math

import pytest
import torch

import pika_h3_flex_amd as pk
from oracle import rows_oracle as O
from pika_h3_flex_amd import _lib
from pika_h3_flex_amd import rows as front
from tests.rows_cases import CASES

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
ACTIVATIONS = ("none", "silu", "gelu", "gelu_tanh")


class Framed:
    """A matrix in one full of NaN, 8 columns and 2 rows from its corner."""

    def __init__(self, values=None, shape=None, dtype=BF16):
        rows, cols = shape if values is None else values.shape
        self.big = torch.full((rows + 4, cols + 24), math.nan, dtype=dtype, device=DEV)
        self.view = self.big[2:2 + rows, 8:8 + cols]
        if values is not None:
            self.view.copy_(values)

    def at(self):
        return self.view.data_ptr(), self.view.stride(0)

    def frame_is_left(self):
        rows, cols = self.view.shape
        b = self.big
        return all(part.isnan().all() for part in (b[:2], b[2 + rows:], b[2:2 + rows, :8], b[2:2 + rows, 8 + cols:]))


def _whole(gen, *shape):
    """-2 .. 2"""
    return torch.randint(-2, 3, shape, generator=gen, device=DEV).to(BF16)


def _unit(K):
    """A power of two that brings a sum of K products of such numbers to about 1.5."""
    return 2.0 ** round(math.log2(1.5 / (2.0 * math.sqrt(K))))


def _equal(got, want, what):
    assert torch.equal(got, want.to(got.dtype)), (what, (got.double() - want.double()).abs().max().item(), (got != want.to(got.dtype)).sum().item())


def _within(got, want, what):
    y, bound = want
    assert got.isfinite().all(), what
    worst = ((got.double() - y).abs() / bound).max().item()
    assert worst <= 1.0, (what, worst)


def _case(kind):
    return pytest.mark.parametrize("tile,share,M,N,K", [c[1:] for c in CASES if c[0] == kind])


@_case("plain")
def test_plain(tile, share, M, N, K):
    gen = torch.Generator(device=DEV).manual_seed(M + N + K)
    unit = _unit(K)
    x, w = Framed(_whole(gen, M, K)), Framed(_whole(gen, N, K) * unit)
    bias = (torch.randint(-100, 101, (N,), generator=gen, device=DEV) * unit).float()
    gate, residual = Framed(torch.randn(3, N, generator=gen, device=DEV)), Framed(torch.randn(M, N, generator=gen, device=DEV))
    index = torch.randint(-1, 4, (M,), generator=gen, device=DEV, dtype=torch.int32)
    z = x.view.double() @ w.view.double().t() + bias.double()
    zero = torch.zeros((), dtype=torch.float64, device=DEV)
    out = Framed(shape=(M, N))
    for name in ACTIVATIONS:
        y, pre = pk.linear(x.view, w.view, bias, activation=name, out=out.view, save=True)
        if name == "none":
            _equal(y, z, "none")
        else:
            _equal(pre, z, "pre")
            _within(y, O.finish(z, zero, name), name)
        for g, r in ((gate, None), (None, residual), (gate, residual)):
            args = dict(activation=name, gate=None if g is None else g.view, row_index=None if g is None else index, residual=None if r is None else r.view)
            pk.linear(x.view, w.view, bias, out=out.view, **args)
            _within(out.view, O.finish(z, zero, name, None if g is None else g.view, index, None if r is None else r.view), (name, g is not None, r is not None))
    assert all(m.frame_is_left() for m in (x, w, gate, residual, out))


@_case("gated")
def test_gated(tile, share, M, N, K):
    gen = torch.Generator(device=DEV).manual_seed(M + N + K)
    unit = _unit(K)
    x, w = Framed(_whole(gen, M, K)), Framed(_whole(gen, 2 * N, K) * unit)
    bias = (torch.randint(-100, 101, (2 * N,), generator=gen, device=DEV) * unit).float()
    w_out = torch.zeros(8, N, dtype=BF16, device=DEV)
    z = x.view.double() @ w.view.double().t() + bias.double()
    a, b = z.chunk(2, 1)
    for name in ACTIVATIONS:
        _, saved = pk.feed_forward(x.view, w.view, w_out, bias, activation=name, save=True)
        _equal(saved.pre, z, "pre")
        f = O.act(name, b)
        _within(saved.hidden, O.rounded(a * f, a.abs() * O.act_error(name, b) + 2 * O.HALF_F32 * (a * f).abs()), name)
    assert x.frame_is_left() and w.frame_is_left()


@_case("dx")
def test_dx(tile, share, M, N, K):
    gen = torch.Generator(device=DEV).manual_seed(M + N + K)
    dy, w = Framed(_whole(gen, M, K)), Framed(_whole(gen, K, N) * _unit(K))
    dx, _, _ = pk.linear_backward(dy.view, torch.empty(M, N, dtype=BF16, device=DEV), w.view, weight_grad=False, bias_grad=False)
    _equal(dx, dy.view.double() @ w.view.double(), "dx")


@_case("dw")
def test_dw(tile, share, M, N, K):
    gen = torch.Generator(device=DEV).manual_seed(M + N + K)
    dy, x = Framed(_whole(gen, K, M)), Framed(_whole(gen, K, N) * _unit(K))
    _, dw, _ = pk.linear_backward(dy.view, x.view, torch.empty(M, N, dtype=BF16, device=DEV), x_grad=False, bias_grad=False)
    _equal(dw, dy.view.double().t() @ x.view.double(), "dw")


def _gradients(gen, M, N, K, wide, gated):
    """Arguments, the exact sums, and a call of the entry: f(activation, saved sums) -> (gradient, sums of its columns)"""
    dy, w = Framed(_whole(gen, M, K)), Framed(_whole(gen, K, N) * _unit(K))
    out, pre = Framed(shape=(M, wide)), Framed(shape=(M, wide), dtype=F32)
    sums = torch.full((wide + 16,), math.nan, dtype=BF16, device=DEV)
    flags = _lib.PRODUCT_B_ACROSS | _lib.PRODUCT_GRAD | (_lib.PRODUCT_GATED if gated else 0)

    def call(name, z):
        pre.view.copy_(z)
        front._product(dy.at(), w.at(), out.at(), M, N, K, flags, 0, pre=pre.at(), sums=sums[8:].data_ptr(), act=front.ACTIVATIONS[name])
        assert all(m.frame_is_left() for m in (dy, w, out, pre)) and sums[:8].isnan().all() and sums[8 + wide:].isnan().all()
        return out.view, sums[8:8 + wide]

    return dy.view.double() @ w.view.double(), call


def _exact_sums(v, unit):
    """Sums of columns whose partial sums are all whole multiples of ``unit`` below 2^24 of it."""
    assert (v / unit).abs().sum(0).max() < 1 << 24
    return v.sum(0)


@_case("grad")
def test_grad(tile, share, M, N, K):
    gen = torch.Generator(device=DEV).manual_seed(M + N + K)
    s, call = _gradients(gen, M, N, K, N, False)
    z = 2 * torch.randn(M, N, generator=gen, device=DEV)
    got, sums = call("none", z)
    _equal(got, s, "none")
    _equal(sums, _exact_sums(s, _unit(K)), "sums")
    for name in ACTIVATIONS[1:]:
        v, e = O._grad(s, torch.zeros_like(s), z.double(), 0.0, name)
        got, sums = call(name, z)
        _within(got, O.rounded(v, e), name)
        _within(sums, O._sums(v, e), name)


@_case("gated_grad")
def test_gated_grad(tile, share, M, N, K):
    gen = torch.Generator(device=DEV).manual_seed(M + N + K)
    s, call = _gradients(gen, M, N, K, 2 * N, True)
    z = _whole(gen, M, 2 * N).float()
    a, b = z.double().chunk(2, 1)
    got, sums = call("none", z)
    want = torch.cat([s * b, s * a], 1)
    _equal(got, want, "none")
    _equal(sums, _exact_sums(want, _unit(K)), "sums")
    z = 2 * torch.randn(M, 2 * N, generator=gen, device=DEV)
    a, b = z.double().chunk(2, 1)
    for name in ACTIVATIONS[1:]:
        f, slope = O.act(name, b), O.act_slope(name, b)
        da, p = s * f, s * a
        e_da = s.abs() * 2 * O.act_error(name, b) + 2 * O.HALF_F32 * da.abs()
        e_db = 4e-6 * (1 + b.abs()) * p.abs() + 4 * O.HALF_F32 * (p * slope).abs()
        v, e = torch.cat([da, p * slope], 1), torch.cat([e_da, e_db], 1)
        got, sums = call(name, z)
        _within(got, O.rounded(v, e), name)
        _within(sums, O._sums(v, e), name)
