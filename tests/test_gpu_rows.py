"""Layer norm, products with their epilogues and the feed-forward block against their formulas in float64 (oracle/rows_oracle.py), every element against
the bound that follows from the roundings on its way."""
import math

import pytest
import torch

import pika_h3_flex_amd as pk
from oracle import rows_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
ACTIVATIONS = ("none", "silu", "gelu", "gelu_tanh")


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, *shape, scale=1.0, dtype=BF16):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def _within(got, want, what=""):
    y, bound = want
    assert got.shape == y.shape, (what, got.shape, y.shape)
    off = (got.double() - y).abs()
    assert torch.isfinite(got).all(), what
    worst = (off / bound).max().item() if got.numel() else 0.0
    assert worst <= 1.0, (what, worst, off.max().item())


# ---- layer norm ----

def _norm_bound(x, y, weight, bias, index, eps, dtype):
    """Sums over the width in float32 (mean and squares), then a few roundings: 2 (width + 8) roundings of the largest normalised value of a row would be the worst of all
    orders of summation; the kernel adds up in a tree of depth log2(width) + 8, and the mean's error is of the row's magnitude."""
    width = x.shape[1]
    depth = math.log2(width) + 8 + width / 64
    xh, rstd = O.standard(x, eps)
    size = x.double().abs().mean(-1, keepdim=True) * rstd          # error of the mean in units of the deviation
    w = 1.0 if weight is None else O.take(weight, index, x.shape[0]).abs()
    b = 0.0 if bias is None else O.take(bias, index, x.shape[0]).abs()
    bound = 2 * O.HALF_F32 * (depth * (size + xh.abs()) * w + 2 * (xh.abs() * w + b))
    return bound + (O.HALF_BF16 if dtype is BF16 else O.HALF_F32) * (y.abs() + bound)


NORM_SHAPES = [(1, 8), (3, 16), (7, 248), (5, 512), (9, 520), (2, 1024), (66, 1032), (4, 2048), (3, 2056), (130, 4096), (2, 4104), (2, 8192), (3, 8200), (2, 16384)]


def _norm_inputs(rows, width, dtype, tables, table_type, seed=0):
    gen = _gen(seed)
    x = _randn(gen, rows, width, scale=1.5, dtype=F32) * (0.2 + 2 * torch.rand((rows, 1), generator=gen, device=DEV)) + torch.randn((rows, 1), generator=gen, device=DEV)
    shape = (tables, width) if tables > 1 else (width,)
    w, b = (_randn(gen, *shape, scale=0.5, dtype=F32) + 1).to(table_type), _randn(gen, *shape, scale=0.5, dtype=table_type)
    index = torch.randint(0, tables, (rows,), generator=gen, device=DEV, dtype=torch.int32) if tables > 1 else None
    return x.to(dtype), w, b, index, _randn(gen, rows, width, dtype=dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,width", NORM_SHAPES)
def test_layer_norm(rows, width, dtype):
    for tables, table_type in ((1, F32), (3, BF16)):
        x, w, b, index, _ = _norm_inputs(rows, width, dtype, tables, table_type, rows + width)
        for weight, bias in ((w, b), (w, None), (None, b), (None, None)):
            idx = index if weight is not None or bias is not None else None
            got = pk.layer_norm(x, weight, bias, row_index=idx, eps=1e-5)
            y = O.layer_norm(x, weight, bias, idx, 1e-5)
            assert got.dtype is dtype
            _within(got, (y, _norm_bound(x, y, weight, bias, idx, 1e-5, dtype)), (tables, weight is None, bias is None))


def _norm_grad_bounds(dy, x, w, index, want, eps):
    """float32 sums: dx as the norm's own bound, of the gradients' magnitudes; the tables' sums by the number of rows."""
    rows, width = x.shape
    xh, rstd = O.standard(x, eps)
    g = dy.double() if w is None else dy.double() * O.take(w, index, rows)
    unit = 2 * O.HALF_F32
    depth = math.log2(width) + 16 + width / 64
    size = x.double().abs().mean(-1, keepdim=True) * rstd
    e_xh = unit * depth * (size + xh.abs())
    m = (g * xh).abs().mean(-1, keepdim=True) + (g.abs() * e_xh).mean(-1, keepdim=True) / (unit * depth)
    e_dx = rstd * (unit * depth * (g.abs() + g.abs().mean(-1, keepdim=True) + (xh.abs() + 1) * m + xh.abs() * m) + e_xh * m)
    dx, dw, db = want
    e_dx = e_dx + (O.HALF_BF16 if x.dtype is BF16 else O.HALF_F32) * (dx.abs() + e_dx)
    e_dw = None if dw is None else O.table_sums((dy.double().abs() * (e_xh + unit * (rows + 2) * xh.abs())), index, dw) + unit
    e_db = None if db is None else O.table_sums(dy.double().abs() * unit * (rows + 2), index, db) + unit
    return e_dx, e_dw, e_db


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,width", NORM_SHAPES + [(1, 1024), (17, 640), (200, 264), (1500, 72)])
def test_layer_norm_backward(rows, width, dtype):
    for tables, table_type in ((1, BF16), (3, F32)):
        x, w, b, index, dy = _norm_inputs(rows, width, dtype, tables, table_type, rows + width + 1)
        for weight, bias in ((w, b), (w, None), (None, None)):
            idx = index if weight is not None else None
            got = pk.layer_norm_backward(dy, x, weight, bias, row_index=idx, eps=1e-5)
            want = O.layer_norm_backward(dy, x, weight, bias, idx, 1e-5)
            bounds = _norm_grad_bounds(dy, x, weight, idx, want, 1e-5)
            for name, a, y, e in zip(("dx", "dweight", "dbias"), got, want, bounds):
                assert (a is None) == (y is None)
                if a is not None:
                    assert a.dtype is (dtype if name == "dx" else F32)
                    _within(a, (y, e), (name, tables))


def test_layer_norm_tables_in_runs_and_out_of_range():
    """Table rows that come in runs, again after another, never, and indexes outside of the tables, which are brought into range."""
    rows, width, tables = 3001, 264, 5
    x, w, b, _, dy = _norm_inputs(rows, width, BF16, tables, F32, 5)
    for kind in ("runs", "again", "wild"):
        i = torch.arange(rows, device=DEV)
        index = {"runs": i * 3 // rows, "again": (i // 7) % 2 * 4, "wild": (i // 50) * 1000 - 20000}[kind].to(torch.int32)
        y = O.layer_norm(x, w, b, index)
        _within(pk.layer_norm(x, w, b, row_index=index), (y, _norm_bound(x, y, w, b, index, 1e-6, BF16)), kind)
        got = pk.layer_norm_backward(dy, x, w, b, row_index=index)
        want = O.layer_norm_backward(dy, x, w, b, index)
        for name, a, v, e in zip(("dx", "dweight", "dbias"), got, want, _norm_grad_bounds(dy, x, w, index, want, 1e-6)):
            _within(a, (v, e), (kind, name))
        again = pk.layer_norm_backward(dy, x, w, b, row_index=index)
        assert all(torch.equal(p, q) for p, q in zip(got, again))


def test_layer_norm_of_64_tables_and_constant_rows():
    rows, width = 700, 96
    x, w, b, index, dy = _norm_inputs(rows, width, F32, 64, F32, 6)
    x[3] = 2.5                                                    # no deviation: eps alone
    x[4] = 0.0
    want = O.layer_norm_backward(dy, x, w, b, index)
    for a, v, e in zip(pk.layer_norm_backward(dy, x, w, b, row_index=index), want, _norm_grad_bounds(dy, x, w, index, want, 1e-6)):
        _within(a, (v, e))
    y = O.layer_norm(x, w, b, index)
    _within(pk.layer_norm(x, w, b, row_index=index), (y, _norm_bound(x, y, w, b, index, 1e-6, F32)))


def test_layer_norm_strides_and_in_place():
    gen = _gen(7)
    wide = _randn(gen, 37, 640)
    x, out = wide[:, 64:384], torch.zeros(37, 384, dtype=BF16, device=DEV)[:, 8:328]
    want = pk.layer_norm(x.contiguous())
    assert torch.equal(pk.layer_norm(x, out=out), want) and out.data_ptr() % 16 == 0
    before = wide.clone()
    assert torch.equal(pk.layer_norm(x, out=x), want)
    assert torch.equal(wide[:, :64], before[:, :64]) and torch.equal(wide[:, 384:], before[:, 384:])


def test_layer_norm_of_values_that_are_not_finite():
    """A row with an infinity or a NaN is NaN; its neighbours are what they are."""
    x, w, b, _, dy = _norm_inputs(9, 264, BF16, 1, F32, 8)
    clean = pk.layer_norm(x, w, b)
    bad = x.clone()
    bad[2, 5], bad[6, 100] = math.inf, math.nan
    got = pk.layer_norm(bad, w, b)
    rows = [0, 1, 3, 4, 5, 7, 8]
    assert torch.equal(got[rows], clean[rows]) and got[[2, 6]].isnan().all()
    dx = pk.layer_norm_backward(dy, bad, w, b)[0]
    assert torch.equal(dx[rows], pk.layer_norm_backward(dy, x, w, b)[0][rows])


# ---- products ----

def _linear_inputs(rows, K, N, seed, table_type=F32):
    gen = _gen(seed)
    x, w = _randn(gen, rows, K), _randn(gen, N, K, scale=1.5 / math.sqrt(K))
    b = _randn(gen, N, scale=0.5, dtype=table_type)
    gate, index = _randn(gen, 3, N), torch.randint(-1, 4, (rows,), generator=gen, device=DEV, dtype=torch.int32)
    return x, w, b, gate, index, _randn(gen, rows, N)


LINEAR_SHAPES = [(1, 8, 8), (1, 1024, 264), (2, 40, 24), (3, 72, 1000), (15, 136, 520), (16, 512, 256), (17, 2048, 128), (33, 264, 648), (64, 1000, 512),
                 (65, 96, 136), (100, 4096, 64), (127, 328, 248), (129, 1032, 264), (255, 64, 2056), (257, 520, 512), (300, 11008, 96), (1085, 768, 776),
                 (2003, 200, 1288), (3, 72, 6200), (20, 2056, 6152), (50, 264, 6408)]


@pytest.mark.parametrize("rows,K,N", LINEAR_SHAPES)
def test_linear(rows, K, N):
    for i, name in enumerate(ACTIVATIONS):
        x, w, b, gate, index, residual = _linear_inputs(rows, K, N, rows + K + N + i, (F32, BF16)[i & 1])
        got, pre = pk.linear(x, w, b, activation=name, save=True)
        _within(got, O.linear(x, w, b, name), name)
        if name == "none":
            assert pre is None
        else:
            assert pre.dtype is F32
            _within(pre, O.first_product(x, w, b), "pre")
        assert torch.equal(pk.linear(x, w, b, activation=name), got)
        got = pk.linear(x, w, activation=name, gate=gate, row_index=index, residual=residual)
        _within(got, O.linear(x, w, None, name, gate, index, residual), (name, "gate, residual"))
    _within(pk.linear(x, w, b, gate=gate[:1], out=residual.clone()), O.linear(x, w, b, "none", gate[:1]))
    inplace = residual.clone()
    assert pk.linear(x, w, b, residual=inplace, out=inplace) is inplace
    _within(inplace, O.linear(x, w, b, "none", None, None, residual))


@pytest.mark.parametrize("rows,K,N", LINEAR_SHAPES)
def test_linear_backward(rows, K, N):
    for i, name in enumerate(ACTIVATIONS):
        x, w, b, _, _, dy = _linear_inputs(rows, K, N, rows + K + N + i + 9, (F32, BF16)[i & 1])
        _, pre = pk.linear(x, w, b, activation=name, save=True)
        got = pk.linear_backward(dy, x, w, pre, activation=name)
        for what, a, want in zip(("dx", "dweight", "dbias"), got, O.linear_backward(dy, x, w, b, name)):
            assert a.dtype is BF16
            _within(a, want, (name, what))
    some = pk.linear_backward(dy, x, w, pre, activation=name, weight_grad=False, bias_grad=False)
    assert some[1] is None and some[2] is None and torch.equal(some[0], got[0])


def _block_inputs(rows, width, inner, outputs, gated, seed, table_type=F32):
    gen = _gen(seed)
    first = 2 * inner if gated else inner
    x, w_in = _randn(gen, rows, width), _randn(gen, first, width, scale=1.5 / math.sqrt(width))
    w_out = _randn(gen, outputs, inner, scale=1.5 / math.sqrt(inner))
    return (x, w_in, w_out, _randn(gen, first, scale=0.5, dtype=table_type), _randn(gen, outputs, scale=0.5, dtype=table_type),
            _randn(gen, 3, outputs), torch.randint(0, 3, (rows,), generator=gen, device=DEV, dtype=torch.int32), _randn(gen, rows, outputs))


BLOCK_SHAPES = [(1, 8, 8, 8), (1, 512, 1376, 512), (2, 64, 200, 72), (5, 1024, 344, 1024), (16, 128, 512, 256), (31, 264, 712, 264), (64, 256, 1000, 136),
                (65, 512, 256, 512), (129, 136, 328, 400), (257, 320, 648, 320), (1085, 256, 680, 256)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,width,inner,outputs", BLOCK_SHAPES)
def test_feed_forward(rows, width, inner, outputs, gated):
    for i, name in enumerate(ACTIVATIONS):
        x, w_in, w_out, b_in, b_out, gate, index, residual = _block_inputs(rows, width, inner, outputs, gated, rows + width + inner + i, (BF16, F32)[i & 1])
        _within(pk.feed_forward(x, w_in, w_out, activation=name, gated=gated), O.feed_forward(x, w_in, w_out, None, None, name, gated), name)
        got = pk.feed_forward(x, w_in, w_out, b_in, b_out, activation=name, gated=gated, gate=gate, row_index=index, residual=residual)
        _within(got, O.feed_forward(x, w_in, w_out, b_in, b_out, name, gated, gate, index, residual), (name, "gate, residual"))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,width,inner,outputs", BLOCK_SHAPES)
def test_feed_forward_backward(rows, width, inner, outputs, gated):
    for i, name in enumerate(ACTIVATIONS):
        x, w_in, w_out, b_in, b_out, _, _, dy = _block_inputs(rows, width, inner, outputs, gated, rows + width + inner + i + 5, (BF16, F32)[i & 1])
        y, saved = pk.feed_forward(x, w_in, w_out, b_in, b_out, activation=name, gated=gated, save=True)
        got = pk.feed_forward_backward(dy, x, w_in, w_out, saved, activation=name, gated=gated)
        for what, a, want in zip(("dx", "dw_in", "dw_out", "db_in", "db_out"), got, O.feed_forward_backward(dy, x, w_in, w_out, b_in, b_out, name, gated)):
            _within(a, want, (name, what))
        again = pk.feed_forward_backward(dy, x, w_in, w_out, saved, activation=name, gated=gated)
        assert all(torch.equal(p, q) for p, q in zip(got, again))


def test_no_rows():
    x, w_in, w_out, b_in, b_out, *_ = _block_inputs(4, 64, 128, 72, True, 1)
    none = x[:0]
    y, saved = pk.feed_forward(none, w_in, w_out, b_in, b_out, save=True)
    assert y.shape == (0, 72)
    dx, *rest = pk.feed_forward_backward(y, none, w_in, w_out, saved)
    assert dx.shape == (0, 64) and all(torch.count_nonzero(t) == 0 for t in rest)
    assert pk.linear(none, w_in).shape == (0, 256) and pk.layer_norm(none).shape == (0, 64)
    dx, dw, db = pk.linear_backward(torch.empty(0, 256, dtype=BF16, device=DEV), none, w_in)
    assert torch.count_nonzero(dw) == 0 and torch.count_nonzero(db) == 0 and dw.shape == w_in.shape
    weight = torch.ones(64, device=DEV)
    dx, dw, db = pk.layer_norm_backward(none, none, weight, weight)
    assert torch.count_nonzero(dw) == 0 and torch.count_nonzero(db) == 0


def test_rows_behind_a_matrix_are_not_written_and_what_lies_there_is_not_read():
    """Operands and results are slices of larger buffers full of NaN: nothing of it reaches a result, and nothing around a result changes."""
    gen = _gen(3)
    for rows, K, N in ((1, 40, 24), (13, 72, 136), (70, 264, 520), (131, 1032, 264), (300, 328, 392)):
        def framed(r, c):
            big = torch.full((r + 5, c + 24), math.nan, dtype=BF16, device=DEV)
            view = big[2:2 + r, 8:8 + c]
            view.copy_(_randn(gen, r, c))
            return big, view
        (_, x), (_, w), (_, dy) = framed(rows, K), framed(N, K), framed(rows, N)
        big, out = framed(rows, N)
        frame = torch.ones_like(big, dtype=torch.bool)
        frame[2:2 + rows, 8:8 + N] = False
        pk.linear(x, w, out=out)
        assert torch.equal(out, pk.linear(x.contiguous(), w.contiguous())) and big[frame].isnan().all()
        _within(out, O.linear(x, w))
        pre = pk.linear(x, w, activation="silu", save=True)[1]
        for a, b in zip(pk.linear_backward(dy, x, w, pre, activation="silu"), pk.linear_backward(dy.contiguous(), x.contiguous(), w.contiguous(), pre, activation="silu")):
            assert torch.equal(a, b) and a.isfinite().all()


def test_gradients_against_differences():
    """A sum over the results, differentiated by steps along random directions in float64 on the formulas, against the kernels' gradients: as far as their own bounds reach."""
    x, w_in, w_out, b_in, b_out, _, _, dy = _block_inputs(23, 72, 136, 64, True, 77)
    args = [t.double() for t in (x, w_in, w_out, b_in, b_out)]

    def loss(parts):
        z = parts[0] @ parts[1].t() + parts[3]
        a, b = z.chunk(2, 1)
        y = (a * torch.nn.functional.silu(b)) @ parts[2].t() + parts[4]
        return (y * dy.double()).sum()

    _, saved = pk.feed_forward(x, w_in, w_out, b_in, b_out, save=True)
    got = pk.feed_forward_backward(dy, x, w_in, w_out, saved)
    bounds = O.feed_forward_backward(dy, x, w_in, w_out, b_in, b_out)
    gen = _gen(78)
    for i in range(5):
        way = torch.randn(args[i].shape, generator=gen, device=DEV, dtype=torch.float64)
        step = 1e-5
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + step * way, args[i] - step * way
        slope = (loss(up) - loss(down)) / (2 * step)
        mine = (got[i].double() * way).sum()
        assert (slope - mine).abs() <= (bounds[i][1] * way.abs()).sum() + 1e-6 * slope.abs(), i


# ---- a run of them together, differentiation, streams, graphs ----

def _half_block(x, p):
    y = pk.layer_norm(x, p["weight"], p["bias"])
    return pk.feed_forward(y, p["w_in"], p["w_out"], p["b_in"], p["b_out"], residual=x)


def _half_block_parts(rows=150, width=264, inner=344, seed=11):
    x, w_in, w_out, b_in, b_out, *_ , dy = _block_inputs(rows, width, inner, width, True, seed)
    gen = _gen(seed + 1)
    p = dict(weight=1 + 0.3 * torch.randn(width, generator=gen, device=DEV), bias=0.3 * torch.randn(width, generator=gen, device=DEV), w_in=w_in, w_out=w_out,
             b_in=b_in, b_out=b_out.to(BF16))
    return x, p, dy


def test_half_a_block_together():
    x, p, _ = _half_block_parts()
    got = _half_block(x, p)
    # the norm's result is rounded to bfloat16: what that does to the block comes on top of the block's own bound
    y = O.layer_norm(x, p["weight"], p["bias"])
    y16 = pk.layer_norm(x, p["weight"], p["bias"])
    _within(y16, (y, _norm_bound(x, y, p["weight"], p["bias"], None, 1e-6, BF16)))
    _within(got, O.feed_forward(y16, p["w_in"], p["w_out"], p["b_in"], p["b_out"], residual=x))


def test_differentiation_gives_the_backward_passes():
    x, p, dy = _half_block_parts()
    leaf = x.clone().requires_grad_()
    parts = {k: v.clone().requires_grad_() for k, v in p.items()}
    out = _half_block(leaf, parts)
    assert torch.equal(out.detach(), _half_block(x, p))
    out.backward(dy)
    y = pk.layer_norm(x, p["weight"], p["bias"])
    _, saved = pk.feed_forward(y, p["w_in"], p["w_out"], p["b_in"], p["b_out"], residual=x, save=True)
    dy1, dw_in, dw_out, db_in, db_out = pk.feed_forward_backward(dy, y, p["w_in"], p["w_out"], saved)
    dx, dw, db = pk.layer_norm_backward(dy1, x, p["weight"], p["bias"])
    want = dict(weight=dw, bias=db, w_in=dw_in, w_out=dw_out, b_in=db_in.float(), b_out=db_out)
    for name, t in want.items():
        assert torch.equal(parts[name].grad, t) and parts[name].grad.dtype == parts[name].dtype, name
    assert torch.equal(leaf.grad, dx + dy)
    # frozen weights: only what is asked for
    leaf.grad = None
    _half_block(leaf, p).sum().backward()
    assert leaf.grad.isfinite().all()
    z = pk.linear(leaf, parts["w_in"], parts["b_in"], activation="gelu", residual=None)
    assert z.requires_grad
    with torch.no_grad():
        assert not pk.linear(leaf, parts["w_in"]).requires_grad


def test_calls_on_another_stream_and_captured():
    x, p, dy = _half_block_parts(rows=77)
    index = torch.zeros(77, dtype=torch.int32, device=DEV)

    def step():
        y = pk.layer_norm(x, p["weight"], p["bias"], row_index=index)
        z, saved = pk.feed_forward(y, p["w_in"], p["w_out"], p["b_in"], p["b_out"], residual=x, save=True)
        return [z, *pk.feed_forward_backward(dy, y, p["w_in"], p["w_out"], saved), *pk.layer_norm_backward(dy, x, p["weight"], p["bias"])]

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        x.copy_(_randn(_gen(100 + i), *x.shape))
        dy.copy_(_randn(_gen(200 + i), *dy.shape))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step())), i
