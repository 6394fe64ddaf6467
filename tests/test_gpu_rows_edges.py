"""Layer norm, products and the feed-forward block where calls go wrong: offsets that pass 32 bits, values that are not finite, framed operands of every form of the products,
two streams at once, graphs, several devices' rules, far ends of the activations."""
import math

import pytest
import torch

import pika_h3_flex_amd as pk

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
ACTIVATIONS = ("none", "silu", "gelu", "gelu_tanh")


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, *shape, scale=1.0, dtype=BF16):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def _equal(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0.0, math.inf, -math.inf), b.nan_to_num(0.0, math.inf, -math.inf))


# rows, K, N: the few-row form in its three heights, tiles of 64, 128 and 256 rows, whole and with the contraction cut, ends of a contraction that are no whole chunk
FORMS = [(1, 1000, 264), (13, 2056, 136), (40, 520, 1032), (130, 1032, 264), (300, 328, 392), (1085, 4104, 1544), (2003, 1400, 5160), (4100, 1032, 4104)]


@pytest.mark.parametrize("rows,K,N", FORMS)
def test_framed_operands_of_every_form(rows, K, N):
    """Every operand and result a slice of a buffer full of NaN: the results are those of the operands by themselves, and finite; nothing around a result changes."""
    gen = _gen(rows)

    def framed(r, c, fill=True):
        big = torch.full((r + 5, c + 24), math.nan, dtype=BF16, device=DEV)
        view = big[2:2 + r, 8:8 + c]
        if fill:
            view.copy_(_randn(gen, r, c, scale=c ** -0.25))
        return big, view

    (_, x), (_, w), (_, dy), (_, residual), (_, gate) = framed(rows, K), framed(N, K), framed(rows, N), framed(rows, N), framed(3, N)
    index = torch.randint(0, 3, (rows,), generator=gen, device=DEV, dtype=torch.int32)
    bias = _randn(gen, N, dtype=F32)
    big, out = framed(rows, N, fill=False)
    frame = torch.ones_like(big, dtype=torch.bool)
    frame[2:2 + rows, 8:8 + N] = False
    args = dict(bias=bias, activation="gelu_tanh", row_index=index)
    pk.linear(x, w, gate=gate, residual=residual, out=out, **args)
    xc, wc, dyc = x.contiguous(), w.contiguous(), dy.contiguous()
    want = pk.linear(xc, wc, gate=gate.contiguous(), residual=residual.contiguous(), **args)
    assert torch.equal(out, want) and out.isfinite().all() and big[frame].isnan().all()
    # in place of its residual
    pk.linear(x, w, gate=gate, residual=residual, out=residual, **args)
    assert torch.equal(residual, want)
    pre = pk.linear(x, w, activation="silu", save=True)[1]
    for a, b in zip(pk.linear_backward(dy, x, w, pre, activation="silu"), pk.linear_backward(dyc, xc, wc, pre, activation="silu")):
        assert torch.equal(a, b) and a.isfinite().all()
    # gated, with the block's own backward products
    half = N // 16 * 8
    w_out = framed(K, half)[1]
    z, saved = pk.feed_forward(x, w[:2 * half], w_out, save=True)
    zc, saved_c = pk.feed_forward(xc, wc[:2 * half], w_out.contiguous(), save=True)
    assert torch.equal(z, zc) and torch.equal(saved.pre, saved_c.pre) and z.isfinite().all()
    back = framed(rows, K)[1]
    for a, b in zip(pk.feed_forward_backward(back, x, w[:2 * half], w_out, saved), pk.feed_forward_backward(back.contiguous(), xc, wc[:2 * half], w_out.contiguous(), saved_c)):
        assert torch.equal(a, b) and a.isfinite().all()


@pytest.mark.parametrize("rows,K,N", [(1, 1000, 264), (40, 520, 264), (130, 1032, 264), (1085, 2056, 1544)])
def test_values_that_are_not_finite_stay_in_their_row_and_column(rows, K, N):
    gen = _gen(rows + 1)
    x, w = _randn(gen, rows, K), _randn(gen, N, K, scale=K ** -0.5)
    clean = pk.linear(x, w)
    r, k, n = rows // 2, K - 1, N // 3
    x2, w2 = x.clone(), w.clone()
    x2[r, k] = math.inf
    got = pk.linear(x2, w)
    others = torch.arange(rows, device=DEV) != r
    assert torch.equal(got[others], clean[others])
    assert torch.equal(got[r].float(), torch.sign(w[:, k].float()) * math.inf)          # (no weight is zero)
    w2[n, 0] = math.nan
    got = pk.linear(x, w2)
    columns = torch.arange(N, device=DEV) != n
    assert torch.equal(got[:, columns], clean[:, columns]) and got[:, n].isnan().all()
    # the same for the products of the backward pass
    dy = _randn(gen, rows, N)
    dx, dw, db = pk.linear_backward(dy, x, w)
    dy2 = dy.clone()
    dy2[r, n] = math.nan
    dx2, dw2, db2 = pk.linear_backward(dy2, x, w)
    assert torch.equal(dx2[others], dx[others]) and dx2[r].isnan().all()
    assert torch.equal(dw2[columns], dw[columns]) and dw2[n].isnan().all()
    assert torch.equal(db2[columns], db[columns]) and db2[n].isnan()


def test_far_ends_of_the_activations_and_their_slopes():
    """Sums of any size that float32 holds: the values and slopes are those of the limits, never 0 times infinity."""
    far = torch.tensor([3e38, 1e25, 1e19, 1e5, 100.0, -100.0, -1e5, -1e19, -1e25, -3e38], device=DEV)
    z = far.repeat(8, 1)[:, :8].contiguous(), far.flip(0).repeat(8, 1)[:, :8].contiguous()
    eye = torch.eye(8, device=DEV, dtype=BF16)
    dy = torch.ones(8, 8, device=DEV, dtype=BF16)
    for name in ACTIVATIONS[1:]:
        for pre in z:
            dx, _, _ = pk.linear_backward(dy, dy, eye, pre, activation=name)
            want = (pre > 0).to(BF16)
            assert torch.equal(dx, want), (name, pre[0], dx[0])
            y = pk.linear(pre.to(BF16), eye, activation="none")
            got = pk.linear(y.clamp(-3e38, 3e38), eye, activation=name)
            big = y.float().abs() >= 1e5
            assert torch.equal(got[big].float(), y[big].float().clamp(min=0)), name


def test_offsets_that_pass_32_bits():
    """Rows 8 MiB apart, the largest stride: 1,100 of them lie over 9 GiB.  The results are those of the rows beside each other."""
    rows, K, N, stride = 1100, 136, 264, 1 << 22
    gen = _gen(5)
    buffers = [torch.empty(rows * stride, dtype=BF16, device=DEV).view(rows, stride) for _ in range(3)]
    x, dy, out = buffers[0][:, stride - K:], buffers[1][:, :N], buffers[2][:, 8:8 + N]
    x.copy_(_randn(gen, rows, K)), dy.copy_(_randn(gen, rows, N))
    xc, dyc = x.contiguous(), dy.contiguous()
    w = _randn(gen, N, K)
    assert torch.equal(pk.linear(x, w, residual=dy, out=out), pk.linear(xc, w, residual=dyc))
    assert torch.equal(pk.linear(x[-5:], w), pk.linear(xc[-5:], w))
    for a, b in zip(pk.linear_backward(dy, x, w), pk.linear_backward(dyc, xc, w)):
        assert torch.equal(a, b)
    # weights' rows as far apart, along and across, and the layer norm's rows
    far_w = buffers[2][:N, 512:512 + K]
    far_w.copy_(w)
    assert torch.equal(pk.linear(xc, far_w), pk.linear(xc, w)) and torch.equal(pk.linear(xc[:3], far_w), pk.linear(xc[:3], w))
    assert torch.equal(pk.linear_backward(dyc, xc, far_w)[0], pk.linear_backward(dyc, xc, w)[0])
    weight, bias = 1 + _randn(gen, K, dtype=F32), _randn(gen, K, dtype=F32)
    slot = buffers[1][:, 1024:1024 + K]
    assert torch.equal(pk.layer_norm(x, weight, bias, out=slot), pk.layer_norm(xc, weight, bias))
    for a, b in zip(pk.layer_norm_backward(slot, x, weight, bias), pk.layer_norm_backward(slot.contiguous(), xc, weight, bias)):
        assert torch.equal(a, b)


def test_float32_sums_kept_beyond_4_gib():
    """The saved sums of a block whose offsets pass 32 bits, read back by the backward pass: rows at the end against the same rows by themselves."""
    rows, width, inner = 70_000, 64, 8192
    gen = _gen(6)
    x, w_in, w_out = _randn(gen, rows, width), _randn(gen, 2 * inner, width, scale=0.2), _randn(gen, width, inner, scale=0.02)
    y, saved = pk.feed_forward(x, w_in, w_out, save=True)
    assert saved.pre.numel() * 4 > 1 << 32
    last = slice(rows - 4096, rows)
    # a row's sums depend on its own row alone, in the order of the contraction, which is one chunk here
    few, saved_few = pk.feed_forward(x[last], w_in, w_out, save=True)
    assert torch.equal(saved.pre[last], saved_few.pre) and torch.equal(saved.hidden[last], saved_few.hidden)
    dy = _randn(gen, rows, width)
    dx = pk.feed_forward_backward(dy, x, w_in, w_out, saved, weight_grad=False, bias_grad=False)[0]
    want = pk.feed_forward_backward(dy[last], x[last], w_in, w_out, saved_few, weight_grad=False, bias_grad=False)[0]
    # the contraction of 16,384 may be cut elsewhere in the smaller call: two orders of the same float32 sum, then one rounding each
    off = (dx[last].float() - want.float()).abs()
    assert (off <= 2 * torch.finfo(BF16).eps * want.float().abs() + 1e-3 * want.float().abs().max()).all()


def test_two_streams_at_once():
    """Two streams with work of their own, cut contractions and column sums among it, whose workspaces must not meet."""
    gen = _gen(7)
    sets = []
    for i in range(2):
        x, w_in, w_out = _randn(gen, 302, 1032), _randn(gen, 2 * 1544, 1032, scale=0.03), _randn(gen, 1032, 1544, scale=0.03)
        sets.append((x, w_in, w_out, _randn(gen, 302, 1032), 1 + _randn(gen, 1032, dtype=F32), _randn(gen, 1032, dtype=F32)))

    def step(x, w_in, w_out, dy, weight, bias):
        y = pk.layer_norm(x, weight, bias)
        z, saved = pk.feed_forward(y, w_in, w_out, save=True)
        back = pk.feed_forward_backward(dy, y, w_in, w_out, saved)
        return [z, *back, *pk.layer_norm_backward(back[0], x, weight, bias)]

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(6):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(step(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i]))


def test_two_graphs_replayed_in_turn():
    """Two captured steps of different sizes, replayed in turn with eager work between them."""
    gen = _gen(8)
    sets = [(_randn(gen, rows, 520), _randn(gen, 264, 520, scale=0.05), _randn(gen, rows, 264)) for rows in (302, 77)]

    def step(x, w, dy):
        y, pre = pk.linear(x, w, activation="gelu", save=True)
        return [y, *pk.linear_backward(dy, x, w, pre, activation="gelu")]

    graphs, held = [], []
    for s in sets:
        step(*s)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step(*s))
    for i in range(6):
        for s, graph, mine in zip(sets, graphs, held):
            s[0].copy_(_randn(gen, *s[0].shape))
            s[2].copy_(_randn(gen, *s[2].shape))
            graph.replay()
            want = step(*s)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(mine, want)), i


def test_recorded_gradients_are_refused_in_a_capture():
    x, w = _randn(_gen(9), 16, 64), _randn(_gen(10), 64, 64).requires_grad_()
    pk.linear(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: pk.linear(x, w), lambda: pk.feed_forward(x, w, w, gated=False), lambda: pk.layer_norm(x, w[0])):
            with pytest.raises(RuntimeError, match="captured"):
                call()
        with torch.no_grad():
            y = pk.linear(x, w)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, pk.linear(x, w.detach()))


def test_gradients_of_too_many_tables_are_refused_at_once():
    tables = torch.ones(65, 64, device=DEV, requires_grad=True)
    index = torch.zeros(5, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="64 table rows"):
        pk.layer_norm(_randn(_gen(11), 5, 64), tables, row_index=index)
    assert pk.layer_norm(_randn(_gen(11), 5, 64), tables.detach(), row_index=index).isfinite().all()


def test_gradients_that_torch_hands_back_in_other_forms():
    """One value in all places, a transposed matrix, float32: each gives the gradients of the same matrix laid out in rows."""
    gen = _gen(12)
    x, w, b = _randn(gen, 40, 72), _randn(gen, 64, 72, scale=0.1), _randn(gen, 64, dtype=F32)

    def grads(dy_of):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = pk.linear(*leaves, activation="silu")
        y.backward(dy_of(y))
        return [t.grad for t in leaves]

    for make in (lambda y: torch.ones((), device=DEV, dtype=BF16).expand_as(y), lambda y: _randn(_gen(13), 64, 40).t()):
        want = grads(lambda y: make(y).contiguous())
        for a, c in zip(grads(make), want):
            assert torch.equal(a, c)
    # the same weight in both products, and an input used twice: torch adds the gradients up
    s = _randn(gen, 72, 72, scale=0.1).requires_grad_()
    leaf = x.clone().requires_grad_()
    pk.feed_forward(leaf, s, s, activation="gelu", gated=False, residual=leaf).sum().backward()
    ones = torch.ones(40, 72, device=DEV, dtype=BF16)
    with torch.no_grad():
        _, saved = pk.feed_forward(x, s, s, activation="gelu", gated=False, save=True)
        dx, d1, d2, _, _ = pk.feed_forward_backward(ones, x, s, s, saved, activation="gelu", gated=False)
    assert torch.equal(s.grad, d1 + d2) and torch.equal(leaf.grad, dx + ones)
