"""Calls of the feed-forward half that its own documents allow and that went wrong once: see each test."""
import math

import pytest
import torch

import pika_h3_flex_amd as pk
from oracle import rows_oracle as O
from tests.test_gpu_rows import _norm_grad_bounds, _norm_inputs, _within

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
INF, NAN = math.inf, math.nan


def _same(got, want):
    got, want = got.float().cpu(), torch.as_tensor(want, dtype=torch.float32)
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0, INF, -INF), want.nan_to_num(0.0, INF, -INF))


@pytest.mark.parametrize("rows", [1, 40, 700])
def test_activations_of_infinities(rows):
    """An infinite sum: the activation of +inf is +inf; that of -inf is -inf * 0, NaN, and so is NaN's, as the formulas have it.  700 rows by 4,104 columns take tiles."""
    N = 4104 if rows == 700 else 16
    eye = torch.eye(8, device=DEV, dtype=BF16)
    w = torch.cat([eye] * (N // 8))                       # out[:, n] = x[:, n % 8], as far as that is finite: one value a row besides zeros
    for value, want in ((INF, INF), (-INF, NAN), (NAN, NAN)):
        x = torch.full((rows, 8), 0.0, device=DEV, dtype=BF16)
        bias = torch.zeros(N, device=DEV)
        bias[3] = value
        for name in ("silu", "gelu", "gelu_tanh"):
            y = pk.linear(x, w, bias, activation=name)
            assert _same(y[:, 3], [want] * rows), (name, value, y[0, 3])
            others = torch.arange(N, device=DEV) != 3
            assert torch.count_nonzero(y[:, others]) == 0, name
            # gated: 2 * act(value)
            both = torch.cat([torch.full((N,), 2.0, device=DEV), bias])
            _, saved = pk.feed_forward(x, torch.cat([w, w]), torch.zeros(8, N, device=DEV, dtype=BF16), both, activation=name, save=True)
            assert _same(saved.hidden[:, 3], [want] * rows), (name, value, saved.hidden[0, 3])
            # the pass back: slopes of an infinite sum are the formulas' 0 times infinity
            _, _, db = pk.linear_backward(torch.ones(rows, 8, device=DEV, dtype=BF16), x, eye, bias[:8].expand(rows, 8).contiguous(), activation=name)
            assert db[[0, 1, 2, 4, 5, 6, 7]].isfinite().all() and db[3].isnan(), (name, value)


def test_a_saved_tensor_that_a_call_overwrote_is_noticed():
    """A recorded call saves its input; one that writes in place over that input afterwards has torch refuse the stale backward pass."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    make = lambda *s: torch.randn(s, generator=gen, device=DEV).to(BF16)  # noqa: E731
    w = make(64, 64).requires_grad_()
    for overwrite in (lambda x: pk.layer_norm(x, out=x), lambda x: pk.linear(make(16, 64), w, residual=x, out=x),
                      lambda x: pk.feed_forward(make(16, 64), w, w, gated=False, residual=x, out=x)):
        x = make(16, 64)
        y = pk.linear(x, w)
        with torch.no_grad():
            overwrite(x)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


@pytest.mark.parametrize("rows,width,tables", [(5, 64, 65), (3000, 264, 1000), (40, 2056, 8193)])
def test_gradients_of_rows_under_many_frozen_tables(rows, width, tables):
    x, w, b, index, dy = _norm_inputs(rows, width, BF16, tables, F32, rows)
    leaf = x.clone().requires_grad_()
    pk.layer_norm(leaf, w, b, row_index=index, eps=1e-5).backward(dy)
    want = O.layer_norm_backward(dy, x, w, b, index, 1e-5)
    _within(leaf.grad, (want[0], _norm_grad_bounds(dy, x, w, index, want, 1e-5)[0]), "dx")
    # with the tables' gradients, or one of them, dx has the same bits
    few = index % 64
    both = pk.layer_norm_backward(dy, x, w[:64], b[:64], row_index=few)
    for weight_grad, bias_grad in ((False, False), (True, False), (False, True)):
        got = pk.layer_norm_backward(dy, x, w[:64], b[:64], row_index=few, weight_grad=weight_grad, bias_grad=bias_grad)
        assert torch.equal(got[0], both[0])
        for part, whole, asked in zip(got[1:], both[1:], (weight_grad, bias_grad)):
            assert torch.equal(part, whole) if asked else part is None


@pytest.mark.parametrize("gated", [False, True])
def test_each_recorded_gradient_of_a_block_by_itself(gated):
    """With whichever of the others frozen, a gradient has the bits of the whole pass."""
    gen = torch.Generator(device=DEV).manual_seed(2)
    make = lambda *s: (torch.randn(s, generator=gen, device=DEV) * 0.3).to(BF16)  # noqa: E731
    parts = [make(150, 72), make(272 if gated else 136, 72), make(72, 136), make(272 if gated else 136).float(), make(72), make(150, 72)]
    dy = make(150, 72)

    def grads(wanted):
        leaves = [t.clone().requires_grad_(i in wanted) for i, t in enumerate(parts)]
        pk.feed_forward(*leaves[:5], activation="gelu", gated=gated, residual=leaves[5]).backward(dy)
        return [t.grad for t in leaves]

    whole = grads(range(6))
    for wanted in ([0], [1], [2], [3], [4], [5], [1, 3], [2, 4], [0, 2, 3]):
        for i, g in enumerate(grads(wanted)):
            assert (g is None) == (i not in wanted)
            assert g is None or (torch.equal(g, whole[i]) and g.dtype is parts[i].dtype), (wanted, i)


def test_keys_kept_for_text_states_follow_what_is_written_over_them():
    """The processor keeps a cross-attention's keys by the text states' version: states that a call wrote over in place give their own keys, not the earlier ones."""
    from tests.test_gpu_full import _Attn

    torch.manual_seed(3)
    H, hidden, width = 3, 384, 200
    attn = _Attn(hidden, H, kv_dim=width).cuda().to(BF16)
    enc, x = torch.randn((1, 64, width), device=DEV, dtype=BF16), torch.randn((1, 150, hidden), device=DEV, dtype=BF16)
    w = torch.randn((width, width), device=DEV, dtype=BF16)
    plain, cached = pk.PikaH3AttnProcessor(), pk.PikaH3AttnProcessor(cache_cross_kv=True)
    with torch.no_grad():
        before = cached(attn, x, encoder_hidden_states=enc)
        for write in (lambda e: pk.linear(e.clone(), w, residual=e, out=e), lambda e: pk.layer_norm(e, out=e),
                      lambda e: pk.feed_forward(e.clone(), w, w, gated=False, residual=e, out=e)):
            write(enc[0])
            got = cached(attn, x, encoder_hidden_states=enc)
            assert torch.equal(got, plain(attn, x, encoder_hidden_states=enc)) and not torch.equal(got, before)
            before = got
