"""What the front end of the feed-forward half does around its launches, with the launches left out: tensors of host memory, entries written down in place of being called."""
import pytest
import torch

import pika_h3_flex_amd as pk
from pika_h3_flex_amd import rows as front

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture
def entries(monkeypatch):
    """Names of the C entries that calls come to."""
    names = []
    monkeypatch.setattr(front, "_place", lambda x: -1)
    monkeypatch.setattr(front, "_call", lambda name, args, index: names.append(name))
    return names


def _parts(rows=4, width=64, inner=32):
    x, w_in, w_out = torch.ones(rows, width, dtype=BF16), torch.ones(inner, width, dtype=BF16), torch.ones(width, inner, dtype=BF16)
    return x, w_in, w_out


def _calls(x, w_in, w_out):
    """The three calls with an ``out`` of their own shape."""
    return ((x.shape, lambda out: pk.layer_norm(x, out=out)), ((x.shape[0], w_in.shape[0]), lambda out: pk.linear(x, w_in, out=out)),
            (x.shape, lambda out: pk.feed_forward(x, w_in, w_out, gated=False, out=out)))


def test_what_a_call_overwrites_has_another_version(entries):
    x, w_in, w_out = _parts()
    for shape, call in _calls(x, w_in, w_out):
        out = torch.zeros(shape, dtype=BF16)
        before = out._version
        assert call(out) is out and out._version > before
    residual, before = torch.zeros(4, 32, dtype=BF16), x._version
    pk.linear(x, w_in, residual=residual, out=residual)
    assert residual._version > 0 and x._version == before
    buffer = torch.zeros(4, 128, dtype=BF16)                     # a slice shares the counter of its buffer
    pk.layer_norm(x, out=buffer[:, 64:])
    assert buffer._version > 0
    before = x._version
    pk.layer_norm(x, out=x)
    assert x._version > before


def test_an_output_that_is_differentiated_is_refused(entries):
    x, w_in, w_out = _parts()
    for shape, call in _calls(x, w_in, w_out):
        out = torch.zeros(shape, dtype=BF16, requires_grad=True)
        with pytest.raises(ValueError, match="out"):
            call(out)
        assert not entries
        with torch.no_grad():
            call(out)
        entries.clear()


def test_forward_mode_tangents_are_refused(entries):
    """A dual tensor does not require gradients: its tangent would be lost without a word."""
    x, w_in, w_out = _parts()
    fw = torch.autograd.forward_ad
    dy, hidden = torch.ones(4, 64, dtype=BF16), torch.ones(4, 32, dtype=BF16)
    saved = front.Saved(torch.ones(4, 32), hidden)
    weight = torch.ones(64, dtype=BF16)
    calls = [lambda a, w: pk.layer_norm(a, weight), lambda a, w: pk.linear(a, w), lambda a, w: pk.feed_forward(a, w, w_out, gated=False),
             lambda a, w: pk.linear(hidden, w_out, residual=a), lambda a, w: pk.layer_norm_backward(dy, a, weight), lambda a, w: pk.layer_norm_backward(a, dy, weight),
             lambda a, w: pk.linear_backward(hidden, a, w), lambda a, w: pk.feed_forward_backward(a, dy, w, w_out, saved, gated=False)]
    with fw.dual_level():
        dual, dual_w = fw.make_dual(x, torch.ones_like(x)), fw.make_dual(w_in, torch.ones_like(w_in))
        for i, call in enumerate(calls):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    call(dual, w_in)
        for call in (calls[1], calls[2], calls[6], calls[7]):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(x, dual_w)
        assert not entries
        assert calls[1](x, w_in).shape == (4, 32)                # (without tangents a level changes nothing)
    with pytest.raises(RuntimeError):                            # torch.func's tensors have no address, or a tangent
        torch.func.jvp(lambda a: pk.linear(a, w_in), (x,), (torch.ones_like(x),))


def test_a_gate_without_rows_is_refused(entries):
    """Its address is NULL, which the entry takes for no gate."""
    x, w_in, w_out = _parts()
    index = torch.zeros(4, dtype=torch.int32)
    for call in (lambda g: pk.linear(x, w_in, gate=g, row_index=index), lambda g: pk.linear(x, w_in, gate=g),
                 lambda g: pk.feed_forward(x, w_in, w_out, gated=False, gate=torch.zeros(g.shape[0], 64, dtype=BF16), row_index=index)):
        with pytest.raises(ValueError, match="gate"):
            call(torch.zeros(0, 32, dtype=BF16))
        call(torch.zeros(1, 32, dtype=BF16))


def test_a_row_index_without_a_gate_is_refused_where_gradients_are_recorded(entries):
    """As it is where they are not."""
    x, w_in, w_out = _parts()
    index = torch.zeros(4, dtype=torch.int32)
    for w in (w_in, w_in.clone().requires_grad_()):
        for call in (lambda: pk.linear(x, w, row_index=index), lambda: pk.feed_forward(x, w, w_out, gated=False, row_index=index)):
            with pytest.raises(ValueError, match="row_index"):
                call()
    assert not entries


def test_frozen_tables(lib, entries, monkeypatch):
    """Only the tables' own gradients are bound to 64 rows, and they are formed where they are asked for alone."""
    calls = []
    monkeypatch.setattr(front, "_call", lambda name, args, index: calls.append((name, front._lib.NORM_ARGS_FORMAT.unpack(args))))
    x = torch.ones(4, 64, dtype=BF16, requires_grad=True)
    index = torch.zeros(4, dtype=torch.int32)
    for tables in (3, 65, 1000):
        weight, bias = torch.ones(tables, 64), torch.ones(tables, 64)
        pk.layer_norm(x, weight, bias, row_index=index).sum().backward()
        name, args = calls[-1]
        assert name == "pkh3_layer_norm_backward" and not any(args[i] for i in (7, 8, 9, 10)), tables        # no sums, no workspace
    weight = torch.ones(3, 64, requires_grad=True)
    pk.layer_norm(x, weight, torch.ones(3, 64), row_index=index).sum().backward()
    assert calls[-1][1][7] and not calls[-1][1][8]
    got = pk.layer_norm_backward(x.detach(), x.detach(), weight.detach(), bias[:3], row_index=index, weight_grad=False)
    assert got[1] is None and got[2].shape == (3, 64) and not calls[-1][1][7] and calls[-1][1][8]
    with pytest.raises(pk.Pkh3Error):
        pk.layer_norm_backward(x.detach(), x.detach(), torch.ones(65, 64), row_index=index)
    # the entry (no rows, so that nothing is launched)
    for dweight, code in ((0, front._lib.PKH3_OK), (0x6000000, front._lib.PKH3_ESHAPE)):
        a = front._lib.NormArgs(dweight=dweight, rows=0, width=264, tables=65535)
        assert lib.pkh3_layer_norm_backward(a, None) == code


def test_recorded_passes_form_what_is_asked_for(entries, monkeypatch):
    """The products behind each gradient alone: two weights of a block are two gradients, and none at all takes no launch."""
    monkeypatch.setattr(front, "_product_scratch", lambda *a: 0)
    monkeypatch.setattr(front, "_activation_scratch", lambda *a: 0)
    product, sums = "pkh3_product", "pkh3_activation_grad"
    x, w_in, w_out = _parts()
    b_in, b_out, residual = torch.ones(32), torch.ones(64), torch.ones(4, 64, dtype=BF16)
    # x, w_in, w_out, b_in, b_out, residual; launches of the backward pass
    for wanted, launches in (((1, 0, 0, 0, 0, 0), [product] * 2), ((0, 1, 0, 0, 0, 0), [product] * 2), ((0, 0, 1, 0, 0, 0), [product]), ((0, 0, 0, 1, 0, 0), [product]),
                             ((0, 0, 0, 0, 1, 0), [sums]), ((0, 0, 0, 0, 0, 1), []), ((1, 1, 1, 1, 1, 1), [product] * 4 + [sums])):
        leaves = [t.clone().requires_grad_(bool(w)) for t, w in zip((x, w_in, w_out, b_in, b_out, residual), wanted)]
        y = pk.feed_forward(*leaves[:5], residual=leaves[5], gated=False)
        entries.clear()
        y.sum().backward()
        assert entries == launches, wanted
        assert [t.grad is not None for t in leaves] == [bool(w) for w in wanted]
        assert all(t.grad is None or t.grad.dtype is t.dtype for t in leaves)
    # x, weight, bias, residual
    for activation, wanted, launches in (("silu", (0, 0, 0, 1), []), ("silu", (1, 0, 0, 0), [sums, product]), ("silu", (0, 0, 1, 0), [sums]), ("silu", (1, 1, 1, 1), [sums, product, product]),
                                         ("none", (0, 0, 0, 1), []), ("none", (0, 1, 0, 0), [product]), ("none", (0, 0, 1, 0), [sums])):
        leaves = [t.clone().requires_grad_(bool(w)) for t, w in zip((x, w_in, b_in, torch.ones(4, 32, dtype=BF16)), wanted)]
        y = pk.linear(*leaves[:3], activation=activation, residual=leaves[3])
        entries.clear()
        y.sum().backward()
        assert entries == launches, (activation, wanted)
        assert [t.grad is not None for t in leaves] == [bool(w) for w in wanted]
