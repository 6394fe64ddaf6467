"""Layer norm, products and the feed-forward block without a GPU: refusals of the C entries and of the Python front end, the oracle against torch's own
differentiation, and the sharing out of tiles in a host build."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest
import torch

import pika_h3_flex_amd as pk
from oracle import rows_oracle as O
from pika_h3_flex_amd import _lib
from pika_h3_flex_amd import rows as front

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "pika-h3-flex_amd", "csrc")
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("name,mirror", [("pkh3_norm_args", _lib.NormArgs), ("pkh3_product_args", _lib.ProductArgs)])
def test_struct_layout_matches_header(name, mirror):
    header = open(os.path.join(ROOT, "include", "pkh3_rows.h")).read()
    body = header[header.index("typedef struct %s {" % name): header.index("} %s;" % name)]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S).split("{", 1)[1]
    names = [re.findall(r"[A-Za-z_][A-Za-z_0-9]*", part)[-1] for decl in body.split(";") if decl.strip() for part in decl.split(",")]
    assert names == [f[0] for f in mirror._fields_]


def test_constants_match_header():
    header = open(os.path.join(ROOT, "include", "pkh3_rows.h")).read()
    values = dict(re.findall(r"#define PKH3_(\w+) (\d+)u?\b", header)) | dict(re.findall(r"PKH3_(ACT_\w+) = (\d+)", header))
    assert {k: int(v) for k, v in values.items()} == {k: getattr(_lib, k) for k in values} and len(values) == 13


# ---- refusals of the C entries: made-up addresses, nothing is looked at ----

def _norm_args(backward):
    a = _lib.NormArgs(x=0x1000000, weight=0x2000000, bias=0x2100000, row_index=0x3000000, workspace=0x9000000, workspace_bytes=1 << 30,
                      rows=10, width=264, tables=3, eps=1e-6)
    if backward:
        a.dy, a.dx, a.dweight, a.dbias, a.dy_stride, a.dx_stride = 0x4000000, 0x5000000, 0x6000000, 0x7000000, 264, 264
    else:
        a.out, a.out_stride = 0x5000000, 264
    a.x_stride = 264
    return a


def _set(**kw):
    def change(a):
        for k, v in kw.items():
            setattr(a, k, v)
    return change


NORM_BAD = [
    (_set(x=0), _lib.PKH3_ENULL), (_set(x=0x1000008), _lib.PKH3_EALIGN), (_set(x_stride=100), _lib.PKH3_ESTRIDE), (_set(x_stride=256), _lib.PKH3_ESTRIDE),
    (_set(x_stride=-264), _lib.PKH3_ESTRIDE), (_set(x_stride=(1 << 22) + 8), _lib.PKH3_ESTRIDE), (_set(width=0), _lib.PKH3_ESHAPE), (_set(width=12), _lib.PKH3_ESHAPE),
    (_set(width=16392, x_stride=16392), _lib.PKH3_ESHAPE), (_set(rows=-1), _lib.PKH3_ESHAPE), (_set(rows=(1 << 21) + 1), _lib.PKH3_ESHAPE),
    (_set(tables=0), _lib.PKH3_ESHAPE), (_set(eps=-1.0), _lib.PKH3_EARG), (_set(eps=float("nan")), _lib.PKH3_EARG), (_set(eps=float("inf")), _lib.PKH3_EARG),
    (_set(flags=4), _lib.PKH3_EARG), (_set(weight=0x2000004), _lib.PKH3_EALIGN), (_set(row_index=0x3000002), _lib.PKH3_EALIGN),
]


@pytest.mark.parametrize("i", range(len(NORM_BAD)))
def test_layer_norm_refuses(lib, i):
    change, code = NORM_BAD[i]
    for backward, call in ((False, lib.pkh3_layer_norm), (True, lib.pkh3_layer_norm_backward)):
        a = _norm_args(backward)
        change(a)
        assert call(C.byref(a), None) == code, backward
    assert lib.pkh3_layer_norm(None, None) == _lib.PKH3_ENULL


@pytest.mark.parametrize("change,code", [
    (_set(out=0x1000000 + 264 * 2), _lib.PKH3_EARG), (_set(out=0x2000000), _lib.PKH3_EARG), (_set(out=0x2100000 + 64), _lib.PKH3_EARG), (_set(out=0x3000000), _lib.PKH3_EARG),
    (_set(out=0x1000000, out_stride=528), _lib.PKH3_EARG), (_set(bias=0x2100002), _lib.PKH3_EALIGN), (_set(out=0), _lib.PKH3_ENULL)])
def test_layer_norm_refuses_outputs(lib, change, code):
    a = _norm_args(False)
    change(a)
    assert lib.pkh3_layer_norm(C.byref(a), None) == code


@pytest.mark.parametrize("change,code", [
    (_set(tables=65), _lib.PKH3_ESHAPE), (_set(dx=0x1000000 + 16), _lib.PKH3_EARG), (_set(dx=0x4000000 + 16), _lib.PKH3_EARG), (_set(dx=0x2000000), _lib.PKH3_EARG),
    (_set(dweight=0x1000000), _lib.PKH3_EARG), (_set(dweight=0x4000000), _lib.PKH3_EARG), (_set(dweight=0x5000000), _lib.PKH3_EARG), (_set(dweight=0x2000000), _lib.PKH3_EARG),
    (_set(dbias=0x6000000 + 16), _lib.PKH3_EARG), (_set(dbias=0x3000000), _lib.PKH3_EARG), (_set(dy=0), _lib.PKH3_ENULL), (_set(dx=0), _lib.PKH3_ENULL),
    (_set(dweight=0x6000004), _lib.PKH3_EALIGN), (_set(workspace=0), _lib.PKH3_EWORKSPACE), (_set(workspace=0x9000010), _lib.PKH3_EWORKSPACE),
    (_set(workspace_bytes=100), _lib.PKH3_EWORKSPACE), (_set(rows=0), _lib.PKH3_ESHAPE)])
def test_layer_norm_backward_refuses(lib, change, code):
    a = _norm_args(True)
    change(a)
    assert lib.pkh3_layer_norm_backward(C.byref(a), None) == code


def _product_args(**kw):
    a = _lib.ProductArgs(a=0x1000000, b=0x2000000, out=0x3000000, workspace=0x40000000, workspace_bytes=1 << 30, a_stride=72, b_stride=72, out_stride=136,
                         M=20, N=136, K=72)
    _set(**kw)(a)
    return a


PRODUCT_BAD = [
    (dict(a=0), _lib.PKH3_ENULL), (dict(b=0), _lib.PKH3_ENULL), (dict(out=0), _lib.PKH3_ENULL), (dict(a=0x1000004), _lib.PKH3_EALIGN), (dict(b=0x2000008), _lib.PKH3_EALIGN),
    (dict(out=0x3000002), _lib.PKH3_EALIGN), (dict(a_stride=64), _lib.PKH3_ESTRIDE), (dict(b_stride=76), _lib.PKH3_ESTRIDE), (dict(out_stride=128), _lib.PKH3_ESTRIDE),
    (dict(N=0), _lib.PKH3_ESHAPE), (dict(N=132), _lib.PKH3_ESHAPE), (dict(K=0), _lib.PKH3_ESHAPE), (dict(K=71), _lib.PKH3_ESHAPE), (dict(M=-1), _lib.PKH3_ESHAPE),
    (dict(M=(1 << 21) + 1), _lib.PKH3_ESHAPE), (dict(flags=32), _lib.PKH3_EARG), (dict(activation=4), _lib.PKH3_EARG), (dict(activation=-1), _lib.PKH3_EARG),
    (dict(flags=_lib.PRODUCT_A_ACROSS), _lib.PKH3_EUNSUPPORTED), (dict(flags=_lib.PRODUCT_GRAD), _lib.PKH3_EUNSUPPORTED),
    (dict(flags=_lib.PRODUCT_B_ACROSS | _lib.PRODUCT_GATED), _lib.PKH3_EUNSUPPORTED),
    (dict(flags=_lib.PRODUCT_A_ACROSS | _lib.PRODUCT_B_ACROSS, M=20), _lib.PKH3_ESHAPE),
    (dict(sums=0x5000000), _lib.PKH3_EARG), (dict(gate=0x6000000, gate_stride=136), _lib.PKH3_ESHAPE), (dict(gate=0x6000000, gate_stride=136, gate_rows=2, gate_index=0x7000001), _lib.PKH3_EALIGN),
    (dict(bias=0x6000004), _lib.PKH3_EALIGN), (dict(residual=0x6000000), _lib.PKH3_ESTRIDE), (dict(residual=0x3000010, residual_stride=136), _lib.PKH3_EARG),
    (dict(out=0x1000000), _lib.PKH3_EARG), (dict(out=0x2000000), _lib.PKH3_EARG), (dict(pre=0x3000000, pre_stride=136), _lib.PKH3_EARG),
    (dict(pre=0x1000000, pre_stride=136), _lib.PKH3_EARG), (dict(bias=0x3000000), _lib.PKH3_EARG), (dict(pre=0x8000000, pre_stride=136, bias=0x8000000), _lib.PKH3_EARG),
    (dict(pre=0x8000000, pre_stride=136, residual=0x8000000, residual_stride=136), _lib.PKH3_EARG),
]


@pytest.mark.parametrize("i", range(len(PRODUCT_BAD)))
def test_product_refuses(lib, i):
    kw, code = PRODUCT_BAD[i]
    a = _product_args(**kw)
    assert lib.pkh3_product(C.byref(a), None) == code, lib.pkh3_last_error()
    assert lib.pkh3_product(None, None) == _lib.PKH3_ENULL


def test_products_of_operands_across_refuse_what_goes_with_others(lib):
    for flags, b_stride in ((_lib.PRODUCT_B_ACROSS, 136), (_lib.PRODUCT_A_ACROSS | _lib.PRODUCT_B_ACROSS, 136)):
        good = dict(flags=flags, b_stride=b_stride, M=24, a_stride=72)
        for kw in (dict(bias=0x6000000), dict(activation=1), dict(residual=0x6000000, residual_stride=136), dict(gate=0x6000000, gate_rows=1, gate_stride=136),
                   dict(pre=0x8000000, pre_stride=136)):
            assert lib.pkh3_product(C.byref(_product_args(**good, **kw)), None) == _lib.PKH3_EARG, kw
    for kw in (dict(residual=0x6000000, residual_stride=136), dict(gate=0x6000000, gate_rows=1, gate_stride=136)):
        assert lib.pkh3_product(C.byref(_product_args(flags=_lib.PRODUCT_GATED, **kw)), None) == _lib.PKH3_EARG, kw


def test_product_of_gradients_refuses(lib):
    flags = _lib.PRODUCT_B_ACROSS | _lib.PRODUCT_GRAD
    good = dict(flags=flags, b_stride=136, pre=0x8000000, pre_stride=136, activation=1, sums=0x5000000)
    for kw, code in ((dict(pre=0), _lib.PKH3_ENULL), (dict(bias=0x6000000), _lib.PKH3_EARG), (dict(residual=0x6000000, residual_stride=136), _lib.PKH3_EARG),
                     (dict(gate=0x6000000, gate_rows=1, gate_stride=136), _lib.PKH3_EARG), (dict(out=0x8000000), _lib.PKH3_EARG), (dict(sums=0x3000000), _lib.PKH3_EARG),
                     (dict(sums=0x8000000), _lib.PKH3_EARG), (dict(workspace=0), _lib.PKH3_EWORKSPACE), (dict(workspace_bytes=8), _lib.PKH3_EWORKSPACE),
                     (dict(workspace=0x40000080), _lib.PKH3_EWORKSPACE), (dict(M=0), _lib.PKH3_ESHAPE), (dict(pre_stride=128), _lib.PKH3_ESTRIDE),
                     (dict(flags=flags | _lib.PRODUCT_GATED), _lib.PKH3_ESTRIDE)):
        a = _product_args(**{**good, **kw})
        assert lib.pkh3_product(C.byref(a), None) == code, (kw, lib.pkh3_last_error())


def test_slices_of_one_buffer_do_not_overlap(lib):
    """Columns beside each other in one buffer are apart; the same ones, or some of the same, are not.  (Workspaces are looked at last: a call that is refused
    for its workspace was taken otherwise.)"""
    for at, code in ((72, _lib.PKH3_EWORKSPACE), (64, _lib.PKH3_EARG), (0, _lib.PKH3_EARG), (-136, _lib.PKH3_EWORKSPACE), (-128, _lib.PKH3_EARG), (208, _lib.PKH3_EARG)):
        a = _product_args(flags=_lib.PRODUCT_B_ACROSS | _lib.PRODUCT_GRAD, b_stride=136, sums=0x5000000, a_stride=208, out=0x1000000 + at * 2, out_stride=208, workspace=0)
        assert lib.pkh3_product(C.byref(a), None) == code, at


def test_activation_grad_refuses(lib):
    good = dict(b=0, K=0, a_stride=136, pre=0x8000000, pre_stride=136, activation=2, sums=0x5000000)
    for kw, code in ((dict(a=0), _lib.PKH3_ENULL), (dict(pre=0), _lib.PKH3_ENULL), (dict(out=0), _lib.PKH3_ENULL), (dict(out=0x1000010), _lib.PKH3_EARG),
                     (dict(out=0x8000000), _lib.PKH3_EARG), (dict(sums=0x1000000), _lib.PKH3_EARG), (dict(sums=0x3000000), _lib.PKH3_EARG), (dict(sums=0x8000000), _lib.PKH3_EARG),
                     (dict(flags=1), _lib.PKH3_EARG), (dict(activation=7), _lib.PKH3_EARG), (dict(N=4), _lib.PKH3_ESHAPE), (dict(M=0), _lib.PKH3_ESHAPE),
                     (dict(workspace_bytes=8), _lib.PKH3_EWORKSPACE), (dict(a_stride=128), _lib.PKH3_ESTRIDE)):
        a = _product_args(**{**good, **kw})
        assert lib.pkh3_activation_grad(C.byref(a), None) == code, (kw, lib.pkh3_last_error())


def test_workspace_sizes(lib):
    a = _lib.NormArgs(rows=100, width=512, tables=3)
    n = lib.pkh3_norm_workspace_bytes(C.byref(a))
    assert n > 0 and n % 256 == 0
    a.tables = 65
    assert lib.pkh3_norm_workspace_bytes(C.byref(a)) == 0 and lib.pkh3_last_error()
    a = _product_args(flags=_lib.PRODUCT_B_ACROSS | _lib.PRODUCT_GRAD, sums=256)
    n = lib.pkh3_product_workspace_bytes(C.byref(a))
    assert n > 0 and n % 256 == 0 and not lib.pkh3_last_error()
    a.N = 4
    assert lib.pkh3_product_workspace_bytes(C.byref(a)) == 0 and lib.pkh3_last_error()


# ---- refusals of the front end ----

def test_front_end_refuses_host_memory_and_shapes():
    x, w = torch.zeros(4, 64, dtype=BF16), torch.zeros(32, 64, dtype=BF16)
    for call in (lambda: pk.layer_norm(x), lambda: pk.linear(x, w), lambda: pk.feed_forward(x, w, w), lambda: pk.layer_norm_backward(x, x),
                 lambda: pk.linear_backward(x, x, w), lambda: pk.feed_forward_backward(x, x, w, w, front.Saved(x, x))):
        with pytest.raises(ValueError, match="device memory"):
            call()
    with pytest.raises(ValueError, match="activation"):
        front._activation("tanh")
    with pytest.raises(TypeError):
        front._matrix("x", torch.zeros(4, 64), 4, 64, -1)
    with pytest.raises(ValueError, match="column stride"):
        front._matrix("x", torch.zeros(64, 8, dtype=BF16).t(), 8, 64, -1)
    with pytest.raises(ValueError, match="must be"):
        front._matrix("x", x, 5, 64, -1)
    with pytest.raises(ValueError, match="bias"):
        front._vector("bias", torch.zeros(8, dtype=torch.float16), 8, -1)
    with pytest.raises(ValueError, match="row_index"):
        front._index("row_index", torch.zeros(8, dtype=torch.int64), 8, -1)
    with pytest.raises(ValueError, match="row_index"):
        front._norm_tables(torch.zeros(3, 64), None, None, 4, 64, -1)
    with pytest.raises(ValueError, match="one type"):
        front._norm_tables(torch.zeros(64), torch.zeros(64, dtype=BF16), None, 4, 64, -1)
    with pytest.raises(ValueError, match="row_index goes with a gate"):
        front._finish(None, torch.zeros(4, dtype=torch.int32), None, 4, 64, -1)
    with pytest.raises(ValueError, match="twice a multiple of 8"):
        front._block(x, torch.zeros(24, 64, dtype=BF16), w, True, -1)


# ---- the oracle ----

@pytest.mark.parametrize("name", ["none", "silu", "gelu", "gelu_tanh"])
def test_oracle_activations(name):
    F = torch.nn.functional
    v = torch.linspace(-30, 30, 4001, dtype=torch.float64, requires_grad=True)
    want = {"none": lambda t: t * 1, "silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[name](v)
    slope, = torch.autograd.grad(want.sum(), v)
    assert torch.allclose(O.act(name, v.detach()), want.detach(), rtol=1e-9, atol=1e-14) and torch.allclose(O.act_slope(name, v.detach()), slope, rtol=1e-9, atol=1e-12)
    assert O.act_slope(name, v.detach()).abs().max() <= O.SLOPE[name]
    curve = (O.act_slope(name, v.detach() + 1e-5) - O.act_slope(name, v.detach() - 1e-5)) / 2e-5
    assert curve.abs().max() <= O.CURVATURE[name] + 1e-9


@pytest.mark.parametrize("gated", [False, True])
def test_oracle_gradients_against_torch(gated):
    torch.manual_seed(0)
    F = torch.nn.functional
    make = lambda *s: torch.randn(s, dtype=torch.float64, requires_grad=True)  # noqa: E731
    x, w1, w2, b1, b2 = make(7, 16), make(48 if gated else 24, 16), make(8, 24), make(48 if gated else 24), make(8)
    dy = torch.randn(7, 8, dtype=torch.float64)
    z = F.linear(x, w1, b1)
    h = z[:, :24] * F.gelu(z[:, 24:]) if gated else F.gelu(z)
    y = F.linear(h, w2, b2)
    parts = [t.detach() for t in (x, w1, w2, b1, b2)]
    assert torch.allclose(O.feed_forward(*parts, "gelu", gated)[0], y.detach())
    for got, want in zip(O.feed_forward_backward(dy, *parts, "gelu", gated), torch.autograd.grad(y, (x, w1, w2, b1, b2), dy)):
        assert torch.allclose(got[0], want) and (got[1] >= 0).all()
    weight, bias, index = make(3, 16), make(3, 16), torch.tensor([0, 2, 2, 1, 0, 0, 2], dtype=torch.int32)
    y = F.layer_norm(x, (16,), eps=1e-5) * weight[index.long()] + bias[index.long()]
    dy = torch.randn(7, 16, dtype=torch.float64)
    assert torch.allclose(O.layer_norm(x.detach(), weight.detach(), bias.detach(), index, 1e-5), y.detach())
    for got, want in zip(O.layer_norm_backward(dy, x.detach(), weight.detach(), bias.detach(), index, 1e-5), torch.autograd.grad(y, (x, weight, bias), dy)):
        assert torch.allclose(got, want)
    w = make(8, 16)
    z = F.linear(x, w, b2)
    y = F.silu(z)
    dy = torch.randn(7, 8, dtype=torch.float64)
    assert torch.allclose(O.linear(x.detach(), w.detach(), b2.detach(), "silu")[0], y.detach())
    for got, want in zip(O.linear_backward(dy, x.detach(), w.detach(), b2.detach(), "silu"), torch.autograd.grad(y, (x, w, b2), dy)):
        assert torch.allclose(got[0], want)


# ---- the sharing out of tiles, in a host build ----

PROGRAM = r"""
#include "pkh3_rows_index.h"
#include <stdio.h>
#include <stdlib.h>
#include <vector>
#include <set>
using namespace pkh3;
#define CHECK(c) do { if (!(c)) { printf("failed: %s (line %d) M %d N %d K %d mode %d\n", #c, __LINE__, M, N, K, mode); return 1; } } while (0)
int main() {
  srand(7);
  for (int trial = 0; trial < 4000; ++trial) {
    auto log_size = [](int most) { int bits = 1 + rand() % 21; int v = 1 + rand() % (1 << bits); return v < most ? v : most; };
    int M = log_size(60000), N = (log_size(20000) + 7) / 8 * 8, K = log_size(60000), mode = rand() % 4;
    if ((int64_t)M * N > 400000000ll) continue;
    ProductPlan plan = plan_product(M, N, K, false, mode, mode >= kGrad, trial % 2);
    const ProductShare& s = plan.share;
    const int columns = (mode == kGated ? 16 : 32) * plan.fb, tiles = s.m_tiles * s.n_tiles;
    CHECK(s.groups % 8 == 0 && s.groups * s.rounds + s.rest == tiles && s.rest < s.groups && s.cuts >= 1 && (s.cuts == 1 || s.cuts * 2 <= s.chunks));
    CHECK((int64_t)s.m_tiles * 32 * plan.tb >= M && (int64_t)s.n_tiles * columns >= N && (int64_t)s.chunks * kChunk >= K && (int64_t)(s.chunks - 1) * kChunk < K);
    CHECK(plan.tb != 3 || trial % 2 == 0);
    CHECK(s.blocks >= 1 && s.blocks <= s.n_tiles);
    std::set<std::pair<int, int>> places;
    for (int i = 0; i < tiles; ++i) {
      TilePlace at = tile_of(s, i);
      CHECK(at.m >= 0 && at.m < s.m_tiles && at.n >= 0 && at.n < s.n_tiles);
      CHECK(places.insert({at.m, at.n}).second);
    }
    // as the kernel's workgroups take them: whole tiles, then parts, each once
    std::vector<char> taken(tiles, 0), used(s.rest * s.cuts + 1, 0);
    for (int group = 0; group < s.groups; ++group) {
      for (int turn = 0; turn < s.rounds; ++turn) {
        const int unit = unit_of(s.rounds, turn, group, s.groups);
        CHECK(unit >= 0 && unit < s.rounds * s.groups && !taken[unit]);
        taken[unit] = 1;
      }
      for (int turn = 0; turn < part_turns(s); ++turn) {
        const int unit = unit_of(part_turns(s), turn, group, s.groups);
        CHECK(unit >= 0);
        if (unit >= units_of(s)) break;                // (and so are all that follow)
        CHECK(!used[unit]);
        used[unit] = 1;
      }
    }
    for (int i = 0; i < s.rounds * s.groups; ++i) CHECK(taken[i]);
    for (int i = 0; i < units_of(s); ++i) CHECK(used[i]);
    if (s.rest) {
      CHECK(part_begin(s, 0) == 0 && part_begin(s, s.cuts) == s.chunks);
      for (int part = 0; part < s.cuts; ++part) CHECK(part_begin(s, part + 1) > part_begin(s, part));
    }
    CHECK(s.cuts == 1 || (size_t)units_of(s) * 32 * plan.tb * 32 * plan.fb * 4 <= plan.sums_off);
  }
  printf("ok\n");
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ is not installed")
def test_tiles_are_shared_out_once(tmp_path):
    src, exe = tmp_path / "share.cpp", tmp_path / "share"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr
