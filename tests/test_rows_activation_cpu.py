"""The activations' arithmetic of pkh3_rows.h in float32 on the host, with the constants as they stand there, against the formulas in 64 bits: how far the tail of the normal distribution is off
is what the header says of it, and what the oracle allows of an activation."""
import math
import os
import re

import numpy as np
import pytest
import torch

from oracle import rows_oracle as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = open(os.path.join(ROOT, "pika-h3-flex_amd", "csrc", "pkh3_rows.h")).read()
f = np.float32


def _tail(v):
    """normal_tail(), every operation rounded to float32 (the compiler fuses some of them, which rounds less)."""
    body = HEADER[HEADER.index("float normal_tail(float v)"):]
    body = body[:body.index("\n}")]
    scale = f(re.search(r"1\.0f \+ ([0-9.]+)f \* fabsf\(v\)", body).group(1))
    first = f(re.search(r"float p = (-?[0-9.]+)f;", body).group(1))
    rest = [f(sign + c) for sign, c in re.findall(r"p = p \* t ([+-]) ([0-9.]+)f;", body)]
    assert len(rest) == 7
    t = f(1) / (f(1) + scale * np.abs(v))
    p = np.full_like(v, first)
    for c in rest:
        p = p * t + c
    half = f(0.5) * f(math.log2(math.e))
    return t * np.exp2(p - half * (v * v))


def _errors(lo, hi):
    v = np.linspace(lo, hi, 200001).astype(f)
    want = 0.5 * torch.special.erfc(torch.from_numpy(v.astype(np.float64)) / math.sqrt(2.0)).numpy()
    return v.astype(np.float64), np.abs(_tail(v).astype(np.float64) / want - 1.0)


def test_tail_of_the_normal_distribution():
    """Fit, reciprocal and polynomial: 1.5e-6; an exponent of v^2 / 2 with four roundings (the constant, the square, the product, the difference): 4 * 2^-24 of it."""
    v, off = _errors(0.0, 13.0)
    assert (off <= 1.5e-6 + 4 * O.HALF_F32 * v * v / 2).all(), (off / (1.5e-6 + 4 * O.HALF_F32 * v * v / 2)).max()
    assert _errors(8.0, 13.0)[1].max() > 3e-6          # (the polynomial's share, 8e-7, is not all of it)


@pytest.mark.parametrize("name", ["silu", "gelu", "gelu_tanh"])
def test_oracle_allows_what_float32_costs(name):
    """The activations in float32 with single roundings stay within what the oracle allows for, far tails among them, and that is less than a rounding to bfloat16."""
    v = np.linspace(-80.0, 80.0, 400001).astype(f)
    v = v[{"silu": np.abs(v) < 80, "gelu": np.abs(v) < 12.5, "gelu_tanh": np.abs(v) < 9.5}[name]]
    log2e = f(math.log2(math.e))
    with np.errstate(over="ignore"):
        if name == "silu":
            y = v * (f(1) / (f(1) + np.exp2(-v * log2e)))
        elif name == "gelu":
            y = np.maximum(v, f(0)) - np.abs(v) * _tail(v)
        else:
            once = f(-2.0 * math.sqrt(2.0 / math.pi) * math.log2(math.e))
            y = v * (f(1) / (f(1) + np.exp2(v * (once + f(once * f(0.044715)) * (v * v)))))
    exact = torch.from_numpy(v.astype(np.float64))
    allowed = O.act_error(name, exact)
    assert (np.abs(y.astype(np.float64) - O.act(name, exact).numpy()) <= allowed.numpy()).all()
    assert (allowed <= 0.02 * O.HALF_BF16 * O.act(name, exact).abs() + 1e-36).all()
