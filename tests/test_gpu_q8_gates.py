"""GPU: gated products in 8-bit integers at gates far from zero, by the few-row kernel (3 rows) and by the paired one (40)."""
import math

import pytest
import torch

from test_gpu_q8 import TYPES, U, within

pytestmark = pytest.mark.gpu

ROWS = [3, 40]


def one_column(values):
    """A weight matrix with `values` in its first column, which the rows below have their only value in."""
    w = torch.zeros(len(values), 16)
    w[:, 0] = torch.tensor(values)
    return w.cuda()


def product(x, w):
    """(127 * 127) * row scale * channel scale, every step as the kernels round it."""
    c = torch.tensor(127.0)
    s = torch.tensor(16129.0) * (torch.tensor(abs(x)) / c)
    return torch.stack([s * (torch.tensor(abs(v)) / c) * (math.copysign(1.0, v) * math.copysign(1.0, x)) for v in w])


GATES = [-0.0, -1e-30, -0.5, -10.0, -50.0, -86.9, -87.1, -87.5, -88.0, -88.5, -89.0, -95.0, -100.0, -104.0, -110.0, -200.0, -1e3, -1e6, -1e10, -1e20, -1e30, -3e38, 3.0, 80.0, 1e3]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("y_type", TYPES)
@pytest.mark.parametrize("up", [1.0, -3.0, 1e20])
def test_strongly_negative_gates(ops, cuda, rows, act, y_type, up):
    gates = GATES if y_type != torch.float16 else [g for g in GATES if g <= 0]         # no overflow of the results
    layer = ops.Int8GatedLinear(one_column(gates), one_column([up] * len(gates)), act)
    x = torch.zeros(rows, 16, device="cuda")
    x[:, 0] = 1.0
    y = layer.forward(x, out_dtype=y_type)
    assert layer.device_status() == 0
    z, u = product(1.0, gates).double(), product(1.0, [up]).double()
    p = z if act == 1 else (8 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)
    f = z * torch.sigmoid(p)
    # p: up to six roundings and the constant's (GELU), each of which moves e^p by |p| U of itself; the exponential 2^-22 and the rounding of its argument |p| U, the sum U, the
    # quotient 2^-22, two products 2 U.  16-bit results: the exponential's argument in base 2 (2 |p| U more) and 2^-21.
    few = y_type != torch.float32
    e = 8 * p.abs() * U + 2.0 ** -21 + 4 * U + (2 * p.abs() * U + 2.0 ** -21 if few else 0)
    # From e^-p = 2^128 on (2^126 where the fast quotient takes it) a result may be zero: |z| 2^-128, |z| < 89, or |z| 2^-126; a subnormal activation is off by 2^-149.
    lost = 2.0 ** -119 if few else 2.0 ** -121
    bound = (f.abs() * e.clamp(max=1.0) + lost) * u.abs()
    want, y = (f * u).expand(rows, -1), y.cpu()
    if y_type == torch.float16:                # from 65520 on, half way to the power of two behind the largest value, fp16 rounds to infinity
        beyond = want.abs() - bound >= 65520
        assert torch.equal(y[beyond].double(), want[beyond].sign() * math.inf)
        want, y = torch.where(beyond, 0.0, want), torch.where(beyond, 0.0, y)
    within(y, want, bound.expand(rows, -1), y_type)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("y_type", TYPES)
def test_infinite_gates(ops, cuda, rows, act, y_type):
    """minus infinity times zero is NaN, as it is in the formula; plus infinity stays."""
    layer = ops.Int8GatedLinear(one_column([-1e30, 1e30, 1e-30]), one_column([1e-30] * 3), act)
    x = torch.zeros(rows, 16, device="cuda")
    x[:, 0] = 1e30
    y = layer.forward(x, out_dtype=y_type)
    assert torch.isnan(y[:, 0]).all() and (y[:, 1] == float("inf")).all() and torch.isfinite(y[:, 2]).all()
