"""Norm and gradient of rows up to the type's top, at lengths where their squares pass 32 bits again unless they are lifted
far enough: every kernel (few rows, rings, rows at offsets, rows read again).

Bounds as in test_gpu_add_norm.py, with u = 2^-24, and for rows whose root mean square passes 2^126 what s = 1 / rms
loses as a subnormal: half of 2^-149 of at least 2^-128, 4 u. So N + 4 units in y and in n = h s, 4 more in s g, and
8 more (of n and of s) in s n mean(g n), whose mean is taken with the lifted row.
"""

import numpy as np
import pytest

import vastloom_b200 as vb
from test_gpu_add_norm import EPS, U, additions, backward, check, dt, exact_grad, exact_norm, f64, forward

pytestmark = pytest.mark.gpu

LOW = 4  # units of s as a subnormal
PAIRS = [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")]
# rows, cols, pad, first row's offset: few rows from registers, one by one, read again; rings; rings at offsets
SHAPES = [(2, 8192, 0, 0), (3, 16384, 0, 0), (2, 30000, 0, 0), (2, 1 << 20, 0, 0), (2, 8192, 3, 1), (70, 8192, 0, 0),
          (70, 8192, 3, 0), (66, 16384, 0, 0), (66, 30000, 0, 0), (70, 4099, 0, 0), (70, 5000, 3, 1), (5, 1, 0, 0), (80, 7, 0, 0)]


@pytest.fixture(scope="module")
def dev():
    if vb.device_count() == 0:
        pytest.fail("no CUDA device: GPU tests must run on a B200")
    d = vb.Device(0, install_codebooks=False)
    yield d
    d.close()


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def view(torch, rows, cols, kind, pad, shift, values=None):
    ld = cols + pad
    v = torch.zeros(rows * ld + shift, device="cuda", dtype=dt(torch, kind))[shift:].as_strided((rows, cols), (ld, 1))
    return v if values is None else v.copy_(values)


def tops(torch, g, rows, cols, top):
    """Values of either sign between 0.9 and 1.1 of `top`; the last row ordinary ones."""
    v = top * (0.9 + 0.2 * torch.rand(rows, cols, device="cuda", generator=g))
    v *= torch.where(torch.rand(rows, cols, device="cuda", generator=g) < 0.5, -1.0, 1.0)
    v[-1] = torch.randn(cols, device="cuda", generator=g)
    return v


@pytest.mark.parametrize("xt,rt", PAIRS)
@pytest.mark.parametrize("rows,cols,pad,shift", SHAPES)
@pytest.mark.parametrize("top,more", [(3e38, 0.0), (2.7e38, 4e37)])  # more: the residual's largest
def test_norm_near_the_top(dev, torch, rows, cols, pad, shift, xt, rt, top, more):
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x = view(torch, rows, cols, xt, pad, shift, tops(torch, g, rows, cols, top))
    r = view(torch, rows, cols, rt, pad, shift, more * (2 * torch.rand(rows, cols, device="cuda", generator=g) - 1)) if more else None
    if more:
        r[-1] = torch.randn(cols, device="cuda", generator=g)
    w = 1.0 + 0.3 * torch.randn(cols, device="cuda", generator=g)
    h, y = view(torch, rows, cols, rt, pad, shift), view(torch, rows, cols, xt, pad, shift)
    q, scale = torch.zeros(rows, cols, device="cuda", dtype=torch.int8), torch.zeros(rows, device="cuda")
    forward(dev, torch, x, r, w, xt=xt, rt=rt, h=h, y=y, q=q, scale=scale)
    want_h, want_y = exact_norm(x, r, w, EPS)
    n = additions(cols) / 2 + 8 + LOW
    check(h, want_h, U * np.abs(want_h), rt)
    check(y, want_y, n * U * np.abs(want_y), xt)
    a = np.max(np.abs(want_y), axis=1)
    assert np.all(np.abs(f64(scale) - a / 127) <= (n + 2) * U * a / 127)
    assert np.all(np.abs(f64(q) - want_y * (127 / a)[:, None]) <= 0.5 + 127 * (2 * n + 4) * U)


@pytest.mark.parametrize("xt,rt", PAIRS)
@pytest.mark.parametrize("rows,cols,pad,shift", SHAPES)
def test_gradient_near_the_top(dev, torch, rows, cols, pad, shift, xt, rt):
    """dy large enough for a d that is no subnormal beside s = 3e-39."""
    g = torch.Generator(device="cuda").manual_seed(rows * 3 + cols)
    h = view(torch, rows, cols, rt, pad, shift, tops(torch, g, rows, cols, 3e38))
    dy = view(torch, rows, cols, xt, pad, shift, 1e10 * torch.randn(rows, cols, device="cuda", generator=g))
    dh = view(torch, rows, cols, rt, pad, shift, 1e-29 * torch.randn(rows, cols, device="cuda", generator=g))
    w = 1.0 + 0.3 * torch.randn(cols, device="cuda", generator=g)
    dx, dr = view(torch, rows, cols, xt, pad, shift), view(torch, rows, cols, rt, pad, shift)
    dw = torch.zeros(cols, device="cuda")
    backward(dev, torch, dy, h, w, dh, xt=xt, rt=rt, dx=dx, dr=dr, dw=dw)
    d, bound, want_w, w_bound = exact_grad(dy, h, w, dh, EPS)
    H, G = f64(h), f64(dy) * f64(w)
    s = 1.0 / np.sqrt(np.mean(H * H, axis=1, keepdims=True) + EPS)
    n = H * s
    bound = bound + U * LOW * (np.abs(s * G) + 2 * np.abs(s * n) * np.mean(np.abs(G * n), axis=1, keepdims=True))
    w_bound = w_bound + LOW * U * np.sum(np.abs(f64(dy) * n), axis=0)
    check(dx, d, bound, xt)
    check(dr, d, bound, rt)
    check(dw, want_w, w_bound, "f32")
    lone = view(torch, rows, cols, xt, pad, shift)
    backward(dev, torch, dy, h, w, dh, xt=xt, rt=rt, dx=lone)  # without the weight's: another kernel for long rows
    check(lone, d, bound, xt)
