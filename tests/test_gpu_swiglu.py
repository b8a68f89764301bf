"""SwiGLU rows of the int8 quantizer and of the products, over the whole range of gates and in every
form a call takes (a warp or a CTA a row, rows on 16-byte boundaries or not, few rows in the product).

Bound, in units of 2^-24 relative: exponential 5 (the power of two's 2 ulp, a correction, a rounding),
sum 1, reciprocal 2 (1 ulp), two products and the scale's division 1 each: 11, and 16 are asked of the
scale; an integer is within 0.5 + 127 * 16 * 2^-24 of the exact quotient. A value below 2^-126 of the
exponential's may come out as 0: absolute 1e-35 times the other operand, far below the rows' largest.
"""

import numpy as np
import pytest

import vastloom_b200 as vb
from test_gpu_int8 import KIND, LEGACY, check_product, cuda, dev, dt, product, run_linear, torch  # noqa: F401

pytestmark = pytest.mark.gpu

TOL = 16 * 2.0 ** -24


def exact(gu, cols, limit=0.0):
    gate, up = gu[:, :cols].double().numpy(), gu[:, cols:].double().numpy()
    if limit:
        gate, up = np.minimum(gate, limit), np.clip(up, -limit, limit)
    e = np.exp(-np.abs(gate))
    return gate * np.where(gate > 0, 1.0, e) / (1 + e) * up


def quantize(dev, torch, gu, cols, limit=0.0):  # noqa: F811
    c = gu.cuda()
    rows, x_type = gu.shape[0], {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}[gu.dtype]
    q = torch.full((rows, cols), 99, dtype=torch.int8, device="cuda")
    s = torch.full((rows,), 99.0, device="cuda")
    dev.int8_quantize_device(c.data_ptr(), rows, cols, q.data_ptr(), s.data_ptr(), x_type=KIND[x_type],
                             x_stride=gu.shape[1], up_ptr=c.data_ptr() + cols * c.element_size(), swiglu_limit=limit,
                             stream=LEGACY)
    return q.cpu().numpy(), s.cpu().numpy()


def check(q, s, a):
    top = np.abs(a).max(axis=1)
    assert np.all(np.abs(s - top / 127) <= TOL * top / 127), float(np.max(np.abs(s - top / 127) * 127 / top) * 2.0 ** 24)
    off = np.abs(q - a * (127 / top)[:, None])
    assert np.all(off <= 0.5 + 127 * TOL), float(off.max())


FORMS = [(5, 64), (5, 77), (3, 1024), (2, 5000), (1030, 64), (1025, 77), (1027, 1024)]


@pytest.mark.parametrize("rows,cols", FORMS)
@pytest.mark.parametrize("x_type", ["f32", "f16", "bf16"])
def test_gates_at_the_ends_of_the_type(dev, torch, x_type, rows, cols):  # noqa: F811
    """The type's largest gates on both sides beside ordinary ones: rows that stay finite by the formula."""
    g = torch.Generator().manual_seed(cols)
    gu = 3 * torch.randn(rows, 2 * cols, generator=g)
    big = float(torch.finfo(dt(torch, x_type)).max)
    for r in range(rows):
        c = (7 * r) % cols
        if r % 5 == 0:
            gu[r, c], gu[r, cols + c] = big, 0.25
        elif r % 5 == 1:
            gu[r, c], gu[r, cols + c] = 0.71 * big, -0.5
        elif r % 5 == 2:
            gu[r, c], gu[r, cols + c] = -big, 1.0
        elif r % 5 == 3:
            gu[r, c], gu[r, cols + c] = big, 0.0
        else:
            gu[r, c], gu[r, cols + c] = min(1500.0, big), 1.0
    gu = gu.to(dt(torch, x_type))
    check(*quantize(dev, torch, gu, cols), exact(gu, cols))


@pytest.mark.parametrize("x_type", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 2, 6, 40])
def test_product_of_the_largest_gates(dev, torch, x_type, rows):  # noqa: F811
    K, N = 256, 48
    gu = torch.randn(rows, 2 * K, generator=torch.Generator().manual_seed(rows))
    gu[:, 9], gu[:, K + 9] = float(torch.finfo(dt(torch, x_type)).max), 2.0 ** -120
    gu = gu.to(dt(torch, x_type))
    rng = np.random.default_rng(rows)
    w, sw = rng.integers(-127, 128, (1, N, K), dtype=np.int8), rng.random((1, N), np.float32)
    guc = gu.cuda()
    y = run_linear(dev, torch, guc, cuda(torch, w), cuda(torch, sw), x_type=x_type, cols=K, x_stride=2 * K,
                   up_ptr=guc.data_ptr() + K * guc.element_size())
    q, s = quantize(dev, torch, gu, K)
    check_product(y.cpu().numpy(), product(q, s, w[0], sw[0]), "f32")


@pytest.mark.parametrize("rows,cols", [(8, 64), (8, 77), (1030, 96)])
@pytest.mark.parametrize("x_type", ["f32", "f16", "bf16"])
def test_rows_of_far_gates(dev, torch, x_type, rows, cols):  # noqa: F811
    """Every gate of a row near -40, -50, ... -85: an error of the exponential that grows with the gate
    shows in the row's scale. (Values of 1e-35 and more: normal numbers, also divided by 127.)"""
    g = torch.Generator().manual_seed(cols)
    far = -torch.tensor([40.0, 50.0, 60.0, 70.0, 75.0, 80.0, 83.0, 85.0])[torch.arange(rows) % 8]
    gu = torch.empty(rows, 2 * cols)
    gu[:, :cols] = far[:, None] + torch.rand(rows, cols, generator=g) - 0.5
    gu[:, cols:] = 200 + 100 * torch.rand(rows, cols, generator=g)
    gu = gu.to(dt(torch, x_type))
    check(*quantize(dev, torch, gu, cols), exact(gu, cols))
