"""The forms of vlb_int8_linear_act_device beside each other: rows of y and residual on 16-byte boundaries whose last
columns fill no 16 bytes, and the sign of a zero. Bounds as in test_gpu_act_linear.py."""

import pytest

import vastloom_b200 as vb
from test_gpu_act_linear import ACTS, Case, dt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if vb.device_count() == 0:
        pytest.fail("no CUDA device: GPU tests must run on a B200")
    d = vb.Device(0, install_codebooks=False)
    yield d
    d.int8_status()
    d.close()


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("rows,K,N", [(130, 1024, 4096), (700, 96, 1030), (1500, 512, 2050), (2100, 256, 1028), (300, 256, 134)])
@pytest.mark.parametrize("x,y", [("i8", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f32")])
def test_rows_on_16_bytes(dev, torch, rows, K, N, act, x, y):
    """One CTA a tile and pairs; the columns between a row and the next are left as they were."""
    ny = N // 2 if act == "swiglu" else N
    c = Case(torch, rows + K + N, rows, K, N, x=x, y=y, swiglu=act == "swiglu", res_pad=-ny % 8 + 8)
    got = c.run(dev, torch, act)
    c.check(got, act)
    assert bool((got[:, ny:] == 9).all())


# few rows, a split K, one CTA a tile, pairs, and rows of w off 16-byte boundaries; y on 16 bytes and off
FORMS = [(1, 512, 512, 0), (3, 256, 130, 0), (8, 256, 512, 0), (100, 4096, 512, 0), (700, 96, 1030, 0), (1500, 512, 2048, 0),
         (50, 100, 66, 100)]


@pytest.mark.parametrize("rows,K,N,ld", FORMS)
@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("y", ["f32", "bf16"])
@pytest.mark.parametrize("grouped", [False, True])
def test_sign_of_zero(dev, torch, rows, K, N, ld, pad, y, grouped):
    """Without a residual y is the route weight times act(z): -0 where that is, in every form; with one of +0, +0."""
    c = Case(torch, 1, rows, K, N, G=2 if grouped else 1, x="f32", y=y, ld=ld, residual=False, res_pad=pad,
             offsets=[0, rows // 2, rows] if grouped else None)
    c.bias.fill_(-1e4)  # far below any product: RELU gives +0
    c.weight.fill_(-0.5)
    c.weight[::2] = 0.5
    want = torch.zeros(rows, N, device="cuda", dtype=torch.bool)
    want[1::2] = True
    got = c.run(dev, torch, "relu")[:, :N]
    assert not got.any() and torch.equal(torch.signbit(got), want)
    c.res = torch.zeros(rows, N + pad, device="cuda", dtype=dt(torch, y))
    got = c.run(dev, torch, "relu")[:, :N]
    assert not got.any() and not torch.signbit(got).any()
