"""Int8 products of few rows at the lengths where their quantizer takes four more elements a thread (four times 256, 128,
64 or 32 columns, by the rows of a block) and where a channel has one piece of 512 columns more: what quantizing first
and a product of the integer rows give, bit for bit, and that against the sum in 64 bits.

The integer sum's conversion, the product with the row's scale and that with the channel's round once each: 3 u |y|.
"""

import numpy as np
import pytest

import vastloom_b200 as vb

pytestmark = pytest.mark.gpu

LEGACY = 1
U = 2.0 ** -24


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


LENGTHS = [1, 15, 16, 17, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1009, 1023, 1024, 1025, 1536, 1537, 2047, 2048, 2049, 4096,
           4100, 8191]


@pytest.mark.parametrize("K", LENGTHS)
@pytest.mark.parametrize("rows", [1, 2, 3, 8])
@pytest.mark.parametrize("groups", [1, 3])
@pytest.mark.parametrize("up", [False, True])
def test_lengths(dev, torch, K, rows, groups, up):
    g = torch.Generator(device="cuda").manual_seed(K * 16 + rows)
    N, ld = 50, (K + 15) // 16 * 16
    w = torch.randint(-127, 128, (groups, N, ld), device="cuda", generator=g, dtype=torch.int8)
    ws = torch.rand(groups, N, device="cuda", generator=g) * 0.01 + 0.001
    weights = vb.Int8Weights(w.data_ptr(), ws.data_ptr(), N, K, groups=groups, stride=ld)
    at = [0, rows] if groups == 1 else [0, rows // 2, rows // 2, rows]
    offsets = torch.tensor(at, device="cuda", dtype=torch.int32)
    need = vb.int8_workspace_bytes(rows, K)
    scratch = torch.empty(need, device="cuda", dtype=torch.uint8)
    common = dict(offsets_ptr=offsets.data_ptr() if groups > 1 else 0, ws_ptr=scratch.data_ptr(), ws_bytes=need, stream=LEGACY)
    for kind, t in ((vb.DTYPE_F32, torch.float32), (vb.DTYPE_BF16, torch.bfloat16)):
        x, u = (torch.randn(rows, K, device="cuda", generator=g).to(t) for _ in range(2))
        x[0, K - 1] = 9  # the row's last column its largest
        y, direct = (torch.full((rows, N), 7.0, device="cuda") for _ in range(2))
        dev.int8_linear_device(weights, x.data_ptr(), rows, direct.data_ptr(), x_type=kind, up_ptr=u.data_ptr() if up else 0,
                               swiglu_limit=1.0 if up else 0.0, **common)
        q = torch.full((rows, ld), 99, device="cuda", dtype=torch.int8)
        s = torch.zeros(rows, device="cuda")
        dev.int8_quantize_device(x.data_ptr(), rows, K, q.data_ptr(), s.data_ptr(), x_type=kind, q_stride=ld,
                                 up_ptr=u.data_ptr() if up else 0, swiglu_limit=1.0 if up else 0.0, stream=LEGACY)
        dev.int8_linear_device(weights, q.data_ptr(), rows, y.data_ptr(), x_type=vb.DTYPE_I8, x_stride=ld,
                               x_scale_ptr=s.data_ptr(), **common)
        assert torch.equal(direct, y)
        for e in range(groups):
            lo, hi = at[e], at[e + 1]
            want = (q[lo:hi, :K].double() @ w[e, :, :K].double().T) * s[lo:hi, None].double() * ws[e].double()
            assert bool(((y[lo:hi].double() - want).abs() <= 3 * U * want.abs() * (1 + 1e-6)).all())
            assert not np.isnan(want.cpu().numpy()).any()
