"""The forms that larger calls of the int8 and balance operators take: a warp a row in the quantizer for
every type and width, pairs of CTAs with 16-bit results, the counts' clusters, the layer from every
storage type that needs no codebook. Bounds: those of the operators' own tests."""

import numpy as np
import pytest

import vastloom_b200 as vb
from test_gpu_balance import check as check_balance
from test_gpu_balance import plain as plain_balance
from test_gpu_balance import routes
from test_gpu_balance import run as run_balance
from test_gpu_int8 import KIND, LEGACY, check_product, cuda, dev, dt, product, quantized, run_linear, torch  # noqa: F401
from test_gpu_int8_layer import plain as plain_layer
from test_gpu_swiglu import check as check_swiglu
from test_gpu_swiglu import exact, quantize
from vastloom_b200 import synth
from vastloom_b200.int8 import Int8MoeLayer

pytestmark = pytest.mark.gpu


# ---- quantizer, 1,024 rows and more ----------------------------------------------------------------


@pytest.mark.parametrize("x_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,pad", [(1024, 8, 0), (1025, 500, 12), (1030, 1024, 0), (1024, 1030, 2), (1100, 2047, 1),
                                           (1024, 4096, 0), (1031, 4104, 0), (1024, 300, 1), (1024, 513, 0), (1027, 1100, 3)])
def test_quantize_a_warp_a_row(dev, torch, x_type, rows, cols, pad):  # noqa: F811
    """Rows that start on 16-byte boundaries or not (by their stride), that end inside a vector, zero and
    not-finite rows among them; q with a pitch."""
    g = torch.Generator().manual_seed(cols)
    x = torch.randn(rows, cols + pad, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))
    x[3] = 0
    x[700, cols - 1] = float("nan")
    x[900, 0] = -float("inf")
    x[1000] *= 2.0 ** -20 if x_type == "f16" else 2.0 ** -115
    x = x.to(dt(torch, x_type))
    ld = (cols + 15) // 16 * 16 + 16
    q = torch.full((rows, ld), 99, dtype=torch.int8, device="cuda")
    s = torch.full((rows,), 99.0, device="cuda")
    xc = x.cuda()
    dev.int8_quantize_device(xc.data_ptr(), rows, cols, q.data_ptr(), s.data_ptr(), x_type=KIND[x_type],
                             x_stride=cols + pad, q_stride=ld, stream=LEGACY)
    rq, rs = quantized(x[:, :cols].float().numpy())
    assert np.array_equal(q.cpu().numpy()[:, :cols], rq)
    assert torch.all(q[:, cols:] == 99)
    got = s.cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(rs)) and np.array_equal(got[~np.isnan(rs)], rs[~np.isnan(rs)])


@pytest.mark.parametrize("x_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,limit", [(1024, 512, 0.0), (1025, 1000, 2.0), (1024, 2048, 0.0), (1026, 2100, 0.0),
                                             (1024, 501, 1.0), (1024, 1027, 0.0), (512, 4099, 0.0)])
def test_swiglu_a_warp_a_row(dev, torch, x_type, rows, cols, limit):  # noqa: F811
    gu = 3 * torch.randn(rows, 2 * cols, generator=torch.Generator().manual_seed(cols))
    gu = gu.to(dt(torch, x_type))
    check_swiglu(*quantize(dev, torch, gu, cols, limit), exact(gu, cols, limit))


# ---- products ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("y_type", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("M,N,K", [(1100, 2100, 1000), (2048, 1024, 512), (700, 4096, 272)])
def test_dense_products_of_pairs(dev, torch, y_type, M, N, K):  # noqa: F811
    rng = np.random.default_rng(M)
    ld = (K + 15) // 16 * 16
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(K)).to(dt(torch, "bf16"))
    w, sw = rng.integers(-127, 128, (N, ld), dtype=np.int8), rng.random(N, np.float32) * np.float32(0.01)
    q, s = quantized(x.float().numpy())
    y = run_linear(dev, torch, x.cuda(), cuda(torch, w[None]), cuda(torch, sw[None]), x_type="bf16", y_type=y_type, cols=K)
    check_product(y.float().cpu().numpy(), product(q, s, w[:, :K], sw), y_type)


@pytest.mark.parametrize("x_type,y_type", [("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("counts,N,K", [([150, 0, 260, 101, 300, 1], 520, 300), ([257] * 7, 1030, 640),
                                        ([0, 0, 900, 31, 33], 256, 1040)])
def test_grouped_products_of_pairs(dev, torch, x_type, y_type, counts, N, K):  # noqa: F811
    """A hundred rows a group and more; gathered rows, weights, 16-bit results."""
    rng = np.random.default_rng(N)
    G, rows, T = len(counts), sum(counts), 400
    ld = (K + 15) // 16 * 16
    off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(N)).to(dt(torch, x_type))
    index, rw = rng.integers(0, T, rows).astype(np.int32), rng.random(rows, np.float32)
    w, sw = rng.integers(-127, 128, (G, N, ld), dtype=np.int8), rng.random((G, N), np.float32) * np.float32(0.01)
    ic, rc, oc = (cuda(torch, a) for a in (index, rw, off))
    y = run_linear(dev, torch, x.cuda(), cuda(torch, w), cuda(torch, sw), x_type=x_type, y_type=y_type, rows=rows, cols=K,
                   x_rows=T, row_index_ptr=ic.data_ptr(), row_weight_ptr=rc.data_ptr(), offsets_ptr=oc.data_ptr())
    q, s = quantized(x.float().numpy())
    out = y.float().cpu().numpy()
    for g in range(G):
        sl = slice(off[g], off[g + 1])
        check_product(out[sl], product(q[index[sl]], s[index[sl]], w[g, :, :K], sw[g], rw[sl]), y_type)


# ---- balance -------------------------------------------------------------------------------------------


@pytest.mark.parametrize("T,E,k,offsets", [(4097, 64, 8, None), (8200, 200, 3, None), (17000, 512, 1, None),
                                           (40000, 96, 2, None), (30000, 33, 5, [1, 29000, 29990])])
@pytest.mark.parametrize("masked", [False, True])
def test_counts_through_clusters(dev, torch, T, E, k, offsets, masked):  # noqa: F811
    rng = np.random.default_rng(T)
    z = rng.standard_normal((T, E)).astype(np.float32)
    idx = np.argsort(rng.random((T, E)), axis=1)[:, :k]
    mask = rng.random(T) < 0.7 if masked else None
    got = run_balance(dev, torch, torch.from_numpy(z).cuda(), idx, score="sigmoid", coef=2.0, mask=mask, offsets=offsets)
    check_balance(got, plain_balance(z, idx, "sigmoid", 2.0, mask, offsets), "f32")
    again = run_balance(dev, torch, torch.from_numpy(z).cuda(), idx, score="sigmoid", coef=2.0, mask=mask, offsets=offsets)
    assert again[0] == got[0] and np.array_equal(again[1], got[1]) and torch.equal(again[3], got[3])


def test_a_half_gradient_scaled_through_upstream(dev, torch):  # noqa: F811
    """f16 logits of a large batch: the gradient's elements lie below f16's smallest (6e-8) and are 0;
    with upstream 2^16 they are there, to f16's unit."""
    T, E, k = 20000, 64, 4
    rng = np.random.default_rng(1)
    z = torch.from_numpy(rng.standard_normal((T, E))).to(torch.float16)
    idx = routes(rng, T, E, k)
    want = plain_balance(z.double().numpy(), idx, "softmax", 0.01)
    assert np.abs(want[2]).max() < 6e-8 / 2
    assert np.all(run_balance(dev, torch, z.cuda(), idx, x="f16", coef=0.01)[2] == 0)
    up = 2.0 ** 16
    got = run_balance(dev, torch, z.cuda(), idx, x="f16", coef=0.01, up=up)
    check_balance(got, plain_balance(z.double().numpy(), idx, "softmax", 0.01, up=up), "f16")
    assert np.mean(got[2] != 0) > 0.9


# ---- layer ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["Q4_K", "Q5_K", "Q6_K", "MXFP4"])
def test_layer_from_every_codebook_free_type(dev, kind):  # noqa: F811
    """Rows of these synthetic blocks have their largest value at 5 to 8 deviations: 2 % of the norm for
    each weight rounding; with the tokens' 0.9 % and SwiGLU's 1.8 % the squares' root is 3.5 %, and 5 % is
    asked."""
    rng = np.random.default_rng(len(kind))
    E, I, H, k, T = 3, 256, 256, 2, 12
    t = getattr(vb, "TYPE_" + kind)
    make = lambda rows, cols, i: dev.upload_matrix(t, rows, cols,  # noqa: E731
                                                   synth.matrix(rng, t, rows, cols, synth.D_SCALE[t]), identity=500 + i)
    ms = [[make(I, H, i) for i in range(E)], [make(I, H, 10 + i) for i in range(E)], [make(H, I, 20 + i) for i in range(E)]]
    router = rng.standard_normal((E, H)).astype(np.float32) * 0.1
    x = rng.standard_normal((T, H)).astype(np.float32)
    layer = Int8MoeLayer(dev, router=router, w1=ms[0], w3=ms[1], w2=ms[2], top_k=k, max_tokens=T)
    try:
        out = layer.forward(x)
        idx, wt = dev.route(dev.router_logits(x, router), k)
        with np.errstate(over="ignore"):
            want = plain_layer(x, idx, wt, *[[dev.dequantize(m) for m in row] for row in ms], None, 0.0)
        assert np.linalg.norm(out - want) <= 0.05 * np.linalg.norm(want)
    finally:
        layer.close()
        for row in ms:
            for m in row:
                dev.release_matrix(m)
