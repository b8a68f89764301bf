"""Products on 8-bit integers (vlb_int8_quantize_device, vlb_int8_linear_device,
vlb_route_plan_device) against plain 64-bit forms.

Bounds, from the operations the entry points promise:
  * quantized integers and scales of plain rows: equal to the 32-bit definition, bit for bit;
  * SwiGLU rows: exp, sum, division, two products and the row's step are each within 2 units of
    2^-24, so q is within 0.5 + 127 * 16 * 2^-24 of the exact quotient and the scale within
    16 * 2^-24 relative;
  * products: the integer sum is exact; its conversion and three products round once each, and the
    output type once: relative 4 * 2^-24 + u, u = 0 / 2^-11 / 2^-8 for f32 / f16 / bf16 (f16 also
    2^-25 absolute below its normal range).
"""

import numpy as np
import pytest

import vastloom_b200 as vb

pytestmark = pytest.mark.gpu

LEGACY = 1  # cudaStreamLegacy, torch's default stream


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


def dt(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


KIND = {"f32": vb.DTYPE_F32, "f16": vb.DTYPE_F16, "bf16": vb.DTYPE_BF16, "i8": vb.DTYPE_I8}
UNIT = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def quantized(x):
    """The definition in 32-bit steps on a float32 array: (q, scale)."""
    x = np.asarray(x, np.float32)
    a = np.max(np.abs(x), axis=1).astype(np.float32)
    lift = np.where(a < np.float32(2.0 ** -100), np.float32(2.0 ** 100), np.float32(1))
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        inv = np.where(a > 0, np.float32(127) / (a * lift), np.float32(0)).astype(np.float32)
        q = np.rint((x * lift[:, None]) * inv[:, None])
    bad = ~np.isfinite(a)
    q[bad | (a == 0)] = 0
    s = (a / np.float32(127)).astype(np.float32)
    s[bad] = np.nan
    return q.astype(np.int8), s


def product(q, s, w, ws, rw=None):
    y = (q.astype(np.float64) @ w.astype(np.float64).T) * s.astype(np.float64)[:, None]
    y *= ws.astype(np.float64)[None, :]
    return y if rw is None else y * rw.astype(np.float64)[:, None]


def check_product(got, want, y):
    got = got.astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    bound = (4 * 2.0 ** -24 + UNIT[y]) * np.abs(want) + (2.0 ** -25 if y == "f16" else 0.0)
    assert np.all(np.abs(got - want)[ok] <= bound[ok]), float(np.max((np.abs(got - want) - bound)[ok]))


def run_linear(dev, torch, x, w, ws, *, x_type="f32", y_type="f32", w_stride=0, rows=None, y=None, ws_buf=None, **kw):
    """x, w, ws: CUDA tensors (w [groups, N, stride] int8)."""
    G, N, ld = w.shape
    K = kw.pop("cols", ld)
    rows = x.shape[0] if rows is None else rows
    y = torch.full((rows, N), 7.0, device="cuda", dtype=dt(torch, y_type)) if y is None else y
    W = vb.Int8Weights(w.data_ptr(), ws.data_ptr(), N, K, groups=G, stride=w_stride or ld)
    need = vb.int8_workspace_bytes(rows, K)
    buf = torch.full((max(need, 16),), 0x55, dtype=torch.uint8, device="cuda") if ws_buf is None else ws_buf
    dev.int8_linear_device(W, x.data_ptr(), rows, y.data_ptr(), x_type=KIND[x_type], y_type=KIND[y_type],
                           ws_ptr=buf.data_ptr(), ws_bytes=need, **{"stream": LEGACY, **kw})
    return y


def cuda(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ---- quantizer -------------------------------------------------------------------------------


@pytest.mark.parametrize("x_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (2, 31), (5, 64), (4, 129), (33, 1000), (2, 4096), (1, 20001)])
def test_quantize_equals_the_definition(dev, torch, x_type, rows, cols):
    g = torch.Generator().manual_seed(rows * 1000 + cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))).to(dt(torch, x_type))
    q = torch.full((rows, cols), 99, dtype=torch.int8, device="cuda")
    s = torch.full((rows,), 99.0, device="cuda")
    xc = x.cuda()
    dev.int8_quantize_device(xc.data_ptr(), rows, cols, q.data_ptr(), s.data_ptr(), x_type=KIND[x_type], stream=LEGACY)
    rq, rs = quantized(x.float().numpy())
    assert np.array_equal(q.cpu().numpy(), rq)
    assert np.array_equal(s.cpu().numpy().view(np.uint32), rs.view(np.uint32))


@pytest.mark.parametrize("cols", [5, 64, 512, 3001])
def test_quantize_rows_where_it_can_go_wrong(dev, torch, cols):
    """Zero rows, the smallest and largest magnitudes, one value alone, ties, NaN and infinities."""
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((12, cols)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e-44)
    x[2] *= np.float32(2.0 ** -110)
    x[3] = np.sign(x[3]) * np.float32(3.4e38)
    x[4] = 0
    x[4, cols - 1] = -2.5
    x[5] = np.arange(cols) % 255 - 127 + np.float32(0.5)
    x[5, 0] = 127
    x[6, cols // 2] = np.nan
    x[7, 0] = np.inf
    x[8, cols - 1] = -np.inf
    x[9] = np.nan
    x[10] = -0.0
    q, s = dev.int8_quantize(x)
    rq, rs = quantized(x)
    assert np.array_equal(q, rq)
    assert np.array_equal(np.isnan(s), np.isnan(rs)) and np.array_equal(s[~np.isnan(s)], rs[~np.isnan(rs)])


def test_quantize_strides_gather_and_missing_rows(dev, torch):
    """Rows of a wider matrix at an odd offset; an index outside x is a row of zeros."""
    base = torch.randn(9, 77).cuda()
    x = base[1:, 3:68]  # 8 rows, 65 columns, stride 77, 4-byte aligned only
    index = torch.tensor([7, 0, 0, 8, 3, -1], dtype=torch.int32).cuda()
    q = torch.full((6, 80), 99, dtype=torch.int8, device="cuda")
    s = torch.full((6,), 99.0, device="cuda")
    dev.int8_quantize_device(x.data_ptr(), 6, 65, q.data_ptr(), s.data_ptr(), x_stride=77, x_rows=8,
                             row_index_ptr=index.data_ptr(), q_stride=80, stream=LEGACY)
    xs = x.cpu().numpy()
    want = np.stack([xs[7], xs[0], xs[0], xs[0] * 0, xs[3], xs[0] * 0])
    rq, rs = quantized(want)
    assert np.array_equal(q.cpu().numpy()[:, :65], rq) and np.array_equal(s.cpu().numpy(), rs)
    assert torch.all(q[:, 65:] == 99)  # the pitch beyond the columns is the caller's


@pytest.mark.parametrize("x_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,limit", [(1, 8, 0.0), (3, 129, 0.0), (5, 256, 1.5), (2, 2048, 7.0), (40, 96, 0.25)])
def test_swiglu_rows(dev, torch, x_type, rows, cols, limit):
    g = torch.Generator().manual_seed(cols)
    gu = (3 * torch.randn(rows, 2 * cols, generator=g)).to(dt(torch, x_type))
    gu[0, :2] = torch.tensor([-90.0, 60.0])  # the exponential's far ends
    guc = gu.cuda()
    q = torch.zeros(rows, cols, dtype=torch.int8, device="cuda")
    s = torch.zeros(rows, device="cuda")
    dev.int8_quantize_device(guc.data_ptr(), rows, cols, q.data_ptr(), s.data_ptr(), x_type=KIND[x_type],
                             x_stride=2 * cols, up_ptr=guc.data_ptr() + cols * guc.element_size(), swiglu_limit=limit,
                             stream=LEGACY)
    gate, up = gu.double().numpy()[:, :cols], gu.double().numpy()[:, cols:]
    if limit:
        gate, up = np.minimum(gate, limit), np.clip(up, -limit, limit)
    a = gate / (1 + np.exp(-gate)) * up
    top = np.abs(a).max(axis=1)
    tol = 16 * 2.0 ** -24
    assert np.all(np.abs(s.cpu().numpy() - top / 127) <= tol * top / 127)
    assert np.all(np.abs(q.cpu().numpy() - a * (127 / top)[:, None]) <= 0.5 + 127 * tol)


def test_swiglu_nan_and_clamp_keep_a_nan(dev, torch):
    gu = torch.randn(3, 64)
    gu[1, 5] = float("nan")
    gu[2, 40] = float("nan")
    c = gu.cuda()
    q = torch.full((3, 32), 9, dtype=torch.int8, device="cuda")
    s = torch.zeros(3, device="cuda")
    dev.int8_quantize_device(c.data_ptr(), 3, 32, q.data_ptr(), s.data_ptr(), x_stride=64, up_ptr=c.data_ptr() + 128,
                             swiglu_limit=1.0, stream=LEGACY)
    assert np.array_equal(np.isnan(s.cpu().numpy()), [False, True, True])
    assert torch.all(q[1:] == 0)


# ---- one matrix ------------------------------------------------------------------------------


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 33, 64, 65, 128, 130, 257])
@pytest.mark.parametrize("N,K", [(1, 1), (8, 16), (100, 33), (128, 128), (129, 500), (300, 640), (65, 1040)])
def test_linear_int8_rows(dev, torch, M, N, K):
    """Given integers, at sizes around the tiles' edges; bytes past K are not the matrix's."""
    rng = np.random.default_rng(M * 7 + N * 3 + K)
    ld = (K + 15) // 16 * 16
    x, w = (rng.integers(-128, 128, (n, ld), dtype=np.int8) for n in (M, N))
    sx, sw = rng.random(M, np.float32) + np.float32(0.1), rng.standard_normal(N).astype(np.float32)
    xc, wc, sxc, swc = (cuda(torch, a) for a in (x, w[None], sx, sw[None]))
    y = run_linear(dev, torch, xc, wc, swc, x_type="i8", x_stride=ld, cols=K, x_scale_ptr=sxc.data_ptr())
    check_product(y.cpu().numpy(), product(x[:, :K], sx, w[:, :K], sw), "f32")


@pytest.mark.parametrize("x_type,y_type", [("f32", "f32"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"),
                                           ("bf16", "f32"), ("f16", "bf16")])
@pytest.mark.parametrize("M,N,K", [(1, 64, 256), (1, 2048, 2048), (3, 1000, 777), (16, 257, 1024), (77, 141, 1001),
                                   (200, 512, 640), (300, 130, 96)])
def test_linear_float_rows(dev, torch, x_type, y_type, M, N, K):
    g = torch.Generator().manual_seed(M + N + K)
    x = torch.randn(M, K, generator=g).to(dt(torch, x_type))
    rng = np.random.default_rng(K)
    ld = (K + 15) // 16 * 16
    w, sw = rng.integers(-127, 128, (N, ld), dtype=np.int8), rng.random(N, np.float32) * np.float32(0.01)
    q, s = quantized(x.float().numpy())
    y = run_linear(dev, torch, x.cuda(), cuda(torch, w[None]), cuda(torch, sw[None]), x_type=x_type, y_type=y_type, cols=K)
    check_product(y.float().cpu().numpy(), product(q, s, w[:, :K], sw), y_type)


@pytest.mark.parametrize("shift,ld", [(0, 131), (1, 144), (4, 132), (8, 136), (16, 144)])
@pytest.mark.parametrize("M", [1, 5, 40, 140])
def test_linear_alignments_and_strides(dev, torch, shift, ld, M):
    """Weight rows at every alignment, x rows of a wider matrix, y rows with a pitch."""
    rng = np.random.default_rng(ld)
    K, N = 131, 70
    flat = cuda(torch, rng.integers(-128, 128, shift + N * ld + 64, dtype=np.int8))
    w = flat[shift:shift + N * ld].view(1, N, ld)
    sw = cuda(torch, rng.random((1, N), np.float32))
    wide = torch.randn(M, 150).cuda()
    x = wide[:, 5:5 + K]
    y = torch.full((M, N + 3), 7.0, device="cuda")
    run_linear(dev, torch, x, w, sw, cols=K, x_stride=150, y=y, y_stride=N + 3)
    q, s = quantized(x.cpu().numpy())
    out = y.cpu().numpy()
    check_product(out[:, :N], product(q, s, w[0, :, :K].cpu().numpy(), sw[0].cpu().numpy()), "f32")
    assert np.all(out[:, N:] == 7.0)


@pytest.mark.parametrize("M", [1, 20, 130])
@pytest.mark.parametrize("pad", [0, 1])
def test_longest_row_of_the_largest_integers(dev, torch, M, pad):
    """131,071 products of -128 * -128: the sum's last bits in 32 bits, on both alignments."""
    K, N = 131071, 3
    ld = K + pad
    x = torch.full((M, ld), -128, dtype=torch.int8, device="cuda")
    w = torch.full((1, N, ld), -128, dtype=torch.int8, device="cuda")
    one, sw = torch.ones(M, device="cuda"), torch.ones(1, N, device="cuda")
    y = run_linear(dev, torch, x, w, sw, x_type="i8", x_stride=ld, cols=K, x_scale_ptr=one.data_ptr())
    assert torch.all(y == float(np.float32(131071 * 16384)))


@pytest.mark.parametrize("M,K", [(1, 256), (3, 100), (40, 256), (200, 384)])
def test_nan_stays_in_its_row(dev, torch, M, K):
    x = torch.randn(M, K)
    x[M - 1, K // 2] = float("nan")
    if M > 2:
        x[1, 0] = float("inf")
        x[0] = 0.0
    ld = (K + 15) // 16 * 16
    rng = np.random.default_rng(3)
    w, sw = rng.integers(-127, 128, (50, ld), dtype=np.int8), rng.random(50, np.float32)
    y = run_linear(dev, torch, x.cuda(), cuda(torch, w[None]), cuda(torch, sw[None]), cols=K)
    q, s = quantized(x.numpy())
    check_product(y.cpu().numpy(), product(q, s, w[:, :K], sw), "f32")


def test_no_rows_is_no_work(dev, torch):
    w, sw = torch.zeros(1, 4, 16, dtype=torch.int8, device="cuda"), torch.zeros(1, 4, device="cuda")
    W = vb.Int8Weights(w.data_ptr(), sw.data_ptr(), 4, 16)
    dev.int8_linear_device(W, 0, 0, 0)
    dev.int8_quantize_device(0, 0, 16, 0, 0)


def test_another_stream(dev, torch):
    """The call runs on the stream it is given, behind what that stream holds already."""
    s = torch.cuda.Stream()
    x = torch.zeros(32, 512, device="cuda")
    w = torch.randint(-127, 128, (1, 256, 512), dtype=torch.int8, device="cuda")
    sw = torch.rand(1, 256, device="cuda")
    src = torch.randn(32, 512).cuda()
    y = torch.zeros(32, 256, device="cuda")
    buf = torch.zeros(vb.int8_workspace_bytes(32, 512), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(20):
            x.add_(1.0)
        x.copy_(src)
        run_linear(dev, torch, x, w, sw, y=y, ws_buf=buf, stream=s.cuda_stream)
        x.zero_()
    s.synchronize()
    q, sc = quantized(src.cpu().numpy())
    check_product(y.cpu().numpy(), product(q, sc, w[0].cpu().numpy(), sw[0].cpu().numpy()), "f32")


@pytest.mark.parametrize("M", [1, 40, 700])
def test_inputs_written_just_before(dev, torch, M):
    """Weights and rows that the kernels ahead on the stream write, and rewrite as soon as the product
    has been enqueued: launches that come up early still see this call's."""
    K, N, n = 1024, 512, 6
    src_w, src_x = torch.randn(n, N, K).cuda(), torch.randn(n, M, K).cuda()
    w, sw = torch.zeros(1, N, K, dtype=torch.int8, device="cuda"), torch.zeros(1, N, device="cuda")
    x = torch.zeros(M, K, device="cuda")
    y = torch.zeros(n, M, N, device="cuda")
    buf = torch.zeros(vb.int8_workspace_bytes(M, K), dtype=torch.uint8, device="cuda")
    for i in range(n):
        dev.int8_quantize_device(src_w[i].data_ptr(), N, K, w.data_ptr(), sw.data_ptr(), stream=LEGACY)
        x.copy_(src_x[i])
        run_linear(dev, torch, x, w, sw, y=y[i], ws_buf=buf)
        x.fill_(float("nan"))
        w.fill_(1)
        sw.fill_(3.0)
    for i in range(n):
        qw, ws = quantized(src_w[i].cpu().numpy())
        q, s = quantized(src_x[i].cpu().numpy())
        check_product(y[i].cpu().numpy(), product(q, s, qw, ws), "f32")


@pytest.mark.parametrize("M", [3, 100, 600])
def test_two_streams_at_once(dev, torch, M):
    """Two streams with workspaces of their own, their calls interleaved."""
    K, N, n = 512, 1500, 8
    w, sw = torch.randint(-127, 128, (1, N, K), dtype=torch.int8, device="cuda"), torch.rand(1, N, device="cuda")
    x = [torch.randn(M, K).cuda() for _ in range(2)]
    y = [torch.zeros(n, M, N, device="cuda") for _ in range(2)]
    bufs = [torch.zeros(vb.int8_workspace_bytes(M, K), dtype=torch.uint8, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(n):
        for j in range(2):
            run_linear(dev, torch, x[j], w, sw, y=y[j][i], ws_buf=bufs[j], stream=streams[j].cuda_stream)
    torch.cuda.synchronize()
    for j in range(2):
        q, s = quantized(x[j].cpu().numpy())
        check_product(y[j][0].cpu().numpy(), product(q, s, w[0].cpu().numpy(), sw[0].cpu().numpy()), "f32")
        assert all(torch.equal(y[j][0], y[j][i]) for i in range(n))


def test_captured_in_a_graph(dev, torch):
    x = torch.randn(5, 256).cuda()
    w = torch.randint(-127, 128, (1, 300, 256), dtype=torch.int8, device="cuda")
    sw = torch.rand(1, 300, device="cuda")
    y = torch.zeros(5, 300, device="cuda")
    buf = torch.zeros(vb.int8_workspace_bytes(5, 256), dtype=torch.uint8, device="cuda")
    run_linear(dev, torch, x, w, sw, y=y, ws_buf=buf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run_linear(dev, torch, x, w, sw, y=y, ws_buf=buf, stream=torch.cuda.current_stream().cuda_stream)
    for k in range(2):
        x.copy_(torch.randn(5, 256))
        graph.replay()
        torch.cuda.synchronize()
        q, s = quantized(x.cpu().numpy())
        check_product(y.cpu().numpy(), product(q, s, w[0].cpu().numpy(), sw[0].cpu().numpy()), "f32")


# ---- groups ----------------------------------------------------------------------------------


@pytest.mark.parametrize("counts", [[1], [0, 3], [5, 0, 0, 1], [0, 0, 0], [16, 17, 1, 0, 40], [130, 1, 0, 257, 64],
                                    [1] * 9, [0, 300]])
@pytest.mark.parametrize("N,K", [(40, 48), (128, 256), (200, 500)])
def test_groups(dev, torch, counts, N, K):
    """Groups without a row, of one row, across tile edges; gathered rows and route weights."""
    rng = np.random.default_rng(len(counts) * 100 + N)
    G, rows, T = len(counts), sum(counts), 23
    ld = (K + 15) // 16 * 16
    off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    x = rng.standard_normal((T, K)).astype(np.float32)
    index = rng.integers(0, T, rows).astype(np.int32)
    rw = rng.random(rows, np.float32)
    w = rng.integers(-127, 128, (G, N, ld), dtype=np.int8)
    sw = rng.random((G, N), np.float32)
    xc, ic, rc, oc, wc, swc = (cuda(torch, a) for a in (x, index, rw, off, w, sw))
    y = run_linear(dev, torch, xc, wc, swc, rows=rows, cols=K, x_rows=T, row_index_ptr=ic.data_ptr() if rows else 0,
                   row_weight_ptr=rc.data_ptr() if rows else 0, offsets_ptr=oc.data_ptr())
    q, s = quantized(x)
    out = y.cpu().numpy()
    for g in range(G):
        sl = slice(off[g], off[g + 1])
        check_product(out[sl], product(q[index[sl]], s[index[sl]], w[g, :, :K], sw[g], rw[sl]), "f32")


@pytest.mark.parametrize("M,N,K", [(2049, 2600, 160), (1500, 4097, 400), (300, 20000, 129), (5000, 1030, 1024)])
def test_linear_large(dev, torch, M, N, K):
    """Products of many tiles: several a CTA, ragged at every edge."""
    rng = np.random.default_rng(M)
    ld = (K + 15) // 16 * 16
    x, w = (rng.integers(-128, 128, (n, ld), dtype=np.int8) for n in (M, N))
    sx, sw = rng.random(M, np.float32) + np.float32(0.1), rng.standard_normal(N).astype(np.float32)
    xc, wc, sxc, swc = (cuda(torch, a) for a in (x, w[None], sx, sw[None]))
    y = run_linear(dev, torch, xc, wc, swc, x_type="i8", x_stride=ld, cols=K, x_scale_ptr=sxc.data_ptr())
    check_product(y.cpu().numpy(), product(x[:, :K], sx, w[:, :K], sw), "f32")


@pytest.mark.parametrize("counts,N,K", [([700, 0, 300, 513, 1, 2000], 1100, 300), ([0, 1300, 1300], 2000, 64),
                                        ([400] * 20, 1000, 96), ([0, 5000, 3], 700, 500),
                                        ([9000, 0, 7411, 30], 300, 1037)])
def test_large_groups(dev, torch, counts, N, K):
    rng = np.random.default_rng(N)
    G, rows, T = len(counts), sum(counts), 900
    ld = (K + 15) // 16 * 16
    off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    x = rng.standard_normal((T, K)).astype(np.float32)
    index = rng.integers(0, T, rows).astype(np.int32)
    rw = rng.random(rows, np.float32)
    w, sw = rng.integers(-127, 128, (G, N, ld), dtype=np.int8), rng.random((G, N), np.float32)
    xc, ic, rc, oc, wc, swc = (cuda(torch, a) for a in (x, index, rw, off, w, sw))
    y = run_linear(dev, torch, xc, wc, swc, rows=rows, cols=K, x_rows=T, row_index_ptr=ic.data_ptr(),
                   row_weight_ptr=rc.data_ptr(), offsets_ptr=oc.data_ptr())
    q, s = quantized(x)
    out = y.cpu().numpy()
    for g in range(G):
        sl = slice(off[g], off[g + 1])
        check_product(out[sl], product(q[index[sl]], s[index[sl]], w[g, :, :K], sw[g], rw[sl]), "f32")


def test_gathered_rows_that_are_not_there(dev, torch):
    """Indices past x are rows of zeros, also where the rows are quantized apart from their copies."""
    rng = np.random.default_rng(12)
    T, K, N = 70, 1024, 40
    for rows in (6, 300, 16400):
        x, w = rng.standard_normal((T, K)).astype(np.float32), rng.integers(-127, 128, (1, N, K), dtype=np.int8)
        index = rng.integers(0, T + 9, rows).astype(np.int32)
        index[rows // 2] = -1
        sw = rng.random((1, N), np.float32)
        ic = cuda(torch, index)
        y = run_linear(dev, torch, cuda(torch, x), cuda(torch, w), cuda(torch, sw), rows=rows, x_rows=T,
                       row_index_ptr=ic.data_ptr()).cpu().numpy()
        there = (index >= 0) & (index < T)
        q, s = quantized(x)
        src = np.where(there, index, 0)
        check_product(y, product(q[src], s[src] * there, w[0], sw[0]), "f32")


@pytest.mark.parametrize("offsets", [[2, 5, 9], [0, 4, 100], [0, 7, 3], [50, 60, 70], [-1, 5, 9]])
def test_offsets_are_kept_inside_the_rows(dev, torch, offsets):
    """Ranges that start late, pass the rows, fall or lie outside: rows of no group stay as they are."""
    rng = np.random.default_rng(5)
    rows, K, N = 9, 64, 33
    x, w = rng.standard_normal((rows, K)).astype(np.float32), rng.integers(-127, 128, (2, N, K), dtype=np.int8)
    sw = rng.random((2, N), np.float32)
    oc = cuda(torch, np.array(offsets, np.int32))
    y = run_linear(dev, torch, cuda(torch, x), cuda(torch, w), cuda(torch, sw), offsets_ptr=oc.data_ptr()).cpu().numpy()
    q, s = quantized(x)
    want = np.full((rows, N), 7.0)
    u = np.array(offsets, np.int32).view(np.uint32).astype(np.int64)
    for g in range(2):
        lo, hi = min(u[g], rows), max(min(u[g], rows), min(u[g + 1], rows))
        want[lo:hi] = product(q[lo:hi], s[lo:hi], w[g], sw[g])
    check_product(y, want, "f32")


@pytest.mark.parametrize("y_type", ["f16", "bf16"])
@pytest.mark.parametrize("rows,K,N,G", [(6, 64, 48, 3), (100, 256, 128, 4), (1, 512, 96, 2)])
def test_swiglu_entry(dev, torch, y_type, rows, K, N, G):
    """SwiGLU rows into a grouped product: against the product of the quantizer's own integers."""
    g = torch.Generator().manual_seed(rows)
    gu = (2 * torch.randn(rows, 2 * K, generator=g)).to(dt(torch, y_type)).cuda()
    rng = np.random.default_rng(rows)
    w, sw = rng.integers(-127, 128, (G, N, K), dtype=np.int8), rng.random((G, N), np.float32) * np.float32(0.02)
    off = np.sort(rng.integers(0, rows + 1, G + 1)).astype(np.int32)
    off[0], off[-1] = 0, rows
    oc = cuda(torch, off)
    y = run_linear(dev, torch, gu, cuda(torch, w), cuda(torch, sw), x_type=y_type, y_type=y_type, cols=K, x_stride=2 * K,
                   up_ptr=gu.data_ptr() + 2 * K, swiglu_limit=2.0, offsets_ptr=oc.data_ptr())
    q, s = torch.zeros(rows, K, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
    dev.int8_quantize_device(gu.data_ptr(), rows, K, q.data_ptr(), s.data_ptr(), x_type=KIND[y_type], x_stride=2 * K,
                             up_ptr=gu.data_ptr() + 2 * K, swiglu_limit=2.0, stream=LEGACY)
    q, s, out = q.cpu().numpy(), s.cpu().numpy(), y.float().cpu().numpy()
    for e in range(G):
        sl = slice(off[e], off[e + 1])
        check_product(out[sl], product(q[sl], s[sl], w[e], sw[e]), y_type)


def test_equal_inputs_give_equal_bits(dev, torch):
    x = torch.randn(70, 1000).cuda()
    w = torch.randint(-127, 128, (3, 260, 1008), dtype=torch.int8, device="cuda")
    sw = torch.rand(3, 260, device="cuda")
    off = torch.tensor([0, 3, 60, 70], dtype=torch.int32).cuda()
    y = [run_linear(dev, torch, x, w, sw, cols=1000, offsets_ptr=off.data_ptr()) for _ in range(5)]
    assert all(torch.equal(y[0], v) for v in y)


def test_a_matrix_past_32_bit_offsets(dev, torch):
    """Weights and rows whose bytes lie beyond 2^31 and 2^32 from their starts."""
    G, N, K = 34, 4096, 32768  # 4.6 GB of weights; the last group's start past 2^32
    w = torch.zeros(G, N, K, dtype=torch.int8, device="cuda")
    w[G - 1] = torch.randint(-127, 128, (N, K), dtype=torch.int8, device="cuda")
    sw = torch.rand(G, N, device="cuda")
    x = torch.randn(3, K).cuda()
    off = torch.zeros(G + 1, dtype=torch.int32)
    off[G] = 3
    off = off.cuda()
    y = run_linear(dev, torch, x, w, sw, offsets_ptr=off.data_ptr())
    q, s = quantized(x.cpu().numpy())
    check_product(y.cpu().numpy(), product(q, s, w[G - 1].cpu().numpy(), sw[G - 1].cpu().numpy()), "f32")


# ---- route plan ------------------------------------------------------------------------------


@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (5, 2, 7), (64, 8, 256), (700, 3, 16)])
def test_route_plan(dev, torch, T, k, E):
    rng = np.random.default_rng(T)
    idx = np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32)
    wt = rng.random((T, k), np.float32)
    n = T * k
    ic, wc = cuda(torch, idx), cuda(torch, wt)
    ri, er = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
    rw, off = torch.zeros(n, device="cuda"), torch.zeros(E + 2, dtype=torch.int32, device="cuda")
    wsb = torch.zeros(int(dev.lib.vlb_ep_workspace_bytes(T, k, E)), dtype=torch.uint8, device="cuda")
    dev.route_plan_device(ic.data_ptr(), wc.data_ptr(), T, k, E, wsb.data_ptr(), ri.data_ptr(), rw.data_ptr(),
                          er.data_ptr(), off.data_ptr(), stream=LEGACY)
    order = np.argsort(idx.reshape(-1), kind="stable")
    assert np.array_equal(ri.cpu().numpy(), order // k)
    assert np.array_equal(rw.cpu().numpy(), wt.reshape(-1)[order])
    assert np.array_equal(er.cpu().numpy()[order], np.arange(n))
    assert np.array_equal(off.cpu().numpy()[:E + 1], np.concatenate([[0], np.cumsum(np.bincount(idx.reshape(-1), minlength=E))]))
    ic[T - 1, k - 1] = E
    with pytest.raises(vb.VlbError, match="invalid_format"):
        dev.route_plan_device(ic.data_ptr(), wc.data_ptr(), T, k, E, wsb.data_ptr(), ri.data_ptr(), rw.data_ptr(),
                              er.data_ptr(), off.data_ptr(), stream=LEGACY)


# ---- refusals --------------------------------------------------------------------------------


def refusals():
    return [
        (dict(rows=0, cols=0), "must be positive"),
        (dict(out_cols=0), "must be positive"),
        (dict(groups=0), "must be positive"),
        (dict(cols=131072), "131071"),
        (dict(groups=1025), "1024 groups"),
        (dict(groups=3), "offsets"),
        (dict(y_type=vb.DTYPE_I8), "y_type"),
        (dict(y_type=9), "y_type"),
        (dict(x_type=4), "x_type"),
        (dict(w=None), "null"),
        (dict(w_scale=None), "null"),
        (dict(y=None), "null"),
        (dict(x=None), "x is null"),
        (dict(y=2), "aligned"),
        (dict(w_scale=2), "aligned"),
        (dict(x=2), "x is null or not aligned"),
        (dict(x_stride=15), "x_stride"),
        (dict(w_stride=15), "stride"),
        (dict(y_stride=3), "stride"),
        (dict(x_rows=1), "fewer rows"),
        (dict(swiglu_limit=-1.0), "swiglu_limit"),
        (dict(swiglu_limit=float("nan")), "swiglu_limit"),
        (dict(x_scale=16), "x_scale"),
        (dict(ws=None), "workspace"),
        (dict(ws=8), "workspace"),
        (dict(ws_bytes=16), "workspace"),
        (dict(x_type=vb.DTYPE_I8), "x_scale"),
        (dict(x_type=vb.DTYPE_I8, x_scale=16, row_index=16), "neither"),
        (dict(x_type=vb.DTYPE_I8, x_scale=16, up=16), "neither"),
    ]


@pytest.mark.parametrize("change,words", refusals())
def test_refusals(dev, torch, change, words):
    """Each is refused on the host, before anything is launched."""
    import ctypes as C

    keep = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    p = keep.data_ptr()
    d = dict(x=p, x_stride=0, x_rows=0, row_index=None, up=None, x_scale=None, row_weight=None, w=p, w_scale=p,
             w_stride=0, offsets=None, y=p, y_stride=0, ws=p, ws_bytes=4096, rows=2, cols=16, out_cols=4, groups=1,
             x_type=vb.DTYPE_F32, y_type=vb.DTYPE_F32, swiglu_limit=0.0, reserved0=0)
    d.update({k: (p + v if k in ("x", "y", "ws", "w_scale", "x_scale", "row_index", "up") and v else v)
              for k, v in change.items()})
    st = dev.lib.vlb_int8_linear_device(dev.h, C.byref(vb._Int8LinearDesc(**d)), None)
    assert st in (1, 8)
    buf = C.create_string_buffer(512)
    dev.lib.vlb_last_error(dev.h, buf, 512)
    assert words in buf.value.decode(), buf.value.decode()


def test_null_arguments(dev):
    assert dev.lib.vlb_int8_linear_device(dev.h, None, None) == 1
    assert dev.lib.vlb_int8_linear_device(None, None, None) == 1
    for args in ((0, 0, 0), (4, 4, 0)):
        with pytest.raises(vb.VlbError):
            dev.int8_quantize_device(args[0], 1, 0, args[1], args[2])
    with pytest.raises(ValueError):
        dev.int8_quantize(np.zeros((2, 2), np.int32))
