"""The residual's addition with its RMS norm and int8 rows, and the gradient (vlb_add_rms_norm_device,
vlb_add_rms_norm_grad_device) against the formulas in 64 bits.

Bounds, in units u = 2^-24 of 32-bit rounding; K = cols / 32 + 16 bounds the additions in a row that any one
product passes through, a row being shared by 32 threads or more:
  * h is one addition: u |h|, and its type's rounding;
  * the mean of squares: h's rounding twice, the square's, K additions and a division: (K + 4) u relative,
    half of it in s, and the addition of eps and the root: (K / 2 + 4) u;
  * y = h s w: h, s and two (lifted: three) products: N = K / 2 + 8 units, and the type's rounding;
  * q is within 0.5 + 127 (2 N + 4) u of y / scale, the scale within (N + 2) u;
  * the gradient: s g within (K / 2 + 8) u; s n mean(g n) with the mean's sum within (K + N + 6) u of
    mean |g n|: (2 K + 30) u of |s n| mean |g n|; two additions of terms that size;
  * dweight: n and a product, and the additions over the rows, up to rows / 444 + 80 in a column:
    (N + rows / 444 + 80) u of the sum of |dy n|.
"""

import numpy as np
import pytest

import vastloom_b200 as vb

pytestmark = pytest.mark.gpu

LEGACY = 1  # cudaStreamLegacy, torch's default stream
U = 2.0 ** -24
KIND = {"f32": vb.DTYPE_F32, "f16": vb.DTYPE_F16, "bf16": vb.DTYPE_BF16}
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half a step of the subnormals (f32: a step)
PAIRS = [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")]
EPS = 1e-6


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


def dt(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def f64(t):
    return t.double().cpu().numpy()


def additions(cols):
    return cols / 32 + 16


def rows_of(torch, g, rows, cols, kind, scale=1.0, pad=0, shift=0):
    """A [rows, cols] view: `pad` more elements a row, the first row `shift` elements in."""
    ld = cols + pad
    flat = torch.zeros(rows * ld + shift, device="cuda", dtype=dt(torch, kind))
    view = flat[shift:].as_strided((rows, cols), (ld, 1))
    view.copy_((scale * torch.randn(rows, cols, device="cuda", generator=g)).to(dt(torch, kind)))
    return view


def exact_norm(x, r, w, eps):
    h = f64(x) + (0 if r is None else f64(r))
    s = 1.0 / np.sqrt(np.mean(h * h, axis=1, keepdims=True) + eps)
    return h, h * s * (1.0 if w is None else f64(w))


def check(got, want, bound, kind):
    got = f64(got)
    assert np.all(np.isfinite(got))
    over = np.abs(got - want) - (bound + UNIT[kind] * np.abs(want) * (1 + 2.0 ** -9) + TINY[kind])
    assert np.all(over <= 0), float(over.max())


def check_int8(q, scale, y, cols):
    n = additions(cols) / 2 + 8
    a = np.max(np.abs(y), axis=1)
    assert np.all(np.abs(f64(scale) - a / 127) <= (n + 2) * U * a / 127)
    q = f64(q)
    assert np.all(np.abs(q - y * (127 / a)[:, None]) <= 0.5 + 127 * (2 * n + 4) * U)
    assert np.all(np.max(np.abs(q), axis=1) == 127)


def forward(dev, torch, x, r, w, *, xt, rt, eps=EPS, h=None, y=None, q=None, scale=None, stream=LEGACY):
    p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    ld = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
    dev.add_rms_norm_device(p(x), x.shape[0], x.shape[1], x_type=KIND[xt], residual_type=KIND[rt], x_stride=ld(x),
                            residual_ptr=p(r), residual_stride=ld(r), weight_ptr=p(w), eps=eps, residual_out_ptr=p(h),
                            residual_out_stride=ld(h), y_ptr=p(y), y_stride=ld(y), q_ptr=p(q), q_stride=ld(q),
                            q_scale_ptr=p(scale), stream=stream)


SIZES = [(1, 1), (1, 7), (3, 8), (1, 4096), (2, 2048), (5, 1411), (64, 64), (33, 96), (300, 1000), (9, 4100), (130, 4096),
         (2100, 512), (1, 16384), (7, 12345), (3, 40000), (200, 1), (70, 3), (1000, 5), (65, 2049), (70, 8191)]


@pytest.mark.parametrize("xt,rt", PAIRS)
@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (3, 0), (3, 1)])
def test_norm_matches_the_formula(dev, torch, rows, cols, xt, rt, pad, shift):
    g = torch.Generator(device="cuda").manual_seed(rows * 131 + cols)
    x = rows_of(torch, g, rows, cols, xt, 1.0, pad, shift)
    r = rows_of(torch, g, rows, cols, rt, 3.0, pad, shift)
    w = 1.0 + 0.3 * torch.randn(cols + shift, device="cuda", generator=g)[shift:]
    h, y = (rows_of(torch, g, rows, cols, k, 1.0, pad, shift) for k in (rt, xt))
    q = torch.full((rows, cols + pad), 99, device="cuda", dtype=torch.int8)[:, :cols]
    scale = torch.zeros(rows, device="cuda")
    before = [t.as_strided((rows * (cols + pad),), (1,), shift * (t is not q)).clone() for t in (h, y, q)]
    forward(dev, torch, x, r, w, xt=xt, rt=rt, h=h, y=y, q=q, scale=scale)
    want_h, want_y = exact_norm(x, r, w, EPS)
    n = additions(cols) / 2 + 8
    check(h, want_h, U * np.abs(want_h), rt)
    check(y, want_y, n * U * np.abs(want_y), xt)
    check_int8(q, scale, want_y, cols)
    # what lies between the rows is left as it was
    for t, old in zip((h, y, q), before):
        now = t.as_strided((rows * (cols + pad),), (1,), shift * (t is not q))
        off = torch.arange(rows * (cols + pad), device="cuda") % (cols + pad) >= cols
        off[(rows - 1) * (cols + pad) + cols:] = False  # not this tensor's
        assert torch.equal(now[off], old[off])


@pytest.mark.parametrize("rows,cols,q_pad,q_shift", [(300, 1095, 9, 0), (300, 1095, 0, 3), (90, 2048, 5, 1), (3, 520, 1, 0)])
@pytest.mark.parametrize("xt,rt", [("bf16", "bf16"), ("f16", "f32"), ("f32", "f32")])
def test_int8_rows_at_an_offset_of_their_own(dev, torch, rows, cols, q_pad, q_shift, xt, rt):
    g = torch.Generator(device="cuda").manual_seed(cols)
    x, r = rows_of(torch, g, rows, cols, xt), rows_of(torch, g, rows, cols, rt)
    flat = torch.full((rows * (cols + q_pad) + q_shift,), 77, device="cuda", dtype=torch.int8)
    q = flat[q_shift:].as_strided((rows, cols), (cols + q_pad, 1))
    s, h = torch.zeros(rows, device="cuda"), torch.zeros_like(r)
    forward(dev, torch, x, r, None, xt=xt, rt=rt, h=h, q=q, scale=s)
    want_h, want = exact_norm(x, r, None, EPS)
    check(h, want_h, U * np.abs(want_h), rt)
    check_int8(q, s, want, cols)
    between = flat[q_shift: q_shift + (rows - 1) * (cols + q_pad)].view(rows - 1, cols + q_pad)[:, cols:]
    assert bool((between == 77).all()) and bool((flat[:q_shift] == 77).all())


def test_norm_of_more_elements_than_32_bits(dev, torch):
    """Offsets past 2^31 elements: the last rows of a large call, forward and gradient."""
    rows, cols = 530000, 4099
    x = torch.empty(rows, cols, device="cuda", dtype=torch.bfloat16).normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    y = torch.zeros_like(x)
    forward(dev, torch, x, None, None, xt="bf16", rt="bf16", y=y)
    dx = torch.zeros_like(x)
    backward(dev, torch, x, x, None, None, xt="bf16", rt="bf16", dx=dx)
    n = additions(cols) / 2 + 8
    for at in (slice(0, 3), slice(rows // 2, rows // 2 + 2), slice(rows - 3, rows)):
        _, want = exact_norm(x[at], None, None, EPS)
        check(y[at], want, n * U * np.abs(want), "bf16")
        d, bound, _, _ = exact_grad(x[at], x[at], None, None, EPS)
        check(dx[at], d, bound, "bf16")


@pytest.mark.parametrize("xt,rt", PAIRS)
def test_norm_outputs_one_by_one(dev, torch, xt, rt):
    g = torch.Generator(device="cuda").manual_seed(5)
    rows, cols = 37, 1024
    x, r = rows_of(torch, g, rows, cols, xt), rows_of(torch, g, rows, cols, rt)
    new = lambda k: torch.zeros(rows, cols, device="cuda", dtype=dt(torch, k))  # noqa: E731
    h, y, q, s = new(rt), new(xt), torch.zeros(rows, cols, device="cuda", dtype=torch.int8), torch.zeros(rows, device="cuda")
    forward(dev, torch, x, r, None, xt=xt, rt=rt, h=h, y=y, q=q, scale=s)
    for kw in ({"h": new(rt)}, {"y": new(xt)}, {"q": torch.zeros_like(q), "scale": torch.zeros_like(s)}):
        forward(dev, torch, x, r, None, xt=xt, rt=rt, **kw)
        for name, t in kw.items():
            assert torch.equal(t, {"h": h, "y": y, "q": q, "scale": s}[name])
    n = additions(cols) / 2 + 8
    _, want = exact_norm(x, None, None, EPS)  # no residual: h = x
    y2, h2 = new(xt), new(rt)
    forward(dev, torch, x, None, None, xt=xt, rt=rt, h=h2, y=y2)
    check(y2, want, n * U * np.abs(want), xt)
    assert torch.equal(h2, x.to(dt(torch, rt)))


@pytest.mark.parametrize("rows,cols", [(40, 2048), (40, 1001), (3, 50000)])
@pytest.mark.parametrize("xt,rt", PAIRS)
def test_norm_in_place(dev, torch, rows, cols, xt, rt):
    """The stream updated where it lies, and the norm over the branch's rows."""
    g = torch.Generator(device="cuda").manual_seed(6)
    x, r = rows_of(torch, g, rows, cols, xt), rows_of(torch, g, rows, cols, rt)
    h, y = torch.zeros_like(r), torch.zeros_like(x)
    forward(dev, torch, x, r, None, xt=xt, rt=rt, h=h, y=y)
    forward(dev, torch, x, r, None, xt=xt, rt=rt, h=r, y=x)
    assert torch.equal(r, h) and torch.equal(x, y)


@pytest.mark.parametrize("rows,cols", [(6, 512), (6, 999), (6, 30000)])
def test_norm_of_extreme_rows(dev, torch, rows, cols):
    """Zeros, values whose squares pass 32 bits, tiny ones, an infinity, a NaN: each row on its own."""
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(rows, cols, device="cuda", generator=g)
    x[0] = 0
    x[1] *= 1e30
    x[2] *= 1e-20
    x[3, cols // 2] = float("inf")
    x[4, 1] = float("nan")
    y, q, s = torch.zeros_like(x), torch.full(x.shape, 5, device="cuda", dtype=torch.int8), torch.zeros(rows, device="cuda")
    h = torch.zeros_like(x)
    forward(dev, torch, x, None, None, xt="f32", rt="f32", h=h, y=y, q=q, scale=s)
    n = additions(cols) / 2 + 8
    ok = [0, 1, 2, 5]
    _, want = exact_norm(x[ok], None, None, EPS)
    check(y[ok], want, n * U * np.abs(want), "f32")
    assert not q[0].any() and float(s[0]) == 0.0
    check_int8(q[[1, 2, 5]], s[[1, 2, 5]], want[1:], cols)
    y3 = f64(y[3])
    assert np.isnan(y3[cols // 2]) and not np.delete(y3, cols // 2).any()
    assert torch.isnan(y[4]).all()
    for i in (3, 4):
        assert torch.isnan(s[i]) and not q[i].any()
    assert torch.equal(h.nan_to_num(1.0), x.nan_to_num(1.0))


def exact_grad(dy, h, w, dh, eps):
    h, dy = f64(h), f64(dy)
    s = 1.0 / np.sqrt(np.mean(h * h, axis=1, keepdims=True) + eps)
    g, n = dy * (1.0 if w is None else f64(w)), h * s
    m, m_abs = np.mean(g * n, axis=1, keepdims=True), np.mean(np.abs(g * n), axis=1, keepdims=True)
    d = s * (g - n * m) + (0 if dh is None else f64(dh))
    k = additions(h.shape[1])
    bound = U * ((k / 2 + 8) * np.abs(s * g) + (2 * k + 30) * np.abs(s * n) * m_abs + 2 * np.abs(d) +
                 (0 if dh is None else np.abs(f64(dh))))
    w_bound = (k / 2 + 8 + h.shape[0] / 444 + 80) * U * np.sum(np.abs(dy * n), axis=0)
    return d, bound, np.sum(dy * n, axis=0), w_bound


def backward(dev, torch, dy, h, w, dh, *, xt, rt, eps=EPS, dx=None, dr=None, dw=None, stream=LEGACY):
    p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    ld = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
    nbytes = vb.add_rms_norm_grad_workspace_bytes(*h.shape)
    ws = torch.full((nbytes + 64,), 0xAB, device="cuda", dtype=torch.uint8)  # not cleared, and a guard behind
    dev.add_rms_norm_grad_device(p(dy), p(h), h.shape[0], h.shape[1], x_type=KIND[xt], residual_type=KIND[rt],
                                 dy_stride=ld(dy), h_stride=ld(h), weight_ptr=p(w), eps=eps, dh_ptr=p(dh), dh_stride=ld(dh),
                                 dx_ptr=p(dx), dx_stride=ld(dx), dresidual_ptr=p(dr), dresidual_stride=ld(dr),
                                 dweight_ptr=p(dw), ws_ptr=ws.data_ptr(), ws_bytes=nbytes, stream=stream)
    assert bool((ws[nbytes:] == 0xAB).all())


@pytest.mark.parametrize("xt,rt", PAIRS)
@pytest.mark.parametrize("rows,cols", SIZES + [(1500, 2048), (5000, 64), (1000, 1411)])
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (3, 0), (3, 1)])
def test_gradient_matches_the_formula(dev, torch, rows, cols, xt, rt, pad, shift):
    g = torch.Generator(device="cuda").manual_seed(rows * 17 + cols)
    dy = rows_of(torch, g, rows, cols, xt, 1.0, pad, shift)
    h, dh = rows_of(torch, g, rows, cols, rt, 3.0, pad, shift), rows_of(torch, g, rows, cols, rt, 1.0, pad, shift)
    w = 1.0 + 0.3 * torch.randn(cols + shift, device="cuda", generator=g)[shift:]
    dx, dr = (rows_of(torch, g, rows, cols, k, 1.0, pad, shift) for k in (xt, rt))
    dw = torch.full((cols + shift,), 7.0, device="cuda")[shift:]
    backward(dev, torch, dy, h, w, dh, xt=xt, rt=rt, dx=dx, dr=dr, dw=dw)
    d, bound, want_w, w_bound = exact_grad(dy, h, w, dh, EPS)
    check(dx, d, bound, xt)
    check(dr, d, bound, rt)
    check(dw, want_w, w_bound, "f32")
    again = torch.zeros_like(dw)
    backward(dev, torch, dy, h, w, dh, xt=xt, rt=rt, dw=again)  # equal inputs, equal bits; also alone
    assert torch.equal(again, dw)
    lone = torch.zeros(rows, cols, device="cuda", dtype=dt(torch, xt))
    backward(dev, torch, dy, h, w, dh, xt=xt, rt=rt, dx=lone)
    check(lone, d, bound, xt)


@pytest.mark.parametrize("rows,cols", [(50, 2048), (50, 1001), (3, 50000)])
@pytest.mark.parametrize("xt,rt", PAIRS)
def test_gradient_in_place(dev, torch, rows, cols, xt, rt):
    g = torch.Generator(device="cuda").manual_seed(8)
    dy, h, dh = rows_of(torch, g, rows, cols, xt), rows_of(torch, g, rows, cols, rt), rows_of(torch, g, rows, cols, rt)
    a = [torch.zeros_like(dy), torch.zeros_like(dh), torch.zeros(cols, device="cuda")]
    b = torch.zeros(cols, device="cuda")
    backward(dev, torch, dy, h, None, dh, xt=xt, rt=rt, dx=a[0], dr=a[1], dw=a[2])
    backward(dev, torch, dy, h, None, dh, xt=xt, rt=rt, dx=dy, dr=dh, dw=b)
    assert torch.equal(dy, a[0]) and torch.equal(dh, a[1]) and torch.equal(b, a[2])


@pytest.mark.parametrize("cols", [512, 999, 30000])
def test_gradient_of_extreme_rows(dev, torch, cols):
    g = torch.Generator(device="cuda").manual_seed(9)
    h, dy = (torch.randn(4, cols, device="cuda", generator=g) for _ in range(2))
    h[0] = 0
    h[1] *= 1e28
    h[2, 3] = float("nan")
    dx, dw = torch.zeros_like(h), torch.zeros(cols, device="cuda")
    backward(dev, torch, dy, h, None, None, xt="f32", rt="f32", dx=dx, dw=dw)
    ok = [0, 1, 3]
    d, bound, _, _ = exact_grad(dy[ok], h[ok], None, None, EPS)
    check(dx[ok], d, bound, "f32")
    assert torch.isnan(dx[2]).all() and torch.isnan(dw).all()  # the column sums take every row


def test_gradient_matches_differences(dev, torch):
    """dx and dweight against central differences of the forward kernel itself, along random directions.
    F = sum y * dy + sum h * dh. The step e = 2^-6 leaves a truncation that 64-bit differences show; the
    kernel's noise in F is within the bound of y (and u |h|) summed against |dy| (|dh|), twice over 2 e."""
    g = torch.Generator(device="cuda").manual_seed(10)
    rows, cols, e = 6, 640, 2.0 ** -6
    x, r, dy, dh = (torch.randn(rows, cols, device="cuda", generator=g) for _ in range(4))
    w = 1.0 + 0.3 * torch.randn(cols, device="cuda", generator=g)
    h = torch.zeros_like(x)
    forward(dev, torch, x, r, w, xt="f32", rt="f32", h=h)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    backward(dev, torch, dy, h, w, dh, xt="f32", rt="f32", dx=dx, dw=dw)

    def F(x, w):
        y, h = torch.zeros_like(x), torch.zeros_like(x)
        forward(dev, torch, x, r, w, xt="f32", rt="f32", y=y, h=h)
        return np.sum(f64(y) * f64(dy)) + np.sum(f64(h) * f64(dh))

    def F64(x, w):
        h = x + f64(r)
        y = h / np.sqrt(np.mean(h * h, axis=1, keepdims=True) + EPS) * w
        return np.sum(y * f64(dy)) + np.sum(h * f64(dh))

    want_h, want_y = exact_norm(x, r, w, EPS)
    n = additions(cols) / 2 + 10
    noise = 2 * (np.sum(n * U * np.abs(want_y * f64(dy))) + np.sum(2 * U * np.abs(want_h * f64(dh)))) / (2 * e) * 1.1
    _, bound, _, w_bound = exact_grad(dy, h, w, dh, EPS)
    for seed in range(3):
        v = torch.randn(rows, cols, device="cuda", generator=g)
        a, b = x + e * v, x - e * v
        mid = (f64(a) - f64(b)) / (2 * e)  # the step as it was rounded
        cut = (F64(f64(a), f64(w)) - F64(f64(b), f64(w))) / (2 * e)
        d, _, _, _ = exact_grad(dy, want(torch, want_h), w, dh, EPS)
        trunc = abs(cut - np.sum(d * mid))
        got = (F(a, w) - F(b, w)) / (2 * e)
        assert abs(got - np.sum(f64(dx) * mid)) <= noise + trunc + np.sum((bound + 2 * U * np.abs(d)) * np.abs(mid))
        u = torch.randn(cols, device="cuda", generator=g)
        a, b = w + e * u, w - e * u
        mid = (f64(a) - f64(b)) / (2 * e)
        got = (F(x, a) - F(x, b)) / (2 * e)  # linear in w: nothing is cut off
        assert abs(got - np.sum(f64(dw) * mid)) <= noise + np.sum((w_bound + 2 * U * np.abs(f64(dw))) * np.abs(mid))


def want(torch, a):
    return torch.from_numpy(a).cuda()


def test_gradient_of_no_rows(dev, torch):
    dw = torch.full((100,), 3.0, device="cuda")
    dev.add_rms_norm_grad_device(0, 0, 0, 100, dweight_ptr=dw.data_ptr(), stream=LEGACY)
    torch.cuda.synchronize()
    assert not dw.any()
    dev.add_rms_norm_device(0, 0, 100, y_ptr=dw.data_ptr(), stream=LEGACY)
    dev.add_rms_norm_grad_device(0, 0, 0, 100, dx_ptr=dw.data_ptr(), stream=LEGACY)
    assert not dw.any()


def test_norm_captured_and_on_other_streams(dev, torch):
    """Forward and gradient in one graph, replayed on inputs that change; then eagerly on the handle's stream."""
    g = torch.Generator(device="cuda").manual_seed(11)
    rows, cols = 77, 2048
    x, r, dy = (torch.randn(rows, cols, device="cuda", generator=g).bfloat16() for _ in range(3))
    w = torch.ones(cols, device="cuda")
    h, y, dx, dw = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x), torch.zeros(cols, device="cuda")
    nbytes = vb.add_rms_norm_grad_workspace_bytes(rows, cols)
    ws = torch.zeros(nbytes, device="cuda", dtype=torch.uint8)

    def both(stream):
        forward(dev, torch, x, r, w, xt="bf16", rt="bf16", h=h, y=y, stream=stream)
        dev.add_rms_norm_grad_device(dy.data_ptr(), h.data_ptr(), rows, cols, x_type=KIND["bf16"], residual_type=KIND["bf16"],
                                     weight_ptr=w.data_ptr(), eps=EPS, dx_ptr=dx.data_ptr(), dweight_ptr=dw.data_ptr(),
                                     ws_ptr=ws.data_ptr(), ws_bytes=nbytes, stream=stream)

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    both(side.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        both(side.cuda_stream)
    for seed in range(2):
        x.copy_(torch.randn(rows, cols, device="cuda", generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (h, y, dx, dw)]
        for t in (h, y, dx, dw):
            t.zero_()
        torch.cuda.synchronize()
        both(0)  # the handle's own stream
        dev.synchronize()
        for a, b in zip(got, (h, y, dx, dw)):
            assert torch.equal(a, b)


def test_host_form(dev):
    rng = np.random.default_rng(3)
    for xt, rt in ((np.float32, np.float32), (np.float16, np.float16), (np.float16, np.float32)):
        x, r = rng.standard_normal((5, 300)).astype(xt), rng.standard_normal((5, 300)).astype(rt)
        w = rng.standard_normal(300).astype(np.float32)
        h, y, q, s = dev.add_rms_norm(x, w, 1e-5, r)
        H = x.astype(np.float64) + r.astype(np.float64)
        Y = H / np.sqrt(np.mean(H * H, axis=1, keepdims=True) + 1e-5) * w
        unit = 2.0 ** -11 if xt == np.float16 else 2.0 ** -24
        assert h.dtype == rt and y.dtype == xt
        assert np.all(np.abs(h - H) <= (2.0 ** -11 if rt == np.float16 else U) * np.abs(H) * 1.01 + 2.0 ** -25)
        assert np.all(np.abs(y - Y) <= (unit + (additions(300) / 2 + 8) * U) * np.abs(Y) * 1.01 + 2.0 ** -25)
        assert np.all(np.abs(q * s[:, None] - Y) <= 0.51 * s[:, None])


def test_refusals(dev, torch):
    x = torch.zeros(4, 64, device="cuda")
    a = x.data_ptr()

    def refused(code, call, *args, **kw):
        with pytest.raises(vb.VlbError) as e:
            call(*args, **kw)
        assert e.value.code == code, e.value

    f, b = dev.add_rms_norm_device, dev.add_rms_norm_grad_device
    bad = "invalid_argument"
    refused(bad, f, a, 4, 64)  # no output
    refused(bad, f, 0, 4, 64, y_ptr=a)
    refused(bad, f, a, 4, 0, y_ptr=a)
    refused(bad, f, a, 4, 64, y_ptr=a, eps=0.0)
    refused(bad, f, a, 4, 64, y_ptr=a, eps=float("nan"))
    refused(bad, f, a, 4, 64, y_ptr=a, eps=float("inf"))
    refused(bad, f, a, 4, 64, y_ptr=a, x_stride=63)
    refused(bad, f, a, 4, 64, y_ptr=a + 2)
    refused(bad, f, a, 4, 64, y_ptr=a, x_type=vb.DTYPE_I8)
    refused(bad, f, a, 4, 64, y_ptr=a, x_type=vb.DTYPE_F16, residual_type=vb.DTYPE_BF16)
    refused(bad, f, a, 4, 64, y_ptr=a, x_type=vb.DTYPE_F32, residual_type=vb.DTYPE_BF16)
    refused(bad, f, a, 4, 64, q_ptr=a)
    refused(bad, f, a, 4, 64, y_ptr=a, q_scale_ptr=a)
    refused(bad, f, a, 4, 64, y_ptr=a, weight_ptr=a + 1)
    refused(bad, f, a, 1 << 31, 64, y_ptr=a)
    refused(bad, b, a, a, 4, 64)
    refused(bad, b, 0, a, 4, 64, dx_ptr=a)
    refused(bad, b, a, a, 4, 64, dweight_ptr=a)  # no workspace
    need = vb.add_rms_norm_grad_workspace_bytes(4, 64)
    refused(bad, b, a, a, 4, 64, dweight_ptr=a, ws_ptr=a, ws_bytes=need - 1)
    refused(bad, b, a, a, 4, 64, dweight_ptr=a, ws_ptr=a + 4, ws_bytes=need)
    refused(bad, b, a, a, 4, 64, dx_ptr=a, dx_stride=1)
    torch.cuda.synchronize()
    assert not x.any()
