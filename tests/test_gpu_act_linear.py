"""Int8 products with bias, activation, route weight and residual in the epilogue
(vlb_int8_linear_act_device) against 64-bit forms.

Bounds, u = 2^-24. The rows' integers and scales are the quantizer's, equal to the 32-bit definition.
  * z: the integer sum's conversion, the product with the row's scale and the last product and addition round once
    each: ez = 2 u |sum s w| + u |z|.
  * activations have slopes of at most 1.13 and add: RELU nothing; SILU 10 u |a| (exponential 5, sum 1, reciprocal 2,
    products 2); GELU 16 u |z| (its documentation); GELU_TANH 16 u |z| (argument 4 u |v| with |v| sigma' <= 0.23, then
    as SILU); SWIGLU |up| 1.1 ez(gate) + |silu| ez(up) + 12 u |a|.
  * the route weight and the residual round once, the output type once.
"""

import math

import numpy as np
import pytest

import vastloom_b200 as vb

pytestmark = pytest.mark.gpu

LEGACY = 1
U = 2.0 ** -24
KIND = {"f32": vb.DTYPE_F32, "f16": vb.DTYPE_F16, "bf16": vb.DTYPE_BF16, "i8": vb.DTYPE_I8}
UNIT = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
ACTS = {"none": vb.ACT_NONE, "relu": vb.ACT_RELU, "silu": vb.ACT_SILU, "gelu": vb.ACT_GELU, "gelu_tanh": vb.ACT_GELU_TANH,
        "swiglu": vb.ACT_SWIGLU}


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
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}[name]


def f64(t):
    return t.double().cpu().numpy()


def quantized(x):
    """The definition in 32-bit steps: (q, scale)."""
    x = np.asarray(x, np.float32)
    a = np.max(np.abs(x), axis=1).astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(a > 0, np.float32(127) / a, np.float32(0)).astype(np.float32)
    return np.rint(x * inv[:, None]), (a / np.float32(127)).astype(np.float32)


def sigmoid(v):
    return np.where(v >= 0, 1 / (1 + np.exp(-np.abs(v))), np.exp(-np.abs(v)) / (1 + np.exp(-np.abs(v))))


def activated(z, ez, act, limit):
    """(act(z), its error)."""
    if act == "none":
        return z, ez
    if act == "relu":
        return np.maximum(z, 0), ez
    if act == "silu":
        a = z * sigmoid(z)
        return a, 1.13 * ez + 10 * U * np.abs(a)
    if act == "gelu":
        a = 0.5 * z * np.vectorize(math.erfc)(-z / math.sqrt(2.0))
        return a, 1.13 * ez + 16 * U * np.abs(z)
    if act == "gelu_tanh":
        a = z * sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        return a, 1.13 * ez + 16 * U * np.abs(z)
    g, u, eg, eu = z[:, 0::2], z[:, 1::2], ez[:, 0::2], ez[:, 1::2]
    if limit:
        g, u = np.minimum(g, limit), np.clip(u, -limit, limit)
    s = g * sigmoid(g)
    return s * u, 1.13 * eg * np.abs(u) + np.abs(s) * eu + 12 * U * np.abs(s * u)


class Case:
    """Inputs of one product; groups G with `offsets` over the rows, w rows `ld` apart."""

    def __init__(self, torch, seed, rows, K, N, G=1, x="f32", y="f32", ld=0, bias=True, residual=True, weight=True,
                 swiglu=False, res_pad=0, offsets=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        self.rows, self.K, self.N, self.G, self.xt, self.yt = rows, K, N, G, x, y
        self.ld = ld or (K + 15) // 16 * 16
        flat = torch.randint(-127, 128, (G * N * self.ld + 16,), device="cuda", generator=g, dtype=torch.int8)
        self.w = flat[: G * N * self.ld].view(G, N, self.ld)
        self.ws = rnd(G, N).abs() * (0.02 / math.sqrt(K)) + 1e-4
        if x == "i8":
            xld = (K + 15) // 16 * 16
            self.x = torch.randint(-127, 128, (max(1, rows), xld), device="cuda", generator=g, dtype=torch.int8)
            self.x_scale = torch.rand(max(1, rows), device="cuda", generator=g) * 0.03 + 0.01
            self.q, self.s = f64(self.x[:rows, :K]), f64(self.x_scale)[:rows]
        else:
            self.x, self.x_scale = rnd(rows, K).to(dt(torch, x)), None
            self.q, s = quantized(self.x.float().cpu().numpy())
            self.s = s.astype(np.float64)
        self.bias = rnd(G, N) if bias else None
        self.ny = N // 2 if swiglu else N
        self.res_ld = self.ny + res_pad
        self.res = rnd(rows, self.res_ld).to(dt(torch, y)) if residual else None
        self.weight = torch.rand(rows, device="cuda", generator=g) - 0.2 if weight else None
        self.offsets = None if offsets is None else torch.tensor(offsets, device="cuda", dtype=torch.int32)
        self.at = [(0, rows)] if offsets is None else list(zip(offsets[:-1], offsets[1:]))

    def run(self, dev, torch, act, limit=0.0, y=None, stream=LEGACY, ws=None):
        p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        if y is None:
            y = torch.full((self.rows, self.res_ld), 9.0, device="cuda", dtype=dt(torch, self.yt))
        need = vb.int8_workspace_bytes(self.rows, self.K)
        ws = torch.empty(need + 16, device="cuda", dtype=torch.uint8) if ws is None else ws
        weights = vb.Int8Weights(p(self.w), p(self.ws), self.N, self.K, groups=self.G, stride=self.ld)
        dev.int8_linear_act_device(weights, p(self.x), self.rows, p(y), act=ACTS[act], act_limit=limit, bias_ptr=p(self.bias),
                                   residual_ptr=p(self.res), residual_stride=self.res_ld, x_type=KIND[self.xt],
                                   y_type=KIND[self.yt], x_stride=self.x.stride(0), x_scale_ptr=p(self.x_scale),
                                   row_weight_ptr=p(self.weight), offsets_ptr=p(self.offsets), y_stride=self.res_ld,
                                   ws_ptr=p(ws), ws_bytes=need, stream=stream)
        return y

    def want(self, act, limit=0.0):
        y, e = np.full((self.rows, self.ny), 9.0), np.zeros((self.rows, self.ny))
        for g, (lo, hi) in enumerate(self.at):
            t = (self.q[lo:hi] @ f64(self.w[g, :, : self.K]).T) * self.s[lo:hi, None] * f64(self.ws[g])
            z = t + (0 if self.bias is None else f64(self.bias[g]))
            a, ea = activated(z, 2 * U * np.abs(t) + U * np.abs(z), act, limit)
            rw = 1.0 if self.weight is None else f64(self.weight)[lo:hi, None]
            y[lo:hi] = rw * a + (0 if self.res is None else f64(self.res)[lo:hi, : self.ny])
            e[lo:hi] = np.abs(rw) * ea + U * np.abs(y[lo:hi])
        return y, e

    def check(self, got, act, limit=0.0, was=None):
        want, e = self.want(act, limit)
        bound = e * (1 + UNIT[self.yt]) + UNIT[self.yt] * np.abs(want) + (2.0 ** -25 if self.yt == "f16" else 2.0 ** -126)
        got = f64(got)[:, : self.ny]
        live = np.zeros(self.rows, bool)
        for lo, hi in self.at:
            live[lo:hi] = True
        over = (np.abs(got - want) - bound)[live]
        assert over.size == 0 or over.max() <= 0, float(over.max())
        if was is not None:
            assert np.array_equal(got[~live], f64(was)[~live, : self.ny])
        else:
            assert np.all(got[~live] == 9)


# each form of the product: few rows, one CTA a tile, a split K, pairs, and rows of w off 16-byte boundaries
DENSE = [(1, 512, 512, 0), (1, 64, 2, 0), (3, 777, 130, 0), (8, 256, 1000, 0), (40, 2048, 640, 0), (130, 1024, 4096, 0),
         (100, 4096, 512, 0), (700, 96, 1030, 0), (1500, 512, 2048, 0), (300, 1001, 258, 1001), (17, 33, 34, 35), (1, 40, 6, 41)]


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("rows,K,N,ld", DENSE)
@pytest.mark.parametrize("x,y", [("f32", "f32"), ("bf16", "bf16"), ("i8", "f16"), ("f16", "f32")])
def test_dense(dev, torch, rows, K, N, ld, act, x, y):
    c = Case(torch, rows + K + N, rows, K, N, x=x, y=y, ld=ld, swiglu=act == "swiglu", res_pad=3)
    c.check(c.run(dev, torch, act), act)


@pytest.mark.parametrize("act", ["none", "gelu", "swiglu"])
@pytest.mark.parametrize("rows,K,N,ld", [(2, 512, 512, 0), (90, 512, 256, 0), (600, 256, 1024, 0), (50, 100, 66, 100)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("weight", [False, True])
def test_parts_one_by_one(dev, torch, rows, K, N, ld, act, bias, residual, weight):
    c = Case(torch, rows + K, rows, K, N, x="f32", y="f32", ld=ld, bias=bias, residual=residual, weight=weight,
             swiglu=act == "swiglu")
    got = c.run(dev, torch, act)
    c.check(got, act)
    if act == "none" and not (bias or residual or weight):  # what the plain call gives, bit for bit
        y = torch.zeros_like(got)
        ws = torch.empty(vb.int8_workspace_bytes(rows, K) + 16, device="cuda", dtype=torch.uint8)
        dev.int8_linear_device(vb.Int8Weights(c.w.data_ptr(), c.ws.data_ptr(), N, K, stride=c.ld), c.x.data_ptr(), rows,
                               y.data_ptr(), ws_ptr=ws.data_ptr(), ws_bytes=vb.int8_workspace_bytes(rows, K), stream=LEGACY)
        assert torch.equal(y, got)


@pytest.mark.parametrize("rows,K,N", [(2, 256, 128), (64, 256, 128), (900, 256, 512)])
@pytest.mark.parametrize("limit", [0.0, 0.7])
def test_swiglu_limit(dev, torch, rows, K, N, limit):
    c = Case(torch, 3, rows, K, N, x="bf16", y="f32", swiglu=True)
    c.bias *= 4
    c.check(c.run(dev, torch, "swiglu", limit), "swiglu", limit)


# groups with none, one and many rows, rows of no group at the end, and offsets that fill the call
GROUPED = [(8, 256, 128, [0, 3, 3, 8]), (20, 512, 64, [0, 1, 2, 10, 20]), (64, 384, 256, [0, 0, 30, 30, 31, 50]),
           (700, 256, 512, [0, 300, 310, 310, 650]), (3000, 128, 256, [0, 1500, 1600, 2900]), (60, 100, 66, [0, 10, 50]),
           (5, 64, 32, [0, 0, 0])]


@pytest.mark.parametrize("act", ["none", "silu", "swiglu"])
@pytest.mark.parametrize("rows,K,N,offsets", GROUPED)
@pytest.mark.parametrize("x,y", [("f32", "f32"), ("i8", "bf16")])
@pytest.mark.parametrize("ld_odd", [False, True])
def test_grouped(dev, torch, rows, K, N, offsets, act, x, y, ld_odd):
    c = Case(torch, rows + N, rows, K, N, G=len(offsets) - 1, x=x, y=y, ld=K + 1 if ld_odd else 0, swiglu=act == "swiglu",
             offsets=offsets)
    c.check(c.run(dev, torch, act), act)


@pytest.mark.parametrize("act", ["none", "gelu_tanh", "swiglu"])
@pytest.mark.parametrize("rows,K,N,ld,offsets", [(4, 256, 128, 0, None), (100, 4096, 256, 0, None), (800, 256, 768, 0, None),
                                                 (70, 90, 40, 91, None), (600, 256, 256, 0, [0, 200, 500])])
def test_onto_the_residual(dev, torch, act, rows, K, N, ld, offsets):
    """y in the residual's memory: the same bits, and rows outside every group as they were."""
    c = Case(torch, 8, rows, K, N, G=1 if offsets is None else len(offsets) - 1, x="f32", y="bf16", ld=ld,
             swiglu=act == "swiglu", offsets=offsets)
    apart = c.run(dev, torch, act)
    c.check(apart, act)
    was = c.res.clone()
    c.run(dev, torch, act, y=c.res)
    live = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for lo, hi in c.at:
        live[lo:hi] = True
    assert torch.equal(c.res[live], apart[live]) and torch.equal(c.res[~live], was[~live])


@pytest.mark.parametrize("rows,K,N", [(3, 256, 128), (60, 512, 256), (900, 512, 768), (40, 90, 40)])
@pytest.mark.parametrize("up", [False, True])
def test_gathered_and_swiglu_rows_as_the_plain_call(dev, torch, rows, K, N, up):
    """Rows by index, SwiGLU of two operands, groups: what the plain call gives, bit for bit, where the epilogue adds
    nothing; and the residual on top of it, rounded once more."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows // 2 + 1, K, device="cuda", generator=g).bfloat16()
    u = torch.randn(rows // 2 + 1, K, device="cuda", generator=g).bfloat16() if up else None
    index = torch.randint(0, rows // 2 + 3, (rows,), device="cuda", generator=g, dtype=torch.int32)  # some past the rows
    offsets = torch.tensor([0, rows // 3, rows // 3, rows - 1], device="cuda", dtype=torch.int32)
    ld = (K + 15) // 16 * 16
    w = torch.randint(-127, 128, (3, N, ld), device="cuda", generator=g, dtype=torch.int8)
    ws = torch.rand(3, N, device="cuda", generator=g) * 0.01
    res = torch.randn(rows, N, device="cuda", generator=g)
    need = vb.int8_workspace_bytes(rows, K)
    scratch = torch.empty(need, device="cuda", dtype=torch.uint8)
    y = [torch.full((rows, N), 9.0, device="cuda") for _ in range(3)]
    kw = dict(x_type=KIND["bf16"], x_rows=x.shape[0], row_index_ptr=index.data_ptr(), up_ptr=u.data_ptr() if up else 0,
              swiglu_limit=2.0 if up else 0.0, offsets_ptr=offsets.data_ptr(), ws_ptr=scratch.data_ptr(), ws_bytes=need,
              stream=LEGACY)
    weights = vb.Int8Weights(w.data_ptr(), ws.data_ptr(), N, K, groups=3, stride=ld)
    dev.int8_linear_device(weights, x.data_ptr(), rows, y[0].data_ptr(), **kw)
    dev.int8_linear_act_device(weights, x.data_ptr(), rows, y[1].data_ptr(), **kw)
    dev.int8_linear_act_device(weights, x.data_ptr(), rows, y[2].data_ptr(), residual_ptr=res.data_ptr(), **kw)
    assert torch.equal(y[0], y[1])
    live = slice(0, rows - 1)
    assert torch.equal(y[2][live], y[0][live] + res[live]) and bool((y[2][rows - 1] == 9).all())


def test_rows_that_are_not_finite(dev, torch):
    """A row of NaN or infinities is NaN in its own outputs and nowhere else, through every activation."""
    for rows in (3, 300):
        for act in ACTS:
            c = Case(torch, 4, rows, 256, 128, x="f32", y="f32", swiglu=act == "swiglu")
            fine = c.run(dev, torch, act)
            c.x[1, 7] = float("nan")
            c.x[2, 9] = float("inf")
            got = c.run(dev, torch, act)
            assert torch.isnan(got[1:3]).all()
            rest = [0, *range(3, rows)]
            assert torch.equal(got[rest], fine[rest])


def test_captured_and_on_the_handles_stream(dev, torch):
    c = Case(torch, 5, 200, 512, 512, x="bf16", y="bf16", swiglu=True)
    ws = torch.empty(vb.int8_workspace_bytes(200, 512) + 16, device="cuda", dtype=torch.uint8)
    y = torch.zeros(200, 256, device="cuda", dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    c.run(dev, torch, "swiglu", y=y, stream=side.cuda_stream, ws=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        c.run(dev, torch, "swiglu", y=y, stream=side.cuda_stream, ws=ws)
    for _ in range(2):
        c.x.copy_(torch.randn_like(c.x.float()))
        c.res.copy_(torch.randn_like(c.res.float()))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        q, s = quantized(c.x.float().cpu().numpy())
        c.q, c.s = q, s.astype(np.float64)
        c.check(got, "swiglu")
        y.zero_()
        torch.cuda.synchronize()
        c.run(dev, torch, "swiglu", y=y, stream=0, ws=ws)
        dev.synchronize()
        assert torch.equal(y, got)


def test_refusals(dev, torch):
    z = torch.zeros(1 << 16, device="cuda")
    a = z.data_ptr()
    need = vb.int8_workspace_bytes(4, 32)
    base = dict(ws_ptr=a, ws_bytes=need)

    def refused(code, n=16, **kw):
        with pytest.raises(vb.VlbError) as e:
            dev.int8_linear_act_device(vb.Int8Weights(a, a, n, 32), a, 4, a, **{**base, **kw})
        assert e.value.code == code, e.value

    refused("invalid_argument", act=6)
    refused("invalid_argument", act=-1)
    refused("invalid_argument", n=15, act=vb.ACT_SWIGLU)
    refused("invalid_argument", act=vb.ACT_SWIGLU, act_limit=-1.0)
    refused("invalid_argument", act=vb.ACT_SWIGLU, act_limit=float("nan"))
    refused("invalid_argument", bias_ptr=a + 2)
    refused("invalid_argument", residual_ptr=a + 2)
    refused("invalid_argument", residual_ptr=a, residual_stride=15)
    refused("invalid_argument", act=vb.ACT_SWIGLU, residual_ptr=a, residual_stride=7)
    refused("invalid_argument", act=vb.ACT_SWIGLU, y_stride=7)
    refused("invalid_argument", y_stride=15)
    refused("invalid_argument", ws_bytes=need - 1)
    st = dev.lib.vlb_int8_linear_act_device(dev.h, None, vb._INT8_EPILOGUE_PACK(0, 0, 0, 0, 0.0), None)
    assert vb.ERROR_CODES[st] == "invalid_argument"
    st = dev.lib.vlb_int8_linear_act_device(dev.h, vb._INT8_LINEAR_PACK(*[0] * 21, 0.0, 0), None, None)
    assert vb.ERROR_CODES[st] == "invalid_argument"
    torch.cuda.synchronize()
    assert not z.any()
