"""Tokens sorted by expert and back (vlb_sort_tokens_device, vlb_combine_device, vlb_combine_grad_device)
against plain forms: the order in whole numbers, row copies bit for bit, sums in 64 bits.

Bounds, u = 2^-24: a combined element is k products and additions and the residual's addition in 32 bits, (k + 2) u
of the sum of the terms' magnitudes, and its type's rounding; drows one product; dweights H additions over at least 32
threads and one across them, (H / 32 + 24) u of the sum of magnitudes.
"""

import numpy as np
import pytest

import vastloom_b200 as vb

pytestmark = pytest.mark.gpu

LEGACY = 1
U = 2.0 ** -24
KIND = {"f32": vb.DTYPE_F32, "f16": vb.DTYPE_F16, "bf16": vb.DTYPE_BF16, "i8": vb.DTYPE_I8}
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}


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
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}[name]


def f64(t):
    return t.double().cpu().numpy()


def view(torch, rows, cols, kind, pad=0, shift=0, fill=None):
    flat = torch.zeros(rows * (cols + pad) + shift, device="cuda", dtype=dt(torch, kind))
    v = flat[shift:].as_strided((rows, cols), (cols + pad, 1))
    if fill is not None:
        v.copy_(fill.to(dt(torch, kind)) if fill.dtype != torch.int8 else fill)
    return v


def order_of(idx, mask, E):
    """(elem_row [T, k] with -1 for dropped, offsets, the live pairs in order) in plain Python terms."""
    T, k = idx.shape
    key = np.where((idx < E) & (mask[:, None] if mask is not None else True), idx, E).reshape(-1).astype(np.int64)
    order = np.argsort(key, kind="stable")
    order = order[key[order] < E]
    elem_row = np.full(T * k, -1, np.int64)
    elem_row[order] = np.arange(order.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(key, minlength=E + 1)[:E])])
    return elem_row.reshape(T, k), offsets, order


def route(rng, T, k, E, how):
    idx = rng.integers(0, E, (T, k)).astype(np.uint32)
    mask = None
    if how == "skewed":
        idx = np.minimum(rng.geometric(0.5, (T, k)) - 1, E - 1).astype(np.uint32)
    elif how == "one":  # a single expert takes all
        idx[:] = E - 1
    elif how == "dropped":
        idx[rng.random((T, k)) < 0.3] = E
        idx[rng.random((T, k)) < 0.1] = 0xFFFFFFFF
        mask = rng.random(T) < 0.7
    elif how == "none":
        mask = np.zeros(T, bool)
    elif how == "distinct":
        idx = np.argsort(rng.random((T, E)), axis=1)[:, :k].astype(np.uint32)
    return idx, mask


def sort(dev, torch, idx, mask, E, *, x=None, rows=None, kind="f32", weights=None, x_scale=None, stream=LEGACY, lean=False):
    T, k = idx.shape
    p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    i32 = lambda n: torch.full((n,), -7, device="cuda", dtype=torch.int32)  # noqa: E731
    out = {"elem_row": i32(T * k), "offsets": i32(E + 1)}
    if not lean:
        out["row_index"] = i32(T * k)
        if weights is not None:
            out["row_weight"] = torch.full((T * k,), -7.0, device="cuda")
        if x_scale is not None:
            out["row_scale"] = torch.full((T * k,), -7.0, device="cuda")
    nbytes = vb.sort_tokens_workspace_bytes(T, k, E)
    ws = torch.full((nbytes + 64,), 0xAB, device="cuda", dtype=torch.uint8)
    m = None if mask is None else torch.from_numpy(mask.astype(np.uint8)).cuda()
    i = torch.from_numpy(idx.astype(np.int64)).cuda().to(torch.int32) if T else torch.zeros(0, k, device="cuda", dtype=torch.int32)
    dev.sort_tokens_device(p(i), T, k, E, elem_row_ptr=p(out["elem_row"]), offsets_ptr=p(out["offsets"]), ws_ptr=p(ws),
                           ws_bytes=nbytes, x_ptr=p(x), H=0 if x is None else x.shape[1], x_type=KIND[kind],
                           x_stride=0 if x is None else x.stride(0), x_scale_ptr=p(x_scale), weights_ptr=p(weights),
                           mask_ptr=p(m), rows_ptr=p(rows), rows_stride=0 if rows is None else rows.stride(0),
                           row_scale_ptr=p(out.get("row_scale")), row_index_ptr=p(out.get("row_index")),
                           row_weight_ptr=p(out.get("row_weight")), stream=stream)
    torch.cuda.synchronize()
    assert bool((ws[nbytes:] == 0xAB).all())
    return out


ROUTES = [(1, 1, 1, "even"), (1, 8, 64, "distinct"), (3, 2, 5, "dropped"), (16, 6, 16, "one"), (64, 8, 256, "distinct"),
          (100, 8, 300, "dropped"), (129, 4, 1024, "even"), (511, 1, 7, "skewed"), (513, 3, 512, "dropped"), (1000, 64, 33, "even"),
          (2048, 8, 64, "skewed"), (4097, 8, 256, "dropped"), (9, 5, 3, "none"), (20000, 8, 128, "dropped"),
          (70001, 2, 1024, "skewed"), (30000, 7, 1, "dropped"), (131072, 8, 256, "dropped")]


@pytest.mark.parametrize("T,k,E,how", ROUTES)
def test_order(dev, torch, T, k, E, how):
    rng = np.random.default_rng(T + k + E)
    idx, mask = route(rng, T, k, E, how)
    weights = torch.from_numpy(rng.random((T, k), np.float32)).cuda()
    x_scale = torch.from_numpy(rng.random(T, np.float32)).cuda()
    got = sort(dev, torch, idx, mask, E, weights=weights, x_scale=x_scale)
    elem_row, offsets, order = order_of(idx, mask, E)
    n = order.size
    assert np.array_equal(got["elem_row"].cpu().numpy().reshape(T, k), elem_row)
    assert np.array_equal(got["offsets"].cpu().numpy(), offsets)
    index, weight, scale = (got[name].cpu().numpy() for name in ("row_index", "row_weight", "row_scale"))
    assert np.array_equal(index[:n], order // k) and np.all(index[n:] == -7)
    assert np.array_equal(weight[:n], weights.cpu().numpy().reshape(-1)[order]) and np.all(weight[n:] == -7)
    assert np.array_equal(scale[:n], x_scale.cpu().numpy()[order // k]) and np.all(scale[n:] == -7)
    lean = sort(dev, torch, idx, mask, E, lean=True)
    assert torch.equal(lean["elem_row"], got["elem_row"]) and torch.equal(lean["offsets"], got["offsets"])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("T,k,E,H,how", [(1, 8, 64, 4096, "distinct"), (5, 3, 4, 1, "dropped"), (64, 8, 256, 2048, "distinct"),
                                         (77, 6, 16, 1411, "dropped"), (300, 2, 8, 33, "skewed"), (1500, 8, 32, 520, "dropped"),
                                         (3000, 8, 64, 16, "even"), (9, 64, 40, 9000, "dropped"), (40, 8, 8, 24, "none"),
                                         (150, 8, 16, 6525, "even"), (2, 3, 4, 6234, "even"), (5000, 3, 9, 253, "dropped"),
                                         (1, 1, 1, 5, "even"), (33, 20, 7, 7, "even")])
@pytest.mark.parametrize("pad,shift", [(0, 0), (16, 0), (3, 1)])
def test_rows(dev, torch, T, k, E, H, how, kind, pad, shift):
    rng = np.random.default_rng(T * 7 + H)
    idx, mask = route(rng, T, k, E, how)
    bits = torch.from_numpy(rng.integers(0, 256, (T, H * SIZE[kind])).astype(np.uint8)).cuda()  # any bits: NaN too
    x = view(torch, T, H, kind, pad, shift)
    x.copy_(bits.view(dt(torch, kind)))
    rows = view(torch, T * k, H, kind, pad, shift)
    old = rows.as_strided((T * k * (H + pad),), (1,), shift)
    old.fill_(3)
    before = old.clone()
    got = sort(dev, torch, idx, mask, E, x=x, rows=rows, kind=kind, lean=True)
    elem_row, _, order = order_of(idx, mask, E)
    n = order.size
    assert np.array_equal(got["elem_row"].cpu().numpy().reshape(T, k), elem_row)
    as_bytes = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
    want = x[torch.from_numpy(order // k).cuda()]
    assert torch.equal(as_bytes(rows[:n]), as_bytes(want))
    wide = old.view(T * k, H + pad)
    was = before.view(T * k, H + pad)
    assert torch.equal(as_bytes(wide[n:]), as_bytes(was[n:])) and torch.equal(as_bytes(wide[:n, H:]), as_bytes(was[:n, H:]))


TYPES = [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"), ("f32", "bf16"), ("f32", "f16"),
         ("bf16", "f16"), ("f16", "bf16")]
SHAPES = [(1, 1, 1, 1, "even"), (1, 8, 64, 4096, "distinct"), (64, 8, 256, 2048, "dropped"), (7, 6, 16, 1411, "dropped"),
          (200, 3, 8, 40, "skewed"), (1000, 8, 64, 1024, "dropped"), (5, 64, 8, 520, "dropped"), (12, 2, 4, 9001, "none"),
          (3, 9, 4, 20000, "even"), (17, 17, 40, 256, "distinct"), (4000, 1, 3, 128, "dropped"), (900, 4, 8, 7, "dropped"),
          (600, 5, 16, 1003, "even")]


def placed(dev, torch, T, k, E, how, seed):
    rng = np.random.default_rng(seed)
    idx, mask = route(rng, T, k, E, how)
    elem_row, _, order = order_of(idx, mask, E)
    return elem_row, order.size, torch.from_numpy(elem_row).cuda().to(torch.int32)


@pytest.mark.parametrize("kind,out_kind", TYPES)
@pytest.mark.parametrize("T,k,E,H,how", SHAPES)
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (3, 0), (3, 1)])
def test_combine(dev, torch, T, k, E, H, how, kind, out_kind, pad, shift):
    elem_row, n, where = placed(dev, torch, T, k, E, how, T + H)
    g = torch.Generator(device="cuda").manual_seed(T + H)
    rows = view(torch, T * k, H, kind, pad, shift, torch.randn(T * k, H, device="cuda", generator=g))
    rows[n:] = float("nan")  # rows that no pair has are not read
    res = view(torch, T, H, out_kind, pad, shift, torch.randn(T, H, device="cuda", generator=g))
    w = torch.rand(T, k, device="cuda", generator=g) - 0.3
    w[where < 0] = float("nan")  # nor a dropped pair's weight
    for weights, residual in ((w, res), (None, None), (w, None), (None, res)):
        out = view(torch, T, H, out_kind, pad, shift)
        flat = out.as_strided((T * (H + pad),), (1,), shift)
        flat.fill_(5)
        dev.combine_device(rows.data_ptr(), where.data_ptr(), T, k, H, out.data_ptr(), x_type=KIND[kind],
                           y_type=KIND[out_kind], rows_stride=H + pad, weights_ptr=0 if weights is None else w.data_ptr(),
                           residual_ptr=0 if residual is None else res.data_ptr(), residual_stride=H + pad,
                           out_stride=H + pad, stream=LEGACY)
        v = np.where(elem_row[:, :, None] >= 0, f64(rows)[np.maximum(elem_row, 0)], 0.0)
        if weights is not None:
            v = v * np.where(elem_row >= 0, f64(w), 0.0)[:, :, None]
        want, size = v.sum(1), np.abs(v).sum(1)
        if residual is not None:
            want, size = want + f64(res), size + np.abs(f64(res))
        got = f64(out)
        bound = (k + 2) * U * size + UNIT[out_kind] * np.abs(want) * (1 + 2.0 ** -9) + UNIT[out_kind] * (k + 2) * U * size
        assert np.all(np.abs(got - want) <= bound + TINY[out_kind])
        if pad:
            assert bool((flat.view(T, H + pad)[: T - 1, H:] == 5).all())
    if shift == 0:  # onto the residual itself
        want = view(torch, T, H, out_kind, pad)
        for out in (want, res):
            dev.combine_device(rows.data_ptr(), where.data_ptr(), T, k, H, out.data_ptr(), x_type=KIND[kind],
                               y_type=KIND[out_kind], rows_stride=H + pad, residual_ptr=res.data_ptr(),
                               residual_stride=H + pad, out_stride=H + pad, stream=LEGACY)
        assert torch.equal(res, want)


def test_combine_takes_any_rows(dev, torch):
    """elem_row need not come from a sort: rows named twice, numbers past the rows, fewer rows than pairs, none."""
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randn(3, 64, device="cuda", generator=g)
    where = torch.tensor([[0, 0], [2, 3], [-1, 1], [1 << 30, 2]], device="cuda", dtype=torch.int32)
    out = torch.zeros(4, 64, device="cuda")
    dev.combine_device(rows.data_ptr(), where.data_ptr(), 4, 2, 64, out.data_ptr(), n_rows=3, stream=LEGACY)
    assert torch.equal(out, torch.stack([rows[0] + rows[0], rows[2], rows[1], rows[2]]))
    dev.combine_device(0, where.data_ptr(), 4, 2, 64, out.data_ptr(), n_rows=0, stream=LEGACY)
    assert not out.any()


@pytest.mark.parametrize("kind,out_kind", TYPES)
@pytest.mark.parametrize("T,k,E,H,how", SHAPES)
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (3, 1)])
def test_combine_gradient(dev, torch, T, k, E, H, how, kind, out_kind, pad, shift):
    elem_row, n, where = placed(dev, torch, T, k, E, how, T * 3 + H)
    g = torch.Generator(device="cuda").manual_seed(T + 2 * H)
    rows = view(torch, T * k, H, kind, pad, shift, torch.randn(T * k, H, device="cuda", generator=g))
    rows[n:] = float("nan")
    dout = view(torch, T, H, out_kind, pad, shift, torch.randn(T, H, device="cuda", generator=g))
    w = torch.rand(T, k, device="cuda", generator=g) - 0.3
    w[where < 0] = float("nan")
    live = elem_row >= 0
    at, t = elem_row[live], np.nonzero(live)[0]

    def call(weights, drows, dweights, rows=rows):
        p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        dev.combine_grad_device(dout.data_ptr(), where.data_ptr(), T, k, H, x_type=KIND[kind], y_type=KIND[out_kind],
                                dout_stride=H + pad, rows_ptr=p(rows), rows_stride=H + pad, weights_ptr=p(weights),
                                drows_ptr=p(drows), drows_stride=H + pad, dweights_ptr=p(dweights), stream=LEGACY)

    both = [None, None]
    for weights in (w, None):
        drows = view(torch, T * k, H, kind, pad, shift)
        flat = drows.as_strided((T * k * (H + pad),), (1,), shift)
        flat.fill_(5)
        dw = torch.full((T, k), 9.0, device="cuda")
        call(weights, drows, dw)
        want = np.zeros((T * k, H))
        want[at] = f64(dout)[t] * (1.0 if weights is None else f64(w)[live][:, None])
        got = f64(drows)
        assert np.all(np.abs(got - want)[:n] <= (U + UNIT[kind] * (1 + 2.0 ** -9)) * np.abs(want)[:n] + TINY[kind])
        assert np.all(got[n:] == 5)
        if pad:
            assert bool((flat.view(T * k, H + pad)[: T * k - 1, H:] == 5).all())
        prod = f64(dout)[t] * f64(rows)[at]
        got = f64(dw)
        assert np.all(np.abs(got[live] - prod.sum(1)) <= (H / 32 + 24) * U * np.abs(prod).sum(1) + 2.0 ** -149)
        assert not got[~live].any()
        both = [drows, dw]
    alone = view(torch, T * k, H, kind, pad, shift, rows)
    dw = torch.zeros(T, k, device="cuda")
    call(None, None, dw)
    assert torch.equal(dw, both[1])
    call(None, alone, None, rows=None)
    assert torch.equal(alone[:n], both[0][:n])
    call(None, rows, dw)  # the rows' gradient over the rows
    assert torch.equal(rows[:n], both[0][:n]) and torch.equal(dw, both[1])


def test_gradients_match_differences(dev, torch):
    """The chain x -> rows by expert -> weighted sum is linear in x and in the weights: central differences of the
    forward kernels have no truncation, and their noise is the bound of out summed against |dout|."""
    rng = np.random.default_rng(4)
    T, k, E, H, e = 40, 4, 8, 96, 0.5
    idx, mask = route(rng, T, k, E, "dropped")
    g = torch.Generator(device="cuda").manual_seed(2)
    x, dout = torch.randn(T, H, device="cuda", generator=g), torch.randn(T, H, device="cuda", generator=g)
    w = torch.rand(T, k, device="cuda", generator=g)

    def rows_of(x):
        rows = torch.zeros(T * k, H, device="cuda")
        got = sort(dev, torch, idx, mask, E, x=x, rows=rows)
        return rows, got["elem_row"]

    def F(x, w):
        rows, where = rows_of(x)
        out = torch.zeros(T, H, device="cuda")
        dev.combine_device(rows.data_ptr(), where.data_ptr(), T, k, H, out.data_ptr(), weights_ptr=w.data_ptr(), stream=LEGACY)
        return np.sum(f64(out) * f64(dout))

    rows, where = rows_of(x)
    drows, dw, dx = torch.zeros_like(rows), torch.zeros_like(w), torch.zeros_like(x)
    dev.combine_grad_device(dout.data_ptr(), where.data_ptr(), T, k, H, rows_ptr=rows.data_ptr(), weights_ptr=w.data_ptr(),
                            drows_ptr=drows.data_ptr(), dweights_ptr=dw.data_ptr(), stream=LEGACY)
    dev.combine_device(drows.data_ptr(), where.data_ptr(), T, k, H, dx.data_ptr(), stream=LEGACY)
    for _ in range(3):
        v, u = torch.randn(T, H, device="cuda", generator=g), torch.randn(T, k, device="cuda", generator=g)
        size = np.sum(np.abs(f64(dout)) * (np.abs(f64(x)) + e * np.abs(f64(v))) * (np.abs(f64(w)) + e * np.abs(f64(u))).sum(1)[:, None])
        noise = 4 * (k + 2) * U * size / (2 * e) * 2
        a, b = x + e * v, x - e * v
        assert abs((F(a, w) - F(b, w)) / (2 * e) - np.sum(f64(dx) * (f64(a) - f64(b)) / (2 * e))) <= noise
        a, b = w + e * u, w - e * u
        assert abs((F(x, a) - F(x, b)) / (2 * e) - np.sum(f64(dw) * (f64(a) - f64(b)) / (2 * e))) <= noise * (H / 32 + 24)


@pytest.mark.parametrize("H", [8192, 8195])
def test_more_elements_than_32_bits(dev, torch, H):
    """Rows past 2^31 elements: sorted, summed and their gradient, at the first, middle and last tokens."""
    T, k, E = 34000, 8, 64
    rng = np.random.default_rng(H)
    idx, _ = route(rng, T, k, E, "even")
    x = torch.empty(T, H, device="cuda", dtype=torch.bfloat16).normal_(generator=torch.Generator(device="cuda").manual_seed(3))
    rows = torch.zeros(T * k, H, device="cuda", dtype=torch.bfloat16)
    got = sort(dev, torch, idx, None, E, x=x, rows=rows, kind="bf16")
    elem_row, _, order = order_of(idx, None, E)
    assert np.array_equal(got["elem_row"].cpu().numpy().reshape(T, k), elem_row)
    for p in (0, 1, T * k // 2, T * k - 2, T * k - 1):
        assert torch.equal(rows[p], x[int(order[p]) // k])
    w = torch.rand(T, k, device="cuda")
    out, dw, drows = torch.zeros(T, H, device="cuda"), torch.zeros(T, k, device="cuda"), torch.zeros_like(rows)
    where = got["elem_row"]
    dev.combine_device(rows.data_ptr(), where.data_ptr(), T, k, H, out.data_ptr(), x_type=KIND["bf16"],
                       weights_ptr=w.data_ptr(), stream=LEGACY)
    dev.combine_grad_device(out.data_ptr(), where.data_ptr(), T, k, H, x_type=KIND["bf16"], rows_ptr=rows.data_ptr(),
                            weights_ptr=w.data_ptr(), drows_ptr=drows.data_ptr(), dweights_ptr=dw.data_ptr(), stream=LEGACY)
    torch.cuda.synchronize()
    for t in (0, 1, T // 2, T - 2, T - 1):
        v = f64(x[t])[None, :] * f64(w[t])[:, None]
        assert np.all(np.abs(f64(out[t]) - v.sum(0)) <= (k + 2) * U * np.abs(v).sum(0))
        prod = f64(out[t]) * f64(x[t])
        assert np.all(np.abs(f64(dw[t]) - prod.sum()) <= (H / 32 + 24) * U * np.abs(prod).sum())
        for s in range(k):
            want = f64(out[t]) * f64(w[t, s])
            assert np.all(np.abs(f64(drows[elem_row[t, s]]) - want) <= (U + UNIT["bf16"] * 1.01) * np.abs(want) + 2.0 ** -126)


def test_no_tokens(dev, torch):
    got = sort(dev, torch, np.zeros((0, 3), np.uint32), None, 5)
    assert not got["offsets"].any()
    out = torch.full((4,), 2.0, device="cuda")
    dev.combine_device(0, 0, 0, 1, 4, out.data_ptr(), stream=LEGACY)
    dev.combine_grad_device(0, 0, 0, 1, 4, dweights_ptr=out.data_ptr(), stream=LEGACY)
    assert bool((out == 2).all())


@pytest.mark.parametrize("T", [33, 5000])
def test_captured_replayed_and_two_streams(dev, torch, T):
    """Sort, combine and gradient in a graph, replayed over changed routes; two captured graphs with a workspace each
    run at once on two streams."""
    rng = np.random.default_rng(T)
    k, E, H = 8, 64, 256
    sides = [torch.cuda.Stream() for _ in range(2)]
    sets = []
    for side in sides:
        s = {"x": torch.randn(T, H, device="cuda").bfloat16(), "w": torch.rand(T, k, device="cuda"),
             "idx": torch.zeros(T, k, device="cuda", dtype=torch.int32),
             "rows": torch.zeros(T * k, H, device="cuda", dtype=torch.bfloat16), "elem": torch.zeros(T * k, device="cuda", dtype=torch.int32),
             "off": torch.zeros(E + 1, device="cuda", dtype=torch.int32), "out": torch.zeros(T, H, device="cuda"),
             "dx": torch.zeros(T, H, device="cuda"), "dw": torch.zeros(T, k, device="cuda")}
        nbytes = vb.sort_tokens_workspace_bytes(T, k, E)
        s["ws"] = torch.zeros(nbytes, device="cuda", dtype=torch.uint8)

        def run(s=s, stream=side.cuda_stream, nbytes=nbytes):
            p = {n: t.data_ptr() for n, t in s.items() if hasattr(t, "data_ptr")}
            dev.sort_tokens_device(p["idx"], T, k, E, elem_row_ptr=p["elem"], offsets_ptr=p["off"], ws_ptr=p["ws"],
                                   ws_bytes=nbytes, x_ptr=p["x"], H=H, x_type=KIND["bf16"], rows_ptr=p["rows"], stream=stream)
            dev.combine_device(p["rows"], p["elem"], T, k, H, p["out"], x_type=KIND["bf16"], weights_ptr=p["w"], stream=stream)
            dev.combine_grad_device(p["out"], p["elem"], T, k, H, x_type=KIND["bf16"], rows_ptr=p["rows"],
                                    weights_ptr=p["w"], dweights_ptr=p["dw"], stream=stream)

        s["run"] = run
        torch.cuda.synchronize()
        run()
        torch.cuda.synchronize()
        s["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s["graph"], stream=side):
            run()
        sets.append(s)
    for _ in range(3):
        routes = []
        for s in sets:
            idx, _ = route(rng, T, k, E, "dropped")
            routes.append(idx)
            s["idx"].copy_(torch.from_numpy(idx.astype(np.int64)).to(torch.int32))
        torch.cuda.synchronize()
        for s, side in zip(sets, sides):
            with torch.cuda.stream(side):
                s["graph"].replay()
        torch.cuda.synchronize()
        for s, idx in zip(sets, routes):
            elem_row, offsets, order = order_of(idx, None, E)
            assert np.array_equal(s["elem"].cpu().numpy().reshape(T, k), elem_row)
            assert np.array_equal(s["off"].cpu().numpy(), offsets)
            assert torch.equal(s["rows"][: order.size], s["x"][torch.from_numpy(order // k).cuda()])
            v = f64(s["x"])[:, None, :] * (f64(s["w"]) * (elem_row >= 0))[:, :, None]
            assert np.all(np.abs(f64(s["out"]) - v.sum(1)) <= (k + 2) * U * np.abs(v).sum(1))
            prod = f64(s["out"]) * f64(s["x"])
            dw = np.where(elem_row >= 0, prod.sum(1)[:, None], 0.0)
            assert np.all(np.abs(f64(s["dw"]) - dw) <= (H / 32 + 24) * U * np.abs(prod).sum(1)[:, None])


def test_refusals(dev, torch):
    z = torch.zeros(4096, device="cuda")
    a = z.data_ptr()

    def refused(code, call, *args, **kw):
        with pytest.raises(vb.VlbError) as e:
            call(*args, **kw)
        assert e.value.code == code, e.value

    bad, no = "invalid_argument", "unsupported"
    need = vb.sort_tokens_workspace_bytes(4, 2, 8)
    base = dict(elem_row_ptr=a, offsets_ptr=a, ws_ptr=a, ws_bytes=need)
    s, c, d = dev.sort_tokens_device, dev.combine_device, dev.combine_grad_device
    refused(bad, s, a, 4, 0, 8, **base)
    refused(bad, s, a, 4, 2, 0, **base)
    refused(no, s, a, 4, 65, 8, **base)
    refused(no, s, a, 4, 2, 1025, **base)
    refused(no, s, a, 1 << 26, 32, 8, **base)
    refused(bad, s, 0, 4, 2, 8, **base)
    refused(bad, s, a + 1, 4, 2, 8, **base)
    refused(bad, s, a, 4, 2, 8, **{**base, "ws_bytes": need - 1})
    refused(bad, s, a, 4, 2, 8, **{**base, "ws_ptr": a + 8})
    refused(bad, s, a, 4, 2, 8, **{**base, "offsets_ptr": 0})
    refused(bad, s, a, 4, 2, 8, row_weight_ptr=a, **base)
    refused(bad, s, a, 4, 2, 8, row_scale_ptr=a, **base)
    refused(bad, s, a, 4, 2, 8, rows_ptr=a, H=8, **base)
    refused(bad, s, a, 4, 2, 8, rows_ptr=a, x_ptr=a, H=0, **base)
    refused(bad, s, a, 4, 2, 8, rows_ptr=a, x_ptr=a, H=8, x_type=9, **base)
    refused(bad, s, a, 4, 2, 8, rows_ptr=a, x_ptr=a, H=8, x_stride=7, **base)
    refused(bad, s, a, 4, 2, 8, rows_ptr=a + 2, x_ptr=a, H=8, **base)
    refused(bad, c, a, a, 4, 0, 8, a)
    refused(bad, c, a, a, 4, 2, 0, a)
    refused(no, c, a, a, 4, 65, 8, a)
    refused(bad, c, a, a, 4, 2, 8, 0)
    refused(bad, c, a, 0, 4, 2, 8, a)
    refused(bad, c, 0, a, 4, 2, 8, a)
    refused(bad, c, a, a, 4, 2, 8, a, x_type=vb.DTYPE_I8)
    refused(bad, c, a, a, 4, 2, 8, a, out_stride=4)
    refused(bad, c, a, a, 4, 2, 8, a, weights_ptr=a + 2)
    refused(bad, d, a, a, 4, 2, 8)
    refused(bad, d, a, a, 4, 2, 8, dweights_ptr=a)  # no rows
    refused(bad, d, 0, a, 4, 2, 8, drows_ptr=a)
    refused(bad, d, a, a, 4, 2, 8, drows_ptr=a, y_type=vb.DTYPE_I8)
    refused(bad, d, a, a, 4, 2, 8, drows_ptr=a, drows_stride=3)
    torch.cuda.synchronize()
    assert not z.any()
