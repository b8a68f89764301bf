"""Int8 products at the bounds of a launch's resources, each in a process that has made no other call.

A kernel that needs more shared memory than the default is opted in at its first such call, so a width
that is launched without the opt-in works after a wider call and fails before it: only a fresh process
shows it. Bound of a product: the integer sum is exact; its conversion and three products round once
each, relative 4 * 2^-24.
"""

import multiprocessing as mp

import numpy as np
import pytest

import vastloom_b200 as vb

pytestmark = pytest.mark.gpu


def quantized(x):
    """The quantizer's definition in 32-bit steps."""
    a = np.abs(x).max(axis=1)
    inv = (np.float32(127) / a).astype(np.float32)
    return np.rint(x * inv[:, None]).astype(np.int8), (a / np.float32(127)).astype(np.float32)


def _product(out, kind, rows, K, grouped):
    try:
        rng = np.random.default_rng(K + rows)
        N, G = 20, 3 if grouped else 1
        with vb.Device(0, install_codebooks=False) as dev:
            w, sw = rng.integers(-127, 128, (G, N, K), dtype=np.int8), rng.random((G, N), np.float32)
            bufs = [dev.to_device(w), dev.to_device(sw)]
            weights = vb.Int8Weights(bufs[0].address, bufs[1].address, N, K, groups=G)
            if kind == "i8":
                q, s = rng.integers(-127, 128, (rows, K), dtype=np.int8), rng.random(rows, np.float32)
                bufs += [dev.to_device(q), dev.to_device(s)]
                args = dict(x_type=vb.DTYPE_I8, x_scale_ptr=bufs[3].address)
            else:
                x = rng.standard_normal((rows, K)).astype(np.float16 if kind == "f16" else np.float32)
                q, s = quantized(x.astype(np.float32))
                need = vb.int8_workspace_bytes(rows, K)
                bufs += [dev.to_device(x), dev.buffer(need)]
                args = dict(x_type=vb.DTYPE_F16 if kind == "f16" else vb.DTYPE_F32, ws_ptr=bufs[3].address, ws_bytes=need)
            y = dev.buffer(rows * N * 4)
            group = np.zeros(rows, int)
            if grouped:  # the rows lie in groups 1 and 2
                bufs.append(dev.to_device(np.array([0, 0, 1, rows], np.uint32)))
                args["offsets_ptr"] = bufs[-1].address
                group = np.minimum(np.arange(rows), 1) + 1
            dev.int8_linear_device(weights, bufs[2].address, rows, y.address, **args)
            dev.int8_status()
            got = y.download(np.float32, rows * N).reshape(rows, N).astype(np.float64)
        want = np.einsum("rk,rnk->rn", q.astype(np.float64), w[group].astype(np.float64))
        want *= s.astype(np.float64)[:, None] * sw[group].astype(np.float64)
        excess = np.abs(got - want) - 4 * 2.0 ** -24 * np.abs(want)
        out.put(float(excess.max()))
    except BaseException as e:  # the parent has only this to go by
        out.put(repr(e))


# around 48 KB of quantized rows, with and without the kernel's own arrays, and at the most it takes
@pytest.mark.parametrize("kind", ["f32", "f16", "i8"])
@pytest.mark.parametrize("rows,K,grouped", [(2, 24064, False), (2, 24080, False), (2, 24576, False), (2, 32768, False),
                                            (1, 48128, False), (1, 48144, False), (1, 49152, False), (1, 65536, False),
                                            (2, 49152, True), (3, 65536, True)])
def test_few_rows_in_a_fresh_process(kind, rows, K, grouped):
    ctx = mp.get_context("spawn")
    out = ctx.Queue()
    p = ctx.Process(target=_product, args=(out, kind, rows, K, grouped))
    p.start()
    try:
        excess = out.get(timeout=120)
    finally:
        p.join(timeout=60)
        if p.is_alive():
            p.kill()
    assert isinstance(excess, float) and excess <= 0, excess
