"""The report of int8 products whose waits ran out: one word a handle, in host memory, which the kernel
sets and vlb_int8_status reads and clears. The word is set here by the host; no wait is made to run out
on the GPU."""

import ctypes as C

import numpy as np
import pytest

import vastloom_b200 as vb

pytestmark = pytest.mark.gpu


def error_word(dev):
    fn = dev.lib["_ZN3vlb15int8_error_wordEP10vlb_handle"]
    fn.restype, fn.argtypes = C.POINTER(C.c_uint32), [C.c_void_p]
    return fn(dev.h)


def test_a_report_belongs_to_its_handle():
    with vb.Device(0, install_codebooks=False) as a, vb.Device(0, install_codebooks=False) as b:
        w, s = a.to_device(np.ones((4, 16), np.int8)), a.to_device(np.ones(4, np.float32))
        weights = vb.Int8Weights(w.address, s.address, 4, 16)
        x = np.ones((3, 16), np.float32)
        error_word(a)[0] = 1
        b.int8_status()
        assert b.int8_linear(weights, x).shape == (3, 4)  # asks for b's status: a's report stays
        with pytest.raises(vb.VlbError, match="ran out"):
            a.int8_status()
        a.int8_status()  # reported once
        error_word(a)[0] = 1
        with pytest.raises(vb.VlbError, match="ran out"):
            a.int8_linear(weights, x)
        assert np.array_equal(a.int8_linear(weights, x), b.int8_linear(weights, x))


def test_handles_in_several_threads():
    """The first products of several handles at once, one in each thread: equal to a later one."""
    from concurrent.futures import ThreadPoolExecutor

    rng = np.random.default_rng(0)
    w, s = rng.integers(-127, 128, (300, 512), dtype=np.int8), rng.random(300, np.float32)
    x = rng.standard_normal((40, 512)).astype(np.float32)

    def run(rows):
        with vb.Device(0, install_codebooks=False) as dev:
            wb, sb = dev.to_device(w), dev.to_device(s)
            weights = vb.Int8Weights(wb.address, sb.address, 300, 512)
            return [dev.int8_linear(weights, x[:rows]) for _ in range(10)]

    with ThreadPoolExecutor(6) as pool:
        runs = list(pool.map(run, [40, 40, 1, 3, 40, 17]))
    whole = run(40)[0]
    for got, rows in zip(runs, [40, 40, 1, 3, 40, 17]):
        assert all(np.array_equal(y, whole[:rows]) for y in got)


@pytest.mark.parametrize("cols", [1 << 31, (1 << 32) - 300, (1 << 32) - 1])
def test_quantizer_refuses_rows_past_32_bit_steps(cols):
    """On the host, before anything is launched."""
    with vb.Device(0, install_codebooks=False) as dev:
        buf = dev.buffer(4096)
        with pytest.raises(vb.VlbError, match="2\\^31 columns"):
            dev.int8_quantize_device(buf.address, 1, cols, buf.address + 1024, buf.address + 2048)
