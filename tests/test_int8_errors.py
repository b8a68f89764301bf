"""What the int8 host forms do with a product that reports an error: raised on the host, by a fake of
the library's calls."""

import numpy as np
import pytest

import vastloom_b200 as vb


class FakeLibrary:
    """The calls that Device.int8_linear makes; `status` is what the products report."""

    def __init__(self, status):
        self.status, self.calls = status, []

    def vlb_int8_linear_device(self, *a):
        self.calls.append("linear")
        return 0

    def vlb_int8_status(self, h, stream):
        self.calls.append("status")
        return self.status

    def vlb_last_error(self, h, buf, n):
        buf.value = b"internal_error: a wait inside an int8 product ran out"
        return 0


class FakeBuffer:
    address = 4096
    live = 0

    def __init__(self):
        FakeBuffer.live += 1

    def download(self, dtype, count):
        return np.zeros(count, dtype)

    def free(self):
        FakeBuffer.live -= 1


def device(status):
    dev = object.__new__(vb.Device)
    dev.lib, dev.h = FakeLibrary(status), None
    dev.to_device = lambda a, tag="": FakeBuffer()
    dev.buffer = lambda n, tag="": FakeBuffer()
    return dev


def test_host_product_raises_what_the_kernel_reports():
    w = vb.Int8Weights(4096, 4096, 8, 16)
    dev = device(10)
    with pytest.raises(vb.VlbError, match="ran out"):
        dev.int8_linear(w, np.zeros((2, 16), np.float32))
    assert dev.lib.calls == ["linear", "status"] and FakeBuffer.live == 0
    dev = device(0)
    assert dev.int8_linear(w, np.zeros((2, 16), np.float32)).shape == (2, 8)
    assert dev.lib.calls == ["linear", "status"] and FakeBuffer.live == 0
