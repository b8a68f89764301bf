"""Int8Experts.fill and fill_pairs take matrices: a source of another number of dimensions is refused before anything is
uploaded (a [n, cols, 2] one has twice the bytes of the [n, cols] buffer made for it)."""

import numpy as np
import pytest

from vastloom_b200.int8 import Int8Experts


class Refuses:
    """A device whose buffers are made and nothing else."""

    class Buffer:
        address = 4096

        def free(self):
            pass

    def __init__(self):
        self.made = 0

    def buffer(self, n, tag=""):
        self.made += 1
        if self.made > 2:
            raise AssertionError("touched the device")
        return self.Buffer()


@pytest.mark.parametrize("shape", [(), (16,), (4, 16, 2), (4, 16, 1), (1, 4, 16)])
def test_fill_takes_matrices(shape):
    with pytest.raises(ValueError):
        Int8Experts(Refuses(), 2, 4, 16).fill(0, 0, np.zeros(shape, np.float32))


@pytest.mark.parametrize("gate,up", [((2, 16, 2), (2, 16, 2)), ((2, 16), (2, 16, 2)), ((2, 16), (16,)), ((16,), (2, 16)),
                                     ((2, 16), (1, 16)), ((2, 15), (2, 15)), ((4, 16), (4, 16)), ((1, 16), (1, 16))])
def test_fill_pairs_takes_two_halves(gate, up):
    with pytest.raises(ValueError):
        Int8Experts(Refuses(), 2, 4, 16).fill_pairs(0, np.zeros(gate, np.float32), np.zeros(up, np.float32))
