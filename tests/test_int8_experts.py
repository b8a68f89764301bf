"""Int8Experts.fill refuses rows outside the matrices before it touches the device."""

import numpy as np
import pytest

from vastloom_b200.int8 import Int8Experts


class Refuses:
    """A device on which nothing may be done."""

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


@pytest.mark.parametrize("group,row0,n,cols", [(0, -1, 2, 16), (0, 3, 2, 16), (0, 0, 5, 16), (2, 0, 4, 16), (-1, 0, 4, 16),
                                               (0, 0, 4, 15), (1, -4, 4, 16)])
def test_fill_outside(group, row0, n, cols):
    experts = Int8Experts(Refuses(), 2, 4, 16)
    with pytest.raises(ValueError):
        experts.fill(group, row0, np.zeros((n, cols), np.float32))
