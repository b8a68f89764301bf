"""Device.balance_loss's arguments on their way to the device, with the uploads kept on the host."""

import numpy as np
import pytest

import vastloom_b200 as vb


class Kept:
    address = 4096

    def __init__(self, array=None):
        self.array = array

    def download(self, dtype, count):
        return np.zeros(count, dtype)

    def free(self):
        pass


@pytest.mark.parametrize("mask", [[True, False, True], [1, 0, 256], [0.5, 0.0, 2.0], [-1, 0, 1 << 40]])
def test_every_value_but_zero_is_live(mask):
    dev, uploads = object.__new__(vb.Device), []
    dev.to_device = lambda a, tag="": uploads.append(np.array(a)) or Kept(a)
    dev.buffer = lambda n, tag="": Kept()
    dev.balance_loss_device = lambda *a, **kw: None
    dev.synchronize = lambda: None
    dev.balance_loss(np.zeros((3, 4), np.float32), np.zeros((3, 1), np.uint32), mask=mask)
    sent = [a for a in uploads if a.dtype == np.uint8]
    assert len(sent) == 1 and sent[0].tolist() == [1, 0, 1]
    with pytest.raises(ValueError):
        dev.balance_loss(np.zeros((2, 4), np.float32), np.zeros((2, 1), np.uint32), mask=mask)
