"""Calls of every size on what was made for the largest: the int8 layer's batches up to its max_tokens,
and the balance loss in a workspace of its largest call. Bounds: those of test_gpu_int8_layer.py and
test_gpu_balance.py."""

import numpy as np
import pytest

import vastloom_b200 as vb
from test_gpu_balance import KIND, check, dev, routes, torch  # noqa: F401
from test_gpu_balance import plain as plain_balance
from test_gpu_int8_layer import plain, weights
from vastloom_b200.int8 import Int8MoeLayer

pytestmark = pytest.mark.gpu


def test_layer_batches_up_to_its_most_tokens(dev):  # noqa: F811
    rng = np.random.default_rng(0)
    E, I, H, k, most = 6, 48, 64, 2, 8192
    w1, w3, w2 = weights(rng, E, I, H), weights(rng, E, I, H), weights(rng, E, H, I)
    router = rng.standard_normal((E, H)).astype(np.float32) * 0.1
    layer = Int8MoeLayer(dev, router=router, w1=w1, w3=w3, w2=w2, top_k=k, max_tokens=most)
    try:
        for T in (most, 1, 100, 1025, 3000, 4096, 4097):
            x = rng.standard_normal((T, H)).astype(np.float32)
            out = layer.forward(x)
            idx, wt = dev.route(dev.router_logits(x, router), k)
            some = rng.permutation(T)[:200]
            want = plain(x[some], idx[some], wt[some], w1, w3, w2, None, 0.0)
            assert np.linalg.norm(out[some] - want) <= 0.05 * np.linalg.norm(want)
            assert np.array_equal(layer.last_counts, np.bincount(idx.reshape(-1), minlength=E))
    finally:
        layer.close()


@pytest.mark.parametrize("S", [1, 3, 40])
def test_balance_in_the_largest_calls_workspace(dev, torch, S):  # noqa: F811
    """Nothing is written past the size either, whichever call is made in it."""
    rng = np.random.default_rng(S)
    E, k, most = 48, 3, 16384
    n = vb.balance_workspace_bytes(most, E, S)
    ws = torch.full((n + 4096,), 0x5a, dtype=torch.uint8, device="cuda")
    for T in (most, 300, 2049, 4096, 4097, 8192, 8193):
        z, idx = rng.standard_normal((T, E)).astype(np.float32), routes(rng, T, E, k)
        off = [0, *sorted(rng.integers(0, T + 1, S - 1).tolist()), T]
        zc, ic = torch.from_numpy(z).cuda(), torch.from_numpy(idx.astype(np.int32)).cuda()
        oc = torch.tensor(off, dtype=torch.int32).cuda()
        lo, co = torch.zeros(1, device="cuda"), torch.full((S, E), 9, dtype=torch.int32, device="cuda")
        gr = torch.full((T, E), 9.0, device="cuda")
        dev.balance_loss_device(zc.data_ptr(), ic.data_ptr(), T, E, k, counts_ptr=co.data_ptr(), ws_ptr=ws.data_ptr(),
                                ws_bytes=n, seq_offsets_ptr=oc.data_ptr(), n_seqs=S, loss_ptr=lo.data_ptr(),
                                dlogits_ptr=gr.data_ptr(), logits_type=KIND["f32"], stream=1)
        got = (float(lo[0]), co.cpu().numpy(), gr.cpu().numpy().astype(np.float64), None)
        check(got, plain_balance(z, idx, "softmax", 1.0, None, off), "f32")
        assert torch.all(ws[n:] == 0x5a)
