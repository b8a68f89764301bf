"""Rows of the balance loss at their limits.

Which rows of the logits it reads: live ones, and no others (a caller may leave the memory of masked
tokens, and of tokens that no sequence holds, without content or without backing). The logits lie in page-locked host memory, which the GPU reads over its host link: 64 MB of rows that
are not to be read would take 1 ms at 64 GB/s, the link's nominal rate, and the call without them
takes some tens of microseconds. 0.4 ms is asked of the fastest of eight calls, a factor of two and
more on either side. Every row is backed, so that a kernel that reads them is slow and no worse.
"""

import numpy as np
import pytest

import vastloom_b200 as vb
from test_gpu_balance import KIND, SCORES, check, dev, plain, routes, run, torch  # noqa: F401

pytestmark = pytest.mark.gpu

T, E, K = 65536, 256, 2
LIMIT_MS = 0.4


@pytest.mark.parametrize("case", ["all masked", "few live", "outside", "outside, masked"])
def test_rows_that_are_not_live_are_not_read(dev, torch, case):  # noqa: F811
    rng = np.random.default_rng(len(case))
    z = torch.empty(T, E, pin_memory=True)
    z.fill_(float("nan"))
    mask, offsets = None, None
    if "masked" in case or case == "few live":
        mask = np.zeros(T, bool)
        mask[rng.integers(0, T, 64 if case != "all masked" else 0)] = True
    if "outside" in case:  # the first and the last tokens belong to no sequence
        offsets = [30000, 30007, 30007, 30100]
    live = np.ones(T, bool) if mask is None else mask
    if offsets:
        if mask is not None:
            mask[30000:30100:3] = True
        held = np.zeros(T, bool)
        held[offsets[0]:offsets[-1]] = True
        live = live & held
    z[torch.from_numpy(live)] = torch.from_numpy(rng.standard_normal((int(live.sum()), E)).astype(np.float32))
    idx = routes(rng, T, E, K) if live.any() else np.zeros((T, K), np.int64)
    S = 1 if offsets is None else len(offsets) - 1
    ic = torch.from_numpy(idx.astype(np.int32)).cuda()
    mc = None if mask is None else torch.from_numpy(mask.astype(np.uint8)).cuda()
    oc = None if offsets is None else torch.tensor(offsets, dtype=torch.int32).cuda()
    lo, co = torch.full((1,), 9.0, device="cuda"), torch.full((S, E), 9, dtype=torch.int32, device="cuda")
    gr = torch.full((T, E), 9.0, device="cuda")
    n = vb.balance_workspace_bytes(T, E, S)
    ws = torch.full((n,), 0x5a, dtype=torch.uint8, device="cuda")
    times = []
    for _ in range(8):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        a.record()
        dev.balance_loss_device(z.data_ptr(), ic.data_ptr(), T, E, K, counts_ptr=co.data_ptr(), ws_ptr=ws.data_ptr(),
                                ws_bytes=n, logits_type=KIND["f32"], score=SCORES["sigmoid"],
                                mask_ptr=0 if mc is None else mc.data_ptr(), seq_offsets_ptr=0 if oc is None else oc.data_ptr(),
                                n_seqs=S, loss_ptr=lo.data_ptr(), dlogits_ptr=gr.data_ptr(), stream=1)
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    got = (float(lo[0]), co.cpu().numpy(), gr.cpu().numpy().astype(np.float64), None)
    check(got, plain(np.where(live[:, None], z.numpy(), 0), idx, "sigmoid", 1.0, live if offsets is None else mask, offsets),
          "f32")
    assert np.all(got[2][~live] == 0)
    assert min(times) <= LIMIT_MS, times


def test_softmax_far_below_the_row_maximum(dev, torch):  # noqa: F811
    """Scores of logits 10 to 87 below their row's maximum (multiples of 2^-8, so that the difference is
    exact), an expert's that no token chose: the gradient -upstream weight p d, d the share of the chosen
    one. Bound in units of 2^-24: exponential 5, two reciprocals 4, count share 2, weight 3, the sum, d
    and four products 7: 21, and 24 are asked. An error that grew with the distance would pass it."""
    rng = np.random.default_rng(5)
    n, experts = 78, 64
    far = 10 + np.arange(n) + np.floor(256 * rng.random(n)) / 256
    far = np.minimum(far, 87)
    z = np.full((n, experts), 3.25, np.float32)
    z[:, 1:] -= far[:, None].astype(np.float32)
    idx = np.zeros((n, 1), np.int64)  # every token's maximum
    got = run(dev, torch, torch.from_numpy(z).cuda(), idx, score="softmax", coef=1e4, up=1e4)
    p = np.exp(-far) / (1 + (experts - 1) * np.exp(-far))
    d = experts / (1 + (experts - 1) * np.exp(-far))
    want = (-1e8 / n * p * d)[:, None]
    assert np.all(np.abs(got[2][:, 1:] - want) <= 24 * 2.0 ** -24 * np.abs(want)), float(
        np.max(np.abs(got[2][:, 1:] / want - 1)) * 2.0 ** 24)


@pytest.mark.parametrize("T,offsets", [(6000, [0, 5000, 100, 6000]), (6000, [6000, 0, 3000, 10]), (9000, [9000, 4000, 0]),
                                       (6000, [4000000000, 5, 4294967295, 7]), (20000, [0, 20000, 1, 20000, 2, 20000]),
                                       (70, [60, 10]), (6000, [0] + [5000, 3] * 300 + [6000])])
@pytest.mark.parametrize("score", ["softmax", "sqrt_softplus"])
def test_offsets_that_fall_touch_nothing_outside(dev, torch, T, offsets, score):  # noqa: F811
    """Offsets outside the contract, over many tokens, pieces and parts: the results are undefined, but
    every output lies inside its array, no count passes the pairs there are, and the call's neighbours
    (a right one before and after, in the same workspace) are untouched."""
    rng = np.random.default_rng(T)
    n, k, S = 40, 3, len(offsets) - 1
    z, idx = rng.standard_normal((T, n)).astype(np.float32), routes(rng, T, n, k)
    right = [0] + sorted(rng.integers(0, T + 1, S - 1).tolist()) + [T]
    want = plain(z, idx, score, 1.0, None, right)
    zc, ic = torch.from_numpy(z).cuda(), torch.from_numpy(idx.astype(np.int32)).cuda()
    size, guard = vb.balance_workspace_bytes(T, n, S), 1024
    ws = torch.full((size + 4 * guard,), 0x5a, dtype=torch.uint8, device="cuda")
    co = torch.full((S * n + 2 * guard,), 9, dtype=torch.int32, device="cuda")
    gr = torch.full((T * n + 2 * guard,), 9.0, device="cuda")
    for off in (right, offsets, right):
        oc = torch.from_numpy(np.array(off, np.uint32).view(np.int32)).cuda()
        lo = torch.full((3,), 9.0, device="cuda")
        co[guard:-guard] = 9
        gr[guard:-guard] = 9
        dev.balance_loss_device(zc.data_ptr(), ic.data_ptr(), T, n, k, counts_ptr=co[guard:].data_ptr(), ws_ptr=ws.data_ptr(),
                                ws_bytes=size, score=SCORES[score], seq_offsets_ptr=oc.data_ptr(), n_seqs=S,
                                loss_ptr=lo[1:].data_ptr(), dlogits_ptr=gr[guard:].data_ptr(), stream=1)
        torch.cuda.synchronize()
        assert float(lo[0]) == 9 and float(lo[2]) == 9 and torch.all(ws[size:] == 0x5a)
        for a in (co, gr):
            assert torch.all(a[:guard] == 9) and torch.all(a[-guard:] == 9)
        counts, grad = co[guard:-guard].view(S, n).cpu().numpy(), gr[guard:-guard].view(T, n).cpu().numpy()
        assert 0 <= counts.min() and counts.sum(axis=1).max() <= T * k
        if off is right:
            check((float(lo[1]), counts, grad.astype(np.float64), None), want, "f32")
