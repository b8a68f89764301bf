"""The router's balance loss, counts and gradient (vlb_balance_loss_device) against the formula in
64 bits, and the gradient against differences of the 64-bit loss.

Bounds: counts are equal. A row's scores come from at most 12 32-bit operations each within 2 units
of 2^-24 and sums over E scores in a tree (log2 E more); a factor f_e - d_t loses what cancels, so
the gradient's bound is taken on coefficient / (S' n) * p * (|f| + |d|) * r, with 64 * 2^-24 plus the
output type's unit; the loss, a sum of positive terms, has 64 * 2^-24 relative.
"""

import numpy as np
import pytest

import vastloom_b200 as vb

pytestmark = pytest.mark.gpu

SCORES = {"softmax": vb.SCORE_SOFTMAX, "sigmoid": vb.SCORE_SIGMOID, "sqrt_softplus": vb.SCORE_SQRT_SOFTPLUS}
UNIT = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
KIND = {"f32": vb.DTYPE_F32, "f16": vb.DTYPE_F16, "bf16": vb.DTYPE_BF16}
TOL = 64 * 2.0 ** -24


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


def scores(z, score):
    """Normalised scores and r = u'/u in 64 bits; a row without an expert gives zeros."""
    z = np.asarray(z, np.float64)
    with np.errstate(all="ignore"):
        if score == "softmax":
            lu, r = z, np.ones_like(z)
        elif score == "sigmoid":
            lu, r = -np.logaddexp(0, -z), np.exp(-np.logaddexp(0, z))
        else:
            sp = np.logaddexp(0, z)
            lu = np.where(z < -40, 0.5 * z, 0.5 * np.log(np.where(z < -40, 1.0, sp)))
            r = np.where(z < -40, 0.5, 0.5 * np.exp(-np.logaddexp(0, -z)) / np.where(z < -40, 1.0, sp))
        top = lu.max(axis=1, keepdims=True)
        none = np.isneginf(top)[:, 0]
        p = np.exp(lu - np.where(np.isneginf(top), 0, top))
        p /= p.sum(axis=1, keepdims=True)
    p[none] = 0
    r = np.where(np.isneginf(z), 0, r)
    return p, r


def plain(z, idx, score, coef=1.0, mask=None, offsets=None, up=1.0):
    """(loss, counts, gradient, the gradient's bound before rounding) in 64 bits."""
    z = np.asarray(z, np.float64)
    T, E = z.shape
    k = idx.shape[1]
    off = [0, T] if offsets is None else list(offsets)
    live = np.ones(T, bool) if mask is None else np.asarray(mask, bool)
    S = len(off) - 1
    counts, loss = np.zeros((S, E), np.int64), 0.0
    grad, scale = np.zeros((T, E)), np.zeros((T, E))
    rows = [[t for t in range(max(0, off[s]), min(T, off[s + 1])) if live[t]] for s in range(S)]
    alive = sum(1 for r in rows if r)
    for s, ts in enumerate(rows):
        if not ts:
            continue
        ids = idx[ts].reshape(-1)
        counts[s] = np.bincount(ids[ids < E], minlength=E)
        f = counts[s] * (E / (k * len(ts)))
        p, r = scores(z[ts], score)
        d = p @ f
        wt = coef / (alive * len(ts))
        loss += wt * d.sum()
        with np.errstate(invalid="ignore"):
            grad[ts] = up * wt * p * (f[None] - d[:, None]) * r
        scale[ts] = np.abs(up * wt) * p * (f[None] + d[:, None]) * np.abs(r)
    return loss, counts, grad, scale


def run(dev, torch, z, idx, *, x="f32", score="softmax", coef=1.0, mask=None, offsets=None, up=None, grad=True, loss=True,
        stride=None, stream=1):
    """z: a CUDA tensor [T, E] of type x (its row stride taken)."""
    T, E = z.shape
    S = 1 if offsets is None else len(offsets) - 1
    ic = torch.from_numpy(np.ascontiguousarray(idx).astype(np.uint32).view(np.int32)).cuda()
    mc = None if mask is None else torch.from_numpy(np.asarray(mask).astype(np.uint8)).cuda()
    oc = None if offsets is None else torch.tensor(offsets, dtype=torch.int32).cuda()
    uc = None if up is None else torch.tensor([up], device="cuda")
    lo = torch.full((1,), 9.0, device="cuda")
    co = torch.full((S, E), 9, dtype=torch.int32, device="cuda")
    gr = torch.full((T, stride or E), 9.0, device="cuda", dtype=z.dtype)
    n = vb.balance_workspace_bytes(T, E, S)
    ws = torch.full((n,), 0x5a, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    dev.balance_loss_device(z.data_ptr(), ic.data_ptr(), T, E, idx.shape[1], counts_ptr=co.data_ptr(), ws_ptr=ws.data_ptr(),
                            ws_bytes=n, logits_type=KIND[x], logits_stride=z.stride(0) if T else 0, score=SCORES[score],
                            coefficient=coef, mask_ptr=0 if mc is None else mc.data_ptr(),
                            seq_offsets_ptr=0 if oc is None else oc.data_ptr(), n_seqs=S,
                            upstream_ptr=0 if uc is None else uc.data_ptr(), loss_ptr=lo.data_ptr() if loss else 0,
                            dlogits_ptr=gr.data_ptr() if grad else 0, dlogits_stride=stride or 0, stream=stream)
    torch.cuda.synchronize()
    return float(lo[0]), co.cpu().numpy(), gr.float().cpu().numpy().astype(np.float64), gr


def check(got, want, x):
    loss, counts, grad, _ = got
    wl, wc, wg, ws = want
    assert np.array_equal(counts, wc)
    assert abs(loss - wl) <= TOL * abs(wl), (loss, wl)
    bound = (TOL + UNIT[x]) * ws + (2.0 ** -25 if x == "f16" else 2.0 ** -140)
    assert np.all(np.abs(grad - wg) <= bound), float(np.max(np.abs(grad - wg) - bound))


def routes(rng, T, E, k):
    return np.stack([rng.permutation(E)[:k] for _ in range(T)]) if T else np.zeros((0, k), np.int64)


@pytest.mark.parametrize("score", list(SCORES))
@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (2, 33, 3), (17, 64, 8), (100, 31, 5), (300, 256, 8),
                                   (65, 512, 16), (1000, 100, 1), (33, 129, 4)])
def test_loss_counts_gradient(dev, torch, score, x, T, E, k):
    rng = np.random.default_rng(T * E + k)
    z = torch.from_numpy(3 * rng.standard_normal((T, E))).to({"f32": torch.float32, "f16": torch.float16,
                                                              "bf16": torch.bfloat16}[x])
    idx = routes(rng, T, E, k)
    got = run(dev, torch, z.cuda(), idx, x=x, score=score, coef=0.37, up=1.75)
    check(got, plain(z.double().numpy(), idx, score, 0.37, up=1.75), x)


@pytest.mark.parametrize("score", list(SCORES))
@pytest.mark.parametrize("offsets", [[0, 40], [0, 0, 40], [0, 7, 7, 39, 40, 40], [0, 1, 2, 3, 40], [3, 20, 35], [0, 64],
                                     [0, 33, 200]])
@pytest.mark.parametrize("masked", [False, True])
def test_sequences_and_masks(dev, torch, score, offsets, masked):
    """Sequences without a token or without a live one; tokens that no sequence holds; masked logits
    that are not numbers."""
    rng = np.random.default_rng(len(offsets) * 10 + masked)
    T, E, k = 40, 48, 4
    z = rng.standard_normal((T, E)).astype(np.float32)
    mask = None
    if masked:
        mask = rng.random(T) > 0.4
        mask[7:39] &= rng.random(32) > 0.5
        z[~mask] = np.nan
        z[np.flatnonzero(~mask)[0]] = np.inf
    idx = routes(rng, T, E, k)
    got = run(dev, torch, torch.from_numpy(z).cuda(), idx, score=score, coef=0.01, mask=mask, offsets=offsets)
    live = np.ones(T, bool) if mask is None else mask
    check(got, plain(np.where(live[:, None], z, 0), idx, score, 0.01, mask, [min(o, T) for o in offsets]), "f32")
    outside = ~live | (np.arange(T) < offsets[0]) | (np.arange(T) >= offsets[-1])
    assert np.all(got[2][outside] == 0)


def test_offsets_that_fall_hold_no_token(dev, torch):
    rng = np.random.default_rng(1)
    z, idx = rng.standard_normal((20, 8)).astype(np.float32), routes(rng, 20, 8, 2)
    loss, counts, grad, _ = run(dev, torch, torch.from_numpy(z).cuda(), idx, offsets=[0, 12, 5, 20])
    assert np.isfinite(loss) and np.all(np.isfinite(grad)) and counts.sum() <= 40


@pytest.mark.parametrize("score", list(SCORES))
def test_masked_experts_and_empty_rows(dev, torch, score):
    """-inf and the type's lowest value on single experts, on all but one, on all of a row."""
    rng = np.random.default_rng(2)
    T, E, k = 12, 40, 4
    z = rng.standard_normal((T, E)).astype(np.float32)
    low = np.finfo(np.float32).min
    z[0, :] = -np.inf
    z[1, 1:] = -np.inf
    z[2, ::2] = -np.inf
    z[3, :] = low
    z[4, 3:] = low
    z[5, :] -= 200
    z[6, :] += 200
    z[7, 0], z[7, 1:] = 80, -80
    z[8, :] = -1e30
    idx = routes(rng, T, E, k)
    got = run(dev, torch, torch.from_numpy(z).cuda(), idx, score=score)
    want = plain(z, idx, score)
    check(got, want, "f32")
    assert np.all(got[2][0] == 0)


@pytest.mark.parametrize("score", list(SCORES))
def test_a_nan_stays_in_its_row(dev, torch, score):
    rng = np.random.default_rng(3)
    z = rng.standard_normal((9, 64)).astype(np.float32)
    z[4, 10] = np.nan
    z[6, :] = np.nan
    idx = routes(rng, 9, 64, 2)
    loss, counts, grad, _ = run(dev, torch, torch.from_numpy(z).cuda(), idx, score=score)
    assert np.isnan(loss) and counts.sum() == 18
    assert np.all(np.isnan(grad[[4, 6]]).any(axis=1)) and np.all(np.isfinite(np.delete(grad, [4, 6], axis=0)))


def test_dropped_slots_are_not_counted(dev, torch):
    rng = np.random.default_rng(4)
    z, idx = rng.standard_normal((30, 16)).astype(np.float32), routes(rng, 30, 16, 4)
    idx[::3, 1] = 16
    idx[5, :] = 0xFFFFFFFF
    check(run(dev, torch, torch.from_numpy(z).cuda(), idx), plain(z, idx, "softmax"), "f32")


@pytest.mark.parametrize("case", ["no tokens", "all masked", "no sequence"])
def test_nothing_live(dev, torch, case):
    T = 0 if case == "no tokens" else 10
    z = torch.randn(T, 24).cuda()
    idx = routes(np.random.default_rng(0), T, 24, 2)
    mask = np.zeros(T, bool) if case == "all masked" else None
    loss, counts, grad, _ = run(dev, torch, z, idx, mask=mask, offsets=[0, 0, 0] if case == "no sequence" else None)
    assert loss == 0 and counts.sum() == 0 and np.all(grad == 0)


@pytest.mark.parametrize("x", ["f32", "bf16"])
def test_strides_and_left_out_outputs(dev, torch, x):
    """Logits as columns of a wider matrix at an odd offset, a gradient with a pitch, no loss, no
    gradient."""
    rng = np.random.default_rng(6)
    T, E, k = 50, 60, 6
    wide = torch.randn(T, 73).to(torch.float32 if x == "f32" else torch.bfloat16).cuda()
    z = wide[:, 5:65]
    idx = routes(rng, T, E, k)
    want = plain(z.double().cpu().numpy(), idx, "sigmoid")
    loss, counts, grad, full = run(dev, torch, z, idx, x=x, score="sigmoid", stride=67)
    check((loss, counts, grad[:, :E], None), want, x)
    assert torch.all(full[:, E:] == 9)
    _, counts, grad, _ = run(dev, torch, z, idx, x=x, score="sigmoid", loss=False)
    assert np.array_equal(counts, want[1])
    loss, _, grad, _ = run(dev, torch, z, idx, x=x, score="sigmoid", grad=False)
    assert abs(loss - want[0]) <= TOL * want[0] and np.all(grad == 9)


@pytest.mark.parametrize("score", list(SCORES))
def test_gradient_against_differences(dev, torch, score):
    """Central differences of the 64-bit loss with step 1e-4: their own error is below 1e-7 of the
    largest gradient for these logits (third derivatives of order one), far under the 1e-5 asked."""
    rng = np.random.default_rng(7)
    T, E, k = 6, 12, 3
    z, idx = rng.standard_normal((T, E)).astype(np.float32), routes(rng, T, E, k)
    off, mask = [0, 2, 6], np.array([1, 1, 1, 0, 1, 1], bool)
    _, _, grad, _ = run(dev, torch, torch.from_numpy(z).cuda(), idx, score=score, mask=mask, offsets=off)
    h, num = 1e-4, np.zeros((T, E))
    for t in range(T):
        for e in range(E):
            a, b = z.astype(np.float64), z.astype(np.float64)
            a[t, e] += h
            b[t, e] -= h
            num[t, e] = (plain(a, idx, score, 1.0, mask, off)[0] - plain(b, idx, score, 1.0, mask, off)[0]) / (2 * h)
    assert np.max(np.abs(num - grad)) <= 1e-5 * np.max(np.abs(num))


def test_equal_inputs_give_equal_bits(dev, torch):
    rng = np.random.default_rng(8)
    z = torch.randn(5000, 128).cuda()
    idx = routes(rng, 5000, 128, 8)
    runs = [run(dev, torch, z, idx, offsets=[0, 100, 2500, 5000]) for _ in range(4)]
    for r in runs[1:]:
        assert r[0] == runs[0][0] and np.array_equal(r[1], runs[0][1]) and torch.equal(r[3], runs[0][3])


@pytest.mark.parametrize("T,offsets", [(60, None), (3000, None), (3000, [0, 5, 900, 3000])])
def test_inputs_written_just_before(dev, torch, T, offsets):
    """Logits and routes that the kernels ahead on the stream write, and rewrite once the call has been
    enqueued; one workspace for all calls."""
    rng = np.random.default_rng(11)
    E, k, n, S = 96, 4, 5, 1 if offsets is None else len(offsets) - 1
    src = torch.randn(n, T, E).cuda()
    ids = [routes(rng, T, E, k) for _ in range(n)]
    idc = torch.from_numpy(np.stack(ids).astype(np.int32)).cuda()
    oc = None if offsets is None else torch.tensor(offsets, dtype=torch.int32).cuda()
    z, idx = torch.zeros(T, E, device="cuda"), torch.zeros(T, k, dtype=torch.int32, device="cuda")
    lo, co, gr = (torch.zeros(n, device="cuda"), torch.zeros(n, S, E, dtype=torch.int32, device="cuda"),
                  torch.zeros(n, T, E, device="cuda"))
    size = vb.balance_workspace_bytes(T, E, S)
    ws = torch.full((size,), 0x5a, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for i in range(n):
        z.copy_(src[i])
        idx.copy_(idc[i])
        dev.balance_loss_device(z.data_ptr(), idx.data_ptr(), T, E, k, counts_ptr=co[i].data_ptr(), ws_ptr=ws.data_ptr(),
                                ws_bytes=size, seq_offsets_ptr=0 if oc is None else oc.data_ptr(), n_seqs=S,
                                loss_ptr=lo[i:].data_ptr(), dlogits_ptr=gr[i].data_ptr(), stream=1)
        z.fill_(float("nan"))
        idx.fill_(-1)
    torch.cuda.synchronize()
    for i in range(n):
        got = (float(lo[i]), co[i].cpu().numpy(), gr[i].cpu().numpy().astype(np.float64), None)
        check(got, plain(src[i].cpu().numpy(), ids[i], "softmax", 1.0, None, offsets), "f32")


def test_many_sequences_and_host_form(dev, torch):
    rng = np.random.default_rng(9)
    T, E, k = 700, 20, 2
    z, idx = rng.standard_normal((T, E)).astype(np.float32), routes(rng, T, E, k)
    off = np.concatenate([[0], np.sort(rng.integers(0, T + 1, 500)), [T]])
    want = plain(z, idx, "softmax", 0.5, None, off)
    loss, counts, grad = dev.balance_loss(z, idx, coefficient=0.5, seq_offsets=off)
    check((loss, counts, grad.astype(np.float64), None), want, "f32")


def refusals():
    return [
        (dict(E=0), "must be positive"), (dict(k=0), "must be positive"), (dict(k=9), "k <= E"),
        (dict(n_seqs=0), "must be positive"), (dict(E=513, k=1), "512"), (dict(E=512, k=65), "64"),
        (dict(score=5), "score"), (dict(score=-1), "score"), (dict(logits_type=3), "logits_type"),
        (dict(n_seqs=2), "seq_offsets"), (dict(logits=None), "null"), (dict(idx=None), "null"),
        (dict(counts=None), "null"), (dict(logits=2), "aligned"), (dict(idx=2), "aligned"), (dict(loss=2), "aligned"),
        (dict(logits_stride=7), "stride"), (dict(dlogits_stride=7), "stride"),
        (dict(coefficient=float("inf")), "coefficient"), (dict(ws=None), "workspace"), (dict(ws=8), "workspace"),
        (dict(ws_bytes=16), "workspace"),
    ]


@pytest.mark.parametrize("change,words", refusals())
def test_refusals(dev, torch, change, words):
    import ctypes as C

    keep = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    p = keep.data_ptr()
    d = dict(logits=p, logits_stride=0, idx=p, mask=None, seq_offsets=None, upstream=None, loss=p, counts=p, dlogits=p,
             dlogits_stride=0, ws=p, ws_bytes=1 << 16, T=2, E=8, k=2, n_seqs=1, score=0, logits_type=0, coefficient=1.0,
             reserved0=0)
    d.update({k: (p + v if k in ("logits", "idx", "loss", "ws") and v else v) for k, v in change.items()})
    st = dev.lib.vlb_balance_loss_device(dev.h, C.byref(vb._BalanceDesc(**d)), None)
    assert st in (1, 8)
    buf = C.create_string_buffer(512)
    dev.lib.vlb_last_error(dev.h, buf, 512)
    assert words in buf.value.decode(), buf.value.decode()


def test_null_description(dev):
    assert dev.lib.vlb_balance_loss_device(dev.h, None, None) == 1
    assert dev.lib.vlb_balance_loss_device(None, None, None) == 1
