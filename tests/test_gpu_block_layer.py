"""The int8 MoE layer as a residual block (Int8MoeLayer with an input norm): norm to int8 rows, rows by expert, gate/up
products with SwiGLU in the epilogue, down products, combine on the residual - the operators as they run together,
against the block in 64 bits on the unrounded weights.

Bound: as for the layer without a norm, a row rounded to 8 bits is off by 0.9 % of its norm (normal rows, one step's
1 / sqrt(12)), SwiGLU rows by 1.8 %; four roundings in independent directions stay below 3 % of the MoE's output, and 5 %
is asked. The residual adds nothing to it.
"""

import numpy as np
import pytest

import vastloom_b200 as vb
from vastloom_b200.int8 import Int8Experts, Int8MoeLayer

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if vb.device_count() == 0:
        pytest.fail("no CUDA device: GPU tests must run on a B200")
    d = vb.Device(0, install_codebooks=False)
    yield d
    d.close()


def weights(rng, E, I, H):
    return [(rng.standard_normal((I, H)) / np.sqrt(H)).astype(np.float32) for _ in range(E)]


def swiglu(g, u, limit):
    if limit:
        g, u = np.minimum(g, limit), np.clip(u, -limit, limit)
    return g / (1 + np.exp(-g)) * u


def moe(x, idx, wt, w1, w3, w2, shared, limit, shared_limit):
    out = np.zeros_like(x)
    for t in range(x.shape[0]):
        for j in range(idx.shape[1]):
            e = idx[t, j]
            out[t] += wt[t, j] * (w2[e].astype(np.float64) @ swiglu(w1[e] @ x[t], w3[e] @ x[t], limit))
        if shared:
            out[t] += shared[2].astype(np.float64) @ swiglu(shared[0] @ x[t], shared[1] @ x[t], shared_limit)
    return out


@pytest.mark.parametrize("T", [1, 2, 9, 150, 700])
@pytest.mark.parametrize("score,with_shared,limit,H,I", [(vb.SCORE_SQRT_SOFTPLUS, True, 0.0, 512, 256),
                                                         (vb.SCORE_SOFTMAX, False, 1.0, 512, 256),
                                                         (vb.SCORE_SOFTMAX_F64_NORM, True, 0.8, 500, 130)])
def test_block(dev, T, score, with_shared, limit, H, I):
    rng = np.random.default_rng(T + H)
    E, k, eps = 12, 3, 1e-5
    w1, w3, w2 = weights(rng, E, I, H), weights(rng, E, I, H), weights(rng, E, H, I)
    shared = (weights(rng, 1, I, H)[0], weights(rng, 1, I, H)[0], weights(rng, 1, H, I)[0]) if with_shared else None
    router = rng.standard_normal((E, H)).astype(np.float32) * 0.1
    norm = (1 + 0.2 * rng.standard_normal(H)).astype(np.float32)
    x = (3 * rng.standard_normal((T, H))).astype(np.float32)
    layer = Int8MoeLayer(dev, router=router, w1=w1, w3=w3, w2=w2, top_k=k, score=score, shared=shared, swiglu_limit=limit,
                         shared_swiglu_limit=0.0, max_tokens=T, input_norm=(norm, eps))
    try:
        out = layer.forward(x)
        _, normed, _, _ = dev.add_rms_norm(x, norm, eps)
        exact = x.astype(np.float64)
        exact = exact / np.sqrt(np.mean(exact * exact, axis=1, keepdims=True) + eps) * norm
        assert np.max(np.abs(normed - exact)) <= 2.0 ** -18 * np.max(np.abs(exact))
        logits = dev.router_logits(normed, router)
        idx, wt = dev.route(logits, k, score=score)
        want = moe(exact, idx, wt, w1, w3, w2, shared, limit, 0.0)
        assert np.linalg.norm(out - x - want) <= 0.05 * np.linalg.norm(want)
        assert np.array_equal(layer.last_counts, np.bincount(idx.reshape(-1), minlength=E))
        loss, _, _ = dev.balance_loss(logits, idx, score=score)
        assert layer.last_loss == loss
        assert np.array_equal(out, layer.forward(x, logits))
    finally:
        layer.close()


def test_pairs_are_interleaved(dev):
    """fill_pairs puts row i of the two matrices at rows 2i and 2i + 1, each with its own scale."""
    rng = np.random.default_rng(0)
    gate, up = (rng.standard_normal((7, 40)).astype(np.float32) for _ in range(2))
    pairs, halves = Int8Experts(dev, 2, 14, 40), Int8Experts(dev, 2, 14, 40)
    try:
        pairs.fill_pairs(1, gate, up)
        halves.fill(1, 0, gate)
        halves.fill(1, 7, up)
        q = [e._q.download(np.int8, 2 * 14 * e.stride).reshape(2, 14, -1)[1, :, :40] for e in (pairs, halves)]
        s = [e._s.download(np.float32, 28).reshape(2, 14)[1] for e in (pairs, halves)]
        for a, b in (q, s):
            assert np.array_equal(a[0::2], b[:7]) and np.array_equal(a[1::2], b[7:])
        with pytest.raises(ValueError):
            pairs.fill_pairs(2, gate, up)
        with pytest.raises(ValueError):
            pairs.fill_pairs(0, gate[:3], up)
    finally:
        pairs.free()
        halves.free()


def test_block_refusals(dev):
    rng = np.random.default_rng(2)
    w1, w2 = weights(rng, 2, 32, 64), weights(rng, 2, 64, 32)
    router = rng.standard_normal((2, 64)).astype(np.float32)
    with pytest.raises(ValueError):
        Int8MoeLayer(dev, router=router, w1=w1, w3=w1, w2=w2, top_k=1, input_norm=(np.ones(63, np.float32), 1e-5))
    layer = Int8MoeLayer(dev, router=router, w1=w1, w3=w1, w2=w2, top_k=1, input_norm=(np.ones(64, np.float32), 0.0))
    try:
        with pytest.raises(vb.VlbError):
            layer.forward(np.ones((1, 64), np.float32))  # eps must be positive
    finally:
        layer.close()
