"""The int8 MoE layer (vastloom_b200/int8.py) from router to combine, against the layer in 64 bits on
the unrounded weights.

Bound: a row rounded to 8 bits is off by a uniform error of one step's 1/sqrt(12), a step being its
largest value / 127. For the normal rows used here (largest about 4 deviations of 256 to 512 values)
that is 0.9 % of the row's norm. An output passes four such roundings (tokens, gate/up weights,
SwiGLU rows, down weights) in independent directions, and SwiGLU rows have longer tails (largest
about 8 deviations: 1.8 %); together the root of the squares' sum stays below 3 %, and 5 % is asked.
"""

import numpy as np
import pytest

import vastloom_b200 as vb
from vastloom_b200.ep import balanced_slots
from vastloom_b200.int8 import Int8MoeLayer

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


def plain(x, idx, wt, w1, w3, w2, shared, limit):
    x = x.astype(np.float64)
    out = np.zeros_like(x)
    for t in range(x.shape[0]):
        for j in range(idx.shape[1]):
            e = idx[t, j]
            out[t] += wt[t, j] * (w2[e].astype(np.float64) @ swiglu(w1[e] @ x[t], w3[e] @ x[t], limit))
        if shared:
            out[t] += shared[2].astype(np.float64) @ swiglu(shared[0] @ x[t], shared[1] @ x[t], limit)
    return out


@pytest.mark.parametrize("T", [1, 2, 9, 150])
@pytest.mark.parametrize("score,with_shared,limit", [(vb.SCORE_SQRT_SOFTPLUS, True, 0.0), (vb.SCORE_SOFTMAX, False, 1.0)])
def test_layer(dev, T, score, with_shared, limit):
    rng = np.random.default_rng(T)
    E, I, H, k = 12, 256, 512, 3
    w1, w3, w2 = weights(rng, E, I, H), weights(rng, E, I, H), weights(rng, E, H, I)
    shared = (weights(rng, 1, I, H)[0], weights(rng, 1, I, H)[0], weights(rng, 1, H, I)[0]) if with_shared else None
    router = rng.standard_normal((E, H)).astype(np.float32) * 0.1
    x = rng.standard_normal((T, H)).astype(np.float32)
    layer = Int8MoeLayer(dev, router=router, w1=w1, w3=w3, w2=w2, top_k=k, score=score, shared=shared,
                         swiglu_limit=limit, max_tokens=T)
    try:
        out = layer.forward(x)
        logits = dev.router_logits(x, router)
        idx, wt = dev.route(logits, k, score=score)
        want = plain(x, idx, wt, w1, w3, w2, shared, limit)
        assert np.linalg.norm(out - want) <= 0.05 * np.linalg.norm(want)
        counts = np.bincount(idx.reshape(-1), minlength=E)
        assert np.array_equal(layer.last_counts, counts)
        loss, own, _ = dev.balance_loss(logits, idx, score=score)
        assert layer.last_loss == loss and np.array_equal(own[0], counts)
        # the counts place the experts over ranks
        assert sorted(balanced_slots(layer.last_counts, 4)) == list(range(E))
        assert np.array_equal(out, layer.forward(x, logits))
    finally:
        layer.close()


def test_layer_from_resident_matrices(dev):
    """Experts given as resident ggml matrices: their dequantized values, rounded to 8 bits."""
    from vastloom_b200 import synth

    rng = np.random.default_rng(1)
    E, I, H, k, T = 4, 128, 256, 2, 20
    make = lambda rows, cols, i: dev.upload_matrix(vb.TYPE_Q8_0, rows, cols,  # noqa: E731
                                                   synth.matrix(rng, vb.TYPE_Q8_0, rows, cols, 0.002), identity=100 + i)
    ms = [[make(I, H, i) for i in range(E)], [make(I, H, 10 + i) for i in range(E)], [make(H, I, 20 + i) for i in range(E)]]
    router = rng.standard_normal((E, H)).astype(np.float32) * 0.1
    x = rng.standard_normal((T, H)).astype(np.float32)
    layer = Int8MoeLayer(dev, router=router, w1=ms[0], w3=ms[1], w2=ms[2], top_k=k, max_tokens=T)
    try:
        out = layer.forward(x)
        idx, wt = dev.route(dev.router_logits(x, router), k)
        want = plain(x, idx, wt, *[[dev.dequantize(m) for m in row] for row in ms], None, 0.0)
        assert np.linalg.norm(out - want) <= 0.05 * np.linalg.norm(want)
    finally:
        layer.close()
        for row in ms:
            for m in row:
                dev.release_matrix(m)


def test_layer_refusals(dev):
    rng = np.random.default_rng(2)
    w1, w2 = weights(rng, 2, 32, 64), weights(rng, 2, 64, 32)
    router = rng.standard_normal((2, 64)).astype(np.float32)
    with pytest.raises(ValueError):
        Int8MoeLayer(dev, router=router, w1=w1, w3=w1, w2=w1, top_k=1)
    with pytest.raises(ValueError):
        Int8MoeLayer(dev, router=router, w1=w1[:1], w3=w1, w2=w2, top_k=1)
    layer = Int8MoeLayer(dev, router=router, w1=w1, w3=w1, w2=w2, top_k=1, max_tokens=4)
    try:
        with pytest.raises(ValueError):
            layer.forward(np.zeros((5, 64), np.float32))
    finally:
        layer.close()
