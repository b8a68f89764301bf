"""The SwiGLU limits of the int8 layer: one of the routed experts, one of the shared expert. Bound: that
of test_gpu_int8_layer.py (5 % of the norm); limits of 0.3 against none move these outputs by far more."""

import numpy as np
import pytest

import vastloom_b200 as vb
from test_gpu_int8_layer import dev, plain, weights  # noqa: F401
from vastloom_b200.int8 import Int8MoeLayer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("routed,own", [(0.3, 0.0), (0.0, 0.3), (0.3, 1.0), (0.3, None), (0.0, None)])
def test_routed_and_shared_limits(dev, T, routed, own):  # noqa: F811
    rng = np.random.default_rng(T)
    E, I, H, k = 5, 96, 128, 2
    w1, w3, w2 = weights(rng, E, I, H), weights(rng, E, I, H), weights(rng, E, H, I)
    shared = (weights(rng, 1, I, H)[0], weights(rng, 1, I, H)[0], weights(rng, 1, H, I)[0])
    router = rng.standard_normal((E, H)).astype(np.float32) * 0.1
    x = rng.standard_normal((T, H)).astype(np.float32)
    limits = {} if own is None else {"shared_swiglu_limit": own}
    layer = Int8MoeLayer(dev, router=router, w1=w1, w3=w3, w2=w2, top_k=k, shared=shared, swiglu_limit=routed, max_tokens=T,
                         **limits)
    try:
        out = layer.forward(x)
        idx, wt = dev.route(dev.router_logits(x, router), k)

        def want(shared_limit):
            alone = plain(x, idx, wt, w1, w3, w2, None, routed)
            return alone + plain(x, idx, 0 * wt, w1, w3, w2, shared, shared_limit)

        right = want(routed if own is None else own)
        assert np.linalg.norm(out - right) <= 0.05 * np.linalg.norm(right)
        if own is not None:
            assert np.linalg.norm(right - want(routed)) > 0.1 * np.linalg.norm(right)
    finally:
        layer.close()
