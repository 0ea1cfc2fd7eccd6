"""Temperatures past f32's range, whose f32 scale log2(e) / T is infinite or none: the top log-probabilities and the distillation
refuse them before any device is touched, and verification's answer does not depend on how many positions a call has."""
import numpy as np
import pytest

import noetic_rl as nr
from tests.test_draft_refusals import backward, distill, text, top


@pytest.mark.parametrize("call", [top, distill, backward])
@pytest.mark.parametrize("temperature", [1e-300, 1e-40, 1.1754943e-38, 3.403e38, 1e300])
def test_refused(call, temperature):
    assert call(temperature=temperature) == -1 and "temperature" in text() and "f32" in text()


@pytest.mark.parametrize("temperature", [1e-300, 1e-40, 1e-37, 1e37, 1e45, 1e300])
@pytest.mark.gpu
def test_verification_of_few_and_many_positions(temperature):
    """Each call's first sequences are the same: their ids and counts are too, with a keep-mask's excluded tokens."""
    nr.claim(0)
    rng = np.random.default_rng(1)
    S, K, V = 200, 2, 700
    x = rng.normal(0, 1, (S, K + 1, V)).astype(np.float32)
    keep = (rng.random((S, K + 1, V)) < 0.5).astype(np.uint8)
    keep[:, :, 3] = 1
    z = np.where(keep == 0, -np.inf, x)
    tokens = np.argmax(z[:, :K], 2).astype(np.int32)
    u = rng.random((S, K + 1))

    def run(n):
        return [t.to_numpy() for t in nr.verify_drafted(
            nr.Tensor.from_numpy(x[:n]), nr.Tensor.from_numpy(x[:n, :K].copy()), nr.Tensor.from_numpy(tokens[:n]), temperature,
            nr.Tensor.from_numpy(keep[:n], "u8"), None, uniforms=nr.Tensor.from_numpy(u[:n], "f64"))]

    few, many = run(20), run(S)
    for a, b in zip(few[:2], many[:2]):
        assert np.array_equal(a, b[:20])
    assert (many[1] == K).all() and np.array_equal(many[0][:, :K], tokens)   # (the drafter's logits are the target's)
    if temperature < 1:
        assert np.array_equal(many[0][:, K], np.argmax(z[:, K], 1))
