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


@pytest.mark.gpu
def test_tempered_logits_past_f32():
    """Under an additive mask a tempered logit that f32 would round to -inf is excluded and one that it would round to +inf refuses
    its row, in every operator and for few and many positions (1e-37: 5 is held, 50 is not)."""
    nr.claim(0)
    T, V, S, K = 1e-37, 3000, 200, 1
    x = np.full((S, K + 1, V), -50.0, np.float32)
    x[:, :, 7], x[:, :, 2900] = 5.0, 5.0
    x[1, 0, 11] = 50.0
    add = nr.Tensor.from_numpy(np.zeros((1, 1, V), np.float32))
    tokens = np.full((S, K), 2900, np.int32)
    u = np.full((S, K + 1), 0.4)
    bad = np.arange(S) == 1
    for n in (3, S):
        ids, acc, lp = (t.to_numpy() for t in nr.verify_drafted(
            nr.Tensor.from_numpy(x[:n]), None, nr.Tensor.from_numpy(tokens[:n]), T, add, None, uniforms=nr.Tensor.from_numpy(u[:n], "f64"),
            check=False))
        assert np.array_equal(ids[:, 0] < 0, bad[:n]) and np.array_equal(acc, np.where(bad[:n], 0, 1))
        assert (ids[~bad[:n]] == [2900, 7]).all() and (np.abs(lp[~bad[:n]] + np.log(2)) < 1e-6).all()
        rows = nr.Tempered(nr.Tensor.from_numpy(x[:n, 0].copy()), T, nr.Tensor.from_numpy(np.zeros((1, V), np.float32)))
        top, lp = (t.to_numpy() for t in nr.top_logprobs(rows, 3, check=False))
        assert np.array_equal(np.isnan(lp).all(1), bad[:n]) and (top[~bad[:n]] == [7, 2900, -1]).all()
        for listed, loss in (([7, 11], np.inf), ([7, 2900], 0.0)):
            it = nr.Tensor.from_numpy(np.tile(np.array(listed, np.int32), (n, 1)))
            lt = nr.Tensor.from_numpy(np.full((n, 2), np.log(0.5), np.float32))
            got, stats = nr.distill_with_stats(rows, it, lt, check=False)
            got = got.to_numpy()
            assert np.isnan(got[bad[:n]]).all()
            good = got[~bad[:n]]
            assert (good == loss).all() if loss else (np.abs(good) < 1e-6).all()
            grad = nr.distill_grad(rows, it, lt, stats, nr.Tensor.from_numpy(np.full(n, 1e-37, np.float32))).to_numpy()
            assert np.isnan(grad[bad[:n]]).all()
            want = np.zeros(V)
            want[7] += 0.5
            want[2900] += 0.5
            want[listed] -= 0.5
            assert (np.abs(grad[~bad[:n]] - want) < 1e-6).all()
