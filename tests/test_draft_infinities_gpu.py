"""A row with +inf among its allowed logits is refused at any temperature (at 1e37 a reference's limit, so many units
above it, would pass f32's range), and one without is not."""
import numpy as np
import pytest

import noetic_rl as nr

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    nr.claim(0)
    yield


@pytest.mark.parametrize("temperature", [1e-20, 1.0, 1e37])
@pytest.mark.parametrize("rows", [3, 400])
def test_infinities(temperature, rows):
    V, k = 3000, 4
    x = np.random.default_rng(0).normal(0, 1, (rows, 1, V)).astype(np.float32)
    x[1, 0, 5] = np.inf
    x[2, 0, 2999] = np.inf
    bad = np.arange(rows) % rows < 3
    bad[0] = False
    flat = nr.Tempered(nr.Tensor.from_numpy(x.reshape(rows, V)), temperature, None)
    _, lp = nr.top_logprobs(flat, k, check=False)
    assert np.array_equal(np.isnan(lp.to_numpy()).all(1), bad) and np.isfinite(lp.to_numpy()[~bad][:, 0]).all()
    ids = np.broadcast_to(np.arange(k, dtype=np.int32), (rows, k)).copy()
    loss, _ = nr.distill_with_stats(flat, nr.Tensor.from_numpy(ids), nr.Tensor.from_numpy(np.full((rows, k), -2.0, np.float32)))
    assert np.array_equal(np.isnan(loss.to_numpy()), bad)
    u = nr.Tensor.from_numpy(np.full((rows, 1), 0.5), "f64")
    got, acc, lp = nr.verify_drafted(nr.Tensor.from_numpy(x), None, nr.Tensor((rows, 0), "i32"), temperature, None, None,
                                     uniforms=u, check=False)
    assert np.array_equal(got.to_numpy()[:, 0] < 0, bad) and (acc.to_numpy() == 0).all()
    assert np.array_equal(np.isnan(lp.to_numpy()[:, 0]), bad)
