"""Greedy verification under an additive mask that lowers a whole row: the log-probabilities are those of the f32 masked logits
that its tokens are the first largest of, as the sampler's are. Ids and counts are equal; a log-probability is within half an
f32 step of its value and 4.2e-6 (its sums' f32 exponentials)."""
import numpy as np
import pytest

import noetic_rl as nr
from tests import draft_reference as ref
from tests.test_verify_drafted_gpu import run

pytestmark = pytest.mark.gpu
LOWEST = float(np.finfo(np.float32).min)


@pytest.fixture(scope="module", autouse=True)
def device():
    nr.claim(0)
    yield


def lowered(x, add):
    """x + add rounded to f32, as f64."""
    return (np.asarray(x, np.float32) + add).astype(np.float64)


@pytest.mark.parametrize("S", [4, 150])  # several workgroups a position, and one
@pytest.mark.parametrize("V", [7, 1100, 5003])
@pytest.mark.parametrize("value", [-1e5, -1e9, -1e13, LOWEST])
def test_greedy(S, V, value):
    rng = np.random.default_rng(V)
    K = 2
    x = ref.rounded(rng.normal(0, 2, (S, K + 1, V)), "f32")
    add = np.full((1, 1, V), value, np.float32)
    z = lowered(x, add)
    tokens = np.where(rng.random((S, K)) < 0.7, np.argmax(z[:, :K], 2), rng.integers(0, V, (S, K))).astype(np.int32)
    wi, wa, wl = ref.verify(z, None, tokens, None, np.full(S, K), True)
    u, mt = rng.random((S, K + 1)), nr.Tensor.from_numpy(add)
    ids, acc, lp = (t.to_numpy() for t in run(x, None, mt, tokens, u, None, "f32", 0.0))
    assert np.array_equal(ids, wi) and np.array_equal(acc, wa)
    assert (np.abs(lp - wl) <= 2.0 ** -24 * np.abs(wl) + 4.2e-6).all()
    # the sampler's, of the same rows (within its own 4.2e-6 too)
    sampled, slp = (t.to_numpy() for t in nr.sample_logp(ref.tensor(x, "f32"), 0.0, mt, None))
    kept = np.arange(K + 1) <= wa[:, None]
    assert np.array_equal(sampled[kept], wi[kept])
    assert (np.abs(lp - slp)[kept] <= 2.0 ** -23 * np.abs(wl)[kept] + 8.4e-6).all()


@pytest.mark.parametrize("S", [4, 150])
def test_greedy_with_one_token_left(S):
    x = np.full((S, 2, 900), 3.7, np.float32)
    add = np.full((1, 1, 900), -np.inf, np.float32)
    add[..., 77] = -1e9
    tokens = np.full((S, 1), 77, np.int32)
    ids, acc, lp = (t.to_numpy() for t in run(x, None, nr.Tensor.from_numpy(add), tokens, np.full((S, 2), 0.5), None, "f32", 0.0))
    assert (ids == 77).all() and (acc == 1).all() and (lp == 0.0).all()


@pytest.mark.parametrize("value", [-200.3, -1e3, -1e5, -4e5, -1e9])
def test_accepted_drafts_of_many_positions(value):
    """450 positions, one workgroup each, judged by f32 exponentials of f64 differences: what an f32 step of the mask is does
    not reach a log-probability."""
    rng = np.random.default_rng(3)
    S, K, V = 150, 2, 1100
    x = ref.rounded(rng.normal(0, 2, (S, K + 1, V)), "f32")
    y = ref.rounded(x[:, :K] + rng.normal(0, 0.5, (S, K, V)), "f32")
    add = np.full((1, 1, V), value, np.float32)
    z, zq = x + add.astype(np.float64), y + add.astype(np.float64)
    tokens = np.argmax(zq + rng.gumbel(size=zq.shape), 2).astype(np.int32)
    u = rng.random((S, K + 1))
    wi, wa, wl = ref.verify(z, zq, tokens, u, np.full(S, K), False)
    ids, acc, lp = (t.to_numpy() for t in run(x, y, nr.Tensor.from_numpy(add), tokens, u, None, "f32", 1.0))
    assert np.array_equal(ids, wi) and np.array_equal(acc, wa) and (wa > 0).any()
    assert (np.abs(lp - wl) <= 2.0 ** -24 * np.abs(wl) + 4.2e-6).all()


def test_a_certain_token_of_many_positions():
    """The only token that the mask leaves, at -1e5: its log-probability is 0."""
    S = 300
    x = np.full((S, 2, 900), 3.7, np.float32)
    add = np.full((1, 1, 900), -np.inf, np.float32)
    add[..., 77] = -1e5
    ids, acc, lp = (t.to_numpy() for t in run(x, None, nr.Tensor.from_numpy(add), np.full((S, 1), 77, np.int32), np.full((S, 2), 0.5),
                                              None, "f32", 1.0))
    assert (ids == 77).all() and (acc == 1).all() and (np.abs(lp) <= 4.2e-6).all()


@pytest.mark.parametrize("V", [9000, 9001])
def test_sums_far_above_their_references(V):
    """450 positions whose largest logits lie 40 above what their lanes met first: the f32 sums' references stay behind, an
    argument around 57 is rounded to 2^-19, and the ratio of p's and q's sums is further off than the 5e-7 that the drawn row's chunks
    are taken with (0.95e-6 by the root mean square of four such roundings, each over a step of 2^-18): k_verify_pick computes
    them throughout. Ids and counts are equal."""
    rng = np.random.default_rng(V)
    S, K = 150, 2
    x = rng.normal(0, 1, (S, K + 1, V))
    y = rng.normal(0, 1, (S, K, V))
    for r in (x, y):
        r[..., 5000:5002] = 40.0 + rng.normal(0, 1, r[..., 5000:5002].shape)
    x, y = ref.rounded(x, "f32"), ref.rounded(y, "f32")
    tokens = np.where(rng.random((S, K)) < 0.5, 5000, 5001).astype(np.int32)
    u = rng.random((S, K + 1))
    want = ref.verify(x, y, tokens, u, np.full(S, K), False)
    assert (want[1] < K).any()
    got = run(x, y, None, tokens, u, None, "f32", 1.0)
    assert np.array_equal(got[0].to_numpy(), want[0]) and np.array_equal(got[1].to_numpy(), want[1])
    lp = got[2].to_numpy()
    assert (np.abs(lp - want[2]) <= 2.0 ** -24 * np.abs(want[2]) + 4.2e-6).all()
