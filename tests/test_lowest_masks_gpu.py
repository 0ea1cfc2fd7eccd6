"""Rows that an additive mask of f32's lowest value lowers throughout, with columns that it excludes (-inf) and lanes past the
row's end: every token left is as likely as the others, and no row is refused. Top log-probabilities, distillation and
verification, sampled and greedy; tolerances as in the operators' own tests."""
import numpy as np
import pytest

import noetic_rl as nr
from tests import draft_reference as ref
from tests.test_distill_gpu import both
from tests.test_verify_drafted_gpu import compare, run

pytestmark = pytest.mark.gpu
LOWEST = np.finfo(np.float32).min


@pytest.fixture(scope="module", autouse=True)
def device():
    nr.claim(0)
    yield


def lowest(V, excluded):
    add = np.full(V, LOWEST, np.float32)
    if excluded:
        add[2300:4200] = -np.inf     # (whole chunks, after and before others)
        add[:3] = -np.inf
    return add


@pytest.mark.parametrize("excluded", [False, True])
@pytest.mark.parametrize("V", [5003, 8200])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_top_and_distillation(dtype, V, excluded):
    rng = np.random.default_rng(V)
    R, k = 40, 6
    x = ref.rounded(rng.normal(0, 2, (R, V)), dtype)
    add = lowest(V, excluded)
    z = np.broadcast_to(add.astype(np.float64), (R, V))   # (a logit is far below half a step of it)
    mt = nr.Tensor.from_numpy(add[None])
    ids, lp = (t.to_numpy() for t in nr.top_logprobs(nr.Tempered(ref.tensor(x, dtype), 1.0, mt), k))
    wi, wl = ref.top(z, z, k)
    assert np.array_equal(ids, wi) and (np.abs(lp - wl) <= 2.0 ** -24 * np.abs(wl) + 4e-6).all()
    allowed = np.nonzero(add > -np.inf)[0]
    listed = np.stack([rng.permutation(allowed)[:k] for _ in range(R)]).astype(np.int32)
    teacher = np.log(np.full((R, k), 0.1)).astype(np.float32)
    for tail in ("REST", "DROP"):
        both(x, z, mt, listed, teacher, dtype, 1.0, tail, np.random.default_rng(1), "f32")


@pytest.mark.parametrize("excluded", [False, True])
@pytest.mark.parametrize("T", [0.0, 1.0])
@pytest.mark.parametrize("S, V", [(4, 5003), (150, 5003), (150, 8200)])
def test_verification(S, V, T, excluded):
    rng = np.random.default_rng(V)
    K = 2
    x = ref.rounded(rng.normal(0, 2, (S, K + 1, V)), "f32")
    add = lowest(V, excluded)
    z = np.broadcast_to(add.astype(np.float64), x.shape)
    allowed = np.nonzero(add > -np.inf)[0]
    tokens = np.where(rng.random((S, K)) < 0.5, allowed[0], rng.choice(allowed, (S, K))).astype(np.int32)
    u = rng.random((S, K + 1))
    y = None if T == 0.0 else ref.rounded(x[:, :K] + rng.normal(0, 0.5, (S, K, V)), "f32")
    want = ref.verify(z, None if y is None else z[:, :K], tokens, u, np.full(S, K), T == 0.0)
    compare(run(x, y, nr.Tensor.from_numpy(add[None, None]), tokens, u, None, "f32", T), want, T == 0.0)
