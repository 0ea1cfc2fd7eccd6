"""Distillation with the list's weights renormalized from a teacher's logits of any size (a mask lowered all or some of them): they
sum to 1. Against the f64 form with the errors and tolerances of the operator's own tests; a weight's logarithm is a
difference of f32 values, exact in f64 where the teacher's are within 2^29 of each other, and 0 or lost beside 1 where not."""
import numpy as np
import pytest

import noetic_rl as nr
from tests import draft_reference as ref
from tests.test_distill_gpu import both

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    nr.claim(0)
    yield


@pytest.mark.parametrize("value", [-1e4, -1e9, -1e13, float(np.finfo(np.float32).min), 1e30])
@pytest.mark.parametrize("some", [False, True])
@pytest.mark.parametrize("R, V, k", [(6, 900, 8), (3, 2000, 700), (1, 130000, 20)])
def test_teachers_logits_of_any_size(R, V, k, value, some):
    rng = np.random.default_rng(V)
    x = ref.rounded(rng.normal(0, 2, (R, V)), "f32")
    ids = np.stack([rng.permutation(V)[:k] for _ in range(R)]).astype(np.int32)
    ids[:, 1] = -1
    lp = rng.normal(0, 2, (R, k)).astype(np.float32)
    lp[:, k // 2 if some else 0:] += np.float32(value)
    both(x, x, None, ids, lp, "f32", 1.0, "RENORMALIZE", np.random.default_rng(1))
