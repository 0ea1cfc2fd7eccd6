"""Distillation under an additive mask that lowers a whole row: the sums and the listed tokens are of the same values, x / T + mask
in f64, of whose differences an f32 step of the mask is no small part. Against the f64 form in logarithms (where some tokens are
lowered by less, others' probabilities are below f64's range), with the errors and tolerances of the operator's own tests.

At -1e13 a step of z itself, 2^-9 in f64, is no small part either: x / T here and x times 1 / T there, rounded by the addition,
can lie on both sides of a half (247 / 2048 at T 1.3 is 47.5 steps), so by dz = 2^-52 |z| apart (T 1: both are the same sum; at
the lowest value no logit reaches half a step). A loss then moves by at most sum |d / dz| dz <= 2 mass dz, mass <= 1, and each probability
by the factor e^(2 dz), under 1 + 2.1 dz."""
import numpy as np
import pytest

import noetic_rl as nr
from tests import draft_reference as ref
from tests.test_distill_far_rest_gpu import form
from tests.test_distill_gpu import E, TINY

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    nr.claim(0)
    yield


@pytest.mark.parametrize("tail", ["REST", "DROP", "RENORMALIZE"])
@pytest.mark.parametrize("value", [-1e5, -1e9, -1e13, float(np.finfo(np.float32).min)])
@pytest.mark.parametrize("R, V, k, dtype, T, gdt", [
    (5, 1000, 8, "f32", 1.0, None),
    (3, 7, 2, "bf16", 0.7, "f32"),
    (300, 1003, 5, "f16", 1.3, "f32"),
    (1, 130000, 20, "f32", 0.9, None),      # several workgroups
])
def test_a_mask_that_lowers_every_token(R, V, k, dtype, T, gdt, value, tail):
    rng = np.random.default_rng(V + k)
    x = ref.rounded(rng.normal(0, 2, (R, V)), dtype)
    ids = np.stack([rng.permutation(V)[:k] for _ in range(R)]).astype(np.int32)
    lp = ref.log_softmax(np.concatenate([rng.normal(0, 2, (R, k)), np.ones((R, 1))], 1))[:, :k].astype(np.float32)
    add = np.full((1, V), value, np.float32)
    add[0, ::11] += np.float32(abs(value) * 1e-4)   # (some lowered by less)
    logits, it, lt = nr.Tempered(ref.tensor(x, dtype), T, nr.Tensor.from_numpy(add)), nr.Tensor.from_numpy(ids), nr.Tensor.from_numpy(lp)
    loss, stats = nr.distill_with_stats(logits, it, lt, nr.TeacherTail[tail])
    g = rng.normal(0, 1, R).astype(np.float32)
    grad = ref.values(nr.distill_grad(logits, it, lt, stats, nr.Tensor.from_numpy(g), gdt))
    want, wg, tol, first = form(x / T + add.astype(np.float64), ids, lp, tail)
    dz = 0.0 if T == 1.0 or value < -1e30 else 2.0 ** -52 * abs(value)
    assert (np.abs(loss.to_numpy() - want) / (2.0 ** -24 * np.abs(want) + 2 * E * first + 2 * dz + 1e-9)).max() <= 1
    s = g.astype(np.float64)[:, None] / T
    held = gdt or dtype
    tol = tol * (1 + 2.1 * dz / (2 * E)) * np.abs(s) * (1 + 2.0 ** -7) + ref.HALF_ULP[held] * np.abs(wg * s) + TINY[held]
    assert (np.abs(grad - wg * s) / tol).max() <= 1
