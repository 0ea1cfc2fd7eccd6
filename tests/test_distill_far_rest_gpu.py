"""Distillation where what is off the list lies far below (or above) the listed tokens: its sum, the loss's term and
the gradient keep what f32 exponentials next to a listed token would lose.

The formula in logarithms, f64: loss = sum w (ln w - ln q) + rest (ln rest - ln q_off), d / dz = mass q - w at a listed token and
mass q - rest softmax_off elsewhere, softmax_off that of the unlisted tokens alone. Errors as in the operator's own
tests: sums within E relative, so |q_off - rest| E of the loss, and of an unlisted gradient its two terms' (2 E + 2e-5)."""
import numpy as np
import pytest

import noetic_rl as nr
from tests import draft_reference as ref
from tests.test_distill_gpu import E, TINY

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    nr.claim(0)
    yield


def lse(z):
    """The largest and what the log-sum-exp is above it, apart: the largest may be of any size."""
    m = z.max(1, keepdims=True)
    return m, np.log(np.exp(z - m).sum(1, keepdims=True))


def form(z, ids, lp, tail):
    """loss [R], gradient [R, V], its tolerance (without the rounding), |d loss / d ln q_off|."""
    R, V = z.shape
    w, rest = ref.teacher_weights(lp, ids, tail)
    on = np.zeros((R, V), bool)
    np.put_along_axis(on, ids, True, 1)
    (m, above), (m_off, above_off) = lse(z), lse(np.where(on, -np.inf, z))
    lnq, ln_off = (z - m) - above, ((m_off - m) + (above_off - above))[:, 0]
    dense = np.zeros((R, V))
    np.put_along_axis(dense, ids, w, 1)
    mass = w.sum(1) + rest
    with np.errstate(invalid="ignore", divide="ignore"):
        loss = np.where(w > 0, w * (np.log(w) - np.take_along_axis(lnq, ids, 1)), 0.0).sum(1)
        loss = loss + np.where(rest > 0, rest * (np.log(rest) - ln_off), 0.0)
    q = np.exp(lnq)
    alone = rest[:, None] * np.exp(np.minimum((z - m_off) - above_off, 0.0))
    grad = np.where(on, mass[:, None] * q - dense, mass[:, None] * q - alone)
    tol = np.where(on, mass[:, None] * q * 2 * E + 1e-12, (mass[:, None] * q + alone) * (2 * E + 2e-5))
    first = np.abs(np.exp(ln_off) - rest) if tail == "REST" else mass
    return loss, grad, tol, first


def rows(V, gap, T, dtype, R, k, rng):
    """x and z, ids, teacher: the listed tokens `gap` above the others in z, but for one listed among them."""
    x = rng.normal(0, 1, (R, V))
    ids = np.stack([rng.permutation(V)[:k] for _ in range(R)]).astype(np.int32)
    ids[0] = np.arange(k)               # (together, in one lane)
    top = np.take_along_axis(x, ids, 1) + gap * T
    if k > 2:
        top[:, -1] -= gap * T
    np.put_along_axis(x, ids, top, 1)
    x = ref.rounded(x, dtype)
    lp = np.log(np.full((R, k), 0.6 / k)).astype(np.float32)
    return x, x / T, ids, lp


CASES = [(V, gap, T, dtype) for V, T, dtype in [(8, 1.0, "f32"), (5, 0.1, "f16"), (1000, 1.0, "f32"), (1000, 0.1, "bf16"), (4099, 2.0, "f16"),
                                                (130000, 1.0, "f32")] for gap in (60, 90, 120, 300, 900, -300)]


@pytest.mark.parametrize("tail", ["REST", "DROP"])
@pytest.mark.parametrize("V, gap, T, dtype", CASES)
def test_the_loss_of_a_far_rest(V, gap, T, dtype, tail):
    rng = np.random.default_rng(V + abs(gap))
    for R in (2, 300) if V < 100000 else (2,):
        x, z, ids, lp = rows(V, gap, T, dtype, R, min(4, V // 3), rng)
        loss, _ = nr.distill_with_stats(nr.Tempered(ref.tensor(x, dtype), T, None), nr.Tensor.from_numpy(ids),
                                        nr.Tensor.from_numpy(lp), nr.TeacherTail[tail])
        want, _, _, first = form(z, ids, lp, tail)
        assert (np.abs(loss.to_numpy() - want) <= 2.0 ** -24 * np.abs(want) + 2 * E * first + 1e-9).all()


def test_one_unlisted_token_that_the_mask_allows():
    """A keep-mask that leaves the listed tokens and one far below them, in the first one's lane and elsewhere."""
    rng = np.random.default_rng(1)
    R, V, k = 6, 3000, 3
    x = ref.rounded(rng.normal(0, 1, (R, V)), "f32")
    ids = np.tile(np.array([8, 9, 2000], np.int32), (R, 1))
    other = np.array([10, 10, 15, 500, 2999, 2003])
    keep = np.zeros((R, V), np.uint8)
    np.put_along_axis(keep, ids, 1, 1)
    keep[np.arange(R), other] = 1
    x[np.arange(R), other] -= np.array([100.0, 400.0, 2000.0, 100.0, 400.0, 2000.0])
    x = ref.rounded(x, "f32")
    lp = np.log(np.full((R, k), 0.25)).astype(np.float32)
    z = np.where(keep == 0, -np.inf, x)
    loss, _ = nr.distill_with_stats(nr.Tempered(ref.tensor(x, "f32"), 1.0, nr.Tensor.from_numpy(keep, "u8")),
                                    nr.Tensor.from_numpy(ids), nr.Tensor.from_numpy(lp))
    want, _, _, first = form(z, ids, lp, "REST")
    assert (np.abs(loss.to_numpy() - want) <= 2.0 ** -24 * np.abs(want) + 2 * E * first + 1e-9).all() and (want > 20).all()


@pytest.mark.parametrize("tail", ["REST", "DROP"])
@pytest.mark.parametrize("V, gap, T, dtype", CASES)
def test_its_gradient(V, gap, T, dtype, tail):
    rng = np.random.default_rng(V + abs(gap) + 1)
    for R in (2, 300) if V < 100000 else (2,):
        x, z, ids, lp = rows(V, gap, T, dtype, R, min(4, V // 3), rng)
        logits, it, lt = nr.Tempered(ref.tensor(x, dtype), T, None), nr.Tensor.from_numpy(ids), nr.Tensor.from_numpy(lp)
        _, stats = nr.distill_with_stats(logits, it, lt, nr.TeacherTail[tail])
        # (f16: a loss scale)
        g = (rng.uniform(0.5, 1.0, R) * (4096.0 if dtype == "f16" else 1.0)).astype(np.float32)
        got = ref.values(nr.distill_grad(logits, it, lt, stats, nr.Tensor.from_numpy(g)))
        _, want, tol, _ = form(z, ids, lp, tail)
        s = g.astype(np.float64)[:, None] / T
        err = np.abs(got - want * s)
        assert (err <= tol * s * (1 + 2.0 ** -7) + ref.HALF_ULP[dtype] * np.abs(want * s) + TINY[dtype]).all()


def test_excluded_columns_beside_a_far_rest_have_no_gradient():
    rng = np.random.default_rng(2)
    for gap in (50.0, 100.0, 1000.0):
        R, V, k = 4, 2003, 2
        x, z, ids, lp = rows(V, gap, 1.0, "f32", R, k, rng)
        keep = (rng.random((R, V)) < 0.5).astype(np.uint8)
        np.put_along_axis(keep, ids, 1, 1)
        logits = nr.Tempered(ref.tensor(x, "f32"), 1.0, nr.Tensor.from_numpy(keep, "u8"))
        it, lt = nr.Tensor.from_numpy(ids), nr.Tensor.from_numpy(lp)
        _, stats = nr.distill_with_stats(logits, it, lt)
        got = nr.distill_grad(logits, it, lt, stats, nr.Tensor.from_numpy(np.ones(R, np.float32))).to_numpy()
        _, want, tol, _ = form(np.where(keep == 0, -np.inf, z), ids, lp, "REST")
        assert (got[keep == 0] == 0.0).all()
        assert (np.abs(got - want) <= tol + 2.0 ** -24 * np.abs(want) + TINY["f32"]).all()
