"""Distillation from a teacher's listed tokens (distill_with_stats, distill_grad) against a plain f64 form.

Errors. The row's sums are of f32 exponentials: e = 4e-6 relative at the most (the scorer's: see the top
log-probabilities' tests). Loss: its derivative by an error of the sums is sum q - sum w over the list and, with
tail REST, off it too, so |sum w - sum q| e there, and e times the mass for the other tails; second order is below 1e-9.
Gradient of an unlisted column: q (mass - rest / q_off), both factors' sums within e and the exponential within
2^-23 + |t| 3 2^-24 ln 2, t its argument in log2 units (at most 150; smaller ones are 0): (mass + share) q (2 e + 2e-5), and half a
step of the gradient's type; of a listed one mass q e and that half step. Below f32's range nothing is held to a
relative error."""
import ctypes as C

import numpy as np
import pytest

from tests import draft_reference as ref
import noetic_rl as nr
from tests.test_kept_blocks_gpu import Capture

pytestmark = pytest.mark.gpu
E = 4e-6
TINY = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -24}  # half of f16's smallest step is 2^-25


@pytest.fixture(scope="module", autouse=True)
def device():
    nr.claim(0)
    yield


def inputs(R, V, k, dtype, kind, T, rng, shared=False, noise=0.5, std=2.0):
    x = ref.rounded(rng.normal(0, std, (R, V)), dtype)
    mt, add, off = ref.make_mask(kind, R, V, rng, shared=shared)
    z = ref.tempered(x, T, add, off)
    tz = ref.tempered(x + rng.normal(0, noise, (R, V)), T, add, off)
    order = np.argsort(-tz, axis=1, kind="stable")[:, :k]
    lp = np.take_along_axis(ref.log_softmax(tz), order, 1).astype(np.float32)
    ids = np.where(lp > -np.inf, order, -1).astype(np.int32)
    for r in range(R):  # in no order
        s = rng.permutation(k)
        ids[r], lp[r] = ids[r, s], lp[r, s]
    return x, z, mt, ids, lp


def check_loss(loss, want, parts, tail):
    q, listed, w, rest, q_off, mass, share = parts
    first = np.abs(q_off - rest) if tail == "REST" else mass
    fine = np.isfinite(want)
    assert np.array_equal(loss[~fine], want[~fine])
    err = np.abs(loss - want)[fine]
    assert (err <= (2.0 ** -24 * np.abs(want) + 2 * E * first + 1e-9)[fine]).all(), err.max()


def check_grad(grad, want, parts, g, T, dtype):
    q, listed, w, rest, q_off, mass, share = parts
    s = np.abs(g)[:, None] / T
    unlisted = (mass + share)[:, None] * q * (2 * E + 2e-5)
    tol = s * np.where(listed, mass[:, None] * q * 2 * E + 1e-12, unlisted) * (1 + 2.0 ** -7)
    want = want * (g / T)[:, None]
    tol = tol + ref.HALF_ULP[dtype] * np.abs(want) + TINY[dtype]
    err = np.abs(grad - want)
    assert (err <= tol).all(), (np.argwhere(err > tol)[:3], err[err > tol][:3], tol[err > tol][:3])


def both(x, z, mt, ids, lp, dtype, T, tail, rng, gdt=None, scale=1.0):
    logits = nr.Tempered(ref.tensor(x, dtype), T, mt)
    it, lt = nr.Tensor.from_numpy(ids), nr.Tensor.from_numpy(lp)
    loss, stats = nr.distill_with_stats(logits, it, lt, nr.TeacherTail[tail])
    g = (rng.normal(0, 1, len(ids)) * scale).astype(np.float32)
    g[::5] = 0.0
    grad = nr.distill_grad(logits, it, lt, stats, nr.Tensor.from_numpy(g), gdt)
    wl, wg, parts = ref.distill(z, ids, lp, tail)
    check_loss(loss.to_numpy().astype(np.float64), wl, parts, tail)
    gv = ref.values(grad)
    assert (gv[g == 0.0] == 0.0).all()
    check_grad(gv, wg, parts, g.astype(np.float64), T, gdt or dtype)
    return loss, grad, stats


CASES = [
    # (rows, V, k, dtype, mask, shared, T, gradient's dtype)
    (1, 1, 1, "f32", "none", False, 1.0, None),
    (2, 7, 3, "f32", "u8", False, 0.7, "bf16"),
    (3, 7, 7, "f16", "none", False, 1.0, "f32"),      # the whole row is listed
    (5, 511, 16, "bf16", "f32", False, 1.3, None),
    (5, 512, 64, "f16", "u8", True, 2.0, None),
    (4, 4099, 1024, "f32", "none", False, 1.0, None),
    (40, 50257, 50, "f16", "u8", False, 2.0, None),
    (3, 128256, 64, "bf16", "none", False, 1.0, None),
    (1, 300000, 8, "f32", "none", False, 1.0, "f16"),  # more columns than one workgroup's bitmap
    (1100, 5001, 20, "bf16", "none", False, 1.0, "f32"),
    (1030, 4096, 33, "f32", "f32", True, 0.8, None),
    (5000, 1000, 10, "bf16", "u8", False, 1.0, None),
    (260, 2056, 100, "f32", "f32", False, 1.0, "bf16"),
]


@pytest.mark.parametrize("tail", ["REST", "DROP", "RENORMALIZE"])
@pytest.mark.parametrize("case", CASES)
def test_against_the_formula(case, tail):
    R, V, k, dtype, kind, shared, T, gdt = case
    rng = np.random.default_rng(R + V + k)
    x, z, mt, ids, lp = inputs(R, V, k, dtype, kind, T, rng, shared)
    got = both(x, z, mt, ids, lp, dtype, T, tail, np.random.default_rng(1), gdt, 64.0 if (gdt or dtype) == "f16" else 1.0)
    again = both(x, z, mt, ids, lp, dtype, T, tail, np.random.default_rng(1), gdt, 64.0 if (gdt or dtype) == "f16" else 1.0)
    assert got[0].to_numpy().tobytes() == again[0].to_numpy().tobytes()
    assert got[1].to_numpy().tobytes() == again[1].to_numpy().tobytes()


@pytest.mark.parametrize("tail", ["REST", "DROP", "RENORMALIZE"])
def test_gradient_against_differences(tail):
    """The f32 gradient against central differences of the f64 loss: step h = 1e-3, whose error is h^2 / 6 times the third
    derivative, at most 1 over softmaxes: 2e-7, with 1e-5 of the gradient's own."""
    rng = np.random.default_rng(3)
    R, V, k, T, h = 3, 40, 5, 1.7, 1e-3
    x, z, mt, ids, lp = inputs(R, V, k, "f32", "none", T, rng)
    logits, it, lt = nr.Tempered(ref.tensor(x, "f32"), T, None), nr.Tensor.from_numpy(ids), nr.Tensor.from_numpy(lp)
    loss, stats = nr.distill_with_stats(logits, it, lt, nr.TeacherTail[tail])
    grad = nr.distill_grad(logits, it, lt, stats, nr.Tensor.from_numpy(np.ones(R, np.float32))).to_numpy()
    for v in range(V):
        up, down = x.copy(), x.copy()
        up[:, v] += h
        down[:, v] -= h
        d = (ref.distill(up / T, ids, lp, tail)[0] - ref.distill(down / T, ids, lp, tail)[0]) / (2 * h)
        assert (np.abs(grad[:, v] - d) <= 2e-7 + 1e-5 * np.abs(d)).all()


def test_a_student_near_its_teacher():
    """Losses down to 1e-7, a difference of sums around 10: within 1e-5 of their value and 1e-9."""
    rng = np.random.default_rng(4)
    for noise in (0.1, 0.01, 0.001):
        x, z, mt, ids, lp = inputs(16, 30000, 64, "f32", "none", 1.0, rng, noise=noise)
        loss, _ = nr.distill_with_stats(ref.tensor(x, "f32"), nr.Tensor.from_numpy(ids), nr.Tensor.from_numpy(lp))
        want = ref.distill(z, ids, lp, "REST")[0]
        # (|sum q - sum w| off the list is about noise / 10)
        assert (np.abs(loss.to_numpy() - want) <= 1e-5 * want + 2 * E * noise * 0.2 + 1e-9).all()


def test_padding_zero_weights_and_excluded_tokens():
    rng = np.random.default_rng(5)
    R, V, k = 6, 900, 8
    x, z, _, ids, lp = inputs(R, V, k, "f32", "none", 1.0, rng)
    lp[0, 3] = -np.inf                        # a weight of 0
    ids[1, 2] = -1                            # padding, whatever its weight says
    ids[2] = -1                               # nothing listed: all of the teacher is rest, and so is the student
    keep = np.ones((R, V), np.uint8)
    keep[3, ids[3, 0]] = 0                    # a listed token that the student may not take: +inf
    keep[4] = 0
    keep[4, ids[4]] = 1                       # nothing off the list is allowed
    z = np.where(keep == 0, -np.inf, z)
    for tail in ("REST", "DROP", "RENORMALIZE"):
        loss, grad, _ = both(x, z, nr.Tensor.from_numpy(keep, "u8"), ids, lp, "f32", 1.0, tail, np.random.default_rng(2))
        loss = loss.to_numpy()
        assert loss[3] == np.inf and np.isfinite(np.delete(loss, 3)).all()
        assert abs(loss[2]) < 1e-9


def test_refused_rows():
    rng = np.random.default_rng(6)
    R, V, k = 7, 2000, 6
    x, z, _, ids, lp = inputs(R, V, k, "f32", "none", 1.0, rng)
    x = x.astype(np.float32)
    x[0] = -np.inf
    x[1, 7] = np.nan
    x[2, 7] = np.inf
    ids[3, 1] = V
    ids[4, 1] = -2
    ids[5, 5] = ids[5, 0]
    xt, it, lt = nr.Tensor.from_numpy(x), nr.Tensor.from_numpy(ids), nr.Tensor.from_numpy(lp)
    loss, stats = nr.distill_with_stats(xt, it, lt, check=False)
    assert np.isnan(loss.to_numpy()[:6]).all() and np.isfinite(loss.to_numpy()[6])
    g = np.ones(R, np.float32)
    grad = nr.distill_grad(xt, it, lt, stats, nr.Tensor.from_numpy(g)).to_numpy()
    assert np.isnan(grad[:6]).all() and np.isfinite(grad[6]).all()
    g[:6] = 0.0
    assert (nr.distill_grad(xt, it, lt, stats, nr.Tensor.from_numpy(g)).to_numpy()[:6] == 0.0).all()
    with pytest.raises(IndexError, match="position 3 lists a token"):
        nr.distill_with_stats(xt, it, lt)


def test_a_row_past_the_last_and_strides():
    rng = np.random.default_rng(7)
    R, V, ld, gld, k = 3, 1003, 1040, 1017, 9
    x, _, _, ids, lp = inputs(R, ld, k, "f32", "none", 1.0, rng)
    ids = (ids % V).astype(np.int32)
    for r in range(R):
        ids[r] = rng.permutation(V)[:k]
    z = x[:, :V]
    xt, it, lt = ref.tensor(x, "f32"), nr.Tensor.from_numpy(ids), nr.Tensor.from_numpy(lp)
    loss = nr.Tensor.from_numpy(np.full(R + 1, 77, np.float32))
    stats = nr.Tensor.from_numpy(np.full((R + 1, 5), 77.0))
    st = nr.Tensor.from_numpy(np.full(R + 1, 77, np.uint8), "u8")
    grad = nr.Tensor.from_numpy(np.full((R + 1, gld), 77, np.float32))
    g = nr.Tensor.from_numpy(np.ones(R, np.float32))
    a = nr.NtRlDistillArgs(xt.ptr, 0, 0, R, V, ld, None, 0, 1.0, k, it.ptr, lt.ptr, 1, 0, loss.ptr, stats.ptr, st.ptr)
    assert nr.lib().nt_hip_rl_distill(C.byref(a)) == 0
    b = nr.NtRlDistillGradArgs(xt.ptr, 0, 0, R, V, ld, None, 0, 1.0, k, it.ptr, lt.ptr, stats.ptr, g.ptr, grad.ptr, 0, 0, gld)
    assert nr.lib().nt_hip_rl_distill_backward(C.byref(b)) == 0
    wl, wg, parts = ref.distill(z, ids, lp, "DROP")
    check_loss(loss.to_numpy()[:R].astype(np.float64), wl, parts, "DROP")
    grad = grad.to_numpy()
    check_grad(grad[:R, :V], wg, parts, np.ones(R), 1.0, "f32")
    assert (grad[:R, V:] == 77).all() and (grad[R] == 77).all()
    assert loss.to_numpy()[R] == 77 and (stats.to_numpy()[R] == 77).all() and st.to_numpy()[R] == 77


@pytest.mark.parametrize("R", [2, 1100])
def test_captured_calls_replay(R):
    rng = np.random.default_rng(8)
    V, k = 3001, 7
    xt, it, lt = nr.Tensor((R, V), "f32"), nr.Tensor((R, k), "i32"), nr.Tensor((R, k), "f32")
    g = nr.Tensor.from_numpy(np.ones(R, np.float32))
    loss, stats, st, grad = nr.Tensor((R,), "f32"), nr.Tensor((R, 5), "f64"), nr.Tensor((R,), "u8"), nr.Tensor((R, V), "f32")

    def call():
        a = nr.NtRlDistillArgs(xt.ptr, 0, 0, R, V, V, None, 0, 1.0, k, it.ptr, lt.ptr, 0, 0, loss.ptr, stats.ptr, st.ptr)
        nr._check(nr.lib().nt_hip_rl_distill(C.byref(a)), "distill")
        b = nr.NtRlDistillGradArgs(xt.ptr, 0, 0, R, V, V, None, 0, 1.0, k, it.ptr, lt.ptr, stats.ptr, g.ptr, grad.ptr, 0, 0, V)
        nr._check(nr.lib().nt_hip_rl_distill_backward(C.byref(b)), "backward")

    call()
    nr.sync()
    cap = Capture()
    with cap:
        call()
    for _ in range(3):
        x, z, _, ids, lp = inputs(R, V, k, "f32", "none", 1.0, rng)
        new = (x.astype(np.float32), ids, lp)
        for t, v in zip((xt, it, lt), new):
            nr._check(nr.lib().nt_hip_upload(C.c_void_p(t.ptr), np.ascontiguousarray(v).ctypes.data_as(C.c_void_p), t.nbytes), "upload")
        e = [nr.Tensor.from_numpy(v) for v in new]
        wl, ws = nr.distill_with_stats(*e)
        wg = nr.distill_grad(*e, ws, g)
        cap.replay()
        nr.sync()
        assert loss.to_numpy().tobytes() == wl.to_numpy().tobytes()
        assert grad.to_numpy().tobytes() == wg.to_numpy().tobytes()
    cap.close()


def test_a_drafter_learns_and_its_drafts_are_verified():
    """The operators as they are used together: a teacher's top log-probabilities are recorded, a drafter's logits take
    descent steps on the divergence (each within what the gradient's norm promises, 1/2 |g|^2 a step
    of 1 being a lower bound for a softmax, whose curvature is at most 1/2), its sampled drafts are verified."""
    rng = np.random.default_rng(9)
    S, B, K, V, k = 1, 32, 3, 2000, 32
    T = 0.9
    teacher = nr.Tensor.from_numpy(rng.normal(0, 2, (S, B, K + 1, V)).astype(np.float32))
    part = nr.Tensor.from_numpy(teacher.to_numpy()[:, :, :K].copy())
    ids, lp = nr.top_logprobs(nr.Tempered(part, T, None), k)
    student = rng.normal(0, 2, (S, B, K, V)).astype(np.float32)
    ones = nr.Tensor.from_numpy(np.ones((S, B, K), np.float32))
    before = None
    for _ in range(5):
        t = nr.Tempered(nr.Tensor.from_numpy(student), T, None)
        loss, stats = nr.distill_with_stats(t, ids, lp)
        grad = nr.distill_grad(t, ids, lp, stats, ones).to_numpy().astype(np.float64)
        if before is not None:
            assert (loss.to_numpy() <= before + 1e-5).all()
        # (the loss at the next point is below loss - step |g|^2 (1 - step / (4 T^2)))
        step = T * T
        before = loss.to_numpy() - step * (1 - 0.25) * (grad ** 2).sum(-1)
        student = (student - step * grad).astype(np.float32)
    reduced = nr.distillation_loss(nr.Tempered(nr.Tensor.from_numpy(student), T, None), ids, lp)
    per = nr.distill_with_stats(nr.Tempered(nr.Tensor.from_numpy(student), T, None), ids, lp)[0].to_numpy()
    assert abs(reduced.to_numpy()[0] - per.mean()) <= 1e-6 * per.mean() + 1e-7
    draft = nr.Tensor.from_numpy(student)
    tokens, _ = nr.sample_logp(draft, T, None, nr.Rng(1, "draft"))
    r = nr.Rng(2, "verify")
    u = r.clone().uniforms(S * B * (K + 1)).reshape(B, K + 1)
    got = nr.verify_drafted(teacher, draft, tokens, T, None, r)
    want = ref.verify(teacher.to_numpy()[0].astype(np.float64) / T, student[0].astype(np.float64) / T, tokens.to_numpy()[0], u,
                      np.full(B, K), False)
    assert np.array_equal(got[0].to_numpy()[0], want[0]) and np.array_equal(got[1].to_numpy()[0], want[1])
    kept = np.arange(K + 1) <= got[1].to_numpy()[0][:, None]
    assert (got[0].to_numpy()[0][kept] >= 0).all() and (got[0].to_numpy()[0][~kept] == -1).all()
