"""Top log-probabilities (top_logprobs) against a stable sort and an f64 log-softmax.

Ids have to be equal. A log-probability's error is the log-sum-exp's: f32 exponentials of arguments t in log2 units, each
within 2^-23 (the instruction) and |t| 3 2^-24 ln 2 (the difference's, the scale's and the product's roundings),
which weighted by the softmax has |t| below 24, and sums of 64 terms a lane in trees (7 roundings): 4e-6 at the most, and
half an f32 step of the result."""
import ctypes as C

import numpy as np
import pytest

from tests import draft_reference as ref
import noetic_rl as nr
from tests.test_kept_blocks_gpu import Capture

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    nr.claim(0)
    yield


def compare(got, key, z, k):
    ids, lp = (t.to_numpy() for t in got)
    wi, wl = ref.top(key, z, k)
    assert np.array_equal(ids, wi)
    fine = wi >= 0
    assert np.array_equal(lp == -np.inf, ~fine)
    assert (np.abs(lp - wl)[fine] <= 2.0 ** -24 * np.abs(wl)[fine] + 4e-6).all()


CASES = [
    # (rows, V, k, dtype, mask, shared, T)
    (1, 128256, 20, "bf16", "none", False, 1.0),
    (1, 1, 1, "f32", "none", False, 1.0),
    (3, 5, 5, "f16", "u8", False, 0.7),
    (7, 511, 64, "f32", "f32", False, 1.0),
    (5, 513, 513, "bf16", "none", False, 2.0),        # the whole row, sorted
    (4, 2049, 1024, "f32", "u8", False, 1.0),
    (2, 151936, 1024, "f32", "none", False, 1.0),
    (40, 50257, 50, "f16", "f32", True, 0.7),
    (1100, 5001, 64, "bf16", "none", False, 1.0),     # one workgroup a row
    (1030, 8192, 128, "f32", "u8", False, 1.3),
    (1030, 20000, 7, "f16", "u8", True, 1.0),
    (1025, 9000, 256, "f32", "f32", False, 0.5),
    (1024, 36000, 1000, "bf16", "none", False, 1.0),
    (600, 3000, 33, "bf16", "f32", False, 1.0),
]


@pytest.mark.parametrize("case", CASES)
def test_against_a_stable_sort(case):
    R, V, k, dtype, kind, shared, T = case
    rng = np.random.default_rng(R + V + k)
    x = ref.rounded(rng.normal(0, 2, (R, V)), dtype)
    mt, add, off = ref.make_mask(kind, R, V, rng, shared=shared)
    z = ref.tempered(x, T, add, off)
    key = np.where(off, -np.inf, x)
    if kind == "f32":  # ordered by the tempered logits in f32
        key = ((x.astype(np.float32) / np.float32(T)).astype(np.float32) + add.astype(np.float32)).astype(np.float64)
        z = key
    got = nr.top_logprobs(nr.Tempered(ref.tensor(x, dtype), T, mt), k)
    compare(got, key, z, k)
    again = nr.top_logprobs(nr.Tempered(ref.tensor(x, dtype), T, mt), k)
    assert all(a.to_numpy().tobytes() == b.to_numpy().tobytes() for a, b in zip(got, again))


@pytest.mark.parametrize("R", [3, 1025])
@pytest.mark.parametrize("shape", ["equal", "rising", "falling", "two", "zeros", "steps", "late"])
@pytest.mark.parametrize("k", [1, 40, 1024])
def test_rows_that_fill_the_list(R, shape, k):
    """Rows of equal values, rising ones (every tile brings more than the last), both zeros, the largest ones last."""
    V = 20011
    rng = np.random.default_rng(k)
    v = np.arange(V)
    x = {"equal": np.full(V, -3.0), "rising": v / 64.0, "falling": -v / 64.0, "two": (v % 2).astype(float),
         "zeros": np.where(rng.random(V) < 0.5, 0.0, -0.0), "steps": np.floor(v / 999.0),
         "late": np.where(v > V - 3000, 5.0 + rng.random(V), rng.random(V))}[shape]
    x = ref.rounded(np.broadcast_to(x, (R, V)), "f32")
    compare(nr.top_logprobs(ref.tensor(x, "f32"), k), x + 0.0, x, k)


def test_rows_without_tokens_and_bad_ones():
    V, k = 3000, 9
    x = np.random.default_rng(1).normal(0, 1, (6, V)).astype(np.float32)
    x[0] = -np.inf
    x[1, 17] = np.nan
    x[2, 18] = np.inf
    x[3, 4:] = -np.inf                  # four tokens
    keep = np.ones((6, V), np.uint8)
    keep[4] = 0
    keep[5, 17] = 0
    x[5, 17] = np.nan                   # excluded: does not matter
    t = nr.Tempered(nr.Tensor.from_numpy(x), 1.0, nr.Tensor.from_numpy(keep, "u8"))
    ids, lp = (a.to_numpy() for a in nr.top_logprobs(t, k, check=False))
    for r in (0, 1, 2, 4):
        assert (ids[r] == -1).all() and np.isnan(lp[r]).all()
    assert sorted(ids[3][:4]) == [0, 1, 2, 3] and (ids[3][4:] == -1).all() and (lp[3][4:] == -np.inf).all()
    assert (ids[5] >= 0).all() and 17 not in ids[5] and np.isfinite(lp[5]).all()
    with pytest.raises(ValueError, match="position 0 has no allowed token"):
        nr.top_logprobs(t, k)


def test_extreme_logits_and_masks():
    V, k = 4000, 30
    rng = np.random.default_rng(2)
    x = rng.normal(0, 1, (2, V)).astype(np.float32)
    x[0, :10] = 3e38
    x[0, 10:20] = -3e38
    x[1] *= 1e-40                       # subnormal
    add = np.zeros((1, V), np.float32)
    add[0, 100:] = np.finfo(np.float32).min
    for m in (None, nr.Tensor.from_numpy(add)):
        z = x.astype(np.float32) + (0 if m is None else add)
        got = nr.top_logprobs(nr.Tempered(nr.Tensor.from_numpy(x), 1.0, m), k)
        compare(got, z.astype(np.float64), z.astype(np.float64), k)


def test_rows_behind_and_strides():
    rng = np.random.default_rng(3)
    R, V, ld, k = 5, 1003, 1100, 12
    x = rng.normal(0, 1, (R, ld)).astype(np.float32)
    xt = nr.Tensor.from_numpy(x)
    ids, lp = nr.Tensor.from_numpy(np.full((R + 1, k), 77, np.int32)), nr.Tensor.from_numpy(np.full((R + 1, k), 77, np.float32))
    st = nr.Tensor.from_numpy(np.full(R + 1, 77, np.uint8), "u8")
    a = nr.NtRlTopArgs(xt.ptr, 0, 0, R, V, ld, None, 0, 1.0, k, ids.ptr, lp.ptr, st.ptr)
    assert nr.lib().nt_hip_rl_top_logprobs(C.byref(a)) == 0
    ids, lp, st = ids.to_numpy(), lp.to_numpy(), st.to_numpy()
    assert np.array_equal(ids[:R], ref.top(x[:, :V].astype(np.float64), x[:, :V].astype(np.float64), k)[0])
    assert (ids[R] == 77).all() and (lp[R] == 77).all() and st.tolist() == [0] * R + [77]


@pytest.mark.parametrize("R", [2, 1030])
def test_captured_calls_replay(R):
    rng = np.random.default_rng(4)
    V, k = 5000, 10
    xt = nr.Tensor((R, V), "f32")
    ids, lp, st = nr.Tensor((R, k), "i32"), nr.Tensor((R, k), "f32"), nr.Tensor((R,), "u8")

    def call():
        a = nr.NtRlTopArgs(xt.ptr, 0, 0, R, V, V, None, 0, 1.0, k, ids.ptr, lp.ptr, st.ptr)
        nr._check(nr.lib().nt_hip_rl_top_logprobs(C.byref(a)), "top")

    call()
    nr.sync()
    cap = Capture()
    with cap:
        call()
    for _ in range(3):
        x = rng.normal(0, 1, (R, V)).astype(np.float32)
        nr._check(nr.lib().nt_hip_upload(C.c_void_p(xt.ptr), x.ctypes.data_as(C.c_void_p), xt.nbytes), "upload")
        want = nr.top_logprobs(nr.Tensor.from_numpy(x), k)
        cap.replay()
        nr.sync()
        assert ids.to_numpy().tobytes() == want[0].to_numpy().tobytes()
        assert lp.to_numpy().tobytes() == want[1].to_numpy().tobytes()
    cap.close()
