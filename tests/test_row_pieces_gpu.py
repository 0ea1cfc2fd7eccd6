"""Rows so long and so few that several workgroups take one (top log-probabilities, distillation): rows that fill the lists
which they hand on, and graphs, whose workspace is theirs. Tolerances as in the operators' own tests."""
import ctypes as C

import numpy as np
import pytest

import noetic_rl as nr
from tests import draft_reference as ref
from tests.test_kept_blocks_gpu import Capture

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    nr.claim(0)
    yield


@pytest.mark.parametrize("V", [130001, 262144])
@pytest.mark.parametrize("shape", ["normal", "equal", "rising", "steps", "last"])
@pytest.mark.parametrize("k", [1, 100, 1024])
def test_top_of_long_rows(V, shape, k):
    rng = np.random.default_rng(V + k)
    v = np.arange(V)
    x = {"normal": rng.normal(0, 2, V), "equal": np.zeros(V), "rising": v / 128.0, "steps": np.floor(v / 9999.0),
         "last": np.where(v >= V - 1, 1.0, -np.inf)}[shape]
    x = ref.rounded(np.broadcast_to(x, (2, V)), "f32")
    ids, lp = (t.to_numpy() for t in nr.top_logprobs(ref.tensor(x, "f32"), k))
    wi, wl = ref.top(x, x, k)
    assert np.array_equal(ids, wi)
    some = wi >= 0
    assert (np.abs(lp - wl)[some] <= 2.0 ** -24 * np.abs(wl)[some] + 4e-6).all() and (lp[~some] == -np.inf).all()


@pytest.mark.parametrize("op", ["top", "distill"])
def test_captured_calls_of_long_rows_replay(op):
    rng = np.random.default_rng(1)
    R, V, k = 2, 130000, 20
    xt = nr.Tensor((R, V), "f32")
    it = nr.Tensor.from_numpy(np.stack([rng.permutation(V)[:k] for _ in range(R)]).astype(np.int32))
    lt = nr.Tensor.from_numpy(np.full((R, k), -4.0, np.float32))
    ids, lp, st = nr.Tensor((R, k), "i32"), nr.Tensor((R, k), "f32"), nr.Tensor((R,), "u8")
    loss, stats = nr.Tensor((R,), "f32"), nr.Tensor((R, 5), "f64")

    def call():
        if op == "top":
            a = nr.NtRlTopArgs(xt.ptr, 0, 0, R, V, V, None, 0, 1.0, k, ids.ptr, lp.ptr, st.ptr)
            nr._check(nr.lib().nt_hip_rl_top_logprobs(C.byref(a)), "top")
        else:
            a = nr.NtRlDistillArgs(xt.ptr, 0, 0, R, V, V, None, 0, 1.0, k, it.ptr, lt.ptr, 0, 0, loss.ptr, stats.ptr, st.ptr)
            nr._check(nr.lib().nt_hip_rl_distill(C.byref(a)), "distill")

    call()
    nr.sync()
    caps = [Capture(), Capture()]
    for cap in caps:
        with cap:
            call()
    for i in range(4):
        x = rng.normal(0, 1, (R, V)).astype(np.float32)
        nr._check(nr.lib().nt_hip_upload(C.c_void_p(xt.ptr), x.ctypes.data_as(C.c_void_p), xt.nbytes), "upload")
        e = nr.Tensor.from_numpy(x)
        want = nr.top_logprobs(e, k) if op == "top" else nr.distill_with_stats(e, it, lt)[:1]
        caps[i % 2].replay()
        nr.top_logprobs(e, k)
        nr.sync()
        for got, w in zip((ids, lp) if op == "top" else (loss,), want):
            assert got.to_numpy().tobytes() == w.to_numpy().tobytes()
    for cap in caps:
        cap.close()


def test_offsets_past_32_bits():
    """70000 rows of 65536 bf16 columns, 4.6e9 of them: zeros but for the last two rows."""
    R, V, k = 70000, 65536, 3
    rng = np.random.default_rng(2)
    L = nr.lib()
    x, grad = nr.Tensor((R, V), "bf16"), nr.Tensor((R, V), "bf16")
    nr._check(L.nt_hip_memset(C.c_void_p(x.ptr), 0, x.nbytes), "memset")
    tail = ref.rounded(rng.normal(0, 2, (2, V)), "bf16")
    bits = ref.bits_of(tail, "bf16")
    nr._check(L.nt_hip_upload(C.c_void_p(x.ptr + (R - 2) * V * 2), bits.ctypes.data_as(C.c_void_p), bits.nbytes), "upload")
    ids, lp = (t.to_numpy() for t in nr.top_logprobs(x, k))
    assert (ids[:-2] == np.arange(k)).all() and (np.abs(lp[:-2] + np.log(V)) <= 2.0 ** -24 * 12 + 4e-6).all()
    wi, wl = ref.top(tail, tail, k)
    assert np.array_equal(ids[-2:], wi) and (np.abs(lp[-2:] - wl) <= 2.0 ** -24 * np.abs(wl) + 4e-6).all()
    it, lt = nr.Tensor.from_numpy(ids), nr.Tensor.from_numpy(np.full((R, k), -2.0, np.float32))
    loss, stats = nr.distill_with_stats(x, it, lt)
    g = nr.Tensor.from_numpy(np.ones(R, np.float32))
    a = nr.NtRlDistillGradArgs(x.ptr, nr.NT_BF16, 0, R, V, V, None, 0, 1.0, k, it.ptr, lt.ptr, stats.rows.ptr, g.ptr, grad.ptr,
                               nr.NT_BF16, 0, V)
    nr._check(L.nt_hip_rl_distill_backward(C.byref(a)), "backward")
    wl, wg, (q, listed, w, rest, q_off, mass, share) = ref.distill(tail, ids[-2:], np.full((2, k), -2.0, np.float32), "REST")
    assert (np.abs(loss.to_numpy()[-2:] - wl) <= 2.0 ** -24 * np.abs(wl) + 8e-6).all()
    out = np.empty((2, V), np.uint16)
    nr._check(L.nt_hip_download(out.ctypes.data_as(C.c_void_p), C.c_void_p(grad.ptr + (R - 2) * V * 2), out.nbytes), "download")
    got = (out.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    tol = np.where(listed, mass[:, None] * q * 8e-6 + 1e-12, (mass + share)[:, None] * q * 2.8e-5) * 1.01
    assert (np.abs(got - wg) <= tol + 2.0 ** -8 * np.abs(wg) + 2.0 ** -126).all()
    # sequences of one draft: the last one's rows are the last two
    S = R // 2
    u = np.full((S, 2), 0.37)
    tokens = np.zeros((S, 1), np.int32)
    got = nr.verify_drafted(nr.Tensor((S, 2, V), "bf16", x.buf), None, nr.Tensor.from_numpy(tokens), 1.0, None, None,
                            uniforms=nr.Tensor.from_numpy(u, "f64"))
    want = ref.verify(tail[None], None, tokens[-1:], u[-1:], [1], False)
    assert np.array_equal(got[0].to_numpy()[-1:], want[0]) and got[1].to_numpy()[-1] == want[1][0]
    assert (got[1].to_numpy()[:-1] == 0).all()
