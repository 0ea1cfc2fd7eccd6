"""Drafted tokens' verification (verify_drafted) against a plain f64 form of its definition.

Everything that decides a token is evaluated in f64, with exponentials within 2e-14: every id and count has to be equal (a
draw lies within 1e-13 of a token's border with a probability of about 1e-9 a test). A log-probability is a
difference of f64 values within 1e-12, rounded once: half an f32 step of its value and 1e-12. From 256 positions on, and
greedily, an accepted draft's (and the greedy token's) log-sum-exp is of f32 exponentials: within 6e-6 in log2 units, 4.2e-6
here, and of an additive mask's f32 sums within half a step of the largest, 2^-24 of it."""
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


def inputs(S, K, V, dtype, kind, T, rng, shared=False, draft=True, ragged=False, std=2.0):
    """A sequence's rows flat as (s, t); the mask [S, K + 1, V] or [1, 1, V]."""
    x = ref.rounded(rng.normal(0, std, (S, K + 1, V)), dtype)
    y = ref.rounded(x[:, :K] + rng.normal(0, 0.5, (S, K, V)), dtype) if draft else None
    mt, add, off = ref.make_mask(kind, S * (K + 1), V, rng, shared=shared)
    add, off = add.reshape(S, K + 1, V), off.reshape(S, K + 1, V)
    if mt is not None:
        mt = nr.Tensor((1, 1, V) if shared else (S, K + 1, V), mt.dtype, mt.buf)
    z = ref.tempered(x, T or 1.0, add, off)
    zq = ref.tempered(y, T or 1.0, add[:, :K], off[:, :K]) if draft else None
    near = (zq if draft else z[:, :K]) + rng.gumbel(size=(S, K, V)) * (0.3 if T == 0.0 else 1.0)
    tokens = np.argmax(near, 2).astype(np.int32).reshape(S, K)
    lengths = rng.integers(0, K + 1, S).astype(np.int32) if ragged else np.full(S, K, np.int32)
    return x, y, z, zq, mt, tokens, rng.random((S, K + 1)), lengths


def run(x, y, mt, tokens, u, lengths, dtype, T, **kw):
    return nr.verify_drafted(ref.tensor(x, dtype), None if y is None else ref.tensor(y, dtype), nr.Tensor.from_numpy(tokens),
                             T, mt, None, uniforms=nr.Tensor.from_numpy(u, "f64"),
                             lengths=None if lengths is None else nr.Tensor.from_numpy(lengths), **kw)


def compare(got, want, greedy=False, largest=0.0):
    ids, acc, lp = (t.to_numpy() for t in got)
    wi, wa, wl = want
    assert np.array_equal(acc, wa)
    assert np.array_equal(ids, wi)
    f32 = np.full(wl.shape, greedy or wl.size >= 256)
    if not greedy:
        f32[np.arange(len(wl)), wa] = False
    assert (np.abs(lp - wl) <= 2.0 ** -24 * np.abs(wl) + np.where(f32, 4.2e-6 + 2.0 ** -24 * largest, 1e-12)).all()


CASES = [
    # (S, K, V, dtype, mask, shared, T, draft logits, lengths of their own)
    (1, 4, 32000, "bf16", "none", False, 0.8, True, False),
    (3, 1, 1, "f32", "none", False, 1.0, True, False),         # one token
    (5, 2, 7, "f32", "u8", False, 0.7, True, True),
    (4, 3, 511, "bf16", "f32", False, 1.3, True, True),
    (4, 3, 512, "f16", "u8", True, 1.0, True, False),
    (4, 3, 513, "f16", "f32", True, 0.9, False, True),         # certain drafts
    (40, 8, 5003, "bf16", "none", False, 0.7, True, False),    # 360 positions: one workgroup each
    (300, 2, 4096, "f16", "u8", False, 0.6, True, True),
    (70, 5, 9001, "f32", "f32", False, 1.0, True, True),
    (64, 7, 8192, "f32", "none", False, 1.0, False, True),
    (2, 7, 128256, "bf16", "u8", False, 0.7, True, False),
    (9, 0, 3001, "f32", "none", False, 0.9, True, False),      # no drafts: a sampler
    (2, 20, 1500, "f32", "none", False, 1.0, True, True),
    (1, 127, 600, "bf16", "none", False, 1.0, True, False),
    (33, 3, 5000, "f16", "f32", True, 0.0, False, True),       # greedy
    (1, 6, 50257, "bf16", "u8", False, 0.0, True, False),
    (90, 3, 1003, "f32", "none", False, 0.0, False, True),
]


@pytest.mark.parametrize("case", CASES)
def test_against_the_definition(case):
    S, K, V, dtype, kind, shared, T, draft, ragged = case
    rng = np.random.default_rng(S * 1000 + K * 10 + V)
    x, y, z, zq, mt, tokens, u, lengths = inputs(S, K, V, dtype, kind, T, rng, shared, draft and K > 0, ragged)
    want = ref.verify(z, zq, tokens, u, lengths, T == 0.0)
    got = run(x, y, mt, tokens, u, lengths if ragged else None, dtype, T)
    compare(got, want, T == 0.0, np.abs(z.max()) if kind == "f32" else 0.0)
    again = run(x, y, mt, tokens, u, lengths if ragged else None, dtype, T)
    for a, b in zip(got, again):
        assert a.to_numpy().tobytes() == b.to_numpy().tobytes()


def test_ends_of_the_range_are_taken():
    """Both ends happen at these sizes: all drafts accepted, and the first refused."""
    rng = np.random.default_rng(5)
    x, y, z, zq, mt, tokens, u, lengths = inputs(300, 3, 1000, "f32", "none", 1.0, rng)
    acc = ref.verify(z, zq, tokens, u, lengths, False)[1]
    assert {0, 1, 2, 3} == set(acc.tolist())
    compare(run(x, y, mt, tokens, u, None, "f32", 1.0), ref.verify(z, zq, tokens, u, lengths, False))


def test_a_drafters_own_temperature_and_equal_logits():
    rng = np.random.default_rng(6)
    S, K, V = 6, 4, 2000
    x, y, z, zq, mt, tokens, u, lengths = inputs(S, K, V, "f32", "none", 0.7, rng)
    want = ref.verify(z, y / 1.1, tokens, u, lengths, False)
    compare(run(x, y, mt, tokens, u, None, "f32", 0.7, draft_temperature=1.1), want)
    # p = q everywhere: every draft is accepted, whatever u below 1
    u[:] = 1.0 - 2.0 ** -53
    ids, acc, _ = run(x, x[:, :K].copy(), mt, tokens, u, None, "f32", 0.7)
    assert (acc.to_numpy() == K).all() and np.array_equal(ids.to_numpy()[:, :K], tokens)
    # u rounded to 1: refused, and nothing of p is above q, so that p itself is drawn from (its last token)
    u[:] = 1.0
    ids, acc, lp = (t.to_numpy() for t in run(x, x[:, :K].copy(), mt, tokens, u, None, "f32", 0.7))
    assert (acc == 0).all() and (ids[:, 0] == V - 1).all() and (ids[:, 1:] == -1).all() and (lp[:, 1:] == 0).all()


def test_the_drawn_tokens_are_distributed_as_the_targets():
    """20000 sequences of one draft over 8 tokens: the first token's counts are the target's, within five standard
    deviations (5.7e-7 each, two-sided)."""
    rng = np.random.default_rng(7)
    S, V = 20000, 8
    x = np.broadcast_to(rng.normal(0, 1, V).astype(np.float32), (S, 2, V)).copy()
    y = np.broadcast_to(rng.normal(0, 1, V).astype(np.float32), (S, 1, V)).copy()
    q = np.exp(ref.log_softmax(y[0, 0].astype(np.float64)))
    tokens = rng.choice(V, (S, 1), p=q / q.sum()).astype(np.int32)
    ids, _, _ = run(x, y, None, tokens, rng.random((S, 2)), None, "f32", 1.0)
    p = np.exp(ref.log_softmax(x[0, 0].astype(np.float64)))
    n = np.bincount(ids.to_numpy()[:, 0], minlength=V)
    assert (np.abs(n - S * p) <= 5 * np.sqrt(S * p * (1 - p))).all()


def test_far_logits_and_masks_of_the_lowest_value():
    """Logits thousands apart (a reference moves), -inf logits, an additive mask of f32's lowest value."""
    rng = np.random.default_rng(8)
    S, K, V = 5, 2, 3000
    x = rng.normal(0, 1, (S, K + 1, V)).astype(np.float32)
    x[:, :, 1500:] += 3000.0
    x[:, :, 2900] = 20000.0
    x[:, :, 2901] = 19999.5
    x[:, :, ::7] = -np.inf
    y = x[:, :K].copy()
    y[:, :, 2901] += 0.25
    add = np.zeros((1, 1, V), np.float32)
    add[..., 10:20] = np.finfo(np.float32).min
    z, zq = x.astype(np.float64) + add, y.astype(np.float64) + add
    tokens = np.where(rng.random((S, K)) < 0.5, 2900, 2901).astype(np.int32)
    u = rng.random((S, K + 1))
    want = ref.verify(z, zq, tokens, u, np.full(S, K), False)
    compare(run(x, y, nr.Tensor.from_numpy(add), tokens, u, None, "f32", 1.0), want)


@pytest.mark.parametrize("S", [4, 150])  # several workgroups a position, and one
@pytest.mark.parametrize("value", [-1e9, -1e13, float(np.finfo(np.float32).min)])
def test_masks_that_lower_every_token(S, value):
    """A row whose mask leaves nothing but lowers all by one value: what f64 keeps of the logits beside it decides."""
    rng = np.random.default_rng(12)
    K, V = 2, 1100
    x = rng.normal(0, 2, (S, K + 1, V)).astype(np.float32)
    y = (x[:, :K] + rng.normal(0, 0.5, (S, K, V))).astype(np.float32)
    add = np.full((1, 1, V), value, np.float32)
    z, zq = x.astype(np.float64) + add, y.astype(np.float64) + add
    tokens = np.argmax(zq + rng.gumbel(size=zq.shape), 2).astype(np.int32)
    u = rng.random((S, K + 1))
    want = ref.verify(z, zq, tokens, u, np.full(S, K), False)
    ids, acc, lp = (t.to_numpy() for t in run(x, y, nr.Tensor.from_numpy(add), tokens, u, None, "f32", 1.0))
    assert np.array_equal(ids, want[0]) and np.array_equal(acc, want[1])
    at = np.arange(S), acc
    assert (np.abs(lp - want[2])[at] <= 2.0 ** -24 * np.abs(want[2])[at] + 1e-12).all()


def raw(x, y, tokens, u, dtype="f32", T=1.0, lengths=None, mt=None, S=None, K=None, V=None):
    """A direct call with every output larger by a row, filled beforehand; (rc, ids, accepted, logp, status)."""
    S1, K1, V1 = x.shape
    S, K, V = S or S1, K1 - 1 if K is None else K, V or V1
    xt, yt = ref.tensor(x, dtype), None if y is None else ref.tensor(y, dtype)
    tt, ut = nr.Tensor.from_numpy(tokens), nr.Tensor.from_numpy(u, "f64")
    lt = None if lengths is None else nr.Tensor.from_numpy(lengths)
    ids = nr.Tensor.from_numpy(np.full((S + 1, K + 1), 77, np.int32))
    acc = nr.Tensor.from_numpy(np.full(S + 1, 77, np.int32))
    lp = nr.Tensor.from_numpy(np.full((S + 1, K + 1), 77, np.float32))
    st = nr.Tensor.from_numpy(np.full(S + 1, 77, np.uint8), "u8")
    a = nr.NtRlVerifyArgs(xt.ptr, None if yt is None else yt.ptr, nr._dtype_code(xt), 0, S, K, V, V1, V1, None, 0, T, T, tt.ptr,
                          None if lt is None else lt.ptr, ut.ptr, ids.ptr, acc.ptr, lp.ptr, st.ptr)
    rc = nr.lib().nt_hip_rl_verify_drafted(C.byref(a))
    return (rc,) + tuple(t.to_numpy() for t in (ids, acc, lp, st))


@pytest.mark.parametrize("S", [6, 200])  # several workgroups a position, and one
def test_refused_rows_matter_only_where_they_are_reached(S):
    rng = np.random.default_rng(9)
    K, V = 3, 1500
    x = rng.normal(0, 1, (S, K + 1, V)).astype(np.float32)
    y = x[:, :K].copy()
    tokens = rng.integers(0, V, (S, K)).astype(np.int32)
    u = np.full((S, K + 1), 0.5)        # equal p and q: everything is accepted
    lengths = np.full(S, K, np.int32)
    x[0, 2, 5] = np.nan                 # 0: the target's row 2
    x[1, 3] = -np.inf                   # 1: nothing allowed at the end
    y[2, 1, 9] = np.nan                 # 2: the drafter's row 1
    y[3, 0] = -np.inf                   # 3: the drafter's row 0
    tokens[4, 1] = V                    # 4: no such token
    lengths[5] = K + 1                  # 5: no such length
    rc, ids, acc, lp, st = raw(x, y, tokens, u, lengths=lengths)
    assert rc == 0
    assert acc[:6].tolist() == [2, 3, 1, 0, 1, 0]
    assert st[:6].tolist() == [2, 1, 2, 1, 3, 3]
    for s, a in enumerate(acc[:6]):
        good = min(a, 3)
        assert np.array_equal(ids[s, :good], tokens[s, :good]) and (ids[s, good:] == -1).all()
        assert np.isfinite(lp[s, :good]).all() and np.isnan(lp[s, good]) and (lp[s, good + 1:] == 0).all()
    assert (st[6:S] == 0).all() and (acc[6:S] == K).all()
    # rows behind the last sequence are left as they were
    assert (ids[S] == 77).all() and acc[S] == 77 and (lp[S] == 77).all() and st[S] == 77
    # the same rows behind a refusal do not matter
    u[:, 0] = 0.999999
    y2 = y.copy()
    y2[np.arange(S), 0, tokens[:, 0] % V] = 30.0
    y2[3, 0] = 0.0
    y2[3, 0, tokens[3, 0]] = 30.0
    lengths[5] = K
    rc, ids, acc, lp, st = raw(x, y2, tokens, u, lengths=lengths)
    assert rc == 0 and (acc[:S] == 0).all() and (st[:S] == 0).all() and (ids[:S, 0] >= 0).all() and (ids[:S, 1:] == -1).all()
    with pytest.raises(ValueError, match="sequence 0 has a position with no allowed token"):
        run(x, y, None, np.minimum(tokens, V - 1), np.full((S, K + 1), 0.5), None, "f32", 1.0)
    with pytest.raises(IndexError, match="sequence 4"):
        run(np.nan_to_num(x, neginf=0.0), np.nan_to_num(y, neginf=0.0), None, tokens, np.full((S, K + 1), 0.5), None, "f32", 1.0)


def test_rows_with_strides_and_no_sequences():
    rng = np.random.default_rng(10)
    S, K, V = 4, 2, 1001
    x, y = rng.normal(0, 1, (S, K + 1, V + 23)).astype(np.float32), rng.normal(0, 1, (S, K, V + 23)).astype(np.float32)
    tokens, u = rng.integers(0, V, (S, K)).astype(np.int32), rng.random((S, K + 1))
    rc, ids, acc, lp, st = raw(x, y, tokens, u, V=V)
    wi, wa, wl = ref.verify(x[..., :V].astype(np.float64), y[..., :V].astype(np.float64), tokens, u, np.full(S, K), False)
    assert rc == 0 and np.array_equal(ids[:S], wi) and np.array_equal(acc[:S], wa)
    ids, acc, lp = nr.verify_drafted(nr.Tensor((0, 3, 9), "f32"), None, nr.Tensor((0, 2), "i32"), 1.0, None, None,
                                     uniforms=nr.Tensor((0, 3), "f64"))
    assert ids.shape == (0, 3) and acc.shape == (0,)


def test_a_stream_gives_the_uniforms():
    rng = np.random.default_rng(11)
    x, y, z, zq, mt, tokens, u, lengths = inputs(3, 2, 500, "f32", "none", 1.0, rng)
    r = nr.Rng(3, "drafts")
    same = r.clone()
    got = nr.verify_drafted(ref.tensor(x, "f32"), ref.tensor(y, "f32"), nr.Tensor.from_numpy(tokens), 1.0, None, r)
    compare(got, ref.verify(z, zq, tokens, same.uniforms(9).reshape(3, 3), lengths, False))
    assert r.next_u64() == same.next_u64()


@pytest.mark.parametrize("S", [3, 200])
def test_captured_calls_replay(S):
    """Two graphs of the call and eager ones between their replays, on new inputs each time."""
    rng = np.random.default_rng(12)
    K, V = 2, 1200
    shapes = [((S, K + 1, V), "f32"), ((S, K, V), "f32"), ((S, K), "i32"), ((S, K + 1), "f64")]
    ins = [nr.Tensor(s, d) for s, d in shapes]
    outs = [[nr.Tensor((S, K + 1), "i32"), nr.Tensor((S,), "i32"), nr.Tensor((S, K + 1), "f32"), nr.Tensor((S,), "u8")] for _ in range(2)]

    def call(o):
        a = nr.NtRlVerifyArgs(ins[0].ptr, ins[1].ptr, 0, 0, S, K, V, V, V, None, 0, 1.0, 1.0, ins[2].ptr, None, ins[3].ptr,
                              o[0].ptr, o[1].ptr, o[2].ptr, o[3].ptr)
        nr._check(nr.lib().nt_hip_rl_verify_drafted(C.byref(a)), "verify")

    call(outs[0])
    nr.sync()
    caps = [Capture(), Capture()]
    for cap, o in zip(caps, outs):
        with cap:
            call(o)
    for i in range(4):
        x, y, z, zq, mt, tokens, u, lengths = inputs(S, K, V, "f32", "none", 1.0, rng)
        for t, v in zip(ins, (x.astype(np.float32), y.astype(np.float32), tokens, u)):
            v = np.ascontiguousarray(v)
            nr._check(nr.lib().nt_hip_upload(C.c_void_p(t.ptr), v.ctypes.data_as(C.c_void_p), t.nbytes), "upload")
        want = run(x, y, None, tokens, u, None, "f32", 1.0)
        caps[i % 2].replay()
        run(x, y, None, tokens, u, None, "f32", 1.0)
        nr.sync()
        for a, b in zip(outs[i % 2], want):
            assert a.to_numpy().tobytes() == b.to_numpy().tobytes()
    for cap in caps:
        cap.close()
