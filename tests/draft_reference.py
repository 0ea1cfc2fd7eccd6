"""Plain f64 forms of the drafted tokens' verification, the top log-probabilities and the distillation, in numpy, and
the inputs that their tests share."""
import numpy as np

import noetic_rl as nr

HALF_ULP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # relative, of a rounding to nearest


def bits_of(x, dtype):
    """f64 values that the dtype holds exactly, as what Tensor.from_numpy takes."""
    x = np.asarray(x, np.float32)
    if dtype == "f32":
        return x
    if dtype == "f16":
        return x.astype(np.float16).view(np.uint16)
    return (x.view(np.uint32) >> 16).astype(np.uint16)


def rounded(x, dtype):
    """x as the dtype's values (bf16 by truncation), f64."""
    x = np.asarray(x, np.float32)
    if dtype == "f16":
        x = x.astype(np.float16)
    elif dtype == "bf16":
        x = (x.view(np.uint32) & 0xffff0000).view(np.float32)
    return x.astype(np.float64)


def tensor(x, dtype):
    return nr.Tensor.from_numpy(bits_of(x, dtype), dtype)


def values(t):
    return t.to_f64()


def make_mask(kind, rows, V, rng, keep=0.6, shared=False):
    """(the device tensor or None, what it adds to z as [rows, V], what excludes as bool [rows, V])."""
    if kind == "none":
        return None, np.zeros((rows, V)), np.zeros((rows, V), bool)
    n = 1 if shared else rows
    on = rng.random((n, V)) < keep
    on[:, rng.integers(0, V)] = True
    if kind == "u8":
        m = np.where(on, rng.integers(1, 256, on.shape), 0).astype(np.uint8)
        return nr.Tensor.from_numpy(m, "u8"), np.zeros((rows, V)), np.broadcast_to(~on, (rows, V))
    add = np.where(on, rng.normal(0, 0.5, on.shape), rng.choice([-np.inf, -1e9], on.shape)).astype(np.float32)
    return nr.Tensor.from_numpy(add), np.broadcast_to(add.astype(np.float64), (rows, V)), np.zeros((rows, V), bool)


def tempered(x, T, add, off):
    """z in f64, -inf where excluded."""
    return np.where(off, -np.inf, x / T + add)


def log_softmax(z):
    with np.errstate(invalid="ignore", divide="ignore"):
        m = z.max(-1, keepdims=True)
        return (z - m) - np.log(np.exp(z - m).sum(-1, keepdims=True))  # (in this order: m may be far larger)


def verify(z, zq, tokens, u, lengths, greedy):
    """z [S, K + 1, V], zq [S, K, V] or None, tokens [S, K] -> ids, accepted, logp."""
    S, K1, V = z.shape
    ids, acc, lp = np.full((S, K1), -1, np.int32), np.zeros(S, np.int32), np.zeros((S, K1))
    for s in range(S):
        a = 0
        while True:
            lnp = log_softmax(z[s, a])
            p = np.exp(lnp)
            if a == lengths[s]:
                r = p
            elif greedy:
                if int(np.argmax(z[s, a])) != tokens[s, a]:
                    r = p
                else:
                    r = None
            else:
                q = np.eye(1, V, tokens[s, a])[0] if zq is None else np.exp(log_softmax(zq[s, a]))
                r = None if u[s, a] * q[tokens[s, a]] < p[tokens[s, a]] else np.maximum(p - q, 0.0)
            if r is None:
                ids[s, a], lp[s, a] = tokens[s, a], lnp[tokens[s, a]]
                a += 1
                continue
            if greedy:
                t = int(np.argmax(z[s, a]))
            else:
                if not r.sum() > 0:
                    r = p
                c = np.cumsum(r)
                over = np.nonzero((c > u[s, -1] * c[-1]) & (r > 0))[0]
                t = int(over[0] if over.size else np.nonzero(r > 0)[0][-1])
            ids[s, a], lp[s, a], acc[s] = t, lnp[t], a
            break
    return ids, acc, lp


def top(key, z, k):
    """The first k of the stable descending sort by `key`, -1 and -inf past the allowed ones."""
    order = np.argsort(-key, axis=1, kind="stable")[:, :k]
    lnp = np.take_along_axis(log_softmax(z), order, 1)
    return np.where(np.take_along_axis(key, order, 1) > -np.inf, order, -1), lnp


def teacher_weights(logp, ids, tail):
    """(w [R, k], rest [R]) in f64; padding (-1) has none."""
    on = ids >= 0
    lw = np.where(on, logp.astype(np.float64), -np.inf)
    if tail == "RENORMALIZE":
        lw = log_softmax(lw)
    w = np.where(on, np.exp(lw), 0.0)  # (nothing listed: no weights, whatever the tail)
    rest = np.maximum(1.0 - w.sum(1), 0.0) if tail == "REST" else np.zeros(len(w))
    return w, rest


def distill(z, ids, logp, tail):
    """loss [R], d loss / d z [R, V], and (q, the listed columns, w, rest, q off the list) for tolerances."""
    R, V = z.shape
    w, rest = teacher_weights(logp, ids, tail)
    lnq = log_softmax(z)
    q = np.exp(lnq)
    listed = np.zeros((R, V + 1), bool)
    np.put_along_axis(listed, np.where(ids >= 0, ids, V), True, 1)
    listed = listed[:, :V]
    at = np.maximum(ids, 0)
    with np.errstate(invalid="ignore", divide="ignore"):
        terms = np.where(w > 0, w * (np.log(w) - np.take_along_axis(lnq, at, 1)), 0.0)
        q_off = np.where(listed, 0.0, q).sum(1)
        some = (rest > 0) & (q_off > 0)
        loss = terms.sum(1) + np.where(some, rest * np.log(rest / q_off), 0.0)
        share = np.where(some, rest / q_off, 0.0)
    mass = w.sum(1) + rest
    grad = q * (mass[:, None] - np.where(listed, 0.0, share[:, None]))
    dense = np.zeros((R, V + 1))
    np.put_along_axis(dense, np.where(ids >= 0, ids, V), w, 1)
    return loss, grad - dense[:, :V], (q, listed, w, rest, q_off, mass, share)
