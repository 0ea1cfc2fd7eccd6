"""Speculative decoding and the distillation of its drafter: what their operators are measured on.

  verify      noetic_rl.verify_drafted: a drafter's tokens against the target's distribution at each position,
              from given uniforms: how many are accepted, the token drawn in place of the first one refused
              (or after the last), and the target's log-probabilities of what is kept.
  top         noetic_rl.top_logprobs: each row's k most likely tokens and their log-probabilities, what a
              teacher records.
  distill     noetic_rl.distill_with_stats: the divergence of a student's row from a teacher's recorded ones.
  train       the same followed by noetic_rl.distill_grad: its gradient with respect to the student's logits.

With z = x / T (+ mask; a token whose u8 mask is 0 is excluded), p = softmax(z) of the target and q of the
drafter under the same mask: the token x drafted at position t is accepted where u_t q(x) < p(x). At the first
position a that is not (or at the sequence's number of drafts, where q counts as 0), the token is
min {v : sum_{j <= v} r_j > u_K sum r}, r = max(p - q, 0). A drafter that gives no logits is certain: q is 1 at
its token. T = 0 is greedy: a token is accepted where it is the first largest.

A row's top tokens are ordered by z, ties to the lowest index; their log-probabilities are ln p.

With teacher weights w_j at tokens i_j, w = exp(teacher's log-probability): tail "rest" lumps what the list
leaves, r = 1 - sum w, into one outcome: loss = sum w (ln w - ln q_i) + r (ln r - ln sum_{v not listed} q_v);
"drop" leaves r out; "renormalize" divides w by its sum first.
"""
import math
import os
import sys

import torch

own = False

_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_ACCEPTED = 0.78  # how often a drafted token of these inputs is accepted


def listed():
    return [
        # one sequence's drafts of a small model: the latency of a decode step with a drafter
        {"name": "verify_step", "op": "verify", "seqs": 1, "drafts": 4, "vocab": 32000, "dtype": "bf16", "mask": "none",
         "temperature": 0.8, "lookup": False, "ragged": False},
        # a constrained decode batch: a grammar's keep-mask at every position
        {"name": "verify_masked", "op": "verify", "seqs": 64, "drafts": 5, "vocab": 128256, "dtype": "bf16", "mask": "u8",
         "temperature": 0.7, "lookup": False, "ragged": False},
        # a rollout's decode batch at the benchmark's rows and vocabulary
        {"name": "verify_batch", "op": "verify", "seqs": 256, "drafts": 7, "vocab": 128256, "dtype": "bf16",
         "mask": "none", "temperature": 0.7, "lookup": False, "ragged": False},
        # drafts looked up in the prompt (certain, of any number), f16, odd sizes, one additive mask
        {"name": "verify_lookup", "op": "verify", "seqs": 33, "drafts": 3, "vocab": 50257, "dtype": "f16",
         "mask": "f32_shared", "temperature": 0.8, "lookup": True, "ragged": True},
        # a served token's alternatives
        {"name": "top_token", "op": "top", "rows": 1, "vocab": 128256, "dtype": "bf16", "mask": "none",
         "temperature": 1.0, "k": 20},
        # a teacher's record of 4096 positions
        {"name": "top_rollout", "op": "top", "rows": 4096, "vocab": 50304, "dtype": "bf16", "mask": "none",
         "temperature": 1.0, "k": 64},
        # f32 logits of the largest vocabulary under a keep-mask, a long record
        {"name": "top_masked", "op": "top", "rows": 1024, "vocab": 151936, "dtype": "f32", "mask": "u8",
         "temperature": 1.0, "k": 128},
        # odd sizes, f16, one additive mask
        {"name": "top_odd", "op": "top", "rows": 333, "vocab": 50257, "dtype": "f16", "mask": "f32_shared",
         "temperature": 0.7, "k": 50},
        # the divergence over a held-out rollout, no gradient
        {"name": "distill_eval", "op": "distill", "rows": 4096, "vocab": 50304, "dtype": "bf16", "mask": "none",
         "temperature": 1.0, "k": 64, "tail": "rest"},
        # one micro-batch of a small drafter
        {"name": "train_small", "op": "train", "rows": 128, "vocab": 32000, "dtype": "bf16", "mask": "none",
         "temperature": 1.0, "k": 16, "tail": "rest"},
        # a training step of a drafter that shares the target's vocabulary
        {"name": "train_large", "op": "train", "rows": 4096, "vocab": 128256, "dtype": "bf16", "mask": "none",
         "temperature": 1.0, "k": 64, "tail": "rest"},
        # odd sizes, f16, softened, a keep-mask row for each position
        {"name": "train_odd", "op": "train", "rows": 333, "vocab": 50257, "dtype": "f16", "mask": "u8",
         "temperature": 2.0, "k": 50, "tail": "renormalize"},
    ]


def _size(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["verify", "verify", "verify", "top", "top", "distill", "train", "train"])
    vocab = rng.choice([32000, 50304, 128256, 151936]) if rng.random() < 0.3 else _size(rng, 1000, 152000)
    vocab = max(vocab // 8, 1) * 8 if rng.random() < 0.4 else vocab
    case = {"op": op, "vocab": vocab, "dtype": rng.choice(["f32", "bf16", "bf16", "f16"]),
            "mask": rng.choice(["none", "none", "u8", "f32_shared"])}
    elements = 400_000_000 // _SIZE[case["dtype"]] // vocab  # rows of the largest drawn case
    if op == "verify":
        drafts = rng.choice([1, 2, 3, 4, 5, 7, 8])
        return dict(case, seqs=_size(rng, 1, min(256, elements // (2 * drafts + 1))), drafts=drafts,
                    temperature=rng.choice([0.0, 0.6, 0.7, 0.8, 1.0]), lookup=rng.random() < 0.2,
                    ragged=rng.random() < 0.4)
    case.update(temperature=rng.choice([0.7, 1.0, 1.0, 2.0]), k=_size(rng, 1, 256))
    case["rows"] = _size(rng, 1, min(8192, elements))
    if op != "top":
        case["tail"] = rng.choice(["rest", "rest", "drop", "renormalize"])
    return case


# ------------------------------------------------------------------------------------- inputs

def _normal(shape, dtype, g, std):
    return torch.empty(shape, dtype=_TORCH[dtype], device="cuda").normal_(0.0, std, generator=g)


def _near(x, g, std):
    """x and noise, in x's type."""
    return torch.empty(x.shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=g).add_(x).to(x.dtype)


def _mask(case, rows, g):
    if case["mask"] == "none":
        return None
    n, V = (rows, case["vocab"]) if case["mask"] == "u8" else (1, case["vocab"])
    keep = torch.empty((n, V), dtype=torch.bool, device="cuda").bernoulli_(0.3 if case["op"] == "verify" else 0.9, generator=g)
    keep[:, V // 2] = True
    return keep.to(torch.uint8) if case["mask"] == "u8" else torch.where(keep, 0.0, -math.inf)


def _masked(z, mask):
    """z under a u8 keep-mask or an additive one, its rows or one row for all."""
    if mask is None:
        return z
    mask = mask.view(z.shape if mask.shape[0] > 1 or z.numel() == mask.numel() else (1,) * (z.dim() - 1) + (-1,))
    return z.masked_fill(mask == 0, -math.inf) if mask.dtype == torch.uint8 else z + mask


def _inputs(case, seed):
    """Every input as torch tensors, a function of the case and the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    V = case["vocab"]
    if case["op"] == "verify":
        S, K = case["seqs"], case["drafts"]
        x = {"logits": _normal((S, K + 1, V), case["dtype"], g, 2.0), "draft": None,
             "uniforms": torch.rand((S, K + 1), dtype=torch.float64, device="cuda", generator=g).clamp_(min=1e-16),
             "mask": _mask(case, S * (K + 1), g)}
        x["lengths"] = torch.randint(0, K + 1, (S,), device="cuda", generator=g, dtype=torch.int32) if case["ragged"] else None
        if case["lookup"]:  # a likely continuation: one token of each row stands out
            at = torch.randint(0, V, (S, K + 1, 1), device="cuda", generator=g)
            x["logits"].scatter_add_(2, at, torch.full_like(at, 13, dtype=x["logits"].dtype))
            z = _masked(x["logits"].float(), x["mask"])[:, :K]
        else:  # the drafter's own sample
            x["draft"] = _near(x["logits"][:, :K], g, 0.4)
            mask = x["mask"]
            if mask is not None and mask.shape[0] > 1:
                mask = mask.view(S, K + 1, V)[:, :K].reshape(S * K, V)
            z = _masked(x["draft"].float() / (case["temperature"] or 1.0), mask)
            if case["temperature"]:
                z -= torch.empty_like(z).exponential_(generator=g).log_()
        x["tokens"] = z.argmax(2).to(torch.int32)
        return x
    R, k = case["rows"], case["k"]
    x = {"logits": _normal((R, V), case["dtype"], g, 2.0), "mask": _mask(case, R, g)}
    if case["op"] == "top":
        return x
    # the teacher's record under the student's temperature and mask
    lnp = torch.log_softmax(_masked(_near(x["logits"], g, 0.4).float() / case["temperature"], x["mask"]), 1)
    x["teacher_logp"], ids = lnp.topk(k, 1)
    x["ids"] = torch.where(x["teacher_logp"] > -math.inf, ids, -1).to(torch.int32)
    if case["op"] == "train":  # a mean over the positions, f16 gradients under a loss scale; one in 16 is padding
        x["g_loss"] = torch.full((R,), (4096.0 if case["dtype"] == "f16" else 1.0) / R, device="cuda")
        x["g_loss"][torch.rand(R, device="cuda", generator=g) < 1 / 16] = 0.0
    return x


def prepare(case, seed):
    return dict(_inputs(case, seed), case=case)


# ------------------------------------------------------------------------------------- the plain forms

def _first_largest(z):
    """The first index of each row's maximum."""
    return (z == z.amax(-1, keepdim=True)).to(torch.uint8).argmax(-1)


def _softmax_parts(z):
    """exp(z - lse) and the log-sum-exp."""
    base = z.amax(-1, keepdim=True)
    w = (z - base).exp_()
    total = w.sum(-1, keepdim=True)
    return w.div_(total), (base + total.log())[..., 0]


def _plain_verify(s):
    # (in 64 bits: a token is the one whose share of the unit interval holds u)
    case, K = s["case"], s["case"]["drafts"]
    T = case["temperature"] or 1.0
    z = _masked(s["logits"].double().div_(T), s["mask"])
    p, lse = _softmax_parts(z)
    at = s["tokens"].long()
    steps = torch.arange(K + 1, device="cuda")
    length = torch.full((case["seqs"],), K, device="cuda") if s["lengths"] is None else s["lengths"].long()
    n = torch.arange(case["seqs"], device="cuda")
    if case["temperature"] == 0.0:
        ok = _first_largest(z[:, :K]) == at
    else:
        p_at = p[:, :K].gather(2, at[:, :, None])[:, :, 0]
        if s["draft"] is None:
            q_at = torch.ones_like(p_at)
        else:
            mask = s["mask"]
            if mask is not None and mask.shape[0] > 1:
                mask = mask.view(z.shape)[:, :K].reshape(-1, case["vocab"])
            q, _ = _softmax_parts(_masked(s["draft"].double().div_(T), mask))
            q_at = q.gather(2, at[:, :, None])[:, :, 0]
        ok = s["uniforms"][:, :K] * q_at < p_at
    accepted = (ok & (steps[:K] < length[:, None])).long().cumprod(1).sum(1)
    here = p[n, accepted]
    if case["temperature"] == 0.0:
        drawn = _first_largest(z[n, accepted])
    else:
        refused = (accepted < length)[:, None]
        t = accepted.clamp(max=K - 1)
        if s["draft"] is None:
            other = torch.zeros_like(here).scatter_(1, at[n, t][:, None], 1.0)
        else:
            other = q[n, t]
        r = torch.where(refused, (here - other).clamp_(min=0.0), here)
        r = torch.where(r.sum(1, keepdim=True) > 0, r, here)
        last = case["vocab"] - 1 - (r > 0).flip(1).to(torch.uint8).argmax(1)
        run = r.cumsum(1)
        drawn = torch.minimum((run <= s["uniforms"][:, K:] * run[:, -1:]).sum(1), last)
    ids = torch.where(steps < accepted[:, None], torch.nn.functional.pad(at, (0, 1)), -1)
    ids[n, accepted] = drawn
    logp = z.gather(2, ids.clamp(min=0)[:, :, None])[:, :, 0] - lse
    return {"ids": ids.to(torch.int32), "accepted": accepted.to(torch.int32),
            "logp": torch.where(ids >= 0, logp, 0.0).float()}


def _tempered(s):
    # (the quotient rounded as IEEE division rounds it: tokens are ordered by it)
    T = torch.full((), s["case"]["temperature"], device="cuda")
    return _masked(s["logits"].float() / T, s["mask"])


def _plain_top(s):
    k = s["case"]["k"]
    z = _tempered(s)
    _, lse = _softmax_parts(z.double())
    # by the logits themselves where no mask is added: a quotient can make two of them one
    key = z if s["case"]["mask"] == "f32_shared" else _masked(s["logits"].float(), s["mask"])
    ids = key.sort(dim=1, descending=True, stable=True)[1][:, :k]
    logp = (z.gather(1, ids).double() - lse[:, None]).float()
    return {"ids": torch.where(logp > -math.inf, ids, -1).to(torch.int32), "logp": logp}


def _weights(s):
    """(the teacher's weight at each listed token, what the list leaves, their sum) in 64 bits."""
    w = s["teacher_logp"].double()
    tail = s["case"]["tail"]
    if tail == "renormalize":
        w = _softmax_parts(w)[0]
    else:
        w = w.exp()
    rest = (1.0 - w.sum(1)).clamp_(min=0.0) if tail == "rest" else torch.zeros_like(w[:, 0])
    return w, rest, w.sum(1) + rest


def _distill(s):
    # (in 64 bits: a divergence is a small difference of large sums)
    z = _masked(s["logits"].double().div_(s["case"]["temperature"]), s["mask"])
    q, lse = _softmax_parts(z)
    listed_ = s["ids"] >= 0
    at = s["ids"].long().clamp(min=0)
    w, rest, mass = _weights(s)
    lnq = z.gather(1, at) - lse[:, None]
    loss = torch.where(listed_ & (w > 0), w * (w.log() - lnq), 0.0).sum(1)
    # each row's listed columns; a column more takes what is not listed there
    seen = torch.zeros((z.shape[0], z.shape[1] + 1), dtype=torch.bool, device="cuda")
    seen = seen.scatter_(1, torch.where(listed_, at, z.shape[1]), True)[:, :-1]
    q_rest = q.masked_fill(seen, 0.0).sum(1)
    loss += torch.where((rest > 0) & (q_rest > 0), rest * (rest.log() - q_rest.log()), 0.0)
    return {"loss": loss.float()}, (q, seen, at, listed_, w, rest, mass, q_rest)


def _train(s):
    out, (q, seen, at, listed_, w, rest, mass, q_rest) = _distill(s)
    scale = s["g_loss"].double() / s["case"]["temperature"]
    share = torch.where(q_rest > 0, rest / q_rest, 0.0)
    grad = q * (scale * mass)[:, None] - q.masked_fill(seen, 0.0).mul_((scale * share)[:, None])
    grad.scatter_add_(1, at, torch.where(listed_, -scale[:, None] * w, 0.0))
    return dict(out, grad=grad.to(s["logits"].dtype))


# ------------------------------------------------------------------------------------- the framework's operators

class _Held:
    """A torch allocation as the buffer behind a noetic_rl.Tensor."""

    def __init__(self, t):
        self.t, self.ptr = t, t.data_ptr()


class _Export:
    def __init__(self, t):
        self.owner = t
        kind = {"f32": "<f4", "bf16": "<i2", "f16": "<f2", "i32": "<i4"}[t.dtype]
        self.__cuda_array_interface__ = {"shape": t.shape, "typestr": kind, "data": (t.ptr, False), "version": 2}


_NAMES = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16", torch.uint8: "u8", torch.int32: "i32",
          torch.float64: "f64"}


def _framework():
    at = os.path.join(os.getcwd(), "noetic-tensor_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import noetic_rl
    return noetic_rl


def _given(nr, t, shape=None):
    """A contiguous torch tensor as the library's device tensor, in place."""
    return None if t is None else nr.Tensor(tuple(shape or t.shape), _NAMES[t.dtype], _Held(t))


def _taken(t):
    """The library's device tensor as a torch tensor over the same memory (kept alive by it)."""
    x = torch.as_tensor(_Export(t), device="cuda")
    return x.view(torch.bfloat16) if t.dtype == "bf16" else x


def _own_verify(s):
    nr, case = _framework(), s["case"]
    mask = s["mask"]
    if mask is not None:
        mask = _given(nr, mask, s["logits"].shape if mask.shape[0] > 1 else (1, 1, case["vocab"]))
    ids, accepted, logp = nr.verify_drafted(
        _given(nr, s["logits"]), _given(nr, s["draft"]), _given(nr, s["tokens"]), case["temperature"], mask, None,
        uniforms=_given(nr, s["uniforms"]), lengths=_given(nr, s["lengths"]), check=False)
    return {"ids": _taken(ids), "accepted": _taken(accepted), "logp": _taken(logp)}


def _own_tempered(nr, s):
    return nr.Tempered(_given(nr, s["logits"]), s["case"]["temperature"], _given(nr, s["mask"]))


def _own_top(s):
    nr = _framework()
    ids, logp = nr.top_logprobs(_own_tempered(nr, s), s["case"]["k"], check=False)
    return {"ids": _taken(ids), "logp": _taken(logp)}


def _own_distill(s):
    nr = _framework()
    logits, ids, teacher = _own_tempered(nr, s), _given(nr, s["ids"]), _given(nr, s["teacher_logp"])
    tail = nr.TeacherTail[s["case"]["tail"].upper()]
    loss, stats = nr.distill_with_stats(logits, ids, teacher, tail, check=False)
    out = {"loss": _taken(loss)}
    if s["case"]["op"] == "train":
        out["grad"] = _taken(nr.distill_grad(logits, ids, teacher, stats, _given(nr, s["g_loss"])))
    return out


def run(s):
    op = s["case"]["op"]
    if own:
        return {"verify": _own_verify, "top": _own_top, "distill": _own_distill, "train": _own_distill}[op](s)
    if op == "distill":
        return _distill(s)[0]
    return {"verify": _plain_verify, "top": _plain_top, "train": _train}[op](s)


# ------------------------------------------------------------------------------------- work and 64 bits

def work(case):
    """Each input read once and each output written once. Of a sequence's positions, those up to the first token
    that is refused (as these inputs accept them, on average); of a row whose upstream gradient is zero, the loss."""
    V, b = case["vocab"], _SIZE[case["dtype"]]
    shared = 4 * V if case["mask"] == "f32_shared" else 0
    per_row = V if case["mask"] == "u8" else 0
    if case["op"] == "verify":
        S, K = case["seqs"], case["drafts"]
        run_of = lambda n: (1 - _ACCEPTED ** n) / (1 - _ACCEPTED)  # noqa: E731
        lengths = range(K + 1) if case["ragged"] else [K]
        target = S * sum(run_of(n + 1) for n in lengths) / len(lengths)
        draft = 0 if case["lookup"] or case["temperature"] == 0.0 else S * sum(run_of(n) for n in lengths) / len(lengths)
        return {"bytes": (target + draft) * V * b + target * per_row + shared + S * (24 * K + 28), "flops": 0}
    R, k = case["rows"], case["k"]
    row = V * b + per_row + 8 * k
    if case["op"] == "train":
        return {"bytes": R * (row + 8) + R * 15 / 16 * V * b + shared, "flops": 0}
    return {"bytes": R * (row + (4 if case["op"] == "distill" else 0)) + shared, "flops": 0}


def _rows64(x, temperature, mask, first, count):
    """Rows first .. first + count - 1 of ln softmax in 64 bits, under the mask."""
    z = x[first:first + count].double() / temperature
    if mask is not None:
        m = mask[first:first + count] if mask.shape[0] > 1 or x.shape[0] == 1 else mask[0]
        z = torch.where(m != 0, z, -math.inf) if mask.dtype == torch.uint8 else z + m.double()
    return z - torch.logsumexp(z, 1, keepdim=True)


def _verify64(case, x):
    S, K, V = case["seqs"], case["drafts"], case["vocab"]
    T = case["temperature"] if case["temperature"] > 0 else 1.0
    out = {"ids": torch.full((S, K + 1), -1, dtype=torch.int32), "accepted": torch.zeros(S, dtype=torch.int32),
           "logp": torch.zeros((S, K + 1), dtype=torch.float64)}
    tokens, u = x["tokens"].tolist(), x["uniforms"].tolist()
    lengths = [K] * S if x["lengths"] is None else x["lengths"].tolist()
    logits, mask = x["logits"].view(-1, V), x["mask"]
    for i in range(S):
        lnp = _rows64(logits, T, mask, i * (K + 1), K + 1)
        lnq = None
        if x["draft"] is not None:
            m = mask
            if m is not None and m.shape[0] > 1:
                m = m.view(S, K + 1, V)[i, :K]
            lnq = _rows64(x["draft"][i], T, m, 0, K)
        a = 0
        drawn = None
        while drawn is None:
            p = lnp[a].exp()
            best = int(torch.nonzero(lnp[a] == lnp[a].max())[0])
            if a == lengths[i]:
                drawn = best if case["temperature"] == 0 else p
                break
            t = tokens[i][a]
            if case["temperature"] == 0:
                if best != t:
                    drawn = best
            elif lnq is None:
                if not u[i][a] < float(p[t]):
                    p[t] = 0.0
                    drawn = p
            else:
                q = lnq[a].exp()
                if not u[i][a] * float(q[t]) < float(p[t]):
                    r = torch.relu(p - q)
                    drawn = r if float(r.sum()) > 0 else p
            if drawn is None:
                out["ids"][i, a], out["logp"][i, a] = t, float(lnp[a][t])
                a += 1
        if not isinstance(drawn, int):
            c = torch.cumsum(drawn, 0)
            past = torch.nonzero(c > u[i][K] * float(c[-1]))
            drawn = int(past[0] if len(past) else torch.nonzero(drawn)[-1])
        out["ids"][i, a], out["logp"][i, a], out["accepted"][i] = drawn, float(lnp[a][drawn]), a
    return out


def exact(case, seed):
    """run()'s outputs in 64 bits from torch alone, a few rows at a time."""
    x = _inputs(case, seed)
    if case["op"] == "verify":
        return _verify64(case, x)
    R, k, T = case["rows"], case["k"], case["temperature"]
    many = max(1, 100_000_000 // case["vocab"])
    parts = []
    for first in range(0, R, many):
        lnp = _rows64(x["logits"], T, x["mask"], first, many)
        if case["op"] == "top":
            # (which of two tokens comes first is said by run() alone: 64 bits tell some apart that f32 does not)
            parts.append({"logp": lnp.topk(k, 1)[0]})
            continue
        ids, teacher = x["ids"][first:first + many].long(), x["teacher_logp"][first:first + many].double()
        w = torch.exp(teacher)
        if case["tail"] == "renormalize":
            w = w / w.sum(1, keepdim=True)
        on = ids >= 0
        outside = torch.ones_like(lnp, dtype=torch.bool)
        r, c = torch.nonzero(on, as_tuple=True)
        outside[r, ids[r, c]] = False
        dense = torch.zeros_like(lnp)
        dense[r, ids[r, c]] = w[r, c]
        loss = (torch.xlogy(w, w) - torch.where(on & (w > 0), w * lnp.gather(1, ids.clamp(min=0)), 0.0)).sum(1)
        total = w.sum(1)
        q = lnp.exp()
        share = torch.zeros_like(loss)
        if case["tail"] == "rest":
            left = torch.relu(1.0 - total)
            q_left = torch.where(outside, q, 0.0).sum(1)
            some = (left > 0) & (q_left > 0)
            loss = loss + torch.where(some, left * torch.log(left / q_left), 0.0)
            share = torch.where(some, left / q_left, 0.0)
            total = total + left
        part = {"loss": loss}
        if case["op"] == "train":
            d = q * (total[:, None] - torch.where(outside, share[:, None], 0.0)) - dense
            part["grad"] = d * (x["g_loss"][first:first + many].double() / T)[:, None]
        parts.append(part)
    out = {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
    return dict(out, ids=None) if case["op"] == "top" else out
